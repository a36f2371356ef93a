"""What the second launches of csrc/verify.cu may read before their own wait for the first one.

They start while the first launch of the same call still runs. A launch that has not waited is promised nothing about cached lines of memory that earlier launches
wrote, and in a replayed step the same addresses hold new numbers every time, so whatever it reads before its wait must come through EarlyTable (loads at GPU scope).
Read off the source: a race of this kind shows on no GPU at will."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "turbo_fieldfare_b200" / "csrc"
TEXT = (CSRC / "verify.cu").read_text()
TABLES = {"row_offsets", "tokens", "parents", "uniforms", "temperatures"}
# functions that the part before the wait calls, and what says in a call that it is before it
HELPERS = {"Nodes of": "kEarly", "Heat heat": "kEarly", "parent_of": "kEarly", "prob_at": ""}


def before_the_wait(kernel):
    body = TEXT[TEXT.index(f"verify_{kernel}_kernel(const"):]
    body = body[:body.index("\n}\n")]
    return body[:body.rindex("if (a.parts) pdl_wait();")]


def definition(start):
    body = TEXT[TEXT.index(start):]
    return body[:body.index("\n}")]


def test_tables_of_a_verification_are_early_ones():
    members = re.search(r"struct VerifyArgs {(.*?)\n};", TEXT, re.S).group(1)
    assert {n for names in re.findall(r"EarlyTable<\w+> ([\w, ]+);", members) for n in names.split(", ")} == TABLES
    assert not set(re.findall(r"\*\s?(\w+)", members)) & TABLES


@pytest.mark.parametrize("kernel", ["lone", "walk"])
def test_reads_before_the_wait_pass_the_l1_cache(kernel):
    part = before_the_wait(kernel)
    for table in TABLES:
        for use in re.findall(rf"\ba\.{table}\b(.{{0,12}})", part):
            assert use.startswith((".at<true>(", ".p ")), (table, use)
    # logits and probabilities: through tables of their own
    assert re.findall(r"\ba\.(?:logits|probs)\[", part) == []
    assert all("EarlyTable<T> logits{" in line for line in part.splitlines() if "a.logits" in line)
    for name, word in HELPERS.items():
        for call in re.findall(rf"\b{name}\((.*?)\)", part):
            assert word in call, (name, call)
    assert part.count("logits.template at<true>(") == part.count("logits{")
    assert "a.stats" not in part                   # the first launch's, which wait for it


def test_helpers_before_the_wait_read_by_their_argument():
    for start in ("struct Heat {", "struct Nodes {", "__device__ __forceinline__ int32_t parent_of("):
        body = definition(start)
        for table in TABLES:
            uses = re.findall(rf"\ba\.{table}\b(.{{0,12}})", body)
            assert all(u.startswith((".at<EARLY>(", ".p ", ".p)")) for u in uses), (start, table, uses)
    body = definition("__device__ __forceinline__ float prob_at(")
    assert body.count("a.probs)") == body.count("EarlyTable<") == 3 and body.count(".at<true>(at)") == 3


def test_first_launches_are_ordinary_ones():
    """They start when all before them has ended: what they are given is complete when they let the second ones start."""
    for kernel in ("verify_stats_kernel", "verify_sums_kernel"):
        assert f"{kernel}<T, CAP><<<" in TEXT and not re.search(rf"launch_pdl\w*\({kernel}", TEXT)


def test_early_tables_of_16_bits_are_loaded_at_gpu_scope():
    body = re.search(r"struct EarlyTable {(.*?)\n};", (CSRC / "tf_common.cuh").read_text(), re.S).group(1)
    assert "ld.relaxed.gpu.global.u16" in body
