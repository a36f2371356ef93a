"""Numbers that do not fit what the library takes are refused, where ctypes would cut them to 32 bits."""
import pytest
import torch

I32 = dict(dtype=torch.int32)
BEYOND = [-1, 0, 1 << 31, (1 << 32) + 16]


@pytest.mark.parametrize("page_size", BEYOND)
def test_pages_of_other_sizes_are_refused(page_size):
    from turbo_fieldfare_b200 import drafts as dr
    with pytest.raises(ValueError, match="page_size"):
        dr.KVPages(torch.zeros(2, 3, **I32), torch.zeros(2, **I32), torch.zeros(9, **I32), torch.zeros(1, **I32), page_size)
    with pytest.raises(ValueError, match="page_size"):
        dr.KVPages.allocate(2, 3, 9, page_size, device="cpu")


@pytest.mark.parametrize("number", BEYOND)
@pytest.mark.parametrize("which", ["rows", "vocab"])
def test_workspaces_of_other_sizes_are_refused(number, which):
    from turbo_fieldfare_b200 import drafts as dr
    with pytest.raises(ValueError, match=which):
        dr.VerificationWorkspace(None, **{"rows": 4, "vocab": 100, which: number})


def test_the_ends_are_taken():
    from turbo_fieldfare_b200 import drafts as dr
    assert dr.KVPages.allocate(2, 3, 9, 65536, device="cpu")._c.page_size == 65536
    asked = []
    lib = type("Library", (), {"tf_verify_workspace_create": lambda self, *a: asked.append(a[1:3]) or 0, "tf_verify_workspace_destroy": lambda self, h: None})()
    context = type("Context", (), {"lib": lib, "handle": None, "check": lambda self, status: None})()
    dr.VerificationWorkspace(context, 1, (1 << 31) - 1)
    assert asked == [(1, (1 << 31) - 1)]
