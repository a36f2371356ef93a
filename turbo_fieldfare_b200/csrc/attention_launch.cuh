// What the entry points of the attention and its kernels share on the host.
#pragma once

#include "attention_plan.cuh"

struct tf_attention_workspace {
    int device = 0;
    uint32_t head_dim = 0, row_capacity = 0, max_workers = 0;   // rows of one partial slot times blocks
    uint64_t bytes = 0;
    float* partial = nullptr;      // [2 x workers][parts of a head][rows][part + 2], in the kernel for many rows [2 x blocks][rows][part + 3]
    void* info = nullptr;          // [max_workers] ShareInfo
    uint32_t* tickets = nullptr;   // [3 levels][2 slots x 2 parts x max_workers], zero between calls
};

namespace tf {

// The launches for one head size and code width, instantiated in attention_d*.cu (a file each, so that they compile side by side).
template <int D, int BITS>
tf_status attend(tf_context* ctx, cudaStream_t st, const AttnArgs& a, const tf_attention_workspace* ws, bool bf16);

}  // namespace tf
