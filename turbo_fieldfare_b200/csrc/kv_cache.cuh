// The quantised, paged key/value cache as kernels see it: checks of the caller's descriptors and addresses of tokens.
#pragma once

#include "tf_common.cuh"

namespace tf {

constexpr uint32_t kErrKvPage = 0x7F000051u;      // a token's page is outside the table or the planes
constexpr uint32_t kErrKvOffsets = 0x7F000052u;   // row offsets descend or pass the rows

struct KvPlanes {
    uint8_t* codes;
    uint16_t* scales;
    uint16_t* biases;
};

// Descriptor and shape checks of tf_kv_cache and tf_kv_batch; both report through the context like every entry point.
tf_status check_kv_cache(tf_context* ctx, const char* name, const tf_kv_cache* c);
tf_status check_kv_batch(tf_context* ctx, const char* name, const tf_kv_batch* b);

// Makes the context's device current for a call and puts the caller's back.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        if (cudaGetDevice(&before_) == cudaSuccess && before_ != device) changed_ = cudaSetDevice(device) == cudaSuccess;
    }
    ~DeviceScope() { if (changed_) cudaSetDevice(before_); }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
private:
    int before_ = 0;
    bool changed_ = false;
};

inline uint32_t log2_of(uint32_t power) {
    uint32_t n = 0;
    while ((1u << n) < power) ++n;
    return n;
}

// WORDS 32-bit words at p, which is aligned to them (to 16 bytes from four words on).
template <int WORDS>
__device__ __forceinline__ void load_words(uint32_t (&w)[WORDS], const void* p) {
    if constexpr (WORDS == 1) w[0] = *static_cast<const uint32_t*>(p);
    else if constexpr (WORDS == 2) { const uint2 t = *static_cast<const uint2*>(p); w[0] = t.x; w[1] = t.y; }
    else {
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) {
            const uint4 t = static_cast<const uint4*>(p)[i];
            w[4 * i] = t.x; w[4 * i + 1] = t.y; w[4 * i + 2] = t.z; w[4 * i + 3] = t.w;
        }
    }
}
// Page of a token of sequence `seq`, or -1: outside the table or the planes.
struct KvTable {
    const int32_t* table;
    uint32_t stride, pages, page_log2;
    __host__ __device__ __forceinline__ int32_t page(uint32_t seq, int64_t token) const {
        if (token < 0 || (token >> page_log2) >= (int64_t)stride) return -1;
        const int32_t p = table[(size_t)seq * stride + (size_t)(token >> page_log2)];
        return p >= 0 && (uint32_t)p < pages ? p : -1;
    }
};

}  // namespace tf
