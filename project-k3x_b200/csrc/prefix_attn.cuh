// prefix_attn.cuh — what the forms of the shared-prefix attention have in
// common (prefix_attn.cu, prefix_attn_tc.cu).
#pragma once

#include "common.cuh"

namespace k3xb {

constexpr uint32_t kMaxNodes = 64;

// One source of key and value rows; strides in elements.
struct KvSource {
    const void *k, *v, *extra;
    uint64_t k_row, k_head, k_seq, v_row, v_head, v_seq, extra_row, extra_seq;
};

struct AttnArgs {
    uint32_t S, N, heads, kv_heads, main, extra, value;
    float scale;
    uint64_t q_row;
    uint32_t prefix_len, capacity;
    KvSource prefix, suffix;
    const int32_t* suffix_len;
    const void* q;
    void* out;
    float* lse;
    int32_t* status;
    uint64_t ancestors[kMaxNodes];   // bit m: node m is n or on n's path to its root
};

// A sequence's committed rows: -1 where it is idle. A length that the cache
// cannot hold together with the draft rows is an error and counts as idle.
__device__ __forceinline__ int32_t own_rows(const AttnArgs& a, uint32_t s) {
    const int32_t len = a.suffix_len[s];
    if (len < 0) return -1;
    if (static_cast<uint64_t>(len) + a.N <= a.capacity) return len;
    if (threadIdx.x == 0) atomicExch(a.status, K3XB_INVALID_EXTENT);
    return -1;
}

// The tensor-core form: whether it takes a call, and the call.
bool attend_tc_takes(const AttnArgs& a, int32_t type);
int launch_attend_tc(k3xb_ctx* ctx, const AttnArgs& a, bool bf16);

}  // namespace k3xb
