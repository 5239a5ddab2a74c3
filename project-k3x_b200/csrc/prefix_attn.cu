// prefix_attn.cu — attention of draft nodes over a prefix that all sequences
// share, each sequence's own committed rows, and the node's ancestors among
// the draft rows (k3xb_prefix_attention). Per sequence s, node n and head h,
// with the key of a position its own per-head part and, behind it, a part
// that the heads share (model.cpp:785-810 without the gate and o_proj):
//
//   p = softmax over the visible positions of scale * q . [k, extra]
//   out = sum p v,   lse = log sum exp(scale * q . [k, extra])
//
// Visible: every prefix row, own rows below suffix_len[s], and the own rows
// suffix_len[s] + m for the nodes m on the path from n to its root.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "common.cuh"
#include "kernels.cuh"
#include "prefix_attn.cuh"
#include "profile.cuh"

namespace k3xb {

namespace {

constexpr uint32_t kMaxDim = 256;

template <typename E>
__device__ __forceinline__ float to_f(E x) {
    if constexpr (std::is_same_v<E, float>) return x;
    else if constexpr (std::is_same_v<E, __half>) return __half2float(x);
    else return __bfloat162float(x);
}

template <typename E>
__device__ __forceinline__ E from_f(float x) {
    if constexpr (std::is_same_v<E, float>) return x;
    else if constexpr (std::is_same_v<E, __half>) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

// The general form: one CTA per (sequence, node, head), its four warps take
// positions in turn, each with a running maximum and sum; a lane holds every
// 32nd query and value element.
constexpr int kRowThreads = 128, kPer = kMaxDim / 32;

template <typename E>
__global__ void __launch_bounds__(kRowThreads) attend_rows_kernel(const __grid_constant__ AttnArgs a) {
    const uint32_t h = blockIdx.x, n = blockIdx.y, s = blockIdx.z, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t kvh = h / (a.heads / a.kv_heads);
    const size_t row = (static_cast<size_t>(s) * a.N + n) * a.heads + h;
    __shared__ float sm_m[4], sm_l[4], sm_o[4][kMaxDim];
    const int32_t len = own_rows(a, s);
    const E* q = static_cast<const E*>(a.q) + (static_cast<size_t>(s) * a.N + n) * a.q_row + static_cast<size_t>(h) * (a.main + a.extra);
    float qv[kPer], o[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const uint32_t c = lane + 32 * i;
        qv[i] = c < a.main + a.extra ? to_f(q[c]) * a.scale : 0.0f;
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    auto visit = [&](const KvSource& src, uint32_t seq, uint64_t p) {
        const E* k = static_cast<const E*>(src.k) + seq * src.k_seq + p * src.k_row + kvh * src.k_head;
        const E* v = static_cast<const E*>(src.v) + seq * src.v_seq + p * src.v_row + kvh * src.v_head;
        const E* e = static_cast<const E*>(src.extra) + seq * src.extra_seq + p * src.extra_row;
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t c = lane + 32 * i;
            if (c < a.main) x = fmaf(qv[i], to_f(k[c]), x);
            else if (c < a.main + a.extra) x = fmaf(qv[i], to_f(e[c - a.main]), x);
        }
        x = warp_sum(x);
        const float top = fmaxf(m, x);
        const float base = top == -INFINITY ? 0.0f : top;
        const float keep = expf(m - base), p_here = expf(x - base);
        l = fmaf(l, keep, p_here);
        m = isnan(x) ? x : top;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t c = lane + 32 * i;
            if (c < a.value) o[i] = fmaf(o[i], keep, p_here * to_f(v[c]));
        }
    };
    if (len >= 0) {
        for (uint32_t p = warp; p < a.prefix_len; p += 4) visit(a.prefix, 0, p);
        for (uint32_t p = warp; p < static_cast<uint32_t>(len); p += 4) visit(a.suffix, s, p);
        for (uint32_t j = warp; j <= n; j += 4)
            if (a.ancestors[n] >> j & 1u) visit(a.suffix, s, static_cast<uint64_t>(len) + j);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) sm_o[warp][lane + 32 * i] = o[i];
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
    __syncthreads();
    float top = -INFINITY, total = 0.0f, w[4];
    for (int i = 0; i < 4; ++i) top = isnan(sm_m[i]) || isnan(top) ? NAN : fmaxf(top, sm_m[i]);
    const float base = top == -INFINITY ? 0.0f : top;
    for (int i = 0; i < 4; ++i) {
        w[i] = expf(sm_m[i] - base);
        total = fmaf(sm_l[i], w[i], total);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;   // nothing visible: a zero row
    for (uint32_t c = threadIdx.x; c < a.value; c += kRowThreads) {
        float x = 0.0f;
        for (int i = 0; i < 4; ++i) x = fmaf(sm_o[i][c], w[i], x);
        static_cast<E*>(a.out)[row * a.value + c] = from_f<E>(x * inv);
    }
    if (a.lse && threadIdx.x == 0) a.lse[row] = total == 0.0f ? -INFINITY : top + logf(total);
}

template <typename E>
int launch_rows(k3xb_ctx* ctx, const AttnArgs& a) {
    attend_rows_kernel<E><<<dim3(a.heads, a.N, a.S), kRowThreads, 0, ctx->stream>>>(a);
    K3XB_LAUNCHED(ctx);
    return K3XB_OK;
}

// A source's strides; all zero: packed [seq][row][head][dim]. A stride over a
// single row, head or sequence is never used, so it gets the packed value.
KvSource source_of(const k3xb_kv_rows& r, const AttnArgs& a, uint32_t sequences) {
    KvSource s{r.k, r.v, r.extra, r.k_row, r.k_head, r.k_seq, r.v_row, r.v_head, r.v_seq, r.extra_row, r.extra_seq};
    const bool packed = !(r.k_row | r.k_head | r.k_seq | r.v_row | r.v_head | r.v_seq | r.extra_row | r.extra_seq);
    if (packed || a.kv_heads == 1) {
        s.k_head = a.main;
        s.v_head = a.value;
    }
    if (packed || r.rows == 1) {
        s.k_row = static_cast<uint64_t>(a.kv_heads) * a.main;
        s.v_row = static_cast<uint64_t>(a.kv_heads) * a.value;
        s.extra_row = a.extra;
    }
    if (packed || sequences == 1) {
        s.k_seq = r.rows * s.k_row;
        s.v_seq = r.rows * s.v_row;
        s.extra_seq = r.rows * s.extra_row;
    }
    return s;
}

}  // namespace
}  // namespace k3xb

using namespace k3xb;

extern "C" int k3xb_prefix_attention(k3xb_ctx* ctx, const k3xb_prefix_attention_io* io) {
    K3XB_ENTER(ctx);
    auto bad = [&](const char* why) { return fail(ctx, K3XB_INVALID_EXTENT, std::string("prefix_attention: ") + why); };
    if (!io || !io->parent || !io->q || !io->suffix_len || !io->out || !io->suffix.k || !io->suffix.v)
        return bad("arguments");
    if (!io->sequences || !io->nodes || io->nodes > kMaxNodes || io->sequences > 65535)
        return bad("1 to 65535 sequences, 1 to 64 nodes");
    if (!io->heads || io->heads > 65535 || !io->kv_heads || io->heads % io->kv_heads)
        return bad("heads must be a multiple of kv_heads");
    if (!io->main_dim || !io->value_dim || io->main_dim + static_cast<uint64_t>(io->extra_dim) > kMaxDim || io->value_dim > kMaxDim)
        return bad("main_dim + extra_dim and value_dim must be 1 to 256");
    if (io->prefix.rows && (!io->prefix.k || !io->prefix.v)) return bad("the prefix has rows but no arrays");
    if (io->extra_dim && ((io->prefix.rows && !io->prefix.extra) || !io->suffix.extra)) return bad("extra_dim without extra rows");
    if (io->prefix.rows > 0x7fffffffu || io->suffix.rows > 0x7fffffffu || io->suffix.rows < io->nodes)
        return bad("the suffix holds fewer rows than nodes, or a row count passes 2^31");
    if (!std::isfinite(io->scale)) return bad("scale must be finite");
    if (io->type != K3XB_TYPE_F32 && io->type != K3XB_TYPE_BF16 && io->type != K3XB_TYPE_F16) return bad("type must be f32, bf16 or f16");
    const size_t el = io->type == K3XB_TYPE_F32 ? 4 : 2;
    auto off = [&](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
    bool odd = off(io->q, el) || off(io->out, el) || off(io->lse, 4) || off(io->suffix_len, 4);
    for (const k3xb_kv_rows* x : {&io->prefix, &io->suffix})
        odd = odd || (x->rows && (off(x->k, el) || off(x->v, el) || (io->extra_dim && off(x->extra, el))));
    if (odd) return bad("an array is not aligned to its type");
    AttnArgs a{};
    a.S = io->sequences;
    a.N = io->nodes;
    a.heads = io->heads;
    a.kv_heads = io->kv_heads;
    a.main = io->main_dim;
    a.extra = io->extra_dim;
    a.value = io->value_dim;
    a.scale = io->scale;
    a.q_row = io->q_row ? io->q_row : static_cast<uint64_t>(a.heads) * (a.main + a.extra);
    a.prefix_len = io->prefix.rows;
    a.capacity = io->suffix.rows;
    a.prefix = source_of(io->prefix, a, 1);
    a.suffix = source_of(io->suffix, a, a.S);
    a.suffix_len = io->suffix_len;
    a.q = io->q;
    a.out = io->out;
    a.lse = io->lse;
    a.status = ctx->status_word;
    for (uint32_t n = 0; n < a.N; ++n) {
        const int32_t p = io->parent[n];
        if (p < -1 || p >= static_cast<int32_t>(n)) return bad("parent[n] must be -1 or < n");
        a.ancestors[n] = (p >= 0 ? a.ancestors[p] : 0) | (1ull << n);
    }
    PhaseScope ph(ctx, K3XB_PHASE_ATTENTION);
    if (attend_tc_takes(a, io->type)) return launch_attend_tc(ctx, a, io->type == K3XB_TYPE_BF16);
    switch (io->type) {
        case K3XB_TYPE_F32: return launch_rows<float>(ctx, a);
        case K3XB_TYPE_BF16: return launch_rows<__nv_bfloat16>(ctx, a);
        default: return launch_rows<__half>(ctx, a);
    }
}
