// kda_seq.cu — the KDA gated delta rule over whole prompts and for one token
// of each sequence (k3xb_kda_prefill, k3xb_kda_step). Per head, with the
// state S [value][key], a = exp(log_decay) and b = beta:
//
//   S <- S diag(a);  delta = b (v - S k);  S <- S + delta k^T;  o = S q
//
// (official_kda.cpp:319-369 token by token, on packed ragged sequences.) The
// sums here are float sums in an order of their own, so results agree with
// k3xb_kda_tree to float tolerance, not bit for bit.
#include <cuda_bf16.h>

#include <atomic>

#include "common.cuh"
#include "kernels.cuh"
#include "profile.cuh"

namespace k3xb {

namespace {

struct SeqArgs {
    const void *q, *k, *v;
    uint64_t row_stride;       // elements between two tokens' rows of q, k and v
    const float *log_decay, *beta;
    const uint32_t* offsets;   // [S + 1] token ranges; NULL: sequence s is token s
    const int32_t* slots;      // state of sequence s, below `states` (NULL: s; negative: idle)
    uint32_t tokens, heads, states;
    const float* state;        // NULL: zeros
    float* state_out;          // NULL: not kept; may be `state`
    void* out;
    int32_t* status;
};

template <typename E>
__device__ __forceinline__ float to_f(E x) {
    if constexpr (sizeof(E) == 4) return x;
    else return __bfloat162float(x);
}

// Four consecutive values as floats; VEC: the address is a multiple of four
// elements.
template <typename E, bool VEC>
__device__ __forceinline__ float4 load4(const E* p) {
    if constexpr (!VEC) {
        return make_float4(to_f(p[0]), to_f(p[1]), to_f(p[2]), to_f(p[3]));
    } else if constexpr (sizeof(E) == 4) {
        return *reinterpret_cast<const float4*>(p);
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u),
                           __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    }
}

template <typename E>
__device__ __forceinline__ void store1(void* p, size_t i, float x) {
    if constexpr (sizeof(E) == 4) static_cast<float*>(p)[i] = x;
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

// The token range of a sequence; false (and the status word set) where the
// offsets are not a range within the tokens.
__device__ __forceinline__ bool token_range(const SeqArgs& a, uint32_t s, uint32_t& t0, uint32_t& t1) {
    if (!a.offsets) {
        t0 = s;
        t1 = s + 1;
        return true;
    }
    t0 = a.offsets[s];
    t1 = a.offsets[s + 1];
    if (t0 <= t1 && t1 <= a.tokens) return true;
    if (threadIdx.x == 0) atomicExch(a.status, K3XB_INVALID_EXTENT);
    return false;
}

// The rule token by token. A CTA owns kRows value rows of one head of one
// sequence; eight lanes share a row (D / 8 keys each, in 16-byte pieces 128
// bytes apart), so a row's two sums take three shuffles. Both are taken in
// one pass over the row: o = (S diag(a)) q + delta (k . q).
constexpr int kRows = 32, kSeqThreads = 128, kRowSets = kRows / (kSeqThreads / 8);

template <int D, typename E, bool VEC>
__global__ void __launch_bounds__(kSeqThreads) kda_recurrent_kernel(const SeqArgs a) {
    constexpr int G = D / 32;   // 16-byte pieces of a row per lane
    const uint32_t s = blockIdx.y, h = blockIdx.x / (D / kRows), r0 = (blockIdx.x % (D / kRows)) * kRows;
    const uint32_t lane = threadIdx.x % 32, sub = lane % 8;
    const uint32_t row = r0 + (threadIdx.x / 32) * 4 + lane / 8;
    const uint32_t P = a.heads * D;
    const E* q = static_cast<const E*>(a.q);
    const E* k = static_cast<const E*>(a.k);
    const E* v = static_cast<const E*>(a.v);
    uint32_t t0, t1;
    if (!token_range(a, s, t0, t1)) return;
    const int32_t slot = a.slots ? a.slots[s] : static_cast<int32_t>(s);
    const bool outside = slot >= 0 && static_cast<uint32_t>(slot) >= a.states;
    if (outside && threadIdx.x == 0) atomicExch(a.status, K3XB_INVALID_EXTENT);
    if (slot < 0 || outside) {   // idle: zero rows, no state
        for (uint32_t t = t0; t < t1; ++t)
            for (uint32_t r = threadIdx.x; r < static_cast<uint32_t>(kRows); r += kSeqThreads)
                store1<E>(a.out, static_cast<size_t>(t) * P + h * D + r0 + r, 0.0f);
        return;
    }
    const size_t base = (static_cast<size_t>(slot) * a.heads + h) * D * D;
    float S[kRowSets][G][4];
#pragma unroll
    for (int i = 0; i < kRowSets; ++i)
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float4 x = a.state ? *reinterpret_cast<const float4*>(a.state + base + (row + 16 * i) * D + g * 32 + sub * 4)
                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            S[i][g][0] = x.x; S[i][g][1] = x.y; S[i][g][2] = x.z; S[i][g][3] = x.w;
        }
    for (uint32_t t = t0; t < t1; ++t) {
        const size_t at = static_cast<size_t>(t) * a.row_stride + h * D;
        float al[G][4], kk[G][4], qq[G][4];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float4 x = load4<float, VEC>(a.log_decay + static_cast<size_t>(t) * P + h * D + g * 32 + sub * 4);
            const float4 y = load4<E, VEC>(k + at + g * 32 + sub * 4), z = load4<E, VEC>(q + at + g * 32 + sub * 4);
            al[g][0] = expf(x.x); al[g][1] = expf(x.y); al[g][2] = expf(x.z); al[g][3] = expf(x.w);
            kk[g][0] = y.x; kk[g][1] = y.y; kk[g][2] = y.z; kk[g][3] = y.w;
            qq[g][0] = z.x; qq[g][1] = z.y; qq[g][2] = z.z; qq[g][3] = z.w;
        }
        const float be = a.beta[static_cast<size_t>(t) * a.heads + h];
        float vv[kRowSets], pred[kRowSets], o[kRowSets], kq = 0.0f;
#pragma unroll
        for (int i = 0; i < kRowSets; ++i) {
            vv[i] = to_f(v[at + row + 16 * i]);
            pred[i] = o[i] = 0.0f;
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                kq = fmaf(kk[g][j], qq[g][j], kq);
#pragma unroll
                for (int i = 0; i < kRowSets; ++i) {
                    S[i][g][j] *= al[g][j];
                    pred[i] = fmaf(S[i][g][j], kk[g][j], pred[i]);
                    o[i] = fmaf(S[i][g][j], qq[g][j], o[i]);
                }
            }
#pragma unroll
        for (int m = 4; m > 0; m >>= 1) {
            kq += __shfl_xor_sync(0xffffffffu, kq, m);
#pragma unroll
            for (int i = 0; i < kRowSets; ++i) {
                pred[i] += __shfl_xor_sync(0xffffffffu, pred[i], m);
                o[i] += __shfl_xor_sync(0xffffffffu, o[i], m);
            }
        }
#pragma unroll
        for (int i = 0; i < kRowSets; ++i) {
            const float delta = (vv[i] - pred[i]) * be;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) S[i][g][j] = fmaf(delta, kk[g][j], S[i][g][j]);
            if (sub == 0) store1<E>(a.out, static_cast<size_t>(t) * P + h * D + row + 16 * i, fmaf(delta, kq, o[i]));
        }
    }
    if (!a.state_out) return;
#pragma unroll
    for (int i = 0; i < kRowSets; ++i)
#pragma unroll
        for (int g = 0; g < G; ++g)
            *reinterpret_cast<float4*>(a.state_out + base + (row + 16 * i) * D + g * 32 + sub * 4) =
                make_float4(S[i][g][0], S[i][g][1], S[i][g][2], S[i][g][3]);
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <int D, typename E>
int launch_recurrent(k3xb_ctx* ctx, const SeqArgs& a, uint32_t sequences) {
    // 16-byte (f32) or 8-byte (bf16) loads where every row allows them
    const bool vec = aligned(a.q, 4 * sizeof(E)) && aligned(a.k, 4 * sizeof(E)) && a.row_stride % 4 == 0 &&
                     aligned(a.log_decay, 16);
    const dim3 grid(a.heads * (D / kRows), sequences);
    if (vec) kda_recurrent_kernel<D, E, true><<<grid, kSeqThreads, 0, ctx->stream>>>(a);
    else kda_recurrent_kernel<D, E, false><<<grid, kSeqThreads, 0, ctx->stream>>>(a);
    K3XB_LAUNCHED(ctx);
    return K3XB_OK;
}

template <typename E>
int launch_seq(k3xb_ctx* ctx, const SeqArgs& a, uint32_t sequences, uint32_t d) {
    switch (d) {
        case 32: return launch_recurrent<32, E>(ctx, a, sequences);
        case 64: return launch_recurrent<64, E>(ctx, a, sequences);
        default: return launch_recurrent<128, E>(ctx, a, sequences);
    }
}

// Checks shared by the two entry points; fills the fields that they share.
int check_seq(k3xb_ctx* ctx, const char* what, int32_t type, uint32_t sequences, uint32_t heads, uint32_t d,
              const SeqArgs& a) {
    const std::string w(what);
    if (type != K3XB_TYPE_F32 && type != K3XB_TYPE_BF16) return fail(ctx, K3XB_INVALID_EXTENT, w + ": type must be f32 or bf16");
    if (d != 32 && d != 64 && d != 128) return fail(ctx, K3XB_INVALID_EXTENT, w + ": head_dim must be 32, 64 or 128");
    // a grid holds 65535 sequences and 2^31 - 1 row groups of heads
    if (!sequences || sequences > 65535 || !heads || heads > (1u << 20))
        return fail(ctx, K3XB_INVALID_EXTENT, w + ": 1 to 65535 sequences, 1 to 2^20 heads");
    if (a.row_stride < static_cast<uint64_t>(heads) * d)
        return fail(ctx, K3XB_INVALID_EXTENT, w + ": row_stride is less than heads * head_dim");
    const size_t el = type == K3XB_TYPE_F32 ? 4 : 2;
    if (!aligned(a.q, el) || !aligned(a.k, el) || !aligned(a.v, el) || !aligned(a.out, el) || !aligned(a.log_decay, 4) ||
        !aligned(a.beta, 4))
        return fail(ctx, K3XB_INVALID_EXTENT, w + ": an array is not aligned to its type");
    if (!aligned(a.state, 16) || !aligned(a.state_out, 16))
        return fail(ctx, K3XB_INVALID_EXTENT, w + ": states must be 16-byte aligned");
    return K3XB_OK;
}

}  // namespace
}  // namespace k3xb

using namespace k3xb;

extern "C" {

int k3xb_kda_prefill(k3xb_ctx* ctx, const void* q, const void* k, const void* v, uint64_t row_stride, int32_t type,
                     const float* log_decay, const float* beta, const uint32_t* offsets, uint32_t sequences,
                     uint32_t tokens, uint32_t heads, uint32_t head_dim, const float* state, float* state_out, void* out) {
    K3XB_ENTER(ctx);
    if (!offsets || (tokens && (!q || !k || !v || !log_decay || !beta || !out)))
        return fail(ctx, K3XB_INVALID_EXTENT, "kda_prefill arguments");
    if (!row_stride) row_stride = static_cast<uint64_t>(heads) * head_dim;
    const SeqArgs a{q, k, v, row_stride, log_decay, beta, offsets, nullptr, tokens, heads, sequences, state, state_out, out, ctx->status_word};
    if (const int st = check_seq(ctx, "kda_prefill", type, sequences, heads, head_dim, a)) return st;
    PhaseScope ph(ctx, K3XB_PHASE_KDA_RECURRENCE);
    ++ctx->stats.kda_calls;
    return type == K3XB_TYPE_F32 ? launch_seq<float>(ctx, a, sequences, head_dim)
                                 : launch_seq<__nv_bfloat16>(ctx, a, sequences, head_dim);
}

int k3xb_kda_step(k3xb_ctx* ctx, const void* q, const void* k, const void* v, uint64_t row_stride, int32_t type,
                  const float* log_decay, const float* beta, uint32_t sequences, uint32_t heads, uint32_t head_dim,
                  const int32_t* slots, uint32_t states, float* state, void* out) {
    K3XB_ENTER(ctx);
    if (!q || !k || !v || !log_decay || !beta || !state || !out)
        return fail(ctx, K3XB_INVALID_EXTENT, "kda_step arguments");
    if (!slots && states < sequences) return fail(ctx, K3XB_INVALID_EXTENT, "kda_step: fewer states than sequences");
    if (!row_stride) row_stride = static_cast<uint64_t>(heads) * head_dim;
    const SeqArgs a{q, k, v, row_stride, log_decay, beta, nullptr, slots, sequences, heads, states, state, state, out, ctx->status_word};
    if (const int st = check_seq(ctx, "kda_step", type, sequences, heads, head_dim, a)) return st;
    PhaseScope ph(ctx, K3XB_PHASE_KDA_RECURRENCE);
    ++ctx->stats.kda_calls;
    return type == K3XB_TYPE_F32 ? launch_seq<float>(ctx, a, sequences, head_dim)
                                 : launch_seq<__nv_bfloat16>(ctx, a, sequences, head_dim);
}

}  // extern "C"
