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
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kernels.cuh"
#include "profile.cuh"
#include "tc.cuh"

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
    uint32_t from, below;      // sequences that a kernel takes: from <= tokens < below
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

// The token range of a sequence; false where the kernel does not take its
// length, and (with the status word set) where the offsets are no range
// within the tokens.
__device__ __forceinline__ bool token_range(const SeqArgs& a, uint32_t s, uint32_t& t0, uint32_t& t1) {
    if (!a.offsets) {
        t0 = s;
        t1 = s + 1;
        return true;
    }
    t0 = a.offsets[s];
    t1 = a.offsets[s + 1];
    if (t0 <= t1 && t1 <= a.tokens) return t1 - t0 >= a.from && t1 - t0 < a.below;
    if (threadIdx.x == 0) atomicExch(a.status, K3XB_INVALID_EXTENT);
    return false;
}

// The rule token by token. A CTA owns kRows value rows of one head of one
// sequence; eight lanes share a row (D / 8 keys each, in 16-byte pieces 128
// bytes apart), so a row's two sums take three shuffles. Both are taken in
// one pass over the row: o = (S diag(a)) q + delta (k . q).
//
// One token of each sequence is bound by its state, read and written once as a
// stream (one B200, 32 heads of 128): 64 sequences 45 us = 6.1 TB/s, 312 of a
// pool of 400 209 us = 6.3 TB/s, 0.93 and 0.97 of the measured copy rate. Two
// warps of 256 bytes in flight a thread beat four of 128 (54 and 241 us) and
// eight of 64 (66 and 292 us); without the streaming hint 49 and 202 us.
constexpr int kRows = 32, kSeqThreads = 64, kSetRows = kSeqThreads / 8, kRowSets = kRows / kSetRows;

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
    asm volatile("griddepcontrol.launch_dependents;");   // chunks of other sequences may start
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
            const float4 x = a.state ? __ldcs(reinterpret_cast<const float4*>(a.state + base + (row + kSetRows * i) * D + g * 32 + sub * 4))
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
            vv[i] = to_f(v[at + row + kSetRows * i]);
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
            if (sub == 0) store1<E>(a.out, static_cast<size_t>(t) * P + h * D + row + kSetRows * i, fmaf(delta, kq, o[i]));
        }
    }
    if (!a.state_out) return;
#pragma unroll
    for (int i = 0; i < kRowSets; ++i)
#pragma unroll
        for (int g = 0; g < G; ++g)
            __stcs(reinterpret_cast<float4*>(a.state_out + base + (row + kSetRows * i) * D + g * 32 + sub * 4),
                   make_float4(S[i][g][0], S[i][g][1], S[i][g][2], S[i][g][3]));
}

// ---- chunks of 16 tokens ------------------------------------------------------
//
// Within a chunk, with p_i the decay from the chunk's start to token i, e_j
// the decay from token j to its end and D_ij the decay from j to i:
//
//   A_ij = k_i . (D_ij k_j)  (j < i),   P_ij = q_i . (D_ij k_j)  (j <= i)
//   T = (1 + diag(b) A)^-1 diag(b),   W = T (p K)
//   U = T V - W S0^T,   O = (p Q) S0^T + P U
//   S = S0 diag(p_15) + U^T (e K)
//
// which is the rule's own sums in another order. Decays are products of the
// tokens' own, never quotients: for a pair (i, j) D_ij is split where the
// halves of the smallest aligned block that holds both meet, D_ij = (decay
// from there to i) (decay from j to there). Four block sizes (16, 8, 4, 2)
// make four products of 8 upper by 8 lower rows, of which a token is in one
// side each.
//
// Two kernels. chunk_operands_kernel makes every chunk's operands, all chunks
// and heads side by side. chunk_scan_kernel goes along the sequences: a warp
// owns 16 value rows and keeps S in registers, in the accumulator layout of
// mma.m16n8k16, which is also the layout its left operand is read in: S, V
// and U go from accumulators straight into the next product, without shared
// memory. (Both in one kernel, with producer warps beside the scan's, the
// producers took 7900 cycles a chunk and the scan 2700, and half the GPU was
// idle at one sequence: 8192 tokens of 32 heads 2.48 ms, apart 1.23.) A
// chunk's operands cross memory once, 1.3 times the bytes of its inputs, as an
// image of the shared memory that the scan copies them to.
//
// Measured (one B200): 8192 tokens, 32 heads of 128, f32: operands 266 us (3.6
// TB/s, the issue slots 53% busy: ~2250 instructions a warp and chunk, most
// of them splits), scan 563 us, 1.1 us a chunk: a chain of products (96 MMAs a
// warp), row maxima and splits from one chunk's state to the next's.
//
// Terms. An f16 operand is two terms of a power-of-two multiple (hi + lo: 22
// bits down to 2^-17 of the multiple's end, 2^-39 of it below) and a product hi hi +
// hi lo + lo hi in f32 accumulators: float accuracy at three times the MMA
// work, where plain f16 or bf16 operands would leave the f32 state with 3
// digits. The long products are of that kind (S by value rows, W and p Q by
// tokens, e K and U by value rows; small products summed apart, since a
// tensor core truncates each sum). T, V, P and U, whose elements may be of any
// size beside each other, are three bf16 terms (24 bits at any size) in their
// short products (U two in P U for bf16 outputs).
//
// Tokens of unlike size. What one token may lose to another's size is taken
// out beforehand, by powers of two and thus exactly: token j's key times
// 2^(x + dx_j), so that every token's largest is alike (up to 2^40 apart), its query
// times 2^z_j, its decay times 2^-e_j, so that its largest channel is 1/2 to 1 (down to
// 2^-80 from the chunk's start). With E_j the sum of the e up to j the rule holds for
//   b_j 2^(-2 dx_j),  v_j 2^(dx_j - E_j + c),  u_j 2^(-dx_j - E_j + c),  o_j 2^(z_j - E_j)
// in place of b, v, u and o: the powers go to T's columns, P's rows and
// the rows' factors fw and fq. So an output is off by float roundings of its
// own query times its own row's content, and no later token changes it.
//
// Infinities and NaN become NaN where the rule takes them: in their token's
// outputs and, but for a query's, in all later ones (a value's or a state's in its own row).

constexpr int kChunk = 16, kStages = 3;
constexpr uint32_t kShort = 9;   // sequences below go token by token where there are some
constexpr int kKeySpread = 40, kLeastDecay = -80, kMostDecay = 100;
// Operands held at a time: longer batches go in segments of chunks.
constexpr size_t kOperandBytes = size_t(1) << 30;

template <int D>
struct __align__(128) ChunkStage {
    // f16 hi, lo; [tok][channel] rows of D + 8 values: ldmatrix reads 8 of them
    // without a bank conflict; 16 + 8 likewise
    __half w[2][kChunk][D + 8], q[2][kChunk][D + 8], ke[2][kChunk][D + 8];   // W, p Q, e K
    __nv_bfloat16 t[3][kChunk][kChunk + 8], p[3][kChunk][kChunk + 8];        // three bf16 terms
    float total[D];                 // p_15
    float fw[kChunk], fq[kChunk];   // what a token's products with w and q are still to be multiplied by
    int exp;                        // U^T (e K) is to be multiplied by 2^exp
};

template <int D>
struct __align__(16) ChunkScratch {
    __half k[2][kChunk][D + 8];           // p K
    // per block size: 8 upper rows of k, 8 of q, 8 lower rows of k
    __half level[4][2][24][D + 8];
    float T[kChunk][kChunk];
    float At[kChunk][kChunk];             // At[j][i] = A_ij
    float P[kChunk][kChunk];
    float diag[D / 32][kChunk];           // q_i . k_i by warp
    float beta[kChunk], bs[kChunk];       // as they are, and as the evened tokens have them
    uint32_t top[3][D / 32][kChunk / 2];  // largest |k|, |q|, decay of each token by warp: two tokens' upper halves
    // powers of two by token: of k, q and the decay (each warp's own); of T's columns, P's rows and its diagonal
    float sk[D / 32][kChunk], sq[D / 32][kChunk], sa[D / 32][kChunk], ft[kChunk], fp[kChunk], fd[kChunk];
    float fx;                             // of all keys' products
    int wexp;                             // of the products with W, besides its rows' own
};

// The chunks of a call lie in slots: sequence s from offsets[s] / 16 + s on
// (a sequence of n tokens ends before the next one's: n / 16 rounded up is at
// most the distance). A segment is a range of slots.
struct ChunkPlan {
    uint32_t slot0, slots;     // this segment
    uint32_t sequences, stride;   // slots that a CTA of the first kernel steps over
    void* stages;              // [slots][heads] ChunkStage
    const float* carry_in;     // states at the segment's start of sequences that began before it
    float* carry_out;          // states at its end
};
// The chunks [first, last) of a sequence that lie in the segment.
__device__ __forceinline__ void segment_chunks(const ChunkPlan& p, uint32_t s, uint32_t t0, uint32_t t1, uint32_t& first,
                                               uint32_t& last, uint32_t& base) {
    base = t0 / kChunk + s;
    const uint32_t n = (t1 - t0 + kChunk - 1) / kChunk;
    first = min(n, p.slot0 > base ? p.slot0 - base : 0u);
    last = min(n, p.slot0 + p.slots > base ? p.slot0 + p.slots - base : 0u);
}

// The chunk in a slot (whole warps): its first token and its sequence's end,
// found in the offsets, 32 of them at a time (up to 31 sequences' in `mine`, a
// lane each); false where the slot holds none.
__device__ __forceinline__ bool chunk_in(const SeqArgs& a, const ChunkPlan& p, uint32_t slot, uint32_t lane, uint32_t mine, uint32_t& first,
                                         uint32_t& t1) {
    uint32_t s = 0, t0;
    if (p.sequences < 32) {
        const uint32_t found = __ballot_sync(0xffffffffu, lane < p.sequences && mine / kChunk + lane <= slot);
        if (!found) return false;
        s = 31 - __clz(found);
        t0 = __shfl_sync(0xffffffffu, mine, s);
        t1 = __shfl_sync(0xffffffffu, mine, s + 1);
    } else {
        for (uint32_t n = p.sequences; n > 1;) {
            const uint32_t step = (n + 31) / 32, i = lane * step;
            const uint32_t found = __ballot_sync(0xffffffffu, i < n && a.offsets[s + i] / kChunk + s + i <= slot);
            if (!found) return false;
            const uint32_t k = 31 - __clz(found);
            s += k * step;
            n = min(step, n - k * step);
        }
        t0 = a.offsets[s];
        t1 = a.offsets[s + 1];
    }
    const uint32_t chunk = slot - (t0 / kChunk + s);
    first = t0 + chunk * kChunk;
    return t0 <= t1 && t1 <= a.tokens && t1 - t0 >= a.from && t1 - t0 < a.below && chunk < (t1 - t0 + kChunk - 1) / kChunk;
}

// The power of two that takes a maximum to [2^14, 2^15) (f16 ends at 2^16);
// zero, infinity and NaN keep theirs.
__device__ __forceinline__ int scale_exp(float top) {
    const int e = static_cast<int>(__float_as_uint(top) >> 23);
    return top == 0.0f || e == 255 ? 0 : min(126, 14 + 127 - e);
}
// 2^e, e clamped to what a float holds normalised
__device__ __forceinline__ float pow2(int e) { return exp2i(max(-126, min(127, e))); }
// 2^e to the ends of a float, subnormals included (|e| up to 252)
__device__ __forceinline__ float two_to(int e) { return pow2(e / 2) * pow2(e - e / 2); }

__device__ __forceinline__ float2 mul2(float2 x, float2 y) { return make_float2(x.x * y.x, x.y * y.y); }
__device__ __forceinline__ float2 mul1(float2 x, float y) { return make_float2(x.x * y, x.y * y); }

// Two neighbours as packed hi and lo.
__device__ __forceinline__ void split_pair(float2 x, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __float22half2_rn(x);
    const float2 b = __half22float2(h);
    const __half2 l = __floats2half2_rn(x.x - b.x, x.y - b.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
template <int ROWS, int W>
__device__ __forceinline__ void store_pair(__half (&dst)[2][ROWS][W], int row, int col, float2 x) {
    uint32_t hi, lo;
    split_pair(x, hi, lo);
    *reinterpret_cast<uint32_t*>(&dst[0][row][col]) = hi;
    *reinterpret_cast<uint32_t*>(&dst[1][row][col]) = lo;
}

// Two neighbours as three packed bf16 terms: 24 bits at any size.
__device__ __forceinline__ void split_bf16(float2 x, uint32_t (&w)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const __nv_bfloat162 h = __float22bfloat162_rn(x);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
        x.x -= __uint_as_float(w[i] << 16);
        x.y -= __uint_as_float(w[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* row) {
    const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(row));
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}

// big += x hi * y hi, small += the cross products, for two n-tiles.
__device__ __forceinline__ void mma_terms(float (&big)[2][4], float (&small)[2][4], const uint32_t (&xh)[4], const uint32_t (&xl)[4],
                                          const uint32_t (&yh)[4], const uint32_t (&yl)[4]) {
#pragma unroll
    for (int n = 0; n < 2; ++n) mma_f16(big[n], xh, yh[2 * n], yh[2 * n + 1]);
#pragma unroll
    for (int n = 0; n < 2; ++n) mma_f16(small[n], xl, yh[2 * n], yh[2 * n + 1]);
#pragma unroll
    for (int n = 0; n < 2; ++n) mma_f16(small[n], xh, yl[2 * n], yl[2 * n + 1]);
}

// The same for a contraction of one step, in one accumulator: the small
// products first, so that the sum is truncated once at its full size.
__device__ __forceinline__ void mma_terms1(float (&c)[2][4], const uint32_t (&xh)[4], const uint32_t (&xl)[4], const uint32_t (&yh)[4],
                                           const uint32_t (&yl)[4]) {
#pragma unroll
    for (int n = 0; n < 2; ++n) mma_f16(c[n], xl, yh[2 * n], yh[2 * n + 1]);
#pragma unroll
    for (int n = 0; n < 2; ++n) mma_f16(c[n], xh, yl[2 * n], yl[2 * n + 1]);
#pragma unroll
    for (int n = 0; n < 2; ++n) mma_f16(c[n], xh, yh[2 * n], yh[2 * n + 1]);
}

// c += x y^T over a chunk's tokens in bf16 terms (NX of x, in accumulator
// layout; three of y in shared memory, `row` this lane's ldmatrix row of the
// first), the small products first.
template <int NX>
__device__ __forceinline__ void split_tokens(const float (&x)[2][4], uint32_t (&xw)[3][4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[3];
        split_bf16(make_float2(x[i / 2][i % 2 * 2], x[i / 2][i % 2 * 2 + 1]), w);
#pragma unroll
        for (int n = 0; n < NX; ++n) xw[n][i] = w[n];
    }
}
template <int NX>
__device__ __forceinline__ void mma_tokens(float (&c)[2][4], const uint32_t (&xw)[3][4], const __nv_bfloat16* row) {
    uint32_t y[3][4];
#pragma unroll
    for (int i = 0; i < 3; ++i) ldmatrix4<false>(y[i], row + i * kChunk * (kChunk + 8));
#pragma unroll
    for (int order = 2; order >= 0; --order)
#pragma unroll
        for (int i = 0; i < NX; ++i)
            if (i <= order)
#pragma unroll
                for (int n = 0; n < 2; ++n) mma_bf16(c[n], xw[i], y[order - i][2 * n], y[order - i][2 * n + 1]);
}

// Two neighbouring values as floats; VEC: at a multiple of two elements.
template <typename E, bool VEC>
__device__ __forceinline__ float2 load2(const E* p) {
    if constexpr (!VEC) {
        return make_float2(to_f(p[0]), to_f(p[1]));
    } else if constexpr (sizeof(E) == 4) {
        return *reinterpret_cast<const float2*>(p);
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
}

__device__ __forceinline__ uint32_t max_halves(uint32_t x, uint32_t y) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
}
// Largest |x| of each of 8 tokens over a half warp, by the floats' upper
// halves (which order like the floats): a lane ends with tokens 2 i and 2 i + 1,
// i = lane / 4 % 4, each exchange halving the tokens that it still has.
__device__ __forceinline__ uint32_t token_tops(const float2 (&x)[8], uint32_t lane) {
    uint32_t m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        m[i] = max_halves(__byte_perm(__float_as_uint(x[2 * i].x), __float_as_uint(x[2 * i + 1].x), 0x7632) & 0x7fff7fffu,
                          __byte_perm(__float_as_uint(x[2 * i].y), __float_as_uint(x[2 * i + 1].y), 0x7632) & 0x7fff7fffu);
#pragma unroll
    for (int w = 2; w > 0; w >>= 1)
#pragma unroll
        for (int i = 0; i < w; ++i) {
            const bool up = lane & (4 * w);
            const uint32_t give = up ? m[i] : m[i + w], keep = up ? m[i + w] : m[i];
            m[i] = max_halves(keep, __shfl_xor_sync(0xffffffffu, give, 4 * w));
        }
    m[0] = max_halves(m[0], __shfl_xor_sync(0xffffffffu, m[0], 2));
    return max_halves(m[0], __shfl_xor_sync(0xffffffffu, m[0], 1));
}

// Row maxima of two rows over a quad's lanes, and as scale exponents.
__device__ __forceinline__ float2 row_exps(float m0, float m1, int (&ex)[2]) {
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
    }
    ex[0] = scale_exp(m0);
    ex[1] = scale_exp(m1);
    return make_float2(m0, m1);
}
__device__ __forceinline__ float2 row_exps(const float (&x)[2][4], int (&ex)[2]) {
    return row_exps(fmaxf(fmaxf(fabsf(x[0][0]), fabsf(x[0][1])), fmaxf(fabsf(x[1][0]), fabsf(x[1][1]))),
             fmaxf(fmaxf(fabsf(x[0][2]), fabsf(x[0][3])), fmaxf(fabsf(x[1][2]), fabsf(x[1][3]))), ex);
}

// The first tokens of two rows (16 tokens in accumulator layout) whose elements
// are not finite (kChunk: none; the second row's above the first's 8 bits);
// zeros take the place of such elements.
constexpr int kNone = kChunk | kChunk << 8;
__device__ __forceinline__ int first_bad(float (&x)[2][4], uint32_t t) {
    int bad[2] = {kChunk, kChunk};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!isfinite(x[i][e])) {
                bad[e / 2] = min(bad[e / 2], static_cast<int>(8 * i + 2 * t) + e % 2);
                x[i][e] = 0.0f;
            }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1)
#pragma unroll
        for (int r = 0; r < 2; ++r) bad[r] = min(bad[r], __shfl_xor_sync(0xffffffffu, bad[r], o));
    return bad[0] | bad[1] << 8;
}

// [16 rows][16] in accumulator layout (two n-tiles) as the two terms of a left operand.
__device__ __forceinline__ void split_rows(const float (&x)[4], const float (&y)[4], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    split_pair(make_float2(x[0], x[1]), hi[0], lo[0]);
    split_pair(make_float2(x[2], x[3]), hi[1], lo[1]);
    split_pair(make_float2(y[0], y[1]), hi[2], lo[2]);
    split_pair(make_float2(y[2], y[3]), hi[3], lo[3]);
}

// D threads: each two neighbouring channels of eight tokens, lanes 0-15 the
// chunk's first half, 16-31 the same channels' second half.
template <int D, typename E, bool VEC>
__global__ void __launch_bounds__(D, D == 128 ? 3 : 1) chunk_operands_kernel(const SeqArgs a, const ChunkPlan plan) {
    extern __shared__ __align__(16) unsigned char chunk_mem[];
    ChunkScratch<D>& sc = *reinterpret_cast<ChunkScratch<D>*>(chunk_mem);
    constexpr int NP = D / 32;   // warps
    asm volatile("griddepcontrol.launch_dependents;");   // the scan's CTAs may start as these run out
    const uint32_t h = blockIdx.x % a.heads;
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, th = lane / 16, P = a.heads * D;
    const uint32_t c = warp * 32 + lane % 16 * 2;
    const E* q = static_cast<const E*>(a.q) + h * D + c;
    const E* k = static_cast<const E*>(a.k) + h * D + c;
    const float* ld = a.log_decay + h * D + c;
    // the next chunk's values; past the end k = q = beta = 0 and a decay of 1
    // leave everything as it is
    float2 kk[8], qq[8], al[8];
    float bb = 0.0f;
    auto fetch = [&](uint32_t first, uint32_t t1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t tok = first + 8 * th + i;
            const float2 zero = make_float2(0.0f, 0.0f);
            const size_t t = tok;
            kk[i] = tok < t1 ? load2<E, VEC>(k + t * a.row_stride) : zero;
            qq[i] = tok < t1 ? load2<E, VEC>(q + t * a.row_stride) : zero;
            al[i] = tok < t1 ? load2<float, VEC>(ld + t * P) : zero;
        }
        if (threadIdx.x < kChunk)
            bb = first + threadIdx.x < t1 ? a.beta[static_cast<size_t>(first + threadIdx.x) * a.heads + h] : 0.0f;
    };
    // the next chunk's rows on their way to L2, 128 bytes a thread, a chunk's
    // work before they are loaded (13 ragged turns: 978 -> 922 us in all)
    auto prefetch = [&](uint32_t first, uint32_t t1) {
        constexpr uint32_t qk = (D * sizeof(E) + 127) / 128, all = 2 * qk + (D * 4 + 127) / 128;
        const size_t tok = first + threadIdx.x % kChunk;
        if (tok >= t1) return;
#pragma unroll
        for (uint32_t p = 0; p < all; p += D / kChunk) {
            const uint32_t x = p + threadIdx.x / kChunk;
            const char* at = x < qk       ? reinterpret_cast<const char*>(static_cast<const E*>(a.q) + tok * a.row_stride + h * D) + 128 * x
                             : x < 2 * qk ? reinterpret_cast<const char*>(static_cast<const E*>(a.k) + tok * a.row_stride + h * D) + 128 * (x - qk)
                                          : reinterpret_cast<const char*>(a.log_decay + tok * P + h * D) + 128 * (x - 2 * qk);
            if (all % (D / kChunk) == 0 || x < all) asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
        }
    };
    const uint32_t arow = lane % 16, acol = lane / 16 * 8;         // ldmatrix: left operands, and k-major ones transposed
    uint32_t slot = blockIdx.x / a.heads, first, t1;
    const uint32_t mine = a.offsets[min(lane, plan.sequences)];
    auto seek = [&] {   // from `slot` on
        while (slot < plan.slots && !chunk_in(a, plan, plan.slot0 + slot, lane, mine, first, t1)) slot += plan.stride;
        return slot < plan.slots;
    };
    bool more = seek();
    if (more) fetch(first, t1);
    while (more) {
        ChunkStage<D>& st = static_cast<ChunkStage<D>*>(plan.stages)[static_cast<size_t>(slot) * a.heads + h];
        slot += plan.stride;
        more = seek();
        if (more) prefetch(first, t1);
#pragma unroll
        for (int i = 0; i < 8; ++i) al[i] = make_float2(expf(al[i].x), expf(al[i].y));
        {
            const uint32_t top[3] = {token_tops(kk, lane), token_tops(qq, lane), token_tops(al, lane)};
            if (lane % 4 == 0)
#pragma unroll
                for (int e = 0; e < 3; ++e) sc.top[e][warp][4 * th + lane / 4 % 4] = top[e];
            // q_i . k_i over the warp's channels: each exchange halves the
            // values that a lane still sums; lane l ends with token l / 2 % 8
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = fmaf(qq[i].x, kk[i].x, qq[i].y * kk[i].y);
#pragma unroll
            for (int w = 8; w > 1; w >>= 1)
#pragma unroll
                for (int i = 0; i < w / 2; ++i) {
                    const bool up = lane & w;
                    const float give = up ? d[i] : d[i + w / 2], keep = up ? d[i + w / 2] : d[i];
                    d[i] = keep + __shfl_xor_sync(0xffffffffu, give, w);
                }
            d[0] += __shfl_xor_sync(0xffffffffu, d[0], 1);
            if (lane % 2 == 0) sc.diag[warp][8 * th + lane % 16 / 2] = d[0];
        }
        if (threadIdx.x < kChunk) sc.beta[threadIdx.x] = bb;
        __syncthreads();
        float ftotal;      // p_15's power
        uint32_t poison;   // the first token with a key, decay or beta that is not finite
        {   // the tokens' powers of two, a lane each, every warp for itself
            const uint32_t tok = lane % 16;
            uint32_t top[3];
#pragma unroll
            for (int e = 0; e < 3; ++e) {
                top[e] = 0;
#pragma unroll
                for (int w = 0; w < NP; ++w) top[e] = max(top[e], static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(sc.top[e][w])[tok]));
            }
            const int ek = scale_exp(__uint_as_float(top[0] << 16)), z = scale_exp(__uint_as_float(top[1] << 16));
            const float be = sc.beta[tok];
            const uint32_t odd = __ballot_sync(0xffffffffu, top[0] >= 0x7f80 || top[2] >= 0x7f80 || !(fabsf(be) < INFINITY));
            poison = odd ? min(16, __ffs(odd) - 1) : 16;
            const bool sized = top[0] && tok < poison;
            const int least = __reduce_min_sync(0xffffffffu, sized ? ek : 1000), x = least == 1000 ? 0 : least;
            const int dx = sized ? min(kKeySpread, ek - x) : 0;
            // 2^ae over the decay's largest channel (up to 1.008 counts as 1)
            const int ae = (top[2] >= 0x3f00 && top[2] <= 0x3f80) || tok >= poison ? 0 : max(kLeastDecay, min(kMostDecay, static_cast<int>(top[2] >> 7) - 126));
            int sum = ae;
#pragma unroll
            for (int o = 1; o < kChunk; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, sum, o, kChunk);
                if (tok >= static_cast<uint32_t>(o)) sum += y;
            }
            if (__any_sync(0xffffffffu, ae > 0)) {   // a decay that grows: the limits apply token by token
                int y = 0;
                for (int i = 0; i < kChunk; ++i) {
                    y = max(kLeastDecay, min(kMostDecay, y + __shfl_sync(0xffffffffu, ae, i, kChunk)));
                    if (tok == static_cast<uint32_t>(i)) sum = y;
                }
            } else {
                sum = max(sum, kLeastDecay);
            }
            const int before = __shfl_up_sync(0xffffffffu, sum, 1, kChunk), end = __shfl_sync(0xffffffffu, sum, 15, kChunk), mid = end >> 1;
            if (lane < 16) {
                sc.sk[warp][tok] = exp2i(x + dx);
                sc.sq[warp][tok] = exp2i(z);
                sc.sa[warp][tok] = exp2i((tok ? before : 0) - sum);
                if (warp == 0) {
                    sc.bs[tok] = sized ? be * exp2i(-2 * dx) : 0.0f;   // a zero key writes nothing, whatever its u
                    sc.ft[tok] = pow2(dx - sum + mid);
                    sc.fp[tok] = two_to(sum - mid - z);
                    sc.fd[tok] = pow2(dx + sum - mid);
                    st.fq[tok] = tok < poison ? two_to(sum - z) : NAN;
                    if (lane == 0) {
                        sc.fx = two_to(-x);
                        sc.wexp = mid + 20 - x;
                        st.exp = end - mid - x;
                    }
                }
            }
            ftotal = poison < 16 ? NAN : exp2i(end);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(&sc.sa[warp][8 * th + i]);
            const float4 y = *reinterpret_cast<const float4*>(&sc.sk[warp][8 * th + i]);
            const float4 z = *reinterpret_cast<const float4*>(&sc.sq[warp][8 * th + i]);
            const float fa[4] = {x.x, x.y, x.z, x.w}, fk[4] = {y.x, y.y, y.z, y.w}, fq[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                al[i + e] = mul1(al[i + e], fa[e]);
                kk[i + e] = mul1(kk[i + e], fk[e]);
                qq[i + e] = mul1(qq[i + e], fq[e]);
            }
        }
        // decays within blocks of 8 (pre, suf), 8's halves (f1), 4's (f2) and
        // 2's (al): upper tokens from the middle, lower ones to it
        float2 f1[8], f2[8], pre[8], suf[8];
        const float2 one = make_float2(1.0f, 1.0f);
#pragma unroll
        for (int b = 0; b < 8; b += 4) {
            f2[b] = al[b + 1];
            f2[b + 1] = one;
            f2[b + 2] = al[b + 2];
            f2[b + 3] = mul2(al[b + 2], al[b + 3]);
        }
        f1[3] = one;
        f1[2] = al[3];
        f1[1] = f2[3];
        f1[0] = mul2(al[1], f2[3]);
        f1[4] = al[4];
        f1[5] = mul2(al[4], al[5]);
        f1[6] = mul2(f1[5], al[6]);
        f1[7] = mul2(f1[5], f2[7]);
        pre[0] = al[0];
        pre[1] = mul2(al[0], al[1]);
        pre[2] = mul2(pre[1], al[2]);
        pre[3] = mul2(pre[1], f2[3]);
        suf[7] = one;
        suf[6] = al[7];
        suf[5] = f2[7];
        suf[4] = mul2(al[5], f2[7]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pre[4 + i] = mul2(pre[3], f1[4 + i]);
            suf[i] = mul2(f1[i], f1[7]);
        }
        // the other half's whole decay
        const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, pre[7].x, 16), __shfl_xor_sync(0xffffffffu, pre[7].y, 16));
        if (th) *reinterpret_cast<float2*>(&st.total[c]) = mul1(mul2(pre[7], other), ftotal);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int tok = 8 * th + i;
            const float2 ks = kk[i], qs = qq[i];
            const float2 from = th ? mul2(pre[i], other) : pre[i], to = th ? suf[i] : mul2(suf[i], other);
            store_pair(sc.k, tok, c, mul2(ks, from));
            store_pair(st.q, tok, c, mul2(qs, from));
            store_pair(st.ke, tok, c, mul2(ks, to));
            // blocks of 16: the second half is upper
            const float2 g = th ? pre[i] : suf[i], k0 = mul2(ks, g);
            store_pair(sc.level[0], th ? i : 16 + i, c, k0);
            if (th) {
                const float2 q0 = mul2(qs, g);
                store_pair(sc.level[0], 8 + i, c, q0);
            }
#pragma unroll
            for (int l = 1; l < 4; ++l) {
                const int half = 8 >> l;
                const int row = 4 * th + i / (2 * half) * half + i % half;   // of its side's 8
                const float2 f = l == 1 ? f1[i] : l == 2 ? f2[i] : i % 2 ? al[i] : one;
                const float2 kl = mul2(ks, f);
                if (i & half) {
                    const float2 ql = mul2(qs, f);
                    store_pair(sc.level[l], row, c, kl);
                    store_pair(sc.level[l], 8 + row, c, ql);
                } else {
                    store_pair(sc.level[l], 16 + row, c, kl);
                }
            }
        }
        // From `poison` on fq, and at the end the state's factor, are NaN. Zeros
        // in p K and T keep the tokens before clear of it (T's and P's own zeros
        // times a NaN would not).
        if (poison < 16)
            for (int i = max(0, static_cast<int>(poison) - static_cast<int>(8 * th)); i < 8; ++i)
                store_pair(sc.k, 8 * th + i, c, make_float2(0.0f, 0.0f));
        if (more) fetch(first, t1);
        __syncthreads();
        for (int l = warp; l < 4; l += NP) {
            float b[4] = {}, x[4] = {};
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                uint32_t yh[4], yl[4];
                ldmatrix4<false>(yh, &sc.level[l][0][16 + lane % 8][32 * j + lane / 8 * 8]);
                ldmatrix4<false>(yl, &sc.level[l][1][16 + lane % 8][32 * j + lane / 8 * 8]);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t xh[4], xl[4];
                    ldmatrix4<false>(xh, &sc.level[l][0][arow][32 * j + 16 * e + acol]);
                    ldmatrix4<false>(xl, &sc.level[l][1][arow][32 * j + 16 * e + acol]);
                    mma_f16(b, xh, yh[2 * e], yh[2 * e + 1]);
                    mma_f16(x, xl, yh[2 * e], yh[2 * e + 1]);
                    mma_f16(x, xh, yl[2 * e], yl[2 * e + 1]);
                }
            }
            const int half = 8 >> l, u = lane / 4, i = u / half * 2 * half + half + u % half;
            const float fx = sc.fx;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int w = lane % 4 * 2 + e, j = w / half * 2 * half + w % half;
                if (u / half != w / half) continue;
                sc.At[j][i] = (b[e] + x[e]) * fx * fx;
                sc.P[i][j] = (b[2 + e] + x[2 + e]) * sc.fp[i] * fx;
            }
        }
        __syncthreads();
        if (warp == 0) {   // T, a lane per column, one row's multiple after the other
            const uint32_t j = lane % 16;
            float x[kChunk];
#pragma unroll
            for (int i = 0; i < kChunk; ++i) x[i] = 0.0f;
#pragma unroll
            for (int m = 0; m < kChunk; ++m) {
                x[m] = fmaf(-sc.bs[m], x[m], m == static_cast<int>(j) ? 1.0f : 0.0f);
#pragma unroll
                for (int i = m + 1; i < kChunk; ++i) x[i] = fmaf(sc.At[m][i], x[m], x[i]);
            }
            const float b = sc.bs[j];
#pragma unroll
            for (int i = 0; i < kChunk / 2; ++i)   // a half warp has half of the rows
                sc.T[8 * th + i][j] = 8 * th + i < poison ? (th ? x[8 + i] : x[i]) * b : 0.0f;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < kChunk * kChunk / 2; e += D) {   // T and P for the scan
            const int i = e / 8, j = e % 8 * 2;
            uint32_t w[3];
            split_bf16(mul2(*reinterpret_cast<const float2*>(&sc.T[i][j]), *reinterpret_cast<const float2*>(&sc.ft[j])), w);
#pragma unroll
            for (int n = 0; n < 3; ++n) *reinterpret_cast<uint32_t*>(&st.t[n][i][j]) = w[n];
            float2 x = *reinterpret_cast<const float2*>(&sc.P[i][j]);
            float diag = 0.0f;
#pragma unroll
            for (int n = 0; n < NP; ++n) diag += sc.diag[n][i];
            diag *= sc.fd[i];
            x.x = i > j ? x.x : i == j ? diag : 0.0f;
            x.y = i > j + 1 ? x.y : i == j + 1 ? diag : 0.0f;
            split_bf16(x, w);
#pragma unroll
            for (int n = 0; n < 3; ++n) *reinterpret_cast<uint32_t*>(&st.p[n][i][j]) = w[n];
        }
        {   // W = T (p K): 16 sums of products below 2^30, kept as multiples of 2^20
            float x[2][4];   // rows lane / 4 and 8 on, each by a power of its own
            int e[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = *reinterpret_cast<const float2*>(&sc.T[lane / 4 + 8 * (i % 2)][8 * (i / 2) + lane % 4 * 2]);
                x[i / 2][i % 2 * 2] = v.x;
                x[i / 2][i % 2 * 2 + 1] = v.y;
            }
            row_exps(x, e);
            if (warp == 0 && lane % 4 < 2) st.fw[lane / 4 + lane % 4 * 8] = two_to(sc.wexp - (lane % 4 ? e[1] : e[0]));
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < 4; ++n) x[i][n] *= exp2i(e[n / 2]);
            uint32_t xh[4], xl[4];
            split_rows(x[0], x[1], xh, xl);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = warp * 32 + 16 * j;
                float w[2][4] = {};
                uint32_t yh[4], yl[4];
                ldmatrix4<true>(yh, &sc.k[0][arow][col + acol]);
                ldmatrix4<true>(yl, &sc.k[1][arow][col + acol]);
                mma_terms1(w, xh, xl, yh, yl);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        store_pair(st.w, lane / 4 + 8 * r, col + 8 * e + lane % 4 * 2,
                                   mul1(make_float2(w[e][2 * r], w[e][2 * r + 1]), 0x1p-20f));
            }
        }
        __syncthreads();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");   // ends after the token form before it
}

template <int D, int NW, int KS>
struct __align__(128) ScanSmem {
    ChunkStage<D> stage[kStages];
    // odd and even chunks, row group, half, what (W S0^T, Q S0^T), token tile: a lane's sums
    float4 part[2][KS > 1 ? NW : 1][KS][2][2][32];
    uint64_t full[kStages], empty[kStages];
    int abort;
};

// The blockIdx.y-th sequence of the batch, the longest ones first (they then
// start first, and the last round of CTAs is short: 13 ragged turns 1027 -> 922
// us in all); the given order for many or short ones, where sorting costs more.
__device__ __forceinline__ uint32_t sequence_of(const SeqArgs& a, uint32_t y, uint32_t* found) {
    const uint32_t n = gridDim.y;
    if (n == 1 || n > 64 || a.tokens < 256 * n) return y;
    for (uint32_t s = threadIdx.x; s < n; s += blockDim.x) {
        const uint32_t len = a.offsets[s + 1] - a.offsets[s];
        uint32_t rank = 0;
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t other = a.offsets[i + 1] - a.offsets[i];
            rank += other > len || (other == len && i < s);
        }
        if (rank == y) *found = s;
    }
    __syncthreads();
    return *found;
}

// A row group is 16 value rows of one head, and KS warps of it take a part of
// the key channels each: with one sequence there are SMs for all of them, and
// a warp's MMAs per chunk halve (an MMA holds up its warp's issue for its 8
// cycles); the parts of W S0^T and Q S0^T are added through shared memory. A
// last warp copies the operands.
template <int D, int NW, int KS, int PER_SM, typename E>
__global__ void __launch_bounds__(32 * NW * KS + 32, PER_SM) chunk_scan_kernel(const SeqArgs a, const ChunkPlan plan) {
    extern __shared__ __align__(128) unsigned char scan_mem[];
    ScanSmem<D, NW, KS>& bar = *reinterpret_cast<ScanSmem<D, NW, KS>*>(scan_mem);
    ChunkStage<D>* stages = bar.stage;
    volatile int* abort = &bar.abort;
    __shared__ uint32_t found;
    constexpr uint32_t slices = D / (16 * NW);
    const uint32_t s = sequence_of(a, blockIdx.y, &found), h = blockIdx.x / slices, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint32_t t0, t1, chunk, chunk_end, base;
    if (!token_range(a, s, t0, t1)) return;
    segment_chunks(plan, s, t0, t1, chunk, chunk_end, base);
    // a sequence without tokens passes its state on in the first segment
    if (chunk >= chunk_end && (t0 < t1 || plan.slot0)) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            tc::mbar_init(&bar.full[i], 1);
            tc::mbar_init(&bar.empty[i], NW * KS);
        }
        bar.abort = 0;
        tc::fence_barrier_init();
    }
    __syncthreads();
    if (warp == NW * KS) {
        const ChunkStage<D>* src = static_cast<const ChunkStage<D>*>(plan.stages) + static_cast<size_t>(base + chunk - plan.slot0) * a.heads + h;
        const E* v = static_cast<const E*>(a.v) + h * D + blockIdx.x % slices * (16 * NW);
        uint32_t n = 0;
        bool ok = true;
        asm volatile("griddepcontrol.wait;" ::: "memory");   // the operands are written
        for (; ok && chunk + n < chunk_end; ++n, src += a.heads) {
            // this CTA's columns of v, for the warps to find in L2
            const uint32_t tok = t0 + (chunk + n) * kChunk + lane / 2;
            if (tok < t1) {
                const E* at = v + static_cast<size_t>(tok) * a.row_stride + lane % 2 * (8 * NW);
                asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
            }
            if (lane == 0) {
                ok = tc::mbar_wait(&bar.empty[n % kStages], n / kStages & 1u ^ 1u, abort);
                if (ok) {
                    tc::mbar_arrive_expect_tx(&bar.full[n % kStages], sizeof(ChunkStage<D>));
                    tc::bulk_load(&stages[n % kStages], src, sizeof(ChunkStage<D>), &bar.full[n % kStages]);
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        if (!ok) --n;   // the last one was not copied
        if (lane == 0) {
            volatile int never = 0;   // copies in flight end before the CTA does
            for (uint32_t i = 0; i < kStages && i < n; ++i)
                tc::mbar_wait(&bar.full[(n - 1 - i) % kStages], (n - 1 - i) / kStages & 1u, &never, 200000000ull);
            if (*abort) atomicExch(a.status, K3XB_BACKEND_UNAVAILABLE);
        }
        return;
    }
    constexpr int DK = D / KS;   // this warp's key channels, from k0 on
    constexpr int NV = sizeof(E) == 2 ? 1 : 3;   // bf16 values are one term
    // U in P U: for bf16 outputs two terms, off by 2^-18 of the products, where
    // the outputs' own rounding takes 2^-9 (13 ragged turns 922 -> 904 us)
    constexpr int NU = sizeof(E) == 2 ? 2 : 3;
    const uint32_t half = warp % KS, k0 = half * DK;
    const uint32_t row0 = blockIdx.x % slices * (16 * NW) + warp / KS * 16;
    const uint32_t g = lane / 4, t = lane % 4, P = a.heads * D;
    const size_t state_at = (static_cast<size_t>(s) * a.heads + h) * D * D + static_cast<size_t>(row0 + g) * D + k0 + 2 * t;
    const E* v = static_cast<const E*>(a.v) + h * D + row0 + g;
    const float* state = chunk ? plan.carry_in : a.state;
    float* state_out = chunk_end * kChunk < t1 - t0 ? plan.carry_out : a.state_out;
    float S[DK / 8][4];
#pragma unroll
    for (int j = 0; j < DK / 8; ++j) {
        float2 x = make_float2(0.0f, 0.0f), y = x;
        if (state) {
            x = *reinterpret_cast<const float2*>(state + state_at + 8 * j);
            y = *reinterpret_cast<const float2*>(state + state_at + 8 * D + 8 * j);
        }
        S[j][0] = x.x; S[j][1] = x.y; S[j][2] = y.x; S[j][3] = y.y;
    }
    // v of tokens 2t, 2t+1, 2t+8, 2t+9 and rows g, g + 8, in accumulator order
    float vv[2][4];
    auto fetch = [&](uint32_t first) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t tok = first + 8 * n + 2 * t + e % 2;
                vv[n][e] = tok < t1 ? to_f(v[static_cast<size_t>(tok) * a.row_stride + 8 * (e / 2)]) : 0.0f;
            }
    };
    fetch(t0 + chunk * kChunk);
    // ldmatrix rows: n-major operands (lanes 0-7: tile 0, k 0-7; 8-15: k 8-15; 16-31: tile 1)
    const uint32_t mrow = lane % 8 + lane / 16 * 8, mcol = lane / 8 % 2 * 8;
    // k-major ones, transposed (lanes 0-7: tile 0, k 0-7; 8-15: k 8-15; 16-31: tile 1)
    const uint32_t krow = lane % 16, kcol = lane / 16 * 8;
    int sx[2] = {0, 0};   // S holds the state's rows times 2^sx
    // A value that is not finite would meet T's zeros above the diagonal: a
    // zero stands for it, and after the chunk its row's state and this lane's
    // outputs from its token on become NaN.
    int spoilt = kNone;
    auto spoil = [&](uint32_t first) {
        for (int i = 0; i < 8; ++i) {
            const uint32_t at = 8 * (i / 4) + 2 * t + i % 2, r = i / 2 % 2;
            if ((KS > 1 && i / 4 != static_cast<int>(half)) || static_cast<int>(at) < (r ? spoilt >> 8 : spoilt & 255) || first + at >= t1) continue;
            store1<E>(a.out, static_cast<size_t>(first + at) * P + h * D + row0 + g + 8 * r, NAN);
        }
    };
    for (uint32_t n = 0; chunk + n < chunk_end; ++n) {
        const uint32_t first = t0 + (chunk + n) * kChunk;
        const ChunkStage<D>& st = stages[n % kStages];
        int ux[2];
        {
            float m0 = 0.0f, m1 = 0.0f, zero[2] = {0.0f, 0.0f};   // zero: NaN where a value is not finite
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) zero[i] = fmaf(vv[i][e], 0.0f, zero[i]);
#pragma unroll
            for (int j = 0; j < DK / 8; ++j) {
                m0 = fmaxf(m0, fmaxf(fabsf(S[j][0]), fabsf(S[j][1])));
                m1 = fmaxf(m1, fmaxf(fabsf(S[j][2]), fabsf(S[j][3])));
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
                m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
            }
            // a row's multiple changes when its largest element leaves
            // [2^8, 2^15]: f16 holds it then, with 32 bits below it
            const bool off0 = m0 > 0x1p15f || (m0 < 0x1p8f && m0 != 0.0f && sx[0] < 126) || sx[0] > 30;
            const bool off1 = m1 > 0x1p15f || (m1 < 0x1p8f && m1 != 0.0f && sx[1] < 126) || sx[1] > 30;
            if (__any_sync(0xffffffffu, off0 || off1 || zero[0] + zero[1] != 0.0f || spoilt != kNone)) {
                const int before = spoilt;
                if (before != kNone) spoil(first - kChunk);
                spoilt = first_bad(vv, t);
                // it stays below 2^90 over that of the values to come, so that a
                // small state's multiple does not carry their sums past a float's end
                int vx[2];
                const float2 top = row_exps(vv, vx);
                const int cap0 = top.x == 0.0f ? 126 : min(126, vx[0] + 90), cap1 = top.y == 0.0f ? 126 : min(126, vx[1] + 90);
                const bool in0 = m0 == 0.0f || (m0 >= 0x1p8f && m0 <= 0x1p15f), in1 = m1 == 0.0f || (m1 >= 0x1p8f && m1 <= 0x1p15f);
                const int d0 = min(in0 ? 0 : scale_exp(m0) - 2, cap0 - sx[0]), d1 = min(in1 ? 0 : scale_exp(m1) - 2, cap1 - sx[1]);
                const float f0 = (before & 255) < kChunk ? NAN : pow2(d0), f1 = before >> 8 < kChunk ? NAN : pow2(d1);
                sx[0] += d0;
                sx[1] += d1;
#pragma unroll
                for (int j = 0; j < DK / 8; ++j) {
                    S[j][0] *= f0;
                    S[j][1] *= f0;
                    S[j][2] *= f1;
                    S[j][3] *= f1;
                }
            }
        }
        uint32_t xh[4], xl[4], yh[4], yl[4], vw[3][4];
        split_tokens<NV>(vv, vw);
        if (chunk + n + 1 < chunk_end) fetch(first + kChunk);
        tc::mbar_pass(&bar.full[n % kStages], n / kStages & 1u, abort);
        __syncwarp();
        uint32_t uw[3][4];
        // T V, W S0^T and (p Q) S0^T
        float u[2][4] = {}, wb[2][4] = {}, ws[2][4] = {}, ob[2][4] = {}, os[2][4] = {};
        mma_tokens<NV>(u, vw, &st.t[0][mrow][mcol]);
#pragma unroll
        for (int j = 0; j < DK / 16; ++j) {
            split_rows(S[2 * j], S[2 * j + 1], xh, xl);
            ldmatrix4<false>(yh, &st.w[0][mrow][k0 + 16 * j + mcol]);
            ldmatrix4<false>(yl, &st.w[1][mrow][k0 + 16 * j + mcol]);
            mma_terms(wb, ws, xh, xl, yh, yl);
            ldmatrix4<false>(yh, &st.q[0][mrow][k0 + 16 * j + mcol]);
            ldmatrix4<false>(yl, &st.q[1][mrow][k0 + 16 * j + mcol]);
            mma_terms(ob, os, xh, xl, yh, yl);
        }
        {
            const float fs[2] = {pow2(-sx[0]), pow2(-sx[1])};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 fw = *reinterpret_cast<const float2*>(&st.fw[8 * i + 2 * t]), fq = *reinterpret_cast<const float2*>(&st.fq[8 * i + 2 * t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    wb[i][e] = (wb[i][e] + ws[i][e]) * fs[e / 2] * (e % 2 ? fw.y : fw.x);
                    ob[i][e] = (ob[i][e] + os[i][e]) * fs[e / 2] * (e % 2 ? fq.y : fq.x);
                }
            }
            if constexpr (KS > 1) {   // the halves' sums, in the same order in both warps
                float4 (*part)[2][2][32] = bar.part[n % 2][warp / KS];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    part[half][0][i][lane] = make_float4(wb[i][0], wb[i][1], wb[i][2], wb[i][3]);
                    part[half][1][i][lane] = make_float4(ob[i][0], ob[i][1], ob[i][2], ob[i][3]);
                }
                asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(warp / KS)), "n"(32 * KS) : "memory");
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 x = part[0][0][i][lane], y = part[1][0][i][lane], z = part[half ^ 1][1][i][lane];
                    wb[i][0] = x.x + y.x; wb[i][1] = x.y + y.y; wb[i][2] = x.z + y.z; wb[i][3] = x.w + y.w;
                    ob[i][0] += z.x; ob[i][1] += z.y; ob[i][2] += z.z; ob[i][3] += z.w;
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) u[i][e] -= wb[i][e];
            split_tokens<NU>(u, uw);
            row_exps(u, ux);
            // a product's powers together stay within a float's
            ux[0] = min(ux[0], 126 + sx[0] + st.exp);
            ux[1] = min(ux[1], 126 + sx[1] + st.exp);
            const float f0 = pow2(ux[0]), f1 = pow2(ux[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) u[i][e] *= e < 2 ? f0 : f1;
            split_rows(u[0], u[1], xh, xl);
        }
        {   // S = S diag(total) + U^T (e K)
            const float f0 = pow2(sx[0] - ux[0] + st.exp), f1 = pow2(sx[1] - ux[1] + st.exp);
#pragma unroll
            for (int j = 0; j < DK / 16; ++j) {
                float c[2][4] = {};
                uint32_t zh[4], zl[4];
                ldmatrix4<true>(zh, &st.ke[0][krow][k0 + 16 * j + kcol]);
                ldmatrix4<true>(zl, &st.ke[1][krow][k0 + 16 * j + kcol]);
                mma_terms1(c, xh, xl, zh, zl);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 tot = *reinterpret_cast<const float2*>(&st.total[k0 + 16 * j + 8 * i + 2 * t]);
                    float (&x)[4] = S[2 * j + i];
                    x[0] = fmaf(c[i][0], f0, x[0] * tot.x);
                    x[1] = fmaf(c[i][1], f0, x[1] * tot.y);
                    x[2] = fmaf(c[i][2], f1, x[2] * tot.x);
                    x[3] = fmaf(c[i][3], f1, x[3] * tot.y);
                }
            }
        }
        {   // O = (p Q) S0^T + P U
            float c[2][4] = {};
            mma_tokens<NU>(c, uw, &st.p[0][mrow][mcol]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (KS > 1 && i != static_cast<int>(half)) continue;   // a half writes one tile of tokens
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t tok = first + 8 * i + 2 * t + e % 2;
                    const float o = c[i][e] + ob[i][e];
                    if (tok < t1) store1<E>(a.out, static_cast<size_t>(tok) * P + h * D + row0 + g + 8 * (e / 2), o);
                }
            }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&bar.empty[n % kStages]);
    }
    if (spoilt != kNone) spoil(t0 + (chunk_end - 1) * kChunk);
    if (!state_out) return;
    const float f0 = (spoilt & 255) < kChunk ? NAN : pow2(-sx[0]), f1 = spoilt >> 8 < kChunk ? NAN : pow2(-sx[1]);
#pragma unroll
    for (int j = 0; j < DK / 8; ++j) {
        *reinterpret_cast<float2*>(state_out + state_at + 8 * j) = make_float2(S[j][0] * f0, S[j][1] * f0);
        *reinterpret_cast<float2*>(state_out + state_at + 8 * D + 8 * j) = make_float2(S[j][2] * f1, S[j][3] * f1);
    }
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

template <int D, int NW, int KS, int PER_SM, typename E>
int launch_scan(k3xb_ctx* ctx, const SeqArgs& a, const ChunkPlan& p, uint32_t sequences) {
    static std::atomic<uint64_t> configured{0};   // per template instance
    const dim3 grid(a.heads * (D / (16 * NW)), sequences);
    // Where every CTA can have an SM of its own it asks for more than half of
    // the shared memory: two on one SM while others idle share its issue
    // slots (8192 tokens of 32 heads 1087 us so, 804 apart, when the kernel's
    // registers left room for two).
    constexpr size_t need = sizeof(ScanSmem<D, NW, KS>), alone = std::max(need, size_t(116) << 10);
    const size_t smem = static_cast<uint64_t>(grid.x) * grid.y <= static_cast<uint64_t>(ctx->sm_count) ? alone : need;
    const int cst = configure_once(ctx, configured, [&]() -> int {
        K3XB_CUDA(ctx, cudaFuncSetAttribute(chunk_scan_kernel<D, NW, KS, PER_SM, E>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            static_cast<int>(alone)));
        return K3XB_OK;
    });
    if (cst) return cst;
    // starts beside the operands kernel's tail; its copying warp waits for the
    // end of that kernel, and nothing else here reads what it writes
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(32 * NW * KS + 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    K3XB_CUDA(ctx, cudaLaunchKernelEx(&cfg, chunk_scan_kernel<D, NW, KS, PER_SM, E>, a, p));
    ++ctx->stats.kernel_launches;
    return K3XB_OK;
}

template <int D, int NW, typename E, bool VEC>
int launch_chunks_as(k3xb_ctx* ctx, const SeqArgs& a, uint32_t sequences) {
    static std::atomic<uint64_t> configured{0};   // per template instance
    const int cst = configure_once(ctx, configured, [&]() -> int {
        K3XB_CUDA(ctx, cudaFuncSetAttribute(chunk_operands_kernel<D, E, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            static_cast<int>(sizeof(ChunkScratch<D>))));
        return K3XB_OK;
    });
    if (cst) return cst;
    const uint32_t slots = a.tokens / kChunk + sequences;
    const size_t per_slot = a.heads * sizeof(ChunkStage<D>);
    const uint32_t step = static_cast<uint32_t>(std::min<size_t>(slots, std::max<size_t>(1, kOperandBytes / per_slot)));
    // states between segments: in state_out, or in scratch where that is not wanted
    const size_t carry = step < slots && !a.state_out ? static_cast<size_t>(sequences) * a.heads * D * D : 0;
    Sizer sz;
    sz.take<unsigned char>(step * per_slot);
    sz.take<float>(carry);
    void* mem;
    if (const int st = ensure_scratch(ctx, sz.used, &mem)) return st;
    Carver cv(mem);
    ChunkPlan p{};
    p.stages = cv.take<unsigned char>(step * per_slot);
    float* between = cv.take<float>(carry);
    if (!carry) between = a.state_out;
    p.carry_in = p.carry_out = between;
    const uint64_t scans = static_cast<uint64_t>(a.heads) * (D / 32) * sequences;
    for (uint32_t x = 0; x < slots; x += step) {
        p.slot0 = x;
        p.slots = std::min(step, slots - x);
        // sixteen CTAs for each that the GPU holds at a time (three per SM), so
        // that they even out and a CTA has chunks to load ahead
        p.sequences = sequences;
        p.stride = static_cast<uint32_t>(std::min<uint64_t>((48ull * ctx->sm_count + a.heads - 1) / a.heads, p.slots));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(p.stride * a.heads);
        cfg.blockDim = dim3(D);
        cfg.dynamicSmemBytes = sizeof(ChunkScratch<D>);
        cfg.stream = ctx->stream;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = x == 0 && a.from ? 1 : 0;   // beside the token form of the short sequences
        K3XB_CUDA(ctx, cudaLaunchKernelEx(&cfg, chunk_operands_kernel<D, E, VEC>, a, p));
        ++ctx->stats.kernel_launches;
        // few sequences: an SM for every 32 rows, with two warps to a row
        // group; else two CTAs per SM where there are that many
        int st;
        if (D == 128 && scans <= static_cast<uint64_t>(ctx->sm_count)) st = launch_scan<D, 2, D == 128 ? 2 : 1, 1, E>(ctx, a, p, sequences);
        else if (scans > 2ull * ctx->sm_count) st = launch_scan<D, NW, 1, 2, E>(ctx, a, p, sequences);
        else st = launch_scan<D, NW, 1, 1, E>(ctx, a, p, sequences);
        if (st) return st;
    }
    return K3XB_OK;
}

template <int D, int NW, typename E>
int launch_chunk(k3xb_ctx* ctx, const SeqArgs& a, uint32_t sequences) {
    // two channels a load where every row starts at one
    const bool vec = aligned(a.q, 2 * sizeof(E)) && aligned(a.k, 2 * sizeof(E)) && a.row_stride % 2 == 0 && aligned(a.log_decay, 8);
    return vec ? launch_chunks_as<D, NW, E, true>(ctx, a, sequences) : launch_chunks_as<D, NW, E, false>(ctx, a, sequences);
}

template <typename E>
int launch_prefill(k3xb_ctx* ctx, const SeqArgs& a, uint32_t sequences, uint32_t d) {
    switch (d) {
        case 32: return launch_chunk<32, 2, E>(ctx, a, sequences);
        case 64: return launch_chunk<64, 4, E>(ctx, a, sequences);
        default: return launch_chunk<128, 4, E>(ctx, a, sequences);
    }
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
    SeqArgs a{q, k, v, row_stride, log_decay, beta, offsets, nullptr, tokens, heads, sequences, state, state_out, out, ctx->status_word, 0, ~0u};
    if (const int st = check_seq(ctx, "kda_prefill", type, sequences, heads, head_dim, a)) return st;
    PhaseScope ph(ctx, K3XB_PHASE_KDA_RECURRENCE);
    ++ctx->stats.kda_calls;
    const bool f32 = type == K3XB_TYPE_F32;
    if (tokens <= 16ull * sequences || sequences >= 16) {
        // Short sequences are likely, or there may be many beside long ones: up to
        // 8 tokens go token by token, the others in chunks (a chunk costs the same
        // for 1 as for 16: 64 sequences of 32 heads take 55, 76 and 134 us with 1, 4
        // and 8 tokens each and 136 to 140 in chunks, 300 take 229, 404, 596 and 589
        // to 609, 16 take 12, 21, 31 and 40). Where there are none this costs a
        // launch beside the first kernel's start.
        a.below = kShort;
        if (const int st = f32 ? launch_seq<float>(ctx, a, sequences, head_dim) : launch_seq<__nv_bfloat16>(ctx, a, sequences, head_dim))
            return st;
        if (tokens < kShort) return K3XB_OK;
        a.from = kShort;
        a.below = ~0u;
    }
    return f32 ? launch_prefill<float>(ctx, a, sequences, head_dim) : launch_prefill<__nv_bfloat16>(ctx, a, sequences, head_dim);
}

int k3xb_kda_step(k3xb_ctx* ctx, const void* q, const void* k, const void* v, uint64_t row_stride, int32_t type,
                  const float* log_decay, const float* beta, uint32_t sequences, uint32_t heads, uint32_t head_dim,
                  const int32_t* slots, uint32_t states, float* state, void* out) {
    K3XB_ENTER(ctx);
    if (!q || !k || !v || !log_decay || !beta || !state || !out)
        return fail(ctx, K3XB_INVALID_EXTENT, "kda_step arguments");
    if (!slots && states < sequences) return fail(ctx, K3XB_INVALID_EXTENT, "kda_step: fewer states than sequences");
    if (!row_stride) row_stride = static_cast<uint64_t>(heads) * head_dim;
    const SeqArgs a{q, k, v, row_stride, log_decay, beta, nullptr, slots, sequences, heads, states, state, state, out, ctx->status_word, 0, ~0u};
    if (const int st = check_seq(ctx, "kda_step", type, sequences, heads, head_dim, a)) return st;
    PhaseScope ph(ctx, K3XB_PHASE_KDA_RECURRENCE);
    ++ctx->stats.kda_calls;
    return type == K3XB_TYPE_F32 ? launch_seq<float>(ctx, a, sequences, head_dim)
                                 : launch_seq<__nv_bfloat16>(ctx, a, sequences, head_dim);
}

}  // extern "C"
