// prefix_attn_tc.cu — the tensor-core form of the shared-prefix attention
// (bf16 and f16, key parts of 64 or 128 and values of 64 or 128).
//
// The rows of one kv head are r = (sequence * N + node) * group + g, R in
// all. Three kernels:
//
// 1. prefix_kernel: all R rows against the prefix, 128 rows a tile on
//    tcgen05, so that a prefix row crosses HBM once for up to 256 rows. The
//    work is one flat list of 128-key steps over (kv head, row tiles), cut
//    into equal ranges, one per CTA; a range that ends inside a row tile
//    leaves a part: the running maximum m (less kLift), sum l and
//    unnormalised output o of its keys. One sequence's short prefix goes
//    with 2 instead.
// 2. own_kernel: a sequence's own rows and its draft rows for 16 rows at a
//    time on mma.sync (a sequence has few rows; the bound is the read of its
//    cache). It runs beside the tail of 1 and then joins the parts:
//       M = max m_i,  out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.
// 3. join_kernel, only where 2 may split long caches into several CTAs, for
//    the sequences that it did split.
//
// Scores stay float; m is kept in log2 units (score * scale * log2 e).
//
// Measured (one B200, 32 heads, keys of 128 + 64, values of 128, prefix 16384):
// 64 x 9 rows a head: prefix_kernel 198 us (0.97 PFLOP/s of tensor work, 58% of
// the measured peak), own_kernel 66 us; 64 rows: 60 us (4.5 TB/s) and 49 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "kernels.cuh"
#include "prefix_attn.cuh"
#include "tc.cuh"

namespace k3xb {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
template <bool BF16>
constexpr float kLazy = BF16 ? 8.0f : 2.0f;
template <bool BF16>
constexpr float kLift = BF16 ? 0.0f : 13.0f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

// Two floats in one register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t pair_bits(uint32_t x, uint32_t y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y));
    return r;
}
__device__ __forceinline__ uint64_t pair_of(float x, float y) { return pair_bits(__float_as_uint(x), __float_as_uint(y)); }
__device__ __forceinline__ void split_pair(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

// Two floats rounded to the 16-bit type, `lo` in the low half.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// ---- the split of the prefix ---------------------------------------------------

constexpr uint32_t kTile = 128;          // rows and keys of a tile
constexpr uint32_t kAtom = kTile * 128;  // bytes of 128 rows x 64 values
constexpr uint32_t kMaxSlots = 12;       // ring slots of one atom
constexpr uint32_t kFullBars = 16;       // more than the blocks that the ring can hold
// Three warpgroups, launched with 168 registers a thread (64,512 in all):
// the two softmax ones take 208, the third keeps 88 (64,512).
constexpr uint32_t kPrefixThreads = 384;

// Row tiles are taken in pairs that share a step's keys; a last odd tile
// takes two key blocks a step instead, one per half of the CTA.
struct PrefixPlan {
    uint32_t rows, group;
    uint32_t blocks;           // 128-key blocks of the prefix
    uint32_t pairs, odd;       // row tile pairs; 1: a last single tile
    uint32_t steps_per_head;
    uint32_t range, max_seg;   // steps of a CTA; parts it may leave
    uint32_t total;            // steps in all; 0: no prefix
};

// A (kv head, row tile pair) and where its steps lie in the flat list.
struct Job {
    uint32_t head, pair, index, begin, steps;
};
__device__ __forceinline__ Job job_of(const PrefixPlan& p, uint32_t step) {
    Job j;
    j.head = step / p.steps_per_head;
    j.pair = min((step - j.head * p.steps_per_head) / p.blocks, p.pairs);
    j.index = j.head * (p.pairs + p.odd) + j.pair;
    j.begin = j.head * p.steps_per_head + j.pair * p.blocks;
    j.steps = j.pair < p.pairs ? p.blocks : (p.blocks + 1) / 2;
    return j;
}

struct Parts {
    float* o;     // [cta][seg][half][128][value]
    float2* ml;   // [cta][seg][half][128]: m, l
};

struct PrefixBars {
    uint64_t full[kFullBars], empty[kMaxSlots], s_full[2], p_ready[2][2], q_ready[2], o_done[2], teardown;
    uint32_t tmem_base;
    int abort;
};

__host__ __device__ constexpr uint32_t ring_slots(uint32_t key_atoms) { return key_atoms == 3 ? 8 : key_atoms == 2 ? 10 : 12; }
constexpr size_t prefix_smem(uint32_t key_atoms) {
    return (2 * key_atoms + ring_slots(key_atoms)) * size_t(kAtom) + sizeof(PrefixBars) + 1024;
}

// One segment of a CTA's range: steps [first, first + n) of a job. In key
// mode half t of the CTA takes block 2 * step + t, else both take block
// `step`; active(t) counts the steps in which the half has a block.
struct Segment {
    Job job;
    uint32_t first, n;
    bool keys;
    __device__ __forceinline__ uint32_t active(uint32_t t, uint32_t blocks) const {
        if (!keys || t == 0) return n;
        return 2 * (first + n - 1) + 1 < blocks ? n : n - 1;
    }
    __device__ __forceinline__ uint32_t block(uint32_t t, uint32_t i) const { return keys ? 2 * (first + i) + t : first + i; }
};
__device__ __forceinline__ Segment segment_at(const PrefixPlan& p, uint32_t x, uint32_t end) {
    Segment s;
    s.job = job_of(p, x);
    s.first = x - s.job.begin;
    s.n = min(end, s.job.begin + s.job.steps) - x;
    s.keys = s.job.pair == p.pairs;
    return s;
}

// A wait that runs out sets the abort flag; every later one returns at once
// then, the loops run to their end on what is in memory (the loads stop), and
// the status word reports it.
//
// What bounds a step (two tiles of 128 x 128 scores: 40 MMAs of 64 cycles = 2560
// cycles; measured 5200): an S product reads both operands from shared memory
// at its full 128 bytes a cycle, so the 80 KB that the loads write per step cost
// it 640 cycles more, and about 900 go in the way scores - softmax -
// probabilities - product that the other half's products do not cover (without
// loads and softmax the same issue order takes 3600 cycles).
//
// Warps 0-3 and 4-7 are the softmax of row tile (or key half) 0 and 1, a
// thread per row; warp 8 loads, warp 9 issues the MMAs (10 and 11 only fill
// the warpgroup). TMEM: output 0, 1 and scores 0, 1, 128 columns each; the
// probabilities overwrite the scores they come from (two per column), and the
// next score tile is issued behind the product that reads them.
//
// The running maximum is lazy: rows keep an old m until a score passes it by
// more than kLazy powers of two, so that the accumulator is rescaled a few times
// per row instead of once per block (p <= 2^8 of it then with bf16, 2^2 with
// f16). The sum is of the unrounded p. f16 ends at 2^-24: there the base that p
// is relative to lies kLift powers below m, so that p ends at 2^15 and keeps its
// 11 bits down to 2^-27 of the largest, and 2^-38 of it is the least that counts.
template <bool BF16, uint32_t NK, uint32_t NV>
__global__ void __launch_bounds__(kPrefixThreads, 1) prefix_kernel(const __grid_constant__ CUtensorMap map_k,
                                                        const __grid_constant__ CUtensorMap map_e,
                                                        const __grid_constant__ CUtensorMap map_v,
                                                        const __grid_constant__ AttnArgs a, const PrefixPlan p,
                                                        const Parts parts) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr uint32_t slots = ring_slots(NK), value = 64 * NV;
    uint8_t* q_smem = base;                       // [2][NK] atoms
    uint8_t* ring = base + 2 * NK * kAtom;        // [slots] atoms
    PrefixBars& bar = *reinterpret_cast<PrefixBars*>(ring + slots * kAtom);
    volatile int* abort = &bar.abort;
    // the shuffle tells the compiler that a warp agrees on its role
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    asm volatile("griddepcontrol.launch_dependents;");
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kFullBars; ++s) tc::mbar_init(&bar.full[s], 1);
        for (uint32_t s = 0; s < slots; ++s) tc::mbar_init(&bar.empty[s], 1);
        for (uint32_t t = 0; t < 2; ++t) {
            tc::mbar_init(&bar.s_full[t], 1);
            tc::mbar_init(&bar.p_ready[t][0], 4);
            tc::mbar_init(&bar.p_ready[t][1], 4);
            tc::mbar_init(&bar.q_ready[t], 4);
            tc::mbar_init(&bar.o_done[t], 1);
        }
        tc::mbar_init(&bar.teardown, 1);
        bar.abort = 0;
        tc::fence_barrier_init();
    }
    if (warp == 9) tc::tmem_alloc(&bar.tmem_base, 512);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = bar.tmem_base;
    const uint32_t lo = blockIdx.x * p.range, hi = min(p.total, lo + p.range);

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8 && lane == 0) {
            // ---------------- loads, in the order the MMAs use them ----------------
            const uint32_t nm = a.main / 64;
            uint32_t pos = 0, blk = 0;   // atoms and key or value blocks so far
            bool ok = true;
            // slots for a block's N atoms; its barrier counts their bytes
            auto begin = [&](uint32_t n) {
                for (uint32_t i = 0; i < n; ++i)
                    ok = ok && tc::mbar_wait(&bar.empty[(pos + i) % slots], (((pos + i) / slots) & 1u) ^ 1u, abort);
                if (ok) tc::mbar_arrive_expect_tx(&bar.full[blk++ % kFullBars], n * kAtom);
                return ok;
            };
            auto load_k = [&](uint32_t head, uint32_t block) {
                uint64_t* full = &bar.full[blk % kFullBars];
                if (!begin(NK)) return;
#pragma unroll
                for (uint32_t i = 0; i < NK; ++i, ++pos) {
                    uint8_t* dst = ring + pos % slots * kAtom;
                    if (i < nm) tc::tma_load_3d(dst, &map_k, full, i * 128, head, block * kTile);
                    else tc::tma_load_3d(dst, &map_e, full, 0, 0, block * kTile);
                }
            };
            auto load_v = [&](uint32_t head, uint32_t block) {
                uint64_t* full = &bar.full[blk % kFullBars];
                if (!begin(NV)) return;
#pragma unroll
                for (uint32_t i = 0; i < NV; ++i, ++pos)   // an atom: 64 keys of 128 values, or 128 keys of 64
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e)
                        tc::tma_load_3d(ring + pos % slots * kAtom + e * (kAtom / 2), &map_v, full, NV == 2 ? e * 128 : 0, head,
                                        block * kTile + (NV == 2 ? i : e) * 64);
            };
            for (uint32_t x = lo; x < hi && ok;) {
                const Segment s = segment_at(p, x, hi);
                const uint32_t h = s.job.head, n1 = s.active(1, p.blocks);
                load_k(h, s.block(0, 0));
                if (s.keys && n1) load_k(h, s.block(1, 0));
                for (uint32_t i = 0; i < s.n && ok; ++i) {
                    load_v(h, s.block(0, i));
                    if (i + 1 < s.n) load_k(h, s.block(0, i + 1));
                    if (s.keys && i < n1) {
                        load_v(h, s.block(1, i));
                        if (i + 1 < n1) load_k(h, s.block(1, i + 1));
                    }
                }
                x += s.n;
            }
            volatile int never = 0;   // these waits must not be cut short by the abort flag
            for (uint32_t i = 0; i < slots && i < blk; ++i) {
                const uint32_t j = blk - 1 - i;
                tc::mbar_wait(&bar.full[j % kFullBars], (j / kFullBars) & 1u, &never, 200000000ull);
            }
        } else if (warp == 9) {
            // ---------------- MMA issue, by one lane of the whole warp ----------------
            constexpr uint32_t id_s = tc::idesc_f16(kTile, BF16, false), id_o = tc::idesc_f16(value, BF16, true);
            const uint64_t q0 = tc::desc_sw128(q_smem), k0 = tc::desc_sw128(ring), v0 = tc::desc_sw128_n(ring, kAtom / 2);
            uint32_t pos = 0, blk = 0, seg = 0, p_phase = 0;   // atoms, blocks, segments; bit t: phase of p_ready[t]
            uint32_t ka = 0, va = 0;                           // where the key and value blocks in use start
            auto next_k = [&]() {
                tc::mbar_pass(&bar.full[blk % kFullBars], blk / kFullBars & 1u, abort);
                ++blk;
                ka = pos;
                pos += NK;
            };
            auto next_v = [&]() {
                tc::mbar_pass(&bar.full[blk % kFullBars], blk / kFullBars & 1u, abort);
                ++blk;
                va = pos;
                pos += NV;
            };
            // scores of half t from the key block at ka
            auto scores = [&](uint32_t t, bool release) {
                tc::fence_after_sync();
                if (tc::elect_one()) {
#pragma unroll
                    for (uint32_t i = 0; i < NK; ++i) {
                        const uint32_t st = (ka + i) % slots;
                        const uint64_t qd = q0 + (t * NK + i) * (kAtom >> 4), kd = k0 + st * (kAtom >> 4);
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) tc::mma_bf16(tmem + 256 + t * 128, qd + 2 * j, kd + 2 * j, id_s, i || j);
                        if (release) tc::commit(&bar.empty[st]);
                    }
                    tc::commit(&bar.s_full[t]);
                }
                __syncwarp();
            };
            // output of half t: its probabilities times the value block at
            // va, 64 keys at a time (the softmax hands them over so)
            auto values = [&](uint32_t t, bool accumulate, bool release, bool last) {
                const uint32_t d = tmem + t * 128, pr = tmem + 256 + t * 128;
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    const uint32_t st = (va + (NV == 2 ? i : 0)) % slots;
                    const uint64_t vd = v0 + st * (kAtom >> 4) + (NV == 2 ? 0 : i * (kAtom >> 5));
                    tc::mbar_pass(&bar.p_ready[t][i], p_phase >> t & 1u, abort);
                    tc::fence_after_sync();
                    if (tc::elect_one()) {
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j)   // 16 keys: 8 columns of p, 2 KB of values
                            tc::mma_f16_ts(d, pr + 32 * i + 8 * j, vd + 128 * j, id_o, i || j ? 1u : accumulate);
                        if (release && (NV == 2 || i)) tc::commit(&bar.empty[st]);
                        if (last && i) tc::commit(&bar.o_done[t]);
                    }
                    __syncwarp();
                }
                p_phase ^= 1u << t;
            };
            for (uint32_t x = lo; x < hi; ++seg) {
                const Segment s = segment_at(p, x, hi);
                const uint32_t n1 = s.active(1, p.blocks);
                for (uint32_t t = 0; t < 2; ++t) tc::mbar_pass(&bar.q_ready[t], seg & 1u, abort);
                next_k();
                scores(0, s.keys);
                if (n1) {
                    if (s.keys) next_k();
                    scores(1, true);
                }
                for (uint32_t i = 0; i < s.n; ++i) {
                    next_v();
                    values(0, i > 0, s.keys, i + 1 == s.n);
                    if (i + 1 < s.n) {
                        next_k();
                        scores(0, s.keys);
                    }
                    if (i >= n1) continue;
                    if (s.keys) next_v();
                    values(1, i > 0, true, i + 1 == n1);
                    if (i + 1 < n1) {
                        if (s.keys) next_k();
                        scores(1, true);
                    }
                }
                if (!n1 && tc::elect_one()) tc::commit(&bar.o_done[1]);   // keeps the halves' phases in step
                __syncwarp();
                x += s.n;
            }
            volatile int never = 0;   // all issued MMAs finish before TMEM is freed
            if (tc::elect_one()) tc::commit(&bar.teardown);
            __syncwarp();
            tc::mbar_wait(&bar.teardown, 0, &never, 200000000ull);
            __syncwarp();
        }
    } else {
        // ---------------- softmax ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const uint32_t t = warp / 4, tid = threadIdx.x % 128, row = tid;
        const uint32_t lanes = (32u * (warp % 4)) << 16;
        const uint32_t scores_at = tmem + lanes + 256 + t * 128, out_at = tmem + lanes + t * 128;
        const float c = fabsf(a.scale) * kLog2e;
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;   // a negative scale: -q
        uint32_t s_uses = 0, seg = 0;
        auto wait = [&](uint64_t* b, uint32_t parity) {
            tc::mbar_pass(b, parity, abort);
            __syncwarp();
            tc::fence_after_sync();
        };
        auto arrive = [&](uint64_t* b) {   // one for the warp: arrivals on a barrier are taken one by one
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(b);
        };
        for (uint32_t x = lo; x < hi; ++seg) {
            const Segment s = segment_at(p, x, hi);
            const uint32_t tile = 2 * s.job.pair + (s.keys ? 0 : t), n = s.active(t, p.blocks);
            // the tile's query rows, swizzled as the MMA reads them: eight
            // threads a row, the loads of four rows in flight
            {
                const uint32_t ch = tid % 8;
#pragma unroll
                for (uint32_t r0 = tid / 8; r0 < kTile; r0 += 64) {
                    uint4 w[4][NK];
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u) {
                        const uint32_t gr = tile * kTile + r0 + 16 * u;
                        const uint64_t at = gr / p.group * a.q_row +
                                            static_cast<uint64_t>(s.job.head * p.group + gr % p.group) * (64 * NK);
#pragma unroll
                        for (uint32_t i = 0; i < NK; ++i) {
                            w[u][i] = make_uint4(0, 0, 0, 0);
                            if (gr < p.rows)
                                w[u][i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + at) + 8 * i + ch);
                        }
                    }
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u) {
                        const uint32_t r = r0 + 16 * u;
#pragma unroll
                        for (uint32_t i = 0; i < NK; ++i)
                            *reinterpret_cast<uint4*>(q_smem + (t * NK + i) * kAtom + r * 128 + ((ch ^ (r % 8)) << 4)) =
                                make_uint4(w[u][i].x ^ flip, w[u][i].y ^ flip, w[u][i].z ^ flip, w[u][i].w ^ flip);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(&bar.q_ready[t]);
            float m = -INFINITY, l = 0.0f;
            for (uint32_t i = 0; i < n; ++i) {
                wait(&bar.s_full[t], s_uses++ & 1u);
                uint32_t v[128];
#pragma unroll
                for (int j = 0; j < 4; ++j) tc::tmem_ld32(scores_at + 32 * j, v + 32 * j);
                tc::tmem_wait_ld();
                const uint32_t valid = min(kTile, a.prefix_len - s.block(t, i) * kTile);
                if (valid < kTile)
#pragma unroll
                    for (int j = 0; j < 128; ++j)
                        if (j >= static_cast<int>(valid)) v[j] = 0xff800000u;
                float top[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) top[j] = __uint_as_float(v[j]);
#pragma unroll
                for (int j = 4; j < 124; j += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(v[j + e]), __uint_as_float(v[j + 4 + e]));
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], __uint_as_float(v[124 + e]));
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
                if (i == 0) {
                    m = mx;
                } else if (__any_sync(0xffffffffu, mx > m + kLazy<BF16>)) {
                    // the product of the block before is done: its scores' successor is
                    const float mn = mx > m + kLazy<BF16> ? mx : m;
                    const float keep = mn == -INFINITY ? 1.0f : ex2(m - mn);
                    l *= keep;
                    m = mn;
                    for (uint32_t cc = 0; cc < value; cc += 16) {
                        float o[16];
                        tc::tmem_ld16(out_at + cc, o);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] *= keep;
                        tc::tmem_st16(out_at + cc, o);
                    }
                }
                const float off = m == -INFINITY ? 0.0f : m - kLift<BF16>;
                // x * c - off for two columns at a time, the sums too
                const uint64_t c2 = pair_of(c, c), off2 = pair_of(-off, -off);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float p0, p1;
                        split_pair(fma2(pair_bits(v[32 * q4 + 2 * j], v[32 * q4 + 2 * j + 1]), c2, off2), p0, p1);
                        p0 = ex2(p0);
                        p1 = ex2(p1);
                        sum[j % 2] = add2(sum[j % 2], pair_of(p0, p1));
                        w[j] = pack2<BF16>(p0, p1);
                    }
                    tc::tmem_st16(scores_at + 16 * q4, w);
                    if (q4 % 2) {   // 64 keys for the product
                        tc::tmem_wait_st();
                        arrive(&bar.p_ready[t][q4 / 2]);
                    }
                }
                float s0, s1;
                split_pair(add2(sum[0], sum[1]), s0, s1);
                l += s0 + s1;
            }
            // the segment's part
            const size_t part = (static_cast<size_t>(blockIdx.x) * p.max_seg + seg) * 2 + t;
            parts.ml[part * kTile + row] = make_float2(m - kLift<BF16>, l);
            wait(&bar.o_done[t], seg & 1u);
            if (n) {
                // through the tile's query rows, which no product reads any
                // more: a thread has a row, a store should have a few (16-byte
                // chunk c of row r stands at c ^ r)
                constexpr uint32_t cols = NK > 1 ? 64 : 32, chunks = cols / 4;
                float4* stage = reinterpret_cast<float4*>(q_smem + t * NK * kAtom) + (warp % 4) * 32 * chunks;
                float* dst = parts.o + (part * kTile + 32 * (warp % 4)) * value;
                const uint32_t rows = min(32u, p.rows - min(p.rows, tile * kTile + 32 * (warp % 4)));
                for (uint32_t cc = 0; cc < value; cc += cols) {
#pragma unroll
                    for (uint32_t c0 = 0; c0 < cols; c0 += 32) {
                        uint32_t o[32];
                        tc::tmem_ld32(out_at + cc + c0, o);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (uint32_t j = 0; j < 8; ++j)
                            stage[lane * chunks + ((c0 / 4 + j) ^ (lane % chunks))] =
                                make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]), __uint_as_float(o[4 * j + 2]),
                                            __uint_as_float(o[4 * j + 3]));
                    }
                    __syncwarp();
#pragma unroll 4
                    for (uint32_t r = lane / chunks; r < rows; r += 32 / chunks)
                        *reinterpret_cast<float4*>(dst + r * value + cc + lane % chunks * 4) =
                            stage[r * chunks + ((lane % chunks) ^ (r % chunks))];
                    __syncwarp();
                }
                asm volatile("bar.sync %0, 128;" ::"r"(1 + static_cast<int>(t)) : "memory");   // before the next queries
                tc::fence_before_sync();
            }
            x += s.n;
        }
    }
    __syncthreads();
    if (*abort && threadIdx.x == 0) atomicExch(a.status, K3XB_BACKEND_UNAVAILABLE);
    if (warp == 9) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, 512);
    }
}

// ---- own rows, draft rows and the join --------------------------------------------

__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1, bool bf16) {
    if (bf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}

struct OwnPlan {
    uint32_t row_tiles;   // 16-row tiles of a sequence's rows per kv head
    uint32_t splits;      // tasks along a sequence's keys, where it is long enough
    uint32_t least;       // tiles of 16 keys that a task has at least
    uint32_t tasks;       // [kv head][row tile][split] of a sequence
    uint32_t warps;       // 1 or 4 to a task
    uint32_t prefix;      // 1: the tasks read the prefix too
    float* o;             // [seq][kv head][row tile][split][16][value] where splits > 1
    float2* ml;           // [seq][kv head][row tile][split][16]
};

// The tasks that a sequence's keys are split into: what its length on the
// device asks for (the host knows the cache's capacity only).
__device__ __forceinline__ uint32_t splits_of(const OwnPlan& own, uint32_t tiles) { return max(1u, min(own.splits, tiles / own.least)); }
__device__ __forceinline__ uint32_t tiles_of(const AttnArgs& a, const OwnPlan& own, int32_t len, uint32_t& prefix) {
    prefix = own.prefix && len >= 0 ? (a.prefix_len + 15) / 16 : 0;
    return len < 0 ? 0 : prefix + (static_cast<uint32_t>(len) + a.N + 15) / 16;
}

// A running join of parts for one row and C of its columns.
template <int C>
struct Join {
    float m = -INFINITY, l = 0.0f, o[C];
    __device__ __forceinline__ Join() {
#pragma unroll
        for (int i = 0; i < C; ++i) o[i] = 0.0f;
    }
    __device__ __forceinline__ void add(float2 ml, const float (&x)[C]) {
        if (ml.x == -INFINITY && ml.y == 0.0f) return;   // no visible key: o was never written
        const float mn = fmaxf(m, ml.x), at = mn == -INFINITY ? 0.0f : mn;
        const float w0 = ex2(m - at), w1 = ex2(ml.x - at);
        l = fmaf(l, w0, ml.y * w1);
        m = mn;
#pragma unroll
        for (int i = 0; i < C; ++i) o[i] = fmaf(o[i], w0, x[i] * w1);
    }
};
template <int C>
__device__ __forceinline__ void load_cols(const float* src, float (&x)[C]) {
    if constexpr (C == 4) {
        const float4 v = *reinterpret_cast<const float4*>(src);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
        const float2 v = *reinterpret_cast<const float2*>(src);
        x[0] = v.x; x[1] = v.y;
    }
}

// The prefix's parts of one row of a kv head, as rows of Parts (32-bit: the
// host checks their count).
struct RowParts {
    uint32_t first, second, step;   // rows of the first CTA's part and the next one's; from CTA to CTA
    uint32_t n, pairs;              // parts; 1: two halves to a CTA
    __device__ __forceinline__ RowParts(const PrefixPlan& p, uint32_t h, uint32_t r) {
        const uint32_t tile = r / kTile, pair = min(tile / 2, p.pairs);
        const bool keys = pair == p.pairs;
        const uint32_t begin = h * p.steps_per_head + pair * p.blocks;
        const uint32_t end = begin + (keys ? (p.blocks + 1) / 2 : p.blocks);
        const uint32_t c0 = begin / p.range, c1 = (end - 1) / p.range;
        // the job is one of the segments of CTA c0 and the first one of the CTAs behind it
        const uint32_t seg0 = h * (p.pairs + p.odd) + pair - job_of(p, c0 * p.range).index;
        pairs = keys ? 1 : 0;
        n = (c1 - c0 + 1) << pairs;
        step = p.max_seg * 2 * kTile;
        second = (c0 + 1) * step + (keys ? 0 : tile % 2) * kTile + r % kTile;
        first = second - step + seg0 * 2 * kTile;
    }
    __device__ __forceinline__ uint32_t part(uint32_t i) const {
        const uint32_t c = i >> pairs, half = (i & pairs) * kTile;
        return half + (c ? second + (c - 1) * step : first);
    }
};

// Joins the prefix's parts to two rows' sums, a lane C columns, up to eight
// loads in flight.
template <int C>
__device__ __forceinline__ void join_prefix(Join<C> (&j)[2], const PrefixPlan& p, const Parts& parts, uint32_t h, const uint32_t (&r)[2],
                                            const bool (&there)[2], uint32_t col, uint32_t value) {
    RowParts rows[2] = {RowParts(p, h, r[0]), RowParts(p, h, r[0])};
    rows[1].first += r[1] - r[0];
    rows[1].second += r[1] - r[0];
    if (r[1] / kTile != r[0] / kTile) rows[1] = RowParts(p, h, r[1]);
    const uint32_t n[2] = {there[0] ? rows[0].n : 0, there[1] ? rows[1].n : 0}, most = max(n[0], n[1]);
    for (uint32_t i0 = 0; i0 < most; i0 += 4) {
        float x[2][4][C];
        float2 ml[2][4];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (i0 + i < n[k]) {
                    const uint32_t at = rows[k].part(i0 + i);
                    ml[k][i] = parts.ml[at];
                    load_cols<C>(parts.o + static_cast<size_t>(at) * value + col, x[k][i]);
                }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (i0 + i < n[k]) j[k].add(ml[k][i], x[k][i]);
    }
}

template <bool BF16, int C>
__device__ __forceinline__ void write_row(const AttnArgs& a, const Join<C>& j, uint32_t s, uint32_t node, uint32_t head,
                                          uint32_t col) {
    const size_t row = (static_cast<size_t>(s) * a.N + node) * a.heads + head;
    const float inv = j.l == 0.0f ? 0.0f : 1.0f / j.l;   // nothing visible: a zero row
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + row * a.value + col);
#pragma unroll
    for (int i = 0; i < C / 2; ++i) dst[i] = pack2<BF16>(j.o[2 * i] * inv, j.o[2 * i + 1] * inv);
    if (a.lse && col == 0) a.lse[row] = j.l == 0.0f ? -INFINITY : (j.m + __log2f(j.l)) * kLn2;
}

// Replaces the infinities and NaN of two values by zeros.
template <bool BF16>
__device__ __forceinline__ void drop_nonfinite(uint32_t& w) {
    constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
    if ((w & e) == e) w &= 0xffff0000u;
    if ((w >> 16 & e) == e) w &= 0x0000ffffu;
}

// acc + 0 * w in both halves: zeros as long as every w was finite.
template <bool BF16>
__device__ __forceinline__ uint32_t add_zero_times(uint32_t w, uint32_t acc) {
    uint32_t r;
    if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(acc));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(acc));
    return r;
}

template <bool BF16>
__device__ __forceinline__ float half_of(uint16_t w) {
    if constexpr (BF16) return decode_bf16(w);
    else return __half2float(__ushort_as_half(w));
}

constexpr uint32_t kOwnThreads = 128;

// A task is 16 rows of one sequence and kv head (and a split of its keys), 16
// keys at a time: one warp's where there are many tasks, four warps' that
// take tiles in turn where there are few. Key and value rows go straight from
// global memory to MMA fragments, 16 bytes a lane: the contraction over key
// dimensions may run in any order, so lane t of a quad reads 8 neighbouring
// dimensions and feeds them to two steps of 16 (the queries are read alike),
// and value column g of an output tile j stands for dimension 8 g + j.
//
// Draft rows are masked by the node's ancestors. A masked key's probability
// is zero, but zero times a value that is infinite or NaN is not, so the
// product takes such values of draft rows as zeros, and the rows that do see
// them add them one by one.
template <int DQ, int DV, bool BF16, uint32_t W>
__global__ void __launch_bounds__(kOwnThreads, DQ + DV <= 192 ? 3 : 2) own_kernel(const __grid_constant__ AttnArgs a, const PrefixPlan p,
                                                          const Parts parts, const OwnPlan own) {
    constexpr int SEG = DQ / 32, H = DV / 64, LD = DV + 4;
    // a warp's output rows; before, a task's queries as each lane's fragments
    // need them ([SEG][2][32] of 16 bytes, at its first warp's rows)
    constexpr int WARP = 16 * LD > SEG * 256 ? 16 * LD : SEG * 256;
    __shared__ __align__(16) float buf[4][WARP];
    __shared__ float2 sm_ml[4][16];
    const uint32_t all = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    float (*sm_o)[LD] = reinterpret_cast<float (*)[LD]>(buf[all]);
    uint4 (*sm_q)[2][32] = reinterpret_cast<uint4 (*)[2][32]>(buf[all / W * W]);
    const uint32_t warp = all % W, mine = all / W, rows_at = blockIdx.x * (4 / W) + mine;   // warp of a task; task of the CTA
    if (rows_at >= a.kv_heads * own.row_tiles) return;   // a whole warp (W = 1); with W = 4 there is a CTA per task
    auto sync = [&] {
        if constexpr (W == 1) __syncwarp();
        else __syncthreads();
    };
    // splits come last: where sequences are short, theirs have nothing to do
    const uint32_t split = blockIdx.z, rt = rows_at % own.row_tiles, h = rows_at / own.row_tiles, s = blockIdx.y;
    const uint32_t task = rows_at * own.splits + split;
    const uint32_t group = a.heads / a.kv_heads, rows = a.N * group;
    const int32_t len = own_rows(a, s);
    const float c = fabsf(a.scale) * kLog2e;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    // this task's tiles of 16 keys: first the prefix's, where they are read
    // here, then the sequence's own
    uint32_t pre;
    const uint32_t tiles = tiles_of(a, own, len, pre), splits = splits_of(own, tiles);
    if (split >= splits) return;   // (those that there are wait for the prefix kernel, and thus this kernel's end)
    const uint32_t per_split = (tiles + splits - 1) / splits, end = min(tiles, (split + 1) * per_split);
    uint32_t tile = split * per_split + warp;

    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4 kr[2][SEG], vr[4][H];
    // this lane's pieces of the tile to load, taken along by pointers (an
    // address from 64-bit strides costs a dozen instructions a load)
    const uint32_t main_seg = a.main / 32;
    const uint16_t *kp[2], *ep[2], *vp[4];
    uint64_t k_step, e_step, v_step;
    auto aim = [&](uint32_t i) {   // at tile i of its source
        const KvSource& x = i < pre ? a.prefix : a.suffix;
        const uint64_t seq = i < pre ? 0 : s, k0 = (i < pre ? i : i - pre) * 16ull;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint64_t key = k0 + 8 * e + g;
            kp[e] = static_cast<const uint16_t*>(x.k) + seq * x.k_seq + h * x.k_head + key * x.k_row + t * 8;
            ep[e] = static_cast<const uint16_t*>(x.extra) + seq * x.extra_seq + key * x.extra_row + t * 8 - a.main;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            vp[e] = static_cast<const uint16_t*>(x.v) + seq * x.v_seq + h * x.v_head + (k0 + 2 * t + (e & 1) + 8 * (e >> 1)) * x.v_row + g * 8;
        k_step = 16 * W * x.k_row;
        e_step = 16 * W * x.extra_row;
        v_step = 16 * W * x.v_row;
    };
    // keys of tile i's source from its first one on
    auto left = [&](uint32_t i) { return i < pre ? a.prefix_len - i * 16 : static_cast<uint32_t>(len) + a.N - (i - pre) * 16; };
    auto load_k = [&](uint32_t n) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const bool in = 8 * x + g < n;
#pragma unroll
            for (int j = 0; j < SEG; ++j) {
                const uint16_t* src = j < 2 || static_cast<uint32_t>(j) < main_seg ? kp[x] : ep[x];   // main_dim is 64 at least
                kr[x][j] = in ? __ldg(reinterpret_cast<const uint4*>(src + j * 32)) : zero;
            }
        }
    };
    auto load_v = [&](uint32_t n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const bool in = 2 * t + (x & 1) + 8 * (x >> 1) < n;
#pragma unroll
            for (int j = 0; j < H; ++j) vr[x][j] = in ? __ldg(reinterpret_cast<const uint4*>(vp[x] + j * 64)) : zero;
        }
    };
    auto advance = [&](uint32_t i) {   // from tile i - W to tile i
        if (i >= pre && i - W < pre) {
            aim(i);
            return;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            kp[x] += k_step;
            ep[x] += e_step;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) vp[x] += v_step;
    };
    // the first tile's rows come while the queries do, a later one's while
    // the tile before is worked on
    if (tile < end) {
        aim(tile);
        load_k(left(tile));
        load_v(left(tile));
    }
    uint64_t seen[2];   // draft rows that rows g and g + 8 see
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t r = rt * 16 + g + 8 * i;
        const bool there = r < rows;
        const uint32_t node = there ? r / group : 0;
        seen[i] = there ? a.ancestors[node] : 0;
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + (static_cast<size_t>(s) * a.N + node) * a.q_row +
                              static_cast<size_t>(h * group + r % group) * DQ + t * 8;
        for (uint32_t j = warp; j < SEG; j += W) {
            uint4 w = zero;
            if (there) w = __ldg(reinterpret_cast<const uint4*>(src + j * 32));
            sm_q[j][i][lane] = make_uint4(w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip);
        }
    }
    sync();
    float o[H][8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < H; ++x)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[x][j][e] = 0.0f;

    for (; tile < end; tile += W) {
        const bool own_tile = tile >= pre, more = tile + W < end;
        const uint32_t n = left(tile), k0 = own_tile ? (tile - pre) * 16 : 0;
        float sc[2][4] = {};
#pragma unroll
        for (int j = 0; j < SEG; ++j) {
            const uint4 q0 = sm_q[j][0][lane], q1 = sm_q[j][1][lane];
            const uint32_t a0[4] = {q0.x, q1.x, q0.y, q1.y}, a1[4] = {q0.z, q1.z, q0.w, q1.w};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                mma16(sc[x], a0, kr[x][j].x, kr[x][j].y, BF16);
                mma16(sc[x], a1, kr[x][j].z, kr[x][j].w, BF16);
            }
        }
        // the next tile's keys; its values when this one's are used
        if (more) {
            advance(tile + W);
            load_k(left(tile + W));
        }
        const bool drafts = own_tile && k0 + 16 > static_cast<uint32_t>(len);
        uint32_t vis = 0xffu;   // bit 4 x + e: key of sc[x][e] is visible to its row
        if (drafts) {
            vis = 0;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t at = 8 * x + 2 * t + (e & 1), key = k0 + at;
                    const bool see = key < static_cast<uint32_t>(len) || (at < n && (seen[e >> 1] >> (key - len) & 1u));
                    if (see) vis |= 1u << (4 * x + e);
                    else sc[x][e] = -INFINITY;
                }
        } else if (n < 16) {   // the prefix's last tile
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (8 * x + 2 * t + (e & 1) >= n) sc[x][e] = -INFINITY;
        }
        float top[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float v = fmaxf(fmaxf(sc[0][2 * i], sc[0][2 * i + 1]), fmaxf(sc[1][2 * i], sc[1][2 * i + 1]));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
            top[i] = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2)) * c;
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float mn = fmaxf(m[i], top[i]), keep = mn == -INFINITY ? 1.0f : ex2(m[i] - mn);
                m[i] = mn;
                l[i] *= keep;
#pragma unroll
                for (int x = 0; x < H; ++x)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        o[x][j][2 * i] *= keep;
                        o[x][j][2 * i + 1] *= keep;
                    }
            }
        }
        // p is relative to m, in f16 to kLift powers below it (as in prefix_kernel)
        const float off[2] = {m[0] == -INFINITY ? 0.0f : m[0] - kLift<BF16>, m[1] == -INFINITY ? 0.0f : m[1] - kLift<BF16>};
        float pr[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pr[x][e] = ex2(fmaf(sc[x][e], c, -off[e >> 1]));
                l[e >> 1] += pr[x][e];
            }
        uint32_t finite = 0;   // stays zero (of either sign) unless a draft row has an infinity or NaN
        if (drafts) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int j = 0; j < H; ++j) {
                    finite = add_zero_times<BF16>(vr[x][j].x, finite);
                    finite = add_zero_times<BF16>(vr[x][j].y, finite);
                    finite = add_zero_times<BF16>(vr[x][j].z, finite);
                    finite = add_zero_times<BF16>(vr[x][j].w, finite);
                }
        }
        if (drafts && __any_sync(0xffffffffu, finite & 0x7fff7fffu)) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int j = 0; j < H; ++j) {
                    drop_nonfinite<BF16>(vr[x][j].x);
                    drop_nonfinite<BF16>(vr[x][j].y);
                    drop_nonfinite<BF16>(vr[x][j].z);
                    drop_nonfinite<BF16>(vr[x][j].w);
                }
            // one key at a time: its probabilities from the lane that has
            // them, its values from memory
            for (uint32_t kk = 0; kk < min(16u, n); ++kk) {
                const uint32_t src = (lane & ~3u) | (kk % 8 / 2), bit = 4 * (kk / 8) + kk % 2;
                const uint32_t sv = __shfl_sync(0xffffffffu, vis, src);
                float pk[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float lo = kk % 2 ? pr[0][2 * i + 1] : pr[0][2 * i], hi = kk % 2 ? pr[1][2 * i + 1] : pr[1][2 * i];
                    pk[i] = __shfl_sync(0xffffffffu, kk < 8 ? lo : hi, src);
                }
                const uint16_t* row = static_cast<const uint16_t*>(a.suffix.v) + s * a.suffix.v_seq + h * a.suffix.v_head +
                                      static_cast<uint64_t>(k0 + kk) * a.suffix.v_row;
#pragma unroll
                for (int x = 0; x < H; ++x)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float v = half_of<BF16>(row[x * 64 + (2 * t + e) * 8 + j]);
                            if (isfinite(v)) continue;
                            if (sv >> bit & 1u) o[x][j][e] = fmaf(pk[0], v, o[x][j][e]);
                            if (sv >> (bit + 2) & 1u) o[x][j][2 + e] = fmaf(pk[1], v, o[x][j][2 + e]);
                        }
            }
        }
        const uint32_t pa[4] = {pack2<BF16>(pr[0][0], pr[0][1]), pack2<BF16>(pr[0][2], pr[0][3]),
                                pack2<BF16>(pr[1][0], pr[1][1]), pack2<BF16>(pr[1][2], pr[1][3])};
#pragma unroll
        for (int x = 0; x < H; ++x) {
            const uint32_t v0[4] = {vr[0][x].x, vr[0][x].y, vr[0][x].z, vr[0][x].w}, v1[4] = {vr[1][x].x, vr[1][x].y, vr[1][x].z, vr[1][x].w};
            const uint32_t v2[4] = {vr[2][x].x, vr[2][x].y, vr[2][x].z, vr[2][x].w}, v3[4] = {vr[3][x].x, vr[3][x].y, vr[3][x].z, vr[3][x].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t pick = j % 2 ? 0x7632u : 0x5410u;
                mma16(o[x][j], pa, __byte_perm(v0[j / 2], v1[j / 2], pick), __byte_perm(v2[j / 2], v3[j / 2], pick), BF16);
            }
        }
        if (more) load_v(left(tile + W));
    }
    // the task's results to rows of lanes, then the rows' parts
    sync();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (t == 0) sm_ml[all][g + 8 * i] = make_float2(m[i] - kLift<BF16>, l[i]);
#pragma unroll
        for (int x = 0; x < H; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    *reinterpret_cast<float4*>(&sm_o[g + 8 * i][x * 64 + (2 * t + e) * 8 + j]) =
                        make_float4(o[x][j][2 * i + e], o[x][j + 1][2 * i + e], o[x][j + 2][2 * i + e], o[x][j + 3][2 * i + e]);
    }
    sync();
    constexpr int C = DV / 32;
    const uint32_t col = lane * C, here = min(16u, rows - rt * 16);
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the prefix's parts
    for (uint32_t row = 2 * warp; row < here; row += 2 * W) {   // two rows at a time
        Join<C> j[2];
        const bool there[2] = {true, row + 1 < here};
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            if (!there[i]) continue;
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) {
                float x[C];
                load_cols<C>(&buf[mine * W + w][(row + i) * LD + col], x);
                j[i].add(sm_ml[mine * W + w][row + i], x);
            }
            if (splits == 1) continue;
            const size_t at = (static_cast<size_t>(s) * own.tasks + task) * 16 + row + i;
            if (lane == 0) own.ml[at] = make_float2(j[i].m, j[i].l);
#pragma unroll
            for (int e = 0; e < C; ++e) own.o[at * DV + col + e] = j[i].o[e];
        }
        if (splits > 1) continue;
        const uint32_t r[2] = {rt * 16 + row, rt * 16 + row + there[1]};
        if (p.total && len >= 0) join_prefix<C>(j, p, parts, h, {s * rows + r[0], s * rows + r[1]}, there, col, DV);
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i)
            if (there[i]) write_row<BF16>(a, j[i], s, r[i] / group, h * group + r[i] % group, col);
    }
}

// The join on its own, of sequences whose keys own_kernel split: a warp per two rows.
template <int DV, bool BF16>
__global__ void __launch_bounds__(kOwnThreads) join_kernel(const __grid_constant__ AttnArgs a, const PrefixPlan p,
                                                           const Parts parts, const OwnPlan own) {
    constexpr int C = DV / 32;
    const uint32_t rt = blockIdx.x % own.row_tiles, h = blockIdx.x / own.row_tiles, s = blockIdx.y;
    const uint32_t group = a.heads / a.kv_heads, rows = a.N * group;
    const uint32_t col = threadIdx.x % 32 * C, here = min(16u, rows - rt * 16);
    const int32_t len = own_rows(a, s);
    uint32_t pre;
    const uint32_t splits = splits_of(own, tiles_of(a, own, len, pre));
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (splits == 1) return;
    for (uint32_t row = threadIdx.x / 32 * 2; row < here; row += 8) {
        Join<C> j[2];
        const bool there[2] = {true, row + 1 < here};
        const uint32_t r[2] = {rt * 16 + row, rt * 16 + row + there[1]};
        if (len >= 0) {
            const size_t at = (static_cast<size_t>(s) * own.tasks + blockIdx.x * own.splits) * 16 + row;
            for (uint32_t k0 = 0; k0 < splits; k0 += 6) {   // six splits' loads in flight
                float x[2][6][C];
                float2 ml[2][6];
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                    for (uint32_t k = 0; k < 6; ++k)
                        if (there[i] && k0 + k < splits) {
                            ml[i][k] = own.ml[at + 16 * (k0 + k) + i];
                            load_cols<C>(own.o + (at + 16 * (k0 + k) + i) * DV + col, x[i][k]);
                        }
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                    for (uint32_t k = 0; k < 6; ++k)
                        if (there[i] && k0 + k < splits) j[i].add(ml[i][k], x[i][k]);
            }
            if (p.total) join_prefix<C>(j, p, parts, h, {s * rows + r[0], s * rows + r[1]}, there, col, DV);
        }
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i)
            if (there[i]) write_row<BF16>(a, j[i], s, r[i] / group, h * group + r[i] % group, col);
    }
}

template <int DQ, int DV, bool BF16>
int launch_own(k3xb_ctx* ctx, const AttnArgs& a, const PrefixPlan& p, const Parts& parts, const OwnPlan& own) {
    cudaLaunchConfig_t cfg{};
    const uint32_t ctas = a.kv_heads * own.row_tiles;
    cfg.gridDim = dim3(own.warps == 1 ? (ctas + 3) / 4 : ctas, a.S, own.splits);
    cfg.blockDim = dim3(kOwnThreads);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    // beside the prefix kernel's tail (it waits there before it joins or ends)
    cfg.numAttrs = p.total ? 1 : 0;
    if (own.warps == 1) K3XB_CUDA(ctx, cudaLaunchKernelEx(&cfg, own_kernel<DQ, DV, BF16, 1>, a, p, parts, own));
    else K3XB_CUDA(ctx, cudaLaunchKernelEx(&cfg, own_kernel<DQ, DV, BF16, 4>, a, p, parts, own));
    ++ctx->stats.kernel_launches;
    if (own.splits > 1) {
        cfg.gridDim = dim3(ctas, a.S);
        cfg.numAttrs = 1;   // it waits for the parts at its start
        K3XB_CUDA(ctx, cudaLaunchKernelEx(&cfg, join_kernel<DV, BF16>, a, p, parts, own));
        ++ctx->stats.kernel_launches;
    }
    return K3XB_OK;
}

template <uint32_t NK, uint32_t NV, bool BF16>
int launch_both(k3xb_ctx* ctx, const AttnArgs& a, const PrefixPlan& p, const Parts& parts, const OwnPlan& own) {
    if (p.total) {
        static std::atomic<uint64_t> configured{0};   // per template instance
        const int cst = configure_once(ctx, configured, [&]() -> int {
            K3XB_CUDA(ctx, cudaFuncSetAttribute(prefix_kernel<BF16, NK, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                static_cast<int>(prefix_smem(NK))));
            return K3XB_OK;
        });
        if (cst) return cst;
        CUtensorMap map_k, map_v, map_e;
        const KvSource& x = a.prefix;
        int st;
        if ((st = make_row_map(ctx, &map_k, x.k, 2ull * a.main, a.kv_heads, a.prefix_len, 2 * x.k_head, 2 * x.k_row, kTile))) return st;
        if ((st = make_row_map(ctx, &map_v, x.v, 2ull * a.value, a.kv_heads, a.prefix_len, 2 * x.v_head, 2 * x.v_row, kTile / 2))) return st;
        map_e = map_k;
        if (a.extra && (st = make_row_map(ctx, &map_e, x.extra, 2ull * a.extra, 1, a.prefix_len, 2 * x.extra_row, 2 * x.extra_row, kTile)))
            return st;
        prefix_kernel<BF16, NK, NV><<<(p.total + p.range - 1) / p.range, kPrefixThreads, prefix_smem(NK), ctx->stream>>>(map_k, map_e, map_v, a, p, parts);
        K3XB_LAUNCHED(ctx);
    }
    return launch_own<64 * NK, 64 * NV, BF16>(ctx, a, p, parts, own);
}

template <bool BF16>
int launch_typed(k3xb_ctx* ctx, const AttnArgs& a, const PrefixPlan& p, const Parts& parts, const OwnPlan& own) {
    switch ((a.main + a.extra) / 64 * 10 + a.value / 64) {
        case 11: return launch_both<1, 1, BF16>(ctx, a, p, parts, own);
        case 12: return launch_both<1, 2, BF16>(ctx, a, p, parts, own);
        case 21: return launch_both<2, 1, BF16>(ctx, a, p, parts, own);
        case 22: return launch_both<2, 2, BF16>(ctx, a, p, parts, own);
        case 31: return launch_both<3, 1, BF16>(ctx, a, p, parts, own);
        default: return launch_both<3, 2, BF16>(ctx, a, p, parts, own);
    }
}

bool whole16(const void* ptr, std::initializer_list<uint64_t> strides) {
    bool ok = reinterpret_cast<uintptr_t>(ptr) % 16 == 0;
    for (uint64_t s : strides) ok = ok && s % 8 == 0 && s < (1ull << 38);
    return ok;
}

}  // namespace

bool attend_tc_takes(const AttnArgs& a, int32_t type) {
    if (type != K3XB_TYPE_BF16 && type != K3XB_TYPE_F16) return false;
    if ((a.main != 64 && a.main != 128) || (a.extra != 0 && a.extra != 64) || (a.value != 64 && a.value != 128)) return false;
    bool ok = whole16(a.q, {a.q_row}) && whole16(a.out, {});
    for (const KvSource* x : {&a.prefix, &a.suffix}) {
        if (x == &a.prefix && !a.prefix_len) continue;
        ok = ok && whole16(x->k, {x->k_row, x->k_head, x->k_seq}) && whole16(x->v, {x->v_row, x->v_head, x->v_seq}) &&
             (!a.extra || whole16(x->extra, {x->extra_row, x->extra_seq}));
    }
    // a tensor map steps over no zero stride (a broadcast prefix)
    if (a.prefix_len)
        ok = ok && a.prefix.k_row && a.prefix.k_head && a.prefix.v_row && a.prefix.v_head && (!a.extra || a.prefix.extra_row);
    // masked scores are -inf times the scale, and row indices of a kv head 32-bit
    return ok && a.scale != 0.0f && static_cast<uint64_t>(a.S) * a.N * (a.heads / a.kv_heads) < (1ull << 31);
}

int launch_attend_tc(k3xb_ctx* ctx, const AttnArgs& a, bool bf16) {
    const uint32_t sms = static_cast<uint32_t>(ctx->sm_count), group = a.heads / a.kv_heads;
    PrefixPlan p{};
    p.rows = a.S * a.N * group;
    p.group = group;
    p.blocks = static_cast<uint32_t>((static_cast<uint64_t>(a.prefix_len) + kTile - 1) / kTile);
    OwnPlan own{};
    own.row_tiles = (a.N * group + 15) / 16;
    // One sequence's few rows read a short prefix with their own rows, which saves
    // a launch and a wait (32 heads of 128 + 64 / 128, one row: prefixes of 200 and 400
    // 12.1 and 13.6 us, apart 14.4 and 14.5; 700 and 2000 18.0 and 28.6, apart 15.4 and 19.6;
    // 16 rows of each of 2 tiles a head: 128 17.5, apart 17.8; 256 21.7, apart 18.5;
    // 4 tiles of one kv head: 700 18.4, apart 19.9; 1500 23.0, apart 18.8).
    own.prefix = a.S == 1 && own.row_tiles <= 4 && a.prefix_len <= 1024 &&
                 static_cast<uint64_t>(a.kv_heads) * own.row_tiles * a.prefix_len <= 96ull * sms;
    const uint32_t tiles = (p.rows + kTile - 1) / kTile;
    p.pairs = tiles / 2;
    p.odd = tiles % 2;
    const uint64_t per_head = static_cast<uint64_t>(p.pairs) * p.blocks + p.odd * ((p.blocks + 1) / 2);
    if (per_head * a.kv_heads >= (1ull << 31)) return fail(ctx, K3XB_INVALID_EXTENT, "prefix_attention: rows times prefix too large");
    p.steps_per_head = static_cast<uint32_t>(per_head);
    p.total = own.prefix ? 0 : p.steps_per_head * a.kv_heads;
    uint32_t ctas = 0;
    if (p.total) {
        // A tensor core truncates each sum, 16 keys at a time, so a part of n keys may
        // be short by n / 16 2^-24: 2^-13 (f16) or 2^-10 (bf16) at most in 2^15 and 2^18
        // keys, an eighth and a quarter of what rounding the output costs.
        // Where that many lie in a CTA's range, the ranges go in several rounds.
        const uint32_t most = bf16 ? 2048 : 256;   // steps
        const uint64_t rounds = p.blocks > most ? (p.total + static_cast<uint64_t>(sms) * most - 1) / (static_cast<uint64_t>(sms) * most) : 1;
        p.range = static_cast<uint32_t>((p.total + sms * rounds - 1) / (sms * rounds));
        ctas = (p.total + p.range - 1) / p.range;
        p.max_seg = p.range / (p.odd ? (p.blocks + 1) / 2 : p.blocks) + 2;
        if (static_cast<uint64_t>(ctas) * p.max_seg * 2 * kTile >= (1ull << 31))
            return fail(ctx, K3XB_INVALID_EXTENT, "prefix_attention: too many rows");
    }
    // A task has one warp where there are tasks for every one that the GPU holds (64 x 32
    // tasks: 116 us with two warps each, 110 with one), else four (6 x 64 tasks:
    // 50 us with one, 38 with four).
    const uint64_t whole = static_cast<uint64_t>(a.S) * a.kv_heads * own.row_tiles;
    own.warps = whole >= 8ull * sms ? 1 : 4;
    // Room for three times as many warps as the GPU holds (twelve per SM), since
    // sequences are of unlike lengths; how many tasks a sequence becomes is up to its
    // length on the device, 512 keys to one at least (48 sequences of up to
    // 2100, 16 heads of 64: 64 us; 256 and 1024 66 and 73 us), or 64 where latency
    // counts. Lengths, not the capacity, so that a cache with room for 16384 costs
    // no more than a full one (21 x 5 rows after 5003 + up to 331: 37.4 us; by
    // capacity 69).
    own.least = own.prefix ? 4 : 32;
    const uint64_t rows_read = a.capacity + (own.prefix ? static_cast<uint64_t>(a.prefix_len) : 0);
    const uint64_t wanted = own.prefix ? 36 * sms : 36 * sms / own.warps;
    own.splits = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>((wanted + whole - 1) / whole, rows_read / (16 * own.least))));
    if (static_cast<uint64_t>(a.kv_heads) * own.row_tiles * own.splits >= (1ull << 31))
        return fail(ctx, K3XB_INVALID_EXTENT, "prefix_attention: too many rows per sequence");
    own.tasks = a.kv_heads * own.row_tiles * own.splits;
    Parts parts{};
    auto carve = [&](auto& c) {
        const size_t n = static_cast<size_t>(ctas) * p.max_seg * 2 * kTile;
        const size_t k = own.splits > 1 ? static_cast<size_t>(own.tasks) * a.S * 16 : 0;
        parts.o = c.template take<float>(n * a.value);
        parts.ml = c.template take<float2>(n);
        own.o = c.template take<float>(k * a.value);
        own.ml = c.template take<float2>(k);
    };
    Sizer sz;
    carve(sz);
    void* mem;
    if (const int st = ensure_scratch(ctx, sz.used, &mem)) return st;
    Carver cv(mem);
    carve(cv);
    return bf16 ? launch_typed<true>(ctx, a, p, parts, own) : launch_typed<false>(ctx, a, p, parts, own);
}

}  // namespace k3xb
