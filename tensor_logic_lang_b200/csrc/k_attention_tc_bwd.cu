// Attention backward on the tensor cores: 16-bit operands, head size up to
// 128, or fp32 arrays as pairs of fp16 (attn_tc.h, SplitArray).  With p = exp(s - lse), dp = dout v^T, D = dout . o by row,
//   dx = p (dp - D) (1 - tanh^2),  dq = scale dx k,  dk = scale dx^T q,  dv = p^T dout
// the scores are taken again from q and k (S is never stored), twice:
//
//   k_attn_prep    by tile of 128 queries: log2(e) lse and D, ready for the
//                  kernels below; the largest row norms of dout and v (fp16;
//                  fp32 arrays: all of it falls out of the splitting)
//   k_attn_tc_dkv  a block per (key tile, head): dk and dv stay in TMEM while
//                  the query tiles pass; the heads of a group form a cluster
//                  and add their sums through distributed shared memory in a
//                  fixed order
//   k_attn_tc_dq   a block per (query tile, head): dq stays in TMEM while the
//                  key tiles pass
//
// Seven products where one kernel for all three would need five, but no
// atomics on dq: the results do not depend on the order of the blocks, and
// there is no fp32 copy of dq in memory.  Four warpgroups take 32 columns of
// the 128 x 128 scores each; P (dx) goes back to TMEM as a 16-bit operand over
// the part of S (dp) its warpgroup has read.  While the exponentials of one
// tile run, the products of the tile before and the scores of the next do.
//
// 16-bit roundings: p and dx as operands of the last products (tensor cores
// take 16-bit operands), each off by half a step of its own size.  fp16 ends
// at 2^-24, so p is written 2^14 larger, and dx times the power of two that
// puts its bound, 2 max|dout_i| max|v_j| (norms; |dp| and |D| are at most half
// of it), at 2^15: neither can overflow, and small gradients keep their bits.
// fp32 arrays: p and dx are written as hi and lo, each product is three, and
// the sums over the tiles are added by the rows' threads (the tensor cores cut
// theirs, see k_attention_tc.cu).  Of head sizes above 64 (WIDE) the resident
// operands fill shared memory but for two tiles of 64 columns, so the passing
// ones come in halves, each as often as a product needs it (twice, from the L2
// cache), and dk and dv, which leave no room for sums in TMEM, are added to
// the outputs tile by tile (sums of 4 tiles on the tensor cores lost 2.4e-6 of dk
// and dv, of one 6e-7).
//
// Bound by the element work between the products: a pair of tiles takes about 4600 clocks
// in the dq kernel and 5700 in the other (2 x 16/4 heads x 2048 x 128, cap 30, starts and ends
// of walks of 1 to 16 tiles among them), of which the products fill 1536 and 2048; instructions
// issue in 52 % of the clocks.  16 heads of 16384 queries and keys, bf16, causal, five products
// counted: d 128 3400 to 3900 us (the power cap), 810 to 710 TFLOP/s, cap 50 4490; d 64 2870 us, 479 TFLOP/s,
// cap 50 3510.  fp32, 8 heads of 4096: d 64 214 us, d 96 455.
#include <algorithm>

#include "attn_tc.h"

namespace tl {
namespace {

constexpr int BW_COMPUTE = 512, BW_THREADS = BW_COMPUTE + 128, BW_STAGES = 2;
constexpr int BW_MMA = BW_COMPUTE / 32, BW_TMA = BW_MMA + 1;   // warps
constexpr int BW_COLS = 32;   // scores of a thread
// Registers a thread: at launch, of the computing warps, of the last warpgroup.
// fp32 (hi and lo of everything) gains most from the larger share (causal backward of 8 heads x
// 4096 x 64: 278 us without a split, 223 with 104 and 64, 213 with 112 and 32); with
// 16 bits, and in halves, the MMA and TMA warps need more than 32 (2 x 16 heads over 4 x 2048 x
// 128, step of both passes: 235 us, 231, 240).
constexpr int BW_REGS = 96;
template <bool FP32> struct BwRegs {
    static constexpr int MORE = FP32 ? 112 : 104, FEWER = FP32 ? 32 : 64;
    static_assert(BW_COMPUTE * MORE + 128 * FEWER <= BW_THREADS * BW_REGS, "the split waits for ever");
};
struct BwArgs {
    AttnCall a;
    const float* stats;          // [b, hq, query tiles][2][128]
    const uint32_t* norms;       // fp16, fp32: [b, hkv][2] largest |dout_i|^2, |v_j|^2 as bits
    const DocRange *q_ranges, *k_ranges;
    SplitTops tops;              // fp32 arrays
    int q_tiles, k_tiles;
    int cluster, abreast, parts;   // dkv: its blocks take `abreast` heads at once, `parts` of them share a head's query tiles
    // a block a query head instead of a key head's group: its dk and dv go to
    // sums of its own, which k_sum_heads adds (WIDE, heads that share keys)
    int by_head;
    HeadsView dk, dv;
    int* err;
};

template <int DP>
struct BwSmem {
    static constexpr bool WIDE = DP > 128;   // halves of 64 columns, hi and lo
    static constexpr int CH = WIDE ? 2 : DP / 64, TILE_B = CH * CHUNK_BYTES;
    // two resident tiles, stages of two tiles and the statistics; WIDE: four
    // resident halves, a ring of two
    static constexpr int FIX = 0, RING = (WIDE ? 4 : 2) * TILE_B, STAT = 6 * TILE_B, BAR = STAT + BW_STAGES * STAT_BYTES,
                         DOCS = BAR + 256, BYTES = DOCS + 64 + 1024;
    // the cluster's sums: dv and dk as fp32 rows padded by 16 bytes, over the tiles
    static constexpr int SUM_LD = DP + 4;
    static_assert(WIDE || 2 * TILE * SUM_LD * 4 <= STAT, "the sums lie over the tiles");
};

// ---------------------------------------------------------------- preparation
// |row|^2 of 8 columns, and the dot product with another row
template <typename T>
__device__ __forceinline__ void dot8(const uint4& x, const uint4& y, float& xy, float& xx) {
    const T* a = reinterpret_cast<const T*>(&x);
    const T* b = reinterpret_cast<const T*>(&y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float u = to_f32(a[i]);
        xy = fmaf(u, to_f32(b[i]), xy);
        xx = fmaf(u, u, xx);
    }
}

// Blocks of half a tile, 16 lanes a row, 4 rows of a half warp in flight:
// first the query tiles, then (fp16) the key tiles' norms of v.
template <typename T>
__global__ void __launch_bounds__(256)
    k_attn_prep(const __grid_constant__ AttnCall a, float* __restrict__ stats, uint32_t* __restrict__ norms, int q_tiles, int k_tiles) {
    let_next_start();
    constexpr int R = 4;
    const int half = threadIdx.x / 16, sub = threadIdx.x % 16, c0 = sub * 8;
    int64_t blk = blockIdx.x / 2;
    const int r0 = blockIdx.x % 2 * (TILE / 2) + half * R;
    const int64_t n_q = (int64_t)a.b * a.hq * q_tiles;
    float top = 0.f;
    const bool keys = blk >= n_q;
    int group_of;
    uint4 x[R], y[R];
    if (!keys) {
        const int i0 = (int)(blk % q_tiles) * TILE + r0;
        const int h = (int)(blk / q_tiles % a.hq), b = (int)(blk / q_tiles / a.hq);
        group_of = b * a.hkv + h / (a.hq / a.hkv);
        const T* dout = static_cast<const T*>(a.dout.p) + b * a.dout.sb + h * a.dout.sh + c0;
        const T* o = static_cast<const T*>(a.o.p) + b * a.o.sb + h * a.o.sh + c0;
        float lse = -INFINITY;   // of row sub, of the first R lanes
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t i = i0 + k;
            const bool on = i < a.nq && (!a.q_doc || a.q_doc[(int64_t)b * a.nq + i] >= 0);
            x[k] = y[k] = make_uint4(0, 0, 0, 0);
            if (on && c0 < a.d) {
                x[k] = *reinterpret_cast<const uint4*>(dout + i * a.dout.ss);
                y[k] = *reinterpret_cast<const uint4*>(o + i * a.o.ss);
            }
            if (on && sub == k) lse = a.lse[((int64_t)b * a.hq + h) * a.nq + i];
        }
        float mine = 0.f;
#pragma unroll
        for (int k = 0; k < R; ++k) {
            float xy = 0.f, xx = 0.f;
            dot8<T>(x[k], y[k], xy, xx);
#pragma unroll
            for (int w = 8; w; w >>= 1) {
                xy += __shfl_xor_sync(0xffffffffu, xy, w);
                xx += __shfl_xor_sync(0xffffffffu, xx, w);
            }
            top = fmaxf(top, finite(xx));
            if (sub == k) mine = xy;
        }
        if (sub < R) {
            float* st = stats + blk * 2 * TILE + r0 + sub;
            // a row that sees nothing has p = 2^-inf = 0 everywhere
            st[0] = lse == -INFINITY ? -INFINITY : PLift<T>::log2 - lse * kLog2e;
            st[TILE] = -mine;
        }
    } else {
        blk -= n_q;
        const int64_t j0 = (blk % k_tiles) * TILE + r0;
        const int h = (int)(blk / k_tiles % a.hkv), b = (int)(blk / k_tiles / a.hkv);
        group_of = b * a.hkv + h;
        const int kv = a.kv_len ? min(max(a.kv_len[b], 0), a.nk) : a.nk;
        const T* v = static_cast<const T*>(a.v.p) + b * a.v.sb + h * a.v.sh + c0;
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t j = j0 + k;
            x[k] = make_uint4(0, 0, 0, 0);
            if (j < kv && (!a.k_doc || a.k_doc[(int64_t)b * a.nk + j] >= 0) && c0 < a.d)
                x[k] = *reinterpret_cast<const uint4*>(v + j * a.v.ss);
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            float xy = 0.f, xx = 0.f;
            dot8<T>(x[k], x[k], xy, xx);
#pragma unroll
            for (int w = 8; w; w >>= 1) xx += __shfl_xor_sync(0xffffffffu, xx, w);
            top = fmaxf(top, finite(xx));
        }
    }
    wait_for_previous();   // the norms start at 0; the documents' ranges, which the kernel behind this one reads
    if (norms) {
        // non-negative floats order like their bits; a maximum does not depend on the order
        __shared__ uint32_t most[8];
        const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        if ((threadIdx.x & 31) == 0) most[threadIdx.x / 32] = m;
        __syncthreads();
        if (threadIdx.x < 32) {
            const uint32_t all = __reduce_max_sync(0xffffffffu, most[threadIdx.x & 7]);
            if (threadIdx.x == 0) atomicMax(&norms[2 * group_of + (keys ? 1 : 0)], all);
        }
    }
}

// The power of two that dx is written with (see the top of the file).  Split
// operands: beside those that dout and v carry.
template <typename T>
__device__ __forceinline__ float dx_lift(const BwArgs& g, int b, int kvh) {
    if (PLift<T>::log2 == 0.f) return 1.f;
    const uint32_t* n = g.norms + 2 * ((int64_t)b * g.a.hkv + kvh);
    const float bound = 2.f * sqrtf(__uint_as_float(n[0])) * sqrtf(__uint_as_float(n[1]));
    if (!(bound > 0.f)) return 1.f;
    return exp2f(fminf(fmaxf(floorf(15.f - log2f(bound)), -100.f), 100.f));
}

// a, of split operands times 2^e in two factors, each within fp32
template <bool SPLIT>
struct Factors {
    float mul, post;
    __device__ __forceinline__ Factors(float a, int e) : mul(SPLIT ? a * pow2(e / 2) : a), post(SPLIT ? pow2(e - e / 2) : 1.f) {}
    __device__ __forceinline__ float of(uint32_t bits) const { return __uint_as_float(bits) * mul * post; }
};

// ---------------------------------------------------------------- elements
// 32 scores q.k of a row -> p in base 2 (16-bit pairs) and p (1 - tanh^2).
// off: position of column 0 relative to the row's (|off + c| is the distance);
// nl(i): minus log2(e) lse of the columns 2i, 2i + 1.
// SPLIT: p16 and low take hi and lo, and the tanh is good to fp32.
template <typename T, bool CAP, bool BIAS, bool SPLIT, typename NL>
__device__ __forceinline__ void grad_row(f2 (&x)[16], uint32_t (&p16)[16], uint32_t (&low)[16], float c1, const CapCoef<SPLIT>& cap, float slope2, int off,
                                         bool masked, uint32_t bits, NL nl) {
    f2 bend[CAP ? 16 : 1];
    if (CAP) {
        cap_scores<BIAS>(x, cap);
        // 1 - tanh^2, the tanh from the score
        const float inv = -1.f / (cap.top * cap.top);
#pragma unroll
        for (int i = 0; i < 16; ++i) bend[i] = fma2(mul2(x[i], pack2(inv, inv)), x[i], pack2(1.f, 1.f));
    }
    const f2 c = CAP ? pack2(1.f, 1.f) : pack2(c1, c1);
    if (BIAS) {
        const bool after = __all_sync(0xffffffffu, off >= 0), before = __all_sync(0xffffffffu, off + 31 <= 0);
        if (after || before) {
            const float k = after ? -slope2 : slope2, kb = k * (float)off;
            const f2 kk = pack2(k, k), base = pack2(kb, kb);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fma2(x[i], c, fma2(kk, pack2((float)(2 * i), (float)(2 * i + 1)), base));
        } else {
            const float at = (float)off;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                x[i] = fma2(x[i], c, pack2(-slope2 * fabsf(at + (float)(2 * i)), -slope2 * fabsf(at + (float)(2 * i + 1))));
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float lo, hi;
        unpack2(CAP || BIAS ? add2(x[i], nl(i)) : fma2(x[i], c, nl(i)), lo, hi);
        if (masked) {
            lo = (bits >> (2 * i)) & 1 ? lo : -INFINITY;
            hi = (bits >> (2 * i + 1)) & 1 ? hi : -INFINITY;
        }
        lo = ex2(lo);
        hi = ex2(hi);
        if (SPLIT) split16(lo, hi, p16[i], low[i]);
        else p16[i] = pack16<T>(lo, hi);
        x[i] = pack2(lo, hi);
        if (CAP) x[i] = mul2(x[i], bend[i]);
    }
}

// dx = pb (dp - D), zero where the key is not seen (there dp may be anything)
template <typename T, bool SPLIT, typename ND>
__device__ __forceinline__ void grad_dx(const f2 (&pb)[16], const uint32_t (&dp)[32], uint32_t (&out)[16], uint32_t (&low)[16],
                                        float lift, bool masked,
                                        uint32_t bits, ND nd) {
    const f2 up = pack2(lift, lift);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const f2 d2 = pack2(__uint_as_float(dp[2 * i]), __uint_as_float(dp[2 * i + 1]));
        float lo, hi;
        unpack2(mul2(pb[i], PLift<T>::log2 == 0.f ? add2(d2, nd(i)) : fma2(d2, up, nd(i))), lo, hi);
        if (masked) {
            lo = (bits >> (2 * i)) & 1 ? lo : 0.f;
            hi = (bits >> (2 * i + 1)) & 1 ? hi : 0.f;
        }
        if (SPLIT) split16(lo, hi, out[i], low[i]);
        else out[i] = pack16<T>(lo, hi);
    }
}

// What the two gradient kernels share: barriers, TMEM, the documents of the block's rows.
struct BwBlock {
    uint64_t *fix, *full, *empty, *s_full, *p_full, *dp_full, *dx_full, *done, *stat_full;
    uint32_t* tmem_slot;
    int* docs;
    __device__ __forceinline__ BwBlock(uint8_t* bars, uint8_t* docs_at) {
        uint64_t* bar = reinterpret_cast<uint64_t*>(bars);
        fix = bar;
        full = bar + 1;
        empty = full + BW_STAGES;
        s_full = empty + BW_STAGES;   // two in the dq kernel
        p_full = s_full + 2;
        dp_full = p_full + 1;
        dx_full = dp_full + 1;
        done = dx_full + 1;
        stat_full = done + 1;         // two; WIDE
        tmem_slot = reinterpret_cast<uint32_t*>(bar + 24);
        docs = reinterpret_cast<int*>(docs_at);
    }
    // returns the TMEM base; `doc`: documents of the block's rows, or null
    __device__ __forceinline__ uint32_t setup(const int32_t* doc, int rows, DocRange* mine, bool wait) {
        const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
        if (threadIdx.x == 0) {
            mbar_init(fix, 1);
            for (int s = 0; s < BW_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
            mbar_init(&s_full[0], 1); mbar_init(&s_full[1], 1);
            mbar_init(&stat_full[0], 1); mbar_init(&stat_full[1], 1);
            mbar_init(p_full, BW_COMPUTE); mbar_init(dp_full, 1); mbar_init(dx_full, BW_COMPUTE); mbar_init(done, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            docs[0] = 0x7fffffff; docs[1] = -1; docs[2] = 0;
        }
        if (warp == BW_MMA) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (wait) wait_for_previous();   // the statistics, the documents' ranges, the split operands
        *mine = no_docs();
        if (doc) {
            const int r = threadIdx.x;
            const int d = r < rows ? doc[r] : -1;
            const int lo = __reduce_min_sync(0xffffffffu, d >= 0 ? d : 0x7fffffff), hi = __reduce_max_sync(0xffffffffu, d);
            const int pad = __any_sync(0xffffffffu, d < 0);
            if (lane == 0) {
                atomicMin(&docs[0], lo);
                atomicMax(&docs[1], hi);
                if (pad && warp * 32 < rows) docs[2] = 1;
            }
            __syncthreads();
            *mine = {docs[0], docs[1], docs[2], 0};
        }
        return *tmem_slot;
    }
    __device__ __forceinline__ void finish(uint32_t tmem) {
        tc_fence_before();
        __syncthreads();
        if (threadIdx.x / 32 == BW_MMA) {
            tc_fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
        }
    }
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, bool ok, int* err) {
    ok = ok && mbar_wait(bar, parity, err);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    return ok;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
                 "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// WIDE: the ring of two halves (64 columns, hi and lo) that pass, entry by entry
// in the same order for the warp that loads and the one that multiplies.
struct HalfRing {
    static constexpr int HALF = 2 * CHUNK_BYTES;
    const BwBlock& bb;
    uint8_t* at;
    int* err;
    int e = 0;
    __device__ __forceinline__ HalfRing(const BwBlock& b, uint8_t* ring, int* er) : bb(b), at(ring), err(er) {}
    // both halves of a tile of rows
    __device__ __forceinline__ void load2(const HeadMap& m, int tile, int h, int b, bool& ok) {
        for (int f = 0; f < 2; ++f) {
            const int s = e % 2;
            if (e >= 2) ok = warp_wait(&bb.empty[s], ((e / 2) & 1) ^ 1, ok, err);
            if (!ok) return;
            if (elect_one()) {
                mbar_expect_tx(&bb.full[s], HALF);
                tma_tile(smem_u32(at + s * HALF), m, &bb.full[s], 2, tile * TILE, h, b, 2 * f);
            }
            __syncwarp();
            ++e;
        }
    }
    // copies in flight land before the block ends
    __device__ __forceinline__ void drain(bool ok) {
        if (!ok)
            for (int i = max(0, e - 2); i < e; ++i) mbar_wait(&bb.full[i % 2], (i / 2) & 1, err);
    }
    // D = X Y^T over both halves: X resident, Y passes
    template <typename T>
    __device__ __forceinline__ void rows2(uint32_t d, uint32_t x, int ksteps, uint64_t* done, bool& ok) {
        for (int f = 0; f < 2; ++f, ++e) {
            const int s = e % 2;
            ok = warp_wait(&bb.full[s], (e / 2) & 1, ok, err);
            if (ok && elect_one()) {
                if (f == 0) mma_rows_split<T>(d, x, smem_u32(at + s * HALF), 4);
                else mma_rows_split<T, true>(d, x + HALF, smem_u32(at + s * HALF), ksteps - 4);
                umma_commit(&bb.empty[s]);
                if (f == 1) umma_commit(done);
            }
            __syncwarp();
        }
    }
    // columns 0..63 and 64.. of D = A Y: Y passes
    template <typename T>
    __device__ __forceinline__ void parts2(uint32_t d, uint32_t a, int ksteps, bool& ok) {
        for (int f = 0; f < 2; ++f, ++e) {
            const int s = e % 2;
            ok = warp_wait(&bb.full[s], (e / 2) & 1, ok, err);
            if (ok && elect_one()) {
                mma_parts_split<BW_COLS>(d + 64 * f, a, smem_u32(at + s * HALF), f16_idesc<T>(f ? 16 * (ksteps - 4) : 64, true), 0);
                umma_commit(&bb.empty[s]);
            }
            __syncwarp();
        }
    }
};

// A row's columns col0 .. col0 + N - 1 of an fp32 output (+)= N TMEM columns times
// f.  The thread alone owns them, so additions that the L2 makes, which nothing
// waits for, come in one order (loads and stores took 6 us more a tile of 96 columns).
template <int N, bool SPLIT>
__device__ __forceinline__ void add_row(const HeadsView& v, int b, int h, int64_t row, int col0, bool on, int d, uint32_t taddr,
                                        const Factors<SPLIT>& f, bool fresh) {
    float* p = static_cast<float*>(v.p) + b * v.sb + h * v.sh + row * v.ss + col0 * v.sd;
    const bool wide = v.sd == 1 && d % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
#pragma unroll 1
    for (int k = 0; k < N; k += 16) {
        const int left = on ? d - col0 - k : 0;   // columns from here on
        uint32_t o[16];
        tmem_ld16(taddr + k, o);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 16; q += 4) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = f.of(o[q + e]);
            float* at = p + (k + q) * v.sd;
            if (wide && fresh) {
                if (q < left) *reinterpret_cast<float4*>(at) = make_float4(x[0], x[1], x[2], x[3]);
            } else if (wide) {
                if (q < left)
                    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3])
                                 : "memory");
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (q + e < left) {
                        if (fresh) at[e * v.sd] = x[e];
                        else asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(at + e * v.sd), "f"(x[e]) : "memory");
                    }
            }
        }
    }
}

// The powers of two that split operands carry.
struct SplitExps {
    int q, k, v, dout;
};
template <bool SPLIT>
__device__ __forceinline__ SplitExps split_exps(const BwArgs& g, int b, int kvh) {
    const int i = b * g.a.hkv + kvh;
    if (!SPLIT) return {0, 0, 0, 0};
    return {split_exp(g.tops.q, i), split_exp(g.tops.k, i), split_exp(g.tops.v, i), split_exp(g.tops.dout, i)};
}

// ---------------------------------------------------------------- dk, dv
// TMEM: S^T (P^T) 0..127, dp^T (dx^T) 128..255, dv, dk (DO columns each; split
// operands: their sums over the tiles behind them).
// T: operands, U: the arrays' type (float: split operands).
template <typename T, typename U, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(BW_THREADS, 1)
    k_attn_tc_dkv(const __grid_constant__ HeadMap mq, const __grid_constant__ HeadMap mk, const __grid_constant__ HeadMap mv,
                  const __grid_constant__ HeadMap mdo, const __grid_constant__ BwArgs g) {
    using L = BwSmem<DP>;
    constexpr bool SPLIT = !std::is_same<T, U>::value;
    constexpr bool WIDE = L::WIDE;
    constexpr int DO = SPLIT ? DP / 2 : DP;   // columns of a result
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const AttnCall& a = g.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    // block -> (key tile, sequence and key head, head of the group); a causal
    // call's first keys are seen by the most queries and go first
    const int heads = g.by_head ? a.hq : a.hkv, group = a.hq / a.hkv, rank = blockIdx.x % g.cluster;
    const unsigned unit = blockIdx.x / g.cluster, bhs = (unsigned)a.b * heads;
    const int kt = (int)(unit / bhs), out_h = (int)(unit % bhs % heads), b = (int)(unit % bhs / heads);
    const int kvh = g.by_head ? out_h / group : out_h;
    const int j0 = kt * TILE;
    const SeqMask mask(a, b);
    const int32_t* qd = a.q_doc ? a.q_doc + (int64_t)b * a.nq : nullptr;
    const int32_t* kd = a.k_doc ? a.k_doc + (int64_t)b * a.nk : nullptr;
    BwBlock bb(smem + L::BAR, smem + L::DOCS);
    DocRange mine;
    const uint32_t tmem = bb.setup(kd ? kd + j0 : nullptr, min(TILE, a.nk - j0), &mine, true);
    // the dq kernel may start on the SMs that this one leaves: what it reads is there
    let_next_start();
    const uint32_t t_s = tmem, t_dp = tmem + TILE, t_dv = tmem + 2 * TILE, t_dk = tmem + 2 * TILE + DO;
    const uint32_t t_dva = tmem + 3 * TILE, t_dka = t_dva + 64;   // split operands: the sums over the tiles

    // query tiles that see some of the keys; from `clear` on they see all of them
    int begin = 0, end = g.q_tiles, clear = 0;
    if (mask.causal && j0 >= mask.prefix) begin = max(0, j0 - mask.p0) / TILE;
    if (mask.causal && j0 + TILE > mask.prefix) clear = max(0, j0 + TILE - 1 - mask.p0 + TILE - 1) / TILE;
    if (j0 >= mask.kv) end = 0;
    if (mask.kv < a.nk && j0 + TILE > mask.kv) clear = end;
    const DocRange* ranges = qd ? g.q_ranges + (int64_t)b * g.q_tiles : nullptr;
    TileWalk<true> walk;
    bool masked, ok = true;
    // (head, query tile) pairs in order; qt < 0 after the last
    int h = (g.by_head ? out_h : kvh * group + rank / g.parts) - g.abreast;
    const int h_end = g.by_head ? out_h + 1 : (kvh + 1) * group;
    int qt = -1;
    auto first = [&]() { walk.start(0, 0, 0, 0, ranges, mine); };
    auto next = [&]() {
        qt = walk.next(&masked);
        while (qt < 0) {
            h += g.abreast;
            if (h >= h_end) return;
            walk.start(begin, end, clear, end, ranges, mine, g.parts, rank & (g.parts - 1));
            qt = walk.next(&masked);
        }
    };
    first();
    next();
    const bool any = qt >= 0;

    if (warp >= BW_MMA) {
        fewer_registers<BwRegs<SPLIT && !WIDE>::FEWER>();
        if (warp == BW_TMA) {
            // ------------------------------------------------ TMA
            if (any && lane == 0) {
                mbar_expect_tx(bb.fix, L::RING);
                for (int f = 0; f < (WIDE ? 2 : 1); ++f) {
                    tma_tile(smem_u32(smem + L::FIX + f * L::TILE_B), mk, bb.fix, L::CH, j0, kvh, b, 2 * f);
                    tma_tile(smem_u32(smem + L::FIX + L::RING / 2 + f * L::TILE_B), mv, bb.fix, L::CH, j0, kvh, b, 2 * f);
                }
            }
            int n = 0;
            if (WIDE) {
                // Q and dout halves in the order in which the products take them: of
                // tile n, n's S and dp, then dv of n, S of n + 1, dk of n, dp of n + 1
                HalfRing ring(bb, smem + L::RING, g.err);
                int n_qt = qt, n_h = h;
                auto stats_of = [&]() {
                    if (!elect_one()) return;
                    mbar_expect_tx(&bb.stat_full[n & 1], STAT_BYTES);
                    bulk_load(smem + L::STAT + (n & 1) * STAT_BYTES, g.stats + (((int64_t)b * a.hq + n_h) * g.q_tiles + n_qt) * 2 * TILE,
                              STAT_BYTES, &bb.stat_full[n & 1]);
                };
                if (n_qt >= 0) {
                    stats_of();
                    ring.load2(mq, n_qt, n_h, b, ok);
                    ring.load2(mdo, n_qt, n_h, b, ok);
                }
                while (n_qt >= 0 && ok) {
                    const int p_qt = n_qt, p_h = n_h;
                    ring.load2(mdo, p_qt, p_h, b, ok);
                    next();
                    n_qt = qt;
                    n_h = h;
                    ++n;
                    if (n_qt >= 0) {
                        ring.load2(mq, n_qt, n_h, b, ok);
                        if (ok) stats_of();   // over those of n - 2: the ring is past dk of n - 2
                        __syncwarp();
                    }
                    ring.load2(mq, p_qt, p_h, b, ok);
                    if (n_qt >= 0) ring.load2(mdo, n_qt, n_h, b, ok);
                }
                ring.drain(ok);
            }
            for (; !WIDE && qt >= 0 && ok; next(), ++n) {
                const int s = n % BW_STAGES;
                if (n >= BW_STAGES) ok = warp_wait(&bb.empty[s], ((n / BW_STAGES) & 1) ^ 1, ok, g.err);
                if (ok && lane == 0) {
                    mbar_expect_tx(&bb.full[s], 2 * L::TILE_B + STAT_BYTES);
                    const uint32_t at = smem_u32(smem + L::RING + s * 2 * L::TILE_B);
                    tma_tile(at, mq, &bb.full[s], L::CH, qt * TILE, h, b);
                    tma_tile(at + L::TILE_B, mdo, &bb.full[s], L::CH, qt * TILE, h, b);
                    const float* st = g.stats + (((int64_t)b * a.hq + h) * g.q_tiles + qt) * 2 * TILE;
                    bulk_load(smem + L::STAT + s * STAT_BYTES, st, STAT_BYTES, &bb.full[s]);
                }
            }
            if (!WIDE && !ok)   // copies in flight land before the block ends
                for (int e = max(0, n - 1 - BW_STAGES); e < n - 1; ++e)
                    mbar_wait(&bb.full[e % BW_STAGES], (e / BW_STAGES) & 1, g.err);
        } else if (warp == BW_MMA) {
            // ------------------------------------------------ tensor cores
            const int ksteps = (a.d + 15) / 16;
            const uint32_t idesc = f16_idesc<T>(16 * ksteps, true);
            const uint32_t sk = smem_u32(smem + L::FIX), sv = sk + L::RING / 2;
            auto rows = [&](uint32_t d, uint32_t x, uint32_t y) {
                if (SPLIT) mma_rows_split<T>(d, x, y, ksteps);
                else mma_rows<T, DP / 16>(d, x, y, ksteps);
            };
            auto parts = [&](uint32_t d, uint32_t x, uint32_t y, bool more) {
                if (SPLIT) mma_parts_split<BW_COLS>(d, x, y, idesc, 0);
                else mma_parts<BW_COLS>(d, x, y, idesc, more);
            };
            // query rows of negative documents: 0 times what they hold could be NaN
            auto clean = [&](int s) {
                if (SPLIT || !qd || !masked) return;
                auto bad = [&](int r) { const int i = qt * TILE + r; return i < a.nq && qd[i] < 0; };
                clear_rows(smem + L::RING + s * 2 * L::TILE_B, L::CH, bad);
                clear_rows(smem + L::RING + s * 2 * L::TILE_B + L::TILE_B, L::CH, bad);
                fence_proxy_async_smem();
                __syncwarp();
            };
            int n = 0;
            if (WIDE && any) {
                HalfRing ring(bb, smem + L::RING, g.err);
                ok = warp_wait(bb.fix, 0, ok, g.err);
                ring.rows2<T>(t_s, sk, ksteps, &bb.s_full[0], ok);
                ring.rows2<T>(t_dp, sv, ksteps, bb.dp_full, ok);
                while (qt >= 0 && ok) {
                    ok = warp_wait(bb.p_full, n & 1, ok, g.err);
                    ring.parts2<T>(t_dv, t_s, ksteps, ok);
                    next();
                    if (qt >= 0) ring.rows2<T>(t_s, sk, ksteps, &bb.s_full[0], ok);
                    ok = warp_wait(bb.dx_full, n & 1, ok, g.err);
                    ring.parts2<T>(t_dk, t_dp, ksteps, ok);
                    if (qt >= 0) ring.rows2<T>(t_dp, sv, ksteps, bb.dp_full, ok);
                    else if (ok && elect_one()) umma_commit(bb.done);
                    __syncwarp();
                    ++n;
                }
            }
            if (!WIDE && any) {
                ok = warp_wait(bb.fix, 0, ok, g.err);
                // keys of padding: their scores would have a say in the tanh's form of their warps
                if (CAP && !SPLIT && ((kd && mine.pad) || (mask.kv < a.nk && j0 + TILE > mask.kv))) {
                    clear_rows(smem + L::FIX, L::CH, [&](int r) { return j0 + r < a.nk && (j0 + r >= mask.kv || (kd && kd[j0 + r] < 0)); });
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                ok = warp_wait(&bb.full[0], 0, ok, g.err);
                if (ok) clean(0);
                const uint32_t sq = smem_u32(smem + L::RING);
                if (ok && elect_one()) {
                    rows(t_s, sk, sq);
                    umma_commit(&bb.s_full[0]);
                    rows(t_dp, sv, sq + L::TILE_B);
                    umma_commit(bb.dp_full);
                }
                __syncwarp();
            }
            while (!WIDE && qt >= 0 && ok) {
                const int s = n % BW_STAGES, s1 = (n + 1) % BW_STAGES;
                const uint32_t sq = smem_u32(smem + L::RING + s * 2 * L::TILE_B);
                const uint32_t sq1 = smem_u32(smem + L::RING + s1 * 2 * L::TILE_B);
                ok = warp_wait(bb.p_full, n & 1, ok, g.err);
                if (ok && elect_one()) parts(t_dv, t_s, sq + L::TILE_B, n > 0);
                __syncwarp();
                next();
                if (qt >= 0) {
                    ok = warp_wait(&bb.full[s1], ((n + 1) / BW_STAGES) & 1, ok, g.err);
                    if (ok) clean(s1);
                    if (ok && elect_one()) {
                        rows(t_s, sk, sq1);
                        umma_commit(&bb.s_full[0]);
                    }
                    __syncwarp();
                }
                ok = warp_wait(bb.dx_full, n & 1, ok, g.err);
                if (ok && elect_one()) {
                    parts(t_dk, t_dp, sq, n > 0);
                    umma_commit(&bb.empty[s]);
                    if (qt >= 0) {
                        rows(t_dp, sv, sq1 + L::TILE_B);
                        umma_commit(bb.dp_full);
                    } else {
                        umma_commit(bb.done);
                    }
                }
                __syncwarp();
                ++n;
            }
        }
        __syncwarp();
        if (g.cluster > 1) {   // as the computing warps below, which keep their registers to the end
            cluster_sync();
            cluster_sync();
        }
    } else {
        // ---------------------------------------------------- 32 queries of a key per thread
        more_registers<BwRegs<SPLIT && !WIDE>::MORE>();
        const int wg = warp / 4, r = threadIdx.x % TILE, j = j0 + r;
        // at the end: dv (dk) and half of its columns
        constexpr int DH = DO / 2;
        const int which = wg / 2, col0 = wg % 2 * DH;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const SplitExps ex = split_exps<SPLIT>(g, b, kvh);
        const float scale = SPLIT ? split_scale(a.scale, ex.q + ex.k) : a.scale, c1 = scale * kLog2e;
        const CapCoef<SPLIT> cap(scale, CAP ? a.cap : 1.f);
        const float lift = dx_lift<T>(g, b, kvh), up = lift * PLift<T>::back;   // (split operands: dp and D carry the powers of dout and v)
        const int doc = kd && j < a.nk ? kd[j] : -1;
        // dk = scale dx^T q, dv = p^T dout
        const Factors<SPLIT> f(which ? (SPLIT ? a.scale : a.scale / lift) : PLift<T>::back,
                               SPLIT ? -(which ? ilogbf(lift) + ex.dout + ex.v + ex.q : ex.dout) : 0);
        int n = 0;
        for (; qt >= 0 && ok; next(), ++n) {
            const int i0 = qt * TILE + wg * BW_COLS;
            uint32_t bits = 0xffffffffu;
            if (masked) {
                // queries from `from` on see the key
                int from = mask.causal && j >= mask.prefix ? j - mask.p0 - i0 : 0;
                if (j >= mask.kv) from = BW_COLS;
                bits = ~low_bits(from, 0);
                if (qd) {
                    const int other[1] = {i0 + lane < a.nq ? __ldg(qd + i0 + lane) : -1};
                    uint32_t same[1];
                    doc_bits(other, doc, same);
                    bits &= same[0];
                }
            }
            const float slope2 = BIAS && a.slopes ? __ldg(a.slopes + h) * kLog2e : 0.f;
            const float* st = reinterpret_cast<const float*>(smem + L::STAT + (n % BW_STAGES) * STAT_BYTES) + wg * BW_COLS;
            uint64_t* landed = WIDE ? &bb.stat_full[n & 1] : &bb.full[n % BW_STAGES];   // the statistics
            ok = warp_wait(landed, (n / 2) & 1, ok, g.err);
            ok = warp_wait(&bb.s_full[0], n & 1, ok, g.err);
            if (!ok) break;
            f2 x[16];
            {
                // dv of the tile before, done before this S
                if (WIDE) {
                    if (which == 0 && n > 0)
                        add_row<DH>(g.dv, b, out_h, j, col0, j < a.nk, a.d, t_dv + lanes + col0, f, n == 1);
                } else if (SPLIT && which == 0 && n > 0) {
                    tmem_add<DH>(t_dva + lanes + col0, t_dv + lanes + col0, n == 1);
                }
                tmem_load(t_s + lanes + wg * BW_COLS, x);
                uint32_t p16[16], low[16];
                grad_row<T, CAP, BIAS, SPLIT>(x, p16, low, c1, cap, slope2, mask.p0 + i0 - j, masked, bits,
                                       [&](int i) { return *reinterpret_cast<const f2*>(st + 2 * i); });
                tmem_st16(t_s + lanes + wg * BW_COLS, p16);
                if (SPLIT) tmem_st16(t_s + lanes + wg * BW_COLS + 16, low);
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bb.p_full);
            ok = warp_wait(bb.dp_full, n & 1, ok, g.err);
            if (!ok) break;
            {
                // dk of the tile before, done before this dp
                if (WIDE) {
                    if (which == 1 && n > 0)
                        add_row<DH>(g.dk, b, out_h, j, col0, j < a.nk, a.d, t_dk + lanes + col0, f, n == 1);
                } else if (SPLIT && which == 1 && n > 0) {
                    tmem_add<DH>(t_dka + lanes + col0, t_dk + lanes + col0, n == 1);
                }
                uint32_t dp[32], dx[16], low[16];
                tmem_load(t_dp + lanes + wg * BW_COLS, dp);
                const f2 up2 = pack2(up, up);
                grad_dx<T, SPLIT>(x, dp, dx, low, up, masked, bits, [&](int i) {
                    const f2 d = *reinterpret_cast<const f2*>(st + TILE + 2 * i);
                    return PLift<T>::log2 == 0.f ? d : mul2(d, up2);
                });
                tmem_st16(t_dp + lanes + wg * BW_COLS, dx);
                if (SPLIT) tmem_st16(t_dp + lanes + wg * BW_COLS + 16, low);
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bb.dx_full);
        }
        if (any) ok = warp_wait(bb.done, 0, ok, g.err);
        uint32_t mine_at = (which ? t_dk : t_dv) + lanes + col0;
        if (SPLIT && !WIDE) {
            const uint32_t acc = (which ? t_dka : t_dva) + lanes + col0;
            if (any && ok) {
                tmem_add<DH>(acc, mine_at, n == 1);
                tmem_wait_st();
            }
            mine_at = acc;
        }
        if (WIDE && any) {
            if (ok) add_row<DH>(which ? g.dk : g.dv, b, out_h, j, col0, j < a.nk, a.d, mine_at, f, n <= 1);
        } else if (g.cluster == 1) {
            HeadsView v = which ? g.dk : g.dv;
            v.p = static_cast<U*>(v.p) + col0 * v.sd;
            if (ok) store_row<U, DH>(v, b, out_h, j, j < a.nk, a.d - col0, mine_at, any, any, f.mul, f.post);
        } else if (ok) {
            float* row = reinterpret_cast<float*>(smem) + (which * TILE + r) * L::SUM_LD + col0;
            for (int k = 0; k < DH / 16; ++k) {
                uint32_t o[16] = {};
                if (any) {
                    tmem_ld16(mine_at + 16 * k, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4*>(row + 16 * k + 4 * q) =
                        make_float4(f.of(o[4 * q]), f.of(o[4 * q + 1]), f.of(o[4 * q + 2]), f.of(o[4 * q + 3]));
            }
        }
        __syncwarp();
        if (g.cluster > 1) {
            // each block adds its share of the rows over the cluster, in the order of the heads
            cluster_sync();
            const int share = TILE / g.cluster, r0 = rank * share;
            const uint32_t sums = smem_u32(smem);
            constexpr int V = DO / 4;
            for (int e = threadIdx.x; e < 2 * share * V; e += BW_COMPUTE) {
                const int c = e % V, r = r0 + e / V % share, wg = e / V / share;
                if (j0 + r >= a.nk || 4 * c >= a.d) continue;
                float s[4] = {0.f, 0.f, 0.f, 0.f};
                for (int q = 0; q < g.cluster; ++q) {
                    float x[4];
                    load_cluster4(in_block(sums + ((wg * TILE + r) * L::SUM_LD + 4 * c) * 4, q), x);
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[k] += x[k];
                }
                const HeadsView& v = wg ? a.dk : a.dv;
                U* p = static_cast<U*>(v.p) + b * v.sb + kvh * v.sh + (int64_t)(j0 + r) * v.ss;
                if constexpr (SPLIT) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (4 * c + k < a.d) p[(4 * c + k) * v.sd] = s[k];
                } else {
                    *reinterpret_cast<uint2*>(p + 4 * c) = make_uint2(pack16<T>(s[0], s[1]), pack16<T>(s[2], s[3]));
                }
            }
            __syncwarp();
            // a block's sums stay until the others have read them
            cluster_sync();
        }
    }
    bb.finish(tmem);
}

// ---------------------------------------------------------------- dq
// TMEM: S of two tiles 0..255, dp (dx) 256..383, dq 384..511 (WIDE: S of one
// tile, dp, dq, its sum).
template <typename T, typename U, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(BW_THREADS, 1)
    k_attn_tc_dq(const __grid_constant__ HeadMap mq, const __grid_constant__ HeadMap mk, const __grid_constant__ HeadMap mv,
                 const __grid_constant__ HeadMap mdo, const __grid_constant__ BwArgs g) {
    using L = BwSmem<DP>;
    constexpr bool SPLIT = !std::is_same<T, U>::value;
    constexpr bool WIDE = L::WIDE;
    constexpr int DO = SPLIT ? DP / 2 : DP;   // columns of a result
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const AttnCall& a = g.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const unsigned bhs = (unsigned)a.b * a.hq;
    const int qt = g.q_tiles - 1 - (int)(blockIdx.x / bhs);
    const int h = (int)(blockIdx.x % bhs % a.hq), b = (int)(blockIdx.x % bhs / a.hq), kvh = h / (a.hq / a.hkv);
    const int i0 = qt * TILE, rows = min(TILE, a.nq - i0);
    const SeqMask mask(a, b);
    const int32_t* qd = a.q_doc ? a.q_doc + (int64_t)b * a.nq : nullptr;
    const int32_t* kd = a.k_doc ? a.k_doc + (int64_t)b * a.nk : nullptr;
    BwBlock bb(smem + L::BAR, smem + L::DOCS);
    DocRange mine;
    const uint32_t tmem = bb.setup(qd ? qd + i0 : nullptr, rows, &mine, false);
    const uint32_t t_dp = tmem + (WIDE ? 1 : 2) * TILE, t_dq = t_dp + TILE;
    const uint32_t t_dqa = t_dq + DO;   // split operands: the sum over the tiles
    TileWalk<> walk;
    walk.start(0, (max(mask.key_end(i0, rows), 0) + TILE - 1) / TILE, 0, max(mask.key_end(i0, 1), 0) / TILE,
               kd ? g.k_ranges + (int64_t)b * g.k_tiles : nullptr, mine);
    bool masked, ok = true;
    int kt = walk.next(&masked);
    const bool any = kt >= 0;

    if (warp >= BW_MMA) {
        fewer_registers<BwRegs<SPLIT && !WIDE>::FEWER>();
        if (warp == BW_TMA) {
            // ------------------------------------------------ TMA
            if (any && lane == 0) {
                mbar_expect_tx(bb.fix, L::RING);
                for (int f = 0; f < (WIDE ? 2 : 1); ++f) {
                    tma_tile(smem_u32(smem + L::FIX + f * L::TILE_B), mq, bb.fix, L::CH, i0, h, b, 2 * f);
                    tma_tile(smem_u32(smem + L::FIX + L::RING / 2 + f * L::TILE_B), mdo, bb.fix, L::CH, i0, h, b, 2 * f);
                }
            }
            int n = 0;
            if (WIDE) {
                // K and V halves in the order in which the products take them: of tile
                // n, S and dp, then dq of n (K again), S and dp of n + 1
                HalfRing ring(bb, smem + L::RING, g.err);
                for (; kt >= 0 && ok; kt = walk.next(&masked)) {
                    ring.load2(mk, kt, kvh, b, ok);
                    if (ok) ring.load2(mv, kt, kvh, b, ok);
                    if (ok) ring.load2(mk, kt, kvh, b, ok);
                }
                ring.drain(ok);
            }
            for (; !WIDE && kt >= 0 && ok; kt = walk.next(&masked), ++n) {
                const int s = n % BW_STAGES;
                if (n >= BW_STAGES) ok = warp_wait(&bb.empty[s], ((n / BW_STAGES) & 1) ^ 1, ok, g.err);
                if (ok && lane == 0) {
                    mbar_expect_tx(&bb.full[s], 2 * L::TILE_B);
                    const uint32_t at = smem_u32(smem + L::RING + s * 2 * L::TILE_B);
                    tma_tile(at, mk, &bb.full[s], L::CH, kt * TILE, kvh, b);
                    tma_tile(at + L::TILE_B, mv, &bb.full[s], L::CH, kt * TILE, kvh, b);
                }
            }
            if (!WIDE && !ok)
                for (int e = max(0, n - 1 - BW_STAGES); e < n - 1; ++e)
                    mbar_wait(&bb.full[e % BW_STAGES], (e / BW_STAGES) & 1, g.err);
        } else if (warp == BW_MMA) {
            // ------------------------------------------------ tensor cores
            const int ksteps = (a.d + 15) / 16;
            const uint32_t idesc = f16_idesc<T>(16 * ksteps, true);
            const uint32_t sq = smem_u32(smem + L::FIX), sdo = sq + L::RING / 2;
            auto rows = [&](uint32_t d, uint32_t x, uint32_t y) {
                if (SPLIT) mma_rows_split<T>(d, x, y, ksteps);
                else mma_rows<T, DP / 16>(d, x, y, ksteps);
            };
            auto parts = [&](uint32_t d, uint32_t x, uint32_t y, bool more) {
                if (SPLIT) mma_parts_split<BW_COLS>(d, x, y, idesc, 0);
                else mma_parts<BW_COLS>(d, x, y, idesc, more);
            };
            // keys that must not count: 0 times what they hold could be NaN
            auto clean = [&](int s) {
                if (SPLIT || !((kd && masked) || (mask.kv < a.nk && (kt + 1) * TILE > mask.kv))) return;
                clear_rows(smem + L::RING + s * 2 * L::TILE_B, L::CH, [&](int r) {
                    const int j = kt * TILE + r;
                    return j >= mask.kv || (kd && kd[j] < 0);
                });
                fence_proxy_async_smem();
                __syncwarp();
            };
            int n = 0;
            if (WIDE && any) {
                HalfRing ring(bb, smem + L::RING, g.err);
                ok = warp_wait(bb.fix, 0, ok, g.err);
                while (kt >= 0 && ok) {
                    ring.rows2<T>(tmem, sq, ksteps, &bb.s_full[0], ok);
                    ring.rows2<T>(t_dp, sdo, ksteps, bb.dp_full, ok);
                    ok = warp_wait(bb.dx_full, n & 1, ok, g.err);
                    ring.parts2<T>(t_dq, t_dp, ksteps, ok);
                    ++n;
                    kt = walk.next(&masked);
                }
                if (ok && elect_one()) umma_commit(bb.done);
                __syncwarp();
            }
            if (!WIDE && any) {
                ok = warp_wait(bb.fix, 0, ok, g.err);
                // queries of padding, likewise
                if (CAP && !SPLIT && qd && mine.pad) {
                    clear_rows(smem + L::FIX, L::CH, [&](int r) { return i0 + r < a.nq && qd[i0 + r] < 0; });
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                ok = warp_wait(&bb.full[0], 0, ok, g.err);
                if (ok) clean(0);
                const uint32_t sk = smem_u32(smem + L::RING);
                if (ok && elect_one()) {
                    rows(tmem, sq, sk);
                    umma_commit(&bb.s_full[0]);
                    rows(t_dp, sdo, sk + L::TILE_B);
                    umma_commit(bb.dp_full);
                }
                __syncwarp();
            }
            while (!WIDE && kt >= 0 && ok) {
                const int s = n % BW_STAGES, s1 = (n + 1) % BW_STAGES;
                const uint32_t sk = smem_u32(smem + L::RING + s * 2 * L::TILE_B);
                const uint32_t sk1 = smem_u32(smem + L::RING + s1 * 2 * L::TILE_B);
                kt = walk.next(&masked);
                if (kt >= 0) {
                    ok = warp_wait(&bb.full[s1], ((n + 1) / BW_STAGES) & 1, ok, g.err);
                    if (ok) clean(s1);
                    // the scores before last have been read: their dx came before
                    if (ok && elect_one()) {
                        rows(tmem + ((n + 1) & 1) * TILE, sq, sk1);
                        umma_commit(&bb.s_full[(n + 1) & 1]);
                    }
                    __syncwarp();
                }
                ok = warp_wait(bb.dx_full, n & 1, ok, g.err);
                if (ok && elect_one()) {
                    parts(t_dq, t_dp, sk, n > 0);
                    umma_commit(&bb.empty[s]);
                    if (kt >= 0) {
                        rows(t_dp, sdo, sk1 + L::TILE_B);
                        umma_commit(bb.dp_full);
                    } else {
                        umma_commit(bb.done);
                    }
                }
                __syncwarp();
                ++n;
            }
        }
    } else {
        // ---------------------------------------------------- 32 keys of a query per thread
        more_registers<BwRegs<SPLIT && !WIDE>::MORE>();
        const int wg = warp / 4, r = threadIdx.x % TILE, i = i0 + r;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const SplitExps ex = split_exps<SPLIT>(g, b, kvh);
        const float scale = SPLIT ? split_scale(a.scale, ex.q + ex.k) : a.scale, c1 = scale * kLog2e;
        const CapCoef<SPLIT> cap(scale, CAP ? a.cap : 1.f);
        const float slope2 = BIAS && a.slopes ? a.slopes[h] * kLog2e : 0.f;
        const float lift = dx_lift<T>(g, b, kvh), up = lift * PLift<T>::back;   // (split operands: dp and D carry the powers of dout and v)
        const float* st = g.stats + (((int64_t)b * a.hq + h) * g.q_tiles + qt) * 2 * TILE;
        const float nl = st[r], nd = st[TILE + r] * up;
        const f2 nl2 = pack2(nl, nl), nd2 = pack2(nd, nd);
        const int doc = qd && i < a.nq ? qd[i] : -1, limit = mask.key_end(i, 1);
        int n = 0;
        for (; kt >= 0 && ok; kt = walk.next(&masked), ++n) {
            const int jw = kt * TILE + wg * BW_COLS;
            uint32_t bits = 0xffffffffu;
            if (masked) {
                bits = low_bits(limit - jw, 0);
                if (kd) {
                    const int other[1] = {jw + lane < a.nk ? __ldg(kd + jw + lane) : -1};
                    uint32_t same[1];
                    doc_bits(other, doc, same);
                    bits &= same[0];
                }
            }
            const int buf = WIDE ? 0 : n & 1;
            ok = warp_wait(&bb.s_full[buf], (WIDE ? n : n / 2) & 1, ok, g.err);
            if (!ok) break;
            f2 x[16];
            tmem_load(tmem + buf * TILE + lanes + wg * BW_COLS, x);
            {
                uint32_t unused[16], low[16];
                grad_row<T, CAP, BIAS, SPLIT>(x, unused, low, c1, cap, slope2, jw - (mask.p0 + i), masked, bits,
                                       [&](int) { return nl2; });
            }
            ok = warp_wait(bb.dp_full, n & 1, ok, g.err);
            if (!ok) break;
            {
                // dq of the tile before, done before this dp
                if (SPLIT && n > 0) tmem_add<DO / 4>(t_dqa + lanes + wg * (DO / 4), t_dq + lanes + wg * (DO / 4), n == 1);
                uint32_t dp[32], dx[16], low[16];
                tmem_load(t_dp + lanes + wg * BW_COLS, dp);
                grad_dx<T, SPLIT>(x, dp, dx, low, up, masked, bits, [&](int) { return nd2; });
                tmem_st16(t_dp + lanes + wg * BW_COLS, dx);
                if (SPLIT) tmem_st16(t_dp + lanes + wg * BW_COLS + 16, low);
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bb.dx_full);
        }
        if (any) ok = warp_wait(bb.done, 0, ok, g.err);
        // each warpgroup writes a quarter of the columns
        if (ok) {
            constexpr int PART = DO / 4;
            uint32_t at = t_dq + lanes + wg * PART;
            if (SPLIT) {
                if (any) {
                    tmem_add<PART>(t_dqa + lanes + wg * PART, at, n == 1);
                    tmem_wait_st();
                }
                at = t_dqa + lanes + wg * PART;
            }
            const Factors<SPLIT> f(SPLIT ? a.scale : a.scale / lift, SPLIT ? -(ilogbf(lift) + ex.dout + ex.v + ex.k) : 0);
            HeadsView v = a.dq;
            v.p = static_cast<U*>(v.p) + wg * PART * v.sd;
            store_row<U, PART>(v, b, h, i, i < a.nq, a.d - wg * PART, at, any, any, f.mul, f.post);
        }
    }
    wait_for_previous();   // the dk, dv kernel, which this one did not need, so that its end is the call's
    bb.finish(tmem);
}

// dk and dv of a key head: the sums of its group's heads, in their order.
// Blocks of 8 rows of a key head, a warp a row.
__global__ void __launch_bounds__(256) k_sum_heads(const __grid_constant__ AttnCall a, const float* __restrict__ dk, const float* __restrict__ dv) {
    const int64_t n = (int64_t)a.nk * a.d;
    const int group = a.hq / a.hkv, lane = threadIdx.x & 31, blocks = (a.nk + 7) / 8;
    const int bh = blockIdx.x / blocks, row = blockIdx.x % blocks * 8 + threadIdx.x / 32;
    wait_for_previous();
    if (row >= a.nk) return;
    for (int w = 0; w < 2; ++w) {
        const float* p = (w ? dv : dk) + bh * group * n + (int64_t)row * a.d;
        const HeadsView& v = w ? a.dv : a.dk;
        float* out = static_cast<float*>(v.p) + bh / a.hkv * v.sb + bh % a.hkv * v.sh + row * v.ss;
        float sum[4] = {};   // columns lane, lane + 32, ...
        for (int q = 0; q < group; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (lane + 32 * e < a.d) sum[e] += p[q * n + lane + 32 * e];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (lane + 32 * e < a.d) out[(lane + 32 * e) * v.sd] = sum[e];
    }
}

bool sums_by_head(const AttnCall& a) { return a.dtype == TL_TYPE_F32 && a.d > 64 && a.hq > a.hkv; }

struct BwPlan {
    int q_tiles, k_tiles;
    size_t stats, norms, q_ranges, k_ranges, split, sums, bytes;
    explicit BwPlan(const AttnCall& a) {
        q_tiles = (a.nq + TILE - 1) / TILE;
        k_tiles = (a.nk + TILE - 1) / TILE;
        auto take = [&](size_t n) { const size_t at = bytes; bytes += (n + 255) / 256 * 256; return at; };
        bytes = 0;
        stats = take((size_t)a.b * a.hq * q_tiles * STAT_BYTES);
        norms = take(a.dtype == TL_TYPE_F16 ? (size_t)a.b * a.hkv * 8 : 0);
        q_ranges = take(a.q_doc ? (size_t)a.b * q_tiles * sizeof(DocRange) : 0);
        k_ranges = take(a.q_doc ? (size_t)a.b * k_tiles * sizeof(DocRange) : 0);
        split = take(a.dtype == TL_TYPE_F32 ? SplitPlan(a, true).bytes : 0);
        sums = take(sums_by_head(a) ? 2 * (size_t)a.b * a.hq * a.nk * a.d * sizeof(float) : 0);
    }
};

template <typename T, typename U, int DP, bool CAP, bool BIAS>
tl_status launch(tl_ctx* c, const HeadMap* m, const BwArgs& g, cudaStream_t s) {
    static std::atomic<uint64_t> done_kv{0}, done_q{0};
    constexpr int smem = BwSmem<DP>::BYTES;
    TL_TRY(kernel_smem(c, k_attn_tc_dkv<T, U, DP, CAP, BIAS>, smem, done_kv, BW_REGS));
    TL_TRY(kernel_smem(c, k_attn_tc_dq<T, U, DP, CAP, BIAS>, smem, done_q, BW_REGS));
    const AttnCall& a = g.a;
    cudaEvent_t ev[2];
    launch_begin_on(c, s, "attention_tc_dkv", 0, 8.0 * a.d * attn_pairs(a), ev);
    TL_CK(c, launch_with(k_attn_tc_dkv<T, U, DP, CAP, BIAS>, dim3((unsigned)((int64_t)g.k_tiles * a.b * (g.by_head ? a.hq : a.hkv * g.cluster))), g.cluster,
                         BW_THREADS, smem, true, s, m[0], m[1], m[2], m[3], g));
    TL_TRY(launch_end_on(c, s, ev));
    launch_begin_on(c, s, "attention_tc_dq", 0, 6.0 * a.d * attn_pairs(a), ev);
    TL_CK(c, launch_with(k_attn_tc_dq<T, U, DP, CAP, BIAS>, dim3((unsigned)((int64_t)g.q_tiles * a.b * a.hq)), 1, BW_THREADS, smem, true, s,
                         m[0], m[1], m[2], m[3], g));
    return launch_end_on(c, s, ev);
}

template <typename T, typename U, int DP>
tl_status launch_scores(tl_ctx* c, const HeadMap* m, const BwArgs& g, cudaStream_t s) {
    const bool bias = takes_slopes(g.a);
    if (g.a.cap > 0.f) return bias ? launch<T, U, DP, true, true>(c, m, g, s) : launch<T, U, DP, true, false>(c, m, g, s);
    return bias ? launch<T, U, DP, false, true>(c, m, g, s) : launch<T, U, DP, false, false>(c, m, g, s);
}

}  // namespace

bool attn_tc_backward_takes(const AttnCall& a) {
    if (!attn_tc_takes(a) || a.nq == 0 || a.hq == 0) return false;
    if (a.dtype == TL_TYPE_F32) return true;
    return tc_array(a.dout, a.b, a.hq, a.nq) && tc_array(a.dq, a.b, a.hq, a.nq) &&
           tc_array(a.dk, a.b, a.hkv, a.nk) && tc_array(a.dv, a.b, a.hkv, a.nk);
}

size_t attn_tc_backward_workspace(const AttnCall& a) { return BwPlan(a).bytes; }

tl_status launch_attn_tc_backward(tl_ctx* c, const AttnCall& a, void* ws, cudaStream_t s) {
    const BwPlan plan(a);
    uint8_t* w = static_cast<uint8_t*>(ws);
    float* stats = reinterpret_cast<float*>(w + plan.stats);
    uint32_t* norms = a.dtype == TL_TYPE_F16 ? reinterpret_cast<uint32_t*>(w + plan.norms) : nullptr;
    BwArgs g;
    g.a = a;
    g.stats = stats;
    g.norms = norms;
    g.q_tiles = plan.q_tiles;
    g.k_tiles = plan.k_tiles;
    const int group = a.hq / a.hkv;
    // clusters of two, larger ones only where that gives the GPU its blocks: a
    // cluster waits for as many free SMs of one GPC (2 x 2048 x 16 heads over 4:
    // clusters of 1, 2, 4 took 185, 109, 138 us; 8 x 512 x 16 over 2: 74, 45, 68)
    g.cluster = group % 2 ? 1 : 2;
    while (g.cluster > 1 && g.cluster < 8 && group % (2 * g.cluster) == 0 &&
           (int64_t)plan.k_tiles * a.b * a.hkv * g.cluster < c->sm_count * 2 / 3)
        g.cluster *= 2;
    // two blocks of the cluster for a head's query tiles where they and dq's
    // blocks find SMs of their own (2 x 512 x 4 heads over 2: bf16 24 -> 21, fp32
    // 42 -> 33 us; 2 x 512 x 8 heads, too many: bf16 22 -> 28); fp32 walks, longer
    // a tile, gain from a causal call's shorter longest one for longer (2048 x 4 heads 78 -> 62,
    // 1024 x 8 54 -> 49, but 2 x 512 x 8 42 -> 43, 1024 x 16 over 4 60 -> 81).  Four never paid.
    const int64_t kv_blocks = (int64_t)plan.k_tiles * a.b * a.hkv * g.cluster, q_blocks = (int64_t)plan.q_tiles * a.b * a.hq;
    g.abreast = g.cluster;
    g.parts = 1;
    if (g.cluster <= 4 && plan.q_tiles > 1 &&
        2 * kv_blocks + q_blocks <= (a.dtype == TL_TYPE_F32 && a.causal ? c->sm_count * 3 / 2 : c->sm_count)) {
        g.parts = 2;
        g.cluster *= 2;
    }
    g.by_head = 0;
    g.dk = a.dk;
    g.dv = a.dv;
    g.err = c->d_flags + 8;
    c->flags_armed = true;
    DocRange *q_ranges = reinterpret_cast<DocRange*>(w + plan.q_ranges), *k_ranges = reinterpret_cast<DocRange*>(w + plan.k_ranges);
    g.q_ranges = q_ranges;
    g.k_ranges = k_ranges;
    HeadMap m[4];
    const double rows = (double)a.b * a.hq * a.nq;
    const int64_t tiles = (int64_t)a.b * a.hq * plan.q_tiles;
    cudaEvent_t ev[2];
    if (a.dtype == TL_TYPE_F32) {
        uint8_t* sw = w + plan.split;
        const SplitPlan sp(a, true);
        TL_TRY(launch_split(c, a, stats, sw, m, q_ranges, k_ranges, s));
        g.norms = reinterpret_cast<const uint32_t*>(sw + sp.norms);
        g.tops.q = reinterpret_cast<const uint32_t*>(sw + sp.top);
        g.tops.k = g.tops.q + (size_t)a.b * a.hkv;
        g.tops.v = g.tops.k + (size_t)a.b * a.hkv;
        g.tops.dout = g.tops.v + (size_t)a.b * a.hkv;
        if (a.d > 64) {
            g.cluster = g.abreast = g.parts = 1;
            if (!sums_by_head(a)) return launch_scores<__half, float, 256>(c, m, g, s);
            float* sums = reinterpret_cast<float*>(w + plan.sums);
            const int64_t one = (int64_t)a.b * a.hq * a.nk * a.d;
            g.by_head = 1;
            g.dk = {sums, (int64_t)a.hq * a.nk * a.d, (int64_t)a.nk * a.d, a.d, 1};
            g.dv = {sums + one, g.dk.sb, g.dk.sh, g.dk.ss, 1};
            TL_TRY((launch_scores<__half, float, 256>(c, m, g, s)));
            launch_begin_on(c, s, "attention_sum_heads", 4.0 * 2 * (one + one / a.hq * a.hkv), 0, ev);
            TL_CK(c, launch_with(k_sum_heads, dim3((unsigned)((int64_t)a.b * a.hkv * ((a.nk + 7) / 8))), 1, 256, 0, false, s, a,
                                 static_cast<const float*>(sums), static_cast<const float*>(sums + one)));
            return launch_end_on(c, s, ev);
        }
        return launch_scores<__half, float, 128>(c, m, g, s);
    }
    g.tops = {nullptr, nullptr, nullptr, nullptr};
    if (!make_head_map(&m[0], a.q, a.dtype, a.b, a.hq, a.nq, a.d) || !make_head_map(&m[1], a.k, a.dtype, a.b, a.hkv, a.nk, a.d) ||
        !make_head_map(&m[2], a.v, a.dtype, a.b, a.hkv, a.nk, a.d) || !make_head_map(&m[3], a.dout, a.dtype, a.b, a.hq, a.nq, a.d))
        return fail(c, TL_ERR_CUDA, "attention: tensor maps");
    TL_TRY(launch_attn_begin(c, a, q_ranges, k_ranges, norms, norms ? (int64_t)a.b * a.hkv * 2 : 0, s));
    const int64_t blocks = tiles + (norms ? (int64_t)a.b * a.hkv * plan.k_tiles : 0);
    launch_begin_on(c, s, "attention_prep", 4.0 * rows * a.d, 2.0 * rows * a.d, ev);
    // early behind launch_attn_begin's kernel where there is one
    TL_CK(c, launch_with(a.dtype == TL_TYPE_F16 ? k_attn_prep<__half> : k_attn_prep<__nv_bfloat16>, dim3((unsigned)(2 * blocks)), 1, 256, 0,
                         norms || a.q_doc, s, a, stats, norms, plan.q_tiles, plan.k_tiles));
    TL_TRY(launch_end_on(c, s, ev));
    if (a.dtype == TL_TYPE_F16)
        return a.d <= 64 ? launch_scores<__half, __half, 64>(c, m, g, s) : launch_scores<__half, __half, 128>(c, m, g, s);
    return a.d <= 64 ? launch_scores<__nv_bfloat16, __nv_bfloat16, 64>(c, m, g, s)
                     : launch_scores<__nv_bfloat16, __nv_bfloat16, 128>(c, m, g, s);
}

}  // namespace tl
