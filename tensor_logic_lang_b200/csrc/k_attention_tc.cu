// Attention forward on the tensor cores: 16-bit operands, or fp32 arrays as
// pairs of fp16 (attn_tc.h, SplitArray), head size up to 128; one pass over the
// keys with a running maximum and sum.
//
// A block owns two tiles of 128 queries that read the same keys: the same
// rows of two heads of a group where the group has an even number of heads
// (each causal tile then needs exactly the keys the block loads), else
// neighbouring rows of one head; or one tile (launch_tiles says when), and two
// such blocks share an SM.  Few queries: a tile holds those of all heads of a
// group (packed_queries).  Few tiles: a cluster's blocks share the keys of one,
// every parts-th key tile each, and add up.  Warps of two tiles:
//   0-7, 8-15  tile 0, 1: a thread has 64 of a query's 128 scores: scores out
//              of TMEM, softmax statistics (the two halves of a row agree on
//              its maximum through shared memory), probabilities (16-bit) back
//              into TMEM over the scores
//   16         tensor cores: S = Q K^T (SMEM x SMEM), O += P V (TMEM x SMEM)
//   17         TMA: Q once, then K and V tiles through a ring of four (two
//              where two blocks share the shared memory)
// TMEM: S0 S1 (128 columns each, P over the first half of each 64), O0 O1.  While one
// tile's softmax runs, the other tile's products do; S of the next keys is
// issued right behind P V of these, which orders it after P is read.
//
// With m the row's reference maximum, p = 2^(s log2 e - m): O is rescaled only
// when a row's maximum has grown by more than 2^8 (fp32 sums and 16-bit p have
// the range), so most tiles touch O not at all.  l sums the unrounded p.
// P is rounded to the operand type: the tensor cores take 16-bit operands;
// each p is off by half a step, which weighs like the rounding of v.
//
// fp32 arrays: Q, K and V come as hi and lo, P is written as hi (over the first
// half of S) and lo (over the second), and each product is three.  The tensor
// cores cut their sums by 2^-23 a step, which over many keys adds up to more
// than fp32 loses, so P V of a tile goes into columns of its own, and the row's
// thread adds them to the sum, also in TMEM, behind S, with rounded additions.
//
// Bound by the softmax threads' chain (TMEM loads, maximum, exponentials, TMEM
// stores; with a cap the tanh's polynomial too), not by the products: 1 x 32/8 heads x 4096 x
// 128, cap 50, keep the tensor pipe busy for 41 % of the clocks, the exponentials' pipe for 42 %.
// 16 heads of 16384 queries and keys, bf16, causal: d 128 950 to 1070 us (the power cap), 1160 to
// 1030 TFLOP/s, cap 50 1260; d 64 780 us, 705 TFLOP/s, cap 50 946.
// With a thread a whole row, and MMAs issued by lane 0 with descriptors made for
// each, 910 and 669 TFLOP/s where this reached 1083 and 867 (not causal).
#include <algorithm>

#include "attn_tc.h"

namespace tl {
namespace {

// Capped scores lie in +-top (base 2), so bf16, which has the range of fp32,
// needs no maximum: p = 2^s lies in 2^-top .. 2^top, and up to top = 72.5 (softcap 50.2)
// its products with v and their sums stay normal numbers of fp32 for |v| of 2^-53 to
// 2^54 / keys.  No maxima, no agreeing on them, no rescaling (1 x 32/8 heads x 4096 x 128,
// causal, cap 50: 161 us, 174 with them).
constexpr float kFixTop = 72.5f;
constexpr float kFuseTop = 0x1p12f;   // half a step of it is 2^-12, less than P's rounding
constexpr float kGrow = 8.f;   // rescale when the maximum grew by 2^8

struct FwArgs {
    AttnCall a;
    const DocRange* k_ranges;   // [b, key tiles] with documents
    int pair_heads;             // two tiles: heads h, h + 1 (else rows i0, i0 + 128)
    int pack;                   // one tile: queries of it, of all heads of a group, head after head; 0: one head's
    int key_tiles;
    int parts;                  // one tile: blocks (a cluster) that share its keys
    SplitTops tops;             // fp32 arrays
    int* err;
};

// NT query tiles a block.  One: two blocks share an SM where TMEM and shared
// memory allow it, with half of each.
template <typename T, typename U, int DP, int NT>
struct Fw {
    static constexpr bool SPLIT = !std::is_same<T, U>::value;
    static constexpr int HALVES = DP > 128 ? 2 : 1;   // split operands of more than 64 columns: a tile is two, one behind the other
    static constexpr int DO = SPLIT ? DP / 2 : DP;    // columns of O
    static constexpr int SOFTMAX = 256 * NT, THREADS = SOFTMAX + (HALVES == 2 ? 64 : 128), MMA = SOFTMAX / 32, TMA = MMA + 1;   // threads, warps
    // registers a thread: at launch, of the softmax warps, of the last warpgroup (bf16, 32/8
    // heads of 4096, d 128, cap 50: 182 us without a split, 165 with; fp32, 8 heads of 2048, d 64: 65, 60)
    static constexpr int REGS = HALVES == 2 ? 0 : NT == 2 ? 96 : 80, MORE = NT == 2 ? 112 : 104, FEWER = 32;
    static_assert(!REGS || SOFTMAX * MORE + 128 * FEWER <= THREADS * REGS, "the split waits for ever");
    static constexpr int CH = DP / HALVES / 64, TILE_B = CH * CHUNK_BYTES;
    static constexpr int PER_SM = NT == 1 && HALVES == 1 ? 2 : 1;
    static constexpr int STAGES = PER_SM == 2 && CH == 2 ? 2 : 4;
    // TMEM: S of the tiles, O of the tiles, split operands: the sums over the key tiles
    static constexpr int T_O = NT * TILE, T_ACC = T_O + NT * DO, TMEM = T_ACC + (SPLIT ? NT * DO : 0) <= 256 ? 256 : 512;
    static_assert(T_ACC + (SPLIT ? NT * DO : 0) <= 512 && PER_SM * TMEM <= 512, "TMEM columns");
    static constexpr int Q = 0, KV = NT * HALVES * TILE_B, BAR = KV + STAGES * TILE_B, DOCS = BAR + 256, ROWS = DOCS + 64,
                         BYTES = ROWS + 2 * 2 * NT * TILE * 4 + 1024;   // ROWS: [parity][tile][half][row]
    // shared keys, behind the walk: O as rows padded by 16 bytes, m and l of each row
    static constexpr int OUT_ROW = DO + 4, STATS = TILE * OUT_ROW * 4;
    static_assert(STATS + TILE * 8 <= BAR, "the rows to add fit where Q, K and V were");
};

// Behind which a call's other kernels start early: the smallest and largest
// document of each query and key tile (a warp a tile; null: not wanted), and
// words that maxima are taken in.
struct BeginArgs {
    const int32_t *q_doc, *k_doc;
    int nq, nk;
    int64_t q_total, k_total;      // tiles of all sequences
    DocRange *q_out, *k_out;
    uint32_t* zero;
    int64_t words;
};
__global__ void __launch_bounds__(256) k_attn_begin(const __grid_constant__ BeginArgs g) {
    let_next_start();
    const int lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (int64_t w = at; w < g.words; w += (int64_t)gridDim.x * blockDim.x) g.zero[w] = 0;
    int64_t t = at >> 5;
    if (t >= g.q_total + g.k_total) return;
    const bool keys = t >= g.q_total;
    if (keys) t -= g.q_total;
    const int32_t* doc = keys ? g.k_doc : g.q_doc;
    const int n = keys ? g.nk : g.nq, tiles = (n + TILE - 1) / TILE;
    const int64_t b = t / tiles;
    const int j0 = (int)(t % tiles) * TILE;
    DocRange r = no_docs();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int j = j0 + 32 * w + lane;
        const int d = j < n ? doc[b * n + j] : -1;
        if (d >= 0) { r.lo = min(r.lo, d); r.hi = max(r.hi, d); }
        else r.pad = 1;
    }
    r.lo = __reduce_min_sync(0xffffffffu, r.lo);
    r.hi = __reduce_max_sync(0xffffffffu, r.hi);
    r.pad = __reduce_max_sync(0xffffffffu, r.pad);
    if (lane == 0) (keys ? g.k_out : g.q_out)[t] = r;
}

// 64 scores of this thread's row: x (q.k) in registers becomes the
// score in base 2 times c (see below), with -inf where the key is not seen.
// Returns the row's largest c-scaled score.
//   !CAP && !BIAS: x is left as it is and c = scale log2 e; else c = 1.
//   FINE: the tanh to fp32; FIX: no maximum is taken
template <bool CAP, bool BIAS, bool FINE, bool FIX>
__device__ __forceinline__ float score_row(f2 (&x)[32], float c1, const CapCoef<FINE>& cap, float slope2, int p, int j0,
                                           bool masked, uint32_t bits0, uint32_t bits1) {
    if (CAP) cap_scores<BIAS>(x, cap);
    if (BIAS) {
        // -slope |p - j| is linear in j on either side of p
        const bool before = __all_sync(0xffffffffu, j0 + 63 <= p), after = __all_sync(0xffffffffu, j0 >= p);
        const f2 c = CAP ? pack2(1.f, 1.f) : pack2(c1, c1);
        if (before || after) {
            const float k = before ? slope2 : -slope2, kb = k * (float)(j0 - p);
            const f2 kk = pack2(k, k), base = pack2(kb, kb);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const f2 bias = fma2(kk, pack2((float)(2 * i), (float)(2 * i + 1)), base);
                x[i] = CAP ? add2(x[i], bias) : fma2(x[i], c, bias);
            }
        } else {
            const float at = (float)(j0 - p);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const f2 bias = pack2(-slope2 * fabsf(at + (float)(2 * i)), -slope2 * fabsf(at + (float)(2 * i + 1)));
                x[i] = CAP ? add2(x[i], bias) : fma2(x[i], c, bias);
            }
        }
    }
    if (masked) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float lo, hi;
            unpack2(x[i], lo, hi);
            const uint32_t w = i < 16 ? bits0 : bits1;
            lo = (w >> (2 * i % 32)) & 1 ? lo : -INFINITY;
            hi = (w >> (2 * i % 32 + 1)) & 1 ? hi : -INFINITY;
            x[i] = pack2(lo, hi);
        }
    }
    if (FIX) return 0.f;
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        float lo, hi;
        unpack2(x[i], lo, hi);
        top[i % 4] = fmaxf(top[i % 4], fmaxf(lo, hi));
    }
    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

// The rows of a tile whose keys the blocks of a cluster shared: with m and l of
// block q, w_q = 2^(m_q - max m), o = sum w_q O_q / sum w_q l_q, added in the
// order of the blocks.  Each block stores TILE / parts rows, a warp a row.
template <typename T, typename U, typename L, bool FIX>
__device__ void join_parts(uint8_t* smem, const FwArgs& g, int part, int b, int h0, int kvh, int i0) {
    const AttnCall& a = g.a;
    const int parts = g.parts, rows = g.pack ? g.pack * (a.hq / a.hkv) : TILE;
    const int lane = threadIdx.x & 31, share = TILE / parts, d0 = 4 * lane;
    const float out_scale = L::SPLIT ? pow2(-split_exp(g.tops.v, b * a.hkv + kvh)) : 1.f;
    for (int r = part * share + threadIdx.x / 32; r < min((part + 1) * share, rows); r += L::SOFTMAX / 32) {
        const int i = g.pack ? i0 + r % g.pack : i0 + r, h = g.pack ? h0 + r / g.pack : h0;
        if (i >= a.nq) continue;
        float m = -INFINITY, l = 0.f;
        if (lane < parts)
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(m), "=f"(l) : "r"(in_block(smem_u32(smem + L::STATS) + r * 8, lane)));
        if (l == 0.f) m = -INFINITY;
        float top = m;
        for (int s = 4; s; s /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s, 8));
        const float w = l == 0.f ? 0.f : ex2(m - top);
        float sum = 0.f, o[4] = {};
        for (int q = 0; q < parts; ++q) {
            const float wq = __shfl_sync(0xffffffffu, w, q);
            sum += wq * __shfl_sync(0xffffffffu, l, q);
            if (d0 < L::DO) {
                float x[4];
                load_cluster4(in_block(smem_u32(smem) + (r * L::OUT_ROW + d0) * 4, q), x);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] += wq * x[e];
            }
        }
        const bool none = sum == 0.f;
        const float inv = none ? 0.f : 1.f / sum;
        U* p = static_cast<U*>(a.o.p) + b * a.o.sb + h * a.o.sh + i * a.o.ss;
        if constexpr (std::is_same<U, float>::value) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d0 + e < a.d) p[(d0 + e) * a.o.sd] = none ? 0.f : o[e] * inv * out_scale;
        } else if (d0 < a.d) {   // d is a multiple of 8, the rows lie on 16 bytes
            *reinterpret_cast<uint2*>(p + d0) =
                none ? make_uint2(0, 0) : make_uint2(pack16<U>(o[0] * inv, o[1] * inv), pack16<U>(o[2] * inv, o[3] * inv));
        }
        if (a.lse && lane == 0)
            a.lse[((int64_t)b * a.hq + h) * a.nq + i] =
                none ? -INFINITY : (FIX ? 0.f : top - Lift<T>::log2) * kLn2 + logf(sum);
    }
}

// T: operands, U: the arrays' type (float: split operands, DP = 128 or 256 columns
// of hi and lo).  FIX: see kFixTop.
template <typename T, typename U, int DP, int NT, bool CAP, bool BIAS, bool FIX>
__global__ void __launch_bounds__(Fw<T, U, DP, NT>::THREADS, Fw<T, U, DP, NT>::PER_SM)
    k_attn_tc(const __grid_constant__ HeadMap mq, const __grid_constant__ HeadMap mk, const __grid_constant__ HeadMap mv,
              const __grid_constant__ FwArgs g) {
    using L = Fw<T, U, DP, NT>;
    constexpr bool SPLIT = L::SPLIT;
    constexpr int HALVES = L::HALVES, DO = L::DO;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::BAR);
    uint64_t *q_full = bar, *full = bar + 1, *empty = full + L::STAGES, *s_full = empty + L::STAGES, *p_full = s_full + 2,
             *o_done = p_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 24);
    int* docs = reinterpret_cast<int*>(smem + L::DOCS);   // lo, hi, pad of the block's rows
    const AttnCall& a = g.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;

    // block -> (rows, heads, sequence); the last rows, which see the most keys
    // of a causal call, go first
    const int group = a.hq / a.hkv;
    const int pack = NT == 1 ? g.pack : 0;
    const int units = pack ? a.hkv : g.pair_heads ? a.hq / 2 : a.hq;
    const int span = pack ? pack : g.pair_heads ? TILE : NT * TILE;
    const int row_blocks = (a.nq + span - 1) / span;
    const unsigned per_row = (unsigned)units * a.b;
    const int parts = NT == 1 ? g.parts : 1, part = NT == 1 ? blockIdx.x % g.parts : 0;
    const unsigned block = NT == 1 ? blockIdx.x / g.parts : blockIdx.x;
    const int rb = row_blocks - 1 - (int)(block / per_row);
    const unsigned u = block % per_row;
    const int b = u / units, h0 = (u % units) * (pack ? group : g.pair_heads ? 2 : 1), kvh = h0 / group;
    const int i0 = rb * span, rows = min(span, a.nq - i0);
    const SeqMask mask(a, b);
    const int32_t* qd = NT == 1 && a.q_doc ? a.q_doc + (int64_t)b * a.nq : nullptr;
    const int32_t* kd = NT == 1 && a.k_doc ? a.k_doc + (int64_t)b * a.nk : nullptr;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int s = 0; s < L::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int t = 0; t < NT; ++t) { mbar_init(&s_full[t], 1); mbar_init(&p_full[t], 2 * TILE); mbar_init(&o_done[t], 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        docs[0] = 0x7fffffff; docs[1] = -1; docs[2] = 0;
    }
    if (warp == L::MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)L::TMEM));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (pack) {
        // rows of no query: what they hold would have a say in their warp's common choices
        // (rescaling, the tanh's form), and so in the last bits of the others
        const int first = pack * group * 128, n = (CHUNK_BYTES - first) / 16;
        for (int e = threadIdx.x; e < HALVES * L::CH * n; e += L::THREADS)
            *reinterpret_cast<uint4*>(smem + L::Q + e / n * CHUNK_BYTES + first + e % n * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
    }
    if (warp == L::TMA && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&mq.map)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&mk.map)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&mv.map)) : "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    wait_for_previous();   // the documents' ranges, the split operands
    DocRange mine = no_docs();
    if (qd) {
        const int r = threadIdx.x;
        const int d = r < rows ? qd[i0 + r] : -1;
        const int lo = __reduce_min_sync(0xffffffffu, d >= 0 ? d : 0x7fffffff), hi = __reduce_max_sync(0xffffffffu, d);
        const int pad = __any_sync(0xffffffffu, d < 0);
        if (lane == 0) {
            atomicMin(&docs[0], lo);
            atomicMax(&docs[1], hi);
            if (pad && warp * 32 < rows) docs[2] = 1;
        }
        __syncthreads();
        mine = {docs[0], docs[1], docs[2], 0};
    }
    TileWalk<NT == 1> walk;
    {
        const int end = (max(mask.key_end(i0, rows), 0) + TILE - 1) / TILE;
        // every row sees the keys that the first one sees
        const int clear = max(mask.key_end(i0, 1), 0) / TILE;
        walk.start(0, end, 0, clear, kd ? g.k_ranges + (int64_t)b * g.key_tiles : nullptr, mine, parts, part);
    }
    bool masked, ok = true;
    // by every warp: gives the TMEM back
    auto end_of_walk = [&]() {
        tc_fence_before();
        __syncthreads();
        if (warp == L::MMA) {
            tc_fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::TMEM));
        }
    };

    if (warp >= L::MMA) {
        if constexpr (L::REGS > 0) fewer_registers<L::FEWER>();
        if (warp == L::TMA) {
            // ------------------------------------------------ TMA
            int kt = walk.next(&masked);
            int n = 0;   // ring entries filled
            if (kt >= 0 && lane == 0) {
                mbar_expect_tx(q_full, pack ? HALVES * L::CH * pack * group * 128 : NT * HALVES * L::TILE_B);
                for (int t = 0; t < NT; ++t)
                    for (int f = 0; f < HALVES; ++f)
                        tma_tile(smem_u32(smem + L::Q + (t * HALVES + f) * L::TILE_B), mq, q_full, L::CH,
                                 i0 + (g.pair_heads ? 0 : t * TILE), h0 + (g.pair_heads ? t : 0), b, f * L::CH);
            }
            for (; kt >= 0 && ok; kt = walk.next(&masked)) {
                for (int w = 0; w < 2 * HALVES && ok; ++w, ++n) {
                    const int s = n % L::STAGES;
                    ok = n < L::STAGES || mbar_wait(&empty[s], ((n / L::STAGES) & 1) ^ 1, g.err);
                    ok = __all_sync(0xffffffffu, ok);
                    if (ok && lane == 0) {
                        mbar_expect_tx(&full[s], L::TILE_B);
                        tma_tile(smem_u32(smem + L::KV + s * L::TILE_B), w / HALVES ? mv : mk, &full[s], L::CH, kt * TILE, kvh, b,
                                 w % HALVES * L::CH);
                    }
                }
            }
            if (!ok)   // copies in flight land before the block ends
                for (int e = max(0, n - L::STAGES); e < n - 1; ++e) mbar_wait(&full[e % L::STAGES], (e / L::STAGES) & 1, g.err);
        } else if (warp == L::MMA) {
            // ------------------------------------------------ tensor cores
            const int ksteps = (a.d + 15) / 16;
            const uint32_t idesc_o = f16_idesc<T>(16 * ksteps, true);
            int kt = walk.next(&masked);
            int n = 0;
            auto wait_full = [&](uint64_t* bars, int i, int stages) {
                ok = ok && mbar_wait(&bars[i % stages], (i / stages) & 1, g.err);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after();
            };
            // the ring entry e's tile
            auto entry = [&](int e) { return smem_u32(smem + L::KV + e % L::STAGES * L::TILE_B); };
            auto scores = [&](int t, int e) {
                if (ok && elect_one()) {
                    const uint32_t sq = smem_u32(smem + L::Q + t * HALVES * L::TILE_B);
                    if (HALVES == 2) {
                        mma_rows_split<T>(tmem + t * TILE, sq, entry(e), 4);
                        mma_rows_split<T, true>(tmem + t * TILE, sq + L::TILE_B, entry(e + 1), ksteps - 4);
                    } else if (SPLIT) {
                        mma_rows_split<T>(tmem + t * TILE, sq, entry(e), ksteps);
                    } else {
                        mma_rows<T, DP / 16>(tmem + t * TILE, sq, entry(e), ksteps);
                    }
                    umma_commit(&s_full[t]);
                }
                __syncwarp();
            };
            auto free_entries = [&](int e) {   // by one lane
                for (int f = 0; f < HALVES; ++f) umma_commit(&empty[(e + f) % L::STAGES]);
            };
            auto wait_entries = [&](int e) {
                for (int f = 0; f < HALVES; ++f) wait_full(full, e + f, L::STAGES);
            };
            // Rows of padding are zeros where they count: those of V, since 0 probability times
            // what they hold could be NaN; with a cap those of K and Q, whose scores would
            // have a say in the tanh's form of their warps, and so in the others' last bits.
            auto padded = [&](int tile, bool mk) { return !SPLIT && ((kd && mk) || (mask.kv < a.nk && (tile + 1) * TILE > mask.kv)); };
            auto clean = [&](int e, int tile) {
                clear_rows(smem + L::KV + e % L::STAGES * L::TILE_B, L::CH, [&](int r) {
                    const int j = tile * TILE + r;
                    return j >= mask.kv || (kd && kd[j] < 0);
                });
                fence_proxy_async_smem();
                __syncwarp();
            };
            if (kt >= 0) {
                wait_full(q_full, 0, 1);
                if (CAP && !SPLIT && ok && qd && mine.pad) {
                    clear_rows(smem + L::Q, L::CH, [&](int r) {
                        const int i = i0 + (pack ? r % pack : r);
                        return i < a.nq && qd[i] < 0;
                    });
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                wait_entries(n);
                if (CAP && ok && padded(kt, masked)) clean(n, kt);
                for (int t = 0; t < NT; ++t) scores(t, n);
                if (ok && elect_one()) free_entries(n);
                n += HALVES;
            }
            for (int it = 0; kt >= 0 && ok; ++it) {
                const int vs = n;   // V's entries
                wait_entries(n);
                n += HALVES;
                if (ok && padded(kt, masked)) clean(vs, kt);
                bool next_masked;
                const int next = walk.next(&next_masked);
                if (next >= 0) {
                    wait_entries(n);   // the next keys: nothing waits between P V and S
                    if (CAP && ok && padded(next, next_masked)) clean(n, next);
                }
                for (int t = 0; t < NT; ++t) {
                    ok = ok && mbar_wait(&p_full[t], it & 1, g.err);
                    ok = __all_sync(0xffffffffu, ok);
                    tc_fence_after();
                    if (ok && elect_one()) {
                        const uint32_t to = tmem + L::T_O + t * DO, tp = tmem + t * TILE;
                        if (HALVES == 2) {
                            mma_parts_split<64>(to, tp, entry(vs), f16_idesc<T>(64, true), 0);
                            mma_parts_split<64>(to + 64, tp, entry(vs + 1), f16_idesc<T>(16 * (ksteps - 4), true), 0);
                        } else if (SPLIT) {
                            mma_parts_split<64>(to, tp, entry(vs), idesc_o, 0);
                        } else {
                            mma_parts<64>(to, tp, entry(vs), idesc_o, it > 0);
                        }
                        if (next < 0) umma_commit(&o_done[t]);
                    }
                    __syncwarp();
                    if (next >= 0) scores(t, n);
                }
                if (ok && elect_one()) {
                    free_entries(vs);
                    if (next >= 0) free_entries(n);
                }
                __syncwarp();
                if (next >= 0) n += HALVES;
                kt = next;
                masked = next_masked;
            }
        }
        __syncwarp();
        end_of_walk();
        if (NT == 1 && parts > 1) {   // as the softmax warps below, which keep their registers to the end
            cluster_sync();
            cluster_sync();
        }
    } else {
        // ---------------------------------------------------- half a row per thread
        if constexpr (L::REGS > 0) more_registers<L::MORE>();
        const int t = warp / 8, half = warp / 4 % 2, r = threadIdx.x % TILE;
        const int head = pack ? r / pack : 0;   // of the group
        const int i = pack ? i0 + r % pack : i0 + r + (g.pair_heads ? 0 : t * TILE);
        const int h = h0 + (pack ? min(head, group - 1) : g.pair_heads ? t : 0);
        const bool on = i < a.nq && (!pack || head < group);
        const int p = mask.p0 + i, limit = mask.key_end(i, 1);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        constexpr int DH = DO / 2;            // this thread's columns of O
        const uint32_t ts = tmem + t * TILE + half * 64 + lanes, to = tmem + L::T_O + t * DO + half * DH + lanes;
        const uint32_t acc = SPLIT ? to + NT * DO : to;   // the sum over the tiles
        float* rows_at = reinterpret_cast<float*>(smem + L::ROWS) + t * 2 * TILE + r;   // [parity][tile][half][row]
        // split operands carry powers of two of their heads
        const int e_qk = SPLIT ? split_exp(g.tops.q, b * a.hkv + kvh) + split_exp(g.tops.k, b * a.hkv + kvh) : 0;
        const float scale = SPLIT ? split_scale(a.scale, e_qk) : a.scale;
        const float c1 = scale * kLog2e, c = CAP || BIAS ? 1.f : c1;
        const CapCoef<SPLIT> cap(scale, CAP ? a.cap : 1.f);
        const float slope2 = BIAS && a.slopes ? a.slopes[h] * kLog2e : 0.f;
        const int doc = qd && i < a.nq ? qd[i] : -1;
        float m = -INFINITY, l = 0.f;
        int it = 0;
        for (int kt = walk.next(&masked); kt >= 0; kt = walk.next(&masked), ++it) {
            const int j0 = kt * TILE + half * 64;
            uint32_t bits0 = 0xffffffffu, bits1 = 0xffffffffu;
            if (masked) {
                bits0 = low_bits(limit - j0, 0);
                bits1 = low_bits(limit - j0, 1);
                if (kd) {
                    const int other[2] = {j0 + lane < a.nk ? __ldg(kd + j0 + lane) : -1,
                                          j0 + 32 + lane < a.nk ? __ldg(kd + j0 + 32 + lane) : -1};
                    uint32_t same[2];
                    doc_bits(other, doc, same);
                    bits0 &= same[0];
                    bits1 &= same[1];
                }
            }
            // a warp whose wait runs out walks on without waiting: the other warps of the tile meet it at
            // the barrier of the maxima once a key tile, which has no limit
            ok = ok && mbar_wait(&s_full[t], it & 1, g.err);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            if (SPLIT && it > 0) tmem_add<DH>(acc, to, it == 1);   // P V of the tile before, done before this S
            f2 x[32];
            tmem_load(ts, x);
            float top = c * score_row<CAP, BIAS, SPLIT, FIX>(x, c1, cap, slope2, p, j0, masked, bits0, bits1);
            if (!FIX) {
                // the row's other half
                float* mine_at = rows_at + (it & 1) * 2 * NT * TILE;
                mine_at[half * TILE] = top;
                asm volatile("bar.sync %0, 256;" ::"r"(1 + t) : "memory");
                top = fmaxf(top, mine_at[(1 - half) * TILE]);
                // a new reference maximum, for the first seen key of a row or a large step
                if (__any_sync(0xffffffffu, top > m + kGrow || (m == -INFINITY && top > m))) {
                    const float nm = fmaxf(m, top);
                    const float by = nm == -INFINITY ? 1.f : ex2(m - nm);
                    l *= by;
                    m = nm;
                    if (it > 0) {
                        if (SPLIT) tmem_wait_st();
                        const f2 by2 = pack2(by, by);
#pragma unroll 1
                        for (int k = 0; k < DH / 16; ++k) {
                            uint32_t o[16];
                            tmem_ld16(acc + 16 * k, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                float lo, hi;
                                unpack2(mul2(pack2(__uint_as_float(o[2 * q]), __uint_as_float(o[2 * q + 1])), by2), lo, hi);
                                o[2 * q] = __float_as_uint(lo);
                                o[2 * q + 1] = __float_as_uint(hi);
                            }
                            tmem_st16(acc + 16 * k, o);
                        }
                    }
                }
            }
            // p = 2^(c x - m), -inf gives 0; a row with no key yet keeps m = 0 here
            const float ref = (m == -INFINITY ? 0.f : m) - Lift<T>::log2;
            // c x - m in one step keeps what rounding m cut off, half a step of m: nothing of
            // the row's sum is left, or more than fp16 holds, where that is many powers of two.
            // Large scores are rounded before, as m was (rows beside theirs then too, by at
            // most 2^-12 of a power of two).
            float by = c;
            if (!CAP && !BIAS && __any_sync(0xffffffffu, m > -INFINITY && fabsf(m) > kFuseTop)) {
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = mul2(x[i], pack2(c, c));
                by = 1.f;
            }
            const f2 c2 = pack2(by, by), ref2 = pack2(-ref, -ref);
            f2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t out[16], low[SPLIT ? 16 : 1];
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    float lo, hi;
                    unpack2(FIX ? x[16 * k + q] : CAP || BIAS ? add2(x[16 * k + q], ref2) : fma2(x[16 * k + q], c2, ref2), lo, hi);
                    lo = ex2(lo);
                    hi = ex2(hi);
                    sum[q & 1] = add2(sum[q & 1], pack2(lo, hi));
                    if (SPLIT) split16(lo, hi, out[q], low[SPLIT ? q : 0]);
                    else out[q] = pack16<T>(lo, hi);
                }
                tmem_st16(ts + 16 * k, out);
                if (SPLIT) tmem_st16(ts + 32 + 16 * k, low);
            }
            {
                float lo, hi;
                unpack2(add2(sum[0], sum[1]), lo, hi);
                l += lo + hi;
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[t]);
        }
        // ---------------------------------------------------- o = O / l, lse
        if (it > 0 && ok) {
            ok = mbar_wait(&o_done[t], 0, g.err);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
        }
        float* mine_at = rows_at + (it & 1) * 2 * NT * TILE;
        mine_at[half * TILE] = l;
        asm volatile("bar.sync %0, 256;" ::"r"(1 + t) : "memory");
        l += mine_at[(1 - half) * TILE];
        const bool none = it == 0 || l == 0.f;   // no key seen
        const float inv = none ? 0.f : 1.f / l;
        float post = 1.f;
        if (ok && SPLIT && it > 0) {
            tmem_add<DH>(acc, to, it == 1);
            tmem_wait_st();
            post = pow2(-split_exp(g.tops.v, b * a.hkv + kvh));
        }
        if (NT == 1 && parts > 1) {
            if (ok) {
                float* to_row = reinterpret_cast<float*>(smem) + r * L::OUT_ROW + half * DH;
                for (int k = 0; k < DH / 16; ++k) {
                    uint32_t w[16] = {};
                    if (it > 0) {
                        tmem_ld16(acc + 16 * k, w);
                        tmem_wait_ld();
                    }
                    if (none)
#pragma unroll
                        for (int q = 0; q < 16; ++q) w[q] = 0;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        reinterpret_cast<uint4*>(to_row + 16 * k)[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
                }
                if (half == 0) reinterpret_cast<float2*>(smem + L::STATS)[r] = make_float2(FIX ? 0.f : m, none ? 0.f : l);
            }
        } else if (ok) {
            HeadsView o = a.o;
            o.p = static_cast<U*>(o.p) + half * DH * o.sd;
            store_row<U, DH>(o, b, h, i, on, a.d - half * DH, acc, !none, it > 0, inv, post);
            if (a.lse && on && half == 0)
                a.lse[((int64_t)b * a.hq + h) * a.nq + i] = none ? -INFINITY : (FIX ? 0.f : m - Lift<T>::log2) * kLn2 + logf(l);
        }
        end_of_walk();
        if (NT == 1 && parts > 1) {
            // TMEM is given back: no block holds any while it waits for its cluster
            cluster_sync();
            if (ok) join_parts<T, U, L, FIX>(smem, g, part, b, h0, kvh, i0);
            __syncwarp();
            cluster_sync();   // its rows are read
        }
    }
}

template <typename T, typename U, int DP, int NT, bool CAP, bool BIAS, bool FIX = false>
tl_status launch(tl_ctx* c, const HeadMap* m, const FwArgs& g, cudaStream_t s) {
    using L = Fw<T, U, DP, NT>;
    static std::atomic<uint64_t> done{0};
    TL_TRY(kernel_smem(c, k_attn_tc<T, U, DP, NT, CAP, BIAS, FIX>, L::BYTES, done, L::REGS));
    const AttnCall& a = g.a;
    const int span = g.pack ? g.pack : g.pair_heads ? TILE : NT * TILE;
    const int64_t grid = (int64_t)a.b * (g.pack ? a.hkv : g.pair_heads ? a.hq / 2 : a.hq) * ((a.nq + span - 1) / span) * g.parts;
    cudaEvent_t ev[2];
    launch_begin_on(c, s, "attention_tc", 0, 4.0 * a.d * attn_pairs(a), ev);
    // early behind a kernel of this call
    TL_CK(c, launch_with(k_attn_tc<T, U, DP, NT, CAP, BIAS, FIX>, dim3((unsigned)grid), g.parts, L::THREADS, L::BYTES,
                         L::SPLIT || a.k_doc != nullptr, s, m[0], m[1], m[2], g));
    return launch_end_on(c, s, ev);
}

template <typename T, typename U, int DP, int NT>
tl_status launch_scores(tl_ctx* c, const HeadMap* m, const FwArgs& g, cudaStream_t s) {
    const bool bias = takes_slopes(g.a);
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        if (g.a.cap > 0.f && !bias && g.a.cap * kLog2e <= kFixTop) return launch<T, U, DP, NT, true, false, true>(c, m, g, s);
    if (g.a.cap > 0.f) return bias ? launch<T, U, DP, NT, true, true>(c, m, g, s) : launch<T, U, DP, NT, true, false>(c, m, g, s);
    return bias ? launch<T, U, DP, NT, false, true>(c, m, g, s) : launch<T, U, DP, NT, false, false>(c, m, g, s);
}

template <typename T, typename U, int DP>
tl_status launch_tiles(tl_ctx* c, const HeadMap* m, FwArgs g, cudaStream_t s) {
    using L = Fw<T, U, DP, 1>;
    const AttnCall& a = g.a;
    // Two tiles a block read each key tile once for both and keep the tensor
    // cores busier; one leaves two blocks an SM, which even out walks of
    // different lengths.  bf16, d 128, one tile / two, us: 128 tiles of 2048
    // keys 36 / 40; causal, 288 tiles 39 / 42, 512 tiles of 512 keys 29 / 30,
    // of 1024 36 / 38, of 2048 50 / 50; not causal, 192 tiles 46 / 41, 512
    // tiles 85 / 79.  fp32, d 64: causal, 288 tiles 86 / 83, 512 112 / 107; 128 tiles 79 /
    // 73, but 58 with keys shared by two blocks.  Documents (when two tiles had them): 512
    // causal tiles of 4096 keys in 16 28 / 31, in 4 44 / 46, in one 95 / 81; their
    // lengths are not known here: many.
    const int64_t tiles = g.pack ? (int64_t)a.b * a.hkv * ((a.nq + g.pack - 1) / g.pack) : (int64_t)a.b * a.hq * ((a.nq + TILE - 1) / TILE);
    const bool one = g.pack || tiles <= c->sm_count || (a.causal && !L::SPLIT && (tiles <= 2 * c->sm_count || a.nk <= 1024)) || (a.q_doc && a.k_doc);
    g.pair_heads = 0;
    g.parts = 1;
    if constexpr (DP <= 128)
        if (!one) {
            g.pair_heads = a.hq / a.hkv % 2 == 0;
            return launch_scores<T, U, DP, 2>(c, m, g, s);
        }
    // Blocks that would leave the GPU half empty share the keys of a tile among
    // up to eight, a cluster, which add their rows in shared memory (2 to 4 us).
    // One block a tile / shared, us: bf16, d 128, 16 tiles of 32768 keys 507 / 78 (two 267,
    // four 139), of 2048 35 / 17; 128 tiles of 2048 36 / 33; 32 tiles of 512 keys, four 16 / 15,
    // two 17, of 256, two 13 / 15; fp32, d 64, of 512 28 / 25, 64 tiles of 1024 41 / 31.  A tile of
    // packed documents meets few of the keys: 64 tiles of 2048 keys in four 17 / 19.
    // Where a block fills an SM (fp32, d 128, 16 tiles of 2048 keys) 80, 57, 42, 48 by 1, 2, 4, 8:
    // few clusters of eight find their SMs.
    const int least = a.q_doc ? 32 : L::SPLIT ? 4 : 8;   // key tiles
    while (g.key_tiles >= least && g.parts < (L::PER_SM == 1 ? 4 : 8) && tiles * g.parts * 2 <= c->sm_count * L::PER_SM &&
           g.parts * 2 <= g.key_tiles)
        g.parts *= 2;
    return launch_scores<T, U, DP, 1>(c, m, g, s);
}

}  // namespace

bool tc_array(const HeadsView& v, int b, int h, int64_t n) {
    auto fits = [](int64_t count, int64_t stride) { return count <= 1 || (stride % 8 == 0 && stride < (int64_t(1) << 38)); };
    return v.sd == 1 && reinterpret_cast<uintptr_t>(v.p) % 16 == 0 && fits(n, v.ss) && v.ss != 0 && fits(h, v.sh) && fits(b, v.sb);
}

bool attn_tc_takes(const AttnCall& a) {
    // a scale that keeps the order of the scores (the row maximum is taken
    // before scaling)
    if (a.nk == 0 || !(a.scale > 0.f) || a.cuda_cores) return false;
    if (a.dtype == TL_TYPE_F32) return a.d <= kSplitMaxHead;   // its operands are copies, the arrays may lie anyhow
    return a.d % 8 == 0 && a.d <= 128 && tc_array(a.q, a.b, a.hq, a.nq) && tc_array(a.k, a.b, a.hkv, a.nk) &&
           tc_array(a.v, a.b, a.hkv, a.nk) && tc_array(a.o, a.b, a.hq, a.nq);
}

bool make_head_map(HeadMap* m, const HeadsView& v, int dtype, int b, int h, int64_t n, int d, int box_rows, int box_heads) {
    typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode enc = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool got = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                         q == cudaDriverEntryPointSuccess;
        return reinterpret_cast<Encode>(got ? p : nullptr);
    }();
    if (!enc) return false;
    // a dim of 1, or one whose stride is 0, is mapped as one element
    m->mh = h > 1 && v.sh != 0;
    m->mb = b > 1 && v.sb != 0;
    cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)n, m->mh ? (cuuint64_t)h : 1, m->mb ? (cuuint64_t)b : 1};
    const int64_t row = n > 1 ? v.ss : (d + 7) / 8 * 8;
    cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)(m->mh ? v.sh : row) * 2, (cuuint64_t)(m->mb ? v.sb : row) * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_heads, 1}, one[4] = {1, 1, 1, 1};
    return enc(&m->map, dtype == TL_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, v.p, dims,
               strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// documents: the ranges of the key tiles; fp32: the split operands
static size_t ranges_bytes(const AttnCall& a) {
    return a.k_doc ? ((size_t)a.b * ((a.nk + TILE - 1) / TILE) * sizeof(DocRange) + 255) / 256 * 256 : 0;
}
size_t attn_tc_workspace(const AttnCall& a) {
    return ranges_bytes(a) + (a.dtype == TL_TYPE_F32 ? SplitPlan(a, false).bytes : 0);
}

tl_status launch_attn_begin(tl_ctx* c, const AttnCall& a, DocRange* q_out, DocRange* k_out, uint32_t* zero, int64_t words,
                            cudaStream_t s) {
    BeginArgs g = {a.q_doc, a.k_doc, a.nq, a.nk, 0, 0, q_out, k_out, zero, words};
    if (a.q_doc && q_out) g.q_total = (int64_t)a.b * ((a.nq + TILE - 1) / TILE);
    if (a.k_doc && k_out) g.k_total = (int64_t)a.b * ((a.nk + TILE - 1) / TILE);
    const int64_t total = g.q_total + g.k_total, zeros = std::min<int64_t>((words + 255) / 256, 64);
    if (!total && !words) return TL_OK;
    cudaEvent_t ev[2];
    launch_begin_on(c, s, "attention_begin", 4.0 * total * TILE, 0, ev);
    k_attn_begin<<<(unsigned)std::max((total + 7) / 8, zeros), 256, 0, s>>>(g);
    return launch_end_on(c, s, ev);
}

// Queries of a tile that holds them for all heads of a group, where that makes
// fewer tiles (0: it does not): 16 x 64 heads over 8, 8 queries over 4096 keys of
// bf16, d 128, 260 us by head, 61 packed.
static int packed_queries(const AttnCall& a) {
    const int group = a.hq / a.hkv;
    if (group < 2 || group > TILE || (a.dtype != TL_TYPE_F32 && a.q.sh == 0)) return 0;
    const int n = std::min(a.nq, TILE / group);
    return (a.nq + n - 1) / n < (int64_t)group * ((a.nq + TILE - 1) / TILE) ? n : 0;
}

tl_status launch_attn_tc(tl_ctx* c, const AttnCall& a, void* ws, cudaStream_t s) {
    FwArgs g;
    g.a = a;
    g.k_ranges = static_cast<DocRange*>(ws);
    g.key_tiles = (a.nk + TILE - 1) / TILE;
    g.err = c->d_flags + 8;
    c->flags_armed = true;
    HeadMap m[4];
    g.pack = packed_queries(a);
    const int group = a.hq / a.hkv, q_rows = g.pack ? g.pack : TILE, q_heads = g.pack ? group : 1;
    if (a.dtype == TL_TYPE_F32) {
        uint8_t* w = static_cast<uint8_t*>(ws) + ranges_bytes(a);
        TL_TRY(launch_split(c, a, nullptr, w, m, nullptr, static_cast<DocRange*>(ws), s));
        g.tops.q = reinterpret_cast<const uint32_t*>(w + SplitPlan(a, false).top);
        g.tops.k = g.tops.q + (size_t)a.b * a.hkv;
        g.tops.v = g.tops.k + (size_t)a.b * a.hkv;
        g.tops.dout = nullptr;
        const int64_t width = split_width(a.d);
        const HeadsView q = {w + SplitPlan(a, false).data[0], a.hq * a.nq * width, a.nq * width, width, 1};
        if (g.pack && !make_head_map(&m[0], q, TL_TYPE_F16, a.b, a.hq, a.nq, (int)width, q_rows, q_heads))
            return fail(c, TL_ERR_CUDA, "attention: tensor maps");
        return a.d > 64 ? launch_tiles<__half, float, 256>(c, m, g, s) : launch_tiles<__half, float, 128>(c, m, g, s);
    }
    TL_TRY(launch_attn_begin(c, a, nullptr, static_cast<DocRange*>(ws), nullptr, 0, s));
    g.tops = {nullptr, nullptr, nullptr, nullptr};
    if (!make_head_map(&m[0], a.q, a.dtype, a.b, a.hq, a.nq, a.d, q_rows, q_heads) || !make_head_map(&m[1], a.k, a.dtype, a.b, a.hkv, a.nk, a.d) ||
        !make_head_map(&m[2], a.v, a.dtype, a.b, a.hkv, a.nk, a.d))
        return fail(c, TL_ERR_CUDA, "attention: tensor maps");
    if (a.dtype == TL_TYPE_F16)
        return a.d <= 64 ? launch_tiles<__half, __half, 64>(c, m, g, s) : launch_tiles<__half, __half, 128>(c, m, g, s);
    return a.d <= 64 ? launch_tiles<__nv_bfloat16, __nv_bfloat16, 64>(c, m, g, s)
                     : launch_tiles<__nv_bfloat16, __nv_bfloat16, 128>(c, m, g, s);
}

}  // namespace tl
