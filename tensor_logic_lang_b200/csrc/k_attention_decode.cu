// Attention of few queries over many keys (a token or a few of each sequence
// over its cache): bound by reading the cache once.
//
// The queries of a group's heads that read one key head are the rows of a
// unit (16 of them, or 4 on the CUDA cores; more rows make more units).  A unit's keys are cut
// into tiles (of 64, or 128 of head sizes up to 64), the tiles of all units form one line, and each block takes
// an equal piece of it, whatever the sequences' lengths: all blocks run at
// once and end together.  A piece that covers a unit whole writes its output;
// the pieces of a unit that lies over several blocks leave their sums,
// maxima and unnormalised outputs in the workspace (at most two a block), and
// k_decode_join adds them in the order of the keys.  Where a call has few units
// and short caches, a cluster of 8 blocks shares each unit instead and joins its
// pieces through distributed shared memory: one launch, no line to divide.
//
//   k_decode_mma   16-bit types with aligned rows and head sizes up to 128: TMA
//                  tiles (128-byte swizzle) through a ring; each of four
//                  warps takes a quarter of a tile's keys for all rows, with
//                  mma.sync.m16n8k16 (at a few rows a key the tensor work is a
//                  fraction of the time the key's bytes take)
//                  16 x 32 heads over 8, caches up to 32768, d 128: 186 us, 6.5 TB/s; 5
//                  sequences x 3 tokens of 16 heads, 4099, d 64: 20 us with the join, 2.4
//                  TB/s: starts and ends of pieces of a few tiles
//   k_decode_any   any type, stride and head size: tiles as fp32 in shared
//                  memory, FFMA; fp32, 16 x 32 heads over 8, 4096, d 128: 85 us, 3.6 TB/s of 6.5, its
//                  five barriers a tile leave the loads uneven
#include <algorithm>

#include "attn_tc.h"

namespace tl {
namespace {

constexpr int JOIN_THREADS = 128;
constexpr int kSms = 148;

struct DecArgs {
    AttnCall a;
    int tile;          // keys of a tile
    int cluster;       // blocks that share a unit, or 1: the blocks share the line
    int rows;          // of a unit
    int row_blocks;    // units of a key head
    int blocks;        // of the kernel that reads the cache
    const int2* spans; // [b] with documents: the first and one past the last key that may be seen
    float* part;       // [blocks][2][rows][d + 2]: o, m, l of a piece
    int* err;
};

// Documents' spans come out of the workspace.  Where a caller lets other work write there
// meanwhile, results are lost, but what is made of the spans stays within the
// arrays: here, in find_place and in the join.
__device__ __forceinline__ int2 seq_tiles(const DecArgs& g, int b) {
    const SeqMask mask(g.a, b);
    int end = max(mask.key_end(0, g.a.nq), 0), begin = 0;
    if (g.spans) {
        const int2 s = g.spans[b];
        begin = min(max(s.x, 0), end);
        end = min(s.y, end);
    }
    if (end <= begin) return make_int2(0, 0);
    return make_int2(begin / g.tile, (end + g.tile - 1) / g.tile);
}

// Sum over the block; every thread gets it.  NW warps, red[NW] words.
template <int NW>
__device__ __forceinline__ int64_t block_total(int64_t v, int64_t* red) {
#pragma unroll
    for (int w = 16; w; w >>= 1) v += __shfl_xor_sync(0xffffffffu, v, w);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    int64_t s = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) s += red[w];
    return s;
}

// Tiles of all sequences, and of those before `upto`.
template <int NW>
__device__ __forceinline__ int64_t tiles_before(const DecArgs& g, int upto, int64_t* all, int64_t* red) {
    int64_t t = 0, p = 0;
    for (int b = threadIdx.x; b < g.a.b; b += NW * 32) {
        const int2 s = seq_tiles(g, b);
        t += s.y - s.x;
        if (b < upto) p += s.y - s.x;
    }
    // two sums in one reduction: a sequence has less than 2^24 tiles of 64 keys
    // and a call at most 2^29 sequences, so the halves are taken apart only
    // where both fit (else one after the other)
    if (g.a.b <= 256) {
        const int64_t both = block_total<NW>(t << 32 | p, red);
        *all = both >> 32;
        return both & 0xffffffff;
    }
    *all = block_total<NW>(t, red);
    return block_total<NW>(p, red);
}

// The line of tiles, from a place on: sequence, unit within it, tile of it.
struct Place {
    int b, unit;       // unit of the sequence: key head * row_blocks + row block
    int2 span;         // its tiles
    int64_t tile;      // next tile (span.x ..)
};

// The place where a block's share of the line starts, and its length (0: it
// has none).  The shares are equal, in the order of the blocks.
template <int NW>
__device__ __forceinline__ Place find_place(const DecArgs& g, int64_t* left, int64_t* red, int64_t* found) {
    const int units = g.a.hkv * g.row_blocks, lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const bool once = g.a.b <= NW * 32;   // one sequence a thread: the sum of all comes with the scan
    int64_t all = 0, before = 0, at = 0;
    if (!once) {
        int64_t t = 0;
        for (int b = threadIdx.x; b < g.a.b; b += NW * 32) {
            const int2 s = seq_tiles(g, b);
            t += s.y - s.x;
        }
        all = block_total<NW>(t, red) * units;
    }
    Place p;
    p.b = 0; p.unit = 0; p.span = make_int2(0, 0); p.tile = 0;
    *left = 0;
    for (int b0 = 0; b0 < g.a.b; b0 += NW * 32) {
        const int b = b0 + threadIdx.x;
        int64_t n = 0;
        if (b < g.a.b) {
            const int2 s = seq_tiles(g, b);
            n = (int64_t)(s.y - s.x) * units;
        }
        int64_t sum = n;   // inclusive over the warp
#pragma unroll
        for (int w = 1; w < 32; w <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, sum, w);
            if (lane >= w) sum += o;
        }
        __syncthreads();
        if (lane == 31) red[warp] = sum;
        if (threadIdx.x == 0) found[0] = -1;
        __syncthreads();
        int64_t base = before, total = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < warp) base += red[w];
            total += red[w];
        }
        if (once) all = total;
        if (b0 == 0) {
            const int64_t per = (all + g.blocks - 1) / g.blocks;
            at = per * blockIdx.x;
            *left = min(per, all - at);
            if (*left <= 0) return p;
        }
        const int64_t lo = base + sum - n, hi = base + sum;
        if (lo <= at && at < hi) { found[0] = b; found[1] = lo; }
        __syncthreads();
        if (found[0] >= 0) break;
        before += total;
    }
    if (found[0] < 0) {
        *left = 0;
        return p;
    }
    p.b = (int)found[0];
    p.span = seq_tiles(g, p.b);
    const int n = max(p.span.y - p.span.x, 1);
    const int64_t in = at - found[1];
    p.unit = (int)min(in / n, (int64_t)units - 1);
    p.tile = p.span.x + in % n;
    return p;
}

// One piece: the tiles [t0, t1) of a unit, and where its sums go.
struct Piece {
    int b, kvh, rb, t0, t1;
    bool whole;       // all of the unit's tiles
    int slot;
};

// The pieces of a block, in order; every thread (and warp role) walks the same ones.
struct PieceWalk {
    Place at;
    int64_t left;      // tiles left for this block
    bool first;
    __device__ __forceinline__ bool next(const DecArgs& g, Piece* p) {
        if (g.cluster > 1) {   // the block's share of its cluster's unit, which may be empty
            if (!first) return false;
            first = false;
            const int unit = blockIdx.x / g.cluster, rank = blockIdx.x % g.cluster, n = at.span.y - at.span.x;
            p->b = at.b;
            p->kvh = unit / g.row_blocks % g.a.hkv;
            p->rb = unit % g.row_blocks;
            p->t0 = at.span.x + n * rank / g.cluster;
            p->t1 = at.span.x + n * (rank + 1) / g.cluster;
            p->whole = false;
            p->slot = 0;
            return true;
        }
        if (left <= 0) return false;
        const int units = g.a.hkv * g.row_blocks;
        while (at.tile >= at.span.y || at.span.x >= at.span.y) {   // the next unit with tiles
            if (at.span.x < at.span.y && at.unit + 1 < units) {
                ++at.unit;
            } else {
                if (at.b + 1 >= g.a.b) return false;
                ++at.b;
                at.unit = 0;
                at.span = seq_tiles(g, at.b);
            }
            at.tile = at.span.x;
        }
        p->b = at.b;
        p->kvh = at.unit / g.row_blocks;
        p->rb = at.unit % g.row_blocks;
        p->t0 = (int)at.tile;
        p->t1 = (int)min((int64_t)at.span.y, at.tile + left);
        p->whole = p->t0 == at.span.x && p->t1 == at.span.y;
        p->slot = first ? 0 : 1;
        first = false;
        left -= p->t1 - p->t0;
        at.tile = p->t1;
        return true;
    }
};

template <int NW>
__device__ __forceinline__ PieceWalk block_pieces(const DecArgs& g, int64_t* red, int64_t* found) {
    PieceWalk w;
    w.first = true;
    if (g.cluster > 1) {
        w.at.b = blockIdx.x / g.cluster / (g.a.hkv * g.row_blocks);
        w.at.span = seq_tiles(g, w.at.b);
    } else {
        w.at = find_place<NW>(g, &w.left, red, found);
    }
    return w;
}

// Row r of a unit: query i of head h.
__device__ __forceinline__ void unit_row(const AttnCall& a, int kvh, int row, int* i, int* h) {
    const int group = a.hq / a.hkv;
    *i = row / group;
    *h = kvh * group + row % group;
}

// What a row needs to score and mask keys.
struct DecRow {
    int p, limit, doc;
    float slope2;
    bool on;
    __device__ __forceinline__ void set(const AttnCall& a, const SeqMask& mask, int b, int kvh, int row) {
        on = row < a.nq * (a.hq / a.hkv);
        int i, h;
        unit_row(a, kvh, on ? row : 0, &i, &h);
        p = mask.p0 + i;
        limit = on ? mask.key_end(i, 1) : 0;
        doc = a.q_doc ? a.q_doc[(int64_t)b * a.nq + i] : -1;
        slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    }
};

// The end of a piece: `warps` sums of o (rows x ld fp32 each), m, l in shared
// memory -> the output, or the block's part (in a cluster: `shared`).
template <typename T>
__device__ __forceinline__ void finish_piece(const DecArgs& g, const Piece& pc, const float* o, int warps, int wstride, int ld,
                                             const float* m, const float* l, int row0, int rows, int thread, int threads, float* shared) {
    const AttnCall& a = g.a;
    const int d2 = a.d + 2, used = min(rows, a.nq * (a.hq / a.hkv) - pc.rb * g.rows - row0);
    for (int e = thread; e < used * a.d; e += threads) {
        const int r = e / a.d, c = e % a.d;
        const int row = pc.rb * g.rows + row0 + r;
        float top = -INFINITY;
        for (int w = 0; w < warps; ++w) top = fmaxf(top, m[w * rows + r]);
        float sum = 0.f, out = 0.f;
        for (int w = 0; w < warps; ++w) {
            const float by = m[w * rows + r] == -INFINITY && top == -INFINITY ? 0.f : ex2(m[w * rows + r] - top);
            sum = fmaf(by, l[w * rows + r], sum);
            out = fmaf(by, o[(size_t)w * wstride + r * ld + c], out);
        }
        if (pc.whole) {
            int i, h;
            unit_row(a, pc.kvh, row, &i, &h);
            const bool none = sum == 0.f;
            static_cast<T*>(a.o.p)[pc.b * a.o.sb + h * a.o.sh + i * a.o.ss + c * a.o.sd] = from_f32<T>(none ? 0.f : out / sum);
            if (a.lse && c == 0)
                a.lse[((int64_t)pc.b * a.hq + h) * a.nq + i] = none ? -INFINITY : top * kLn2 + logf(sum);
        } else {
            float* part = (g.cluster > 1 ? shared : g.part + (size_t)(blockIdx.x * 2 + pc.slot) * g.rows * d2) + (row0 + r) * d2;
            part[c] = out;
            if (c == 0) { part[a.d] = top; part[a.d + 1] = sum; }
        }
    }
}

// The pieces of a cluster's unit, each in its block's `shared`, joined in the
// order of the keys: the blocks take rows x columns in turn.
template <typename T>
__device__ __forceinline__ void join_cluster(const DecArgs& g, const Piece& pc, const float* shared, int threads) {
    const AttnCall& a = g.a;
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int rank = blockIdx.x % g.cluster, d2 = a.d + 2;
    const int used = min(g.rows, a.nq * (a.hq / a.hkv) - pc.rb * g.rows);
    for (int e = rank * threads + threadIdx.x; threadIdx.x < threads && e < used * a.d; e += threads * g.cluster) {
        const int r = e / a.d, c = e % a.d;
        float o[8], m[8], l[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            uint32_t at;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(shared + r * d2)), "r"(min(q, g.cluster - 1)));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o[q]) : "r"(at + 4 * c));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(m[q]) : "r"(at + 4 * a.d));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(l[q]) : "r"(at + 4 * a.d + 4));
        }
        float top = -INFINITY, sum = 0.f, out = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (q < g.cluster) top = fmaxf(top, m[q]);
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (q < g.cluster) {
                const float by = top == -INFINITY ? 0.f : ex2(m[q] - top);
                sum = fmaf(by, l[q], sum);
                out = fmaf(by, o[q], out);
            }
        int i, h;
        unit_row(a, pc.kvh, pc.rb * g.rows + r, &i, &h);
        const bool none = sum == 0.f;
        static_cast<T*>(a.o.p)[pc.b * a.o.sb + h * a.o.sh + i * a.o.ss + c * a.o.sd] = from_f32<T>(none ? 0.f : out / sum);
        if (a.lse && c == 0) a.lse[((int64_t)pc.b * a.hq + h) * a.nq + i] = none ? -INFINITY : top * kLn2 + logf(sum);
    }
    __syncwarp();
    // a block's part stays until the others have read it
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A block a row: rows of units that lie over several blocks, and of sequences
// without keys.
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) k_decode_join(const __grid_constant__ DecArgs g) {
    __shared__ int64_t red[JOIN_THREADS / 32];
    __shared__ float weight[2 * kSms], sums[2 * kSms], tops[JOIN_THREADS / 32];   // of at most every block
    const AttnCall& a = g.a;
    const int rows = a.nq * (a.hq / a.hkv), units = a.hkv * g.row_blocks;
    const int row = blockIdx.x % rows, kvh = blockIdx.x / rows % a.hkv, b = blockIdx.x / rows / a.hkv;
    const int unit = kvh * g.row_blocks + row / g.rows, r = row % g.rows;
    int64_t all;   // from the lengths, which were there before the kernel that reads the cache
    const int64_t before = tiles_before<JOIN_THREADS / 32>(g, b, &all, red) * units;
    all *= units;
    const int2 span = seq_tiles(g, b);
    const int n = span.y - span.x, d2 = a.d + 2;
    const int64_t per = max((int64_t)1, (all + g.blocks - 1) / g.blocks);
    const int64_t u0 = before + (int64_t)unit * n, u1 = u0 + n;
    const int first = (int)min(u0 / per, (int64_t)g.blocks - 1), last = n ? (int)min((u1 - 1) / per, (int64_t)g.blocks - 1) : first;
    // before any return: where no row is split over blocks, what follows this
    // kernel would else start before the outputs are written
    wait_for_previous();
    if (n && first == last) return;   // one block wrote it
    int i, h;
    unit_row(a, kvh, row, &i, &h);
    // a block's second piece is the one that starts inside it
    auto part = [&](int q) { return g.part + ((size_t)(q * 2 + ((int64_t)q * per < u0 ? 1 : 0)) * g.rows + r) * d2; };
    // the parts' maxima and sums, a thread a part; weights for the columns
    const int parts = n ? last - first + 1 : 0;
    float top = -INFINITY;
    for (int q = threadIdx.x; q < parts; q += JOIN_THREADS) {
        const float* p = part(first + q);
        weight[q] = p[a.d];
        sums[q] = p[a.d + 1];
        top = fmaxf(top, weight[q]);
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JOIN_THREADS / 32; ++w) top = fmaxf(top, tops[w]);
    for (int q = threadIdx.x; q < parts; q += JOIN_THREADS) weight[q] = top == -INFINITY ? 0.f : ex2(weight[q] - top);
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += JOIN_THREADS) {
        float sum = 0.f, out = 0.f;
#pragma unroll 8
        for (int q = 0; q < parts; ++q) {
            sum = fmaf(weight[q], sums[q], sum);
            out = fmaf(weight[q], part(first + q)[c], out);
        }
        const bool none = sum == 0.f;
        static_cast<T*>(a.o.p)[b * a.o.sb + h * a.o.sh + i * a.o.ss + c * a.o.sd] = from_f32<T>(none ? 0.f : out / sum);
        if (a.lse && c == 0) a.lse[((int64_t)b * a.hq + h) * a.nq + i] = none ? -INFINITY : top * kLn2 + logf(sum);
    }
}

// First and one past the last key whose document is one of a sequence's
// queries' (a document that lies in one piece is all of that).
__global__ void __launch_bounds__(256) k_doc_spans(const __grid_constant__ AttnCall a, int2* __restrict__ spans) {
    __shared__ int lo, hi, dlo, dhi;
    const int b = blockIdx.x;
    if (threadIdx.x == 0) { lo = 0x7fffffff; hi = 0; dlo = 0x7fffffff; dhi = -1; }
    __syncthreads();
    for (int i = threadIdx.x; i < a.nq; i += 256) {
        const int d = a.q_doc[(int64_t)b * a.nq + i];
        if (d >= 0) { atomicMin(&dlo, d); atomicMax(&dhi, d); }
    }
    __syncthreads();
    int first = 0x7fffffff, last = 0;
    const int32_t* kd = a.k_doc + (int64_t)b * a.nk;
#pragma unroll 8
    for (int j = threadIdx.x; j < a.nk; j += 256) {
        const int d = __ldg(kd + j);
        if (d >= dlo && d <= dhi) { first = min(first, j); last = max(last, j + 1); }
    }
    atomicMin(&lo, first);
    atomicMax(&hi, last);
    __syncthreads();
    if (threadIdx.x == 0) spans[b] = make_int2(min(lo, hi), hi);
}

// ---------------------------------------------------------------- tensor cores

template <int DP>
struct DmSmem {
    static constexpr int KW = DP == 64 ? 32 : 16, DT = 4 * KW;   // keys of a warp, of a tile
    static constexpr int WARPS = 4, THREADS = 32 * (WARPS + 1), PER_SM = 2;   // and one of TMA
    static constexpr int CH = DP / 64, CHUNK = DT * 128, TILE_B = CH * CHUNK, STAGES = 2;
    static constexpr int LQ = DP + 8;   // 16-bit query rows, padded by 16 bytes
    static constexpr int KV = 0, Q = STAGES * 2 * TILE_B, MERGE = Q + 16 * LQ * 2, LO = DP + 4,
                         STAT = MERGE + WARPS * 16 * LO * 4, PART = STAT + 2 * WARPS * 16 * 4, BAR = PART + 16 * (DP + 2) * 4, BYTES = BAR + 256 + 1024;
};

__device__ __forceinline__ void ldsm4(uint32_t at, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t at, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if (TypeOf<T>::id == TL_TYPE_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int DP>
__global__ void __launch_bounds__(DmSmem<DP>::THREADS, DmSmem<DP>::PER_SM)
    k_decode_mma(const __grid_constant__ HeadMap mk, const __grid_constant__ HeadMap mv, const __grid_constant__ DecArgs g) {
    using L = DmSmem<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR);
    uint64_t* empty = full + L::STAGES;
    __shared__ int64_t red[L::THREADS / 32], found[2];
    const AttnCall& a = g.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    let_next_start();
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], L::WARPS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    PieceWalk walk = block_pieces<L::THREADS / 32>(g, red, found);
    __syncthreads();
    Piece pc;
    int n = 0;
    bool ok = true;
    if (warp == L::WARPS) {
        while (ok && walk.next(g, &pc))
            for (int t = pc.t0; t < pc.t1 && ok; ++t, ++n) {
                const int s = n % L::STAGES;
                if (n >= L::STAGES) ok = mbar_wait(&empty[s], ((n / L::STAGES) & 1) ^ 1, g.err);
                ok = __all_sync(0xffffffffu, ok);
                if (ok && lane == 0) {
                    mbar_expect_tx(&full[s], 2 * L::TILE_B);
                    for (int w = 0; w < 2; ++w)
                        for (int c = 0; c < L::CH; ++c) {
                            const HeadMap& m = w ? mv : mk;
                            asm volatile(
                                "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, "
                                "%6}], [%2];" ::"r"(smem_u32(smem + L::KV + (2 * s + w) * L::TILE_B + c * L::CHUNK)),
                                "l"(reinterpret_cast<uint64_t>(&m.map)), "r"(smem_u32(&full[s])), "r"(64 * c), "r"(t * L::DT),
                                "r"(pc.kvh * m.mh), "r"(pc.b * m.mb)
                                : "memory");
                        }
                }
                __syncwarp();
            }
        if (!ok)
            for (int e = max(0, n - 1 - L::STAGES); e < n - 1; ++e) mbar_wait(&full[e % L::STAGES], (e / L::STAGES) & 1, g.err);
        if (g.cluster > 1) join_cluster<T>(g, pc, reinterpret_cast<float*>(smem + L::PART), 32 * L::WARPS);
        return;
    }

    const CapCoef<false> cap(a.scale, a.cap > 0.f ? a.cap : 1.f);
    const int gid = lane >> 2, tid = lane & 3, mi = lane >> 3, mr = lane & 7;
    const int ksteps = (a.d + 15) / 16;
    T* qs = reinterpret_cast<T*>(smem + L::Q);
    float* merge = reinterpret_cast<float*>(smem + L::MERGE);
    float *m_s = reinterpret_cast<float*>(smem + L::STAT), *l_s = m_s + L::WARPS * 16;
    while (walk.next(g, &pc)) {
        const SeqMask mask(a, pc.b);
        const int32_t* kd = a.k_doc ? a.k_doc + (int64_t)pc.b * a.nk : nullptr;
        // the unit's query rows (zeros past the last one, past the head size and of padding)
        for (int e = threadIdx.x; e < 16 * DP / 8; e += 32 * L::WARPS) {
            const int r = e / (DP / 8), c = e % (DP / 8) * 8, row = pc.rb * g.rows + r;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row < a.nq * (a.hq / a.hkv) && c < a.d) {
                int i, h;
                unit_row(a, pc.kvh, row, &i, &h);
                if (!a.q_doc || a.q_doc[(int64_t)pc.b * a.nq + i] >= 0)
                    v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q.p) + pc.b * a.q.sb + h * a.q.sh + i * a.q.ss + c);
            }
            *reinterpret_cast<uint4*>(qs + r * L::LQ + c) = v;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * L::WARPS) : "memory");
        DecRow row[2];
        float m[2], l[2], o[DP / 8][4];
        const int left = a.nq * (a.hq / a.hkv) - pc.rb * g.rows;   // rows from the unit's first on
        int all_see = 0x7fffffff;                                  // keys that every row sees
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            row[e].set(a, mask, pc.b, pc.kvh, pc.rb * g.rows + gid + 8 * e);
            if (row[e].on) all_see = min(all_see, row[e].limit);
            m[e] = -INFINITY;
            l[e] = 0.f;
        }
        all_see = __reduce_min_sync(0xffffffffu, all_see);
#pragma unroll
        for (int c = 0; c < DP / 8; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][e] = 0.f;
        for (int t = pc.t0; t < pc.t1 && ok; ++t, ++n) {
            constexpr int KW = L::KW, NK = KW / 8;   // tiles of 8 keys of a warp
            const int st = n % L::STAGES, j0 = t * L::DT + warp * KW;
            ok = mbar_wait(&full[st], (n / L::STAGES) & 1, g.err);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            uint8_t* kt = smem + L::KV + 2 * st * L::TILE_B;
            uint8_t* vt = kt + L::TILE_B;
            // keys that must not count: 0 times what V holds could be NaN, and scores of what K
            // holds would have a say in the tanh's form
            const int jl = j0 + lane % KW;
            const int jdoc = kd && jl < a.nk ? __ldg(kd + jl) : -1;
            const bool bad = jl >= mask.kv || (kd && jdoc < 0);
            const bool dirty = __any_sync(0xffffffffu, bad);
            if (dirty) {
                auto clear = [&](uint8_t* tile) {
                    for (int c = 0; c < L::CH; ++c)
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            *reinterpret_cast<uint4*>(tile + c * L::CHUNK + (warp * KW + lane) * 128 + 16 * k) = make_uint4(0, 0, 0, 0);
                };
                if (bad && lane < KW) {
                    clear(vt);
                    if (a.cap > 0.f) clear(kt);
                }
                __syncwarp();
            }
            // scores of the warp's keys, 8 to a tile
            float s[NK][4];
#pragma unroll
            for (int e = 0; e < 4 * NK; ++e) s[e / 4][e % 4] = 0.f;
            {
                const int key = warp * KW + (mi >> 1) * 8 + mr;
                const uint32_t kb = smem_u32(kt) + key * 128;
                const uint32_t qb = smem_u32(qs) + ((mi & 1) * 8 + mr) * (L::LQ * 2) + (mi >> 1) * 16;
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    if (k >= ksteps) break;
                    const int c16 = 2 * (k % 4) + (mi & 1);
                    uint32_t kf[NK / 2][4];
#pragma unroll
                    for (int x = 0; x < NK / 2; ++x)
                        ldsm4(kb + x * 16 * 128 + (k / 4) * L::CHUNK + ((c16 ^ (key & 7)) << 4), kf[x]);
                    uint32_t qf[4];
                    ldsm4(qb + k * 32, qf);
#pragma unroll
                    for (int x = 0; x < NK / 2; ++x) {
                        mma16816<T>(s[2 * x], qf, kf[x][0], kf[x][1]);
                        mma16816<T>(s[2 * x + 1], qf, kf[x][2], kf[x][3]);
                    }
                }
            }
            uint32_t p[NK / 2][4];
            // scores to probabilities; E: 4, or 2 where rows 8..15 are not there
            auto soft = [&](auto e_count) {
                constexpr int E = decltype(e_count)::value;
                const bool masked = kd || j0 + KW > all_see;
                float top[2] = {-INFINITY, -INFINITY};
                f2 y[NK * E / 2];   // pairs of keys of a row
#pragma unroll
                for (int i = 0; i < NK * E / 2; ++i) y[i] = pack2(s[i % NK][i / NK * 2], s[i % NK][i / NK * 2 + 1]);
                if (a.cap > 0.f) {
                    cap_scores<true>(y, cap);
                } else {
#pragma unroll
                    for (int i = 0; i < NK * E / 2; ++i) y[i] = mul2(y[i], pack2(cap.mul, cap.mul));
                }
#pragma unroll
                for (int i = 0; i < NK * E / 2; ++i) {
                    const int x = i % NK, e = i / NK * 2;
                    const DecRow& w = row[e >> 1];
                    const float at = (float)(w.p - j0 - 8 * x - 2 * tid);
                    float lo, hi;
                    unpack2(y[i], lo, hi);
                    s[x][e] = fmaf(-w.slope2, fabsf(at), lo);
                    s[x][e + 1] = fmaf(-w.slope2, fabsf(at - 1.f), hi);
                }
                if (masked) {
#pragma unroll
                    for (int x = 0; x < NK; ++x)
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const DecRow& w = row[e >> 1];
                            const int col = 8 * x + 2 * tid + (e & 1);
                            const int cdoc = kd ? __shfl_sync(0xffffffffu, jdoc, col) : -1;
                            if (!(j0 + col < w.limit && (!kd || (w.doc >= 0 && cdoc == w.doc)))) s[x][e] = -INFINITY;
                        }
                }
#pragma unroll
                for (int x = 0; x < NK; ++x)
#pragma unroll
                    for (int e = 0; e < E; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[x][e]);
#pragma unroll
                for (int e = 0; e < E / 2; ++e) {
                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
                }
                // the reference maximum moves for a row's first key and by steps of 2^8
                bool move = false;
#pragma unroll
                for (int e = 0; e < E / 2; ++e) move |= top[e] > m[e] + 8.f || (m[e] == -INFINITY && top[e] > m[e]);
                if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                    for (int e = 0; e < E / 2; ++e) {
                        const float nm = fmaxf(m[e], top[e]);
                        const float by = nm == -INFINITY ? 1.f : ex2(m[e] - nm);
                        m[e] = nm;
                        l[e] *= by;
#pragma unroll
                        for (int c = 0; c < DP / 8; ++c) {
                            o[c][2 * e] *= by;
                            o[c][2 * e + 1] *= by;
                        }
                    }
                }
                float ref[2];
#pragma unroll
                for (int e = 0; e < E / 2; ++e) ref[e] = (m[e] == -INFINITY ? 0.f : m[e]) - Lift<T>::log2;
#pragma unroll
                for (int x = 0; x < NK; ++x) {
                    float pr[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        pr[e] = ex2(s[x][e] - ref[e >> 1]);
                        l[e >> 1] += pr[e];
                    }
                    p[x / 2][2 * (x % 2)] = pack16<T>(pr[0], pr[1]);
                    p[x / 2][2 * (x % 2) + 1] = E == 4 ? pack16<T>(pr[2], pr[3]) : 0u;
                }
            };
            if (left > 8) soft(std::integral_constant<int, 4>());
            else soft(std::integral_constant<int, 2>());
            {
                const int key = warp * KW + (mi & 1) * 8 + mr;
                const uint32_t vb = smem_u32(vt) + key * 128;
#pragma unroll
                for (int c = 0; c < DP / 8; c += 2) {
                    if (8 * c >= a.d) break;
                    const int c16 = c % 8 + (mi >> 1);
#pragma unroll
                    for (int x = 0; x < NK / 2; ++x) {
                        uint32_t vf[4];
                        ldsm4t(vb + x * 16 * 128 + (c / 8) * L::CHUNK + ((c16 ^ (key & 7)) << 4), vf);
                        mma16816<T>(o[c], p[x], vf[0], vf[1]);
                        mma16816<T>(o[c + 1], p[x], vf[2], vf[3]);
                    }
                }
            }
            if (dirty) fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
        // the warps' sums
        float* mw = merge + warp * 16 * L::LO;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
            if (tid == 0) {
                m_s[warp * 16 + gid + 8 * e] = m[e] == -INFINITY ? -INFINITY : m[e] - Lift<T>::log2;
                l_s[warp * 16 + gid + 8 * e] = l[e];
            }
        }
#pragma unroll
        for (int c = 0; c < DP / 8; ++c) {
            *reinterpret_cast<float2*>(mw + gid * L::LO + 8 * c + 2 * tid) = make_float2(o[c][0], o[c][1]);
            *reinterpret_cast<float2*>(mw + (gid + 8) * L::LO + 8 * c + 2 * tid) = make_float2(o[c][2], o[c][3]);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * L::WARPS) : "memory");
        if (ok) finish_piece<T>(g, pc, merge, L::WARPS, 16 * L::LO, L::LO, m_s, l_s, 0, 16, threadIdx.x, 32 * L::WARPS,
                                reinterpret_cast<float*>(smem + L::PART));
        asm volatile("bar.sync 1, %0;" ::"n"(32 * L::WARPS) : "memory");
    }
    if (g.cluster > 1) join_cluster<T>(g, pc, reinterpret_cast<float*>(smem + L::PART), 32 * L::WARPS);
}

// ---------------------------------------------------------------- any type
constexpr int DA_THREADS = 256, DA_T = 64;   // threads, keys of a tile

template <int DP, int RB>
struct DaSmem {
    static constexpr int LD = DP + 16;   // rows half of the banks apart
    static constexpr int K = 0, V = K + DA_T * LD * 4, Q = V + DA_T * LD * 4, P = Q + RB * DP * 4, STAT = P + DA_T * RB * 4,
                         BYTES = STAT + 3 * RB * 4;
    static_assert(8 * RB * DP <= 2 * DA_T * LD, "the warps' sums lie over the tiles");
};

// Scores: four threads a key, each a quarter of its columns for all rows.
// Sums: warp w takes keys w, w + 8, ... of the tile, a lane 4 columns of every
// 128, for all rows.
template <typename T, int DP, int RB, bool VEC>
__global__ void __launch_bounds__(DA_THREADS) k_decode_any(const __grid_constant__ DecArgs g) {
    using L = DaSmem<DP, RB>;
    extern __shared__ __align__(16) uint8_t smem[];
    float *K = reinterpret_cast<float*>(smem + L::K), *V_ = reinterpret_cast<float*>(smem + L::V);
    float *Q = reinterpret_cast<float*>(smem + L::Q), *P = reinterpret_cast<float*>(smem + L::P);
    float *m_s = reinterpret_cast<float*>(smem + L::STAT), *l_s = m_s + RB, *by_s = l_s + RB;
    __shared__ int64_t red[DA_THREADS / 32], found[2];
    const AttnCall& a = g.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    let_next_start();
    PieceWalk walk = block_pieces<DA_THREADS / 32>(g, red, found);
    const int group = a.hq / a.hkv;
    constexpr int NC = DP >= 128 ? DP / 128 : 1, LANES = DP >= 128 ? 32 : DP / 4;
    Piece pc;
    while (walk.next(g, &pc)) {
        const SeqMask mask(a, pc.b);
        const int32_t* kd = a.k_doc ? a.k_doc + (int64_t)pc.b * a.nk : nullptr;
        __syncthreads();
        for (int e = threadIdx.x; e < RB * DP; e += DA_THREADS) {
            const int r = e / DP, c = e % DP, row = pc.rb * g.rows + r;
            float v = 0.f;
            if (row < a.nq * group && c < a.d) {
                int i, h;
                unit_row(a, pc.kvh, row, &i, &h);
                v = to_f32(static_cast<const T*>(a.q.p)[pc.b * a.q.sb + h * a.q.sh + i * a.q.ss + c * a.q.sd]);
            }
            Q[r * DP + c] = v;
        }
        if (threadIdx.x < RB) { m_s[threadIdx.x] = -INFINITY; l_s[threadIdx.x] = 0.f; }
        DecRow rows[RB / 4];   // of the scores this thread writes: rows threadIdx.x % 4, + 4, ...
#pragma unroll
        for (int r = 0; r < RB / 4; ++r) rows[r].set(a, mask, pc.b, pc.kvh, pc.rb * g.rows + 4 * r + threadIdx.x % 4);
        float o[RB][NC][4];
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[r][c][e] = 0.f;
        const T* kp = static_cast<const T*>(a.k.p) + pc.b * a.k.sb + pc.kvh * a.k.sh;
        const T* vp = static_cast<const T*>(a.v.p) + pc.b * a.v.sb + pc.kvh * a.v.sh;
        // 16-byte vectors of the tile after this one are in registers while this
        // one is used (VEC: rows and head size allow them)
        constexpr int V = 16 / sizeof(T), NV = DA_T * DP / V / DA_THREADS;
        uint4 kr[VEC ? NV : 1], vr[VEC ? NV : 1];
        auto fetch = [&](int t) {
            if constexpr (VEC) {
#pragma unroll
                for (int e = 0; e < NV; ++e) {
                    const int at = threadIdx.x + e * DA_THREADS, r = at / (DP / V), c = at % (DP / V) * V;
                    const int64_t j = (int64_t)t * DA_T + r;
                    const bool on = t < pc.t1 && j < mask.kv && c < a.d && (!kd || kd[j] >= 0);
                    kr[e] = on ? *reinterpret_cast<const uint4*>(kp + j * a.k.ss + c) : make_uint4(0, 0, 0, 0);
                    vr[e] = on ? *reinterpret_cast<const uint4*>(vp + j * a.v.ss + c) : make_uint4(0, 0, 0, 0);
                }
            }
        };
        fetch(pc.t0);
        for (int t = pc.t0; t < pc.t1; ++t) {
            const int j0 = t * DA_T;
            __syncthreads();
            if constexpr (VEC) {
#pragma unroll
                for (int e = 0; e < NV; ++e) {
                    const int at = threadIdx.x + e * DA_THREADS, r = at / (DP / V), c = at % (DP / V) * V;
                    const T *ke = reinterpret_cast<const T*>(&kr[e]), *ve = reinterpret_cast<const T*>(&vr[e]);
#pragma unroll
                    for (int f = 0; f < V; f += 4) {
                        *reinterpret_cast<float4*>(K + r * L::LD + c + f) =
                            make_float4(to_f32(ke[f]), to_f32(ke[f + 1]), to_f32(ke[f + 2]), to_f32(ke[f + 3]));
                        *reinterpret_cast<float4*>(V_ + r * L::LD + c + f) =
                            make_float4(to_f32(ve[f]), to_f32(ve[f + 1]), to_f32(ve[f + 2]), to_f32(ve[f + 3]));
                    }
                }
            } else {
#pragma unroll 4
                for (int e = threadIdx.x; e < DA_T * DP; e += DA_THREADS) {
                    const int r = e / DP, c = e % DP;
                    const int64_t j = j0 + r;
                    const bool on = j < mask.kv && c < a.d && (!kd || kd[j] >= 0);
                    K[r * L::LD + c] = on ? to_f32(kp[j * a.k.ss + c * a.k.sd]) : 0.f;
                    V_[r * L::LD + c] = on ? to_f32(vp[j * a.v.ss + c * a.v.sd]) : 0.f;
                }
            }
            __syncthreads();
            fetch(t + 1);
            {
                const int key = threadIdx.x / 4, part = threadIdx.x % 4;
                float s[RB];
#pragma unroll
                for (int r = 0; r < RB; ++r) s[r] = 0.f;
#pragma unroll 4
                for (int c = 4 * part; c < DP; c += 16) {
                    const float4 k = *reinterpret_cast<const float4*>(K + key * L::LD + c);
#pragma unroll
                    for (int r = 0; r < RB; ++r) {
                        const float4 q = *reinterpret_cast<const float4*>(Q + r * DP + c);
                        s[r] = fmaf(k.x, q.x, fmaf(k.y, q.y, fmaf(k.z, q.z, fmaf(k.w, q.w, s[r]))));
                    }
                }
#pragma unroll
                for (int r = 0; r < RB; ++r) {
                    s[r] += __shfl_xor_sync(0xffffffffu, s[r], 1);
                    s[r] += __shfl_xor_sync(0xffffffffu, s[r], 2);
                }
                const int j = j0 + key, jdoc = kd && j < mask.kv ? kd[j] : -1;
#pragma unroll
                for (int r = 0; r < RB; ++r)
                    if (r % 4 == part) {
                        const DecRow& row = rows[r / 4];
                        float x = s[r];
                        float y = a.cap > 0.f ? a.cap * kLog2e * tanhf(x * (a.scale / a.cap)) : x * (a.scale * kLog2e);
                        y -= row.slope2 * fabsf((float)(row.p - j));
                        P[key * RB + r] = j < row.limit && (!kd || (row.doc >= 0 && jdoc == row.doc)) ? y : -INFINITY;
                    }
            }
            __syncthreads();
            // a warp's rows: maximum, exponentials, sum
            for (int r = warp; r < RB; r += DA_THREADS / 32) {
                const float x0 = P[lane * RB + r], x1 = P[(lane + 32) * RB + r];
                float top = fmaxf(x0, x1);
#pragma unroll
                for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                const float old = m_s[r], nm = fmaxf(old, top), ref = nm == -INFINITY ? 0.f : nm;
                const float e0 = exp2f(x0 - ref), e1 = exp2f(x1 - ref);
                P[lane * RB + r] = e0;
                P[(lane + 32) * RB + r] = e1;
                float sum = e0 + e1;
#pragma unroll
                for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
                __syncwarp();
                if (lane == 0) {
                    const float by = nm == -INFINITY ? 1.f : exp2f(old - nm);
                    by_s[r] = by;
                    l_s[r] = l_s[r] * by + sum;
                    m_s[r] = nm;
                }
            }
            __syncthreads();
            if (lane < LANES) {
#pragma unroll
                for (int r = 0; r < RB; ++r) {
                    const float by = by_s[r];
                    if (by != 1.f)
#pragma unroll
                        for (int c = 0; c < NC; ++c)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[r][c][e] *= by;
                }
#pragma unroll 2
                for (int key = warp; key < DA_T; key += DA_THREADS / 32) {
                    float4 v[NC];
#pragma unroll
                    for (int c = 0; c < NC; ++c) v[c] = *reinterpret_cast<const float4*>(V_ + key * L::LD + 128 * c + 4 * lane);
#pragma unroll
                    for (int r = 0; r < RB; ++r) {
                        const float p = P[key * RB + r];
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            o[r][c][0] = fmaf(p, v[c].x, o[r][c][0]);
                            o[r][c][1] = fmaf(p, v[c].y, o[r][c][1]);
                            o[r][c][2] = fmaf(p, v[c].z, o[r][c][2]);
                            o[r][c][3] = fmaf(p, v[c].w, o[r][c][3]);
                        }
                    }
                }
            }
        }
        // the warps' sums over the tiles' memory; one maximum and sum for all
        __syncthreads();
        float* merge = K;
        if (lane < LANES)
#pragma unroll
            for (int r = 0; r < RB; ++r)
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    *reinterpret_cast<float4*>(merge + (warp * RB + r) * DP + 128 * c + 4 * lane) =
                        make_float4(o[r][c][0], o[r][c][1], o[r][c][2], o[r][c][3]);
        __syncthreads();
        for (int e = threadIdx.x; e < RB * DP; e += DA_THREADS) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) s += merge[w * RB * DP + e];
            Q[e] = s;
        }
        __syncthreads();
        finish_piece<T>(g, pc, Q, 1, 0, DP, m_s, l_s, 0, RB, threadIdx.x, DA_THREADS, K);
        __syncthreads();
        if (g.cluster > 1) join_cluster<T>(g, pc, K, DA_THREADS);
    }
}

bool few_takes_mma(const AttnCall& a) { return a.dtype != TL_TYPE_F32 && attn_tc_takes(a); }
int few_rows(const AttnCall& a) {
    const int64_t rows = (int64_t)a.nq * (a.hq / a.hkv);
    return !few_takes_mma(a) && rows <= 4 ? 4 : 16;
}
int few_blocks(const AttnCall& a) { return a.d > 128 ? kSms : 2 * kSms; }

struct DecPlan {
    size_t part, spans, bytes;
    explicit DecPlan(const AttnCall& a) {
        part = 0;
        bytes = ((size_t)few_blocks(a) * 2 * few_rows(a) * (a.d + 2) * 4 + 255) / 256 * 256;
        spans = bytes;
        if (a.k_doc) bytes += ((size_t)a.b * sizeof(int2) + 255) / 256 * 256;
    }
};

template <typename T, int DP>
tl_status launch_mma(tl_ctx* c, const DecArgs& g, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr int smem = DmSmem<DP>::BYTES;
    TL_TRY(kernel_smem(c, k_decode_mma<T, DP>, smem, done));
    const AttnCall& a = g.a;
    HeadMap mk, mv;
    if (!make_head_map(&mk, a.k, a.dtype, a.b, a.hkv, a.nk, a.d, DmSmem<DP>::DT) ||
        !make_head_map(&mv, a.v, a.dtype, a.b, a.hkv, a.nk, a.d, DmSmem<DP>::DT))
        return fail(c, TL_ERR_CUDA, "attention: tensor maps");
    c->flags_armed = true;
    TL_CK(c, launch_with(k_decode_mma<T, DP>, dim3(g.blocks), g.cluster, DmSmem<DP>::THREADS, smem, false, s, mk, mv, g));
    return TL_OK;
}

template <typename T, int DP, int RB, bool VEC>
tl_status launch_any_as(tl_ctx* c, const DecArgs& g, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr int smem = DaSmem<DP, RB>::BYTES;
    TL_TRY(kernel_smem(c, k_decode_any<T, DP, RB, VEC>, smem, done));
    TL_CK(c, launch_with(k_decode_any<T, DP, RB, VEC>, dim3(g.blocks), g.cluster, DA_THREADS, smem, false, s, g));
    return TL_OK;
}

template <typename T, int DP, int RB>
tl_status launch_any(tl_ctx* c, const DecArgs& g, cudaStream_t s) {
    // rows of whole 16-byte vectors
    const AttnCall& a = g.a;
    const int64_t n = 16 / sizeof(T);
    auto fits = [&](const HeadsView& v) {
        return v.sd == 1 && reinterpret_cast<uintptr_t>(v.p) % 16 == 0 && (a.nk <= 1 || v.ss % n == 0) && (a.hkv <= 1 || v.sh % n == 0) &&
               (a.b <= 1 || v.sb % n == 0);
    };
    if (a.d % n == 0 && fits(a.k) && fits(a.v)) return launch_any_as<T, DP, RB, true>(c, g, s);
    return launch_any_as<T, DP, RB, false>(c, g, s);
}

template <typename T>
tl_status launch_type(tl_ctx* c, const DecArgs& g, cudaStream_t s) {
    const AttnCall& a = g.a;
    cudaEvent_t ev[2];
    launch_begin_on(c, s, "attention_decode", 2.0 * a.b * a.hkv * (double)a.nk * a.d * sizeof(T), 4.0 * a.d * attn_pairs(a), ev);
    if constexpr (!std::is_same<T, float>::value) {
        if (few_takes_mma(a)) {
            if (a.d <= 64) TL_TRY((launch_mma<T, 64>(c, g, s)));
            else TL_TRY((launch_mma<T, 128>(c, g, s)));
            return launch_end_on(c, s, ev);
        }
    }
    if (a.d <= 64) TL_TRY((g.rows == 4 ? launch_any<T, 64, 4>(c, g, s) : launch_any<T, 64, 16>(c, g, s)));
    else if (a.d <= 128) TL_TRY((g.rows == 4 ? launch_any<T, 128, 4>(c, g, s) : launch_any<T, 128, 16>(c, g, s)));
    else TL_TRY((g.rows == 4 ? launch_any<T, 256, 4>(c, g, s) : launch_any<T, 256, 16>(c, g, s)));
    return launch_end_on(c, s, ev);
}

}  // namespace

// Where these kernels are faster than the tiles of 128 queries, if the tensor
// cores take the call at all.  us here / there, one head a group:
//   bf16, d 128, 16 x 8 heads of 4096 keys: 4 rows 51 / 55, 12 rows 60 / 55; with
//     lengths of their own the pieces here stay equal
//   fp16, d 64, the same: 12 rows 37 / 39, 48 rows 80 / 42
//   fp32, d 64, 4 x 16 heads of 4096 keys: 4 rows 49 / 141, 12 rows 172 / 141
// and where few tiles, each shared by eight blocks at most, would walk a long
// cache: 64 rows of one head, 65536 keys: bf16, d 128 50 / 123, fp16, d 64 28 / 105,
// fp32, d 64 171 / 211; of two heads, 32768 keys: 42 / 68, 25 / 57, 169 / 126.
bool attn_few_takes(const AttnCall& a) {
    const int64_t rows = (int64_t)a.nq * (a.hq / a.hkv);
    if (a.nk == 0 || rows > 64) return false;
    if (!attn_tc_takes(a)) return true;
    const bool f32 = a.dtype == TL_TYPE_F32;
    if (a.nk >= 8192 && (int64_t)a.b * a.hkv * ((rows + 15) / 16) <= (f32 ? 4 : a.d <= 64 ? 32 : 12)) return true;
    return rows <= (f32 ? 4 : a.d <= 64 || a.kv_len ? 16 : 8);
}

size_t attn_few_workspace(const AttnCall& a) { return DecPlan(a).bytes; }

tl_status launch_attn_few(tl_ctx* c, const AttnCall& a, void* ws, cudaStream_t s) {
    const DecPlan plan(a);
    uint8_t* w = static_cast<uint8_t*>(ws);
    DecArgs g;
    g.a = a;
    g.rows = few_rows(a);
    g.row_blocks = (int)(((int64_t)a.nq * (a.hq / a.hkv) + g.rows - 1) / g.rows);
    g.part = reinterpret_cast<float*>(w + plan.part);
    g.spans = nullptr;
    g.err = c->d_flags + 8;
    // no more blocks than tiles there can be
    const int64_t units = (int64_t)a.b * a.hkv * g.row_blocks, rows = (int64_t)a.nq * (a.hq / a.hkv);
    g.tile = few_takes_mma(a) && a.d <= 64 ? 128 : 64;
    const int64_t tiles = (a.nk + g.tile - 1) / g.tile;
    // A cluster a unit while all of them run at once and a block has few tiles: one
    // launch for two.  Cluster / line, us: bf16, 1 x 32 heads over 8, 512 keys 6.9 / 8.8,
    // 2048 9.9 / 11.8, 2 x 32 heads, 4096 14.9 / 13.9; fp32, 512 keys 9.3 / 11.0, 1024 14.3 /
    // 13.5, 2048 18 / 15.
    g.cluster = units * 8 <= kSms && tiles <= (few_takes_mma(a) ? 32 : 8) ? 8 : 1;
    g.blocks = g.cluster > 1 ? (int)units * g.cluster : (int)std::min<int64_t>(few_blocks(a), units * tiles);
    cudaEvent_t ev[2];
    if (a.k_doc) {
        int2* spans = reinterpret_cast<int2*>(w + plan.spans);
        g.spans = spans;
        launch_begin_on(c, s, "attention_doc_spans", 4.0 * a.b * a.nk, 0, ev);
        k_doc_spans<<<a.b, 256, 0, s>>>(a, spans);
        TL_TRY(launch_end_on(c, s, ev));
    }
    switch (a.dtype) {
    case TL_TYPE_F32: TL_TRY(launch_type<float>(c, g, s)); break;
    case TL_TYPE_F16: TL_TRY(launch_type<__half>(c, g, s)); break;
    default: TL_TRY(launch_type<__nv_bfloat16>(c, g, s));
    }
    if (g.cluster > 1) return TL_OK;
    launch_begin_on(c, s, "attention_decode_join", 0, 0, ev);
    cudaError_t e;
    switch (a.dtype) {
    case TL_TYPE_F32: e = launch_with(k_decode_join<float>, dim3((unsigned)((int64_t)a.b * a.hkv * rows)), 1, JOIN_THREADS, 0, true, s, g); break;
    case TL_TYPE_F16: e = launch_with(k_decode_join<__half>, dim3((unsigned)((int64_t)a.b * a.hkv * rows)), 1, JOIN_THREADS, 0, true, s, g); break;
    default: e = launch_with(k_decode_join<__nv_bfloat16>, dim3((unsigned)((int64_t)a.b * a.hkv * rows)), 1, JOIN_THREADS, 0, true, s, g);
    }
    TL_CK(c, e);
    return launch_end_on(c, s, ev);
}

}  // namespace tl
