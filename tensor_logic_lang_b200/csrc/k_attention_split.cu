// fp32 arrays as pairs of fp16 for the tensor-core attention kernels: the
// largest value of every group of heads, then hi and lo of every value (attn_tc.h,
// SplitArray), and what the backward pass needs of the rows.  HBM-bound: the arrays are read twice (the second time mostly
// from the L2 cache) and their 4 bytes a value written once.
//
// Three fp16 products of 11-bit parts give 22 bits; TF32 would take the same
// three at half the rate, and fp32 on the CUDA cores runs at a tenth of it.
#include <algorithm>

#include "attn_tc.h"

namespace tl {
namespace {

constexpr int SP_ROWS = 64;   // of a block of 8 warps

struct SplitArgs {
    AttnCall a;
    SplitArray arr[4];
    // backward: of operands with their powers of two, so that no square leaves fp32
    uint32_t* norms;
    float* stats;     // [b, hq, query tiles][2][128], -log2(e) lse + lift and -D = -dout.out of each row
};

__device__ __forceinline__ bool row_counts(const AttnCall& a, const SplitArray& x, int b, int64_t r) {
    if (r >= x.n) return false;
    if (!x.keys) return !a.q_doc || a.q_doc[(int64_t)b * a.nq + r] >= 0;
    const int kv = a.kv_len ? min(max(a.kv_len[b], 0), a.nk) : a.nk;
    return r < kv && (!a.k_doc || a.k_doc[(int64_t)b * a.nk + r] >= 0);
}

// Columns c and c + 1 of a row (0 past the head size); pairs: as one load (4 x 8 x
// 1024 x 128, forward call: 77 us, 82 with two).
__device__ __forceinline__ float2 two(const float* row, int64_t sd, int c, int d, bool pairs) {
    if (pairs) return c < d ? *reinterpret_cast<const float2*>(row + c) : make_float2(0.f, 0.f);
    return make_float2(c < d ? row[c * sd] : 0.f, c + 1 < d ? row[(c + 1) * sd] : 0.f);
}
__device__ __forceinline__ bool in_pairs(const HeadsView& v, int d) {
    return v.sd == 1 && d % 2 == 0 && (v.ss | v.sh | v.sb) % 2 == 0 && reinterpret_cast<uintptr_t>(v.p) % 8 == 0;
}

// The largest of a block's values into *to.  Non-negative floats order like their
// bits; a maximum does not depend on the order.
__device__ __forceinline__ void block_max(float v, uint32_t* to) {
    __shared__ uint32_t most[8];
    const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
    if ((threadIdx.x & 31) == 0) most[threadIdx.x / 32] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t all = 0;
        for (int k = 0; k < 8; ++k) all = max(all, most[k]);
        atomicMax(to, all);
    }
}

// A warp takes 8 rows, a lane columns 2 lane and 2 lane + 1 of every 64.
template <bool WRITE, int HALVES>
__global__ void __launch_bounds__(256) k_split(const __grid_constant__ SplitArgs g) {
    let_next_start();
    if (WRITE) wait_for_previous();   // the largest values
    const AttnCall& a = g.a;
    const SplitArray& x = g.arr[blockIdx.y];
    const unsigned blocks = (x.n + TILE - 1) / TILE * (TILE / SP_ROWS);
    if (blockIdx.x >= (int64_t)blocks * x.h * a.b) return;
    const int bh = blockIdx.x / blocks, b = bh / x.h, h = bh % x.h;
    const int group = b * a.hkv + h / (x.h / a.hkv);
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, c = 2 * lane;
    const int64_t r0 = (int64_t)(blockIdx.x % blocks) * SP_ROWS + warp * 8;
    const float* p = static_cast<const float*>(x.v.p) + b * x.v.sb + h * x.v.sh;
    const bool pairs = in_pairs(x.v, a.d);
    float2 u[8][HALVES];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const bool on = row_counts(a, x, b, r0 + k);
#pragma unroll
        for (int f = 0; f < HALVES; ++f)
            u[k][f] = on ? two(p + (r0 + k) * x.v.ss, x.v.sd, c + 64 * f, a.d, pairs) : make_float2(0.f, 0.f);
    }
    if (WRITE) {
        const float up = pow2(split_exp(x.top, group));
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int f = 0; f < HALVES; ++f) u[k][f] = make_float2(u[k][f].x * up, u[k][f].y * up);
        __half* out = x.out + ((int64_t)bh * x.n + r0) * (128 * HALVES) + c;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (r0 + k >= x.n) break;
#pragma unroll
            for (int f = 0; f < HALVES; ++f) {
                uint32_t hi, lo;
                split16(u[k][f].x, u[k][f].y, hi, lo);
                *reinterpret_cast<uint32_t*>(out + (k * HALVES + f) * 128) = hi;
                *reinterpret_cast<uint32_t*>(out + (k * HALVES + f) * 128 + 64) = lo;
            }
        }
        if (g.stats && blockIdx.y == 3) {
            // dout: D of its rows, and the statistics of whole tiles
            const float* o = static_cast<const float*>(a.o.p) + b * a.o.sb + h * a.o.sh;
            const float up_o = pow2(split_exp(g.arr[2].top, group));   // o's values are within those of v
            const int64_t qt = r0 / TILE, q_tiles = blocks / (TILE / SP_ROWS);
            float* st = g.stats + ((int64_t)bh * q_tiles + qt) * 2 * TILE + r0 % TILE;
            const bool live = lane < 8 && row_counts(a, x, b, r0 + lane);
            const float lse = live ? a.lse[(int64_t)bh * a.nq + r0 + lane] : -INFINITY;
            const bool o_pairs = in_pairs(a.o, a.d);
            float dot[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                dot[k] = 0.f;
                if (!row_counts(a, x, b, r0 + k)) continue;
#pragma unroll
                for (int f = 0; f < HALVES; ++f) {
                    const float2 y = two(o + (r0 + k) * a.o.ss, a.o.sd, c + 64 * f, a.d, o_pairs);
                    dot[k] = fmaf(u[k][f].x, y.x * up_o, fmaf(u[k][f].y, y.y * up_o, dot[k]));
                }
            }
            float d = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
#pragma unroll
                for (int m = 16; m; m >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], m);
                if (lane == k) d = dot[k];
            }
            if (lane < 8) {
                // a row that sees nothing has p = 2^-inf = 0 everywhere
                st[lane] = lse == -INFINITY ? -INFINITY : PLift<__half>::log2 - lse * kLog2e;
                st[TILE + lane] = -d;
            }
        }
        if (x.norm >= 0) {
            float norm = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                float n2 = 0.f;
#pragma unroll
                for (int f = 0; f < HALVES; ++f) n2 = fmaf(u[k][f].x, u[k][f].x, fmaf(u[k][f].y, u[k][f].y, n2));
#pragma unroll
                for (int m = 16; m; m >>= 1) n2 += __shfl_xor_sync(0xffffffffu, n2, m);
                norm = fmaxf(norm, finite(n2));
            }
            block_max(norm, &g.norms[2 * group + x.norm]);
        }
    } else {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int f = 0; f < HALVES; ++f) top = fmaxf(top, fmaxf(finite(fabsf(u[k][f].x)), finite(fabsf(u[k][f].y))));
        wait_for_previous();   // the maxima start at 0
        block_max(top, &x.top[group]);
    }
}

}  // namespace

SplitPlan::SplitPlan(const AttnCall& a, bool backward) {
    bytes = 0;
    auto take = [&](size_t n) { const size_t at = bytes; bytes += (n + 255) / 256 * 256; return at; };
    // the words that start at zero lie together
    const size_t groups = (size_t)a.b * a.hkv;
    top = take(groups * (4 * 4 + 8));
    norms = top + groups * 4 * 4;
    const size_t row = 2 * (size_t)split_width(a.d), q = row * a.b * a.hq * a.nq, k = row * a.b * a.hkv * a.nk;
    data[0] = take(q);
    data[1] = take(k);
    data[2] = take(k);
    data[3] = take(backward ? q : 0);
}

tl_status launch_split(tl_ctx* c, const AttnCall& a, float* stats, uint8_t* ws, HeadMap* maps, DocRange* q_ranges, DocRange* k_ranges,
                       cudaStream_t s) {
    const bool backward = stats != nullptr;
    const SplitPlan plan(a, backward);
    SplitArgs g;
    g.a = a;
    g.stats = stats;
    uint32_t* top = reinterpret_cast<uint32_t*>(ws + plan.top);
    g.norms = reinterpret_cast<uint32_t*>(ws + plan.norms);
    const int count = backward ? 4 : 3;
    const HeadsView* views[4] = {&a.q, &a.k, &a.v, &a.dout};
    int64_t grid = 0;
    for (int i = 0; i < count; ++i) {
        SplitArray& x = g.arr[i];
        x.keys = i == 1 || i == 2;
        x.v = *views[i];
        x.h = x.keys ? a.hkv : a.hq;
        x.n = x.keys ? a.nk : a.nq;
        x.norm = !backward ? -1 : i == 3 ? 0 : i == 2 ? 1 : -1;
        x.out = reinterpret_cast<__half*>(ws + plan.data[i]);
        x.top = top;
        top += (size_t)a.b * a.hkv;
        grid = std::max<int64_t>(grid, (int64_t)a.b * x.h * ((x.n + TILE - 1) / TILE * (TILE / SP_ROWS)));
        const int64_t w = split_width(a.d);
        const HeadsView flat = {x.out, x.h * x.n * w, x.n * w, w, 1};
        if (!make_head_map(&maps[i], flat, TL_TYPE_F16, a.b, x.h, x.n, (int)w)) return fail(c, TL_ERR_CUDA, "attention: tensor maps");
    }
    TL_TRY(launch_attn_begin(c, a, q_ranges, k_ranges, reinterpret_cast<uint32_t*>(ws + plan.top), (int64_t)a.b * a.hkv * 6, s));
    const double bytes = (double)a.b * a.d * ((double)(backward ? 2 : 1) * a.hq * a.nq + 2.0 * a.hkv * a.nk);
    cudaEvent_t ev[2];
    launch_begin_on(c, s, "attention_split_top", 4 * bytes, 0, ev);
    const bool wide = a.d > 64;
    TL_CK(c, launch_with(wide ? k_split<false, 2> : k_split<false, 1>, dim3((unsigned)grid, count), 1, 256, 0, true, s, g));
    TL_TRY(launch_end_on(c, s, ev));
    launch_begin_on(c, s, "attention_split", 8 * bytes, 0, ev);
    TL_CK(c, launch_with(wide ? k_split<true, 2> : k_split<true, 1>, dim3((unsigned)grid, count), 1, 256, 0, true, s, g));
    return launch_end_on(c, s, ev);
}

}  // namespace tl
