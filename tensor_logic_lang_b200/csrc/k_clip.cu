// The global norm of a list of arrays and their scaling to a largest norm.
//
//   k_clip_norm   every block sums the squares of its chunks of the list in 64
//                 bits and writes one partial sum;
//   k_clip_scale  every block adds the partial sums in one order (all blocks
//                 get the same norm, whatever ran first), and multiplies its
//                 chunks by min(1, max_norm / norm).  In place and under the
//                 limit it has nothing to do.
//
// HBM-bound: the list is read once for the norm, and read and written once
// more where it is scaled.  A chunk is a piece of one array; the list travels
// in the launch's parameters (no copy, so a captured call keeps it).
#include <math.h>

#include <algorithm>

#include "attention.h"

namespace tl {
namespace {

constexpr int CL_THREADS = 256, CL_CHUNK = 32768, CL_MAX_BLOCKS = 148 * 8;

struct ClipEntry {
    const void* in;
    void* out;
    int64_t n;
    uint32_t first;      // chunk number of its first element within the launch
    uint16_t in_type, out_type;
};
// 32-byte entries in at most 32764 bytes of parameters
template <int CAP>
struct ClipList {
    int32_t count;
    uint32_t chunks;
    ClipEntry e[CAP];
};

template <int CAP>
__device__ __forceinline__ int find_entry(const ClipList<CAP>& list, uint32_t chunk) {
    int lo = 0, hi = list.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (list.e[mid].first <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int w = 16; w; w >>= 1) v += __shfl_xor_sync(0xffffffffu, v, w);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0;
#pragma unroll
    for (int w = 0; w < CL_THREADS / 32; ++w) s += red[w];
    __syncthreads();
    return s;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int64_t n) {
    double s = 0;
    for (int64_t i = threadIdx.x; i < n; i += CL_THREADS) {
        const double x = to_f32(p[i]);
        s = fma(x, x, s);
    }
    return s;
}

template <int CAP>
__global__ void __launch_bounds__(CL_THREADS) k_clip_norm(const __grid_constant__ ClipList<CAP> list, double* __restrict__ part) {
    __shared__ double red[CL_THREADS / 32];
    double s = 0;
    for (uint32_t ch = blockIdx.x; ch < list.chunks; ch += gridDim.x) {
        const ClipEntry& e = list.e[find_entry(list, ch)];
        const int64_t at = (int64_t)(ch - e.first) * CL_CHUNK;
        const int64_t n = min((int64_t)CL_CHUNK, e.n - at);
        if (e.in_type == TL_TYPE_F32) s += chunk_squares(static_cast<const float*>(e.in) + at, n);
        else if (e.in_type == TL_TYPE_F16) s += chunk_squares(static_cast<const __half*>(e.in) + at, n);
        else s += chunk_squares(static_cast<const __nv_bfloat16*>(e.in) + at, n);
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <typename T, typename U>
__device__ __forceinline__ void chunk_scale(const T* in, U* out, int64_t n, float by) {
    for (int64_t i = threadIdx.x; i < n; i += CL_THREADS) out[i] = from_f32<U>(to_f32(in[i]) * by);
}

template <typename T>
__device__ __forceinline__ void chunk_scale_to(const T* in, const ClipEntry& e, int64_t at, int64_t n, float by) {
    if (e.out_type == TL_TYPE_F32) chunk_scale(in, static_cast<float*>(e.out) + at, n, by);
    else if (e.out_type == TL_TYPE_F16) chunk_scale(in, static_cast<__half*>(e.out) + at, n, by);
    else chunk_scale(in, static_cast<__nv_bfloat16*>(e.out) + at, n, by);
}

template <int CAP>
__global__ void __launch_bounds__(CL_THREADS)
    k_clip_scale(const __grid_constant__ ClipList<CAP> list, const double* __restrict__ part, int n_part, double max_norm,
                 float* __restrict__ norm_out) {
    __shared__ double red[CL_THREADS / 32];
    double s = 0;
    for (int i = threadIdx.x; i < n_part; i += CL_THREADS) s += part[i];
    const double norm = sqrt(block_sum(s, red));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float by = isfinite(norm) && norm > max_norm ? (float)(max_norm / norm) : 1.f;
    for (uint32_t ch = blockIdx.x; ch < list.chunks; ch += gridDim.x) {
        const ClipEntry& e = list.e[find_entry(list, ch)];
        if (by == 1.f && e.in == e.out && e.in_type == e.out_type) continue;
        const int64_t at = (int64_t)(ch - e.first) * CL_CHUNK;
        const int64_t n = min((int64_t)CL_CHUNK, e.n - at);
        if (e.in_type == TL_TYPE_F32) chunk_scale_to(static_cast<const float*>(e.in) + at, e, at, n, by);
        else if (e.in_type == TL_TYPE_F16) chunk_scale_to(static_cast<const __half*>(e.in) + at, e, at, n, by);
        else chunk_scale_to(static_cast<const __nv_bfloat16*>(e.in) + at, e, at, n, by);
    }
}

template <int CAP>
tl_status clip(tl_ctx* c, const std::vector<ClipItem>& items, double max_norm, float* norm, double* part, cudaStream_t s) {
    // launches of at most CAP arrays and 2^31 chunks
    std::vector<ClipList<CAP>> lists;
    double bytes = 0, wrote = 0;
    for (const ClipItem& it : items) {
        const int64_t ch = (it.n + CL_CHUNK - 1) / CL_CHUNK;
        if (ch > 0x7fffffff) return fail(c, TL_ERR_TOO_LARGE, "clip: an array of %lld elements", (long long)it.n);
        if (lists.empty() || lists.back().count == CAP || lists.back().chunks + ch > 0x7fffffff) {
            lists.emplace_back();
            lists.back().count = 0;
            lists.back().chunks = 0;
        }
        auto& l = lists.back();
        l.e[l.count++] = {it.in, it.out, it.n, l.chunks, (uint16_t)it.in_type, (uint16_t)it.out_type};
        l.chunks += (uint32_t)ch;
        bytes += (double)it.n * type_size(it.in_type);
        wrote += it.in == it.out ? 0.0 : (double)it.n * type_size(it.out_type);
    }
    if (lists.empty()) lists.emplace_back();   // the norm of nothing
    if (items.empty()) { lists[0].count = 0; lists[0].chunks = 0; }
    const int per = std::max(1, CL_MAX_BLOCKS / (int)lists.size());
    if ((int64_t)per * (int64_t)lists.size() > CL_MAX_BLOCKS)
        return fail(c, TL_ERR_TOO_LARGE, "clip: %zu arrays", items.size());
    int n_part = 0;
    cudaEvent_t ev[2];
    std::vector<int> grid;
    for (auto& l : lists) {
        const int g = (int)std::min<uint32_t>(per, std::max(1u, l.chunks));
        grid.push_back(g);
        launch_begin_on(c, s, "clip_norm", bytes / lists.size(), 0, ev);
        k_clip_norm<CAP><<<g, CL_THREADS, 0, s>>>(l, part + n_part);
        TL_TRY(launch_end_on(c, s, ev));
        n_part += g;
    }
    for (size_t i = 0; i < lists.size(); ++i) {
        launch_begin_on(c, s, "clip_scale", (bytes + wrote) / lists.size(), 0, ev);
        k_clip_scale<CAP><<<grid[i], CL_THREADS, 0, s>>>(lists[i], part, n_part, max_norm, i == 0 ? norm : nullptr);
        TL_TRY(launch_end_on(c, s, ev));
    }
    return TL_OK;
}

}  // namespace

size_t clip_workspace_bytes() { return CL_MAX_BLOCKS * sizeof(double); }

tl_status launch_clip(tl_ctx* c, const std::vector<ClipItem>& items, double max_norm, float* norm, void* ws, cudaStream_t s) {
    double* part = static_cast<double*>(ws);
    if (items.size() <= 16) return clip<16>(c, items, max_norm, norm, part, s);
    return clip<1000>(c, items, max_norm, norm, part, s);
}

}  // namespace tl
