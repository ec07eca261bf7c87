// The global norm of a list of arrays and their scaling to a largest norm.
//
//   k_clip_norm   every block sums the squares of its chunks of the list and
//                 writes one partial sum (64 bits);
//   k_clip_scale  every block adds the partial sums in one order (all blocks
//                 get the same norm, whatever ran first), and multiplies its
//                 chunks by min(1, max_norm / norm).  In place and under the
//                 limit it has nothing to do.
//
// HBM-bound: the list is read once for the norm, and read and written once
// more where it is scaled, the last chunks first: the L2 cache still holds
// those.  The blocks take the chunks in turn.  400M bf16 into fp32, one array: 514 us, 6.2 TB/s of the 3.2 GB that
// two reads and a write are; 291 arrays of six sizes: 563 to 573 us; 360 MB of fp32 under the limit:
// 64 to 67 us, 5.5 TB/s, in place over it 193 us, 5.6 TB/s.  A chunk is a piece of one array; the list travels in the launch's
// parameters (no copy, so a captured call keeps it).  128-bit loads, eight
// in flight a thread (four: 585 us), stores of up to 256 bits; a chunk whose array
// starts between 16-byte boundaries peels its first elements.
//
// The squares of a 128-bit load are added in fp32 and go into a 64-bit sum;
// where they could leave the range of fp32 (a sum outside 2^-90 .. 2^120, zeros
// included) they are taken again in 64 bits.
#include <math.h>

#include <algorithm>

#include "attention.h"

namespace tl {
namespace {

constexpr int CL_THREADS = 256, CL_MAX_BLOCKS = 148 * 4, CL_MAX_CHUNK = 65536, CL_MIN_CHUNK = 2048;
constexpr int CL_FLIGHT = 8;   // loads in flight a thread

struct ClipEntry {
    const void* in;
    void* out;
    int64_t n;
    uint32_t first;      // chunk number of its first element within the launch
    uint16_t in_type, out_type;
};
// The elements before an array's first 16-byte boundary belong to its first
// chunk, so every other chunk starts on one and the full ones are equal.
__host__ __device__ inline int64_t head_of(const void* p, int64_t n, int type) {
    const int64_t size = type == TL_TYPE_F32 ? 4 : 2;
    const int64_t h = (16 - (int64_t)(reinterpret_cast<uintptr_t>(p) & 15)) % 16 / size;
    return h < n ? h : n;
}
struct Run {
    int64_t at, n;
    __device__ __forceinline__ Run(const ClipEntry& e, uint32_t k, int64_t chunk) {
        const int64_t h = head_of(e.in, e.n, e.in_type), to = h + (k + 1) * chunk;
        at = k ? h + k * chunk : 0;
        n = (to < e.n ? to : e.n) - at;
    }
};

// 32-byte entries: 1000 of them stay below the 32764 bytes of a launch's parameters.
template <int CAP>
struct ClipList {
    int32_t count;
    uint32_t chunks;
    int64_t chunk;       // elements of a chunk
    alignas(16) ClipEntry e[CAP];
};

// The list in shared memory, and the search for a chunk's array.  Generic
// loads of the parameters: through the constant cache, threads that index them
// take turns, and every chunk's entry would be a miss (12 us of 63 for 57
// arrays of 360 MB together).
template <int CAP>
struct Index {
    ClipEntry e[CAP];
    __device__ __forceinline__ void fill(const ClipList<CAP>& list) {
        uint4* to = reinterpret_cast<uint4*>(e);
        for (int i = threadIdx.x; i < 2 * list.count; i += CL_THREADS) {
            uint4 v;
            asm volatile("ld.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "l"(reinterpret_cast<const uint4*>(list.e) + i));
            to[i] = v;
        }
        __syncthreads();
    }
    __device__ __forceinline__ const ClipEntry& find(int count, uint32_t chunk) const {
        int lo = 0, hi = count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (e[mid].first <= chunk) lo = mid; else hi = mid - 1;
        }
        return e[lo];
    }
};

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

// A chunk as elements before the first 16-byte boundary, 128-bit vectors, and
// the elements behind them.
template <typename T>
struct Parts {
    static constexpr int V = 16 / sizeof(T);
    int64_t head, vecs;
    __device__ __forceinline__ Parts(const T* p, int64_t n) {
        head = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) % 16 / sizeof(T);
        if (head > n) head = n;
        vecs = (n - head) / V;
    }
};

template <typename T>
__device__ __forceinline__ double square(T v) {
    const double x = to_f32(v);
    return x * x;
}

template <typename T>
__device__ __forceinline__ double vec_squares(const uint4& raw) {
    const T* x = reinterpret_cast<const T*>(&raw);
    constexpr int V = Parts<T>::V;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) s = fmaf(to_f32(x[i]), to_f32(x[i]), s);
    if (TypeOf<T>::id == TL_TYPE_F16 || (s > 0x1p-90f && s < 0x1p120f)) return s;
    double d = 0;
    if (s != 0.f || ((raw.x | raw.y | raw.z | raw.w) & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)))
        for (int i = 0; i < V; ++i) d += square(x[i]);
    return d;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int64_t n) {
    const Parts<T> parts(p, n);
    double s = 0;
    if (threadIdx.x < parts.head) s += square(p[threadIdx.x]);
    const uint4* v = reinterpret_cast<const uint4*>(p + parts.head);
    int64_t i = threadIdx.x, full = parts.vecs / (CL_FLIGHT * CL_THREADS);
    for (; full; --full, i += CL_FLIGHT * CL_THREADS) {
        uint4 raw[CL_FLIGHT];
#pragma unroll
        for (int k = 0; k < CL_FLIGHT; ++k) raw[k] = __ldg(v + i + k * CL_THREADS);
#pragma unroll
        for (int k = 0; k < CL_FLIGHT; ++k) s += vec_squares<T>(raw[k]);
    }
    if (i < parts.vecs) {
        uint4 raw[CL_FLIGHT];
#pragma unroll
        for (int k = 0; k < CL_FLIGHT; ++k)
            raw[k] = i + k * CL_THREADS < parts.vecs ? __ldg(v + i + k * CL_THREADS) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < CL_FLIGHT; ++k) s += vec_squares<T>(raw[k]);
    }
    const int64_t rest = parts.head + parts.vecs * Parts<T>::V + threadIdx.x;
    if (rest < n) s += square(p[rest]);
    return s;
}

template <int CAP>
__global__ void __launch_bounds__(CL_THREADS) k_clip_norm(const __grid_constant__ ClipList<CAP> list, double* __restrict__ part) {
    __shared__ double red[CL_THREADS / 32];
    let_next_start();
    __shared__ __align__(16) Index<CAP> index;
    index.fill(list);
    double s = 0;
    for (uint32_t ch = blockIdx.x; ch < list.chunks; ch += gridDim.x) {
        const ClipEntry& e = index.find(list.count, ch);
        const Run run(e, ch - e.first, list.chunk);
        const int64_t at = run.at, n = run.n;
        if (e.in_type == TL_TYPE_F32) s += chunk_squares(static_cast<const float*>(e.in) + at, n);
        else if (e.in_type == TL_TYPE_F16) s += chunk_squares(static_cast<const __half*>(e.in) + at, n);
        else s += chunk_squares(static_cast<const __nv_bfloat16*>(e.in) + at, n);
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// 16 bytes of T, scaled, as elements of U
template <typename T, typename U>
__device__ __forceinline__ void vec_scale(const uint4& raw, U* out, float by, bool aligned) {
    constexpr int V = Parts<T>::V, W = V * sizeof(U);   // bytes written: 8, 16 or 32
    const T* x = reinterpret_cast<const T*>(&raw);
    __align__(32) U y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = from_f32<U>(to_f32(x[i]) * by);
    if (!aligned) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = y[i];
    } else if (W == 32) {
        const float* f = reinterpret_cast<const float*>(y);
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "f"(f[0]), "f"(f[1]), "f"(f[2]),
                     "f"(f[3]), "f"(f[4 % V]), "f"(f[5 % V]), "f"(f[6 % V]), "f"(f[7 % V])
                     : "memory");
    } else if (W == 8) {
        *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(y);
    } else {
        *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(y);
    }
}

// in and out may be one array: a thread writes only what it has read
template <typename T, typename U>
__device__ __forceinline__ void chunk_scale(const T* in, U* out, int64_t n, float by) {
    const Parts<T> parts(in, n);
    constexpr int V = Parts<T>::V, W = V * sizeof(U);
    if (threadIdx.x < parts.head) out[threadIdx.x] = from_f32<U>(to_f32(in[threadIdx.x]) * by);
    const uint4* v = reinterpret_cast<const uint4*>(in + parts.head);
    U* o = out + parts.head;
    const bool aligned = reinterpret_cast<uintptr_t>(o) % W == 0;
    int64_t i = threadIdx.x, full = parts.vecs / (CL_FLIGHT * CL_THREADS);
    for (; full; --full, i += CL_FLIGHT * CL_THREADS) {
        uint4 raw[CL_FLIGHT];
#pragma unroll
        for (int k = 0; k < CL_FLIGHT; ++k) raw[k] = v[i + k * CL_THREADS];
#pragma unroll
        for (int k = 0; k < CL_FLIGHT; ++k) vec_scale<T>(raw[k], o + (i + k * CL_THREADS) * V, by, aligned);
    }
    if (i < parts.vecs) {
        uint4 raw[CL_FLIGHT];
#pragma unroll
        for (int k = 0; k < CL_FLIGHT; ++k)
            if (i + k * CL_THREADS < parts.vecs) raw[k] = v[i + k * CL_THREADS];
#pragma unroll
        for (int k = 0; k < CL_FLIGHT; ++k)
            if (i + k * CL_THREADS < parts.vecs) vec_scale<T>(raw[k], o + (i + k * CL_THREADS) * V, by, aligned);
    }
    const int64_t rest = parts.head + parts.vecs * V + threadIdx.x;
    if (rest < n) out[rest] = from_f32<U>(to_f32(in[rest]) * by);
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
    __shared__ __align__(16) Index<CAP> index;
    index.fill(list);
    wait_for_previous();
    double s = 0;
    for (int i = threadIdx.x; i < n_part; i += CL_THREADS) s += part[i];
    const double norm = sqrt(block_sum(s, red));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float by = isfinite(norm) && norm > max_norm ? (float)(max_norm / norm) : 1.f;
    for (uint32_t back = blockIdx.x; back < list.chunks; back += gridDim.x) {
        const uint32_t ch = list.chunks - 1 - back;
        const ClipEntry& e = index.find(list.count, ch);
        if (by == 1.f && e.in == e.out && e.in_type == e.out_type) continue;
        const Run run(e, ch - e.first, list.chunk);
        const int64_t at = run.at, n = run.n;
        if (e.in_type == TL_TYPE_F32) chunk_scale_to(static_cast<const float*>(e.in) + at, e, at, n, by);
        else if (e.in_type == TL_TYPE_F16) chunk_scale_to(static_cast<const __half*>(e.in) + at, e, at, n, by);
        else chunk_scale_to(static_cast<const __nv_bfloat16*>(e.in) + at, e, at, n, by);
    }
}

template <int CAP>
tl_status clip(tl_ctx* c, const std::vector<ClipItem>& items, double max_norm, float* norm, double* part, cudaStream_t s) {
    double bytes = 0, wrote = 0, total = 0;
    for (const ClipItem& it : items) {
        bytes += (double)it.n * type_size(it.in_type);
        wrote += it.in == it.out ? 0.0 : (double)it.n * type_size(it.out_type);
        total += (double)it.n;
    }
    // short lists: one chunk a block, all of its loads in flight at once
    const int64_t chunk = std::min<int64_t>(
        CL_MAX_CHUNK, ((int64_t)(total / CL_MAX_BLOCKS) / CL_MIN_CHUNK + 1) * CL_MIN_CHUNK);
    // launches of at most CAP arrays and 2^31 chunks
    std::vector<ClipList<CAP>> lists;
    for (const ClipItem& it : items) {
        const int64_t ch = std::max<int64_t>(1, (it.n - head_of(it.in, it.n, it.in_type) + chunk - 1) / chunk);
        if (ch > 0x7fffffff) return fail(c, TL_ERR_TOO_LARGE, "clip: an array of %lld elements", (long long)it.n);
        if (lists.empty() || lists.back().count == CAP || lists.back().chunks + ch > 0x7fffffff) {
            lists.emplace_back();
            lists.back().count = 0;
            lists.back().chunks = 0;
            lists.back().chunk = chunk;
        }
        auto& l = lists.back();
        l.e[l.count++] = {it.in, it.out, it.n, l.chunks, (uint16_t)it.in_type, (uint16_t)it.out_type};
        l.chunks += (uint32_t)ch;
    }
    if (lists.empty()) {   // the norm of nothing
        lists.emplace_back();
        lists[0].count = 0;
        lists[0].chunks = 0;
        lists[0].chunk = chunk;
    }
    const int per = CL_MAX_BLOCKS / (int)std::min<size_t>(lists.size(), CL_MAX_BLOCKS);
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
        // long lists are scaled by half as many blocks: with fewer streams of
        // writes open the scaling of 400M bf16 into fp32 takes 392 us, not 420
        if (lists[i].chunks > CL_MAX_BLOCKS) grid[i] = (grid[i] + 1) / 2;
        launch_begin_on(c, s, "clip_scale", (bytes + wrote) / lists.size(), 0, ev);
        if (lists.size() == 1) {
            TL_CK(c, launch_with(k_clip_scale<CAP>, dim3(grid[i]), 1, CL_THREADS, 0, true, s, lists[i], static_cast<const double*>(part), n_part,
                                  max_norm, norm));
        } else {
            k_clip_scale<CAP><<<grid[i], CL_THREADS, 0, s>>>(lists[i], part, n_part, max_norm, i == 0 ? norm : nullptr);
        }
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
