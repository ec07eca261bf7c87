// Attention with modified scores for any type, stride and head size up to
// 256 (where the tensor-core kernels' rules do not hold, attn_tc_takes): tiles of
// queries against tiles of keys in shared memory, fp32 FFMA products, one pass
// over the keys with a running maximum and sum.
//
//   forward   a block per (sequence, head, query tile):
//               s = scores(q k), m' = max(m, s), l = l e^{m-m'} + sum e^{s-m'},
//               o = o e^{m-m'} + e^{s-m'} v;  o / l and lse = m + log l at the end
//   backward  D = dout . o by row, then a block per query tile for dq = dx k
//             and a block per key tile for dv = p^T dout, dk = dx^T q, summed
//             over the query tiles and the heads that share the keys in a
//             fixed order (no atomics).
//
// A tile is TS x TS scores; each of the 256 threads holds a TS/16 x TS/16
// block of them and as many rows of DP/16 columns of a result, so a product
// step costs 8 128-bit shared loads for 64 FMAs (TS = 64).  Rows are padded
// by 16 bytes, which spreads the 16 rows that a half warp reads over the
// banks.  Head sizes above 128 take TS = 32 (four operand tiles of 64 x 260
// floats do not fit in 227 KB).
#include <algorithm>

#include "attention.h"

namespace tl {
namespace {

constexpr int GA_THREADS = 256;
constexpr float kNegInf = -__builtin_huge_valf();

template <int TS, int DP>
struct GaTile {
    static constexpr int LD = DP + 4, LP = TS + 4, R = TS / 16, C = DP / 16;
    static constexpr int OPERAND = TS * LD * 4, SCORES = TS * LP * 4;
};

// Rows [row0, row0 + TS) of one head as fp32, zeros past n rows and d columns
// and at rows of a negative document (what they hold must not count).
template <typename T, int TS, int DP>
__device__ __forceinline__ void load_rows(float* dst, const HeadsView& v, int b, int h, int row0, int n, int d,
                                          const int32_t* doc) {
    const T* base = static_cast<const T*>(v.p) + b * v.sb + h * v.sh;
    for (int i = threadIdx.x; i < TS * DP; i += GA_THREADS) {
        const int r = i / DP, col = i % DP;
        const int64_t row = row0 + r;
        float x = 0.f;
        if (row < n && col < d && (!doc || doc[row] >= 0)) x = to_f32(base[row * v.ss + col * v.sd]);
        dst[r * GaTile<TS, DP>::LD + col] = x;
    }
}

// acc[i][j] = A[ty R + i] . B[tx + 16 j]
template <int TS, int DP>
__device__ __forceinline__ void dot_rows(float (&acc)[TS / 16][TS / 16], const float* A, const float* B, int ty, int tx) {
    using G = GaTile<TS, DP>;
#pragma unroll
    for (int i = 0; i < G::R; ++i)
#pragma unroll
        for (int j = 0; j < G::R; ++j) acc[i][j] = 0.f;
#pragma unroll 4
    for (int k = 0; k < DP; k += 4) {
        float4 x[G::R], y[G::R];
#pragma unroll
        for (int i = 0; i < G::R; ++i) x[i] = *reinterpret_cast<const float4*>(A + (ty * G::R + i) * G::LD + k);
#pragma unroll
        for (int j = 0; j < G::R; ++j) y[j] = *reinterpret_cast<const float4*>(B + (tx + 16 * j) * G::LD + k);
#pragma unroll
        for (int i = 0; i < G::R; ++i)
#pragma unroll
            for (int j = 0; j < G::R; ++j) {
                acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]);
                acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
                acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]);
                acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
            }
    }
}

// out[i][c] += sum_k W[ty R + i][k] X[k][col(c)]; thread tx owns columns
// 4 tx .. 4 tx + 3 of every 64 (DP = 32: 2 tx, 2 tx + 1)
template <int DP>
__device__ __forceinline__ int out_col(int tx, int c) {
    return DP >= 64 ? tx * 4 + (c / 4) * 64 + c % 4 : tx * 2 + c;
}
template <int TS, int DP>
__device__ __forceinline__ void add_product(float (&out)[TS / 16][DP / 16], const float* W, const float* X, int ty, int tx) {
    using G = GaTile<TS, DP>;
#pragma unroll 2
    for (int k = 0; k < TS; k += 4) {
        float4 w[G::R];
#pragma unroll
        for (int i = 0; i < G::R; ++i) w[i] = *reinterpret_cast<const float4*>(W + (ty * G::R + i) * G::LP + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int c0 = 0; c0 < G::C; c0 += 4) {
                const float4 x = *reinterpret_cast<const float4*>(X + (k + kk) * G::LD + out_col<DP>(tx, c0));
#pragma unroll
                for (int i = 0; i < G::R; ++i) {
                    const float a = kk == 0 ? w[i].x : kk == 1 ? w[i].y : kk == 2 ? w[i].z : w[i].w;
                    out[i][c0] = fmaf(a, x.x, out[i][c0]);
                    out[i][c0 + 1] = fmaf(a, x.y, out[i][c0 + 1]);
                    out[i][c0 + 2] = fmaf(a, x.z, out[i][c0 + 2]);
                    out[i][c0 + 3] = fmaf(a, x.w, out[i][c0 + 3]);
                }
            }
    }
}

template <typename T, int TS, int DP>
__device__ __forceinline__ void store_rows(const HeadsView& v, int b, int h, int row0, int n, int d,
                                           const float (&out)[TS / 16][DP / 16], const float (&mul)[TS / 16], int ty, int tx) {
    T* base = static_cast<T*>(v.p) + b * v.sb + h * v.sh;
#pragma unroll
    for (int i = 0; i < TS / 16; ++i) {
        const int64_t row = row0 + ty * (TS / 16) + i;
        if (row >= n) continue;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
            const int col = out_col<DP>(tx, c);
            if (col < d) base[row * v.ss + col * v.sd] = from_f32<T>(out[i][c] * mul[i]);
        }
    }
}

// The score of a query at position p and a key at j from x = scale q.k; *bend
// is d(score) / dx.
__device__ __forceinline__ float bent_score(float x, float cap, float inv_cap, float slope, int p, int j, float* bend) {
    float y = x;
    *bend = 1.f;
    if (cap > 0.f) {
        const float t = tanhf(x * inv_cap);
        y = cap * t;
        *bend = 1.f - t * t;
    }
    return y - slope * fabsf((float)(p - j));
}

struct RowSet {
    int b, h, g, row0;
};
// block -> (sequence, head of `heads`, tile)
__device__ __forceinline__ RowSet block_rows(int n, int heads, int group, int ts) {
    const unsigned tiles = (n + ts - 1) / ts;
    RowSet r;
    r.row0 = (int)(blockIdx.x % tiles) * ts;
    const unsigned bh = blockIdx.x / tiles;
    r.h = bh % heads;
    r.b = bh / heads;
    r.g = r.h / group;
    return r;
}

template <typename T, int TS, int DP>
__global__ void __launch_bounds__(GA_THREADS) k_attn_general(const __grid_constant__ AttnCall a) {
    using G = GaTile<TS, DP>;
    extern __shared__ __align__(16) float sm[];
    float* Q = sm;
    float* K = Q + TS * G::LD;
    float* V = K + TS * G::LD;
    float* P = V + TS * G::LD;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const RowSet rs = block_rows(a.nq, a.hq, a.hq / a.hkv, TS);
    const SeqMask mask(a, rs.b);
    const int32_t* qd = a.q_doc ? a.q_doc + (int64_t)rs.b * a.nq : nullptr;
    const int32_t* kd = a.k_doc ? a.k_doc + (int64_t)rs.b * a.nk : nullptr;
    const float slope = a.slopes ? a.slopes[rs.h] : 0.f;
    const float inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
    const int kend = mask.key_end(rs.row0, min(TS, a.nq - rs.row0));
    load_rows<T, TS, DP>(Q, a.q, rs.b, rs.h, rs.row0, a.nq, a.d, qd);
    int docs[G::R];
#pragma unroll
    for (int i = 0; i < G::R; ++i) {
        const int row = rs.row0 + ty * G::R + i;
        docs[i] = qd && row < a.nq ? qd[row] : -1;
    }
    float m[G::R], l[G::R], o[G::R][G::C];
#pragma unroll
    for (int i = 0; i < G::R; ++i) {
        m[i] = kNegInf; l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < G::C; ++c) o[i][c] = 0.f;
    }
    for (int j0 = 0; j0 < kend; j0 += TS) {
        __syncthreads();
        load_rows<T, TS, DP>(K, a.k, rs.b, rs.g, j0, mask.kv, a.d, kd);
        load_rows<T, TS, DP>(V, a.v, rs.b, rs.g, j0, mask.kv, a.d, kd);
        __syncthreads();
        float s[G::R][G::R];
        dot_rows<TS, DP>(s, Q, K, ty, tx);
#pragma unroll
        for (int i = 0; i < G::R; ++i) {
            const int row = rs.row0 + ty * G::R + i;
            float top = m[i];
#pragma unroll
            for (int j = 0; j < G::R; ++j) {
                const int key = j0 + tx + 16 * j;
                float bend;
                s[i][j] = bent_score(s[i][j] * a.scale, a.cap, inv_cap, slope, mask.p0 + row, key, &bend);
                const bool seen = mask.sees(row, key) && (!kd || (docs[i] >= 0 && kd[key] == docs[i]));
                s[i][j] = seen ? s[i][j] : kNegInf;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int w = 8; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float safe = top == kNegInf ? 0.f : top;
            const float old = expf(m[i] - safe);
            m[i] = top;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < G::R; ++j) {
                const float p = expf(s[i][j] - safe);
                sum += p;
                P[(ty * G::R + i) * G::LP + tx + 16 * j] = p;
            }
            l[i] = l[i] * old + sum;
#pragma unroll
            for (int c = 0; c < G::C; ++c) o[i][c] *= old;
        }
        __syncthreads();
        add_product<TS, DP>(o, P, V, ty, tx);
    }
    float mul[G::R];
#pragma unroll
    for (int i = 0; i < G::R; ++i) {
#pragma unroll
        for (int w = 8; w; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
        mul[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
        const int row = rs.row0 + ty * G::R + i;
        if (a.lse && tx == 0 && row < a.nq)
            a.lse[((int64_t)rs.b * a.hq + rs.h) * a.nq + row] = l[i] == 0.f ? kNegInf : m[i] + logf(l[i]);
    }
    store_rows<T, TS, DP>(a.o, rs.b, rs.h, rs.row0, a.nq, a.d, o, mul, ty, tx);
}

// D[row] = dout . o, a warp per row; rows of a negative document count as 0.
template <typename T>
__global__ void __launch_bounds__(256) k_attn_delta(const __grid_constant__ AttnCall a, float* __restrict__ delta) {
    const int64_t rows = (int64_t)a.b * a.hq * a.nq;
    const int lane = threadIdx.x & 31;
    for (int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < rows;
         r += ((int64_t)gridDim.x * blockDim.x) >> 5) {
        const int64_t i = r % a.nq, bh = r / a.nq, h = bh % a.hq, b = bh / a.hq;
        float sum = 0.f;
        if (!a.q_doc || a.q_doc[b * a.nq + i] >= 0) {
            const T* x = static_cast<const T*>(a.dout.p) + b * a.dout.sb + h * a.dout.sh + i * a.dout.ss;
            const T* y = static_cast<const T*>(a.o.p) + b * a.o.sb + h * a.o.sh + i * a.o.ss;
            for (int c = lane; c < a.d; c += 32) sum = fmaf(to_f32(x[c * a.dout.sd]), to_f32(y[c * a.o.sd]), sum);
        }
#pragma unroll
        for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if (lane == 0) delta[r] = sum;
    }
}

// p and dx of one (query, key) from q.k and dout.v
__device__ __forceinline__ void grad_scores(const AttnCall& a, const SeqMask& mask, float qk, float dv, float inv_cap,
                                            float slope, int i, int j, bool doc, float lse, float delta, float* p, float* dx) {
    float bend;
    const float s = bent_score(qk * a.scale, a.cap, inv_cap, slope, mask.p0 + i, j, &bend);
    const bool seen = doc && i < a.nq && mask.sees(i, j);
    const float e = expf(s - lse);
    *p = seen ? e : 0.f;
    *dx = seen ? e * (dv - delta) * bend * a.scale : 0.f;
}

template <typename T, int TS, int DP>
__global__ void __launch_bounds__(GA_THREADS) k_attn_general_dq(const __grid_constant__ AttnCall a,
                                                                const float* __restrict__ delta) {
    using G = GaTile<TS, DP>;
    extern __shared__ __align__(16) float sm[];
    float* Q = sm;
    float* O = Q + TS * G::LD;   // dout
    float* K = O + TS * G::LD;
    float* V = K + TS * G::LD;
    float* X = V + TS * G::LD;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const RowSet rs = block_rows(a.nq, a.hq, a.hq / a.hkv, TS);
    const SeqMask mask(a, rs.b);
    const int32_t* qd = a.q_doc ? a.q_doc + (int64_t)rs.b * a.nq : nullptr;
    const int32_t* kd = a.k_doc ? a.k_doc + (int64_t)rs.b * a.nk : nullptr;
    const float slope = a.slopes ? a.slopes[rs.h] : 0.f;
    const float inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
    const int kend = mask.key_end(rs.row0, min(TS, a.nq - rs.row0));
    load_rows<T, TS, DP>(Q, a.q, rs.b, rs.h, rs.row0, a.nq, a.d, qd);
    load_rows<T, TS, DP>(O, a.dout, rs.b, rs.h, rs.row0, a.nq, a.d, qd);
    float lse[G::R], dl[G::R], dq[G::R][G::C], one[G::R];
    int docs[G::R];
#pragma unroll
    for (int i = 0; i < G::R; ++i) {
        const int row = rs.row0 + ty * G::R + i;
        const int64_t at = ((int64_t)rs.b * a.hq + rs.h) * a.nq + row;
        lse[i] = row < a.nq ? a.lse[at] : 0.f;
        dl[i] = row < a.nq ? delta[at] : 0.f;
        docs[i] = qd && row < a.nq ? qd[row] : -1;
        one[i] = 1.f;
#pragma unroll
        for (int c = 0; c < G::C; ++c) dq[i][c] = 0.f;
    }
    for (int j0 = 0; j0 < kend; j0 += TS) {
        __syncthreads();
        load_rows<T, TS, DP>(K, a.k, rs.b, rs.g, j0, mask.kv, a.d, kd);
        load_rows<T, TS, DP>(V, a.v, rs.b, rs.g, j0, mask.kv, a.d, kd);
        __syncthreads();
        float s[G::R][G::R], t[G::R][G::R];
        dot_rows<TS, DP>(s, Q, K, ty, tx);
        dot_rows<TS, DP>(t, O, V, ty, tx);
#pragma unroll
        for (int i = 0; i < G::R; ++i)
#pragma unroll
            for (int j = 0; j < G::R; ++j) {
                const int row = rs.row0 + ty * G::R + i, key = j0 + tx + 16 * j;
                const bool doc = !kd || (key < mask.kv && docs[i] >= 0 && kd[key] == docs[i]);
                float p, dx;
                grad_scores(a, mask, s[i][j], t[i][j], inv_cap, slope, row, key, doc, lse[i], dl[i], &p, &dx);
                X[(ty * G::R + i) * G::LP + tx + 16 * j] = dx;
            }
        __syncthreads();
        add_product<TS, DP>(dq, X, K, ty, tx);
    }
    store_rows<T, TS, DP>(a.dq, rs.b, rs.h, rs.row0, a.nq, a.d, dq, one, ty, tx);
}

template <typename T, int TS, int DP>
__global__ void __launch_bounds__(GA_THREADS) k_attn_general_dkv(const __grid_constant__ AttnCall a,
                                                                 const float* __restrict__ delta) {
    using G = GaTile<TS, DP>;
    extern __shared__ __align__(16) float sm[];
    float* K = sm;
    float* V = K + TS * G::LD;
    float* Q = V + TS * G::LD;
    float* O = Q + TS * G::LD;   // dout
    float* P = O + TS * G::LD;   // p^T, then dx^T
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int group = a.hq / a.hkv;
    const RowSet rs = block_rows(a.nk, a.hkv, 1, TS);
    const SeqMask mask(a, rs.b);
    const int32_t* qd = a.q_doc ? a.q_doc + (int64_t)rs.b * a.nq : nullptr;
    const int32_t* kd = a.k_doc ? a.k_doc + (int64_t)rs.b * a.nk : nullptr;
    const float inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
    load_rows<T, TS, DP>(K, a.k, rs.b, rs.g, rs.row0, mask.kv, a.d, kd);
    load_rows<T, TS, DP>(V, a.v, rs.b, rs.g, rs.row0, mask.kv, a.d, kd);
    float dk[G::R][G::C], dv[G::R][G::C], one[G::R];
    int docs[G::R];
#pragma unroll
    for (int i = 0; i < G::R; ++i) {
        const int key = rs.row0 + ty * G::R + i;
        docs[i] = kd && key < a.nk ? kd[key] : -1;
        one[i] = 1.f;
#pragma unroll
        for (int c = 0; c < G::C; ++c) dk[i][c] = dv[i][c] = 0.f;
    }
    // the first query that may see the tile's first key
    int first = 0;
    if (mask.causal && rs.row0 >= mask.prefix) first = max(0, rs.row0 - mask.p0);
    if (rs.row0 >= mask.kv) first = a.nq;
    for (int h = rs.h * group; h < (rs.h + 1) * group; ++h) {
        const float slope = a.slopes ? a.slopes[h] : 0.f;
        const int64_t at0 = ((int64_t)rs.b * a.hq + h) * a.nq;
        for (int i0 = first / TS * TS; i0 < a.nq; i0 += TS) {
            __syncthreads();
            load_rows<T, TS, DP>(Q, a.q, rs.b, h, i0, a.nq, a.d, qd);
            load_rows<T, TS, DP>(O, a.dout, rs.b, h, i0, a.nq, a.d, qd);
            __syncthreads();
            float s[G::R][G::R], t[G::R][G::R];
            dot_rows<TS, DP>(s, K, Q, ty, tx);
            dot_rows<TS, DP>(t, V, O, ty, tx);
#pragma unroll
            for (int j = 0; j < G::R; ++j) {
                const int row = i0 + tx + 16 * j;
                const float lse = row < a.nq ? a.lse[at0 + row] : 0.f, dl = row < a.nq ? delta[at0 + row] : 0.f;
                const int qdoc = qd && row < a.nq ? qd[row] : -1;
#pragma unroll
                for (int i = 0; i < G::R; ++i) {
                    const int key = rs.row0 + ty * G::R + i;
                    const bool doc = !kd || (qdoc >= 0 && docs[i] == qdoc);
                    float p, dx;
                    grad_scores(a, mask, s[i][j], t[i][j], inv_cap, slope, row, key, doc, lse, dl, &p, &dx);
                    P[(ty * G::R + i) * G::LP + tx + 16 * j] = p;
                    s[i][j] = dx;
                }
            }
            __syncthreads();
            add_product<TS, DP>(dv, P, O, ty, tx);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < G::R; ++i)
#pragma unroll
                for (int j = 0; j < G::R; ++j) P[(ty * G::R + i) * G::LP + tx + 16 * j] = s[i][j];
            __syncthreads();
            add_product<TS, DP>(dk, P, Q, ty, tx);
        }
    }
    store_rows<T, TS, DP>(a.dk, rs.b, rs.h, rs.row0, a.nk, a.d, dk, one, ty, tx);
    store_rows<T, TS, DP>(a.dv, rs.b, rs.h, rs.row0, a.nk, a.d, dv, one, ty, tx);
}

unsigned blocks(int64_t bh, int n, int ts) { return (unsigned)(bh * ((n + ts - 1) / ts)); }

template <typename T, int TS, int DP>
tl_status forward(tl_ctx* c, const AttnCall& a, cudaStream_t s) {
    using G = GaTile<TS, DP>;
    constexpr int smem = 3 * G::OPERAND + G::SCORES;
    static std::atomic<uint64_t> done{0};
    TL_TRY(kernel_smem(c, k_attn_general<T, TS, DP>, smem, done));
    cudaEvent_t ev[2];
    launch_begin_on(c, s, "attention_general", 0, 4.0 * a.d * attn_pairs(a), ev);
    k_attn_general<T, TS, DP><<<blocks((int64_t)a.b * a.hq, a.nq, TS), GA_THREADS, smem, s>>>(a);
    return launch_end_on(c, s, ev);
}

template <typename T, int TS, int DP>
tl_status backward(tl_ctx* c, const AttnCall& a, float* delta, cudaStream_t s) {
    using G = GaTile<TS, DP>;
    constexpr int smem = 4 * G::OPERAND + G::SCORES;
    static std::atomic<uint64_t> done_q{0}, done_kv{0};
    TL_TRY(kernel_smem(c, k_attn_general_dq<T, TS, DP>, smem, done_q));
    TL_TRY(kernel_smem(c, k_attn_general_dkv<T, TS, DP>, smem, done_kv));
    const int64_t rows = (int64_t)a.b * a.hq * a.nq;
    cudaEvent_t ev[2];
    if (rows > 0) {
        launch_begin_on(c, s, "attention_delta", 2.0 * rows * a.d * sizeof(T), 2.0 * rows * a.d, ev);
        k_attn_delta<T><<<(unsigned)std::min<int64_t>((rows + 7) / 8, 148 * 16), 256, 0, s>>>(a, delta);
        TL_TRY(launch_end_on(c, s, ev));
        launch_begin_on(c, s, "attention_general_dq", 0, 6.0 * a.d * attn_pairs(a), ev);
        k_attn_general_dq<T, TS, DP><<<blocks((int64_t)a.b * a.hq, a.nq, TS), GA_THREADS, smem, s>>>(a, delta);
        TL_TRY(launch_end_on(c, s, ev));
    }
    if (a.nk > 0) {
        launch_begin_on(c, s, "attention_general_dkv", 0, 8.0 * a.d * attn_pairs(a), ev);
        k_attn_general_dkv<T, TS, DP><<<blocks((int64_t)a.b * a.hkv, a.nk, TS), GA_THREADS, smem, s>>>(a, delta);
        TL_TRY(launch_end_on(c, s, ev));
    }
    return TL_OK;
}

template <typename F>
tl_status by_type_and_size(const AttnCall& a, F f) {
    auto size = [&](auto t) {
        if (a.d <= 64) return f(t, std::integral_constant<int, 64>(), std::integral_constant<int, 64>());
        if (a.d <= 128) return f(t, std::integral_constant<int, 64>(), std::integral_constant<int, 128>());
        return f(t, std::integral_constant<int, 32>(), std::integral_constant<int, 256>());
    };
    switch (a.dtype) {
    case TL_TYPE_F32: return size(float());
    case TL_TYPE_F16: return size(__half());
    default: return size(__nv_bfloat16());
    }
}

}  // namespace

// backward: D of every query row
size_t attn_general_workspace(const AttnCall& a, bool backward) {
    return backward ? (size_t)a.b * a.hq * a.nq * sizeof(float) : 0;
}

tl_status launch_attn_general(tl_ctx* c, const AttnCall& a, void*, cudaStream_t s) {
    return by_type_and_size(a, [&](auto t, auto ts, auto dp) {
        return forward<decltype(t), decltype(ts)::value, decltype(dp)::value>(c, a, s);
    });
}

tl_status launch_attn_general_backward(tl_ctx* c, const AttnCall& a, void* ws, cudaStream_t s) {
    return by_type_and_size(a, [&](auto t, auto ts, auto dp) {
        return backward<decltype(t), decltype(ts)::value, decltype(dp)::value>(c, a, static_cast<float*>(ws), s);
    });
}

}  // namespace tl
