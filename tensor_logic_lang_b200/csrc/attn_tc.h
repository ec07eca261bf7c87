// Device pieces shared by the tensor-core attention kernels (16-bit operands,
// head size up to 128; fp32 arrays of such head sizes as pairs of fp16).
//
// Operand tiles are 128 rows of one head in shared memory as one or two
// chunks of 64 columns (16 KB each, 128-byte swizzle), which TMA writes from a
// [batch, heads, positions, head size] tensor map; rows past the array and
// columns past the head size arrive as zeros.  The same tile is a K-major
// operand (the head size contracted: q k^T, dout v^T) and an MN-major one (the
// rows contracted: p v, dx k, p^T dout, dx^T q).
#pragma once

#include <float.h>

#include "attention.h"
#include "tc_ptx.h"

namespace tl {

constexpr int TILE = 128;                 // queries or keys of a tile
constexpr int CHUNK_BYTES = TILE * 128;   // 64 columns of a tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// fp16 probabilities are written 2^6 times larger: the smallest ones keep
// more bits (fp16 ends at 2^-24), and with the lazy rescaling's 2^8 they stay
// below 2^15.
template <typename T> struct Lift { static constexpr float log2 = 0.f; };
template <> struct Lift<__half> { static constexpr float log2 = 6.f; };

// ---------------------------------------------------------------- packed fp32
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(f2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <typename T> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// 2^e, of e in fp32's normal numbers (their ends beyond)
__device__ __forceinline__ float pow2(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }

// a value >= 0, or 0 for one that is not finite: a power of two taken from the largest of many then stays
// that of the others
__device__ __forceinline__ float finite(float x) { return x <= FLT_MAX ? x : 0.f; }

// ---------------------------------------------------------------- tcgen05
// One lane of a converged warp.  ptxas knows that the branch it guards has one
// thread and keeps descriptors in uniform registers there (a branch on the lane
// number costs about 90 cycles an MMA, more than the MMA).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p)::"memory");
    return p != 0;
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes; the values are there after tmem_wait_ld
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// Instruction descriptor of kind::f16: fp32 sums, A and B of one 16-bit type,
// A K-major, M = 128.
template <typename T>
__device__ __forceinline__ constexpr uint32_t f16_idesc(int n, bool b_mn) {
    const uint32_t t = TypeOf<T>::id == TL_TYPE_BF16 ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(TILE >> 4) << 24);
}
// The MMA warp shares its scheduler with the warps that compute, so every
// instruction it needs beside tcgen05.mma delays the tensor cores: descriptors
// differ only in the address field of their low word (16-byte units, below
// 2^14, no carry), and each MMA costs one addition to it.  (In a cluster a
// shared address carries the block's rank above these bits.)
constexpr uint32_t kDescRows = 1024 >> 4;   // high word without the version and the swizzle: 8 rows (SBO)
constexpr uint32_t kDescHigh = kDescRows | (1u << 14) | (2u << 29);   // version 1, 128-byte swizzle
__device__ __forceinline__ uint32_t desc_rows(uint32_t saddr) { return ((saddr >> 4) & 0x3FFF) | (1u << 16); }   // K-major (LBO unused)
__device__ __forceinline__ uint32_t desc_cols(uint32_t saddr) { return ((saddr >> 4) & 0x3FFF) | ((CHUNK_BYTES >> 4) << 16); }   // MN-major: LBO to the next 64 columns
template <bool ACC>
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
        "mov.b64 x, {%1, %4};\n\tmov.b64 y, {%2, %4};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "n"(kDescHigh), "n"(ACC ? 1 : 0));
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\t"
        "mov.b64 y, {%2, %4};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "n"(kDescHigh), "r"(accumulate));
}

// D[128 x 128] = A B^T over the head size (ksteps of 16, at most N), both
// K-major tiles.  N steps, all of them of the largest head size, are unrolled.
template <typename T, int N>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b, int ksteps) {
    constexpr uint32_t idesc = f16_idesc<T>(TILE, false);
    const uint32_t da = desc_rows(a), db = desc_rows(b);
    auto at = [](int k) { return (uint32_t)((k / 4) * (CHUNK_BYTES >> 4) + (k % 4) * 2); };
    umma_f16_ss<false>(d, da, db, idesc);
    if (ksteps == N) {
#pragma unroll
        for (int k = 1; k < N; ++k) umma_f16_ss<true>(d, da + at(k), db + at(k), idesc);
    } else {
        for (int k = 1; k < ksteps; ++k) umma_f16_ss<true>(d, da + at(k), db + at(k), idesc);
    }
}
// The same with operands in two parts (x = hi + lo, see SplitPlan): chunk 0 of a
// tile holds hi, chunk 1 lo.  lo hi + hi lo + hi hi; lo lo, 2^-22 of the
// product, is left out.  The small products go first: the tensor cores cut
// their fp32 sums (2^-23 of the sum a step), so the large sum should see few
// steps.
// MORE: added to D.
template <typename T, bool MORE = false>
__device__ __forceinline__ void mma_rows_split(uint32_t d, uint32_t a, uint32_t b, int ksteps) {
    constexpr uint32_t idesc = f16_idesc<T>(TILE, false), low = CHUNK_BYTES >> 4;
    const uint32_t da = desc_rows(a), db = desc_rows(b);
    umma_f16_ss<MORE>(d, da + low, db, idesc);
    if (ksteps == 4) {
#pragma unroll
        for (int k = 1; k < 4; ++k) umma_f16_ss<true>(d, da + low + 2 * k, db + 2 * k, idesc);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f16_ss<true>(d, da + 2 * k, db + low + 2 * k, idesc);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f16_ss<true>(d, da + 2 * k, db + 2 * k, idesc);
    } else {
        for (int k = 1; k < ksteps; ++k) umma_f16_ss<true>(d, da + low + 2 * k, db + 2 * k, idesc);
        for (int k = 0; k < ksteps; ++k) umma_f16_ss<true>(d, da + 2 * k, db + low + 2 * k, idesc);
        for (int k = 0; k < ksteps; ++k) umma_f16_ss<true>(d, da + 2 * k, db + 2 * k, idesc);
    }
}
// D[128 x n] (+)= A B: A 128 x 128 16-bit in TMEM, in parts of W columns (W / 2
// TMEM columns each, W apart: each over the fp32 scores it comes from), B the
// tile's 128 rows as contracted index.
template <int W>
__device__ __forceinline__ constexpr uint32_t part_col(int k) { return (16 * k / W) * W + (16 * k % W) / 2; }
template <int W>
__device__ __forceinline__ void mma_parts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    const uint32_t db = desc_cols(b);
    umma_f16_ts(d, a, db, idesc, accumulate);
#pragma unroll
    for (int k = 1; k < TILE / 16; ++k) umma_f16_ts(d, a + part_col<W>(k), db + k * (2048 >> 4), idesc, 1);
}
// The same for split operands (the caller adds the tiles up in fp32): in each
// part's W TMEM columns W / 2 of hi, W / 2 of lo.
template <int W>
__device__ __forceinline__ void mma_parts_split(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    const uint32_t db = desc_cols(b);
#pragma unroll
    for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int k = 0; k < TILE / 16; ++k)
            umma_f16_ts(d, a + part_col<W>(k) + (part == 0 ? W / 2 : 0), db + (part == 1 ? CHUNK_BYTES >> 4 : 0) + k * (2048 >> 4), idesc,
                        part > 0 || k > 0 ? 1u : accumulate);
}
// N columns of the warp's lanes
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&raw)[N]) {
#pragma unroll
    for (int k = 0; k < N / 32; ++k) tmem_ld32(taddr + 32 * k, raw + 32 * k);
    tmem_wait_ld();
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, f2 (&x)[N]) {
    uint32_t raw[2 * N];
    tmem_load(taddr, raw);
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = pack2(__uint_as_float(raw[2 * k]), __uint_as_float(raw[2 * k + 1]));
}
// hi and lo of a pair of values as fp16 pairs
__device__ __forceinline__ void split16(float a, float b, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(b), "f"(a));
    const __half2 h = *reinterpret_cast<const __half2*>(&hi);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(b - __high2float(h)), "f"(a - __low2float(h)));
}
// N TMEM columns at acc = columns at `from` + (fresh: 0, else what is there)
template <int N>
__device__ __forceinline__ void tmem_add(uint32_t acc, uint32_t from, bool fresh) {
#pragma unroll 1
    for (int k = 0; k < N; k += 16) {
        uint32_t x[16], y[16];
        tmem_ld16(from + k, x);
        if (!fresh) tmem_ld16(acc + k, y);
        tmem_wait_ld();
        if (!fresh)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) + __uint_as_float(y[i]));
        tmem_st16(acc + k, x);
    }
}

// A row of DP fp32 sums in TMEM, scaled (by mul and then by post, of fp32 arrays, whose product may pass fp32), as
// values of an array: 16-bit rows are 16-byte aligned (tc_array), fp32 ones may lie anyhow.  any: there are sums
// (else zeros); live: the columns may be read (the same for the whole warp).
template <typename U, int DP>
__device__ __forceinline__ void store_row(const HeadsView& v, int b, int h, int64_t row, bool on, int d, uint32_t taddr, bool any,
                                          bool live, float mul, float post = 1.f) {
    U* p = static_cast<U*>(v.p) + b * v.sb + h * v.sh + row * v.ss;
    const bool wide = std::is_same<U, float>::value && v.sd == 1 && d % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int k = 0; k < DP / 16; ++k) {
        uint32_t o[16];
        if (live) {
            tmem_ld16(taddr + 16 * k, o);
            tmem_wait_ld();
        }
        if (!on) continue;
        if constexpr (std::is_same<U, float>::value) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = 16 * k + 4 * q;
                if (c >= d) break;
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = any ? __uint_as_float(o[4 * q + e]) * mul * post : 0.f;
                if (wide) {
                    *reinterpret_cast<float4*>(p + c) = make_float4(w[0], w[1], w[2], w[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < d) p[(c + e) * v.sd] = w[e];
                }
            }
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (16 * k + 8 * q >= d) break;
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = any ? pack16<U>(__uint_as_float(o[8 * q + 2 * e]) * mul, __uint_as_float(o[8 * q + 2 * e + 1]) * mul) : 0u;
                *reinterpret_cast<uint4*>(p + 16 * k + 8 * q) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

// ---------------------------------------------------------------- TMA
// One head's rows in a 4-D map; strides of 0 and dims of 1 take coordinate 0.
struct HeadMap {
    CUtensorMap map;
    int mh, mb;   // 1, or 0 where every head (sequence) is the same memory
};
__device__ __forceinline__ void tma_tile(uint32_t dst, const HeadMap& m, uint64_t* bar, int chunks, int row, int h, int b, int first = 0) {
    for (int c = 0; c < chunks; ++c)
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
            ::"r"(dst + c * CHUNK_BYTES),
            "l"(reinterpret_cast<uint64_t>(&m.map)), "r"(smem_u32(bar)), "r"(64 * (first + c)), "r"(row), "r"(h * m.mh), "r"(b * m.mb)
            : "memory");
}

// ---------------------------------------------------------------- capped scores
// softcap tanh(x / softcap) as x P((x / softcap)^2), where P has the least
// largest relative error for tanh(u) / u over the range (a linear programme
// over a Chebyshev grid gives it).  16-bit probabilities: |u| <= 0.75, degree 3,
// 1.1e-5, far below the rounding of p.  Fp32: |u| <= 0.625, degree 5, 3.9e-9, below
// the rounding of fp32.  Tiles that hold a larger score take tanh u =
// 1 - 2 / (1 + e^2u), which is off by 1.2e-7 of 1, so its scores by 1.2e-7 of the
// cap: fp32, and 16-bit types where that counts beside P's error (top above
// kFarTop), take it for the larger scores alone, 16-bit types with small caps for
// all of the tile.
template <bool FINE>
__device__ __forceinline__ constexpr float tanh_coef(int i) {
    if (FINE)
        return i == 0 ? 1.0f : i == 1 ? -0.3333325982093811f : i == 2 ? 0.13331125676631927f : i == 3 ? -0.053720925003290176f
               : i == 4 ? 0.020590508356690407f : -0.00565946102142334f;
    return i == 0 ? 0.9999889731407166f : i == 1 ? -0.33269670605659485f : i == 2 ? 0.12742698192596436f : -0.035452794283628464f;
}

constexpr float kFarTop = 128.f;
template <bool FINE>
struct CapCoef {
    static constexpr int N = FINE ? 5 : 3;
    float limit;       // largest |q.k| of the polynomial
    float k2;          // (scale / softcap)^2; fp32
    float mul;         // scale log2 e; fp32
    float wide;        // 2 log2(e) scale / softcap: 2u in base 2
    float top;         // softcap log2 e
    float c[N + 1];    // 16-bit: P's coefficients times scale log2(e) k2^i
    __device__ __forceinline__ CapCoef(float scale, float cap) {
        // split operands have scales of any size; their products are 0 or above 2^-48, so 2^63 bends alike
        const float u = FINE ? fminf(scale / cap, 0x1p63f) : scale / cap;
        k2 = u * u;
        mul = scale * kLog2e;
        wide = FINE ? 2.f * kLog2e * u : 2.f * kLog2e * scale / cap;
        top = cap * kLog2e;
        float f = FINE ? 1.f : mul;
#pragma unroll
        for (int i = 0; i <= N; ++i) {
            c[i] = tanh_coef<FINE>(i) * f;
            if (!FINE) f *= k2;
        }
        // 16-bit: a coefficient below fp32's normal numbers (scale much smaller than
        // the cap) is left out, and the polynomial ends where its term is 1e-6 of the score
        float end = FINE ? 0.625f : 0.75f;
        if (!FINE) {
#pragma unroll
            for (int i = N; i >= 1; --i)
                if (fabsf(c[i]) < 0x1p-126f) {
                    c[i] = 0.f;
                    end = i == 3 ? 0.1f : i == 2 ? 0.05f : 1e-3f;
                }
        }
        limit = fabsf(c[N]) < 3e38f ? end * (cap / scale) : -1.f;   // out of range: never the polynomial
    }
    // score / x in base 2 of a pair within the limit
    __device__ __forceinline__ f2 ratio(f2 x) const {
        f2 z = mul2(x, x);
        if (FINE) z = mul2(z, pack2(k2, k2));
        f2 r = pack2(c[N], c[N]);
#pragma unroll
        for (int i = N - 1; i >= 0; --i) r = fma2(r, z, pack2(c[i], c[i]));
        return FINE ? mul2(r, pack2(mul, mul)) : r;
    }
};
__device__ __forceinline__ float wide_tanh(float x, float wide) { return 1.f - __fdividef(2.f, 1.f + ex2(x * wide)); }
// The largest |score| of a row.
template <int N>
__device__ __forceinline__ float largest(const f2 (&x)[N]) {
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float lo, hi;
        unpack2(x[i], lo, hi);
        big = fmaxf(big, fmaxf(fabsf(lo), fabsf(hi)));
    }
    return big;
}
// 16-bit calls whose cap is far above the scores take the kernels with slopes, of 0 where there are none: the code for
// both forms in one tile costs the others 1 to 4 % (backward, 16 x 2048 x 128 over 4, cap 30: 113.1 us, 115.5 with it).
inline bool takes_slopes(const AttnCall& a) { return a.slopes || (a.dtype != TL_TYPE_F32 && a.cap * kLog2e > kFarTop); }
// The score in base 2 of a pair in a tile with scores past the limit; EACH: those within
// it take the polynomial.
template <bool EACH, bool FINE>
__device__ __forceinline__ f2 wide_score(f2 x, const CapCoef<FINE>& cap) {
    float lo, hi;
    unpack2(x, lo, hi);
    float y = cap.top * wide_tanh(lo, cap.wide), z = cap.top * wide_tanh(hi, cap.wide);
    if (EACH) {
        float a, b;
        unpack2(mul2(x, cap.ratio(x)), a, b);
        y = fabsf(lo) <= cap.limit ? a : y;
        z = fabsf(hi) <= cap.limit ? b : z;
    }
    return pack2(y, z);
}
// The scores in base 2 of a row, in place; one choice for all of a warp's rows.
// FAR: caps above kFarTop come here too.
template <bool FAR, bool FINE, int N>
__device__ __forceinline__ void cap_scores(f2 (&x)[N], const CapCoef<FINE>& cap) {
    if (!__any_sync(0xffffffffu, !(largest(x) <= cap.limit))) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = mul2(x[i], cap.ratio(x[i]));
    } else if (FINE || (FAR && cap.top > kFarTop)) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = wide_score<true>(x[i], cap);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = wide_score<false>(x[i], cap);
    }
}

// ---------------------------------------------------------------- documents
// Smallest and largest document of a tile of positions (padding apart: none
// gives lo > hi), and whether it holds padding.
struct DocRange {
    int lo, hi, pad, _unused;
};
__device__ __forceinline__ DocRange no_docs() { return {0x7fffffff, -1, 0, 0}; }
__device__ __forceinline__ bool docs_meet(const DocRange& a, const DocRange& b) { return a.lo <= b.hi && b.lo <= a.hi && a.lo <= a.hi && b.lo <= b.hi; }
__device__ __forceinline__ bool docs_one(const DocRange& a, const DocRange& b) { return a.lo == a.hi && b.lo == b.hi && a.lo == b.lo && !a.pad && !b.pad; }

// The tiles of [begin, end) that a block has to visit, 32 at a time: ballots
// over a lane per tile.  Every warp of a block walks the same list.
template <bool PART = false>
struct TileWalk {
    int base, end;
    int clear_lo, clear_hi;       // tiles within need no mask of positions
    const DocRange* ranges;       // documents of the tiles, or null
    DocRange mine;                // documents of the block's own rows
    uint32_t active, masked;
    int lane;
    uint32_t ours;                // PART: every `parts`-th tile, of 32 from base on
    __device__ __forceinline__ void fill() {
        const int t = base + lane;
        bool on = t < end, mk = t < clear_lo || t >= clear_hi;
        if (ranges && on) {
            const int4 r4 = __ldg(reinterpret_cast<const int4*>(ranges) + t);
            const DocRange r = {r4.x, r4.y, r4.z, 0};
            on = docs_meet(mine, r);
            mk = mk || !docs_one(mine, r);
        }
        active = __ballot_sync(0xffffffffu, on);
        if (PART) active &= ours;
        masked = __ballot_sync(0xffffffffu, mk);
    }
    __device__ __forceinline__ void start(int begin, int end_, int lo, int hi, const DocRange* r, const DocRange& m, int parts = 1,
                                          int part = 0) {
        base = begin; end = end_; clear_lo = lo; clear_hi = hi; ranges = r; mine = m;
        lane = threadIdx.x & 31;
        if (PART) ours = __ballot_sync(0xffffffffu, ((begin + lane) & (parts - 1)) == part);   // parts divides 32
        active = masked = 0;
        if (base < end) fill();
    }
    // the next tile (-1: none), by all lanes of a warp together
    __device__ __forceinline__ int next(bool* mask) {
        while (!active) {
            base += 32;
            if (base >= end) return -1;
            fill();
        }
        const int bit = __ffs(active) - 1;
        active &= active - 1;
        *mask = (masked >> bit) & 1;
        return base + bit;
    }
};

// Registers of a warpgroup, from those that the block was launched with: the
// warpgroup of the MMA and TMA warps leaves what its two need not.
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// an address of this block's shared memory, in block `rank` of the cluster
__device__ __forceinline__ uint32_t in_block(uint32_t saddr, int rank) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(saddr), "r"(rank));
    return at;
}
__device__ __forceinline__ void load_cluster4(uint32_t at, float (&x)[4]) {
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(at));
}

// Bits of 32 W other positions whose document is `doc`, lane by lane: the lane
// holds the documents of positions lane, 32 + lane, ... in other[W] and wants
// its own row's doc.  The distinct documents of a warp's rows are few (W
// ballots each).
template <int W>
__device__ __forceinline__ void doc_bits(const int (&other)[W], int doc, uint32_t (&bits)[W]) {
    uint32_t left = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < W; ++w) bits[w] = 0;
    while (left) {
        const int d = __shfl_sync(0xffffffffu, doc, __ffs(left) - 1);
        const bool mine = doc == d;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const uint32_t m = __ballot_sync(0xffffffffu, other[w] == d && d >= 0);
            if (mine) bits[w] = m;
        }
        left &= ~__ballot_sync(0xffffffffu, mine);
    }
}
// the low n bits of word w of a row
__device__ __forceinline__ uint32_t low_bits(int n, int w) {
    const int k = n - 32 * w;
    return k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1;
}

// Zeros over the rows of a tile that must not count (a warp; the caller
// fences before the tensor cores read the tile).
template <typename F>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int chunks, F bad) {
    const int lane = threadIdx.x & 31;
    for (int r = lane; r < TILE; r += 32)
        if (bad(r))
            for (int c = 0; c < chunks; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    *reinterpret_cast<uint4*>(tile + c * CHUNK_BYTES + r * 128 + 16 * k) = make_uint4(0, 0, 0, 0);
}

// host: the tensor map of one array (k_attention_tc.cu)
bool make_head_map(HeadMap* m, const HeadsView& v, int dtype, int b, int h, int64_t n, int d, int box_rows = TILE, int box_heads = 1);
// the arrays a tensor-core kernel takes: 16-bit, head size contiguous, 16-byte
// aligned rows
bool tc_array(const HeadsView& v, int b, int h, int64_t n);
// fp32 arrays on the tensor cores (k_attention_split.cu).  A value times a
// power of two of its key head's group (the largest of these heads then lies
// in 2^14 .. 2^15) is hi + lo, two fp16 numbers of 11 bits: 22 bits of it, or 2^-25
// where that is more, which is 2^-39 of the largest.  One array:
// [b, h, n, 128] fp16, columns 0..63 hi, 64..127 lo, zeros past the head size and in
// rows that must not count; head sizes above 64 have two such halves behind one
// another, [b, h, n, 256].
constexpr int kSplitMaxHead = 128;
inline int split_width(int d) { return d <= 64 ? 128 : 256; }
struct SplitArray {
    HeadsView v;
    int h, n;
    bool keys;          // rows count below kv_len and in documents of k_doc (else of q_doc)
    int norm;           // largest row norm^2, of what out holds, into norms[2 * (b * hkv + key head) + norm]; -1: none
    __half* out;
    uint32_t* top;      // [b, hkv] largest |x| of the group's heads as bits
};
struct SplitPlan {
    size_t top, norms, data[4], bytes;   // of q, k, v, dout (backward)
    SplitPlan(const AttnCall& a, bool backward);
};
// queues the splitting, and launch_attn_begin for the ranges; maps: q, k, v, dout;
// stats: of the backward pass, null in a forward one
tl_status launch_split(tl_ctx* c, const AttnCall& a, float* stats, uint8_t* ws, HeadMap* maps, DocRange* q_ranges, DocRange* k_ranges,
                       cudaStream_t s);
// the power of two of a group, from its largest value (below 2^-112, where fp32 itself ends, it stays smaller)
__device__ __forceinline__ int split_exp(const uint32_t* top, int group) {
    const float m = __uint_as_float(top[group]);
    if (!(m > 0.f)) return 0;
    return min(14 - ilogbf(m), 126);
}
// the scale of scores whose operands carry the powers of two e together.  Within 2^-126 .. 2^126 whatever they
// are: products of split operands, below 2^37, are scores of 0 at the lower end, and pass fp32 past the upper one
__device__ __forceinline__ float split_scale(float scale, int e) {
    return fminf(fmaxf(scale * pow2(-e / 2) * pow2(-e - -e / 2), 0x1p-126f), 0x1p126f);
}
struct SplitTops {
    const uint32_t *q, *k, *v, *dout;    // null: operands are the arrays themselves
};

// the documents' ranges of the query and key tiles (null: not wanted), and zeros
tl_status launch_attn_begin(tl_ctx* c, const AttnCall& a, DocRange* q_out, DocRange* k_out, uint32_t* zero, int64_t words,
                            cudaStream_t s);

// ---------------------------------------------------------------- backward
// of a query tile: -log2(e) lse (+ lift), -D
constexpr int STAT_BYTES = 2 * TILE * 4;
template <typename T> struct PLift { static constexpr float log2 = 0.f, back = 1.f; };
template <> struct PLift<__half> { static constexpr float log2 = 14.f, back = 1.f / 16384.f; };

}  // namespace tl
