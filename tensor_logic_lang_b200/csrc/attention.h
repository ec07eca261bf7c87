// Internal declarations of the attention and gradient-clipping operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "tl_internal.h"

namespace tl {

// [batch, heads, positions, head size] with strides in elements
struct HeadsView {
    void* p;
    int64_t sb, sh, ss, sd;
};

// One checked attention call (tl_attention with its sizes taken out).
struct AttnCall {
    int dtype;                    // TL_TYPE_*
    int b, hq, hkv, nq, nk, d;
    HeadsView q, k, v, o, dout, dq, dk, dv;
    float* lse;                   // [b, hq, nq]
    float scale, cap;
    int causal;
    int cuda_cores;               // fp32 arrays of a TL_PREC_FP32 context: no tensor cores
    const float* slopes;
    const int32_t *prefix_len, *q_doc, *k_doc, *kv_len, *q_start;
};

// Which keys the queries of one sequence see.  Positions fit 32 bits: counts
// are at most 2^29 and q_start is clamped to +-2^30.
struct SeqMask {
    int kv;        // keys of the sequence
    int p0;        // position of query 0
    int prefix;    // keys every query of a causal call sees
    int causal;
    __device__ __forceinline__ SeqMask(const AttnCall& a, int b) {
        kv = a.kv_len ? min(max(__ldg(a.kv_len + b), 0), a.nk) : a.nk;
        p0 = a.q_start ? min(max(__ldg(a.q_start + b), -(1 << 30)), 1 << 30) : kv - a.nq;
        causal = a.causal;
        prefix = a.prefix_len ? __ldg(a.prefix_len + b) : 0;
    }
    // keys before this one may be seen by some query of [i0, i0 + n)
    __device__ __forceinline__ int key_end(int i0, int n) const {
        return causal ? min(kv, max(p0 + i0 + n, prefix)) : kv;
    }
    __device__ __forceinline__ bool sees(int i, int j) const {
        return j < kv && (!causal || j <= p0 + i || j < prefix);
    }
};

template <typename T> struct TypeOf;
template <> struct TypeOf<float> { static constexpr int id = TL_TYPE_F32; };
template <> struct TypeOf<__half> { static constexpr int id = TL_TYPE_F16; };
template <> struct TypeOf<__nv_bfloat16> { static constexpr int id = TL_TYPE_BF16; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// The kernel's dynamic shared memory limit, raised once per device (not in
// every call: the attribute may not be set in a capture).  regs: registers a thread that a
// kernel which divides them anew (setmaxnreg) must be launched with; a split that sums up to
// more would wait for ever, so another compiler's kernel is not launched (kNoSplit), and the general kernel takes the
// call.
constexpr tl_status kNoSplit = -1;
template <typename F>
tl_status kernel_smem(tl_ctx* c, F* kernel, int bytes, std::atomic<uint64_t>& done, int regs = 0) {
    const uint64_t bit = uint64_t(1) << (c->device & 63);
    if (c->device < 64 && (done.load() & bit)) return TL_OK;
    TL_CK(c, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (regs) {
        cudaFuncAttributes attr;
        TL_CK(c, cudaFuncGetAttributes(&attr, kernel));
        if ((attr.numRegs + 7) / 8 * 8 != regs) return kNoSplit;   // they are given out by eight
    }
    if (c->device < 64) done.fetch_or(bit);
    return TL_OK;
}

// A launch in clusters of `cluster` blocks along x.  early: its blocks may start
// when every block of the kernel before it in the stream has said
// griddepcontrol.launch_dependents or ended; they wait for its results with
// griddepcontrol.wait.
template <typename... P, typename... A>
cudaError_t launch_with(void (*kernel)(P...), dim3 grid, int cluster, int threads, int smem, bool early, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (early) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

inline size_t type_size(int dtype) { return dtype == TL_TYPE_F32 ? 4 : 2; }

// algorithmic work of a call for the profile: every pair of a query and a key
// it may see by the causal rule alone
double attn_pairs(const AttnCall& a);

// k_attention.cu: any type, strides and head size up to 256, fp32 arithmetic
constexpr int kAttnMaxHead = 256;
size_t attn_general_workspace(const AttnCall& a, bool backward);
tl_status launch_attn_general(tl_ctx* c, const AttnCall& a, void* ws, cudaStream_t s);
tl_status launch_attn_general_backward(tl_ctx* c, const AttnCall& a, void* ws, cudaStream_t s);

// k_attention_tc.cu: 16-bit types with aligned rows, and fp32, of head size up to 128
bool attn_tc_takes(const AttnCall& a);
size_t attn_tc_workspace(const AttnCall& a);
tl_status launch_attn_tc(tl_ctx* c, const AttnCall& a, void* ws, cudaStream_t s);

// k_attention_tc_bwd.cu
bool attn_tc_backward_takes(const AttnCall& a);
size_t attn_tc_backward_workspace(const AttnCall& a);
tl_status launch_attn_tc_backward(tl_ctx* c, const AttnCall& a, void* ws, cudaStream_t s);

// k_attention_decode.cu: few queries over many keys, any type
bool attn_few_takes(const AttnCall& a);
size_t attn_few_workspace(const AttnCall& a);
tl_status launch_attn_few(tl_ctx* c, const AttnCall& a, void* ws, cudaStream_t s);

// k_clip.cu
struct ClipItem {
    const void* in;
    void* out;
    int64_t n;
    int in_type, out_type;
};
size_t clip_workspace_bytes();
tl_status launch_clip(tl_ctx* c, const std::vector<ClipItem>& items, double max_norm, float* norm, void* ws,
                      cudaStream_t s);

}  // namespace tl
