// Entry points of the array operators (include/tl_cuda.h: tl_tensor_array,
// tl_attention_*, tl_clip_*): argument checks, streams, workspaces, dispatch.
// Arguments are checked before any device work.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "attention.h"

namespace tl {
namespace {

constexpr int64_t kMaxCount = int64_t(1) << 29;   // positions, heads, batch
constexpr size_t kMaxStreams = 16;

// The context's device is current while a call runs.
struct DeviceGuard {
    int prev = -1;
    bool ok;
    explicit DeviceGuard(int dev) {
        ok = cudaGetDevice(&prev) == cudaSuccess;
        if (ok && prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
        else if (ok) prev = -1;
    }
    ~DeviceGuard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

// No exception leaves a C entry.
template <typename R, typename F>
R entry(tl_ctx* c, R oom, F f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        try { fail(c, TL_ERR_OOM, "out of host memory"); } catch (...) {}
        return oom;
    } catch (...) {
        return oom;
    }
}

// *capturing: the stream is in capture, where a stream's device may not be
// asked for (a launch on a stream of another device fails by itself).
tl_status check_stream(tl_ctx* c, cudaStream_t s, bool* capturing) {
    *capturing = false;
    if (!s || s == cudaStreamLegacy) return TL_OK;   // the current device's, never in capture
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    TL_CK(c, cudaStreamIsCapturing(s, &cap));
    *capturing = cap != cudaStreamCaptureStatusNone;
    if (*capturing || s == cudaStreamPerThread) return TL_OK;
    int dev = -1;
    TL_CK(c, cudaStreamGetDevice(s, &dev));
    if (dev != c->device) return fail(c, TL_ERR_INVALID, "the stream belongs to device %d, the context to %d", dev, c->device);
    return TL_OK;
}

// Scratch of a call: the caller's, or the context's buffer for the stream.
tl_status op_workspace(tl_ctx* c, cudaStream_t s, bool capturing, size_t need, void* given, int64_t given_bytes, void** out) {
    *out = nullptr;
    if (need == 0) return TL_OK;
    if (given) {
        if (given_bytes < 0 || (size_t)given_bytes < need)
            return fail(c, TL_ERR_INVALID, "workspace of %lld bytes, %zu are needed", (long long)given_bytes, need);
        if (reinterpret_cast<uintptr_t>(given) % 256) return fail(c, TL_ERR_INVALID, "workspace is not 256-byte aligned");
        *out = given;
        return TL_OK;
    }
    if (s == cudaStreamPerThread)
        return fail(c, TL_ERR_INVALID, "the per-thread default stream needs a workspace of the caller's");
    if (capturing)
        return fail(c, TL_ERR_INVALID, "a stream in capture needs a workspace of the caller's (%zu bytes)", need);
    if (s == cudaStreamLegacy) s = nullptr;   // two names of one stream
    auto& all = c->op_ws;
    auto it = std::find_if(all.begin(), all.end(), [&](const StreamWs& w) { return w.stream == s; });
    if (it != all.end() && it->cap >= need) {
        std::rotate(it, it + 1, all.end());
        *out = all.back().ptr;
        return TL_OK;
    }
    // cudaFree waits for the device, so no work still uses what it frees
    if (it == all.end() && all.size() >= kMaxStreams) it = all.begin();
    if (it != all.end()) {
        cudaFree(it->ptr);
        all.erase(it);
    }
    const size_t bytes = std::max(need, (size_t)4 << 20);
    all.reserve(all.size() + 1);
    void* p = nullptr;
    TL_CK(c, cudaMalloc(&p, bytes));
    all.push_back({s, p, bytes});
    *out = p;
    return TL_OK;
}

// ---------------------------------------------------------------------------
// array checks
// ---------------------------------------------------------------------------
tl_status check_array(tl_ctx* c, const tl_array& a, const char* name) {
    if (a.dtype < TL_TYPE_F32 || a.dtype > TL_TYPE_BF16) return fail(c, TL_ERR_INVALID, "%s: unknown element type %d", name, a.dtype);
    if (a.rank < 0 || a.rank > TL_ARRAY_RANK) return fail(c, TL_ERR_INVALID, "%s: rank %d", name, a.rank);
    int64_t n = 1, reach = 0;
    for (int k = 0; k < a.rank; ++k) {
        if (a.dims[k] < 0) return fail(c, TL_ERR_INVALID, "%s: negative dim", name);
        if (a.strides[k] < 0) return fail(c, TL_ERR_INVALID, "%s: negative stride", name);
    }
    for (int k = 0; k < a.rank; ++k)
        if (a.dims[k] == 0) return TL_OK;
    for (int k = 0; k < a.rank; ++k) {
        int64_t span;
        if (__builtin_mul_overflow(n, a.dims[k], &n) || __builtin_mul_overflow(a.dims[k] - 1, a.strides[k], &span) ||
            __builtin_add_overflow(reach, span, &reach) || reach > (int64_t(1) << 58))
            return fail(c, TL_ERR_TOO_LARGE, "%s: sizes and strides pass 64 bits", name);
    }
    if (!a.data) return fail(c, TL_ERR_INVALID, "%s: no data", name);
    if (reinterpret_cast<uintptr_t>(a.data) % type_size(a.dtype)) return fail(c, TL_ERR_INVALID, "%s: misaligned", name);
    return TL_OK;
}

int64_t numel(const tl_array& a) {
    int64_t n = 1;
    for (int k = 0; k < a.rank; ++k) n *= a.dims[k];
    return n;
}

// Dims longer than one by rising stride.
int by_stride(const tl_array& a, int* ax) {
    int n = 0;
    for (int k = 0; k < a.rank; ++k)
        if (a.dims[k] > 1) ax[n++] = k;
    std::sort(ax, ax + n, [&](int x, int y) { return a.strides[x] < a.strides[y]; });
    return n;
}

// No two indices name one element: each stride passes the reach of the smaller ones.
bool distinct(const tl_array& a) {
    if (numel(a) == 0) return true;
    int ax[TL_ARRAY_RANK];
    const int n = by_stride(a, ax);
    int64_t reach = 0;
    for (int k = 0; k < n; ++k) {
        if (a.strides[ax[k]] <= reach) return false;
        reach += (a.dims[ax[k]] - 1) * a.strides[ax[k]];
    }
    return true;
}

// The elements fill their memory in some order.
bool dense(const tl_array& a) {
    int ax[TL_ARRAY_RANK];
    const int n = by_stride(a, ax);
    int64_t next = 1;
    for (int k = 0; k < n; ++k) {
        if (a.strides[ax[k]] != next) return false;
        next *= a.dims[ax[k]];
    }
    return true;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
HeadsView view(const tl_array& a) { return {a.data, a.strides[0], a.strides[1], a.strides[2], a.strides[3]}; }

tl_status check_heads(tl_ctx* c, const tl_array& a, const char* name, const tl_attention& t, int64_t b, int64_t h,
                      int64_t n, int64_t d, bool written) {
    TL_TRY(check_array(c, a, name));
    if (a.rank != 4) return fail(c, TL_ERR_INVALID, "attention: %s has rank %d, not 4", name, a.rank);
    if (a.dtype != t.q.dtype) return fail(c, TL_ERR_INVALID, "attention: %s has another element type than q", name);
    if (a.dims[0] != b || a.dims[1] != h || a.dims[2] != n || a.dims[3] != d)
        return fail(c, TL_ERR_INVALID, "attention: %s is [%lld, %lld, %lld, %lld], not [%lld, %lld, %lld, %lld]", name,
                    (long long)a.dims[0], (long long)a.dims[1], (long long)a.dims[2], (long long)a.dims[3], (long long)b,
                    (long long)h, (long long)n, (long long)d);
    if (written && !distinct(a)) return fail(c, TL_ERR_INVALID, "attention: %s is written and overlaps itself", name);
    return TL_OK;
}

tl_status check_attention(tl_ctx* c, const tl_attention& t, bool backward, AttnCall* out) {
    TL_TRY(check_array(c, t.q, "q"));
    TL_TRY(check_array(c, t.k, "k"));
    if (t.q.rank != 4 || t.k.rank != 4)
        return fail(c, TL_ERR_INVALID, "attention: q has rank %d and k %d, not 4", t.q.rank, t.k.rank);
    const int64_t b = t.q.dims[0], hq = t.q.dims[1], nq = t.q.dims[2], d = t.q.dims[3];
    const int64_t hkv = t.k.dims[1], nk = t.k.dims[2];
    if (d < 1 || d > kAttnMaxHead)
        return fail(c, TL_ERR_UNSUPPORTED, "attention: head size %lld, 1 to %d are supported", (long long)d, kAttnMaxHead);
    if (hkv == 0 ? hq != 0 : hq % hkv != 0)
        return fail(c, TL_ERR_INVALID, "attention: %lld query heads over %lld key heads", (long long)hq, (long long)hkv);
    if (b > kMaxCount || hq > kMaxCount || hkv > kMaxCount || nq > kMaxCount || nk > kMaxCount)
        return fail(c, TL_ERR_TOO_LARGE, "attention: more than 2^29 sequences, heads or positions");
    // blocks are numbered in 31 bits: one a query, or 16 keys of a head, at the least
    const int64_t heads = std::max(hq, hkv);   // keys without queries have gradients of 0 to write
    if (b * heads > kMaxCount / 2 || (double)b * hq * nq > 2147483647.0 || (double)b * heads * ((nk + 15) / 16) > 2147483647.0)
        return fail(c, TL_ERR_TOO_LARGE, "attention: batch x heads x queries above 2^31, or x keys above 2^35");
    TL_TRY(check_heads(c, t.q, "q", t, b, hq, nq, d, false));
    TL_TRY(check_heads(c, t.k, "k", t, b, hkv, nk, d, false));
    TL_TRY(check_heads(c, t.v, "v", t, b, hkv, nk, d, false));
    TL_TRY(check_heads(c, t.o, "o", t, b, hq, nq, d, !backward));
    const tl_array* in[5] = {&t.q, &t.k, &t.v, &t.o, &t.dout};
    const tl_array* wr[3] = {&t.o, nullptr, nullptr};
    int n_in = 3, n_wr = 1;
    if (backward) {
        TL_TRY(check_heads(c, t.dout, "dout", t, b, hq, nq, d, false));
        TL_TRY(check_heads(c, t.dq, "dq", t, b, hq, nq, d, true));
        TL_TRY(check_heads(c, t.dk, "dk", t, b, hkv, nk, d, true));
        TL_TRY(check_heads(c, t.dv, "dv", t, b, hkv, nk, d, true));
        wr[0] = &t.dq; wr[1] = &t.dk; wr[2] = &t.dv;
        n_in = 5; n_wr = 3;
        if (!t.lse && b * hq * nq > 0) return fail(c, TL_ERR_INVALID, "attention: the backward pass needs the forward's lse");
    }
    for (int w = 0; w < n_wr; ++w) {
        if (numel(*wr[w]) == 0) continue;
        for (int i = 0; i < n_in; ++i)
            if (in[i]->data == wr[w]->data && numel(*in[i]) > 0)
                return fail(c, TL_ERR_INVALID, "attention: a written array is an input too");
        for (int i = 0; i < w; ++i)
            if (wr[i]->data == wr[w]->data && numel(*wr[i]) > 0)
                return fail(c, TL_ERR_INVALID, "attention: two written arrays are one");
    }
    const std::pair<const void*, const char*> words[] = {
        {t.lse, "lse"}, {t.slopes, "slopes"}, {t.prefix_len, "prefix_len"}, {t.q_doc, "q_doc"},
        {t.k_doc, "k_doc"}, {t.kv_len, "kv_len"}, {t.q_start, "q_start"}};
    for (const auto& w : words)
        if (reinterpret_cast<uintptr_t>(w.first) % 4) return fail(c, TL_ERR_INVALID, "attention: %s is misaligned", w.second);
    if (!isfinite(t.scale)) return fail(c, TL_ERR_INVALID, "attention: scale is not finite");
    if (fabsf(t.scale) > 0x1p120f)   // times log2(e) it has to stay in fp32
        return fail(c, TL_ERR_UNSUPPORTED, "attention: scale %g is out of range", (double)t.scale);
    if (!isfinite(t.softcap) || t.softcap < 0) return fail(c, TL_ERR_INVALID, "attention: softcap is negative or not finite");
    // what the kernels make of the two (their quotient, its squares, the cap's
    // square) stays within fp32's normal numbers
    const double sc = fabs((double)t.scale), cap = t.softcap;
    if (cap > 0 && (cap < 0x1p-60 || cap > 0x1p100 || sc > cap * 0x1p60))
        return fail(c, TL_ERR_UNSUPPORTED, "attention: softcap %g with scale %g is out of range", cap, (double)t.scale);
    if (t.causal != 0 && t.causal != 1) return fail(c, TL_ERR_INVALID, "attention: causal is 0 or 1");
    if (t.prefix_len && !t.causal) return fail(c, TL_ERR_INVALID, "attention: prefix_len is for causal calls");
    if (!t.q_doc != !t.k_doc) return fail(c, TL_ERR_INVALID, "attention: q_doc and k_doc come together");
    AttnCall a;
    memset(&a, 0, sizeof a);
    a.dtype = t.q.dtype;
    a.b = (int)b; a.hq = (int)hq; a.hkv = (int)hkv; a.nq = (int)nq; a.nk = (int)nk; a.d = (int)d;
    a.q = view(t.q); a.k = view(t.k); a.v = view(t.v); a.o = view(t.o);
    if (backward) { a.dout = view(t.dout); a.dq = view(t.dq); a.dk = view(t.dk); a.dv = view(t.dv); }
    a.lse = t.lse;
    a.scale = t.scale; a.causal = t.causal;
    // q.k below 2^47 is then below 2^-13 of the cap, where the tanh is its argument to 2^-27
    a.cap = cap > sc * 0x1p60 ? 0.f : t.softcap;
    a.slopes = t.slopes; a.prefix_len = t.prefix_len; a.q_doc = t.q_doc; a.k_doc = t.k_doc;
    a.kv_len = t.kv_len; a.q_start = t.q_start;
    a.cuda_cores = c && c->opts.precision == TL_PREC_FP32 && a.dtype == TL_TYPE_F32;
    *out = a;
    return TL_OK;
}

// No query (backward: and no key) to write for.
bool nothing_to_do(const AttnCall& a, bool backward) {
    return (int64_t)a.b * a.hq * a.nq == 0 && (!backward || (int64_t)a.b * a.hkv * a.nk == 0);
}

size_t attention_need(const AttnCall& a, bool backward) {
    if (nothing_to_do(a, backward)) return 0;
    if (backward && attn_tc_backward_takes(a)) return attn_tc_backward_workspace(a);
    if (!backward && attn_few_takes(a)) return attn_few_workspace(a);
    if (!backward && attn_tc_takes(a)) return attn_tc_workspace(a);
    return attn_general_workspace(a, backward);
}

tl_status run_attention(tl_ctx* c, const tl_attention* t, bool backward) {
    if (!t) return fail(c, TL_ERR_INVALID, "attention: no descriptor");
    AttnCall a;
    TL_TRY(check_attention(c, *t, backward, &a));
    if (nothing_to_do(a, backward)) return TL_OK;
    DeviceGuard dev(c->device);
    if (!dev.ok) return fail(c, TL_ERR_CUDA, "cannot make device %d current", c->device);
    cudaStream_t s = static_cast<cudaStream_t>(t->stream);
    bool capturing;
    TL_TRY(check_stream(c, s, &capturing));
    if (capturing) c->flags_captured = true;
    void* ws = nullptr;
    TL_TRY(op_workspace(c, s, capturing, attention_need(a, backward), t->workspace, t->workspace_bytes, &ws));
    if (!backward && attn_few_takes(a)) return launch_attn_few(c, a, ws, s);
    const bool tc = backward ? attn_tc_backward_takes(a) : attn_tc_takes(a);
    if (tc) {
        const tl_status st = backward ? launch_attn_tc_backward(c, a, ws, s) : launch_attn_tc(c, a, ws, s);
        if (st != kNoSplit) return st;   // (what was queued only prepares operands; the general kernels need less workspace)
    }
    return backward ? launch_attn_general_backward(c, a, ws, s) : launch_attn_general(c, a, ws, s);
}

// ---------------------------------------------------------------------------
// clipping
// ---------------------------------------------------------------------------
tl_status check_clip(tl_ctx* c, const tl_array* grads, const tl_array* out, int32_t n, double max_norm,
                     std::vector<ClipItem>* items) {
    if (n < 0 || (n > 0 && !grads)) return fail(c, TL_ERR_INVALID, "clip: no gradients");
    if (!(max_norm >= 0)) return fail(c, TL_ERR_INVALID, "clip: max_norm is negative or not a number");
    std::vector<std::pair<uintptr_t, uintptr_t>> written;
    items->reserve(n);
    written.reserve(n);
    for (int i = 0; i < n; ++i) {
        const tl_array& g = grads[i];
        TL_TRY(check_array(c, g, "clip: gradient"));
        const int64_t count = numel(g);
        if (count > 0 && !dense(g)) return fail(c, TL_ERR_INVALID, "clip: gradient %d is not dense", i);
        const tl_array& o = out ? out[i] : g;
        if (out) {
            TL_TRY(check_array(c, o, "clip: output"));
            bool same = o.rank == g.rank;
            for (int k = 0; same && k < g.rank; ++k)
                same = o.dims[k] == g.dims[k] && (g.dims[k] <= 1 || o.strides[k] == g.strides[k]);
            if (!same) return fail(c, TL_ERR_INVALID, "clip: output %d has other dims or strides than its gradient", i);
        }
        if (count == 0) continue;
        items->push_back({g.data, o.data, count, g.dtype, o.dtype});
        const uintptr_t at = reinterpret_cast<uintptr_t>(o.data);
        written.push_back({at, at + count * type_size(o.dtype)});
    }
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
        if (written[i].first < written[i - 1].second)
            return fail(c, TL_ERR_INVALID, "clip: two of the arrays written share elements");
    if (out) {
        // an input under another array's output would be read half clipped
        for (const ClipItem& it : *items) {
            const uintptr_t lo = reinterpret_cast<uintptr_t>(it.in), hi = lo + it.n * type_size(it.in_type);
            auto w = std::upper_bound(written.begin(), written.end(), std::make_pair(hi - 1, UINTPTR_MAX));
            if (w != written.begin() && std::prev(w)->second > lo && !(it.in == it.out && it.in_type == it.out_type))
                return fail(c, TL_ERR_INVALID, "clip: an output lies over an input");
        }
    }
    return TL_OK;
}

}  // namespace

double attn_pairs(const AttnCall& a) {
    const double nq = a.nq, nk = a.nk;
    double per = nq * nk;
    if (a.causal && !a.prefix_len) per = nk >= nq ? nq * (nk - nq) + nq * (nq + 1) / 2 : nk * (nk + 1) / 2;
    return per * a.b * a.hq;
}

}  // namespace tl

using namespace tl;

extern "C" tl_status tl_tensor_array(tl_tensor* t, int32_t write, tl_array* out) {
    tl_ctx* c = t ? static_cast<tl_ctx*>(t->owner) : nullptr;
    if (!c || !out) return TL_ERR_INVALID;
    return entry(c, (tl_status)TL_ERR_OOM, [&]() -> tl_status {
        if (t->shard != TL_SHARD_NONE && c->world > 1)
            return fail(c, TL_ERR_UNSUPPORTED, "%s: a sharded tensor has no array", t->name.c_str());
        if (t->rank > TL_ARRAY_RANK)
            return fail(c, TL_ERR_UNSUPPORTED, "%s: rank %d, arrays have at most %d", t->name.c_str(), t->rank, TL_ARRAY_RANK);
        DeviceGuard dev(c->device);
        if (!dev.ok) return fail(c, TL_ERR_CUDA, "cannot make device %d current", c->device);
        TL_TRY(ensure_dense(c, t));
        if (write) {
            mark_written_dense(t);
            t->boolean = false;
        }
        memset(out, 0, sizeof *out);
        out->data = t->dense;
        out->dtype = TL_TYPE_F32;
        out->rank = t->rank;
        for (int k = 0; k < t->rank; ++k) { out->dims[k] = t->dims[k]; out->strides[k] = t->strides[k]; }
        return TL_OK;
    });
}

extern "C" tl_status tl_attention_forward(tl_ctx* c, const tl_attention* a) {
    if (!c) return TL_ERR_INVALID;
    return entry(c, (tl_status)TL_ERR_OOM, [&] { return run_attention(c, a, false); });
}

extern "C" tl_status tl_attention_backward(tl_ctx* c, const tl_attention* a) {
    if (!c) return TL_ERR_INVALID;
    return entry(c, (tl_status)TL_ERR_OOM, [&] { return run_attention(c, a, true); });
}

extern "C" int64_t tl_attention_workspace(tl_ctx* c, const tl_attention* t, int32_t backward) {
    return entry(c, (int64_t)-TL_ERR_OOM, [&]() -> int64_t {
        if (!t) return -(int64_t)fail(c, TL_ERR_INVALID, "attention: no descriptor");
        AttnCall a;
        const tl_status st = check_attention(c, *t, backward != 0, &a);
        if (st != TL_OK) return -(int64_t)st;
        size_t n = attention_need(a, backward != 0);
        if (!c && a.dtype == TL_TYPE_F32) {   // enough for a context of either precision
            a.cuda_cores = 1;
            n = std::max(n, attention_need(a, backward != 0));
        }
        return (int64_t)n;
    });
}

extern "C" int64_t tl_clip_workspace(tl_ctx* c, const tl_array* grads, const tl_array* out, int32_t n, double max_norm) {
    return entry(c, (int64_t)-TL_ERR_OOM, [&]() -> int64_t {
        std::vector<ClipItem> items;
        const tl_status st = check_clip(c, grads, out, n, max_norm, &items);
        return st == TL_OK ? (int64_t)clip_workspace_bytes() : -(int64_t)st;
    });
}

extern "C" tl_status tl_clip_gradients(tl_ctx* c, const tl_array* grads, const tl_array* out, int32_t n, double max_norm,
                                       float* d_norm, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!c) return TL_ERR_INVALID;
    return entry(c, (tl_status)TL_ERR_OOM, [&]() -> tl_status {
        std::vector<ClipItem> items;
        TL_TRY(check_clip(c, grads, out, n, max_norm, &items));
        if (reinterpret_cast<uintptr_t>(d_norm) % 4) return fail(c, TL_ERR_INVALID, "clip: norm is misaligned");
        if (items.empty() && !d_norm) return TL_OK;
        DeviceGuard dev(c->device);
        if (!dev.ok) return fail(c, TL_ERR_CUDA, "cannot make device %d current", c->device);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        bool capturing;
        TL_TRY(check_stream(c, s, &capturing));
        void* ws = nullptr;
        TL_TRY(op_workspace(c, s, capturing, clip_workspace_bytes(), workspace, workspace_bytes, &ws));
        return launch_clip(c, items, max_norm, d_norm, ws, s);
    });
}
