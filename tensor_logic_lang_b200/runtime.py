"""Drive libtl_cuda through its C ABI (include/tl_cuda.h).

`Context` owns one tl_ctx on one GPU; `Context.run(program)` executes a
lowered `.tl` program the way the reference's emitted `main()` does
(LLVMCodegen.generate order: statements, fixpoint, queries), and
`Context.tensor(name)` reads a result back as f64 numpy.  There is no CPU
fallback: without the built library or a GPU, construction raises.
"""
import ctypes as C
import struct
from math import prod
from operator import methodcaller

import numpy as np

from . import abi


# tl_array: data, dtype, rank, dims[4], strides[4]
_ARRAY = struct.Struct("=Qii4q4q")
_LIST = np.dtype([("data", "u8"), ("dtype", "i4"), ("rank", "i4"), ("dims", "i8", 4), ("strides", "i8", 4)])
_TYPES = {"torch.float32": abi.TL_TYPE_F32, "torch.float16": abi.TL_TYPE_F16, "torch.bfloat16": abi.TL_TYPE_BF16,
          "float32": abi.TL_TYPE_F32, "float16": abi.TL_TYPE_F16, "bfloat16": abi.TL_TYPE_BF16}
_type_of = {}          # dtype object -> TL_TYPE_*
_DATA, _NUMEL, _DEVICE, _IS_CONTIGUOUS = (methodcaller(n) for n in ("data_ptr", "numel", "get_device", "is_contiguous"))
# tl_attention: eight tl_array, then lse .. stream
_ATTENTION = struct.Struct("=" + "Qii4q4q" * 8 + "QffiiQQQQQQQqQ")
_NO_GRADS = (0,) * (11 * 4)
_PAD = [(0,) * (abi.TL_ARRAY_RANK - r) for r in range(abi.TL_ARRAY_RANK + 1)]


def _in_a_row(shape, strides):
    """Whether an array's elements lie behind one another in the order of its indices."""
    n = 1
    for k, s in zip(reversed(shape), reversed(strides)):
        if k != 1 and s != n:
            return False
        n *= k
    return True



class Context:
    def __init__(self, device=-1, precision=abi.PREC_TF32, rank=0, world_size=1, nccl_id=None,
                 max_sweeps=1000, verbose=False, comm_timeout_ms=30000, lib=None):
        self.lib = lib or abi.load_library()
        opts = abi.InitOpts()
        self.lib.tl_default_opts(C.byref(opts))
        opts.device = device
        opts.precision = precision
        opts.rank = rank
        opts.world_size = world_size
        opts.max_sweeps = max_sweeps
        opts.verbose = 1 if verbose else 0
        opts.comm_timeout_ms = comm_timeout_ms
        if nccl_id is not None:
            for i, b in enumerate(bytes(nccl_id)[:128]):
                opts.nccl_id[i] = b
        h = C.c_void_p()
        st = self.lib.tl_init(C.byref(opts), C.byref(h))
        if st != abi.TL_OK:
            raise abi.TLError(st, "tl_init failed (no CUDA device or bad options)")
        self.h = h
        self.device = self.lib.tl_device(h)

    def close(self):
        if getattr(self, "h", None):
            self.lib.tl_shutdown(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def check(self, st, what=""):
        if st != abi.TL_OK:
            msg = self.lib.tl_last_error(self.h).decode(errors="replace")
            raise abi.TLError(st, f"{what}: {msg}")

    # ------------------------------------------------------------------ program
    def run(self, program):
        self.check(self.lib.tl_program_run(self.h, C.cast(program.stmts, C.POINTER(abi.Statement)), program.n),
                   "tl_program_run")
        return self

    def sync(self):
        self.check(self.lib.tl_sync(self.h), "tl_sync")

    @property
    def sweeps(self):
        return self.lib.tl_last_sweeps(self.h)

    def last_error(self):
        """tl_last_error: the text of the last failure or note (the sweep cap)."""
        return self.lib.tl_last_error(self.h).decode(errors="replace")

    @property
    def launches(self):
        return self.lib.tl_launch_count(self.h)

    @property
    def stream_ptr(self):
        return self.lib.tl_stream(self.h)

    def set_sharding(self, name, mode=abi.SHARD_ROWS):
        self.check(self.lib.tl_set_sharding(self.h, name.encode(), mode), "tl_set_sharding")

    # ------------------------------------------------------------------ tensors
    def _lookup(self, name):
        t = C.c_void_p()
        self.check(self.lib.tl_tensor_lookup(self.h, name.encode(), C.byref(t)), f"lookup {name}")
        return t

    def shape(self, name):
        t = self._lookup(name)
        return tuple(self.lib.tl_tensor_dim(t, k) for k in range(self.lib.tl_tensor_rank(t)))

    def tensor(self, name, rows=None):
        """f64 copy of a tensor (a row-sharded one gives its local rows)."""
        t = self._lookup(name)
        shape = self.shape(name)
        if rows is not None:
            shape = (rows,) + shape[1:]
        out = np.empty(shape, dtype=np.float64)
        self.check(self.lib.tl_tensor_download(t, out.ctypes.data_as(C.POINTER(C.c_double))), f"download {name}")
        return out

    def tensor_f32(self, name, rows=None):
        t = self._lookup(name)
        shape = self.shape(name)
        if rows is not None:
            shape = (rows,) + shape[1:]
        out = np.empty(shape, dtype=np.float32)
        self.check(self.lib.tl_tensor_download_f32(t, out.ctypes.data_as(C.POINTER(C.c_float))), f"download {name}")
        return out

    def bits(self, name, rows=None, out=None, words=None):
        """Bit rows (uint32 words) of a 0/1 rank-2 tensor (into `out` when given,
        e.g. a pinned host buffer).  A row-sharded tensor gives its `rows`
        local rows; a column-sharded one its slice of `words` words per row."""
        t = self._lookup(name)
        r, cols = self.shape(name)
        if rows is not None:
            r = rows
        w = (cols + 31) // 32 if words is None else words
        if out is None:
            out = np.empty((r, w), dtype=np.uint32)
        assert out.dtype == np.uint32 and out.flags.c_contiguous and out.shape == (r, w)
        self.check(self.lib.tl_tensor_download_bits(t, out.ctypes.data_as(C.POINTER(C.c_uint32))), f"bits {name}")
        return out

    def upload(self, name, arr):
        t = self._lookup(name)
        a = np.ascontiguousarray(arr, dtype=np.float64)
        self.check(self.lib.tl_tensor_upload(t, a.ctypes.data_as(C.POINTER(C.c_double))), f"upload {name}")

    def upload_f32(self, name, arr):
        t = self._lookup(name)
        a = np.ascontiguousarray(arr, dtype=np.float32)
        self.check(self.lib.tl_tensor_upload_f32(t, a.ctypes.data_as(C.POINTER(C.c_float))), f"upload {name}")

    def create(self, name, shape):
        t = C.c_void_p()
        dims = (C.c_int64 * max(1, len(shape)))(*shape)
        self.check(self.lib.tl_tensor_create(self.h, name.encode(), len(shape), dims, C.byref(t)), f"create {name}")
        return t

    def query(self, name):
        t = self._lookup(name)
        buf = C.create_string_buffer(4096)
        self.check(self.lib.tl_query_format(t, buf, len(buf)), f"query {name}")
        return buf.value.decode()

    def output(self):
        """What the last program's queries printed (the reference's stdout)."""
        need = C.c_int64()
        self.check(self.lib.tl_program_output(self.h, None, 0, C.byref(need)), "program output")
        buf = C.create_string_buffer(need.value + 1)
        self.check(self.lib.tl_program_output(self.h, buf, len(buf), None), "program output")
        return buf.value.decode()

    # ------------------------------------------------------------------ array operators
    # Arrays are device tensors (torch's, or any object with their data_ptr(), dtype,
    # shape, stride(), get_device(), numel() and is_contiguous()), or names of this context's tensors, which
    # stand for their fp32 storage and are used on the context's own stream alone.  stream: a cudaStream_t handle (torch's
    # current stream: torch.cuda.current_stream().cuda_stream), or None for the
    # context's own stream, on which its programs run.  Device tensors that
    # another stream wrote need that stream's work done or waited for first.
    def _view(self, x, what):
        """(data, type, shape, strides) of an array argument."""
        if isinstance(x, str):
            if self._foreign:
                raise abi.TLError(abi.TL_ERR_INVALID, f"{what}: a tensor's storage is used on the context's own stream")
            a = abi.Array()
            self.check(self.lib.tl_tensor_array(self._lookup(x), 0, C.byref(a)), f"{what} {x}")
            return a.data or 0, a.dtype, tuple(a.dims[:a.rank]), tuple(a.strides[:a.rank])
        t = _type_of.get(x.dtype)
        if t is None:
            t = self._type(x.dtype, what)
        self._on_device(x, what)
        return x.data_ptr(), t, x.shape, x.stride()

    def _wrote(self, xs, what):
        """Tells the tensors among the arrays that a call has been queued which writes their storage."""
        for x in xs:
            if isinstance(x, str):
                self.check(self.lib.tl_tensor_array(self._lookup(x), 1, C.byref(abi.Array())), f"{what} {x}")

    def _type(self, dtype, what):
        t = _TYPES.get(str(dtype))
        if t is None:
            raise abi.TLError(abi.TL_ERR_INVALID, f"{what}: element type {dtype}, not float32, float16 or bfloat16")
        _type_of[dtype] = t
        return t

    def _on_device(self, x, what):
        if x.get_device() != self.device:
            raise abi.TLError(abi.TL_ERR_INVALID, f"{what} is on {x.device}, the context on cuda:{self.device}")

    def _heads(self, x, what):
        """The fields of an array of rank 2 to 4 as [batch, heads, positions, head size]."""
        p, t, shape, strides = self._view(x, what)
        r = len(shape)
        if r != 4:
            if r < 2 or r > 4:
                raise abi.TLError(abi.TL_ERR_INVALID, f"attention: {what} has rank {r}, not 2 to 4")
            shape, strides = (1,) * (4 - r) + tuple(shape), (0,) * (4 - r) + tuple(strides)
        return (p, t, 4, *shape, *strides)

    def _plain(self, x, what, kind, shape):
        """Address of a contiguous device array of one type and shape."""
        if isinstance(x, str):
            if kind != "float32":
                raise abi.TLError(abi.TL_ERR_INVALID, f"{what} is an array of {kind}, not a tensor's name")
            p, _, have, _ = self._view(x, what)
        else:
            self._on_device(x, what)
            if str(x.dtype).rpartition(".")[2] != kind or not x.is_contiguous():
                raise abi.TLError(abi.TL_ERR_INVALID, f"{what} is not a contiguous array of {kind}")
            p, have = x.data_ptr(), tuple(x.shape)
        if have == shape:
            return p
        n = 1
        for k in shape:
            n *= k
        m = 1
        for k in have:
            m *= k
        if m != n or (len(have) == len(shape) and tuple(have) != tuple(shape)):
            raise abi.TLError(abi.TL_ERR_INVALID, f"{what} is {have}, not {tuple(shape)}")
        return p

    def _stream(self, stream):
        own = self.lib.tl_stream(self.h) or 0
        if stream is None:
            stream = own
        self._foreign = stream != own
        return stream

    def _room(self, workspace):
        if workspace is None:
            return 0, 0
        self._on_device(workspace, "workspace")
        if not workspace.is_contiguous():
            raise abi.TLError(abi.TL_ERR_INVALID, "workspace is not contiguous")
        return workspace.data_ptr(), workspace.numel() * workspace.element_size()

    def _attention(self, q, k, v, out, lse, grads, scale, softcap, slopes, causal, prefix_len, q_doc, k_doc, kv_len,
                   q_start, workspace, stream):
        stream = self._stream(stream)
        qa, ka, va, oa = self._heads(q, "q"), self._heads(k, "k"), self._heads(v, "v"), self._heads(out, "out")
        b, hq, nq, d = qa[3:7]
        nk = ka[5]
        ga = _NO_GRADS
        if grads:
            ga = sum((self._heads(x, n) for x, n in zip(grads, ("dout", "dq", "dk", "dv"))), ())
        if scale is None:
            scale = d ** -0.5 if d else 1.0
        ws, room = self._room(workspace)
        plain, one = self._plain, (b,)
        return _ATTENTION.pack(
            *qa, *ka, *va, *oa, *ga, lse is not None and plain(lse, "lse", "float32", (b, hq, nq)), scale, softcap,
            1 if causal else 0, 0, slopes is not None and plain(slopes, "slopes", "float32", (hq,)),
            prefix_len is not None and plain(prefix_len, "prefix_len", "int32", one),
            q_doc is not None and plain(q_doc, "q_doc", "int32", (b, nq)),
            k_doc is not None and plain(k_doc, "k_doc", "int32", (b, nk)),
            kv_len is not None and plain(kv_len, "kv_len", "int32", one),
            q_start is not None and plain(q_start, "q_start", "int32", one), ws, room, stream)

    def attention(self, q, k, v, out, lse=None, *, scale=None, softcap=0.0, slopes=None, causal=False, prefix_len=None,
                  q_doc=None, k_doc=None, kv_len=None, q_start=None, workspace=None, stream=None):
        """out = softmax(scores) v by head, with capped, biased or masked scores (tl_attention_forward).

        q, out [batch, Hq, Nq, d] and k, v [batch, Hkv, Nk, d] (leading dims of 1 may be left out); out is written.
        scale: of q.k, d^-0.5 when None.  softcap: scores become softcap tanh(score / softcap).  slopes [Hq]: score
        minus slope times distance.  causal: a query sees the keys up to its position, and those before
        prefix_len [batch].  q_doc [batch, Nq], k_doc [batch, Nk]: keys of the query's own document alone, a negative
        one is padding.  kv_len [batch]: keys of each sequence.  q_start [batch]: position of its first query,
        kv_len - Nq when None.  lse [batch, Hq, Nq] fp32 receives what the backward pass needs.
        """
        d = self._attention(q, k, v, out, lse, None, scale, softcap, slopes, causal, prefix_len, q_doc, k_doc, kv_len,
                            q_start, workspace, stream)
        self.check(self.lib.tl_attention_forward(self.h, d), "attention")
        self._wrote((out, lse), "attention")
        return out

    def attention_backward(self, q, k, v, out, lse, dout, dq, dk, dv, *, scale=None, softcap=0.0, slopes=None,
                           causal=False, prefix_len=None, q_doc=None, k_doc=None, kv_len=None, q_start=None,
                           workspace=None, stream=None):
        """Writes dq, dk, dv, the gradient of sum(out * dout) (tl_attention_backward); out and lse are the forward's."""
        d = self._attention(q, k, v, out, lse, (dout, dq, dk, dv), scale, softcap, slopes, causal, prefix_len, q_doc,
                            k_doc, kv_len, q_start, workspace, stream)
        self.check(self.lib.tl_attention_backward(self.h, d), "attention_backward")
        self._wrote((dq, dk, dv), "attention_backward")
        return dq, dk, dv

    def attention_workspace(self, q, k, v, out, lse=None, grads=None, *, scale=None, softcap=0.0, slopes=None,
                            causal=False, prefix_len=None, q_doc=None, k_doc=None, kv_len=None, q_start=None):
        """Bytes of workspace of an attention call, with grads = (dout, dq, dk, dv) of its backward pass."""
        d = self._attention(q, k, v, out, lse, grads, scale, softcap, slopes, causal, prefix_len, q_doc, k_doc, kv_len,
                            q_start, None, None)
        n = self.lib.tl_attention_workspace(self.h, d, 1 if grads else 0)
        self.check(max(0, -n), "attention_workspace")
        return n

    def _list(self, arrays, what):
        """Packs arrays as tl_array (a contiguous one as its elements in a row)."""
        n = len(arrays)
        if n > 16 and not any(isinstance(x, str) for x in arrays) and all(map(_IS_CONTIGUOUS, arrays)):
            # long lists a column at a time
            for d in set(map(_DEVICE, arrays)) - {self.device}:
                raise abi.TLError(abi.TL_ERR_INVALID, f"{what} on device {d}, the context on cuda:{self.device}")
            types = [x.dtype for x in arrays]
            for t in set(types) - _type_of.keys():
                self._type(t, what)
            out = np.zeros(n, _LIST)
            out["data"] = np.fromiter(map(_DATA, arrays), np.uint64, n)
            out["dtype"] = [_type_of[t] for t in types]
            out["rank"] = 1
            out["dims"][:, 0] = np.fromiter(map(_NUMEL, arrays), np.int64, n)
            out["strides"][:, 0] = 1
            return out.tobytes()
        parts = []
        for x in arrays:
            p, t, shape, strides = self._view(x, what)
            r = len(shape)
            if _in_a_row(shape, strides) if isinstance(x, str) else x.is_contiguous():
                shape, strides, r = (prod(shape),), (1,), 1
            elif r > abi.TL_ARRAY_RANK:
                raise abi.TLError(abi.TL_ERR_INVALID, f"{what}: rank {r} and not contiguous")
            parts.append(_ARRAY.pack(p, t, r, *shape, *_PAD[r], *strides, *_PAD[r]))
        return b"".join(parts)

    def _clip_lists(self, grads, out):
        if out is not None and len(out) != len(grads):
            raise abi.TLError(abi.TL_ERR_INVALID, f"clip: {len(out)} outputs for {len(grads)} gradients")
        return self._list(grads, "gradient"), None if out is None else self._list(out, "output")

    def clip_gradients(self, grads, max_norm, out=None, norm=None, workspace=None, stream=None):
        """Scales the arrays so that their global norm is at most max_norm (tl_clip_gradients).

        In place, or into the arrays of `out` (any type; the same dims and strides, or contiguous like the gradient and
        with as many elements).  norm: a device fp32 scalar that
        receives the norm before the scaling.  Nothing is copied to the host.
        """
        stream = self._stream(stream)
        a, o = self._clip_lists(grads, out)
        at = None if norm is None else self._plain(norm, "norm", "float32", ())
        self.check(self.lib.tl_clip_gradients(self.h, a, o, len(grads), max_norm,
                                              at, *self._room(workspace), stream), "clip_gradients")
        self._wrote(grads if out is None else out, "clip_gradients")
        self._wrote((norm,), "clip_gradients")
        return grads if out is None else out

    def clip_workspace(self, grads, max_norm, out=None):
        """Bytes of workspace of a clip_gradients call."""
        self._stream(None)
        a, o = self._clip_lists(grads, out)
        n = self.lib.tl_clip_workspace(self.h, a, o, len(grads), max_norm)
        self.check(max(0, -n), "clip_workspace")
        return n

    # ------------------------------------------------------------------ profiling
    def profile(self, on=True):
        self.check(self.lib.tl_profile_enable(self.h, 1 if on else 0), "profile")

    def profile_reset(self):
        self.check(self.lib.tl_profile_reset(self.h), "profile_reset")

    def profile_read(self):
        arr = (abi.KernelStats * 64)()
        n = self.lib.tl_profile_read(self.h, arr, 64)
        return {arr[i].name.decode(): dict(launches=arr[i].launches, total_ms=arr[i].total_ms,
                                           bytes=arr[i].algo_bytes, flops=arr[i].algo_flops)
                for i in range(n)}


def unique_id(lib=None):
    lib = lib or abi.load_library()
    buf = (C.c_uint8 * 128)()
    st = lib.tl_comm_unique_id(buf)
    if st != abi.TL_OK:
        raise abi.TLError(st, "tl_comm_unique_id")
    return bytes(buf)
