"""Argument checks of the array operators (attention, gradient clipping): every refusal happens on the host,
before any device work, so these run without a GPU through the _workspace functions, which make the same checks."""
import ctypes as C
import math

import pytest

from tensor_logic_lang_b200 import abi


@pytest.fixture(scope="module")
def lib():
    from tensor_logic_lang_b200 import build
    build.build()
    return abi.load_library()


def array(dims, strides=None, dtype=abi.TL_TYPE_F32, data=0x10000):
    if strides is None:
        strides, n = [], 1
        for k in reversed(dims):
            strides.insert(0, n)
            n *= k
    a = abi.Array(data=data, dtype=dtype, rank=len(dims))
    for i, (n, s) in enumerate(zip(dims, strides)):
        a.dims[i], a.strides[i] = n, s
    return a


def attention(b=2, hq=4, hkv=2, nq=8, nk=16, d=32, dtype=abi.TL_TYPE_F32, **fields):
    a = abi.Attention(scale=1.0)
    for i, n in enumerate(("q", "o", "dout", "dq")):
        setattr(a, n, array((b, hq, nq, d), dtype=dtype, data=0x100000 * (i + 1)))
    for i, n in enumerate(("k", "v", "dk", "dv")):
        setattr(a, n, array((b, hkv, nk, d), dtype=dtype, data=0x10000000 * (i + 1)))
    a.lse = 0x1000
    for n, v in fields.items():
        setattr(a, n, v)
    return a


def need(lib, a, backward=0):
    return lib.tl_attention_workspace(None, C.byref(a), backward)


def test_accepted(lib):
    for dtype in (abi.TL_TYPE_F32, abi.TL_TYPE_F16, abi.TL_TYPE_BF16):
        assert need(lib, attention(dtype=dtype)) >= 0
        assert need(lib, attention(dtype=dtype), 1) >= 0
    assert need(lib, attention(nq=0)) >= 0
    assert need(lib, attention(nk=0), 1) >= 0
    assert need(lib, attention(b=0), 1) >= 0
    # broadcast keys, any order of the dims, any stride along the head
    assert need(lib, attention(k=array((2, 2, 16, 32), (0, 0, 32, 1)))) >= 0
    assert need(lib, attention(o=array((2, 4, 8, 32), (4 * 8 * 32, 32, 4 * 32, 1)))) >= 0
    assert need(lib, attention(q=array((2, 4, 8, 32), (8192, 2048, 256, 8)))) >= 0


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("bad", [
    dict(q=array((2, 4, 8))),                                          # rank
    dict(v=array((2, 2, 17, 32))),                                     # lengths of k and v
    dict(k=array((2, 3, 16, 32)), v=array((2, 3, 16, 32))),            # heads that do not divide
    dict(k=array((2, 0, 16, 32)), v=array((2, 0, 16, 32))),
    dict(o=array((2, 4, 8, 32), dtype=abi.TL_TYPE_F16)),               # types
    dict(q=array((2, 4, 8, 32), dtype=7)),
    dict(q=array((2, 4, 8, 32), data=0)),                              # no data, misaligned
    dict(q=array((2, 4, 8, 32), data=0x10002)),
    dict(q=array((2, 4, 8, 32), (1024, 256, -32, 1))),
    dict(q=array((-2, 4, 8, 32), (1024, 256, 32, 1))),
    dict(scale=math.nan), dict(softcap=-1.0), dict(softcap=math.inf), dict(causal=2),
    dict(prefix_len=0x1000), dict(q_doc=0x1000), dict(causal=1, k_doc=0x1000), dict(lse=0x1002),
    dict(d=0),
])
def test_refused(lib, bad, backward):
    st = need(lib, attention(**bad), backward)
    assert st in (-abi.TL_ERR_INVALID, -abi.TL_ERR_UNSUPPORTED), st


@pytest.mark.parametrize("name", ["slopes", "prefix_len", "kv_len", "q_start", "q_doc", "k_doc"])
def test_refused_addresses(lib, name):
    # 32-bit values that do not lie on 4 bytes would fault the GPU
    both = {"q_doc": 0x1000, "k_doc": 0x2000} if "doc" in name else {}
    for off in (1, 2):
        a = attention(causal=1, **dict(both, **{name: 0x3000 + off}))
        assert need(lib, a) == need(lib, a, 1) == -abi.TL_ERR_INVALID
    assert need(lib, attention(causal=1, **dict(both, **{name: 0x3004}))) >= 0


def test_refused_scales(lib):
    # times log2(e), 3e38 is infinite, and 0 times that no score
    for scale in (3e38, -3e38, 2.0 ** 121):
        for backward in (0, 1):
            assert need(lib, attention(scale=scale), backward) == -abi.TL_ERR_UNSUPPORTED
    for scale in (2.0 ** 120, -2.0 ** 120, 0.0, 1e-44):
        assert need(lib, attention(scale=scale)) >= 0


def test_refused_caps(lib):
    # caps whose quotients with the scale, or squares, leave fp32
    for scale, softcap in ((1.0, 1e-30), (1.0, 2.0 ** -61), (1e-20, 1e-40), (1e30, 2.0 ** 101), (1e20, 1.0), (-1e20, 1.0)):
        for backward in (0, 1):
            assert need(lib, attention(scale=scale, softcap=softcap), backward) == -abi.TL_ERR_UNSUPPORTED
    for scale, softcap in ((1.0, 2.0 ** -60), (1.0, 2.0 ** 100), (0.0, 1.0), (1e-30, 1e30), (2.0 ** 60, 1.0)):
        assert need(lib, attention(scale=scale, softcap=softcap)) >= 0


def test_refused_sizes(lib):
    assert need(lib, attention(d=257)) == -abi.TL_ERR_UNSUPPORTED
    assert need(lib, attention(d=256)) >= 0
    big = 1 << 40
    a = attention(k=array((2, 2, big, 32), (0, 0, 0, 1)), v=array((2, 2, big, 32), (0, 0, 0, 1)))
    assert need(lib, a) == -abi.TL_ERR_TOO_LARGE
    a = attention(q=array((2, 4, 8, 32), (1 << 61, 1, 1, 1)))
    assert need(lib, a) == -abi.TL_ERR_TOO_LARGE


def test_workspace_without_a_context_is_enough_for_any(lib):
    # a TL_PREC_FP32 context keeps fp32 arrays on the CUDA cores, as every context does at a head size of 200,
    # where a row's part is 202 words (of head size 64: 66)
    for rows in (1, 8, 32):
        on_cuda_cores = need(lib, attention(b=1, hq=rows, hkv=1, nq=1, nk=64, d=200)) * 66 // 202
        assert need(lib, attention(b=1, hq=rows, hkv=1, nq=1, nk=64, d=64)) >= on_cuda_cores


@pytest.mark.parametrize("dtype", [abi.TL_TYPE_F32, abi.TL_TYPE_F16, abi.TL_TYPE_BF16])
def test_no_heads_need_no_workspace(lib, dtype):
    # heads, queries or sequences that are not there: nothing is divided by their number
    for backward in (0, 1):
        for none in (dict(hq=0, hkv=0), dict(b=0), dict(b=0, hq=0, hkv=0), dict(hq=0, hkv=0, nq=0, nk=0)):
            assert need(lib, attention(dtype=dtype, **none), backward) == 0, none
        assert need(lib, attention(dtype=dtype, hq=0), backward) == 0    # keys without queries: dk, dv of zeros
        assert need(lib, attention(dtype=dtype, nq=0), backward) == 0


def test_refused_counts(lib):
    # more queries than blocks can be numbered, without the memory for them
    def wide(b, h, n):
        return array((b, h, n, 1), (0, 0, 0, 1))
    a = attention(b=1, hq=1, hkv=1, nq=1, nk=1, d=1)
    a.q = wide(1 << 14, 1 << 14, 64)
    a.k = a.v = wide(1 << 14, 1 << 14, 1)
    a.o = array((1 << 14, 1 << 14, 64, 1), data=0x70000000)
    assert need(lib, a) == -abi.TL_ERR_TOO_LARGE


def test_refused_counts_of_keys_without_queries(lib):
    # key heads of calls without query heads count like query heads
    for b, h, n in ((1 << 14, 1 << 15, 1), (1 << 14, 1 << 14, 1 << 20), (1, 1 << 40, 1)):
        a = attention(b=1, hq=1, hkv=1, nq=1, nk=1, d=1)
        for i, name in enumerate(("q", "o", "dout", "dq")):
            setattr(a, name, array((b, 0, 1, 1), data=0x1000 * (i + 1)))
        a.k = a.v = array((b, h, n, 1), (0, 0, 0, 1))
        a.dk, a.dv = array((b, h, n, 1), data=1 << 40), array((b, h, n, 1), data=1 << 41)
        assert need(lib, a, 1) == -abi.TL_ERR_TOO_LARGE, (b, h, n)


def test_refused_outputs(lib):
    # written arrays that overlap themselves, an input or one another
    assert need(lib, attention(o=array((2, 4, 8, 32), (0, 256, 32, 1)))) == -abi.TL_ERR_INVALID
    assert need(lib, attention(o=array((2, 4, 8, 32), (1024, 256, 31, 1)))) == -abi.TL_ERR_INVALID
    assert need(lib, attention(dk=array((2, 2, 16, 32), (0, 512, 32, 1))), 1) == -abi.TL_ERR_INVALID
    a = attention()
    a.o = a.q
    assert need(lib, a) == -abi.TL_ERR_INVALID
    a = attention()
    a.dv = a.dk
    assert need(lib, a, 1) == -abi.TL_ERR_INVALID
    a = attention()
    a.dq = a.dout
    assert need(lib, a, 1) == -abi.TL_ERR_INVALID
    assert need(lib, attention(lse=None), 1) == -abi.TL_ERR_INVALID
    assert need(lib, attention(lse=None)) >= 0


def clip(lib, grads, out=None, max_norm=1.0):
    def at(v):
        return (abi.Array * max(1, len(v)))(*v)
    return lib.tl_clip_workspace(None, at(grads), None if out is None else at(out), len(grads), max_norm)


def test_clip_checks(lib):
    g = [array((100,)), array((3, 5), data=0x20000, dtype=abi.TL_TYPE_BF16), array((0,), data=0)]
    assert clip(lib, g) > 0
    assert clip(lib, []) > 0
    assert clip(lib, g, max_norm=math.inf) > 0
    assert clip(lib, [array((3, 5), (1, 3))]) > 0                     # dense, another order
    assert clip(lib, g, [array((100,), data=0x40000), array((3, 5), data=0x50000), array((0,), data=0)]) > 0
    for bad in (math.nan, -1.0):
        assert clip(lib, g, max_norm=bad) == -abi.TL_ERR_INVALID
    assert clip(lib, [array((3, 5), (6, 1))]) == -abi.TL_ERR_INVALID  # gaps
    assert clip(lib, [array((3, 5), (0, 1))]) == -abi.TL_ERR_INVALID  # the same element again
    assert clip(lib, [g[0], g[0]]) == -abi.TL_ERR_INVALID             # the same array twice
    assert clip(lib, [g[0], array((4,), data=0x10000 + 396)]) == -abi.TL_ERR_INVALID
    assert clip(lib, [array((4,), data=0)]) == -abi.TL_ERR_INVALID
    assert clip(lib, [array((4,), dtype=3)]) == -abi.TL_ERR_INVALID
    two = [array((4,), data=0x1000), array((4,), data=0x2000)]
    assert clip(lib, two, [array((4,), data=0x3000), array((5,), data=0x4000)]) == -abi.TL_ERR_INVALID
    assert clip(lib, two, [array((4,), data=0x3000), array((4,), data=0x1008)]) == -abi.TL_ERR_INVALID
    # an array read twice is allowed where it is not written
    assert clip(lib, [two[0], two[0]], [array((4,), data=0x3000), array((4,), data=0x4000)]) > 0
    assert lib.tl_clip_workspace(None, None, None, 2, 1.0) == -abi.TL_ERR_INVALID


class DeviceArray:
    """What Context reads of a contiguous device tensor."""
    device = "cuda:0"

    def __init__(self, at, shape, dtype="float32"):
        self.at, self.shape, self.dtype = at, shape, dtype

    def data_ptr(self):
        return self.at

    def numel(self):
        return math.prod(self.shape)

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def stride(self):
        return tuple(math.prod(self.shape[i + 1:]) for i in range(len(self.shape)))


@pytest.mark.parametrize("count", [1, 2, 16, 17, 60])
def test_clip_lists_of_names_and_arrays(lib, count):
    # names and device arrays pair up the same way in lists of any length
    from tensor_logic_lang_b200.runtime import Context
    shapes = [((40, 3), (7,), (2, 5, 3, 4), (1, 9))[i % 4] for i in range(count)]

    def arrays(at):
        return [DeviceArray(at + 0x1000 * i, s) for i, s in enumerate(shapes)]

    class Named(Context):
        def __init__(self):
            self.device, self.lib, self.h = 0, lib, None
            self.held = dict(zip((f"W{i}" for i in range(count)), arrays(0x10000000)))

        def _view(self, x, what, write=False):
            return super()._view(self.held[x] if isinstance(x, str) else x, what)

    c = Named()
    names, there = list(c.held), arrays(0x20000000)
    mixed = [n if i % 2 else a for i, (n, a) in enumerate(zip(names, arrays(0x30000000)))]
    for grads, out in ((names, there), (there, names), (names, None), (mixed, there), (there, mixed)):
        a, o = c._clip_lists(grads, out)
        assert lib.tl_clip_workspace(None, a, o, count, 1.0) > 0, (grads is names, out is names)
    a, o = c._clip_lists(names, there[1:] + [DeviceArray(0x40000000, (41, 3))])
    assert lib.tl_clip_workspace(None, a, o, count, 1.0) == -abi.TL_ERR_INVALID


def test_null_arguments(lib):
    assert lib.tl_attention_forward(None, None) == abi.TL_ERR_INVALID
    assert lib.tl_attention_backward(None, None) == abi.TL_ERR_INVALID
    assert lib.tl_attention_workspace(None, None, 0) == -abi.TL_ERR_INVALID
    assert lib.tl_clip_gradients(None, None, None, 0, 1.0, None, None, 0, None) == abi.TL_ERR_INVALID
    assert lib.tl_tensor_array(None, 0, None) == abi.TL_ERR_INVALID
    assert lib.tl_device(None) == -1


def test_struct_layout_matches_c(tmp_path):
    import os
    import subprocess
    inc = os.path.join(abi.REPO_DIR, "include")
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tl_cuda.h"\n'
                   'int main(void){printf("%zu %zu %zu %zu\\n", sizeof(tl_array), sizeof(tl_attention),'
                   ' offsetof(tl_attention, lse), offsetof(tl_attention, stream)); return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(abi.Array), C.sizeof(abi.Attention), abi.Attention.lse.offset, abi.Attention.stream.offset]
