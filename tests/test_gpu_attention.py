"""Attention with modified scores and its gradient against 64-bit formulas (attention_ref)."""
import numpy as np
import pytest

from attention_ref import TYPES, check, reference

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    from tensor_logic_lang_b200.runtime import Context
    c = Context(device=0)
    yield c
    c.close()


def stream():
    return torch.cuda.current_stream().cuda_stream


def heads(gen, b, h, n, d, dtype, layout="bhsd"):
    """A [b, h, n, d] array in one of several memory layouts."""
    t = TYPES[dtype]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(t)
    if layout == "bshd":
        return randn(b, n, h, d).transpose(1, 2)
    if layout == "packed":                     # a third of a joint projection
        return randn(b, n, 3, h, d)[:, :, 1].transpose(1, 2)
    if layout == "odd":                        # rows of d + 1, the array one element off its allocation
        return randn(b * h * n * (d + 1) + 1)[1:].view(b, h, n, d + 1)[..., :d]
    if layout == "dim":                        # head size not the contiguous dim
        return randn(b, h, d, n).transpose(2, 3)
    if layout == "broadcast":                  # one head's values for all, in every sequence
        return randn(1, 1, n, d).expand(b, h, n, d)
    return randn(b, h, n, d)


def like(x, layout):
    """An array to write in, with what it must not keep, in a layout of its own."""
    b, h, n, d = x.shape
    if layout in ("bhsd", "broadcast"):
        y = torch.empty((b, h, n, d), dtype=x.dtype, device=x.device)
    elif layout == "odd":
        y = torch.empty((b, h, n, d + 1), dtype=x.dtype, device=x.device)[..., :d]
    elif layout == "dim":
        y = torch.empty((b, h, d, n), dtype=x.dtype, device=x.device).transpose(2, 3)
    else:
        y = torch.empty((b, n, h, d), dtype=x.dtype, device=x.device).transpose(1, 2)
    return y.fill_(float("nan"))


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def modifiers(names, b, hq, nq, nk, seed):
    rng = np.random.default_rng(seed)
    m = {}
    if "cap" in names:
        m["softcap"] = 1.5                      # bends the scores of these inputs well
    if "slopes" in names:
        m["slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / hq) for h in range(hq)], device="cuda")
    if "causal" in names or "prefix" in names:
        m["causal"] = True
    if "prefix" in names:
        m["prefix_len"] = ints([int(x) for x in rng.integers(0, nk + 2, b)])
    if "docs" in names:                         # packed documents, padding between and behind them
        def row(n):
            r = np.sort(rng.integers(0, 4, n))
            r[rng.random(n) < 0.1] = -1
            return r
        m["q_doc"] = ints(np.stack([row(nq) for _ in range(b)])) if nq else ints(np.zeros((b, 0)))
        m["k_doc"] = m["q_doc"] if nq == nk else ints(np.stack([row(nk) for _ in range(b)])) if nk else \
            ints(np.zeros((b, 0)))
    if "ids" in names:                          # documents in no order
        m["q_doc"], m["k_doc"] = ints(rng.integers(-1, 3, (b, nq))), ints(rng.integers(-1, 3, (b, nk)))
    if "len" in names:                          # from no key to more than there are
        m["kv_len"] = ints([(0, nk, nk // 2 + 1, nk + 5, 1)[i % 5] for i in range(b)])
    if "start" in names:
        m["q_start"] = ints([(0, -3, nk // 2, 2 * nk)[i % 4] for i in range(b)])
    return m


def poison(x, ok):
    """Infinities and NaN where what an array holds must not matter."""
    if ok is not None and not bool(ok.all()):
        bad = torch.where(torch.arange(x.shape[2], device=x.device) % 2 == 0, float("nan"), float("inf")).to(x.dtype)
        x.copy_(torch.where(ok[:, None, :, None], x, bad[None, None, :, None].expand_as(x)))


def run(ctx, q, k, v, dout, m, layout="bhsd", **kw):
    out = like(q, layout)
    lse = torch.full(q.shape[:3], float("nan"), device="cuda")
    ctx.attention(q, k, v, out, lse, stream=stream(), **m, **kw)
    got = {"out": out, "lse": lse}
    if dout is not None:
        got["dq"], got["dk"], got["dv"] = like(q, layout), like(k, layout), like(v, layout)
        ctx.attention_backward(q, k, v, out, lse, dout, got["dq"], got["dk"], got["dv"], stream=stream(), **m, **kw)
    torch.cuda.synchronize()
    ctx.sync()
    return got


def compare(ctx, b, hq, hkv, nq, nk, d, dtype, names="", layout="bhsd", seed=0, backward=True, gain=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = heads(gen, b, hq, nq, d, dtype, "bhsd" if layout == "broadcast" else layout)
    if gain != 1.0:
        q.mul_(gain)
    k, v = heads(gen, b, hkv, nk, d, dtype, layout), heads(gen, b, hkv, nk, d, dtype, layout)
    dout = heads(gen, b, hq, nq, d, dtype, "bshd") if backward else None
    m = modifiers(names, b, hq, nq, nk, seed)
    if layout != "broadcast":
        k_ok = torch.ones((b, nk), dtype=torch.bool, device="cuda")
        if "kv_len" in m:
            k_ok &= torch.arange(nk, device="cuda")[None] < m["kv_len"][:, None]
        if "k_doc" in m:
            k_ok &= m["k_doc"] >= 0
        poison(k, k_ok)
        poison(v, k_ok)
    if "q_doc" in m:
        poison(q, m["q_doc"] >= 0)
        if backward:
            poison(dout, m["q_doc"] >= 0)
    want = reference(q, k, v, dout, **m)
    got = run(ctx, q, k, v, dout, m, layout)
    for n in want:
        check(got[n], want[n], n)
    return got


MODIFIERS = ["", "cap", "slopes", "causal", "prefix", "docs", "ids", "len", "causal start", "cap slopes causal docs",
             "cap prefix len start", "slopes docs len"]
SIZES = [(1, 1, 1, 1, 1, 64), (2, 4, 2, 7, 5, 64), (1, 2, 2, 64, 64, 64), (5, 2, 1, 65, 129, 64),
         (2, 3, 3, 200, 333, 128), (1, 8, 1, 257, 257, 128), (4, 2, 1, 130, 31, 80), (2, 4, 4, 3, 300, 128),
         (1, 6, 2, 300, 300, 40)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("names", MODIFIERS)
def test_modifiers(ctx, names, dtype):
    for i, size in enumerate(SIZES):
        compare(ctx, *size, dtype, names, seed=i)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [1, 8, 32, 33, 72, 96, 120, 129, 192, 256])
def test_head_sizes(ctx, d, dtype):
    compare(ctx, 2, 2, 1, 70, 90, d, dtype, "cap causal", seed=d)
    compare(ctx, 2, 2, 2, 2, 90, d, dtype, "slopes len", seed=d)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["bshd", "packed", "odd", "dim", "broadcast"])
def test_layouts(ctx, layout, dtype):
    for nq in (1, 140):
        compare(ctx, 2, 4, 2, nq, 140, 64, dtype, "cap causal len", layout, seed=3)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("step", [8, 3, 0])
def test_rows_that_overlap(ctx, step, dtype):
    # windows over one row of memory: neighbouring positions share elements, or all of them
    gen = torch.Generator(device="cuda").manual_seed(11)

    def windows(b, h, n, d):
        room = n * step + d + 8 - d % 8
        return torch.randn((b, h, room), generator=gen, device="cuda").to(TYPES[dtype]).as_strided((b, h, n, d), (h * room, room, step, 1))
    for nq in (1, 5, 140):
        q, k, v, dout = windows(2, 4, nq, 64), windows(2, 2, 140, 64), windows(2, 2, 140, 64), windows(2, 4, nq, 64)
        m = {"causal": True, "softcap": 3.0}
        got, want = run(ctx, q, k, v, dout, m, "bshd"), reference(q, k, v, dout, **m)
        for n in want:
            check(got[n], want[n], (nq, n))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nk", [(0, 5), (5, 0), (0, 0)])
def test_nothing_to_attend(ctx, nq, nk, dtype):
    got = compare(ctx, 2, 2, 1, nq, nk, 64, dtype)
    for n in ("out", "dq", "dk", "dv"):
        assert not got[n].float().any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nk", [(1, 4097), (2, 1000), (513, 2050), (1500, 1500)])
def test_longer(ctx, nq, nk, dtype):
    compare(ctx, 2, 4, 2, nq, nk, 128, dtype, "cap causal", seed=nq, backward=nk < 2048)
    compare(ctx, 2, 4, 2, nq, nk, 64, dtype, "slopes docs", seed=nq, backward=nk < 2048)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_large_scores(ctx, dtype):
    # rows whose largest key has nearly all of the weight, met late in the row
    compare(ctx, 1, 2, 2, 300, 700, 64, dtype, "", seed=1, gain=6.0)
    compare(ctx, 1, 2, 2, 1, 700, 64, dtype, "", seed=1, gain=6.0)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_small_gradients(ctx, dtype):
    # dout far below 1, as without a loss scale: the gradients keep their bits
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (heads(gen, 1, 2, 400, 64, dtype) for _ in range(3))
    dout = heads(gen, 1, 2, 400, 64, dtype)
    small = (dout.float() * 2.0 ** -10).to(dout.dtype)
    m = {"causal": True}
    want = reference(q, k, v, dout, **m)
    got = run(ctx, q, k, v, small, m)
    for n in ("dq", "dk", "dv"):
        value, bound = want[n]
        check(got[n], (value * 2.0 ** -10, bound * 2.0 ** -10 + 2.0 ** -24), n)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_against_differences(ctx, dtype):
    # sum(out * dout) in 64 bits moves along a direction as the gradients say
    gen = torch.Generator(device="cuda").manual_seed(9)
    q, k, v, dout = (heads(gen, 1, 2, 40, 16, dtype) for _ in range(4))
    m = modifiers("cap slopes causal", 1, 2, 40, 40, 0)
    got = run(ctx, q, k, v, dout, m)
    for n, x in (("dq", q), ("dk", k), ("dv", v)):
        step = torch.randn(x.shape, generator=gen, device="cuda").double()
        ends = []
        for sign in (1e-4, -1e-4):
            moved = {"q": q.double(), "k": k.double(), "v": v.double()}
            moved[n[1]] = moved[n[1]] + sign * step
            ends.append((reference(moved["q"], moved["k"], moved["v"], **m)["out"][0] * dout.double()).sum().item())
        slope = (ends[0] - ends[1]) / 2e-4
        # differences: 1e-8 of the values; the gradient: its bound summed along the direction
        bound = (reference(q, k, v, dout, **m)[n][1] * step.abs()).sum().item() + 1e-6 * (1 + abs(slope))
        assert abs((got[n].double() * step).sum().item() - slope) <= bound


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_runs_repeat_bit_for_bit(ctx, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    for nq in (1, 600):
        q, dout = heads(gen, 2, 8, nq, 64, dtype), heads(gen, 2, 8, nq, 64, dtype)
        k, v = heads(gen, 2, 2, 1100, 64, dtype), heads(gen, 2, 2, 1100, 64, dtype)
        first = run(ctx, q, k, v, dout, {"causal": True, "softcap": 5.0})
        for _ in range(3):
            again = run(ctx, q, k, v, dout, {"causal": True, "softcap": 5.0})
            for n in first:
                assert torch.equal(first[n], again[n]), n


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,nq,nk,d", [(8, 2, 30, 700, 64), (8, 1, 9, 1300, 128), (4, 1, 18, 155, 128), (64, 8, 3, 300, 64),
                                            (24, 8, 17, 600, 100), (16, 2, 40, 40, 32)])
def test_what_ran_before_leaves_no_trace(ctx, hq, hkv, nq, nk, d, dtype):
    # tiles that hold fewer queries than rows: shared memory that other calls left behind does not show in a bit
    gen = torch.Generator(device="cuda").manual_seed(nq)
    q, k, v = heads(gen, 2, hq, nq, d, dtype), heads(gen, 2, hkv, nk, d, dtype), heads(gen, 2, hkv, nk, d, dtype)
    q.mul_(4.0)
    others = [[x.mul_(by) for x in (heads(gen, 2, 16, 256, 128, t), *(heads(gen, 2, 4, 512, 128, t) for _ in range(2)))]
              for t in ("bf16", "f32") for by in (0.0, 1.0, 30.0)]
    for m in ({"causal": True}, {"softcap": 3.0}, {"slopes": torch.full((hq,), 0.02, device="cuda")}):
        first = run(ctx, q, k, v, None, m)
        for a, b, c in others:
            for _ in range(2):
                ctx.attention(a, b, c, torch.empty_like(a), stream=stream())
            again = run(ctx, q, k, v, None, m)
            for n in first:
                assert torch.equal(first[n], again[n]), n


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("names", ["len cap", "docs cap", "ids cap causal", "len docs cap slopes", "len docs", "ids causal slopes"])
@pytest.mark.parametrize("size", [(3, 8, 2, 1, 700, 64), (3, 4, 2, 3, 300, 128), (2, 4, 1, 60, 60, 40), (2, 2, 2, 300, 300, 128),
                                  (3, 4, 2, 150, 333, 64), (2, 6, 2, 11, 150, 192)])
def test_padding_leaves_no_trace(ctx, size, names, dtype):
    # what padding holds does not show in a bit of any result
    b, hq, hkv, nq, nk, d = size
    gen = torch.Generator(device="cuda").manual_seed(nk)
    arrays = [heads(gen, b, h, n, d, dtype) for h, n in ((hq, nq), (hkv, nk), (hkv, nk), (hq, nq))]
    m = modifiers(names, b, hq, nq, nk, 1)
    k_ok = torch.arange(nk, device="cuda")[None] < m.get("kv_len", ints([nk] * b))[:, None]
    q_ok = torch.ones((b, nq), dtype=torch.bool, device="cuda")
    if "k_doc" in m:
        k_ok, q_ok = k_ok & (m["k_doc"] >= 0), m["q_doc"] >= 0
    first = {}
    for fill in (0.0, -3.0, 1000.0, float("inf"), float("nan")):
        q, k, v, dout = (torch.where(ok[:, None, :, None], x, torch.full_like(x, fill))
                         for x, ok in zip(arrays, (q_ok, k_ok, k_ok, q_ok)))
        for softcap in (6.0, 30.0) if "cap" in names else (0.0,):
            got = run(ctx, q, k, v, dout, dict(m, softcap=softcap))
            if fill == 0.0:
                first[softcap] = got
            for n in got:
                assert torch.equal(got[n], first[softcap][n]), (fill, softcap, n)


@pytest.mark.parametrize("nq", [1, 200])
def test_captured_and_replayed(ctx, nq):
    # two graphs with workspaces of their own, replayed side by side on new values
    gen = torch.Generator(device="cuda").manual_seed(4)
    kept = []
    for i in range(2):
        q, dout = heads(gen, 2, 4, nq, 64, "bf16"), heads(gen, 2, 4, nq, 64, "bf16")
        k, v = heads(gen, 2, 2, 2000, 64, "bf16"), heads(gen, 2, 2, 2000, 64, "bf16")
        out, lse = like(q, "bhsd"), torch.empty(q.shape[:3], device="cuda")
        g = (dout, like(q, "bhsd"), like(k, "bhsd"), like(v, "bhsd"))
        m = {"causal": True, "softcap": 4.0}
        ws = torch.empty(256 + max(ctx.attention_workspace(q, k, v, out, lse, **m),
                                   ctx.attention_workspace(q, k, v, out, lse, g, **m)), dtype=torch.uint8, device="cuda")

        def step():
            ctx.attention(q, k, v, out, lse, stream=stream(), workspace=ws, **m)
            ctx.attention_backward(q, k, v, out, lse, *g, stream=stream(), workspace=ws, **m)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        kept.append((graph, q, k, v, out, lse, g, m))
    streams = [torch.cuda.Stream() for _ in kept]
    for _ in range(2):
        for _, q, k, v, out, lse, g, m in kept:
            for x in (q, k, v, g[0]):
                x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        torch.cuda.synchronize()
        for s, (graph, *_) in zip(streams, kept):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, q, k, v, out, lse, g, m in kept:
            want = reference(q, k, v, g[0], **m)
            for n, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *g[1:])):
                check(x, want[n], n)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("b,hkv,nk", [
    (4, 8, 50),        # more units than clusters find SMs for, a tile each: every unit lies in one block
    (64, 8, 30), (37, 8, 64),
    (3, 8, 333)])      # units that lie over several blocks
def test_few_rows_are_written_when_the_call_ends(ctx, b, hkv, nk, dtype):
    # the next node of a captured graph takes what the call wrote
    gen = torch.Generator(device="cuda").manual_seed(b)
    q, k, v = heads(gen, b, 2 * hkv, 1, 128, dtype), heads(gen, b, hkv, nk, 128, dtype), heads(gen, b, hkv, nk, 128, dtype)
    out, lse = like(q, "bhsd"), torch.empty(q.shape[:3], device="cuda")
    kept, kept_lse = torch.empty_like(out), torch.empty_like(lse)
    m = {"causal": True, "softcap": 3.0}
    ws = torch.empty(256 + ctx.attention_workspace(q, k, v, out, lse, **m), dtype=torch.uint8, device="cuda")
    ws = ws[-ws.data_ptr() % 256:]

    def step():
        out.fill_(float("nan")), lse.fill_(float("nan"))
        ctx.attention(q, k, v, out, lse, stream=stream(), workspace=ws, **m)
        kept.copy_(out), kept_lse.copy_(lse)
        k.mul_(-1.0)                            # the cache moves on
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(10):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        want = reference(q, k, v, **m)
        graph.replay()
        check(kept, want["out"], "out")
        check(kept_lse, want["lse"], "lse")


@pytest.mark.parametrize("names", ["docs", "docs len causal", ""])
def test_graphs_that_take_turns_share_a_workspace(ctx, names):
    # two captured calls of different sizes, one replayed when the other's work is done
    gen = torch.Generator(device="cuda").manual_seed(14)
    kept, ws = [], torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    for b, hkv, nq, nk, dtype in ((3, 8, 2, 900, "bf16"), (2, 2, 60, 300, "f32")):
        q, k, v = heads(gen, b, 2 * hkv, nq, 64, dtype), heads(gen, b, hkv, nk, 64, dtype), heads(gen, b, hkv, nk, 64, dtype)
        out, lse = like(q, "bhsd"), torch.empty(q.shape[:3], device="cuda")
        m = modifiers(names, b, 2 * hkv, nq, nk, 3)
        assert ctx.attention_workspace(q, k, v, out, lse, **m) <= ws.numel()
        ctx.attention(q, k, v, out, lse, workspace=ws, stream=stream(), **m)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ctx.attention(q, k, v, out, lse, workspace=ws, stream=stream(), **m)
        kept.append((graph, q, k, v, out, lse, m))
    for _ in range(3):
        for graph, q, k, v, out, lse, m in kept:
            v.copy_(torch.randn(v.shape, generator=gen, device="cuda"))
            graph.replay()
            want = reference(q, k, v, **m)
            check(out, want["out"], "out")
            check(lse, want["lse"], "lse")


def test_capture_needs_a_workspace(ctx):
    from tensor_logic_lang_b200 import abi
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, k, v, dout = (heads(gen, 1, 2, 64, 64, "bf16") for _ in range(4))
    got = run(ctx, q, k, v, dout, {})
    graph = torch.cuda.CUDAGraph()
    said = []
    with torch.cuda.graph(graph):
        q.add_(0)
        try:
            ctx.attention_backward(q, k, v, got["out"], got["lse"], dout, got["dq"], got["dk"], got["dv"], stream=stream())
        except abi.TLError as e:
            said.append(e)
    assert said and said[0].status == abi.TL_ERR_INVALID and "capture" in str(said[0])


def test_workspace_is_checked(ctx):
    from tensor_logic_lang_b200 import abi
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, k, v, dout = (heads(gen, 1, 2, 64, 64, "bf16") for _ in range(4))
    got = run(ctx, q, k, v, dout, {})
    need = ctx.attention_workspace(q, k, v, got["out"], got["lse"], (dout, got["dq"], got["dk"], got["dv"]))
    room = torch.empty(need + 512, dtype=torch.uint8, device="cuda")
    off = -room.data_ptr() % 256
    before = room.clone()
    for ws in (room[off:off + need - 1], room[off + 1:off + 1 + need]):
        with pytest.raises(abi.TLError):
            ctx.attention_backward(q, k, v, got["out"], got["lse"], dout, got["dq"], got["dk"], got["dv"], workspace=ws,
                                   stream=stream())
    assert torch.equal(before, room)
    again = run(ctx, q, k, v, dout, {})
    ctx.attention_backward(q, k, v, got["out"], got["lse"], dout, got["dq"], got["dk"], got["dv"],
                           workspace=room[off:off + need], stream=stream())
    torch.cuda.synchronize()
    for n in got:
        assert torch.equal(got[n], again[n])
    assert torch.equal(before[:off], room[:off]) and torch.equal(before[off + need:], room[off + need:])


def test_streams_side_by_side(ctx):
    # the context keeps a workspace for each stream
    gen = torch.Generator(device="cuda").manual_seed(8)
    jobs = []
    for i in range(4):
        q, dout = heads(gen, 1, 4, 300, 64, "f16"), heads(gen, 1, 4, 300, 64, "f16")
        k, v = heads(gen, 1, 2, 500, 64, "f16"), heads(gen, 1, 2, 500, 64, "f16")
        jobs.append((torch.cuda.Stream(), q, k, v, dout))
    torch.cuda.synchronize()
    results = []
    for _ in range(3):
        results = []
        for s, q, k, v, dout in jobs:
            with torch.cuda.stream(s):
                out, lse = like(q, "bhsd"), torch.empty(q.shape[:3], device="cuda")
                g = (like(q, "bhsd"), like(k, "bhsd"), like(v, "bhsd"))
                ctx.attention(q, k, v, out, lse, causal=True, stream=s.cuda_stream)
                ctx.attention_backward(q, k, v, out, lse, dout, *g, causal=True, stream=s.cuda_stream)
                results.append((out, lse, *g))
    torch.cuda.synchronize()
    for (s, q, k, v, dout), got in zip(jobs, results):
        want = reference(q, k, v, dout, causal=True)
        for n, x in zip(("out", "lse", "dq", "dk", "dv"), got):
            check(x, want[n], n)


def test_calls_after_one_that_found_no_memory(ctx):
    from tensor_logic_lang_b200 import abi
    gen = torch.Generator(device="cuda").manual_seed(4)
    # dk and dv of 8192 heads that share their keys, 430 GB, before they are added up
    q, k = torch.zeros((1, 8192, 1, 100), device="cuda"), torch.zeros((1, 1, 65536, 100), device="cuda")
    lse, dk, dv = torch.zeros(q.shape[:3], device="cuda"), torch.empty_like(k), torch.empty_like(k)
    assert ctx.attention_workspace(q, k, k, q, lse, (q, torch.empty_like(q), dk, dv)) > torch.cuda.get_device_properties(0).total_memory
    with pytest.raises(abi.TLError) as said:
        ctx.attention_backward(q, k, k, q, lse, q, torch.empty_like(q), dk, dv, stream=stream())
    assert said.value.status == abi.TL_ERR_OOM
    compare(ctx, 1, 2, 1, 100, 100, 64, "f32", "causal")
    compare(ctx, 1, 2, 1, 100, 100, 64, "bf16", "causal")
    torch.cuda.synchronize()


def test_refusals_do_nothing(ctx):
    from tensor_logic_lang_b200 import abi
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (heads(gen, 1, 2, 64, 64, "bf16") for _ in range(3))
    out = torch.full_like(q, 7.0)
    for bad in (dict(q=q.cpu()), dict(out=out.float()), dict(v=v[:, :, 1:]), dict(out=q), dict(k=k[..., :32]),
                dict(q=q.double()), dict(q=q[0, 0, 0])):
        with pytest.raises(abi.TLError):
            ctx.attention(bad.get("q", q), bad.get("k", k), bad.get("v", v), bad.get("out", out), stream=stream())
    for bad in (dict(softcap=-1.0), dict(prefix_len=ints([3])), dict(q_doc=ints([[0] * 64])), dict(kv_len=ints([1, 2])),
                dict(kv_len=torch.tensor([3], device="cuda")), dict(slopes=torch.ones(2)),
                dict(slopes=torch.ones(2, dtype=torch.float64, device="cuda")),
                dict(q_doc=ints([[0] * 128])[:, ::2], k_doc=ints([[0] * 64]))):
        with pytest.raises(abi.TLError):
            ctx.attention(q, k, v, out, stream=stream(), **bad)
    torch.cuda.synchronize()
    assert (out == 7.0).all()


def test_rows_outside_are_left(ctx):
    # outputs inside larger buffers: what surrounds them stays
    gen = torch.Generator(device="cuda").manual_seed(6)
    for nq, nk in ((1, 100), (100, 100), (130, 130)):
        q, k, v, dout = heads(gen, 2, 2, nq, 72, "bf16"), heads(gen, 2, 2, nk, 72, "bf16"), \
            heads(gen, 2, 2, nk, 72, "bf16"), heads(gen, 2, 2, nq, 72, "bf16")
        rooms = [torch.full((2, 2, n + 3, 80), 7.0, device="cuda", dtype=torch.bfloat16) for n in (nq, nq, nk, nk)]
        out, dq, dk, dv = (r[:, :, 1:-2, :72] for r in rooms)
        lse = torch.empty((2, 2, nq), device="cuda")
        ctx.attention(q, k, v, out, lse, stream=stream())
        ctx.attention_backward(q, k, v, out, lse, dout, dq, dk, dv, stream=stream())
        torch.cuda.synchronize()
        want = reference(q, k, v, dout)
        for n, x in zip(("out", "dq", "dk", "dv"), (out, dq, dk, dv)):
            check(x, want[n], n)
            x.fill_(7.0)
        for r in rooms:
            assert (r == 7.0).all()


def test_named_tensors(ctx):
    # the storage of a program's tensors, on the context's own stream
    from tensor_logic_lang_b200 import lang
    rng = np.random.default_rng(3)
    s, e, d = 96, 24, 16
    data = {n: rng.standard_normal(shape) for n, shape in
            (("X", (s, e)), ("Wq", (e, d)), ("Wk", (e, d)), ("Wv", (e, d)))}
    src = "".join(f"domain {n}: {k}\n" for n, k in (("s", s), ("e", e), ("d", d)))
    src += "".join(f"{n}[{ix}] = 0\nload {n} \"{n}.bin\"\n" for n, ix in (("X", "s,e"), ("Wq", "e,d"), ("Wk", "e,d"), ("Wv", "e,d")))
    src += "".join(f"{n}[s,d] = X[s,e] W{n.lower()}[e,d]\n" for n in "QKV")
    ctx.run(lang.Program(src, inputs=data))
    ctx.create("O", (s, d))
    ctx.create("Lse", (1, s))
    ctx.attention("Q", "K", "V", "O", "Lse", causal=True, softcap=30.0)
    q, k, v = (torch.tensor(ctx.tensor(n), device="cuda", dtype=torch.float32)[None, None] for n in "QKV")
    want = reference(q, k, v, causal=True, softcap=30.0)
    check(torch.tensor(ctx.tensor("O"), device="cuda")[None, None], want["out"], "O")
    check(torch.tensor(ctx.tensor("Lse"), device="cuda")[None], want["lse"], "Lse")


def test_training_step_of_a_program(ctx):
    """Projections and their gradients from a program, attention and its gradient between them, the gradients
    clipped: the calls as a training step makes them, on the context's stream."""
    from tensor_logic_lang_b200 import lang
    rng = np.random.default_rng(4)
    s, e, d = 80, 32, 32
    x, w = rng.standard_normal((s, e)), {n: rng.standard_normal((e, d)) / e ** 0.5 for n in ("Wq", "Wk", "Wv")}
    g_out = rng.standard_normal((s, d))
    doms = "".join(f"domain {n}: {k}\n" for n, k in (("s", s), ("e", e), ("d", d)))
    src = doms + "X[s,e] = 0\nload X \"x\"\n"
    src += "".join(f"W{n}[e,d] = 0\nload W{n} \"{n}\"\n{n.upper()}[s,d] = X[s,e] W{n}[e,d]\n" for n in "qkv")
    ctx.run(lang.Program(src, inputs=dict(w, X=x)))
    for n, shape in (("O", (s, d)), ("Lse", (1, s)), ("dO", (s, d)), ("dQ", (s, d)), ("dK", (s, d)), ("dV", (s, d))):
        ctx.create(n, shape)
    ctx.upload("dO", g_out)
    m = dict(causal=True, softcap=20.0)
    ctx.attention("Q", "K", "V", "O", "Lse", **m)
    ctx.attention_backward("Q", "K", "V", "O", "Lse", "dO", "dQ", "dK", "dV", **m)
    back = {n: ctx.tensor(n) for n in ("dQ", "dK", "dV")}
    src = doms + "X[s,e] = 0\nload X \"x\"\n"
    src += "".join(f"G{n}[s,d] = 0\nload G{n} \"{n}\"\nd{n}[e,d] = X[s,e] G{n}[s,d]\n" for n in "QKV")
    ctx.run(lang.Program(src, inputs={"X": x, "GQ": back["dQ"], "GK": back["dK"], "GV": back["dV"]}))
    ctx.create("Norm", (1,))
    before = {n: ctx.tensor(n) for n in ("dQ", "dK", "dV")}
    ctx.clip_gradients(["dQ", "dK", "dV"], 0.5, norm="Norm")
    # the same in 64 bits
    X = torch.tensor(x, device="cuda")
    leaf = {n: torch.tensor(v, device="cuda") for n, v in w.items()}
    q, k, v = (X @ leaf[n] for n in ("Wq", "Wk", "Wv"))
    ref = reference(q[None, None], k[None, None], v[None, None], torch.tensor(g_out, device="cuda")[None, None], **m)
    grads = {n: X.T @ ref[n.lower()][0][0, 0] for n in ("dQ", "dK", "dV")}
    norm = torch.sqrt(sum((t ** 2).sum() for t in grads.values())).item()
    assert norm > 0.5
    assert abs(ctx.tensor("Norm")[0] - norm) <= 1e-4 * norm
    for n, t in grads.items():
        t = t.cpu().numpy()
        assert np.abs(before[n] - t).max() <= 1e-3 * np.abs(t).max()
        assert np.abs(ctx.tensor(n) - t * (0.5 / norm)).max() <= 1e-3 * np.abs(t).max() * 0.5 / norm


@pytest.mark.parametrize("cap", [50.0, 50.2, 50.3, 1000.0])
def test_cap_at_the_ends_of_the_tanh(ctx, cap):
    # scores far past the cap on either side, for rows of all high, all low and mixed ones
    gen = torch.Generator(device="cuda").manual_seed(3)
    for dtype in ("bf16", "f16", "f32"):
        for nq in (1, 150):
            q, k, v = heads(gen, 1, 4, nq, 64, dtype), heads(gen, 1, 2, 300, 64, dtype), heads(gen, 1, 2, 300, 64, dtype)
            q[:, 0].abs_(), q[:, 1].abs_().neg_(), k[:, 0].abs_()
            q.mul_(40.0)
            dout = heads(gen, 1, 4, nq, 64, dtype)
            m = {"softcap": cap, "causal": True}
            want = reference(q, k, v, dout, **m)
            got = run(ctx, q, k, v, dout, m)
            for n in want:
                check(got[n], want[n], (dtype, nq, n))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("power", [-40, -30, -20, -12, 12, 30])
def test_values_of_any_size_under_a_cap(ctx, power, dtype):
    # rows whose scores all lie near the lower end of the tanh, all near the upper one, or anywhere, and rows
    # that see one key: the exponentials' size does not show in what they weigh
    if dtype == "f16" and not -12 <= power <= 12:
        pytest.skip("outside fp16")
    gen = torch.Generator(device="cuda").manual_seed(13)
    for hq, nq, nk in ((4, 1, 300), (4, 150, 300), (2, 130, 4300), (32, 700, 700)):
        q, k, v = heads(gen, 1, hq, nq, 64, dtype), heads(gen, 1, 2, nk, 64, dtype), heads(gen, 1, 2, nk, 64, dtype)
        k[:, 0].abs_()
        q[:, 0].abs_().neg_(), q[:, hq // 2 - 1].abs_()
        q.mul_(40.0)
        v.mul_(2.0 ** power)
        m = {"softcap": 50.0, "causal": True}
        got, want = run(ctx, q, k, v, None, m), reference(q, k, v, **m)
        for n in ("out", "lse"):
            check(got[n], want[n], (hq, nq, n))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [200.0, 1e4, 1e6, 3e7, 1e8, 1e12])
def test_caps_far_above_the_scores(ctx, cap, dtype):
    # a cap that bends nothing changes nothing: the scores keep their digits beside it
    gen = torch.Generator(device="cuda").manual_seed(3)
    for b, nq, d in ((1, 1, 64), (3, 3, 128), (1, 150, 128), (2, 300, 64)):
        q, k, v = heads(gen, b, 4, nq, d, dtype), heads(gen, b, 2, 400, d, dtype), heads(gen, b, 2, 400, d, dtype)
        q.mul_(2.0)
        dout = heads(gen, b, 4, nq, d, dtype)
        m = {"softcap": cap, "causal": True}
        want = reference(q, k, v, dout, **m)
        got = run(ctx, q, k, v, dout, m)
        for n in want:
            check(got[n], want[n], (nq, n))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [100.0, 1e4, 1e5])
def test_large_and_small_scores_in_one_tile(ctx, cap, dtype):
    # every third query's scores pass the cap; the rows beside it keep the digits of theirs
    gen = torch.Generator(device="cuda").manual_seed(3)
    for nq in (1, 3, 150):
        q, k, v = heads(gen, 1, 4, nq, 64, dtype), heads(gen, 1, 2, 300, 64, dtype), heads(gen, 1, 2, 300, 64, dtype)
        k.mul_(4.0)
        q.mul_(0.5)
        q[:, 0, ::3].mul_(min(cap, 1e4))        # fp16 ends at 65504
        dout = heads(gen, 1, 4, nq, 64, dtype)
        m = {"softcap": cap, "causal": True}
        want = reference(q, k, v, dout, **m)
        got = run(ctx, q, k, v, dout, m)
        for n in want:
            check(got[n], want[n], (nq, n))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [1e6, 3e7, 1e9])
def test_bent_scores_of_a_large_cap(ctx, cap, dtype):
    # scores up to three quarters of a cap that is 1e7 to 1e10 times the scale: a row's one large weight is
    # that of its largest score, so lse is the bent score itself
    gen = torch.Generator(device="cuda").manual_seed(5)
    for nq in (1, 150):
        q, k, v = heads(gen, 1, 4, nq, 64, dtype), heads(gen, 1, 2, 300, 64, dtype), heads(gen, 1, 2, 300, 64, dtype)
        x = (q.double() @ k.double().repeat_interleave(2, 1).transpose(-1, -2)).abs().amax().item() * 64 ** -0.5
        q.mul_(0.74 * cap / x)
        m = {"softcap": cap}
        got = run(ctx, q, k, v, None, m)
        check(got["lse"], reference(q, k, v, **m)["lse"], nq)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_caps_at_the_ends_of_their_range(ctx, dtype):
    gen = torch.Generator(device="cuda").manual_seed(6)
    for nq in (1, 3, 150):
        q, k, v = heads(gen, 1, 4, nq, 64, dtype), heads(gen, 1, 2, 300, 64, dtype), heads(gen, 1, 2, 300, 64, dtype)
        q[:, 1] = 0.0                           # scores of 0
        dout = heads(gen, 1, 4, nq, 64, dtype)
        for scale, cap in ((0.125, 2.0 ** -60), (0.125, 2.0 ** -40), (0.125, 2.0 ** 56), (0.125, 2.0 ** 100), (2.0 ** 30, 2.0 ** -30),
                           (-0.125, 2.0 ** -60), (-0.125, 2.0 ** 100)):
            m = {"softcap": cap, "causal": True, "scale": scale}
            want = reference(q, k, v, dout, **m)
            got = run(ctx, q, k, v, dout, m)
            for n in ("out", "lse", "dv"):
                check(got[n], want[n], (nq, scale, cap, n))
            for n in ("dq", "dk"):
                # at q = 0 the tanh is its argument, so dq is 2^30 dx k under a scale of 2^30: past 65504, fp16's
                # largest number, where dx k is above 2^-14
                past = want[n][0].abs() + want[n][1] > torch.finfo(got[n].dtype).max
                assert (torch.isfinite(got[n]) | (past & torch.isinf(got[n]))).all(), (nq, scale, cap, n)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [2.0 ** 12, 2.0 ** 21, 2.0 ** 24, 2.0 ** 30, 2.0 ** 60])
def test_scores_without_a_fraction(ctx, scale, dtype):
    # q.k are whole numbers: a row's weight lies on the keys of its largest score alone, in equal parts, so
    # what is off is v's bits (fp32: 22), the sums' and the result's rounding
    gen = torch.Generator(device="cuda").manual_seed(7)
    for hq, nq, nk in ((2, 1, 300), (4, 150, 700), (1, 130, 4300), (8, 600, 600)):
        q, k, v = heads(gen, 2, hq, nq, 64, dtype), heads(gen, 2, 1, nk, 64, dtype), heads(gen, 2, 1, nk, 64, dtype)
        q.mul_(2.0).round_(), k.mul_(2.0).round_()
        m = {"scale": scale, "causal": True}
        got = run(ctx, q, k, v, None, m)
        # (softmax of 64-bit scores of 2^37 would lose bits of the logarithm of the number of equal parts)
        x = q.double() @ k.double().transpose(-1, -2)
        x = x.masked_fill(~torch.ones((nq, nk), dtype=torch.bool, device="cuda").tril(nk - nq), -np.inf)
        largest = x.amax(-1, keepdim=True)
        w = (x == largest).double()
        out = (w / w.sum(-1, keepdim=True)) @ v.double()
        one = torch.finfo(v.dtype).eps / 2 + 2.0 ** -20
        check(got["out"], (out, one * (out.abs() + v.double().abs().amax())), "out")
        lse = largest[..., 0] * scale + w.sum(-1).log()
        check(got["lse"], (lse, 2.0 ** -22 * lse.abs() + 2.0 ** -16), "lse")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_products_whose_squares_pass_fp32(ctx, dtype):
    # under a cap far above them, which counts as none
    gen = torch.Generator(device="cuda").manual_seed(6)
    for nq in (1, 3, 150):
        q, k, v = heads(gen, 1, 4, nq, 64, dtype), heads(gen, 1, 2, 300, 64, dtype), heads(gen, 1, 2, 300, 64, dtype)
        q.mul_(2.0 ** 40), k.mul_(2.0 ** 40)
        m = {"softcap": 2.0 ** 99, "scale": 2.0 ** -10}
        check(run(ctx, q, k, v, None, m)["lse"], reference(q, k, v, **m)["lse"], nq)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_many_sequences(ctx, dtype):
    # more sequences than a block has threads, most of them short or empty
    for b, nq in ((700, 1), (300, 3), (90, 40)):
        gen = torch.Generator(device="cuda").manual_seed(b)
        q, k, v = heads(gen, b, 2, nq, 32, dtype), heads(gen, b, 1, 200, 32, dtype), heads(gen, b, 1, 200, 32, dtype)
        m = {"causal": True, "kv_len": ints([(7 * i) % 230 if i % 3 else 0 for i in range(b)])}
        got = run(ctx, q, k, v, None, m)
        want = reference(q, k, v, **m)
        for n in want:
            check(got[n], want[n], n)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,nq,nk,d,names", [
    (4, 2, 130, 70, 128, "len"), (3, 1, 260, 90, 64, "cap"), (4, 1, 130, 300, 40, "slopes len"),
    (3, 3, 130, 1100, 64, "causal start"), (4, 2, 129, 1030, 96, "cap causal len start"), (6, 2, 200, 130, 72, "docs"),
    (3, 1, 150, 1040, 24, "cap slopes prefix len start")])
def test_more_tiles_than_the_gpu_holds_at_once(ctx, hq, hkv, nq, nk, d, names, dtype):
    compare(ctx, 52, hq, hkv, nq, nk, d, dtype, names, seed=hq + nk, backward=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("names", ["cap causal start len", "slopes docs len", "ids", "prefix start"])
@pytest.mark.parametrize("b,hq,hkv,nq,nk,d", [
    (3, 8, 1, 1, 900, 128), (2, 18, 2, 1, 333, 64), (4, 8, 2, 6, 700, 128), (2, 8, 1, 5, 1300, 64), (3, 4, 4, 50, 260, 72),
    (2, 32, 1, 2, 5000, 128), (40, 6, 2, 11, 150, 128)])
def test_few_rows(ctx, b, hq, hkv, nq, nk, d, names, dtype):
    # 1 to 64 rows a key head
    compare(ctx, b, hq, hkv, nq, nk, d, dtype, names, seed=nq + nk, backward=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("names", ["cap causal start len", "slopes docs len", "ids", "prefix start", ""])
@pytest.mark.parametrize("b,hq,hkv,nq,nk,d,layout", [
    (2, 6, 2, 50, 700, 128, "bhsd"), (1, 40, 2, 30, 260, 64, "bshd"), (3, 8, 1, 16, 1000, 128, "packed"), (2, 10, 2, 27, 520, 40, "bshd"),
    (1, 128, 1, 3, 1100, 64, "bhsd"), (5, 4, 2, 65, 130, 96, "odd")])
def test_heads_of_a_group_in_one_tile(ctx, b, hq, hkv, nq, nk, d, layout, names, dtype):
    compare(ctx, b, hq, hkv, nq, nk, d, dtype, names, layout=layout, seed=nq + nk, backward=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_queries_broadcast_over_heads(ctx, dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)
    for nq in (2, 20, 150):
        q = heads(gen, 1, 1, nq, 64, dtype).expand(2, 8, nq, 64)
        k, v = heads(gen, 2, 2, 300, 64, dtype), heads(gen, 2, 2, 300, 64, dtype)
        m = {"causal": True, "softcap": 2.0}
        want, got = reference(q, k, v, **m), run(ctx, q, k, v, None, m)
        for n in want:
            check(got[n], want[n], n)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("b,hq,hkv,nq,nk,d,names", [
    (1, 1, 1, 130, 4300, 64, "len start"), (2, 2, 1, 200, 1200, 128, "cap causal start"), (5, 1, 1, 140, 1031, 40, "slopes len"),
    (1, 2, 2, 260, 4200, 72, "docs"), (2, 1, 1, 300, 4100, 64, "ids"), (3, 2, 1, 150, 2100, 96, "cap slopes prefix len start"),
    (4, 5, 1, 257, 700, 32, "causal start len"), (4, 1, 1, 135, 9000, 24, "causal start len")])
def test_few_queries_many_keys(ctx, b, hq, hkv, nq, nk, d, names, dtype):
    # blocks that share the keys of a query tile, some without any
    compare(ctx, b, hq, hkv, nq, nk, d, dtype, names, seed=nk)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [3, 8, 12, 64])
def test_groups(ctx, group, dtype):
    compare(ctx, 2, group, 1, 2, 700, 64, dtype, "cap causal len", seed=group)
    compare(ctx, 1, 2 * group, 2, 140, 140, 128, dtype, "causal", seed=group)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_of_very_different_size(ctx, dtype):
    # heads, and q, k, v, dout, of scales far apart: a head's results keep their digits
    gen = torch.Generator(device="cuda").manual_seed(12)
    q, k, v, dout = (heads(gen, 2, 4, 200, 64, dtype) for _ in range(4))
    for i, s in enumerate((1e-12, 1e-4, 1.0, 1e6)):
        v[:, i].mul_(s)
        dout[:, i].mul_(1 / s)
    k.mul_(1e3)
    q.mul_(1e-3)
    m = {"causal": True}
    want = reference(q, k, v, dout, **m)
    got = run(ctx, q, k, v, dout, m)
    for n in want:
        check(got[n], want[n], n)


@pytest.mark.parametrize("sizes", [(1, 1, 1e-30), (1, 1, 1e30), (1, 1, 1e-37), (1e-25, 1e25, 1), (1e27, 1e-27, 1e20), (1e-30, 1, 1),
                                   (1e-25, 1e-25, 1), (1e17, 1e17, 1e-20), (1e-19, 1e20, 1e-24)])
@pytest.mark.parametrize("d", [64, 100])
def test_fp32_values_of_any_size(ctx, d, sizes):
    # q, k and v anywhere in the range of fp32 keep their digits
    gen = torch.Generator(device="cuda").manual_seed(21)
    for hq, nq, nk, names in ((2, 1, 300, ""), (4, 150, 150, "causal"), (2, 130, 4300, "slopes"), (8, 300, 700, "cap causal")):
        q, k, v = heads(gen, 1, hq, nq, d, "f32"), heads(gen, 1, 2, nk, d, "f32"), heads(gen, 1, 2, nk, d, "f32")
        for x, by in zip((q, k, v), sizes):
            x.mul_(by)
        m = modifiers(names, 1, hq, nq, nk, 0)
        got, want = run(ctx, q, k, v, None, m), reference(q, k, v, **m)
        for n in ("out", "lse"):
            check(got[n], want[n], (hq, nq, n))


@pytest.mark.parametrize("sizes", [(1, 1, 1, 1e-24), (1, 1, 1, 1e20), (1, 1, 1e-20, 1e-10), (1, 1, 1e25, 1e-20), (1, 1, 1e20, 1e15),
                                   (1e-10, 1e10, 1e-15, 1e-15), (1e10, 1e-10, 1e-18, 1e10), (1e-20, 1e20, 1e-30, 1e25), (1, 1, 1e-25, 1e-9)])
@pytest.mark.parametrize("d", [64, 100])
def test_fp32_gradients_of_any_size(ctx, d, sizes):
    gen = torch.Generator(device="cuda").manual_seed(22)
    for hq, nq, nk, names in ((2, 150, 150, "causal"), (4, 300, 260, "cap"), (8, 130, 700, "slopes"), (6, 520, 520, "cap causal")):
        q, k, v = heads(gen, 1, hq, nq, d, "f32"), heads(gen, 1, 2, nk, d, "f32"), heads(gen, 1, 2, nk, d, "f32")
        dout = heads(gen, 1, hq, nq, d, "f32")
        for x, by in zip((q, k, v, dout), sizes):
            x.mul_(by)
        m = modifiers(names, 1, hq, nq, nk, 0)
        got, want = run(ctx, q, k, v, dout, m), reference(q, k, v, dout, **m)
        for n in want:
            check(got[n], want[n], (hq, nq, n))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("size", [2.0 ** -10, 1.0, 2.0 ** 20])
def test_one_infinity_stays_in_its_tiles(ctx, dtype, bad, size):
    # a document of one tile holds values that are not finite; the next document's results are its own
    if dtype == "f16" and size > 1:
        pytest.skip("outside fp16")
    gen = torch.Generator(device="cuda").manual_seed(23)
    for d in (64, 128) if dtype != "f32" else (64, 100):
        for names in ("", "cap", "slopes"):
            q, k = heads(gen, 1, 4, 400, d, dtype), heads(gen, 1, 2, 400, d, dtype)
            v, dout = heads(gen, 1, 2, 400, d, dtype), heads(gen, 1, 4, 400, d, dtype)
            v.mul_(size), dout.mul_(size)
            for x in (q, k, v, dout):
                x[0, 1, 5, 3] = bad
            m = modifiers(names, 1, 4, 400, 400, 0)
            docs = ints([[0] * 128 + [1] * 272])
            got = run(ctx, q, k, v, dout, dict(m, causal=True, q_doc=docs, k_doc=docs))
            want = reference(*(x[:, :, 128:] for x in (q, k, v, dout)), causal=True, **m)
            for n in want:
                check(got[n][:, :, 128:], want[n], n)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", ["dout", "v"])
def test_one_infinity_leaves_small_gradients_their_bits(ctx, where, d):
    # fp16: dx of 2^-22 and keys of 2^12, beside a document with an infinity
    gen = torch.Generator(device="cuda").manual_seed(24)
    q, k = heads(gen, 1, 4, 400, d, "f16"), heads(gen, 1, 2, 400, d, "f16")
    v, dout = heads(gen, 1, 2, 400, d, "f16"), heads(gen, 1, 4, 400, d, "f16")
    q.mul_(2.0 ** -12), k.mul_(2.0 ** 12), dout.mul_(2.0 ** -14)
    (dout if where == "dout" else v)[0, 1, 5, 3] = float("inf")
    docs = ints([[0] * 128 + [1] * 272])
    got = run(ctx, q, k, v, dout, dict(causal=True, q_doc=docs, k_doc=docs))
    want = reference(*(x[:, :, 128:] for x in (q, k, v, dout)), causal=True)
    check(got["dq"][:, :, 128:], want["dq"], "dq")


@pytest.mark.parametrize("d", [64, 80, 128])
def test_fp32_errors_do_not_grow_with_the_tiles(ctx, d):
    # of the norm of a result: a tile's sums are cut 24 times (8 steps of 3 products) by half a
    # last place, 2^-24 each, whatever the number of tiles, and either operand has 22 bits
    gen = torch.Generator(device="cuda").manual_seed(d)
    q, dout = heads(gen, 1, 4, 1300, d, "f32"), heads(gen, 1, 4, 1300, d, "f32")
    k, v = heads(gen, 1, 2, 1300, d, "f32"), heads(gen, 1, 2, 1300, d, "f32")
    got = run(ctx, q, k, v, dout, {"causal": True})
    q6, k6, v6 = (x.double().requires_grad_() for x in (q, k, v))
    s = (q6 @ k6.repeat_interleave(2, 1).transpose(2, 3)) * d ** -0.5
    seen = torch.ones(1300, 1300, dtype=torch.bool, device="cuda").tril()
    o6 = s.masked_fill(~seen, -torch.inf).softmax(-1) @ v6.repeat_interleave(2, 1)
    o6.backward(dout.double())
    for n, want in (("out", o6), ("dq", q6.grad), ("dk", k6.grad), ("dv", v6.grad)):
        assert ((got[n].double() - want).norm() / want.norm()).item() <= 24 * 2.0 ** -24 + 2 * 2.0 ** -22, n


def test_fp32_on_the_cuda_cores():
    # a context of that precision keeps all 24 bits of the operands
    from tensor_logic_lang_b200 import abi
    from tensor_logic_lang_b200.runtime import Context
    c = Context(device=0, precision=abi.PREC_FP32)
    try:
        c.profile(True)
        compare(c, 2, 4, 2, 100, 130, 64, "f32", "cap causal")
        names = set(c.profile_read())
        assert "attention_general" in names and not any("tc" in n or "split" in n for n in names), names
    finally:
        c.close()


def test_workspace_of_either_precision(ctx):
    # without a context the size is enough for a context of any precision
    import ctypes as C
    from tensor_logic_lang_b200 import abi
    from tensor_logic_lang_b200.runtime import Context
    gen = torch.Generator(device="cuda").manual_seed(4)
    c = Context(device=0, precision=abi.PREC_FP32)
    try:
        for hq, nq, nk, d in ((32, 1, 64, 64), (2, 20, 70, 128), (2, 100, 100, 96), (2, 1, 900, 200)):
            q, k, v = heads(gen, 1, hq, nq, d, "f32"), heads(gen, 1, 1, nk, d, "f32"), heads(gen, 1, 1, nk, d, "f32")
            out, lse, dout = like(q, "bhsd"), torch.empty(q.shape[:3], device="cuda"), like(q, "bhsd")
            g = (dout, like(q, "bhsd"), like(k, "bhsd"), like(v, "bhsd"))
            for grads in (None, g):
                fields = ctx._attention(q, k, v, out, lse, grads, None, 0.0, None, False, None, None, None, None, None,
                                        None, None)
                any_context = ctx.lib.tl_attention_workspace(None, C.c_char_p(fields), 1 if grads else 0)
                assert any_context >= max(x.attention_workspace(q, k, v, out, lse, grads) for x in (ctx, c))
    finally:
        c.close()


def test_kernels_that_run(ctx):
    # the kernels the rules of the entry point's documentation name
    gen = torch.Generator(device="cuda").manual_seed(1)
    ctx.profile(True)
    for dtype, nq, d, layout, want in (("bf16", 200, 64, "bhsd", "attention_tc"), ("f32", 200, 64, "bhsd", "attention_tc"),
                                       ("f32", 200, 100, "odd", "attention_tc"), ("f16", 200, 128, "bshd", "attention_tc"),
                                       ("bf16", 200, 100, "bhsd", "attention_general"), ("bf16", 200, 64, "odd", "attention_general"),
                                       ("f16", 200, 192, "bhsd", "attention_general"), ("bf16", 1, 64, "bhsd", "attention_decode"),
                                       ("f32", 3, 64, "bhsd", "attention_decode"), ("f16", 2, 100, "odd", "attention_decode")):
        q, k, v = heads(gen, 1, 2, nq, d, dtype, layout), heads(gen, 1, 2, 300, d, dtype, layout), heads(gen, 1, 2, 300, d, dtype, layout)
        ctx.profile_reset()
        ctx.attention(q, k, v, like(q, "bhsd"), stream=stream())
        assert want in ctx.profile_read(), (dtype, nq, d, layout, set(ctx.profile_read()))
    ctx.profile(False)


def test_offsets_past_32_bits(ctx):
    # a cache whose last keys lie behind 2^32 bytes and 2^31 elements of it
    n, d = (1 << 24) + 77, 128
    k = torch.zeros((1, 1, n, d), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros((1, 1, n, d), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(7)
    tail = 300
    k[:, :, -tail:] = torch.randn((1, 1, tail, d), generator=gen, device="cuda").bfloat16()
    v[:, :, -tail:] = torch.randn((1, 1, tail, d), generator=gen, device="cuda").bfloat16()
    for nq in (1, 130):
        q = (torch.randn((1, 1, nq, d), generator=gen, device="cuda") * 8).bfloat16()
        q = torch.cat([q, q], 1)
        out, lse = like(q, "bhsd"), torch.empty((1, 2, nq), device="cuda")
        ctx.attention(q, k, v, out, lse, causal=True, stream=stream())
        torch.cuda.synchronize()
        # keys of zeros have the score 0 and no value
        want = reference(q, k[:, :, -tail:], v[:, :, -tail:], causal=True)
        x = (q.double() @ k[:, :, -tail:].double().transpose(-1, -2)) * d ** -0.5
        seen = torch.arange(tail, device="cuda")[None] <= torch.arange(nq, device="cuda")[:, None] + tail - nq
        x = x.masked_fill(~seen, float("-inf"))
        total = torch.logsumexp(torch.cat([x, torch.full((1, 2, nq, 1), float(np.log(n - tail)), device="cuda", dtype=torch.float64)], -1), -1)
        value = torch.exp(x - total[..., None]) @ v[:, :, -tail:].double()
        check(out, (value, want["out"][1]), "out")
        assert ((lse.double() - total).abs() <= 1e-4 * total.abs()).all()


def test_named_tensors_stay_on_their_stream(ctx):
    from tensor_logic_lang_b200 import abi
    ctx.create("Xq", (8, 16))
    x = torch.zeros((8, 16), device="cuda")
    with pytest.raises(abi.TLError):
        ctx.attention("Xq", x, x, torch.empty_like(x), stream=stream())


def test_names_are_marked_as_written_by_calls_that_write(ctx):
    # asking for a workspace, a refused call and reading leave a 0/1 tensor one (with its bit rows)
    from tensor_logic_lang_b200 import abi
    rows, d = 24, 16
    gen = np.random.default_rng(1)
    for n in ("Mq", "Mk", "Mv", "Mdo"):
        ctx.create(n, (rows, d))
        ctx.upload(n, gen.standard_normal((rows, d)))
    out, lse, grads = "Mo", "Mlse", ("Mdq", "Mdk", "Mdv")
    marked = (out, *grads)
    for n in marked:
        ctx.create(n, (rows, d))
    ctx.create(lse, (1, rows))
    ctx.create("Mnorm", (1, 1))
    for n in (*marked, lse, "Mnorm"):
        ctx.upload(n, np.ones(ctx.shape(n)))

    def still(names):
        for n in names:
            assert (ctx.tensor(n) == 1).all()
            ctx.bits(n)                         # refused where a tensor may hold other values
    ctx.attention_workspace("Mq", "Mk", "Mv", out, lse)
    ctx.attention_workspace("Mq", "Mk", "Mv", out, lse, ("Mdo", *grads))
    ctx.clip_workspace(list(grads), 1.0)
    for bad in (dict(softcap=-1.0), dict(prefix_len=ints([3]))):
        with pytest.raises(abi.TLError):
            ctx.attention("Mq", "Mk", "Mv", out, lse, **bad)
        with pytest.raises(abi.TLError):
            ctx.attention_backward("Mq", "Mk", "Mv", out, lse, "Mdo", *grads, **bad)
    with pytest.raises(abi.TLError):
        ctx.clip_gradients(list(grads), -1.0, norm="Mnorm")
    still((*marked, lse, "Mnorm"))
    ctx.attention_backward("Mq", "Mk", "Mv", out, lse, "Mdo", *grads)
    still((out, lse))
    ctx.attention("Mq", "Mk", "Mv", out, lse)
    ctx.clip_gradients(list(grads), 0.5, norm="Mnorm")
    for n in (*marked, lse, "Mnorm"):
        assert not (ctx.tensor(n) == 1).all()
        with pytest.raises(abi.TLError):
            ctx.bits(n)


def test_replayed_graphs_report_to_sync():
    # tl_sync reads the device's error word after work that may write it: a captured call's replays too
    from tensor_logic_lang_b200.runtime import Context
    c = Context(device=0)

    def read_by_sync():
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
            c.sync()
            torch.cuda.synchronize()
        return any("DtoH" in e.name for e in prof.events())
    try:
        gen = torch.Generator(device="cuda").manual_seed(4)
        q, k, v = (heads(gen, 1, 2, 200, 64, "bf16") for _ in range(3))
        out = like(q, "bhsd")
        c.sync()
        read_by_sync()
        c.attention(q, k, v, out, stream=stream())
        torch.cuda.synchronize()
        if not read_by_sync():
            pytest.skip("the profiler sees no copies here")
        assert not read_by_sync()               # nothing since
        ws = torch.empty(256 + c.attention_workspace(q, k, v, out), dtype=torch.uint8, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.attention(q, k, v, out, stream=stream(), workspace=ws)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert read_by_sync()
    finally:
        c.close()


def test_second_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    from tensor_logic_lang_b200.runtime import Context
    c = Context(device=1)
    try:
        torch.cuda.set_device(0)
        gen = torch.Generator(device="cuda").manual_seed(1)
        q, k, v = (heads(gen, 1, 2, 70, 64, "bf16").to("cuda:1") for _ in range(3))
        out = torch.empty_like(q)
        torch.cuda.synchronize(1)
        c.attention(q, k, v, out, causal=True)
        c.sync()
        assert torch.cuda.current_device() == 0
        check(out, reference(q, k, v, causal=True)["out"], "out")
    finally:
        c.close()
