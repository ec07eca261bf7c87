"""The global gradient norm and clipping against 64-bit sums."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    from tensor_logic_lang_b200.runtime import Context
    c = Context(device=0)
    yield c
    c.close()


def stream():
    return torch.cuda.current_stream().cuda_stream


def expected(xs, max_norm):
    norm = math.sqrt(sum((x.double() ** 2).sum().item() for x in xs))
    by = max_norm / norm if norm > max_norm else 1.0
    return norm, [x.double() * by for x in xs]


def check(got, want, by_half=True):
    # the factor and the product are rounded to fp32 (2^-24 each), the result to its type
    for g, w in zip(got, want):
        t = g.dtype
        tol = 2.0 ** -22 * w.abs() + (0 if t == torch.float32 else torch.finfo(t).eps / 2 * w.abs()) + \
            torch.finfo(t).smallest_normal * torch.finfo(t).eps
        assert ((g.double() - w).abs() <= tol).all()


SIZES = [[1], [3, 5, 7], [32768], [32769, 1, 32767], [100003, 17, 4096 * 10], [8] * 40, [1000, 0, 2] * 12]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["in place", "f32", "f16", "bf16"])
def test_sizes(ctx, dtype, out):
    gen = torch.Generator(device="cuda").manual_seed(1)
    for sizes in SIZES:
        for off in (0, 1, 3):                       # views into one buffer, at any element
            flat = torch.randn(sum(sizes) + off, generator=gen, device="cuda").to(TYPES[dtype])
            xs = [x for x in flat[off:].split(sizes)]
            scale = math.sqrt(sum(sizes))
            for max_norm in (0.3 * scale, 3 * scale, 0.0):
                ys = [x.clone() for x in xs]
                views = xs if out != "in place" else [y for y in flat.clone()[off:].split(sizes)]
                room = None if out == "in place" else \
                    [r for r in torch.full((sum(sizes) + 5,), 9.0, dtype=TYPES[out], device="cuda")[2:-3].split(sizes)]
                norm = torch.zeros((), device="cuda")
                got = ctx.clip_gradients(views, max_norm, out=room, norm=norm, stream=stream())
                torch.cuda.synchronize()
                want_norm, want = expected(ys, max_norm)
                assert abs(norm.item() - want_norm) <= 2.0 ** -22 * want_norm
                check(got, want)
                if room is not None:
                    base = room[0]._base
                    assert (base[:2] == 9.0).all() and (base[-3:] == 9.0).all()


def test_mixed_types_and_layouts(ctx):
    gen = torch.Generator(device="cuda").manual_seed(2)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    xs = [randn(64, 33).t(), randn(3, 4, 5, 6).permute(0, 2, 3, 1).bfloat16(), randn(2, 2, 2, 2, 2).half(), randn(),
          randn(7).half()]
    keep = [x.clone() for x in xs]
    norm = torch.zeros((), device="cuda")
    ctx.clip_gradients(xs, 1.0, norm=norm, stream=stream())
    torch.cuda.synchronize()
    want_norm, want = expected(keep, 1.0)
    assert abs(norm.item() - want_norm) <= 2.0 ** -22 * want_norm
    check(xs, want)


@pytest.mark.parametrize("count", [16, 17, 1000, 1001, 2500])
def test_many_arrays(ctx, count):
    gen = torch.Generator(device="cuda").manual_seed(count)
    sizes = [1 + (37 * i) % 90 for i in range(count)]
    flat = torch.randn(sum(sizes), generator=gen, device="cuda")
    keep = flat.clone()
    norm = torch.zeros((), device="cuda")
    ctx.clip_gradients(list(flat.split(sizes)), 2.0, norm=norm, stream=stream())
    torch.cuda.synchronize()
    want_norm, want = expected([keep], 2.0)
    assert abs(norm.item() - want_norm) <= 2.0 ** -22 * want_norm
    check([flat], want)


def test_range_of_fp32(ctx):
    # squares that pass fp32 on either side
    for s in (1e30, 1e-30):
        x = torch.randn(5000, device="cuda") * s
        keep = x.clone()
        norm = torch.zeros((), device="cuda")
        ctx.clip_gradients([x], s, norm=norm, stream=stream())
        torch.cuda.synchronize()
        want_norm, want = expected([keep], s)
        assert abs(norm.item() - want_norm) <= 2.0 ** -22 * want_norm
        check([x], want)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_norm_not_finite(ctx, bad):
    x, y = torch.ones(5000, device="cuda"), torch.ones(100, device="cuda", dtype=torch.bfloat16)
    x[4321] = bad
    norm = torch.zeros((), device="cuda")
    ctx.clip_gradients([x, y], 0.5, norm=norm, stream=stream())
    torch.cuda.synchronize()
    assert norm.item() == bad or (math.isnan(bad) and math.isnan(norm.item()))
    assert (y == 1).all() and (x[:4321] == 1).all() and (x[4322:] == 1).all()


def test_norm_alone_and_nothing(ctx):
    x = torch.ones(10000, device="cuda")
    norm = torch.zeros((), device="cuda")
    ctx.clip_gradients([x], math.inf, norm=norm, stream=stream())
    torch.cuda.synchronize()
    assert norm.item() == 100.0 and (x == 1).all()
    ctx.clip_gradients([], 1.0, norm=norm, stream=stream())
    torch.cuda.synchronize()
    assert norm.item() == 0.0
    z = torch.zeros(100, device="cuda")
    ctx.clip_gradients([z], 0.0, norm=norm, stream=stream())
    torch.cuda.synchronize()
    assert norm.item() == 0.0 and not z.any()


def test_repeats_bit_for_bit(ctx):
    xs = [torch.randn(n, device="cuda") for n in (1_000_003, 77, 250_000)]
    seen = []
    for _ in range(3):
        ys = [x.clone() for x in xs]
        norm = torch.zeros((), device="cuda")
        ctx.clip_gradients(ys, 1.0, norm=norm, stream=stream())
        torch.cuda.synchronize()
        seen.append([norm] + ys)
    for s in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(s, seen[0]))


def test_captured_and_replayed(ctx):
    xs = [torch.randn(n, device="cuda") for n in (100_003, 77)]
    ys = [torch.empty_like(x) for x in xs]
    norm = torch.zeros((), device="cuda")
    ws = torch.empty(ctx.clip_workspace(xs, 1.0, ys), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.clip_gradients(xs, 1.0, out=ys, norm=norm, workspace=ws, stream=stream())
    for i in range(3):
        for x in xs:
            x.normal_().mul_(i + 1)
        graph.replay()
        torch.cuda.synchronize()
        want_norm, want = expected(xs, 1.0)
        assert abs(norm.item() - want_norm) <= 2.0 ** -22 * want_norm
        check(ys, want)


def test_refusals_do_nothing(ctx):
    from tensor_logic_lang_b200 import abi
    x = torch.ones(100, device="cuda")
    for bad in ([x, x], [x[:60], x[50:]], [x[::2]], [x.cpu()], [x.double()]):
        with pytest.raises(abi.TLError):
            ctx.clip_gradients(bad, 0.5, stream=stream())
    with pytest.raises(abi.TLError):
        ctx.clip_gradients([x], -1.0, stream=stream())
    with pytest.raises(abi.TLError):
        ctx.clip_gradients([x], 1.0, out=[torch.ones(99, device="cuda")], stream=stream())
    with pytest.raises(abi.TLError):
        ctx.clip_gradients([x], 1.0, out=[], stream=stream())
    with pytest.raises(abi.TLError):
        ctx.clip_gradients([x], 1.0, norm=torch.zeros((), device="cuda", dtype=torch.float64), stream=stream())
    torch.cuda.synchronize()
    assert (x == 1).all()


def test_gradients_of_a_program(ctx):
    # what `backward` leaves, clipped in the program's own storage
    import numpy as np
    from tensor_logic_lang_b200 import configs
    p, *_ = configs.program(configs.mlp_train, b=64, i=40, h=96, o=10)
    ctx.run(p)
    before = [ctx.tensor(n) for n in ("dL_dW1", "dL_dW2")]
    norm = math.sqrt(sum((g ** 2).sum() for g in before))
    ctx.clip_gradients(["dL_dW1", "dL_dW2"], norm / 3)
    for n, g in zip(("dL_dW1", "dL_dW2"), before):
        np.testing.assert_allclose(ctx.tensor(n), g / 3, rtol=2.0 ** -22, atol=1e-40)
