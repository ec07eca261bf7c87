"""Attention with modified scores in 64 bits, and how far a kernel's results may be from it.

`reference` evaluates the formulas of include/tl_cuda.h on whole score matrices
and gives each result with a bound for every element:

  out  16-bit operands: the exponentials are rounded before their product with
       v, and the result is rounded, each by at most half a step h = eps / 2
       relative to the value:  h (|out| + sum p |v|)
  dv   h (|dv| + sum p |dout|)
  dq   dx is rounded (h sum |dx| |k|), out was rounded before it went into
       D = dout . out (off by h sum |dout| |out|, which every dx of the row
       takes with its p), and the result is rounded; dk alike with q

and in every type a slack g relative to the sizes of the terms for the 32-bit
arithmetic: scores that are off by s 2^-24 times a few, the exponential and
the tanh (g = 2^-12 beside 16-bit roundings, 2^-16 in fp32).

The tanh of a capped score is held in 32 bits: near 1 it is off by half a step,
2^-24, elsewhere by up to 2^-21 (an exponential and a quotient of 2^-22 each),
so 1 - tanh^2 is off by up to 2^-20 in absolute terms, which counts where it is
small.

An exponential below 2^-126, the smallest normal number of fp32 and bf16, may be
0, and so may a dx: off by that much for every pair that is seen.

fp32 arrays of head size up to 128 go through the tensor cores as pairs of fp16
numbers, hi + lo: a value x below 2^15 keeps 22 bits, or 2^-25 where that is
more (fp16 ends at 2^-24, half a step of it).  In the backward pass p goes in as
2^14 p, so it is off by up to 2^-25 / 2^14 = 2^-39; dx / scale goes in times the
power of two L that puts B = 2 max|dout_i| max|v_j| (norms, over the heads of
a group) between 2^14 and 2^15, L >= 2^14 / B, so it is off by up to
2^-25 / L <= 2^-39 B.  Both are absolute, for every pair that is seen (tiny):
they count where a key's every p is that small.
"""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def reference(q, k, v, dout=None, *, scale=None, softcap=0.0, slopes=None, causal=False, prefix_len=None, q_doc=None,
              k_doc=None, kv_len=None, q_start=None):
    """{name: (value, bound)} of out, lse and, with dout, dq, dk, dv."""
    h = half_step(q.dtype)
    g = 2.0 ** -16 if q.dtype == torch.float32 else 2.0 ** -12
    tiny = torch.finfo(q.dtype).tiny            # results below it lose bits
    b, hq, nq, d = q.shape
    hkv, nk = k.shape[1:3]
    group = hq // hkv if hkv else 1
    scale = d ** -0.5 if scale is None else scale
    dev = q.device
    n = torch.full((b,), nk, device=dev) if kv_len is None else kv_len.long().clamp(0, nk)
    start = n - nq if q_start is None else q_start.long()
    at = (start[:, None] + torch.arange(nq, device=dev))[:, :, None].double()
    key = torch.arange(nk, device=dev)[None, None, :].double()
    seen = (key < n[:, None, None]).expand(b, nq, nk).clone()
    if causal:
        past = key <= at
        if prefix_len is not None:
            past = past | (key < prefix_len[:, None, None])
        seen &= past
    k_ok = key[0] < n[:, None]
    q_ok = torch.ones((b, nq), dtype=torch.bool, device=dev)
    if q_doc is not None:
        seen &= (q_doc[:, :, None] == k_doc[:, None, :]) & (q_doc[:, :, None] >= 0)
        k_ok = k_ok & (k_doc >= 0)
        q_ok = q_doc >= 0

    def clean(x, ok):
        return torch.where(ok[:, None, :, None], x.double(), 0.0)

    Q = clean(q, q_ok)
    K = clean(k, k_ok).repeat_interleave(group, 1)
    V = clean(v, k_ok).repeat_interleave(group, 1)
    seen = seen[:, None]
    x = Q @ K.transpose(-1, -2) * scale
    t = torch.tanh(x / softcap) if softcap else torch.zeros_like(x)
    s = softcap * t if softcap else x
    if slopes is not None:
        s = s - slopes.double()[None, :, None, None] * (at - key)[:, None].abs()
    s = torch.where(seen, s, -math.inf)
    lse = torch.logsumexp(s, -1) if nk else torch.full((b, hq, nq), -math.inf, device=dev, dtype=torch.float64)
    p = torch.where(seen, torch.exp(s - torch.where(lse > -math.inf, lse, 0.0)[..., None]), 0.0)
    # the slack of a row's exponentials grows with the size of its scores
    big = 1 + torch.where(seen, s, 0.0).abs().amax(-1, keepdim=True) / 8 if nk else torch.ones_like(at[:, None])
    out = p @ V
    res = {"out": (out, h * out.abs() + (h + g * big) * (p @ V.abs()) + tiny),
           "lse": (lse, 2.0 ** -16 * (1 + torch.where(lse > -math.inf, lse, 0.0).abs()))}
    if dout is None:
        return res
    DO = clean(dout, q_ok)
    dp = DO @ V.transpose(-1, -2)
    D = (DO * out).sum(-1, keepdim=True)
    bend = (1 - t * t) * scale
    dx = p * (dp - D) * bend
    # every dx: its rounding, the rounding of out within D, the slack of p, dp and D
    off_D = (DO * out).abs().sum(-1, keepdim=True)
    off_dp = DO.abs() @ V.abs().transpose(-1, -2)
    off_bend = 2.0 ** -20 * scale if softcap else 0.0
    off = h * dx.abs() + p * off_bend * (dp - D).abs() + p * bend.abs() * (h * off_D + g * big * ((dp - D).abs() + 2.0 ** -6 * (off_dp + off_D)))

    def grouped(y):
        return y.view(b, hkv, group, nk, d).sum(2)

    off_p = seen * 2.0 ** -126
    off = off + off_p * (1 + (dp - D).abs() * bend.abs())
    if q.dtype == torch.float32:
        def top(y, heads):
            return y.norm(dim=-1).amax(-1).view(b, hkv, heads).amax(-1).repeat_interleave(group, 1)
        both = 2.0 * top(DO, group) * top(V, group) if nq and nk else torch.zeros((b, hq), device=dev)
        off = off + seen * 2.0 ** -39 * both.view(b, hq, 1, 1) * scale
        off_p = off_p + seen * 2.0 ** -39
    dq, dk, dv = dx @ K, grouped(dx.transpose(-1, -2) @ Q), grouped(p.transpose(-1, -2) @ DO)
    res["dq"] = (dq, h * dq.abs() + off @ K.abs() + tiny)
    res["dk"] = (dk, h * dk.abs() + grouped(off.transpose(-1, -2) @ Q.abs()) + tiny)
    res["dv"] = (dv, h * dv.abs() + grouped(((h + g * big) * p + off_p).transpose(-1, -2) @ DO.abs()) + tiny)
    return res


def check(got, want, what):
    value, bound = want
    got = got.double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    same = torch.isinf(value) & (got == value)
    off = torch.where(same, 0.0, (got - value).abs())
    over = ~(off <= bound)                       # a NaN is over
    if over.any():
        at = torch.argmax(torch.where(torch.isnan(off), math.inf, off / bound.clamp(min=1e-300)))
        i = [int(c) for c in torch.unravel_index(at, value.shape)]
        raise AssertionError(f"{what}: {int(over.sum())} of {over.numel()} values off, worst at {i}: "
                             f"{got[tuple(i)].item()} for {value[tuple(i)].item()}, bound {bound[tuple(i)].item():.3g}")
