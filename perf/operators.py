"""The attention and gradient-clipping operators as they are measured: cases, inputs, plain forms, exact values.

Every case is one pass through an operator.  With `own` false `run` computes it from elementary torch
operations in 32 bits (sums of squares in 64); with `own` true it makes the calls of
tensor_logic_lang_b200.runtime.Context.  Kinds of cases:

  prompt   attention of many queries over keys and values; the scores are capped by a tanh, get a bias that
           falls with distance, or are masked (causal, causal with a visible prefix, causal within documents)
  train    the same forward pass and its backward pass
  decode   one or a few new tokens of every sequence over a cache with lengths of its own
  clip     the global norm over a list of gradients, and their scaling to a largest norm

Lengths (of documents, of cached sequences) are a function of the case, dealt in an order that the seed gives,
so a case costs the same under every seed.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_context = []


def _ctx():
    """The program's context, made at the first call."""
    if not _context:
        from tensor_logic_lang_b200.runtime import Context
        _context.append(Context(device=torch.cuda.current_device()))
    return _context[0]


def _attention(name, kind, dtype, b, hq, hkv, nq, nk, d, cap=0.0, slopes=False, mask="causal", docs=0, ragged=False,
               layout="bhsd"):
    return dict(name=name, kind=kind, dtype=dtype, b=b, hq=hq, hkv=hkv, nq=nq, nk=nk, d=d, cap=cap, slopes=slopes,
                mask=mask, docs=docs, ragged=ragged, layout=layout)


def _clip(name, dtype, out, tensors, elements, clipped):
    return dict(name=name, kind="clip", dtype=dtype, out=out, tensors=tensors, elements=elements, clipped=clipped)


def listed():
    return [
        # a long prompt read at once, grouped heads, capped scores: the largest forward pass
        _attention("prompt_cap_causal_bf16", "prompt", "bf16", 1, 32, 8, 4096, 4096, 128, cap=50.0),
        # a pre-training batch's forward pass: documents packed behind one another, distance bias, odd length
        _attention("prompt_docs_bias_f16", "prompt", "f16", 2, 16, 16, 3001, 3001, 64, slopes=True, mask="document",
                   docs=7, layout="bshd"),
        # the framework's own attention block (2048 x 64, fp32 storage) with a visible prefix
        _attention("prompt_prefix_f32", "prompt", "f32", 1, 8, 8, 2048, 2048, 64, mask="prefix"),
        # training, grouped heads, capped scores: the largest backward pass
        _attention("train_cap_causal_bf16", "train", "bf16", 2, 16, 4, 2048, 2048, 128, cap=30.0),
        # training on packed documents with a distance bias, a ragged length and an odd head size
        _attention("train_docs_bias_f16", "train", "f16", 3, 12, 12, 1777, 1777, 80, slopes=True, mask="document",
                   docs=5, layout="bshd"),
        # a small fp32 training step with a prefix that every query sees
        _attention("train_prefix_f32", "train", "f32", 2, 4, 2, 509, 509, 64, cap=20.0, mask="prefix"),
        # one token of one short sequence: latency
        _attention("decode_one_bf16", "decode", "bf16", 1, 32, 8, 1, 517, 128, cap=50.0),
        # a serving batch with long caches of different lengths
        _attention("decode_batch_bf16", "decode", "bf16", 16, 32, 8, 1, 32768, 128, cap=50.0, ragged=True),
        # a few new tokens of each of several sequences, distance bias, every head with keys of its own
        _attention("decode_few_f16", "decode", "f16", 5, 16, 16, 3, 4099, 64, slopes=True, ragged=True,
                   layout="bshd"),
        # the weight gradients of the framework's training benchmark (784 x 4096 and 4096 x 10), clipped
        _clip("clip_mlp_f32", "f32", "f32", 2, 784 * 4096 + 4096 * 10, True),
        # a model's 16-bit gradients, clipped into the fp32 gradients that its optimiser reads
        _clip("clip_model_bf16", "bf16", "f32", 291, 400_000_003, True),
        # gradients under the largest norm stay as they are: the norm alone has to be found
        _clip("clip_under_f32", "f32", "in place", 57, 90_000_001, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("prompt", "train", "decode", "clip"))
    if kind == "clip":
        out = rng.choice(("in place", "f32", "same"))
        dtype = rng.choice(("f32", "f16", "bf16"))
        c = _clip("", dtype, dtype if out == "same" else out, _log(rng, 1, 400), _log(rng, 1000, 200_000_000),
                  out != "in place")
        del c["name"]
        return c
    dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
    hkv = rng.choice((1, 2, 3, 4, 8))
    hq = hkv * rng.choice((1, 2, 3, 4, 8))
    d = rng.choice((32, 40, 64, 64, 80, 96, 128, 128))
    cap = rng.choice((0.0, 20.0, 30.0, 50.0))
    slopes = rng.random() < 0.4
    layout = rng.choice(("bhsd", "bshd"))
    if kind == "decode":
        b = _log(rng, 1, 24)
        nk = _log(rng, 16, 32768)
        while b * hkv * nk * d > 16 * 8 * 32768 * 128 // 2:
            nk = max(16, nk // 2 + 1)
        c = _attention("", kind, dtype, b, hq, hkv, rng.choice((1, 1, 1, 2, 4, 7)), nk, d, cap, slopes,
                       rng.choice(("causal", "causal", "document")), rng.randrange(2, 6), b > 1, layout)
    else:
        b = rng.randrange(1, 5)
        nk = _log(rng, 100, 4000)
        budget = (2e8 if dtype == "f32" else 4e8) / (3.5 if kind == "train" else 1.0)
        while b * hq * nk * nk > budget:
            nk = max(64, nk * 3 // 4 + 1)
        nq = nk if kind == "train" or rng.random() < 0.6 else max(9, nk // rng.randrange(2, 9))
        mask = rng.choice(("causal", "prefix", "document", "full") if nq == nk else ("causal", "prefix", "full"))
        c = _attention("", kind, dtype, b, hq, hkv, nq, nk, d, cap, slopes, mask, rng.randrange(2, 9),
                       b > 1 and mask != "document" and rng.random() < 0.4, layout)
    del c["name"]
    return c


# --------------------------------------------------------------------------- lengths of a case
def _documents(case):
    """Lengths of the documents of one sequence; what is left of it is padding."""
    weights = [1 + (5 * i) % 7 for i in range(max(1, case["docs"]))]
    used = case["nk"] - case["nk"] // 50
    return [max(1, used * w // sum(weights)) for w in weights]


def _lengths(case):
    """Keys of each sequence: all, or from an eighth of them up."""
    b, nk = case["b"], case["nk"]
    if not case["ragged"]:
        return [nk] * b
    return [max(1, nk // 8 + (nk - nk // 8) * i // max(1, b - 1)) for i in range(b)]


def _prefix(case):
    return [case["nk"] // 3 + 5 * i for i in range(case["b"])]


def _sizes(case):
    """Elements of each gradient: a few large matrices, many small vectors, odd sizes."""
    n, total = case["tensors"], case["elements"]
    if n == 2 and total == 784 * 4096 + 4096 * 10:
        return [784 * 4096, 4096 * 10]
    weights = [(1, 4000, 90, 11000, 3, 4000)[i % 6] for i in range(n)]
    sizes = [max(1, total * w // sum(weights)) for w in weights]
    sizes[sizes.index(max(sizes))] += max(0, total - sum(sizes))
    return sizes


def _pairs(case):
    """Visible (query, key) pairs of one head, over the batch."""
    nq, mask, total = case["nq"], case["mask"], 0
    if mask == "document":
        if case["kind"] == "decode":   # the last document alone, whose order the seed gives: its mean
            docs = _documents(case)
            return case["b"] * nq * sum(docs) // len(docs)
        return case["b"] * sum(n * (n + 1) // 2 for n in _documents(case))
    for b, n in enumerate(_lengths(case)):
        start = n - nq if case["kind"] == "decode" else case["nk"] - nq
        seen = torch.arange(start + 1, start + nq + 1, dtype=torch.int64).clamp(0, n)
        if mask == "full":
            seen = torch.full_like(seen, n)
        if mask == "prefix":
            seen = seen.clamp(min=min(_prefix(case)[b], n))
        total += int(seen.sum())
    return total


def work(case):
    if case["kind"] == "clip":
        n, size = sum(_sizes(case)), SIZE[case["dtype"]]
        wrote = 0 if case["out"] == "in place" else SIZE[case["out"]]
        return {"bytes": n * (size + wrote) + 4, "flops": 3 * n}
    b, hq, hkv, nq, d = (case[k] for k in ("b", "hq", "hkv", "nq", "d"))
    size = SIZE[case["dtype"]]
    pairs = _pairs(case)
    keys = sum(_documents(case)) * b // max(1, case["docs"]) if case["mask"] == "document" and case["kind"] == "decode" \
        else sum(_lengths(case))
    q, kv = b * hq * nq * d * size, keys * hkv * d * size
    if case["kind"] == "train":
        # q, k, v, dout read; out, dq, dk, dv written; 2 products forward, 5 backward
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * d * hq * pairs}
    return {"bytes": 2 * q + 2 * kv, "flops": 4 * d * hq * pairs}


# --------------------------------------------------------------------------- inputs
def _normal(gen, shape, dtype, gain=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * gain).to(TYPES[dtype])


def _heads(gen, case, h, n, gain=1.0):
    """[b, h, n, d], as the projections leave it: heads or positions outermost."""
    if case["layout"] == "bshd":
        return _normal(gen, (case["b"], n, h, case["d"]), case["dtype"], gain).transpose(1, 2)
    return _normal(gen, (case["b"], h, n, case["d"]), case["dtype"], gain)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = random.Random(seed)
    if case["kind"] == "clip":
        sizes = _sizes(case)
        flat = _normal(gen, (sum(sizes),), case["dtype"], 1e-3)
        s = {"case": case, "flat": flat, "grads": list(flat.split(sizes))}
        s["norm"] = torch.zeros((), device="cuda")
        true = 1e-3 * math.sqrt(sum(sizes))
        s["max_norm"] = min(1.0, 0.25 * true) if case["clipped"] else 4.0 * true
        if case["out"] != "in place":
            s["out"] = torch.zeros(flat.shape, dtype=TYPES[case["out"]], device="cuda")
            s["outs"] = list(s["out"].split(sizes))
        return s
    b, hq, hkv, nq, nk = (case[k] for k in ("b", "hq", "hkv", "nq", "nk"))
    s = {"case": case, "scale": case["d"] ** -0.5, "cap": case["cap"], "causal": case["mask"] != "full"}
    s["q"] = _heads(gen, case, hq, nq, 2.0)
    s["k"] = _heads(gen, case, hkv, nk)
    s["v"] = _heads(gen, case, hkv, nk)
    s["out"] = torch.zeros_like(s["q"])
    if case["kind"] == "train":
        s["dout"] = _heads(gen, case, hq, nq)
        s["dq"], s["dk"], s["dv"] = (torch.zeros_like(s[n]) for n in ("q", "k", "v"))
        s["lse"] = torch.zeros((b, hq, nq), device="cuda")

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device="cuda") if case["slopes"] \
        else None
    s["kv_len"] = s["q_start"] = s["prefix_len"] = s["q_doc"] = s["k_doc"] = None
    if case["ragged"]:
        n = _lengths(case)
        order.shuffle(n)
        s["kv_len"] = ints(n)
        if case["kind"] != "decode":   # right-padded rows: positions count from the left
            s["q_start"] = ints([nk - nq] * b)
    if case["mask"] == "prefix":
        s["prefix_len"] = ints(_prefix(case))
    if case["mask"] == "document":
        rows = []
        for _ in range(b):
            docs = _documents(case)
            order.shuffle(docs)
            ids = [i for i, n in enumerate(docs) for _ in range(n)][:nk]
            # a training row ends in padding, a cache in the document that is being written
            end = -1 if case["kind"] != "decode" else len(docs) - 1
            rows.append(ids + [end] * (nk - len(ids)))
        s["k_doc"] = ints(rows)
        if case["kind"] != "decode":
            s["q_doc"] = s["k_doc"]
        else:
            n = s["kv_len"] if s["kv_len"] is not None else ints([nk] * b)
            at = (n[:, None] - nq + torch.arange(nq, device="cuda")).clamp(min=0)
            s["q_doc"] = torch.gather(s["k_doc"], 1, at).contiguous()
    return s


# --------------------------------------------------------------------------- the operators
MODIFIERS = ("slopes", "prefix_len", "q_doc", "k_doc", "kv_len", "q_start")


def run(s):
    if s["case"]["kind"] == "clip":
        return _clip_own(s) if own else _clip_plain(s)
    return _attention_own(s) if own else _attention_plain(s)


def _attention_own(s):
    stream = torch.cuda.current_stream().cuda_stream
    more = {n: s[n] for n in MODIFIERS}
    _ctx().attention(s["q"], s["k"], s["v"], s["out"], lse=s.get("lse"), scale=s["scale"], softcap=s["cap"],
                     causal=s["causal"], stream=stream, **more)
    if s["case"]["kind"] != "train":
        return s["out"]
    _ctx().attention_backward(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["dq"], s["dk"], s["dv"],
                              scale=s["scale"], softcap=s["cap"], causal=s["causal"], stream=stream, **more)
    return {"out": s["out"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}


def _clip_own(s):
    stream = torch.cuda.current_stream().cuda_stream
    if "outs" not in s:
        _ctx().clip_gradients(s["grads"], s["max_norm"], norm=s["norm"], stream=stream)
        return {"norm": s["norm"], "grads": s["flat"]}
    _ctx().clip_gradients(s["grads"], s["max_norm"], out=s["outs"], norm=s["norm"], stream=stream)
    return {"norm": s["norm"], "grads": s["out"]}


def _attention_plain(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, hq, nq, d = q.shape
    hkv, nk = k.shape[1], k.shape[2]
    q = q.reshape(b, hkv, hq // hkv * nq, d)          # the queries of a group of heads share its keys
    scores = (q @ k.transpose(-1, -2)).view(b, hkv, hq // hkv, nq, nk) * s["scale"]
    bent = None
    if s["cap"]:
        bent = torch.tanh(scores / s["cap"])
        scores = s["cap"] * bent
    n = s["kv_len"].long() if s["kv_len"] is not None else torch.full((b,), nk, device=q.device)
    start = s["q_start"].long() if s["q_start"] is not None else n - nq
    at = (start[:, None] + torch.arange(nq, device=q.device))[:, :, None]
    key = torch.arange(nk, device=q.device)[None, None, :]
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(1, hkv, -1, 1, 1) * (at - key).abs().float()[:, None, None]
    seen = key < n[:, None, None]
    if s["causal"]:
        past = key <= at
        if s["prefix_len"] is not None:
            past = past | (key < s["prefix_len"][:, None, None])
        seen = seen & past
    if s["q_doc"] is not None:
        seen = seen & (s["q_doc"][:, :, None] == s["k_doc"][:, None, :]) & (s["q_doc"][:, :, None] >= 0)
    seen = seen.expand(b, nq, nk)[:, None, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    del scores
    p = p / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    p = p.view(b, hkv, -1, nk)
    o = p @ v
    out = o.view(b, hq, nq, d).to(s["q"].dtype)
    if s["case"]["kind"] != "train":
        return out
    do = s["dout"].float().reshape(b, hkv, -1, d)
    dv = p.transpose(-1, -2) @ do
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * s["scale"]
    if bent is not None:
        ds = ds * (1 - bent.square().view(b, hkv, -1, nk))
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    return {"out": out, "dq": dq.view(b, hq, nq, d).to(out.dtype), "dk": dk.to(out.dtype), "dv": dv.to(out.dtype)}


def _clip_plain(s):
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
    by = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).float()
    scaled = s["flat"].float() * by
    return {"norm": norm.float(), "grads": scaled.to(s.get("out", s["flat"]).dtype)}


# --------------------------------------------------------------------------- exact values
def exact(case, seed):
    """The definitions in 64 bits, a head at a time."""
    s = prepare(case, seed)
    if case["kind"] == "clip":
        x = s["flat"].double()
        norm = torch.linalg.vector_norm(x)
        by = min(1.0, s["max_norm"] / norm.item()) if norm.item() > 0 else 1.0
        return {"norm": norm, "grads": x.mul_(by)}
    b, hq, nq, d = s["q"].shape
    hkv, nk = s["k"].shape[1:3]
    out = torch.zeros((b, hq, nq, d), dtype=torch.float64, device="cuda")
    grads = [torch.zeros((b, h, n, d), dtype=torch.float64, device="cuda")
             for h, n in ((hq, nq), (hkv, nk), (hkv, nk))] if case["kind"] == "train" else None
    j = torch.arange(nk, device="cuda").double()
    for bi in range(b):
        n = int(s["kv_len"][bi]) if s["kv_len"] is not None else nk
        i = torch.arange(nq, device="cuda").double() + (int(s["q_start"][bi]) if s["q_start"] is not None else n - nq)
        far = i[:, None] - j[None, :]
        hidden = (j >= n)[None, :].expand(nq, nk).clone()
        if s["causal"]:
            ahead = far < 0
            if s["prefix_len"] is not None:
                ahead &= (j >= int(s["prefix_len"][bi]))[None, :]
            hidden |= ahead
        if s["q_doc"] is not None:
            hidden |= (s["q_doc"][bi][:, None] != s["k_doc"][bi][None, :]) | (s["q_doc"][bi] < 0)[:, None]
        none = hidden.all(1)
        for h in range(hq):
            g = h // (hq // hkv)
            q, k, v = (t.double() for t in (s["q"][bi, h], s["k"][bi, g], s["v"][bi, g]))
            x = torch.mm(q, k.t()).mul_(s["scale"])
            slope = torch.ones_like(x)
            if s["cap"]:
                x = torch.tanh(x / s["cap"])
                slope = 1 - x * x
                x = x * s["cap"]
            if s["slopes"] is not None:
                x -= s["slopes"][h].double() * far.abs()
            x[hidden] = -math.inf
            x[none] = 0.0
            p = torch.softmax(x, 1)
            p[none] = 0.0
            o = torch.mm(p, v)
            out[bi, h] = o
            if grads:
                do = s["dout"][bi, h].double()
                dp = torch.mm(do, v.t())
                dx = p * (dp - (p * dp).sum(1, keepdim=True)) * slope * s["scale"]
                grads[0][bi, h] = torch.mm(dx, k)
                grads[1][bi, g] += torch.mm(dx.t(), q)
                grads[2][bi, g] += torch.mm(p.t(), do)
    if not grads:
        return out
    return {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}
