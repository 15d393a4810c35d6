"""The answering end of a scoring step, as cases with sizes, inputs, work, plain forms and 64-bit answers.

Four operators: log probabilities of given tokens with entropy and top alternatives (`ops.logprobs`), the same from hidden
states without the logits matrix (`ops.lm_head_logprobs`), products with 4-bit weights under group scales
(`ops.gemm_w4`), and the quantisation that makes those weights (`ops.quantize_w4`, `ops.dequantize_w4`).

`listed()` holds fixed cases, `draw(rng)` more of the same ranges; `prepare` makes what a program has in hand before the
call and `run` is one pass: the plain form in torch operations, or with `own` the framework's operators.  Vocabulary and
widths are the presets' (1b, 2b, tiny) or generic.
"""
from __future__ import annotations

import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [p for p in (ROOT, os.path.join(ROOT, "minicpm5-vllm-tpu_amd")) if p not in sys.path]

own = False

DEV = "cuda:0"
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
DTYPES = {"f32": F32, "bf16": BF16, "f16": F16}
VOCAB = 130560        # the presets' vocabulary
W_STD = 0.02          # weights N(0, 0.02)
SMALLEST = 2.0 ** -126


def listed():
    return [
        # one reply of a chat: the last token's logits, its token's log probability and the 20 best alternatives
        {"name": "logprobs_1x130560", "kind": "logprobs", "rows": 1, "vocab": VOCAB, "dtype": "f32", "ids": 1, "top": 20,
         "masked": False},
        # the smallest call: two short prompts of the tiny config, four answer letters each, no alternatives
        {"name": "logprobs_2x32768", "kind": "logprobs", "rows": 2, "vocab": 32768, "dtype": "f32", "ids": 4, "top": 0,
         "masked": False},
        # a scoring batch with part of the vocabulary disallowed, an odd vocabulary, four candidates a row
        {"name": "logprobs_33x130559_masked", "kind": "logprobs", "rows": 33, "vocab": VOCAB - 1, "dtype": "f32", "ids": 4,
         "top": 20, "masked": True},
        # the tokens of a long prompt from half-precision logits
        {"name": "logprobs_2048x130560_bf16", "kind": "logprobs", "rows": 2048, "vocab": VOCAB, "dtype": "bf16", "ids": 1,
         "top": 5, "masked": False},
        # every token of a full-context prompt scored from its hidden states (1b head)
        {"name": "head_logprobs_1b_8192", "kind": "head_logprobs", "rows": 8192, "hidden": 1536, "vocab": VOCAB, "ids": 1},
        # a mid-length prompt with an odd number of tokens (2b head)
        {"name": "head_logprobs_2b_645", "kind": "head_logprobs", "rows": 645, "hidden": 2048, "vocab": VOCAB, "ids": 1},
        # four candidates of a few prompts' last tokens (1b head)
        {"name": "head_logprobs_1b_17", "kind": "head_logprobs", "rows": 17, "hidden": 1536, "vocab": VOCAB, "ids": 4},
        # the 1b head in 4 bits for one token
        {"name": "gemm_w4_1b_head_1", "kind": "gemm_w4", "rows": 1, "n": VOCAB, "k": 1536, "group": 128, "out": "f32"},
        # the 2b head in 4 bits for a batch of 40 last tokens, finer groups
        {"name": "gemm_w4_2b_head_40", "kind": "gemm_w4", "rows": 40, "n": VOCAB, "k": 2048, "group": 64, "out": "f32"},
        # a down projection for one token: few rows of weights, latency counts
        {"name": "gemm_w4_1b_down_1", "kind": "gemm_w4", "rows": 1, "n": 1536, "k": 4608, "group": 32, "out": "bf16"},
        # the 1b head into 4 bits
        {"name": "quantize_w4_1b_head", "kind": "quantize_w4", "n": VOCAB, "k": 1536, "group": 128},
        # a 2b down projection into 4 bits
        {"name": "quantize_w4_2b_down", "kind": "quantize_w4", "n": 2048, "k": 6144, "group": 64},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs", "head_logprobs", "gemm_w4", "gemm_w4", "quantize_w4"])
    if kind == "logprobs":
        vocab = _spread(rng, 1000, 160000)
        dtype = rng.choice(["f32", "bf16", "f16"])
        rows = _spread(rng, 1, min(4096, (1 if dtype == "f32" else 2) * 1024 * VOCAB // vocab))
        return {"kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype, "ids": rng.choice([1, 1, 2, 4, 7]),
                "top": rng.choice([0, 1, 5, 20, 32]), "masked": rng.random() < 0.3}
    if kind == "head_logprobs":
        return {"kind": kind, "rows": _spread(rng, 1, 6000), "hidden": 32 * _spread(rng, 8, 64),
                "vocab": _spread(rng, 8000, VOCAB), "ids": rng.choice([1, 1, 2, 5])}
    if kind == "gemm_w4":
        n, k = rng.choice([(_spread(rng, 256, VOCAB), _spread(rng, 96, 2048)), (_spread(rng, 256, 12288), _spread(rng, 96, 8192))])
        return {"kind": kind, "rows": _spread(rng, 1, 64), "n": n, "k": k, "group": rng.choice([32, 64, 128]),
                "out": rng.choice(["f32", "bf16"])}
    return {"kind": kind, "n": _spread(rng, 256, 65536), "k": _spread(rng, 96, 2048), "group": rng.choice([32, 64, 128])}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _logits(g, rows, vocab, dtype, masked):
    """Logits of a language model: a bell around a row's own level, a few tokens far above it; masked: a token in three
    disallowed."""
    x = torch.randn((rows, vocab), generator=g, device=DEV).mul_(2.5)
    x += 3.0 * torch.randn((rows, 1), generator=g, device=DEV) - 4.0
    likely = torch.randint(0, vocab, (rows, 32), generator=g, device=DEV)
    x.scatter_(1, likely, 6.0 + 3.0 * torch.randn((rows, 32), generator=g, device=DEV))
    if masked:
        x.masked_fill_(torch.rand((rows, vocab), generator=g, device=DEV) < 1 / 3, float("-inf"))
    return x.to(dtype)


def _given(g, x, n):
    """Given tokens: the likely ones half of the time, never a disallowed one."""
    w = torch.softmax(0.3 * x.float(), -1)
    if w.shape[0] * w.shape[1] < 1 << 24:
        return torch.multinomial(w, n, replacement=True, generator=g)
    return torch.cat([torch.multinomial(p, n, replacement=True, generator=g) for p in w.split(256)])


def _hidden(g, rows, width):
    """Final-normed hidden rows: unit-sized channels, some larger than others."""
    x = torch.randn((rows, width), generator=g, device=DEV)
    return (x * torch.exp(0.4 * torch.randn((1, width), generator=g, device=DEV))).to(BF16)


def _weight(g, n, k):
    """A linear's weights: N(0, 0.02), rows of different sizes, a few outliers."""
    w = torch.randn((n, k), generator=g, device=DEV).mul_(W_STD)
    w *= torch.exp(0.2 * torch.randn((n, 1), generator=g, device=DEV))
    w[:, :: 97] *= 2.5
    return w.to(BF16)


def _groups(w, group):
    """(n, k) -> (n, groups, group), the last group filled up with zeros."""
    n, k = w.shape
    ng = -(-k // group)
    return torch.nn.functional.pad(w, (0, ng * group - k)).view(n, ng, group)


def _quantize(w, group):
    """The 4-bit format in torch: codes (n, groups, group) f32 in [-7, 7], scales (n, groups, 1) f32 of bf16 values."""
    g = _groups(w.float(), group)
    s = (g.abs().amax(-1, keepdim=True) / 7.0)
    s = torch.where(s < SMALLEST, torch.zeros_like(s), s).to(BF16).float()
    c = torch.where(s > 0, torch.round(g / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(g))
    return c.clamp_(-7, 7), s


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "logprobs":
        st["logits"] = _logits(g, case["rows"], case["vocab"], DTYPES[case["dtype"]], case["masked"])
        st["ids"] = _given(g, st["logits"], case["ids"])
        return st
    if kind == "head_logprobs":
        st["hidden"] = _hidden(g, case["rows"], case["hidden"])
        st["weight"] = _weight(g, case["vocab"], case["hidden"])
        st["ids"] = torch.randint(0, case["vocab"], (case["rows"], case["ids"]), generator=g, device=DEV)
        return st
    w = _weight(g, case["n"], case["k"])
    if kind == "quantize_w4":
        st["weight"] = w
        return st
    st["x"] = _hidden(g, case["rows"], case["k"])
    if own:
        from minicpm5_mk import ops
        st["w4"] = ops.quantize_w4(w, case["group"])
    else:
        c, s = _quantize(w, case["group"])
        st["codes"], st["scales"] = c.to(torch.int8), s
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    from minicpm5_mk import ops
    case = st["case"]
    kind = case["kind"]
    if kind == "logprobs":
        r = ops.logprobs(st["logits"], st["ids"], top=case["top"])
        out = [r.token_logprobs, r.ranks, r.entropy, r.logsumexp]
        return out + [r.top_logprobs, r.top_ids] if case["top"] else out
    if kind == "head_logprobs":
        r = ops.lm_head_logprobs(st["hidden"], st["weight"], st["ids"])
        return [r.token_logprobs, r.entropy, r.logsumexp]
    if kind == "gemm_w4":
        return [ops.gemm_w4(st["x"], st["w4"], dtype=DTYPES[case["out"]])]
    return [ops.dequantize_w4(ops.quantize_w4(st["weight"], case["group"]))]


def _softmax_stats(x):
    """Row maximum, log of the sum of exponentials above it, and entropy of x (rows, vocab) in x's type."""
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    u = (e * torch.where(e > 0, d, torch.zeros_like(d))).sum(-1, keepdim=True)
    ls = torch.log(s)
    return m, ls, (ls - u / s).squeeze(-1)


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "logprobs":
        parts = [_plain_logprobs(x.float(), i, case["top"]) for x, i in zip(st["logits"].split(512), st["ids"].split(512))]
        return [torch.cat(p) for p in zip(*parts)]
    if kind == "head_logprobs":
        w = st["weight"].float()
        parts = []
        for h, i in zip(st["hidden"].split(1024), st["ids"].split(1024)):
            x = h.float() @ w.T
            m, ls, ent = _softmax_stats(x)
            parts.append([(x.gather(1, i) - m) - ls, ent, (m + ls).squeeze(-1)])
        return [torch.cat(p) for p in zip(*parts)]
    if kind == "gemm_w4":
        c = st["codes"]
        w = (c.float() * st["scales"]).reshape(c.shape[0], -1)[:, : case["k"]]
        return [(st["x"].float() @ w.T).to(DTYPES[case["out"]])]
    n, k = st["weight"].shape
    c, s = _quantize(st["weight"], case["group"])
    return [(c * s).reshape(n, -1)[:, :k].to(BF16)]


def _plain_logprobs(x, ids, top):
    m, ls, ent = _softmax_stats(x)
    at = torch.arange(x.shape[1], device=x.device)
    v = x.gather(1, ids)
    rank = torch.stack([1 + (x > v[:, j: j + 1]).sum(-1) + ((x == v[:, j: j + 1]) & (at < ids[:, j: j + 1])).sum(-1)
                        for j in range(ids.shape[1])], 1).to(torch.int32)
    out = [(v - m) - ls, rank, ent, (m + ls).squeeze(-1)]
    if top:
        val, idx = torch.sort(x, dim=-1, descending=True, stable=True)
        out += [(val[:, :top] - m) - ls, idx[:, :top].to(torch.int32)]
    return out


# ------------------------------------------------------------------------------------------------ work, answers
def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        t, v, n, k = case["rows"], case["vocab"], case["ids"], case["top"]
        esz = 4 if case["dtype"] == "f32" else 2
        return {"bytes": t * v * esz + t * n * 8 + t * 4 * (2 * n + 2 * k + 2), "flops": 6 * t * v}
    if kind == "head_logprobs":
        t, v, h, n = case["rows"], case["vocab"], case["hidden"], case["ids"]
        return {"bytes": 2 * (t + v) * h + t * n * 8 + t * 4 * (n + 2), "flops": 2 * t * v * h + 6 * t * v}
    n, k = case["n"], case["k"]
    ng = -(-k // case["group"])
    if kind == "gemm_w4":
        m = case["rows"]
        return {"bytes": n * k // 2 + n * ng * 2 + m * k * 2 + m * n * (4 if case["out"] == "f32" else 2),
                "flops": 2 * m * n * k}
    return {"bytes": n * k * 2 + n * k * 2, "flops": 4 * n * k}


def exact(case, seed):
    """What `run` returns for these inputs, from the definitions in 64 bits."""
    g = _gen(seed)
    kind = case["kind"]
    if kind == "logprobs":
        logits = _logits(g, case["rows"], case["vocab"], DTYPES[case["dtype"]], case["masked"])
        ids = _given(g, logits, case["ids"])
        parts = [_exact_rows(x.to(F64), i, case["top"]) for x, i in zip(logits.split(128), ids.split(128))]
        out = [torch.cat(p) for p in zip(*parts)]
        return out[:1] + [None] + out[1:3] + ([out[3], None] if case["top"] else [])
    if kind == "head_logprobs":
        h = _hidden(g, case["rows"], case["hidden"]).to(F64)
        w = _weight(g, case["vocab"], case["hidden"]).to(F64)
        ids = torch.randint(0, case["vocab"], (case["rows"], case["ids"]), generator=g, device=DEV)
        parts = [_exact_rows(torch.mm(a, w.T), i, 0) for a, i in zip(h.split(512), ids.split(512))]
        return [torch.cat(p) for p in zip(*parts)]
    w = _weight(g, case["n"], case["k"]).to(F64)
    rows, step = [], max(1, (1 << 26) // case["k"])
    x = _hidden(g, case["rows"], case["k"]).to(F64) if kind == "gemm_w4" else None
    for part in w.split(step):
        pieces = []
        for one in part.split(case["group"], dim=1):
            s = (one.abs().amax(1, keepdim=True) / 7).to(BF16).to(F64)
            s[s < SMALLEST] = 0
            c = torch.round(one / torch.where(s > 0, s, torch.full_like(s, math.inf))).clamp(-7, 7)
            pieces.append(c * s)
        q = torch.cat(pieces, 1)
        rows.append(q if x is None else torch.mm(x, q.T))
    return [torch.cat(rows, 0 if x is None else 1)]


def _exact_rows(x, ids, top):
    lse = torch.logsumexp(x, -1, keepdim=True)
    lp = x - lse
    out = [lp.gather(1, ids), -torch.special.xlogy(lp.exp(), lp.exp()).sum(-1), lse.squeeze(-1)]
    return out + [torch.topk(lp, top, -1).values] if top else out
