"""ops.lm_head_logprobs against the definition in float64: stored and fused paths, odd rows and vocabularies, refusals,
streams and graph replay; and the answering end run as one: head, log probabilities, 4-bit head."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")


def _inputs(T, H, V, n, seed=0, std=0.05):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    h = torch.randn((T, H), generator=g, device=DEV).to(BF16)
    w = (std * torch.randn((V, H), generator=g, device=DEV)).to(BF16)
    ids = torch.randint(0, V, (T, n), generator=g, device=DEV)
    return h, w, ids


def _check(h, w, ids, r=None):
    """A logit is H products (exact) added in f32 in some order: off by at most H 2^-24 sum |h w|.  logsumexp is off by at
    most the largest of a row's logit errors, a log probability by two of them, the entropy (mean log probability with
    changed weights) by two and their product with its own size; on top the sums of 2^14 exponentials a lane or tile
    entry, counted 400 half steps."""
    from minicpm5_mk import ops

    r = ops.lm_head_logprobs(h, w, ids) if r is None else r
    assert r.ranks is None and r.top_ids is None and r.top_logprobs is None
    hd, wd = h.double(), w.double()
    x = torch.mm(hd, wd.T.contiguous())
    off = h.shape[1] * 2.0 ** -24 * torch.mm(hd.abs(), wd.abs().T.contiguous()).amax(-1) + 400 * 2.0 ** -24
    lse = torch.logsumexp(x, -1)
    lp = x - lse[:, None]
    ent = -(lp.exp() * lp).sum(-1)
    tol = off * (1 + lse.abs())
    assert ((r.logsumexp.double() - lse).abs() <= tol).all()
    assert ((r.entropy.double() - ent).abs() <= 2 * off * (1 + ent) * 2).all()
    if ids is None:
        assert r.token_logprobs is None
        return r
    i = ids.long().reshape(h.shape[0], -1)
    ok = (i >= 0) & (i < w.shape[0])
    want = torch.where(ok, lp.gather(1, torch.where(ok, i, torch.zeros_like(i))), torch.full_like(lp[:, :1], -INF))
    got = r.token_logprobs.double().reshape(i.shape)
    assert r.token_logprobs.shape == ids.shape
    assert torch.equal(torch.isinf(got), ~ok)
    assert ((got - want).abs()[ok] <= (2 * tol[:, None] * (1 + want.abs()))[ok]).all()
    # the bounds add every rounding's worst; typical errors are those of an f32 product
    assert float((got - want)[ok].norm()) <= 2e-6 * float(want[ok].norm()) + 1e-6
    assert float((r.entropy.double() - ent).norm()) <= 2e-6 * float(ent.norm()) + 1e-6
    return r


@pytest.mark.parametrize("T,H,V,n", [
    (1, 32, 1, 1), (1, 256, 1000, 2), (17, 1536, 8000, 4), (33, 96, 257, 1), (64, 512, 20000, 1), (5, 2048, 33333, 3),
    (65, 32, 256, 1), (65, 64, 255, 2), (66, 96, 1, 1), (100, 1536, 257, 1), (129, 2048, 5000, 64), (255, 224, 1023, 1),
    (256, 1536, 8192, 2), (257, 256, 300, 1), (645, 2048, 3001, 1), (1000, 160, 12345, 5), (2100, 64, 40000, 1),
])
def test_sizes(T, H, V, n):
    h, w, ids = _inputs(T, H, V, n, seed=T)
    _check(h, w, ids)


def test_paths_agree():
    """The rows of a long batch (statistics of tiles) and the same rows alone (stored logits)."""
    from minicpm5_mk import ops

    h, w, ids = _inputs(200, 1536, 9000, 2)
    a, b = ops.lm_head_logprobs(h, w, ids), ops.lm_head_logprobs(h[:40].contiguous(), w, ids[:40].contiguous())
    for x, y in zip((a.token_logprobs, a.entropy, a.logsumexp), (b.token_logprobs, b.entropy, b.logsumexp)):
        assert float((x[:40] - y).abs().max()) <= 1e-5 * (1 + float(y.abs().max()))


def test_ids_outside_and_none():
    h, w, ids = _inputs(70, 128, 500, 3)
    ids[0] = torch.tensor([-1, 500, 2 ** 40], device=DEV)
    ids[69, 1] = -100
    _check(h, w, ids)
    _check(h[:9].contiguous(), w, ids[:9].contiguous())
    _check(h, w, ids[:, 2].contiguous())
    _check(h, w, ids.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32))
    _check(h, w, None)
    _check(h[:9].contiguous(), w, None)
    r = _check(h[:1].contiguous(), w, ids[:1, :0].contiguous())
    assert r.token_logprobs.shape == (1, 0)


@pytest.mark.parametrize("T", [3, 90])
def test_certain_and_not_finite(T):
    """A token of all but certain probability stays at or below 0; a row with an infinity is NaN, the others are not."""
    from minicpm5_mk import ops

    h, w, ids = _inputs(T, 256, 2000, 1)
    h[1] = w[77] * 100
    w[77] *= 20
    h[1] = (w[77].float() * 8).to(BF16)
    ids[1] = 77
    h[2, 5] = INF
    r = ops.lm_head_logprobs(h, w, ids)
    assert torch.isnan(r.token_logprobs[2]).all() and torch.isnan(r.entropy[2]) and torch.isnan(r.logsumexp[2])
    keep = [i for i in range(T) if i != 2]
    assert torch.isfinite(r.token_logprobs[keep]).all() and torch.isfinite(r.entropy[keep]).all()
    assert -1e-4 <= float(r.token_logprobs[1]) <= 0.0 and 0.0 <= float(r.entropy[1]) <= 1e-3
    assert (r.token_logprobs[keep] <= 0).all()


def test_zero_rows_and_equal_logits():
    """Hidden rows of zeros: every token equally likely, ln V."""
    from minicpm5_mk import ops

    for T in (2, 80):
        h, w, ids = _inputs(T, 64, 1000, 2)
        h.zero_()
        r = ops.lm_head_logprobs(h, w, ids)
        ln = torch.log(torch.tensor(1000.0)).item()
        for v in (-r.token_logprobs, r.entropy, r.logsumexp):
            assert float((v - ln).abs().max()) <= 400 * 2.0 ** -24 * (1 + ln)
        assert ops.lm_head_logprobs(h[:0], w, ids[:0]).entropy.shape == (0,)


def test_many_rows():
    """More rows than one pass keeps statistics of."""
    h, w, ids = _inputs(16384 + 77, 32, 300, 1)
    _check(h, w, ids)


@pytest.mark.parametrize("T", [3, 70])
def test_large_weight(T):
    """A head of more than 4 GiB: the vocabulary in slices, given tokens on both sides of the cut."""
    V, H = 270000, 8192
    h, _, _ = _inputs(T, H, 1, 1, seed=3)
    w = torch.empty((V, H), device=DEV, dtype=BF16)
    for part in w.split(30000):
        part.copy_(0.01 * torch.randn(part.shape, device=DEV))
    cut = ((1 << 32) - 1) // (2 * H) // 256 * 256
    ids = torch.tensor([[0, cut - 1, cut, V - 1]] * T, device=DEV)
    x = torch.cat([torch.mm(h.float(), part.float().T.contiguous()) for part in w.split(30000)], 1).double()
    from minicpm5_mk import ops

    r = ops.lm_head_logprobs(h, w, ids)
    lp = torch.log_softmax(x, -1)
    # both sides' logits are f32 sums of 8192 products: relative errors of a few 2^-24 sqrt(8192) in norm
    assert float((r.token_logprobs.double() - lp.gather(1, ids)).norm()) <= 4e-6 * float(lp.gather(1, ids).norm())
    assert float((r.logsumexp.double() - torch.logsumexp(x, -1)).abs().max()) <= 1e-4
    assert float((r.entropy.double() + (lp.exp() * lp).sum(-1)).abs().max()) <= 1e-4


def test_refusals():
    from minicpm5_mk import ops

    h, w, ids = _inputs(4, 64, 100, 1)
    for bad, msg in ((lambda: ops.lm_head_logprobs(h.float(), w, ids), "dtype"),
                     (lambda: ops.lm_head_logprobs(h, w.float(), ids), "dtype"),
                     (lambda: ops.lm_head_logprobs(h[:, :32], w, ids), "contiguous"),
                     (lambda: ops.lm_head_logprobs(h, w[:, :32].contiguous(), ids), "shape"),
                     (lambda: ops.lm_head_logprobs(h[0], w, ids), "expected hidden"),
                     (lambda: ops.lm_head_logprobs(h, w[:0], ids), "empty"),
                     (lambda: ops.lm_head_logprobs(h[:, :48].contiguous(), w[:, :48].contiguous(), ids), "multiple of 32"),
                     (lambda: ops.lm_head_logprobs(h, w, ids[:3].contiguous()), "ids"),
                     (lambda: ops.lm_head_logprobs(h, w, ids.float()), "ids"),
                     (lambda: ops.lm_head_logprobs(h, w, ids.cpu()), "GPU tensor"),
                     (lambda: ops.lm_head_logprobs(h, w, ids.expand(4, 65).contiguous()), "at most 64"),
                     (lambda: ops.logprobs(h, ids, top=101), "top"),
                     (lambda: ops.logprobs(h, ids, top=-1), "top"),
                     (lambda: ops.logprobs(h.double(), ids), "expected 2 dimensions"),
                     (lambda: ops.logprobs(h.T, None), "contiguous"),
                     (lambda: ops.logprobs(h[:, :0], None), "empty")):
        with pytest.raises(ops.MkError, match=msg):
            bad()


@pytest.mark.parametrize("T", [6, 150])
def test_streams_and_graph(T):
    from minicpm5_mk import ops

    h1, w, ids = _inputs(T, 512, 7000, 1, seed=1)
    h2, _, _ = _inputs(T, 512, 1, 1, seed=2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        a = ops.lm_head_logprobs(h1, w, ids)
    with torch.cuda.stream(s2):
        b = ops.lm_head_logprobs(h2, w, ids)
    torch.cuda.synchronize()
    _check(h1, w, ids, a)
    _check(h2, w, ids, b)
    buf = h1.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = ops.lm_head_logprobs(buf, w, ids)
    for h, want in ((h1, a), (h2, b), (h1, a)):
        buf.copy_(h)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(r.token_logprobs, want.token_logprobs) and torch.equal(r.entropy, want.entropy)
        ops.lm_head_logprobs(h2, w, ids)
        torch.cuda.synchronize()


def test_answering_end():
    """Hidden rows through the bf16 head, the fused head and the 4-bit head: the first two agree as f32 sums of one order
    and another do, the third with the logits of the values its weights stand for."""
    from minicpm5_mk import ops

    h, w, ids = _inputs(24, 1536, 32768, 3, seed=11, std=0.02)
    logits = ops.lm_head(h, w)
    a = ops.logprobs(logits, ids, top=20)
    b = ops.lm_head_logprobs(h, w, ids)
    assert float((a.token_logprobs - b.token_logprobs).abs().max()) <= 1e-5 * (1 + float(a.token_logprobs.abs().max()))
    assert float((a.entropy - b.entropy).abs().max()) <= 1e-5 * (1 + float(a.entropy.abs().max()))
    q = ops.quantize_w4(w, 64)
    c = ops.logprobs(ops.gemm_w4(h, q, dtype=F32), ids, top=20)
    v = ops.dequantize_w4(q, dtype=F32)
    want = torch.log_softmax(torch.mm(h.double(), v.double().T.contiguous()), -1)
    assert float((c.token_logprobs.double() - want.gather(1, ids)).abs().max()) <= 1e-4
    best = want.argmax(-1)
    assert ((want.gather(1, best[:, None]) - want.gather(1, c.top_ids[:, :1].long())) <= 1e-4).all()
    # the same token at rank 1 of every listing
    first = ops.logprobs(logits, a.top_ids[:, :1].contiguous())
    assert (first.ranks == 1).all() and torch.equal(first.token_logprobs, a.top_logprobs[:, :1])
