"""ops.logprobs against the definition in float64: values, ranks, order among equals, masked rows, strides, splits,
refusals, streams and graph replay."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
INF = float("inf")


def _ref(x, ids, top):
    """Definition on the CPU in float64; x (T, V) any float type."""
    x = x.detach().cpu().double()
    T, V = x.shape
    m = x.max(-1, keepdim=True).values
    bad = ~((x == x).all(-1) & (m.squeeze(-1) < INF))
    empty = (m.squeeze(-1) == -INF) & ~bad
    safe = torch.where((bad | empty).unsqueeze(-1), torch.zeros_like(x), x)
    lp = torch.log_softmax(safe, -1)
    lse = torch.logsumexp(safe, -1)
    p = lp.exp()
    ent = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    lp[empty] = -INF
    lse[empty], ent[empty] = -INF, 0.0
    lp[bad], lse[bad], ent[bad] = float("nan"), float("nan"), float("nan")
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    place = torch.empty_like(order).scatter_(1, order, torch.arange(1, V + 1).expand(T, V).contiguous())
    out = {"ent": ent, "lse": lse}
    if ids is not None:
        i = ids.detach().cpu().long().reshape(T, -1)
        ok = (i >= 0) & (i < V)
        j = torch.where(ok, i, torch.zeros_like(i))
        nan = bad.unsqueeze(1).expand_as(i)
        out["lp"] = torch.where(ok | nan, lp.gather(1, j), torch.full(i.shape, -INF, dtype=torch.float64)).reshape(ids.shape)
        out["rank"] = torch.where(ok & ~nan, place.gather(1, j), torch.full_like(i, -1)).reshape(ids.shape)
    if top:
        out["top_ids"] = torch.where(bad.unsqueeze(1), torch.full_like(order[:, :top], -1), order[:, :top])
        out["top"] = torch.where(bad.unsqueeze(1), lp[:, :top], lp.gather(1, order[:, :top]))
    return out


def _close(got, want, x, what):
    """Roundings of f32 (half a step, 2^-24 each) counted along one value: 16 + V / 4096 + 1 additions of a lane, 16
    merges of three roundings and two exponentials each, the exponentials' arguments (|d| log2 e, their mean at most
    ln V), the final logarithm, differences and quotient; each relative to what it adds up."""
    V = x.shape[1]
    got = got.detach().cpu().double()
    steps = 17 + V / 4096 + 16 * 7 + 4 * 12 + 8
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), what
    err = (got[fin] - want[fin]).abs() / (1 + want[fin].abs())
    assert err.numel() == 0 or err.max() <= steps * 2.0 ** -24, (what, float(err.max()), steps * 2.0 ** -24)


def _check(x, ids, top, r=None):
    from minicpm5_mk import ops

    r = ops.logprobs(x, ids, top=top) if r is None else r
    want = _ref(x, ids, top)
    _close(r.entropy, want["ent"], x, "entropy")
    _close(r.logsumexp, want["lse"], x, "logsumexp")
    if ids is None:
        assert r.token_logprobs is None and r.ranks is None
    else:
        assert r.token_logprobs.shape == ids.shape and r.ranks.dtype == torch.int32
        _close(r.token_logprobs, want["lp"], x, "token_logprobs")
        assert torch.equal(r.ranks.cpu().long(), want["rank"].long())
    if top:
        assert r.top_ids.dtype == torch.int32 and r.top_ids.shape == (x.shape[0], top)
        assert torch.equal(r.top_ids.cpu().long(), want["top_ids"].long())
        _close(r.top_logprobs, want["top"], x, "top_logprobs")
    else:
        assert r.top_logprobs is None and r.top_ids is None
    return r


def _logits(T, V, dtype, seed=0, scale=2.5):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (scale * torch.randn((T, V), generator=g, device=DEV) + 3).to(dtype)


def _ids(T, V, n, seed=1, dtype=torch.int64):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randint(0, V, (T, n), generator=g, device=DEV, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V,n,top", [
    (1, 1, 1, 1), (1, 2, 2, 2), (3, 63, 1, 20), (2, 64, 1, 64), (5, 1023, 3, 7), (1, 1024, 1, 1), (1, 4096, 1, 5),
    (1, 4097, 1, 5), (2, 32768, 4, 0), (7, 12289, 2, 33), (1, 130560, 1, 20), (3, 130559, 64, 64), (300, 5000, 1, 20),
    (256, 8193, 2, 64), (257, 1000, 1, 3),
])
def test_sizes(T, V, n, top, dtype):
    """Rows in one and in several workgroups, whole and ragged tiles; half-precision logits are full of equals."""
    _check(_logits(T, V, dtype, seed=V), _ids(T, V, n), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [2, 300])
def test_orders(T, dtype):
    """Ascending, descending, constant and few-valued rows: every value beats the list so far, none does, all tie."""
    V = 20000
    up = torch.linspace(-8, 8, V, device=DEV)
    rows = torch.stack([up, up.flip(0), torch.zeros(V, device=DEV), (torch.arange(V, device=DEV) % 3).float(),
                        torch.where(torch.arange(V, device=DEV) < V - 10, -INF, 1.0), -up.abs()])
    x = rows.repeat((T + 5) // 6, 1)[:T].to(dtype).contiguous() if T > 6 else rows.to(dtype)
    _check(x, _ids(x.shape[0], V, 5), 20)
    _check(x, _ids(x.shape[0], V, 5), 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [8, 264])
def test_masks(T, dtype):
    """Masked values: -inf, the type's lowest value, rows that leave one token, three tokens or none; infinities and NaN."""
    V = 9001
    x = _logits(T, V, dtype, seed=3)
    low = torch.finfo(dtype).min
    x[0, :] = -INF
    x[1, :] = low
    x[2, :] = -INF
    x[2, 4242] = 1.5
    x[3, :] = low
    x[3, 17] = -2.0
    x[4, :] = -INF
    x[4, [5, 8000, 9000]] = torch.tensor([0.5, 0.5, -1.0], device=DEV, dtype=dtype)
    x[5, 8999] = float("nan")
    x[6, 0] = INF
    x[7, ::2] = -INF
    ids = _ids(T, V, 6)
    ids[:, 0] = 4242
    ids[:, 1] = 17
    r = _check(x, ids, 12)
    assert torch.isfinite(r.token_logprobs[1]).all()     # equal lowest values: ln(1 / V) each, not 0
    assert float(r.entropy[0]) == 0.0 and float(r.entropy[2]) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,V", [(3, 1), (6, 700), (3, 32768), (2, 130560), (40, 70001), (300, 33000), (1000, 20000)])
def test_certain_tokens(T, V, dtype):
    """Rows where one token outweighs all others: its log probability and the entropy are sums of the others' small
    terms, each off by its exponent's roundings (|d| log2 e at 2^-24 twice, |d| <= 60) and the exponential's 2^-23, then
    a few hundred additions of one sign."""
    from minicpm5_mk import ops

    x = _logits(T, V, dtype, scale=1.0)
    at = _ids(T, V, 1, seed=V)
    for up in (12.0, 20.0, 40.0):
        x.scatter_(1, at, up)
        r = ops.logprobs(x, at, top=1)
        d = x.cpu().double() - up
        rest = d.exp().scatter(1, at.cpu(), 0.0).sum(-1)
        lp, ent = -torch.log1p(rest), torch.log1p(rest) - (d.exp() * d).sum(-1) / (1 + rest)
        tol = (2 * 60 * 1.5 + 2 + 400) * 2.0 ** -24
        assert ((r.token_logprobs[:, 0].cpu().double() - lp).abs() <= tol * lp.abs()).all()
        assert ((r.entropy.cpu().double() - ent).abs() <= tol * ent.abs()).all()
        assert torch.equal(r.top_ids.long(), at) and (r.ranks == 1).all()
        assert torch.equal(r.top_logprobs, r.token_logprobs)


@pytest.mark.parametrize("T", [2, 100, 300, 1000])
def test_one_lowest_value(T):
    """One finite token, the type's lowest, among -inf: certain."""
    from minicpm5_mk import ops

    x = torch.full((T, 40000), -INF, device=DEV)
    x[:, 39001] = torch.finfo(torch.float32).min
    r = ops.logprobs(x, torch.full((T, 1), 39001, device=DEV), top=2)
    assert (r.token_logprobs == 0).all() and (r.entropy == 0).all() and (r.top_ids == torch.tensor([39001, 0], device=DEV)).all()


def test_ids_outside():
    x = _logits(4, 5000, torch.float32)
    ids = torch.tensor([[-1, 0, 4999], [5000, -100, 1], [2 ** 40, -2 ** 40, 2], [3, 3, 3]], device=DEV)
    _check(x, ids, 3)
    _check(x, ids[:, 0].clamp(-5, 6000).contiguous(), 0)          # (T,)
    _check(x, ids.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32), 3)
    _check(x, None, 4)
    _check(x, None, 0)
    _check(x, torch.empty((4, 0), dtype=torch.int64, device=DEV), 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [3, 260])
def test_strides(T, dtype):
    """A slice of a padded vocabulary: odd row stride and start, what lies beside the slice never read as a logit."""
    base = torch.full((T, 7013), float("nan"), device=DEV, dtype=dtype)
    x = base[:, 3:7004]
    x.copy_(_logits(T, 7001, dtype))
    _check(x, _ids(T, 7001, 2), 9)
    col = _logits(T, 1, dtype)
    _check(col, _ids(T, 1, 1), 1)


def test_far_row():
    """Rows beyond 2^31 elements and 2^32 bytes."""
    V, T = 130560, 17000
    x = torch.zeros((T, V), device=DEV, dtype=torch.bfloat16)
    last = _logits(2, V, torch.bfloat16, seed=9)
    x[-2:] = last
    ids = _ids(T, V, 1)
    from minicpm5_mk import ops

    r = ops.logprobs(x, ids, top=5)
    _check(last, ids[-2:], 5, type(r)(*[v[-2:] for v in r]))


def test_no_rows():
    from minicpm5_mk import ops

    r = ops.logprobs(torch.empty((0, 100), device=DEV), torch.empty((0, 2), dtype=torch.int64, device=DEV), top=3)
    assert r.token_logprobs.shape == (0, 2) and r.top_ids.shape == (0, 3) and r.entropy.shape == (0,)


def test_repeats_are_equal():
    x, ids = _logits(5, 100003, torch.float32), _ids(5, 100003, 3)
    from minicpm5_mk import ops

    a = ops.logprobs(x, ids, top=20)
    for _ in range(3):
        b = ops.logprobs(x, ids, top=20)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_streams_and_graph():
    """Another stream than the default, two streams at once, and a captured call replayed on new logits."""
    from minicpm5_mk import ops

    x, y, ids = _logits(3, 50021, torch.float32), _logits(3, 50021, torch.float32, seed=5), _ids(3, 50021, 2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        a = ops.logprobs(x, ids, top=8)
    with torch.cuda.stream(s2):
        b = ops.logprobs(y, ids, top=8)
    torch.cuda.synchronize()
    _check(x, ids, 8, a)
    _check(y, ids, 8, b)

    buf = x.clone()
    with torch.cuda.stream(s1):
        ops.logprobs(buf, ids, top=8)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = ops.logprobs(buf, ids, top=8)
    for src in (x, y, x, y):
        buf.copy_(src)
        g.replay()
        torch.cuda.synchronize()
        eager = ops.logprobs(src, ids, top=8)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(r, eager))
