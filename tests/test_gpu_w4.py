"""4-bit weights with group scales: the quantised values bit by bit against the definition on the CPU, the product against
float64, at odd sizes, strides and every group size; refusals, streams and graph replay."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
SMALLEST = 2.0 ** -126


def _weight(n, k, seed=0, std=0.02):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (std * torch.randn((n, k), generator=g, device=DEV)).to(BF16)


def _x(m, k, seed=1):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn((m, k), generator=g, device=DEV) + 0.1).to(BF16)


def _ref(w, group):
    """Values of the 4-bit format on the CPU in float64 (exact: codes of 4 bits times scales of 8)."""
    w = w.detach().cpu()
    out = torch.empty(w.shape, dtype=torch.float64)
    for k0 in range(0, w.shape[1], group):
        g = w[:, k0:k0 + group].float()
        s = (g.abs().amax(1, keepdim=True) / 7).clone()
        s[s < SMALLEST] = 0
        s = s.to(BF16).double()
        c = torch.where(s > 0, torch.round(g.double() / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(g).double())
        v = c.clamp(-7, 7) * s
        bad = ~torch.isfinite(g).all(1)
        v[bad] = float("nan")
        out[:, k0:k0 + group] = v
    return out


SIZES = [(1, 1), (1, 128), (16, 128), (17, 129), (15, 31), (33, 64), (40, 96), (256, 1536), (100, 1000), (16, 8193), (1000, 777)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", SIZES)
def test_quantize(n, k, group):
    from minicpm5_mk import ops

    w = _weight(n, k, seed=n + k)
    q = ops.quantize_w4(w, group)
    assert (q.n, q.k, q.group) == (n, k, group)
    want = _ref(w, group)
    assert torch.equal(ops.dequantize_w4(q, dtype=F32).cpu().double(), want)
    assert torch.equal(ops.dequantize_w4(q).cpu(), want.to(F32).to(BF16))


def test_quantize_special():
    """Ties between codes, empty and tiny groups, the largest values, infinities and NaN (their own group only)."""
    from minicpm5_mk import ops

    w = torch.zeros((8, 96), device=DEV, dtype=BF16)
    w[0, :15] = torch.arange(-7, 8, device=DEV).to(BF16) / 2          # scale 0.5: whole codes
    w[1, :29] = (torch.arange(-14, 15, device=DEV) / 2).to(BF16)      # scale 1: every code and every tie
    w[2, :4] = torch.tensor([1e-38, -3e-38, 2e-38, 8.2e-38]).to(BF16)  # amax / 7 just below the smallest normal
    w[2, 32:36] = torch.tensor([4.2e-38, -1.2e-37, 2e-37, 2.5e-38]).to(BF16)
    w[3, :3] = torch.tensor([3.38e38, -1.7e38, 1e37]).to(BF16)
    w[4, 40] = float("inf")
    w[4, 3] = 1.0
    w[5, 70] = float("nan")
    w[6] = -0.0
    w[7, ::5] = 1e-40
    got = ops.dequantize_w4(ops.quantize_w4(w, 32), dtype=F32).cpu().double()
    want = _ref(w, 32)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~torch.isnan(got)], want[~torch.isnan(want)])
    assert torch.isnan(got[4, 32:64]).all() and torch.isfinite(got[4, :32]).all()
    # -7 .. 7 in halves under scale 1: halves go to even codes
    assert torch.equal(got[1, :29], torch.round(torch.arange(-14, 15).double() / 2))


def test_quantize_strided():
    from minicpm5_mk import ops

    base = torch.full((50, 301), float("nan"), device=DEV, dtype=BF16)
    w = base[1::2, 3:300]
    w.copy_(_weight(25, 297))
    assert torch.equal(ops.dequantize_w4(ops.quantize_w4(w, 64), dtype=F32).cpu().double(), _ref(w, 64))


def _check_gemm(x, q, dtype, got=None):
    """f32 accumulation: per group of g values the sum of (16 + u) x products on a start of -24 sum x (itself g / 8
    serial and a few tree additions), scaled and added over the groups.  Every rounding is half a step of at most the
    magnitudes summed: 2^-24 (31 + 24) sum |x| |s| per addition and group, g + g / 8 + 8 of them at most, plus the
    groups' additions on the total; then the output's own rounding."""
    from minicpm5_mk import ops

    got = (ops.gemm_w4(x, q, dtype=dtype) if got is None else got)
    assert got.shape == (x.shape[0], q.n) and got.dtype == dtype
    w = ops.dequantize_w4(q, dtype=F32).cpu().double()
    xd = x.cpu().double()
    want = xd @ w.T
    groups = -(-q.k // q.group)
    pad = groups * q.group - q.k
    xs = torch.nn.functional.pad(xd.abs(), (0, pad)).view(x.shape[0], groups, q.group).sum(-1)
    ws = torch.nn.functional.pad(w.abs(), (0, pad)).view(q.n, groups, q.group).amax(-1) / 7 * 1.01   # the groups' scales
    tol = 2.0 ** -24 * ((q.group * 9 / 8 + 8) * 55 * (xs @ ws.T) + (groups + 9) * (xd.abs() @ w.abs().T))
    if dtype == BF16:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
    err = (got.cpu().double() - want).abs()
    assert (err <= tol + 1e-300).all(), float((err / (tol + 1e-300)).max())
    # far inside the bound, which adds every rounding's worst: the errors of an f32 sum, not lost bits
    rel = float(err.norm() / want.norm()) if want.norm() else 0.0
    assert rel <= (2.0 ** -8 if dtype == BF16 else 4e-6), rel


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 16, 128), (2, 17, 33), (3, 100, 1000), (16, 256, 1536), (17, 130, 1100), (32, 64, 4608), (33, 40, 200),
    (64, 1000, 777), (5, 8192, 1536), (1, 1536, 4608), (1, 33000, 256), (40, 70000, 128), (65, 48, 300), (130, 100, 520), (5000, 20, 40),
])
def test_gemm(m, n, k, group):
    from minicpm5_mk import ops

    q = ops.quantize_w4(_weight(n, k, seed=n), group)
    x = _x(m, k, seed=m)
    _check_gemm(x, q, F32)
    _check_gemm(x, q, BF16)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_gemm_one_sided_x(group):
    """x of one sign, whose sums are far larger than the result: no more rounding than 16 half steps of the result's norm
    (an f32 product over the weights' values measures 2)."""
    from minicpm5_mk import ops

    q = ops.quantize_w4(_weight(5000, 1536), group)
    w = ops.dequantize_w4(q, dtype=F32).double()
    g = torch.Generator(device=DEV)
    g.manual_seed(8)
    for x in (torch.rand((6, 1536), generator=g, device=DEV), 3 + torch.randn((6, 1536), generator=g, device=DEV),
              torch.exp(1.5 * torch.randn((6, 1536), generator=g, device=DEV))):
        x = x.to(BF16)
        want = torch.mm(x.double(), w.T.contiguous())
        err = ops.gemm_w4(x, q, dtype=F32).double() - want
        assert float(err.norm()) <= 16 * 2.0 ** -24 * float(want.norm())


def test_gemm_rows_alone():
    """A row's result does not depend on the other rows or how many they are: one block or several a wave, K dealt out or
    not."""
    from minicpm5_mk import ops

    for n, k in ((300, 700), (7000, 2300), (66000, 300)):
        q = ops.quantize_w4(_weight(n, k), 64)
        x = _x(150, k)
        full = ops.gemm_w4(x, q, dtype=F32)
        for m0, m1 in ((0, 1), (7, 8), (3, 19), (20, 53), (60, 124), (149, 150)):
            assert torch.equal(ops.gemm_w4(x[m0:m1], q, dtype=F32), full[m0:m1]), (n, m0, m1)


def test_gemm_strides():
    from minicpm5_mk import ops

    q = ops.quantize_w4(_weight(77, 333), 32)
    base = torch.full((9, 701), float("nan"), device=DEV, dtype=BF16)
    x = base[::2, 5:338]
    x.copy_(_x(5, 333))
    want = ops.gemm_w4(x.contiguous(), q, dtype=F32)
    assert torch.equal(ops.gemm_w4(x, q, dtype=F32), want)
    for dt in (F32, BF16):
        room = torch.full((7, 90), 3.0, device=DEV, dtype=dt)
        out = room[1:6, 7:84]
        assert ops.gemm_w4(x, q, out=out) is out
        assert torch.equal(out, want.to(dt))
        room[1:6, 7:84] = 3.0
        assert (room == 3.0).all()


def test_gemm_special():
    from minicpm5_mk import ops

    w = _weight(40, 256)
    w[3, 100] = float("nan")
    w[5] = 0
    q = ops.quantize_w4(w, 64)
    x = _x(4, 256)
    x[2, 7] = float("inf")
    x[3] = 0
    got = ops.gemm_w4(x, q, dtype=F32).cpu()
    assert torch.isnan(got[:, 3]).all() and torch.isnan(got[2]).all()
    keep = [i for i in range(40) if i != 3]
    assert torch.isfinite(got[:2][:, keep]).all()
    assert (got[[0, 1, 3], 5] == 0).all() and (got[3, keep] == 0).all()
    assert ops.gemm_w4(x[:0], q).shape == (0, 40)


def test_refusals():
    from minicpm5_mk import ops

    q = ops.quantize_w4(_weight(40, 256), 64)
    x = _x(4, 256)
    for bad, msg in ((lambda: ops.quantize_w4(x.float()), "expected 2 dimensions"),
                     (lambda: ops.quantize_w4(x, 48), "group"),
                     (lambda: ops.quantize_w4(x.T, 32), "contiguous"),
                     (lambda: ops.quantize_w4(x[:0], 32), "empty"),
                     (lambda: ops.gemm_w4(x[:, :255], q), "columns"),
                     (lambda: ops.gemm_w4(x, q._replace(n=1000)), "bytes of codes"),
                     (lambda: ops.gemm_w4(x, q._replace(scales=q.scales[:-1])), "bf16 scales"),
                     (lambda: ops.gemm_w4(x, q._replace(scales=q.scales.cpu())), "one device"),
                     (lambda: ops.dequantize_w4(q._replace(k=4000)), "bytes of codes"),
                     (lambda: ops.gemm_w4(x.half(), q), "expected 2 dimensions"),
                     (lambda: ops.gemm_w4(x.expand(2, 4, 256), q), "expected 2 dimensions"),
                     (lambda: ops.gemm_w4(x[:1].expand(4, 256), q), "overlap"),
                     (lambda: ops.gemm_w4(x, q, dtype=torch.float16), "dtype"),
                     (lambda: ops.gemm_w4(x, q, out=torch.empty((3, 40), device=DEV)), "rows"),
                     (lambda: ops.gemm_w4(x, q, out=torch.empty((4, 41), device=DEV)), "columns"),
                     (lambda: ops.gemm_w4(x, q, out=torch.empty((4, 40))), "GPU tensor")):
        with pytest.raises(ops.MkError, match=msg):
            bad()


def test_large_offsets():
    """A weight whose values pass 2^31 elements: its last rows."""
    from minicpm5_mk import ops

    n, k = 1050000, 2048
    w = torch.zeros((n, k), device=DEV, dtype=BF16)
    tail = _weight(24, k)
    w[-24:] = tail
    q = ops.quantize_w4(w, 128)
    del w
    x = _x(2, k)
    got = ops.gemm_w4(x, q, dtype=F32)
    small = ops.quantize_w4(tail, 128)
    want = ops.gemm_w4(x, small, dtype=F32)
    assert (got[:, :-24] == 0).all()
    # another division of K over the waves: the same sums in another order
    assert (got[:, -24:] - want).abs().max() <= 1e-5 * want.abs().max()


def test_streams_and_graph():
    from minicpm5_mk import ops

    w1, w2 = _weight(500, 1536, seed=4), _weight(500, 1536, seed=5)
    x1, x2 = _x(3, 1536, seed=6), _x(3, 1536, seed=7)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        a = ops.gemm_w4(x1, ops.quantize_w4(w1, 64), dtype=F32)
    with torch.cuda.stream(s2):
        b = ops.gemm_w4(x2, ops.quantize_w4(w2, 64), dtype=F32)
    torch.cuda.synchronize()
    _check_gemm(x1, ops.quantize_w4(w1, 64), F32, a)
    _check_gemm(x2, ops.quantize_w4(w2, 64), F32, b)

    wb, xb = w1.clone(), x1.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = ops.quantize_w4(wb, 64)
        y = ops.gemm_w4(xb, q, dtype=F32)
        d = ops.dequantize_w4(q)
    for w, x, want in ((w1, x1, a), (w2, x2, b), (w1, x1, a)):
        wb.copy_(w)
        xb.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert torch.equal(d, ops.dequantize_w4(ops.quantize_w4(w, 64)))
        torch.cuda.synchronize()
