"""The argument checks of the answering-end entry points (log probabilities, LM head with log probabilities, 4-bit
products), on the host: no GPU call is reached."""
import ctypes

import pytest
import torch

from minicpm5_mk import _lib, ops

BOGUS = 1 << 20      # a pointer the checks never follow


def _err():
    return _lib.load().mk_last_error().decode()


def _logprobs(**kw):
    a = dict(logits=BOGUS, type=0, ld=1000, T=2, V=1000, ids=BOGUS, ids64=1, n_ids=1, top=3, token_lp=BOGUS, ranks=BOGUS,
             top_lp=BOGUS, top_ids=BOGUS, entropy=BOGUS, lse=BOGUS, scratch=BOGUS, scratch_bytes=1 << 30)
    a.update(kw)
    return _lib.load().mk_logprobs(*a.values(), None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(type=3), -1, "type"),
    (dict(T=-1), -1, "T must be"),
    (dict(V=0), -1, "V"),
    (dict(n_ids=65), -1, "given tokens"),
    (dict(top=65), -1, "top"),
    (dict(top=5, V=4, ld=4), -1, "top"),
    (dict(ld=999), -1, "stride"),
    (dict(logits=None), -1, "null"),
    (dict(entropy=None), -1, "null"),
    (dict(ranks=None), -1, "given tokens"),
    (dict(top_ids=None), -1, "alternatives"),
    (dict(logits=BOGUS + 2), -1, "aligned"),
    (dict(V=100000, ld=100000, scratch_bytes=16), -4, "scratch"),
    (dict(V=100000, ld=100000, scratch=BOGUS + 8), -1, "16-byte"),
    (dict(T=0), 0, ""),
])
def test_logprobs_refusals(kw, code, msg):
    assert _logprobs(**kw) == code
    if code:
        assert msg in _err()


def test_logprobs_scratch():
    f = _lib.load().mk_logprobs_scratch_bytes
    assert f(2000, 130560, 1, 20) == 0 and f(4, 32768, 1, 20) == 0   # one workgroup a row
    assert f(1, 130560, 1, 20) == 8 * (4 + 2 + 40) * 4               # 8 of 16384 values
    assert f(0, 130560, 1, 20) == 0 and f(1, 0, 1, 1) == 0


def test_logprobs_cpu_tensor():
    with pytest.raises(_lib.MkError, match="GPU tensor"):
        ops.logprobs(torch.zeros(2, 8))
    with pytest.raises(_lib.MkError, match="torch.Tensor"):
        ops.logprobs([[0.0]])


def _head(**kw):
    a = dict(hidden=BOGUS, weight=BOGUS, T=100, H=64, V=1000, ids=BOGUS, ids64=0, n_ids=1, token_lp=BOGUS, entropy=BOGUS,
             lse=BOGUS, scratch=BOGUS, scratch_bytes=1 << 30)
    a.update(kw)
    return _lib.load().mk_lm_head_logprobs(*a.values(), None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(T=-1), -1, "T must be"),
    (dict(V=0), -1, "V"),
    (dict(H=0), -1, "multiple of 32"),
    (dict(H=48), -1, "multiple of 32"),
    (dict(n_ids=65), -1, "given tokens"),
    (dict(hidden=None), -1, "null"),
    (dict(token_lp=None), -1, "given tokens"),
    (dict(hidden=BOGUS + 8), -1, "16-byte"),
    (dict(weight=BOGUS + 2), -1, "16-byte"),
    (dict(scratch=None), -4, "scratch"),
    (dict(scratch_bytes=100), -4, "scratch"),
    (dict(scratch=BOGUS + 4), -1, "16-byte"),
    (dict(T=0), 0, ""),
])
def test_head_logprobs_refusals(kw, code, msg):
    assert _head(**kw) == code
    if code:
        assert msg in _err()


def test_head_logprobs_scratch():
    f = _lib.load().mk_lm_head_logprobs_scratch_bytes
    assert f(8192, 130560, 1) == 510 * 3 * 8192 * 4              # statistics of 256 tokens at a time
    assert f(1 << 20, 130560, 1) == f(16384, 130560, 1)          # in passes
    assert f(2, 1000, 1) == 8192                                 # two rows of logits, in whole 256 bytes
    assert f(0, 1000, 1) == 0


def _w4(name, **kw):
    lib = _lib.load()
    d = dict(x=BOGUS, ldx=256, w=BOGUS, ldw=256, codes=BOGUS, scales=BOGUS, M=2, N=100, K=256, group=64, out=BOGUS, f32=0,
             ldo=256)
    d.update(kw)
    if name == "quantize":
        return lib.mk_w4_quantize(d["w"], d["ldw"], d["N"], d["K"], d["group"], d["codes"], d["scales"], None)
    if name == "dequantize":
        return lib.mk_w4_dequantize(d["codes"], d["scales"], d["N"], d["K"], d["group"], d["out"], d["f32"], d["ldo"], None)
    return lib.mk_gemm_w4(d["x"], d["ldx"], d["codes"], d["scales"], d["M"], d["N"], d["K"], d["group"], d["out"], d["f32"],
                          d["ldo"], None)


@pytest.mark.parametrize("name,kw,code,msg", [
    *[(n, dict(group=g), -1, "group") for n in ("quantize", "dequantize", "gemm") for g in (0, 16, 96, 256)],
    *[(n, kw, -1, "empty") for n in ("quantize", "dequantize", "gemm") for kw in (dict(N=0), dict(K=0))],
    *[(n, dict(codes=None), -1, "null") for n in ("quantize", "dequantize", "gemm")],
    *[(n, dict(scales=BOGUS + 16), -1, "32-byte") for n in ("quantize", "dequantize", "gemm")],
    *[(n, dict(N=1 << 30, K=1 << 30, ldw=1 << 30, ldx=1 << 30, ldo=1 << 30), -1, "large")
      for n in ("quantize", "dequantize", "gemm")],
    ("quantize", dict(w=None), -1, "null"),
    ("quantize", dict(ldw=255), -1, "stride"),
    ("dequantize", dict(out=BOGUS + 2, f32=1), -1, "misaligned"),
    ("dequantize", dict(ldo=255), -1, "stride"),
    ("gemm", dict(M=-1), -1, "M must be"),
    ("gemm", dict(M=(1 << 19) + 1), -1, "M must be"),
    ("gemm", dict(x=None), -1, "null"),
    ("gemm", dict(x=BOGUS + 1), -1, "misaligned"),
    ("gemm", dict(ldx=255), -1, "stride"),
    ("gemm", dict(ldo=99), -1, "stride"),
    ("gemm", dict(M=0), 0, ""),
])
def test_w4_refusals(name, kw, code, msg):
    assert _w4(name, **kw) == code
    if code:
        assert msg in _err()


def test_w4_bytes():
    c, s = ctypes.c_size_t(), ctypes.c_size_t()
    f = _lib.load().mk_w4_bytes
    assert f(33, 130, 32, ctypes.byref(c), ctypes.byref(s)) == 0
    assert (c.value, s.value) == (3 * 2 * 1024, 3 * 2 * 16 * 4 * 2)
    assert f(130560, 1536, 128, ctypes.byref(c), ctypes.byref(s)) == 0
    assert (c.value, s.value) == (130560 * 1536 // 2, 130560 * 12 * 2)
    assert f(1, 1, 32, None, None) == -1


def test_w4_cpu_tensors():
    with pytest.raises(_lib.MkError, match="GPU tensor"):
        ops.quantize_w4(torch.zeros(4, 64, dtype=torch.bfloat16))
    with pytest.raises(_lib.MkError, match="W4Weight"):
        ops.gemm_w4(torch.zeros(1, 64, dtype=torch.bfloat16), torch.zeros(4, 64))
    with pytest.raises(_lib.MkError, match="W4Weight"):
        ops.dequantize_w4(None)
    z = torch.zeros(1024, dtype=torch.uint8)
    w = ops.W4Weight(z, z.bfloat16(), 4, 64, 64)
    with pytest.raises(_lib.MkError, match="dtype"):
        ops.dequantize_w4(w, dtype=torch.float16)
    with pytest.raises(_lib.MkError, match="GPU tensors"):
        ops.gemm_w4(torch.zeros(1, 64, dtype=torch.bfloat16), w)
    with pytest.raises(_lib.MkError, match="group"):
        ops.gemm_w4(torch.zeros(1, 64, dtype=torch.bfloat16), w._replace(group=48))


def test_candidate_ids():
    from minicpm5_mk.engine import candidate_ids

    assert torch.equal(candidate_ids([5, 7], 3, 10), torch.tensor([[5, 7]] * 3))
    assert torch.equal(candidate_ids([[1, 2], [3, 4]], 2, 10), torch.tensor([[1, 2], [3, 4]]))
    assert candidate_ids([], 2, 10).shape == (2, 0)
    assert candidate_ids(torch.tensor([[1], [9]], dtype=torch.int32), 2, 10).dtype == torch.int64
    for bad, msg in (([10], "token ids"), ([-1], "token ids"), ([[1], [2]], "shape"), ([[[1]]], "shape"), ([0.5], "expected"),
                     (list(range(65)), "at most"), ([True], "expected")):
        with pytest.raises(ValueError, match=msg):
            candidate_ids(bad, 3, 10 if len(bad) < 65 else 100)


def test_engine_head_option():
    from minicpm5_mk.engine import MkEngine

    with pytest.raises(ValueError, match="lm_head_quant"):
        MkEngine("tiny", lm_head_quant="w3", log=lambda *a: None)
