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
