"""The launch rules of the answering-end operators (csrc/rules.h), compiled with the host compiler and checked on the CPU."""
import ctypes
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "minicpm5-vllm-tpu_amd", "csrc")

SRC = r"""
#include "rules.h"
extern "C" void logprob_plan(int T, int V, int* out) {
  const mk::LogprobPlan p = mk::logprob_plan(T, V);
  out[0] = p.splits, out[1] = p.waves;
}
extern "C" void w4_plan(int M, long nrb, int nkb, int* out) {
  const mk::W4Plan p = mk::w4_plan(M, nrb, nkb);
  out[0] = p.mg, out[1] = p.r, out[2] = p.kw, out[3] = p.bpc;
}
extern "C" int lse_tile(int T) { return mk::lse_tile(T); }
extern "C" int head_logprobs_stored(int T) { return mk::head_logprobs_stored(T); }
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("answer_rules")
    (d / "rules.cpp").write_text(SRC)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "rules.cpp"), "-o",
                    str(d / "rules.so")], check=True)
    return ctypes.CDLL(str(d / "rules.so"))


def _ints(fn, n, *args):
    out = (ctypes.c_int * n)()
    fn(*args, out)
    return tuple(out)


def test_logprob_plan(rules):
    """One workgroup a row or splits of whole 1024-value tiles, at most one workgroup a CU where rows are split."""
    for T in (1, 2, 3, 33, 64, 85, 86, 128, 129, 255, 256, 257, 896, 897, 5000, 1 << 20):
        for V in (1, 1023, 16384, 32768, 32769, 65536, 130560, 1 << 20, 1 << 30):
            splits, waves = _ints(rules.logprob_plan, 2, T, V)
            assert waves in (4, 8, 16) and splits >= 1
            assert splits == 1 or (waves == 16 and T * splits <= 256 and splits <= -(-V // 16384))
    assert _ints(rules.logprob_plan, 2, 1, 130560) == (8, 16) and _ints(rules.logprob_plan, 2, 33, 130560) == (4, 16)
    assert _ints(rules.logprob_plan, 2, 200, 130560) == (1, 16) and _ints(rules.logprob_plan, 2, 500, 130560) == (1, 8)
    assert _ints(rules.logprob_plan, 2, 2048, 130560) == (1, 4)


def test_w4_plan(rules):
    """The staged x fits its LDS, K is dealt to a divisor of a workgroup's waves and the same for every M."""
    for nrb in (1, 19, 96, 399, 400, 576, 2048, 4095, 4096, 8160, 1 << 26):
        for nkb in (1, 2, 3, 7, 12, 36, 64, 1000):
            deal = set()
            for M in (1, 2, 15, 16, 17, 32, 33, 40, 48, 63, 64, 65, 200, 1 << 19):
                mg, r, kw, bpc = _ints(rules.w4_plan, 4, M, ctypes.c_long(nrb), nkb)
                deal.add((r, kw))
                rows = min(M, 16) if mg == 1 else 16 * mg
                assert 1 <= mg <= 4 and r in (1, 2) and kw in (1, 2, 4, 8) and kw <= nkb and (r == 1 or kw == 1)
                assert bpc >= 1 and bpc % kw == 0 and bpc * rows * 256 <= (64 if mg == 1 else 128) * 1024
                if mg > 1:
                    assert 16 * (mg - 1) < M
            assert len(deal) == 1
    assert _ints(rules.w4_plan, 4, 1, ctypes.c_long(96), 36) == (1, 1, 8, 40)
    assert _ints(rules.w4_plan, 4, 40, ctypes.c_long(8160), 16) == (3, 2, 1, 8)


def test_head_logprob_rules(rules):
    assert [rules.head_logprobs_stored(t) for t in (1, 64, 65, 8192)] == [1, 1, 0, 0]
    assert [rules.lse_tile(t) for t in (65, 128, 129, 192, 193, 256, 257, 320, 321, 384, 385, 512, 513, 640, 645, 768, 8192)] == [
        2, 2, 5, 5, 4, 4, 8, 8, 5, 5, 4, 4, 8, 8, 4, 4, 4]
