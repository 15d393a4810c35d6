"""torch-facing wrappers of libmk's kernel-level entry points.

PyTorch provides device memory and the current HIP stream; every computation runs in libmk's HIP
kernels.  Each wrapper checks dtypes, devices, contiguity and shapes on the host before the launch
(the kernels assume them) and raises `MkError` with libmk's message on any failure.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib
from ._lib import EPI, MkError, check, load

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _need(t: torch.Tensor, name: str, dtype=None, shape=None):
    if not isinstance(t, torch.Tensor):
        raise MkError(f"{name}: expected a torch.Tensor")
    if not t.is_cuda:
        raise MkError(f"{name}: must be a GPU tensor (libmk has no CPU path)")
    if not t.is_contiguous():
        raise MkError(f"{name}: must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise MkError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise MkError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.data_ptr() % 16:
        raise MkError(f"{name}: must be 16-byte aligned")


def _need_rows(t: torch.Tensor, name: str, dtypes, cols: int | None = None):
    """A (rows, cols) GPU tensor of one of `dtypes` whose rows are contiguous, at any row stride and alignment ->
    (rows, cols, row stride)."""
    if not isinstance(t, torch.Tensor):
        raise MkError(f"{name}: expected a torch.Tensor")
    if not t.is_cuda:
        raise MkError(f"{name}: must be a GPU tensor (libmk has no CPU path)")
    if t.ndim != 2 or t.dtype not in dtypes:
        raise MkError(f"{name}: {tuple(t.shape)} {t.dtype}, expected 2 dimensions of {' / '.join(str(d) for d in dtypes)}")
    rows, c = t.shape
    if cols is not None and c != cols:
        raise MkError(f"{name}: {c} columns, expected {cols}")
    s0, s1 = t.stride()
    if (s1 != 1 and c > 1 and rows > 0) or (s0 < c and rows > 1):
        raise MkError(f"{name}: rows must be contiguous and must not overlap")
    return rows, c, s0


def _same_device(t: torch.Tensor, **others):
    for name, o in others.items():
        if o is not None and o.device != t.device:
            raise MkError(f"{name}: on {o.device}, expected {t.device}")


def _call(t: torch.Tensor, fn, what: str, *args):
    """check(fn(*args, stream)) with t's device the current one and that device's current stream (its raw handle: a
    Stream object around it costs 2.7 us of a call)."""
    dev = t.get_device()
    if dev == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        check(rc, what)


def _adr(t):
    return t.data_ptr() if t is not None else None


def attn_scratch_bytes(B: int, S: int, n_kv: int, head_dim: int) -> int:
    return int(load().mk_attn_scratch_bytes(B, S, n_kv, head_dim))


def attn_prefill(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, n_q: int, n_kv: int, head_dim: int,
                 sm_scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA prefill attention (super_gqa_v2, plugin/minicpm5_mk/mk_attn.py:660-710).

    qkv (B, S, (n_q + 2 n_kv) hd) bf16 -> (B, S, n_q hd) bf16; RoPE from the bf16 tables in-kernel."""
    lib = load()
    B, S, D = qkv.shape
    if D != (n_q + 2 * n_kv) * head_dim:
        raise MkError(f"qkv last dim {D} != (n_q + 2 n_kv) * head_dim")
    _need(qkv, "qkv", BF16)
    _need(cos, "cos", BF16)
    _need(sin, "sin", BF16)
    if cos.shape[0] < S or cos.shape[1] != head_dim or sin.shape != cos.shape:
        raise MkError("cos / sin must be (>= S, head_dim)")
    if out is None:
        out = torch.empty((B, S, n_q * head_dim), dtype=BF16, device=qkv.device)
    _need(out, "out", BF16, (B, S, n_q * head_dim))
    nbytes = attn_scratch_bytes(B, S, n_kv, head_dim)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=qkv.device)
    check(lib.mk_attn_prefill(_ptr(qkv), _ptr(cos), _ptr(sin), _ptr(out), _ptr(scratch), nbytes, B, S, n_q, n_kv,
                              head_dim, float(sm_scale), _stream()), "mk_attn_prefill")
    return out


def row_quant(x: torch.Tensor, a: torch.Tensor | None, eps: float = 1e-6, norm: bool = True, recip: bool = True):
    """Per-token dynamic int8 quantisation (+ RMSNorm statistics): returns (q int8 (T, H), sx f32 (T,))."""
    lib = load()
    if x.dim() != 2 or x.dtype not in (BF16, torch.float32):
        raise MkError("row_quant: x must be (T, H) bf16 or f32")
    T, H = x.shape
    _need(x, "x")
    if a is not None:
        _need(a, "a", torch.float32, (H,))
    q = torch.empty((T, H), dtype=torch.int8, device=x.device)
    sx = torch.empty((T,), dtype=torch.float32, device=x.device)
    check(lib.mk_row_quant(_ptr(x), int(x.dtype == torch.float32), _ptr(a), T, H, float(eps), int(norm), int(recip),
                           _ptr(q), _ptr(sx), _stream()), "mk_row_quant")
    return q, sx


ACT_MODES = {"int8d": 0, "fp8d": 1, "int8": 2, "fp8": 3}
FP8 = torch.float8_e4m3fn


def act_quant(x: torch.Tensor, a: torch.Tensor | None, mode: str, eps: float = 1e-6, norm: bool = False,
              recip: bool = False, smul: bool = False):
    """Activation quantisation in one of the reference's modes (include/mk.h, mk_act_quant): returns
    (q (T, H) int8 or float8_e4m3fn, sx f32 (T,))."""
    lib = load()
    if mode not in ACT_MODES:
        raise MkError(f"act_quant: unknown mode {mode!r}")
    if x.dim() != 2 or x.dtype not in (BF16, torch.float32):
        raise MkError("act_quant: x must be (T, H) bf16 or f32")
    T, H = x.shape
    _need(x, "x")
    if a is not None:
        _need(a, "a", torch.float32, (H,))
    q = torch.empty((T, H), dtype=FP8 if mode.startswith("fp8") else torch.int8, device=x.device)
    sx = torch.empty((T,), dtype=torch.float32, device=x.device)
    flags = int(norm) | 2 * int(recip) | 4 * int(smul)
    check(lib.mk_act_quant(_ptr(x), int(x.dtype == torch.float32), _ptr(a), T, H, float(eps), ACT_MODES[mode], flags,
                           _ptr(q), _ptr(sx), _stream()), "mk_act_quant")
    return q, sx


def gemm(A: torch.Tensor, B: torch.Tensor, epi: str, out: torch.Tensor | None = None, res: torch.Tensor | None = None,
         rs: torch.Tensor | None = None, cs: torch.Tensor | None = None, aux: torch.Tensor | None = None):
    """C = A (M, K) @ B (N, K)^T with a fused epilogue (see include/mk.h MK_EPI_*).

    int8 operands -> int8 MFMA with int32 accumulation; bf16 / float8_e4m3fn operands -> bf16 / fp8 MFMA,
    f32 accumulation."""
    lib = load()
    if epi not in EPI:
        raise MkError(f"unknown epilogue {epi!r}")
    if A.dim() != 2 or B.dim() != 2 or A.shape[1] != B.shape[1] or A.dtype != B.dtype:
        raise MkError("gemm: A (M, K) and B (N, K) must share K and dtype")
    if A.dtype not in (torch.int8, BF16, FP8):
        raise MkError("gemm: operands must be int8, bf16 or float8_e4m3fn")
    _need(A, "A")
    _need(B, "B")
    M, K = A.shape
    N = B.shape[0]
    silu = epi in ("dq_silu", "dq_silu_f32a", "silu_bf16")
    n_out = N // 2 if silu else N
    residual = epi in ("res_bf16add", "dq_res_bf16add", "res_f32add", "dq2_res_f32add", "dq2_res_bf16add")
    if residual:
        if res is None:
            raise MkError("gemm: residual epilogue needs `res`")
        _need(res, "res", BF16, (M, N))
    elif out is None:
        dt = {"f32": torch.float32, "i32": torch.int32, "dq_silu_f32a": torch.float32}.get(epi, BF16)
        out = torch.empty((M, n_out), dtype=dt, device=A.device)
    if out is not None:
        _need(out, "out", None, (M, n_out))
    for t, nm, n in ((rs, "rs", M), (cs, "cs", N), (aux, "aux", n_out)):
        if t is not None:
            _need(t, nm, torch.float32, (n,))
    in_type = {BF16: 0, torch.int8: 1, FP8: 2}[A.dtype]
    check(lib.mk_gemm(in_type, EPI[epi], _ptr(A), K, _ptr(B), K, M, N, K, _ptr(out),
                      n_out if out is not None else 0, _ptr(res), N if res is not None else 0, _ptr(rs), _ptr(cs),
                      _ptr(aux), _stream()), "mk_gemm")
    return res if residual else out


def lm_head(hidden: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """logits (B, V) f32 = hidden (B, H) bf16 @ weight (V, H)^T."""
    lib = load()
    B, H = hidden.shape
    V = weight.shape[0]
    _need(hidden, "hidden", BF16)
    _need(weight, "lm_head", BF16, (V, H))
    out = torch.empty((B, V), dtype=torch.float32, device=hidden.device)
    check(lib.mk_lm_head(_ptr(hidden), _ptr(weight), B, H, V, _ptr(out), _stream()), "mk_lm_head")
    return out


class LogProbs(NamedTuple):
    """Log probabilities of T rows (nats, f32).  ids None: no token_logprobs / ranks; top 0: no top_*."""
    token_logprobs: torch.Tensor | None   # of ids' shape
    ranks: torch.Tensor | None            # int32, of ids' shape; 1 = the most likely token
    top_logprobs: torch.Tensor | None     # (T, top), descending
    top_ids: torch.Tensor | None          # (T, top) int32
    entropy: torch.Tensor                 # (T,)
    logsumexp: torch.Tensor               # (T,)


LOGPROBS_MAX = 64
LOGITS_TYPES = {torch.float32: 0, BF16: 1, torch.float16: 2}


def _need_ids(ids, rows: int):
    """Given tokens (rows,) or (rows, n <= 64), int32 or int64 -> n."""
    if not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int32, torch.int64):
        raise MkError("ids: expected an int32 or int64 tensor")
    if not ids.is_cuda:
        raise MkError("ids: must be a GPU tensor (libmk has no CPU path)")
    if ids.dim() not in (1, 2) or ids.shape[0] != rows:
        raise MkError(f"ids: shape {tuple(ids.shape)}, expected ({rows},) or ({rows}, n)")
    if not ids.is_contiguous():
        raise MkError("ids: must be contiguous")
    n = ids.shape[1] if ids.dim() == 2 else 1
    if n > LOGPROBS_MAX:
        raise MkError(f"ids: {n} given tokens a row, at most {LOGPROBS_MAX}")
    return n


def logprobs(logits: torch.Tensor, ids: torch.Tensor | None = None, top: int = 0) -> LogProbs:
    """Log probabilities of rows of logits (T, V) f32 / bf16 / f16 in one pass (include/mk.h, mk_logprobs): of the
    given tokens `ids` (T,) or (T, n) with their ranks, of the `top` most likely tokens, with entropy and logsumexp.

    Equal logits rank by the lower index.  An id outside [0, V): -inf, rank -1.  A row of only -inf (everything
    masked): log probabilities and logsumexp -inf, entropy 0.  A row with NaN or +inf: NaN, ranks and top_ids -1.
    Rows may be strided (a slice of a padded vocabulary).  No gradient."""
    lib = load()
    T, V, ld = _need_rows(logits, "logits", LOGITS_TYPES)
    if V < 1:
        raise MkError("logits: empty vocabulary")
    top = int(top)
    if not 0 <= top <= min(LOGPROBS_MAX, V):
        raise MkError(f"top: {top}, expected 0 .. {min(LOGPROBS_MAX, V)}")
    n = 0
    lp = rk = tl = ti = None
    if ids is not None:
        n = _need_ids(ids, T)
        _same_device(logits, ids=ids)
        lp, rk = logits.new_empty(ids.shape, dtype=F32), logits.new_empty(ids.shape, dtype=I32)
    if top:
        tl, ti = logits.new_empty((T, top), dtype=F32), logits.new_empty((T, top), dtype=I32)
    ent, lse = logits.new_empty((2, T), dtype=F32).unbind()
    nbytes = int(lib.mk_logprobs_scratch_bytes(T, V, n, top))
    scratch = logits.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(logits, lib.mk_logprobs, "mk_logprobs", _adr(logits), LOGITS_TYPES[logits.dtype], ld, T, V, _adr(ids),
          int(n > 0 and ids.dtype == torch.int64), n, top, _adr(lp), _adr(rk), _adr(tl), _adr(ti), _adr(ent), _adr(lse),
          _adr(scratch), nbytes)
    return LogProbs(lp, rk, tl, ti, ent, lse)


def lm_head_logprobs(hidden: torch.Tensor, weight: torch.Tensor, ids: torch.Tensor | None = None) -> LogProbs:
    """logprobs(lm_head(hidden, weight), ids) without ranks and alternatives, and for more than 64 rows without the
    logits: hidden (T, H) bf16, weight (V, H) bf16, H a multiple of 32 (include/mk.h, mk_lm_head_logprobs).

    For the tokens of whole prompts: a (8192, 130560) f32 matrix of logits is 4.3 GB.  No gradient."""
    lib = load()
    _need(hidden, "hidden", BF16)
    if hidden.dim() != 2 or not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise MkError("lm_head_logprobs: expected hidden (T, H) and weight (V, H)")
    T, H = hidden.shape
    V = weight.shape[0]
    _need(weight, "weight", BF16, (V, H))
    if V < 1:
        raise MkError("weight: empty vocabulary")
    n = 0 if ids is None else _need_ids(ids, T)
    _same_device(hidden, weight=weight, ids=ids)
    lp = None if ids is None else hidden.new_empty(ids.shape, dtype=F32)
    ent, lse = hidden.new_empty((2, T), dtype=F32).unbind()
    nbytes = int(lib.mk_lm_head_logprobs_scratch_bytes(T, V, n))
    scratch = hidden.new_empty(nbytes, dtype=torch.uint8)
    _call(hidden, lib.mk_lm_head_logprobs, "mk_lm_head_logprobs", _adr(hidden), _adr(weight), T, H, V, _adr(ids),
          int(n > 0 and ids.dtype == torch.int64), n, _adr(lp), _adr(ent), _adr(lse), _adr(scratch), nbytes)
    return LogProbs(lp, None, None, None, ent, lse)


class W4Weight(NamedTuple):
    """A weight (n, k) in 4 bits with a bf16 scale per row and `group` values of k, in libmk's block layout
    (include/mk.h, mk_w4_quantize).  Made by quantize_w4."""
    codes: torch.Tensor    # uint8
    scales: torch.Tensor   # bf16
    n: int
    k: int
    group: int


@functools.lru_cache(maxsize=256)
def _w4_sizes(n: int, k: int, group: int):
    """Bytes of the codes and the scales."""
    codes, scales = ctypes.c_size_t(), ctypes.c_size_t()
    check(load().mk_w4_bytes(n, k, group, ctypes.byref(codes), ctypes.byref(scales)), "mk_w4_bytes")
    return codes.value, scales.value


def _need_w4(w):
    """The kernels take a W4Weight's sizes on trust: its buffers have to be as large as those say."""
    if not isinstance(w, W4Weight):
        raise MkError("expected a W4Weight (quantize_w4)")
    nc, ns = _w4_sizes(w.n, w.k, w.group)
    c, s = w.codes, w.scales
    if not c.is_cuda or s.device != c.device:
        raise MkError("W4Weight: codes and scales must be GPU tensors of one device")
    if c.dtype != torch.uint8 or s.dtype != BF16 or c.numel() != nc or s.numel() != ns // 2 or not (
            c.is_contiguous() and s.is_contiguous()):
        raise MkError(f"W4Weight: expected {nc} bytes of codes and {ns // 2} bf16 scales, contiguous")


def quantize_w4(weight: torch.Tensor, group: int = 128) -> W4Weight:
    """weight (N, K) bf16 -> 4-bit codes in [-7, 7] under a bf16 scale amax / 7 per row and `group` (32, 64 or 128)
    values of K.  Any N and K; rows may be strided.  A group with a NaN or an infinity gets a NaN scale."""
    lib = load()
    n, k, ld = _need_rows(weight, "weight", (BF16,))
    group = int(group)
    nc, ns = _w4_sizes(n, k, group)
    codes, scales = weight.new_empty(nc, dtype=torch.uint8), weight.new_empty(ns // 2)
    _call(weight, lib.mk_w4_quantize, "mk_w4_quantize", _adr(weight), ld, n, k, group, _adr(codes), _adr(scales))
    return W4Weight(codes, scales, n, k, group)


def dequantize_w4(w: W4Weight, dtype: torch.dtype = BF16) -> torch.Tensor:
    """The values a W4Weight stands for: (N, K) f32 (exact) or bf16 (rounded once)."""
    lib = load()
    if dtype not in (BF16, F32):
        raise MkError(f"dequantize_w4: dtype {dtype}, expected bf16 or f32")
    _need_w4(w)
    out = w.scales.new_empty((w.n, w.k), dtype=dtype)
    _call(out, lib.mk_w4_dequantize, "mk_w4_dequantize", _adr(w.codes), _adr(w.scales), w.n, w.k, w.group, _adr(out),
          int(dtype != BF16), w.k)
    return out


def gemm_w4(x: torch.Tensor, w: W4Weight, dtype: torch.dtype = BF16, out: torch.Tensor | None = None) -> torch.Tensor:
    """x (M, K) bf16 @ w (N, K)^T with 4-bit weights, f32 accumulation -> (M, N) bf16 or f32 (include/mk.h, mk_gemm_w4).

    For few rows: the weights are read once per 64 rows of x.  x and `out` may have strided rows; `out` must not overlap x
    or the weight.  A row's result is the same in every batch."""
    lib = load()
    _need_w4(w)
    M, _, ldx = _need_rows(x, "x", (BF16,), w.k)
    if out is None:
        if dtype not in (BF16, F32):
            raise MkError(f"gemm_w4: dtype {dtype}, expected bf16 or f32")
        _same_device(x, w=w.codes)
        out = x.new_empty((M, w.n), dtype=dtype)
        ldo = w.n
    else:
        rows, _, ldo = _need_rows(out, "out", (BF16, F32), w.n)
        if rows != M:
            raise MkError(f"out: {rows} rows, expected {M}")
        _same_device(x, w=w.codes, out=out)
    _call(x, lib.mk_gemm_w4, "mk_gemm_w4", _adr(x), ldx, _adr(w.codes), _adr(w.scales), M, w.n, w.k, w.group, _adr(out),
          int(out.dtype != BF16), ldo)
    return out


def pack_weight(w: torch.Tensor, map_gu: bool = False, ic: int = 0, inter: int = 0) -> torch.Tensor:
    """(K, N) -> (N, K) repack (the layout mk_model_create builds); map_gu reorders gate/up columns."""
    lib = load()
    K, N = w.shape
    _need(w, "w")
    out = torch.empty((N, K), dtype=w.dtype, device=w.device)
    check(lib.mk_pack_weight(_ptr(w), N, _ptr(out), K, N, w.element_size(), int(map_gu), ic, inter, _stream()),
          "mk_pack_weight")
    return out


__all__ = ["attn_prefill", "attn_scratch_bytes", "row_quant", "act_quant", "gemm", "lm_head", "logprobs", "LogProbs", "lm_head_logprobs",
           "W4Weight", "quantize_w4", "dequantize_w4", "gemm_w4", "pack_weight", "MkError", "_lib"]
