"""Operator interface of the attention hot path on torch CUDA tensors.

The four functions mirror the reference's four kernels (attention.metal:19-299)
with the same buffer roles, order and dtypes, as its host code binds them
(model.h:446-473 forward, model.h:639-665 backward).  Each call goes through the
C ABI of libmetalattn (include/metalattn.h); PyTorch only provides the device
memory and the stream.  Outputs may be passed in (as the reference's
preallocated buffers) or are allocated here, for a call with stream= in that
stream's order.  The inputs of such a call have to be ready on that stream and
kept (or recorded for it, Tensor.record_stream) until its work is done.

Shapes (B sequences of length T = params.M, N = params.N = NH*D):
    X, q, k, v, out, dO, dK, dV : bf16 [B, T, N]
    dQ                          : fp32 [B, T, N]
    l                           : fp32 [B, T, NH]
    D                           : bf16 [B, T, NH]

For long contexts (no counterpart in the reference): rotary positions
(rotaryForward, rotaryBackward), attention with a sliding window and sinks
(windowAttentionForward, windowAttentionBackward) and, for serving, the same
two over a K/V cache (rotaryCacheAppend, windowAttentionCached).  They take
grouped heads (k, v and their gradients [B, T, NKV*D], caches
[B, cap, NKV*D]; query head h uses K/V head h // (NH // NKV)) and padded
batches (lens, int32 [B]: rows from lens[b] on are padding).
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

import torch

from . import _lib
from ._lib import AttentionParams, MetalAttnError  # noqa: F401  (re-exported)


def make_params(T: int, NH: int, D: int) -> AttentionParams:
    """AttentionParams{M=T, N=NH*D, D, NH} as model.h:178 fills it."""
    return AttentionParams(T, NH * D, D, NH)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# The current stream's handle.  torch.cuda.current_stream() builds a Stream
# object first, 3 us of the 10 to 20 us that a small call takes on the host.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream: Optional[torch.cuda.Stream]) -> int:
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple) -> None:
    if type(t) is torch.Tensor and t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.is_cuda and \
            t.get_device() == torch.cuda.current_device():
        return  # as it should be; else find out what is not
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (no CPU path exists)")
    cur = torch.cuda.current_device()
    if t.device.index != cur:
        # the entry points launch on the current device; another device's
        # pointer would be dereferenced from there
        raise ValueError(f"{name} is on {t.device} but the current CUDA device is cuda:{cur}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape) and t.numel() != _numel(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _numel(shape: tuple) -> int:
    n = 1
    for s in shape:
        n *= s
    return n


def _out(t: Optional[torch.Tensor], like: torch.Tensor, shape: tuple, dtype: torch.dtype,
         name: str, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """The output given, checked, or a new one for a call on `stream`."""
    if t is None:
        if stream is not None and stream.cuda_stream != _stream(None):
            # Allocated in that stream's order: memory that work queued on the current
            # stream may still use is not handed out.  Recorded for the current stream,
            # where the caller will read it: dropped, it waits for that work.
            with torch.cuda.stream(stream):
                t = torch.empty(shape, dtype=dtype, device=like.device)
            t.record_stream(torch.cuda.current_stream())
            return t
        if like.dtype is dtype and like.shape == shape and like.is_contiguous():
            return torch.empty_like(like)  # half the host time of torch.empty
        return torch.empty(shape, dtype=dtype, device=like.device)
    _check(t, name, dtype, shape)
    return t


def computeQKV(X: torch.Tensor, q_w: torch.Tensor, k_w: torch.Tensor, v_w: torch.Tensor,
               p: AttentionParams, B: int, q: Optional[torch.Tensor] = None,
               k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None,
               stream: Optional[torch.cuda.Stream] = None):
    """q, k, v = X Wq, X Wk, X Wv (attention.metal:19-53)."""
    act = (B, p.M, p.N)
    _check(X, "X", torch.bfloat16, act)
    for w, n in ((q_w, "q_w"), (k_w, "k_w"), (v_w, "v_w")):
        _check(w, n, torch.bfloat16, (p.N, p.N))
    q = _out(q, X, act, torch.bfloat16, "q", stream)
    k = _out(k, X, act, torch.bfloat16, "k", stream)
    v = _out(v, X, act, torch.bfloat16, "v", stream)
    _lib.call("ma_computeQKV", _ptr(X), _ptr(q), _ptr(k), _ptr(v), _ptr(q_w), _ptr(k_w),
              _ptr(v_w), ctypes.byref(p), B, _stream(stream))
    return q, k, v


def projForward(attn_out: torch.Tensor, proj_w: torch.Tensor, p: AttentionParams, B: int,
                out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
    """out = attn_out . proj_w (attention.metal:395-416)."""
    act = (B, p.M, p.N)
    _check(attn_out, "attn_out", torch.bfloat16, act)
    _check(proj_w, "proj_w", torch.bfloat16, (p.N, p.N))
    out = _out(out, attn_out, act, torch.bfloat16, "out", stream)
    _lib.call("ma_projForward", _ptr(attn_out), _ptr(proj_w), _ptr(out), ctypes.byref(p), B,
              _stream(stream))
    return out


def projBackwarddW(attn_out: torch.Tensor, dZ: torch.Tensor, p: AttentionParams, B: int,
                   dProjw: Optional[torch.Tensor] = None,
                   stream: Optional[torch.cuda.Stream] = None):
    """dProjw = attn_out^T . dZ over all B*M rows (attention.metal:418-430)."""
    act = (B, p.M, p.N)
    _check(attn_out, "attn_out", torch.bfloat16, act)
    _check(dZ, "dZ", torch.bfloat16, act)
    dProjw = _out(dProjw, attn_out, (p.N, p.N), torch.bfloat16, "dProjw", stream)
    _lib.call("ma_projBackwarddW", _ptr(attn_out), _ptr(dZ), _ptr(dProjw), ctypes.byref(p), B,
              _stream(stream))
    return dProjw


def projBackwarddX(dZ: torch.Tensor, proj_w: torch.Tensor, p: AttentionParams, B: int,
                   dAttn: Optional[torch.Tensor] = None,
                   stream: Optional[torch.cuda.Stream] = None):
    """dAttn = dZ . proj_w^T (attention.metal:432-455)."""
    act = (B, p.M, p.N)
    _check(dZ, "dZ", torch.bfloat16, act)
    _check(proj_w, "proj_w", torch.bfloat16, (p.N, p.N))
    dAttn = _out(dAttn, dZ, act, torch.bfloat16, "dAttn", stream)
    _lib.call("ma_projBackwarddX", _ptr(dZ), _ptr(proj_w), _ptr(dAttn), ctypes.byref(p), B,
              _stream(stream))
    return dAttn


def projBackwarddXComputeD(dZ: torch.Tensor, proj_w: torch.Tensor, attn_out: torch.Tensor,
                           p: AttentionParams, B: int, dAttn: Optional[torch.Tensor] = None,
                           D: Optional[torch.Tensor] = None,
                           stream: Optional[torch.cuda.Stream] = None):
    """dAttn = dZ . proj_w^T and D = computeD(dAttn, attn_out) in one launch
    (the D sums formed in the GEMM epilogue)."""
    act = (B, p.M, p.N)
    _check(dZ, "dZ", torch.bfloat16, act)
    _check(proj_w, "proj_w", torch.bfloat16, (p.N, p.N))
    _check(attn_out, "attn_out", torch.bfloat16, act)
    dAttn = _out(dAttn, dZ, act, torch.bfloat16, "dAttn", stream)
    D = _out(D, dZ, (B, p.M, p.NH), torch.bfloat16, "D", stream)
    _lib.call("ma_projBackwarddXComputeD", _ptr(dZ), _ptr(proj_w), _ptr(dAttn), _ptr(attn_out), _ptr(D),
              ctypes.byref(p), B, _stream(stream))
    return dAttn, D


def computeGradDx(q_w: torch.Tensor, k_w: torch.Tensor, v_w: torch.Tensor, dQ: torch.Tensor,
                  dK: torch.Tensor, dV: torch.Tensor, p: AttentionParams, B: int,
                  dX: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
    """dX = dQ.Wq^T + dK.Wk^T + dV.Wv^T in fp32 (attention.metal:301-342)."""
    act = (B, p.M, p.N)
    for w, n in ((q_w, "q_w"), (k_w, "k_w"), (v_w, "v_w")):
        _check(w, n, torch.bfloat16, (p.N, p.N))
    _check(dQ, "dQ", torch.float32, act)
    _check(dK, "dK", torch.bfloat16, act)
    _check(dV, "dV", torch.bfloat16, act)
    dX = _out(dX, dK, act, torch.float32, "dX", stream)
    _lib.call("ma_computeGradDx", _ptr(dX), _ptr(q_w), _ptr(k_w), _ptr(v_w), _ptr(dQ), _ptr(dK),
              _ptr(dV), ctypes.byref(p), B, _stream(stream))
    return dX


def computeGradDw(x: torch.Tensor, dQ: torch.Tensor, dK: torch.Tensor, dV: torch.Tensor,
                  p: AttentionParams, B: int, dQw: Optional[torch.Tensor] = None,
                  dKw: Optional[torch.Tensor] = None, dVw: Optional[torch.Tensor] = None,
                  stream: Optional[torch.cuda.Stream] = None):
    """dQw = X^T.dQ (fp32), dKw = X^T.dK, dVw = X^T.dV (bf16) over all B*M rows
    (attention.metal:344-393)."""
    act = (B, p.M, p.N)
    _check(x, "x", torch.bfloat16, act)
    _check(dQ, "dQ", torch.float32, act)
    _check(dK, "dK", torch.bfloat16, act)
    _check(dV, "dV", torch.bfloat16, act)
    w = (p.N, p.N)
    dQw = _out(dQw, x, w, torch.float32, "dQw", stream)
    dKw = _out(dKw, x, w, torch.bfloat16, "dKw", stream)
    dVw = _out(dVw, x, w, torch.bfloat16, "dVw", stream)
    _lib.call("ma_computeGradDw", _ptr(x), _ptr(dQ), _ptr(dK), _ptr(dV), _ptr(dQw), _ptr(dKw),
              _ptr(dVw), ctypes.byref(p), B, _stream(stream))
    return dQw, dKw, dVw


def flashAttentionForward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, p: AttentionParams,
                          B: int, out: Optional[torch.Tensor] = None,
                          l: Optional[torch.Tensor] = None, shard: Optional[tuple] = None,
                          stream: Optional[torch.cuda.Stream] = None):
    """out, l = causal attention of (q, k, v) (attention.metal:56-164).

    ``shard=(bh_begin, bh_end)`` restricts the work to flat (batch, head) indices
    in that range (ma_flashAttentionForward_shard)."""
    act = (B, p.M, p.N)
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _check(t, n, torch.bfloat16, act)
    out = _out(out, q, act, torch.bfloat16, "out", stream)
    l = _out(l, q, (B, p.M, p.NH), torch.float32, "l", stream)
    if shard is None:
        _lib.call("ma_flashAttentionForward", _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(l),
                  ctypes.byref(p), B, _stream(stream))
    else:
        _lib.call("ma_flashAttentionForward_shard", _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(l),
                  ctypes.byref(p), B, shard[0], shard[1], _stream(stream))
    return out, l


def flashAttentionForwardComputeD(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, dO: torch.Tensor,
                                  p: AttentionParams, B: int, out: Optional[torch.Tensor] = None,
                                  l: Optional[torch.Tensor] = None, D: Optional[torch.Tensor] = None,
                                  shard: Optional[tuple] = None, stream: Optional[torch.cuda.Stream] = None,
                                  zero_dQ: Optional[torch.Tensor] = None):
    """out, l, D = flashAttentionForward then computeD(dO, out), for callers
    that know dO before the forward (ma_flashAttentionForwardComputeD; at
    head size 64 D is formed in the forward's epilogue).  With zero_dQ (fp32
    [B, T, N]) the forward also writes zeros to it for every (row, head) it
    computes (ma_flashAttentionForwardComputeDZeroDQ), for a following
    flashAttentionBackward(..., accumulate_dQ=True)."""
    act = (B, p.M, p.N)
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (dO, "dO")):
        _check(t, n, torch.bfloat16, act)
    out = _out(out, q, act, torch.bfloat16, "out", stream)
    l = _out(l, q, (B, p.M, p.NH), torch.float32, "l", stream)
    D = _out(D, q, (B, p.M, p.NH), torch.bfloat16, "D", stream)
    if zero_dQ is not None:
        _check(zero_dQ, "zero_dQ", torch.float32, act)
        name = "ma_flashAttentionForwardComputeDZeroDQ"
        args = (_ptr(q), _ptr(k), _ptr(v), _ptr(dO), _ptr(out), _ptr(l), _ptr(D), _ptr(zero_dQ),
                ctypes.byref(p), B)
        if shard is None:
            _lib.call(name, *args, _stream(stream))
        else:
            _lib.call(name + "_shard", *args, shard[0], shard[1], _stream(stream))
    elif shard is None:
        _lib.call("ma_flashAttentionForwardComputeD", _ptr(q), _ptr(k), _ptr(v), _ptr(dO), _ptr(out), _ptr(l),
                  _ptr(D), ctypes.byref(p), B, _stream(stream))
    else:
        _lib.call("ma_flashAttentionForwardComputeD_shard", _ptr(q), _ptr(k), _ptr(v), _ptr(dO), _ptr(out),
                  _ptr(l), _ptr(D), ctypes.byref(p), B, shard[0], shard[1], _stream(stream))
    return out, l, D


def computeD(dO: torch.Tensor, O: torch.Tensor, p: AttentionParams, B: int,
             D: Optional[torch.Tensor] = None, shard: Optional[tuple] = None,
             stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """D = rowsum(dO * O) per head, bf16 (attention.metal:166-195)."""
    act = (B, p.M, p.N)
    _check(dO, "dO", torch.bfloat16, act)
    _check(O, "O", torch.bfloat16, act)
    D = _out(D, dO, (B, p.M, p.NH), torch.bfloat16, "D", stream)
    if shard is None:
        _lib.call("ma_computeD", _ptr(dO), _ptr(O), _ptr(D), ctypes.byref(p), B, _stream(stream))
    else:
        _lib.call("ma_computeD_shard", _ptr(dO), _ptr(O), _ptr(D), ctypes.byref(p), B, shard[0],
                  shard[1], _stream(stream))
    return D


def flashAttentionBackward(dZ: torch.Tensor, d: torch.Tensor, l: torch.Tensor, q: torch.Tensor,
                           k: torch.Tensor, v: torch.Tensor, p: AttentionParams, B: int,
                           dQ: Optional[torch.Tensor] = None, dK: Optional[torch.Tensor] = None,
                           dV: Optional[torch.Tensor] = None, shard: Optional[tuple] = None,
                           stream: Optional[torch.cuda.Stream] = None, accumulate_dQ: bool = False):
    """dQ (fp32), dK, dV (bf16) of causal attention (attention.metal:198-299).
    With accumulate_dQ, dQ (given) is added to, as the reference's kernel
    adds into a dQ its host zeroed (ma_flashAttentionBackwardAccumulate);
    otherwise dQ is written."""
    act = (B, p.M, p.N)
    for t, n in ((dZ, "dZ"), (q, "q"), (k, "k"), (v, "v")):
        _check(t, n, torch.bfloat16, act)
    _check(d, "d", torch.bfloat16, (B, p.M, p.NH))
    _check(l, "l", torch.float32, (B, p.M, p.NH))
    if accumulate_dQ and dQ is None:
        raise ValueError("accumulate_dQ needs the dQ tensor to add into")
    dQ = _out(dQ, q, act, torch.float32, "dQ", stream)
    dK = _out(dK, q, act, torch.bfloat16, "dK", stream)
    dV = _out(dV, q, act, torch.bfloat16, "dV", stream)
    args = (_ptr(dZ), _ptr(d), _ptr(l), _ptr(q), _ptr(k), _ptr(v), _ptr(dQ), _ptr(dK), _ptr(dV),
            ctypes.byref(p), B)
    name = "ma_flashAttentionBackwardAccumulate" if accumulate_dQ else "ma_flashAttentionBackward"
    if shard is None:
        _lib.call(name, *args, _stream(stream))
    else:
        _lib.call(name + "_shard", *args, shard[0], shard[1], _stream(stream))
    return dQ, dK, dV


# ------------------------------------------------------------ long contexts
def rotaryFrequencies(rot: int, base: float = 10000.0, factor: float = 1.0, original_length: Optional[int] = None,
                      low: float = 1.0, high: float = 32.0, device="cuda") -> torch.Tensor:
    """Radians per position of a rotation's rot/2 pairs, float64 [rot/2]:
    base^(-2i/rot).  factor > 1 stretches the context: every frequency divided
    by it, or, given original_length, by parts: pairs that make at least
    `high` turns within original_length keep their frequency, pairs with at
    most `low` turns are divided by factor, and those between move linearly
    from one to the other.  (A stretch by parts usually goes with an
    amplitude of 0.1 ln(factor) + 1.)"""
    if rot < 2 or rot % 2:
        raise ValueError(f"rot must be even and at least 2, got {rot}")
    if not base > 0 or not factor > 0 or not high > low:
        raise ValueError("base and factor must be positive and high above low")
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rot)
    if original_length is None:
        return (f / factor).to(device)
    keep = ((original_length * f / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
    return (f * (keep + (1.0 - keep) / factor)).to(device)


def _groups(p: AttentionParams, NKV: Optional[int]) -> int:
    NKV = p.NH if NKV is None else int(NKV)
    if NKV < 1 or p.NH % NKV:
        raise ValueError(f"NKV={NKV} must divide NH={p.NH}")
    return NKV


def _check_all(*specs) -> None:
    """_check for each (tensor, name, dtype, shape)."""
    cur = torch.cuda.current_device() if torch.cuda.is_initialized() else -1
    for t, name, dtype, shape in specs:
        if not (type(t) is torch.Tensor and t.dtype is dtype and t.shape == shape and t.is_contiguous()
                and t.get_device() == cur and t.is_cuda):
            _check(t, name, dtype, shape)


def _check_optional(t: Optional[torch.Tensor], name: str, dtype: torch.dtype, shape: tuple) -> None:
    if t is not None:
        _check(t, name, dtype, shape)


def _rotary(inv_freq: torch.Tensor, NKV: int, interleaved: bool, amplitude: float) -> _lib.Rotary:
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1:
        raise TypeError("inv_freq must be a one-dimensional tensor (rotaryFrequencies)")
    _check(inv_freq, "inv_freq", torch.float64, inv_freq.shape)
    return _lib.Rotary(inv_freq.data_ptr(), 2 * inv_freq.shape[0], bool(interleaved), NKV, amplitude)


def _u32(x: int, name: str) -> int:
    if x < 0:
        raise ValueError(f"{name} must not be negative, got {x}")
    return min(int(x), 0xFFFFFFFF)


def _window(window: int, sinks: int, NKV: int) -> _lib.Window:
    return _lib.Window(NKV, _u32(window, "window"), _u32(sinks, "sinks"))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(M: int, D: int, NH: int, NKV: int, window: int, sinks: int, B: int,
                     cap: Optional[int]) -> int:
    """Bytes of workspace of a backward (cap None) or of a call over a cache."""
    need = ctypes.c_uint64()
    w, p = ctypes.byref(_lib.Window(NKV, window, sinks)), ctypes.byref(make_params(M, NH, D))
    if cap is None:
        _lib.call("ma_windowAttentionBackward_workspace", w, p, B, ctypes.byref(need))
    else:
        _lib.call("ma_windowAttentionCached_workspace", w, p, B, cap, ctypes.byref(need))
    return need.value


def _workspace(like: torch.Tensor, stream: Optional[torch.cuda.Stream], p: AttentionParams, w: _lib.Window, B: int,
               cap: Optional[int] = None) -> Optional[torch.Tensor]:
    """Device memory for a call on `stream`, or None where it needs none."""
    need = _workspace_bytes(p.M, p.D, p.NH, w.NKV, w.window, w.sinks, B, cap)
    if need == 0:
        return None
    if stream is None:
        return torch.empty(need, dtype=torch.uint8, device=like.device)
    with torch.cuda.stream(stream):  # the allocator then reuses it in that stream's order
        return torch.empty(need, dtype=torch.uint8, device=like.device)


def rotaryForward(q: torch.Tensor, k: torch.Tensor, inv_freq: torch.Tensor, p: AttentionParams, B: int,
                  NKV: Optional[int] = None, positions: Optional[torch.Tensor] = None, interleaved: bool = False,
                  amplitude: float = 1.0, q_out: Optional[torch.Tensor] = None,
                  k_out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
    """q_out, k_out = q, k (bf16) with the first 2*len(inv_freq) columns of
    every head turned by positions * inv_freq (float64, rotaryFrequencies) and
    multiplied by amplitude.  Pairs are columns i and i + rot/2, or with
    interleaved 2i and 2i + 1.  positions: int32 [B, T], by default 0 .. T-1.
    q_out may be q and k_out may be k (ma_rotaryForward)."""
    NKV = _groups(p, NKV)
    r = _rotary(inv_freq, NKV, interleaved, amplitude)
    qs, ks = (B, p.M, p.N), (B, p.M, NKV * p.D)
    _check_all((q, "q", torch.bfloat16, qs), (k, "k", torch.bfloat16, ks))
    _check_optional(positions, "positions", torch.int32, (B, p.M))
    q_out = _out(q_out, q, qs, torch.bfloat16, "q_out", stream)
    k_out = _out(k_out, k, ks, torch.bfloat16, "k_out", stream)
    _lib.call("ma_rotaryForward", _ptr(q), _ptr(k), _ptr(q_out), _ptr(k_out), ctypes.byref(r), _ptr(positions),
              ctypes.byref(p), B, _stream(stream))
    return q_out, k_out


def rotaryBackward(dQ: torch.Tensor, dK: torch.Tensor, inv_freq: torch.Tensor, p: AttentionParams, B: int,
                   NKV: Optional[int] = None, positions: Optional[torch.Tensor] = None, interleaved: bool = False,
                   amplitude: float = 1.0, dQ_out: Optional[torch.Tensor] = None,
                   dK_out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
    """The gradients of rotaryForward's inputs from those of its outputs: dQ
    (fp32 or bf16, and dQ_out of the same type) and dK (bf16) turned back.
    In place allowed (ma_rotaryBackward)."""
    NKV = _groups(p, NKV)
    r = _rotary(inv_freq, NKV, interleaved, amplitude)
    qs, ks = (B, p.M, p.N), (B, p.M, NKV * p.D)
    t = torch.float32 if isinstance(dQ, torch.Tensor) and dQ.dtype == torch.float32 else torch.bfloat16
    _check_all((dQ, "dQ", t, qs), (dK, "dK", torch.bfloat16, ks))
    _check_optional(positions, "positions", torch.int32, (B, p.M))
    dQ_out = _out(dQ_out, dQ, qs, t, "dQ_out", stream)
    dK_out = _out(dK_out, dK, ks, torch.bfloat16, "dK_out", stream)
    _lib.call("ma_rotaryBackward", _ptr(dQ), _ptr(dK), _ptr(dQ_out), _ptr(dK_out), int(t == torch.float32),
              ctypes.byref(r), _ptr(positions), ctypes.byref(p), B, _stream(stream))
    return dQ_out, dK_out


def _cap(cache: torch.Tensor, name: str) -> int:
    if not isinstance(cache, torch.Tensor) or cache.dim() != 3:
        raise TypeError(f"{name} must be a [B, cap, NKV*D] tensor")
    return cache.shape[1]


def rotaryCacheAppend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, start: torch.Tensor, inv_freq: torch.Tensor, p: AttentionParams, B: int,
                      NKV: Optional[int] = None, lens: Optional[torch.Tensor] = None, interleaved: bool = False,
                      amplitude: float = 1.0, q_out: Optional[torch.Tensor] = None,
                      stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """p.M new tokens of each sequence enter the caches (bf16 [B, cap, NKV*D]):
    k turned at its position start[b] + i (start: int32 [B]) and v are stored
    in that row.  Returns q turned (rows from lens[b] on: 0); q_out may be q.
    Padding rows, and rows past the caches' end, are not stored
    (ma_rotaryCacheAppend)."""
    NKV = _groups(p, NKV)
    r = _rotary(inv_freq, NKV, interleaved, amplitude)
    qs, ks, cap = (B, p.M, p.N), (B, p.M, NKV * p.D), _cap(k_cache, "k_cache")
    cs = (B, cap, NKV * p.D)
    _check_all((q, "q", torch.bfloat16, qs), (k, "k", torch.bfloat16, ks), (v, "v", torch.bfloat16, ks),
               (k_cache, "k_cache", torch.bfloat16, cs), (v_cache, "v_cache", torch.bfloat16, cs),
               (start, "start", torch.int32, (B,)))
    _check_optional(lens, "lens", torch.int32, (B,))
    q_out = _out(q_out, q, qs, torch.bfloat16, "q_out", stream)
    _lib.call("ma_rotaryCacheAppend", _ptr(q), _ptr(k), _ptr(v), _ptr(q_out), _ptr(k_cache), _ptr(v_cache),
              _ptr(start), _ptr(lens), ctypes.byref(r), ctypes.byref(p), B, cap, _stream(stream))
    return q_out


def windowAttentionForward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, p: AttentionParams, B: int,
                           window: int, sinks: int = 0, NKV: Optional[int] = None,
                           lens: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                           l: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
    """out, l as flashAttentionForward, where the query at i sees key j <= i
    only if i - j < window or j < sinks.  Padding rows: out = 0, l = -inf
    (ma_windowAttentionForward)."""
    NKV = _groups(p, NKV)
    w = _window(window, sinks, NKV)
    qs, ks = (B, p.M, p.N), (B, p.M, NKV * p.D)
    _check_all((q, "q", torch.bfloat16, qs), (k, "k", torch.bfloat16, ks), (v, "v", torch.bfloat16, ks))
    _check_optional(lens, "lens", torch.int32, (B,))
    out = _out(out, q, qs, torch.bfloat16, "out", stream)
    l = _out(l, q, (B, p.M, p.NH), torch.float32, "l", stream)
    _lib.call("ma_windowAttentionForward", _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(l), _ptr(lens),
              ctypes.byref(w), ctypes.byref(p), B, _stream(stream))
    return out, l


def windowAttentionBackward(dO: torch.Tensor, out: torch.Tensor, l: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                            v: torch.Tensor, p: AttentionParams, B: int, window: int, sinks: int = 0,
                            NKV: Optional[int] = None, lens: Optional[torch.Tensor] = None,
                            dQ: Optional[torch.Tensor] = None, dK: Optional[torch.Tensor] = None,
                            dV: Optional[torch.Tensor] = None, dQ_dtype: Optional[torch.dtype] = None,
                            stream: Optional[torch.cuda.Stream] = None):
    """dQ, dK, dV of windowAttentionForward from dO and its out and l (padding
    rows: 0).  dQ is fp32 as flashAttentionBackward's (for computeGradDx and
    computeGradDw), or bf16: by the dQ given, or by dQ_dtype
    (ma_windowAttentionBackward)."""
    NKV = _groups(p, NKV)
    w = _window(window, sinks, NKV)
    qs, ks = (B, p.M, p.N), (B, p.M, NKV * p.D)
    _check_all((dO, "dO", torch.bfloat16, qs), (out, "out", torch.bfloat16, qs), (q, "q", torch.bfloat16, qs),
               (l, "l", torch.float32, (B, p.M, p.NH)), (k, "k", torch.bfloat16, ks), (v, "v", torch.bfloat16, ks))
    _check_optional(lens, "lens", torch.int32, (B,))
    if dQ_dtype is None:
        dQ_dtype = dQ.dtype if isinstance(dQ, torch.Tensor) else torch.float32
    if dQ_dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"dQ must be float32 or bfloat16, got {dQ_dtype}")
    f32 = int(dQ_dtype == torch.float32)
    dQ = _out(dQ, q, qs, dQ_dtype, "dQ", stream)
    dK = _out(dK, k, ks, torch.bfloat16, "dK", stream)
    dV = _out(dV, k, ks, torch.bfloat16, "dV", stream)
    ws = _workspace(q, stream, p, w, B)
    _lib.call("ma_windowAttentionBackward", _ptr(dO), _ptr(out), _ptr(l), _ptr(q), _ptr(k), _ptr(v), _ptr(dQ),
              _ptr(dK), _ptr(dV), f32, _ptr(lens), ctypes.byref(w), ctypes.byref(p), B, _ptr(ws), ws.numel(),
              _stream(stream))
    return dQ, dK, dV


def windowAttentionCached(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, start: torch.Tensor,
                          p: AttentionParams, B: int, window: int, sinks: int = 0, NKV: Optional[int] = None,
                          lens: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                          l: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
    """out, l of p.M >= 1 new queries of each sequence, at positions
    start[b] + i, over caches that already hold their keys and values
    (rotaryCacheAppend); window and sinks as in windowAttentionForward, rows
    from lens[b] on are padding.  start[b] + lens[b] must not exceed the
    caches' rows (ma_windowAttentionCached)."""
    NKV = _groups(p, NKV)
    w = _window(window, sinks, NKV)
    qs, cap = (B, p.M, p.N), _cap(k_cache, "k_cache")
    cs = (B, cap, NKV * p.D)
    _check_all((q, "q", torch.bfloat16, qs), (k_cache, "k_cache", torch.bfloat16, cs),
               (v_cache, "v_cache", torch.bfloat16, cs), (start, "start", torch.int32, (B,)))
    _check_optional(lens, "lens", torch.int32, (B,))
    out = _out(out, q, qs, torch.bfloat16, "out", stream)
    l = _out(l, q, (B, p.M, p.NH), torch.float32, "l", stream)
    ws = _workspace(q, stream, p, w, B, cap=cap)
    _lib.call("ma_windowAttentionCached", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), _ptr(l), _ptr(start),
              _ptr(lens), ctypes.byref(w), ctypes.byref(p), B, cap, _ptr(ws), 0 if ws is None else ws.numel(),
              _stream(stream))
    return out, l


def device_status(stream: Optional[torch.cuda.Stream] = None) -> int:
    """Reads and clears the device's kernel status (0 = no bounded wait ran
    out; else a mask of the _lib.STATUS_* bits), for every entry point
    including flashAttentionBackward_noalloc."""
    st = ctypes.c_uint32(0)
    _lib.call("ma_device_status", ctypes.byref(st), _stream(stream))
    return st.value


def debug_expire_next_wait(kernels: int, wait_ns: int = 1_000_000) -> None:
    """Test hook of the time-out path: the next launch of each kernel in
    `kernels` (_lib.STATUS_FWD_TIMEOUT / _lib.STATUS_BWD_TIMEOUT) lets a wait
    run out after `wait_ns` and winds down as after a real time-out (its bit
    then shows in device_status).  kernels=0 cancels a pending request."""
    _lib.call("ma_debug_expire_next_wait", int(kernels), int(wait_ns))


class CudaAttention:
    """Attention core of one transformer block with reference-style buffers.

    Mirrors the attention part of the reference's MetalAttention harness
    (main.cpp:955-1284) and Model::forward/backward (model.h:446-473,
    639-665): buffers are allocated once for (B, T, NH, D) and reused, forward
    runs flashAttentionForward, backward runs computeD then
    flashAttentionBackward.  The projections around attention are not part of
    this path."""

    def __init__(self, B: int, T: int, NH: int, D: int, device="cuda"):
        self.B, self.T, self.NH, self.D = B, T, NH, D
        self.p = make_params(T, NH, D)
        act = (B, T, NH * D)
        dev = torch.device(device)
        self.out = torch.empty(act, dtype=torch.bfloat16, device=dev)
        self.l = torch.empty((B, T, NH), dtype=torch.float32, device=dev)
        self.Dvec = torch.empty((B, T, NH), dtype=torch.bfloat16, device=dev)
        self.dQ = torch.empty(act, dtype=torch.float32, device=dev)
        self.dK = torch.empty(act, dtype=torch.bfloat16, device=dev)
        self.dV = torch.empty(act, dtype=torch.bfloat16, device=dev)

    def forward(self, q, k, v, stream=None):
        self.q, self.k, self.v = q, k, v
        return flashAttentionForward(q, k, v, self.p, self.B, out=self.out, l=self.l,
                                     stream=stream)

    def backward(self, dO, stream=None):
        computeD(dO, self.out, self.p, self.B, D=self.Dvec, stream=stream)
        return flashAttentionBackward(dO, self.Dvec, self.l, self.q, self.k, self.v, self.p,
                                      self.B, dQ=self.dQ, dK=self.dK, dV=self.dV, stream=stream)


def _check_host(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.is_cuda:
        raise ValueError(f"{name} must be a host (CPU) tensor; use the device entry points for CUDA tensors")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.numel() != _numel(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


class HostPipeline:
    """Attention over host-resident batches (ma_host_pipeline_*): the batch is
    split into chunks of `chunk_B` sequences whose host->device copies,
    kernels and device->host copies overlap on three internal streams.  The
    reference needs no such step (its Metal buffers are shared CPU/GPU memory,
    model.h:236-253); O, l, dK and dV equal the device entry points bit for
    bit, and dQ to fp32 rounding (its reduce-adds arrive in no fixed order).
    Host tensors should be pinned (`tensor.pin_memory()`) for the overlap."""

    def __init__(self, T: int, NH: int, D: int, chunk_B: int, device=None):
        self.p = make_params(T, NH, D)
        self.T, self.NH, self.D, self.chunk_B = T, NH, D, chunk_B
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        h = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            _lib.call("ma_host_pipeline_create", ctypes.byref(self.p), chunk_B, ctypes.byref(h))
        self._h = h

    def close(self) -> None:
        if getattr(self, "_h", None) is not None and self._h.value:
            _lib.call("ma_host_pipeline_destroy", self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _shapes(self, B: int):
        act = (B, self.T, self.NH * self.D)
        return act, (B, self.T, self.NH)

    def forward(self, q, k, v, B: int, out=None, l=None, stream=None):
        """flashAttentionForward of B host sequences -> (out bf16, l fp32), host."""
        act, rows = self._shapes(B)
        for t, n in ((q, "q"), (k, "k"), (v, "v")):
            _check_host(t, n, torch.bfloat16, act)
        out = torch.empty(act, dtype=torch.bfloat16).pin_memory() if out is None else out
        l = torch.empty(rows, dtype=torch.float32).pin_memory() if l is None else l
        _check_host(out, "out", torch.bfloat16, act)
        _check_host(l, "l", torch.float32, rows)
        with torch.cuda.device(self.device):
            _lib.call("ma_flashAttentionForward_host", self._h, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                      out.data_ptr(), l.data_ptr(), B, _stream(stream))
        return out, l

    def forward_backward(self, q, k, v, dO, B: int, out=None, l=None, dQ=None, dK=None, dV=None,
                         stream=None):
        """forward + computeD + backward of B host sequences ->
        (out, l, dQ, dK, dV), host tensors, ready when `stream` is."""
        act, rows = self._shapes(B)
        for t, n in ((q, "q"), (k, "k"), (v, "v"), (dO, "dO")):
            _check_host(t, n, torch.bfloat16, act)
        mk = lambda t, shape, dt: torch.empty(shape, dtype=dt).pin_memory() if t is None else t
        out, l = mk(out, act, torch.bfloat16), mk(l, rows, torch.float32)
        dQ, dK, dV = mk(dQ, act, torch.float32), mk(dK, act, torch.bfloat16), mk(dV, act, torch.bfloat16)
        for t, n, dt, shp in ((out, "out", torch.bfloat16, act), (l, "l", torch.float32, rows),
                              (dQ, "dQ", torch.float32, act), (dK, "dK", torch.bfloat16, act),
                              (dV, "dV", torch.bfloat16, act)):
            _check_host(t, n, dt, shp)
        with torch.cuda.device(self.device):
            _lib.call("ma_attentionForwardBackward_host", self._h, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                      dO.data_ptr(), out.data_ptr(), l.data_ptr(), dQ.data_ptr(), dK.data_ptr(),
                      dV.data_ptr(), B, _stream(stream))
        return out, l, dQ, dK, dV
