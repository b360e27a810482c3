"""Operators over token sequences: (B, T, C) activations with long T, packed sequences and single tokens.

The gated cell's recurrence without its transforms, for each channel in real arithmetic

    D_t = softplus(delta_t + bias),  h_t = kappa exp(-D_t) h_{t-1} + D_t x_t,  y_t = h_t SiLU(z_t)

(:func:`token_scan`, one token at a time :func:`token_scan_step`), the root-mean-square norm behind a residual's
addition (:func:`rms_norm`) and the product of 8-bit operands that its 8-bit output feeds (:func:`scaled_matmul`).
The differentiable forms are in :mod:`cssm_amd.training`.

Tensors live on one GPU; the work is enqueued on torch's current stream of that GPU.  Nothing synchronises, and
nothing falls back: what a kernel does not take raises ValueError or :class:`cssm_amd._lib.CssmError`.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .spectral import _DTYPES, OUTPUT_ACTS, _raw_stream

SEGMENT = 128     # rows between the states a training pass keeps (CSSM_TOKEN_SEGMENT)
KEPT_ROWS, KEPT_CHANNELS = 8, 16     # values of a checkpoint under one exponent


class Blocks8(NamedTuple):
    """A matrix in 8 bits: ``values`` (float8_e4m3fn) times the power of two of their block in ``scales``
    (float8_e8m0fnu).  A block is 128 values of a row (:func:`quantize_rows`, :func:`rms_norm`) or 128 x 128 values
    (:func:`quantize_weight`)."""
    values: torch.Tensor
    scales: torch.Tensor


def _call(dev: int, name: str, *args) -> None:
    """The entry point on the current stream of GPU ``dev``, whatever the current device is."""
    if dev == torch.cuda.current_device():
        _lib.call(name, *args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, _stream(dev))


def _stream(dev: int) -> int:
    return _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


def _gpu(t, name: str) -> int:
    """The GPU's number of a tensor on one."""
    dev = t.get_device() if isinstance(t, torch.Tensor) else -1
    if dev < 0:
        raise ValueError(f"{name} must be a GPU tensor")
    return dev


def _check(t, name: str, shape, dtype, dev: int) -> torch.Tensor:
    """t, contiguous, of this shape and type on this GPU."""
    if _gpu(t, name) != dev:
        raise ValueError(f"{name} is on {t.device}, expected GPU {dev}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _sizes(name: str, shape, *sizes: int) -> None:
    """Refuses sizes that the C entry points' 32-bit arguments would cut."""
    if max(sizes) > 0x7fffffff:
        raise ValueError(f"{name} has shape {tuple(shape)}: a size is over 2^31 - 1")


def _rows(t, name: str, like: torch.Tensor, dev: int, packed: bool) -> _lib.TokenRows:
    """cssm_token_rows of (B, T, C), or (T, C) packed rows / (B, C) tokens: any strides but the channels'."""
    if t is not like:
        if _gpu(t, name) != dev or t.dtype is not like.dtype or t.shape != like.shape:
            raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}, expected {tuple(like.shape)} "
                             f"{like.dtype} on {like.device}")
    elif t.dtype not in _DTYPES:
        raise ValueError(f"{name}: unsupported dtype {t.dtype}")
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have its channels side by side (strides {st})")
    if len(st) == 3:
        return _lib.TokenRows(t.data_ptr(), st[0], st[1])
    return _lib.TokenRows(t.data_ptr(), 0, st[0]) if packed else _lib.TokenRows(t.data_ptr(), st[0], 0)


def _ref(rows):
    return None if rows is None else ctypes.addressof(rows)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _sequences(x, kappa, bias, state, offsets):
    """(GPU, B, T, C, sequences, number of offsets) of checked arguments."""
    dev = _gpu(x, "x")
    if x.dim() != (3 if offsets is None else 2):
        raise ValueError(f"x has shape {tuple(x.shape)}, expected " +
                         ("(B, T, C)" if offsets is None else "(T, C) rows with offsets"))
    C = x.shape[-1]
    _check(kappa, "kappa", (C,), torch.float32, dev)
    _check(bias, "bias", (C,), torch.float32, dev)
    if offsets is None:
        B, T, n, nseq = x.shape[0], x.shape[1], x.shape[0], 0
    else:
        _gpu(offsets, "offsets")
        if offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets must be a tensor of n + 1 row numbers")
        _check(offsets, "offsets", offsets.shape, torch.int32, dev)
        B, T, n, nseq = 1, x.shape[0], offsets.numel() - 1, offsets.numel() - 1
    _sizes("x", x.shape, B, T, C, n)
    if state is not None:
        _check(state, "state", (n, C), torch.float32, dev)
    return dev, B, T, C, n, nseq


def _kept_buffers(planes: int, B: int, T: int, C: int, device):
    return (torch.empty((planes, B, T, C), dtype=torch.uint8, device=device),
            torch.empty((planes, B, -(-T // KEPT_ROWS), -(-C // KEPT_CHANNELS)), dtype=torch.uint8, device=device))


def scan_forward(x, delta, kappa, bias, z=None, state=None, offsets=None, out=None, keep_states=False, keep_e4m3=False):
    """:func:`token_scan` with what its adjoint needs: (y, final state, states, kept, kept scales); ``states`` (B,
    segments, C) where asked for, the last two the 8-bit checkpoint where ``keep_e4m3``, else None."""
    dev, B, T, C, n, nseq = _sequences(x, kappa, bias, state, offsets)
    packed = offsets is not None
    rx, rd = _rows(x, "x", x, dev, packed), _rows(delta, "delta", x, dev, packed)
    rz = None if z is None else _rows(z, "z", x, dev, packed)
    if out is None:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        y = _check(out, "out", x.shape, x.dtype, dev)
    final = torch.empty((n, C), dtype=torch.float32, device=x.device)
    lib = _lib.load()
    states = kept = scales = work = None
    if keep_states or keep_e4m3:
        states = torch.empty((B, lib.cssm_token_scan_chunks(T), C), dtype=torch.float32, device=x.device)
    if keep_e4m3:
        kept, scales = _kept_buffers(2 if z is None else 3, B, T, C, x.device)
    need = lib.cssm_token_scan_workspace_size(B, T, C, 0)
    if need:
        work = torch.empty(need // 8, dtype=torch.int64, device=x.device)
    if B and C:
        _call(dev, "cssm_token_scan", _ref(rx), _ref(rd), _ref(rz), _DTYPES[x.dtype], B, T, C, kappa.data_ptr(),
              bias.data_ptr(), _ptr(state), _ptr(offsets), nseq, y.data_ptr(), int(packed and out is None),
              final.data_ptr(), _ptr(states), _ptr(kept), _ptr(scales), _ptr(work), need)
    return y, final, states, kept, scales


def scan_backward(x, delta, kappa, bias, z, state, offsets, states, kept, scales, dy, dfinal, gated: bool):
    """Adjoint of :func:`token_scan` (cssm_token_scan_bwd): (dx, ddelta, dz, dkappa, dbias, dstate); from the 8-bit
    checkpoint where ``kept`` is given (x, delta and z are then None), dz None without a gate."""
    packed = offsets is not None
    dev, B, T, C, n, nseq = _sequences(dy, kappa, bias, state, offsets)
    rdy = _rows(dy, "dy", dy, dev, packed)
    rows = [None if t is None else _rows(t, name, dy, dev, packed) for t, name in ((x, "x"), (delta, "delta"), (z, "z"))]
    if dfinal is not None:
        _check(dfinal, "dfinal", (n, C), torch.float32, dev)
    chunks = _lib.load().cssm_token_scan_chunks(T)
    _check(states, "states", (B, chunks, C), torch.float32, dev)
    if kept is not None:
        planes = 3 if gated else 2
        _check(kept, "kept", (planes, B, T, C), torch.uint8, dev)
        _check(scales, "scales", (planes, B, -(-T // KEPT_ROWS), -(-C // KEPT_CHANNELS)), torch.uint8, dev)
    elif x is None or delta is None or gated != (z is not None):
        raise ValueError("the adjoint needs x, delta and, with a gate, z, or the kept checkpoint")

    def like():
        return torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
    dx, dd, dz = like(), like(), like() if gated else None
    dk, db = torch.empty_like(kappa), torch.empty_like(bias)
    dh0 = torch.empty((n, C), dtype=torch.float32, device=dy.device)
    need = _lib.load().cssm_token_scan_workspace_size(B, T, C, 1)
    work = torch.empty(max(1, need // 8), dtype=torch.int64, device=dy.device)
    if B and C:
        _call(dev, "cssm_token_scan_bwd", _ref(rows[0]), _ref(rows[1]), _ref(rows[2]), int(gated), _ref(rdy),
              _DTYPES[dy.dtype], B, T, C, kappa.data_ptr(), bias.data_ptr(), _ptr(state), _ptr(offsets), nseq,
              states.data_ptr(), _ptr(kept), _ptr(scales), _ptr(dfinal), dx.data_ptr(), dd.data_ptr(), _ptr(dz),
              dk.data_ptr(), db.data_ptr(), dh0.data_ptr(), work.data_ptr(), need)
    else:
        dk.zero_(), db.zero_()
    return dx, dd, dz, dk, db, dh0


def token_scan(x: torch.Tensor, delta: torch.Tensor, kappa: torch.Tensor, bias: torch.Tensor,
               z: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
               offsets: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gated recurrence over whole sequences: (y, final state).

    ``x``, ``delta``, ``z`` (B, T, C), float32 or bfloat16 and alike, the channels side by side (slices of one
    projection's output will do); ``kappa``, ``bias`` (C) float32; ``state`` (B, C) float32 before the first row
    (None: zeros).  Without ``z`` y is the state itself.  With ``offsets`` (n + 1 int32 row numbers on the GPU, from 0,
    ascending) the rows (T, C) hold n sequences one behind the other, ``state`` and the final state are (n, C), and an
    empty sequence keeps its state.  Rows behind the last sequence are zero, or as they were in ``out``.  A row with
    delta = -inf and finite x only scales the state by kappa.  Not differentiable: see
    :func:`cssm_amd.training.token_scan_train`.
    """
    return scan_forward(x, delta, kappa, bias, z, state, offsets, out)[:2]


def token_scan_step(x: torch.Tensor, delta: torch.Tensor, kappa: torch.Tensor, bias: torch.Tensor, state: torch.Tensor,
                    z: Optional[torch.Tensor] = None, out_state: Optional[torch.Tensor] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token for each sequence: (y, state) from ``x``, ``delta``, ``z`` (B, C) and ``state`` (B, C) float32, which
    ``out_state=state`` updates in place; the same values as :func:`token_scan` of one row."""
    dev = _gpu(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x has shape {tuple(x.shape)}, expected (B, C)")
    B, C = x.shape
    _sizes("x", x.shape, B, C)
    _check(kappa, "kappa", (C,), torch.float32, dev)
    _check(bias, "bias", (C,), torch.float32, dev)
    _check(state, "state", (B, C), torch.float32, dev)
    rx, rd = _rows(x, "x", x, dev, False), _rows(delta, "delta", x, dev, False)
    rz = None if z is None else _rows(z, "z", x, dev, False)
    if out_state is None:
        out_state = torch.empty_like(state)
    elif out_state is not state:
        _check(out_state, "out_state", (B, C), torch.float32, dev)
    y = torch.empty((B, C), dtype=x.dtype, device=x.device)
    if B and C:
        _call(dev, "cssm_token_scan_step", _ref(rx), _ref(rd), _ref(rz), _DTYPES[x.dtype], B, C, kappa.data_ptr(),
              bias.data_ptr(), state.data_ptr(), y.data_ptr(), out_state.data_ptr())
    return y, out_state


def _norm_args(x, weight, residual):
    dev = _gpu(x, "x")
    if x.dtype not in _DTYPES or x.dim() < 1:
        raise ValueError(f"x is {tuple(x.shape)} {x.dtype}, expected rows in float32 or bfloat16")
    _check(x, "x", x.shape, x.dtype, dev)
    C = x.shape[-1]
    _sizes("x", x.shape, C)
    _check(weight, "weight", (C,), torch.float32, dev)
    if residual is not None:
        _check(residual, "residual", x.shape, x.dtype, dev)
    return dev, (x.numel() // C if C else 0), C


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
             out: str = "same"):
    """(y, s): s = x + residual rounded to x's type (x itself without a residual), y = s / rms(s) * weight over the last
    axis, rms(s) = sqrt(mean(s^2) + eps).  ``out`` 'same': y of x's shape and type; 'e4m3': y a :class:`Blocks8` of x's
    shape, an exponent for each 128 of a row.  Not differentiable: see :func:`cssm_amd.training.rms_norm_train`."""
    dev, M, C = _norm_args(x, weight, residual)
    if out not in ("same", "e4m3"):
        raise ValueError(f"out={out!r}: 'same' or 'e4m3'")
    s = x if residual is None else torch.empty_like(x)
    scales = None
    if out == "e4m3":
        y = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty((*x.shape[:-1], -(-C // 128)), dtype=torch.float8_e8m0fnu, device=x.device)
    else:
        y = torch.empty_like(x)
    if M:
        _call(dev, "cssm_rms_norm", x.data_ptr(), _ptr(residual), _DTYPES[x.dtype], M, C, weight.data_ptr(),
              float(eps), None if residual is None else s.data_ptr(), y.data_ptr(), _ptr(scales))
    return (y if scales is None else Blocks8(y, scales)), s


def rms_norm_backward(dy, ds, s, weight, eps: float):
    """(dx, dweight) of :func:`rms_norm` (cssm_rms_norm_bwd): dx is x's and the residual's gradient, ``s`` what the
    forward returned, ``ds`` its gradient or None."""
    dev, M, C = _norm_args(s, weight, None)
    _check(dy, "dy", s.shape, s.dtype, dev)
    if ds is not None:
        _check(ds, "ds", s.shape, s.dtype, dev)
    dx, dw = torch.empty_like(s), torch.empty_like(weight)
    if not M:
        return dx, dw.zero_()
    need = _lib.load().cssm_rms_norm_bwd_workspace_size(M, C)
    work = torch.empty(need // 4, dtype=torch.float32, device=s.device)
    _call(dev, "cssm_rms_norm_bwd", dy.data_ptr(), _ptr(ds), s.data_ptr(), _DTYPES[s.dtype], M, C,
          weight.data_ptr(), float(eps), dx.data_ptr(), dw.data_ptr(), work.data_ptr(), need)
    return dx, dw


def quantize_rows(x: torch.Tensor) -> Blocks8:
    """x (..., K) float32 or bfloat16 in 8 bits, an exponent for each 128 of a row (cssm_quantize_rows)."""
    dev = _gpu(x, "x")
    if x.dim() < 1 or x.dtype not in _DTYPES:
        raise ValueError(f"x is {tuple(x.shape)} {x.dtype}, expected rows in float32 or bfloat16")
    _check(x, "x", x.shape, x.dtype, dev)
    K = x.shape[-1]
    _sizes("x", x.shape, K)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty((*x.shape[:-1], -(-K // 128)), dtype=torch.float8_e8m0fnu, device=x.device)
    if x.numel():
        _call(dev, "cssm_quantize_rows", x.data_ptr(), _DTYPES[x.dtype], x.numel() // K, K, q.data_ptr(),
              s.data_ptr())
    return Blocks8(q, s)


def quantize_weight(kernel: torch.Tensor) -> Blocks8:
    """A Dense kernel (K, N) float32 as :func:`scaled_matmul` reads it: (N, K) in 8 bits, an exponent for each 128 x 128
    (cssm_quantize_weight).  Laid out once for a weight that stays."""
    dev = _gpu(kernel, "kernel")
    if kernel.dim() != 2:
        raise ValueError(f"kernel has shape {tuple(kernel.shape)}, expected (K, N)")
    K, N = kernel.shape
    _sizes("kernel", kernel.shape, K, N)
    _check(kernel, "kernel", (K, N), torch.float32, dev)
    q = torch.empty((N, K), dtype=torch.float8_e4m3fn, device=kernel.device)
    s = torch.empty((-(-N // 128), -(-K // 128)), dtype=torch.float8_e8m0fnu, device=kernel.device)
    _call(dev, "cssm_quantize_weight", kernel.data_ptr(), K, N, q.data_ptr(), s.data_ptr())
    return Blocks8(q, s)


def scaled_matmul(a: Blocks8, w: Blocks8, bias: Optional[torch.Tensor] = None, act: str = "none",
                  out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """act(a W^T + bias) (..., N) of 8-bit rows ``a`` (..., K) and an 8-bit weight ``w`` (N, K), summed in float32;
    ``act`` 'none', 'gelu' (tanh form) or 'silu', ``out_dtype`` float32 or bfloat16.  K a multiple of 16.  With a bfloat16
    output the 8-bit matrix instruction drops what lies about 13 bits below the largest of the few products that it adds
    at once, before they join the float32 sum; with float32 every product counts in full."""
    av, sa = a
    wv, sw = w
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    dev = _gpu(av, "a.values")
    _gpu(wv, "w.values")
    if av.dim() < 1 or wv.dim() != 2:
        raise ValueError("a must be (..., K) rows and w a (N, K) weight in 8 bits")
    K, N = av.shape[-1], wv.shape[0]
    M = av.shape[:-1].numel()
    _sizes("a", av.shape, M, K)
    _sizes("w", wv.shape, N)
    _check(av, "a.values", av.shape, f8, dev)
    _check(sa, "a.scales", (*av.shape[:-1], -(-K // 128)), e8, dev)
    _check(wv, "w.values", (N, K), f8, dev)
    _check(sw, "w.scales", (-(-N // 128), -(-K // 128)), e8, dev)
    if bias is not None:
        _check(bias, "bias", (N,), torch.float32, dev)
    if act not in OUTPUT_ACTS:
        raise ValueError(f"act={act!r}: one of {sorted(OUTPUT_ACTS)}")
    if out_dtype not in _DTYPES:
        raise ValueError(f"unsupported out_dtype {out_dtype}")
    out = torch.empty((*av.shape[:-1], N), dtype=out_dtype, device=av.device)
    if out.numel():
        _call(dev, "cssm_scaled_matmul", av.data_ptr(), sa.data_ptr(), wv.data_ptr(), sw.data_ptr(),
              M, N, K, _ptr(bias), OUTPUT_ACTS[act], out.data_ptr(), _DTYPES[out_dtype])
    return out
