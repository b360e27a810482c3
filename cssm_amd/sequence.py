"""Operators over token sequences: (B, T, C) activations with long T, packed sequences and single tokens.

The gated cell's recurrence without its transforms, for each channel in real arithmetic

    D_t = softplus(delta_t + bias),  h_t = kappa exp(-D_t) h_{t-1} + D_t x_t,  y_t = h_t SiLU(z_t)

(:func:`token_scan`, one token at a time :func:`token_scan_step`), the root-mean-square norm behind a residual's
addition (:func:`rms_norm`) and the product of 8-bit operands that its 8-bit output feeds (:func:`scaled_matmul`); the
gated delta rule, whose state is a matrix for each head (:func:`delta_rule`, :func:`delta_rule_step`), and the norm and
rotation of the heads that feed it (:func:`rotate_heads`).  The differentiable forms are in :mod:`cssm_amd.training`.

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


def _heads(t, name: str, lead, width: int, dtype, dev: int, like: str) -> Tuple[_lib.TokenRows, int]:
    """cssm_token_rows and the number of heads of (..., H, width) whose heads lie side by side; ``lead`` its leading sizes.
    (B, T, H, width), or (T, H, width) packed rows / (B, H, width) tokens as ``like`` says."""
    if _gpu(t, name) != dev:
        raise ValueError(f"{name} is on {t.device}, expected GPU {dev}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != len(lead) + 2 or t.shape[:-2] != lead or (width and t.shape[-1] != width) or not t.shape[-2]:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(lead)} rows of heads" +
                         (f" of {width}" if width else ""))
    H, D = t.shape[-2:]
    st = t.stride()
    if t.numel() and ((D > 1 and st[-1] != 1) or (H > 1 and st[-2] != D)):
        raise ValueError(f"{name} must have its heads side by side (strides {st})")
    return _lead_rows(t, st, like), H


def _lead_rows(t, st, like: str) -> _lib.TokenRows:
    if like == "batch":
        return _lib.TokenRows(t.data_ptr(), st[0], st[1])
    return _lib.TokenRows(t.data_ptr(), 0, st[0]) if like == "packed" else _lib.TokenRows(t.data_ptr(), st[0], 0)


def _gate_rows(t, name: str, lead, H: int, dev: int, like: str) -> _lib.TokenRows:
    """cssm_token_rows of (..., H) float32, any strides but the heads'."""
    if _gpu(t, name) != dev:
        raise ValueError(f"{name} is on {t.device}, expected GPU {dev}")
    if t.dtype is not torch.float32:
        raise ValueError(f"{name} must be torch.float32, got {t.dtype}")
    if t.shape != (*lead, H):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {(*lead, H)}")
    st = t.stride()
    if t.numel() and H > 1 and st[-1] != 1:
        raise ValueError(f"{name} must have its heads side by side (strides {st})")
    return _lead_rows(t, st, like)


_Rows5, _Rows2 = ctypes.c_longlong * 15, ctypes.c_longlong * 6     # cssm_token_rows one behind the other
_ROWS = ctypes.sizeof(_lib.TokenRows)
_MOST = 0x7fffffff


def _fine(t, shape, dtype, dev: int) -> bool:
    """Whether :func:`_check` takes t: what a usual call asks, without naming what is wrong."""
    return isinstance(t, torch.Tensor) and t.get_device() == dev and t.dtype is dtype and t.shape == shape and t.is_contiguous()


def _new(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape, type and GPU."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


class _Delta(NamedTuple):
    """Checked arguments of the delta rule: GPU, rows (addresses in ``rows``), sizes."""
    dev: int
    rows: object
    q: int
    k: int
    v: int
    beta: int
    decay: Optional[int]
    dtype: int
    B: int
    T: int
    Hk: int
    Hv: int
    dk: int
    dv: int
    n: int          # sequences
    nseq: int       # with offsets, else 0


def _plain_delta(q, k, v, beta, decay, state, offsets, step: bool) -> Optional[_Delta]:
    """:func:`_delta` of contiguous tensors that go together: the usual call, without the checks that name what is wrong.
    None for any other."""
    try:
        dev, dt, f32, sv, sk, gate = v.get_device(), v.dtype, torch.float32, v.shape, k.shape, beta.shape
        if len(sv) == 4 and offsets is None and not step:
            B, T, Hv, dv = sv
            n, nseq = B, 0
            same = sk[0] == B and sk[1] == T and gate == (B, T, Hv)
        elif len(sv) == 3 and step:
            B, Hv, dv = sv
            T, n, nseq = 1, B, 0
            same = sk[0] == B and gate == (B, Hv)
        elif len(sv) == 3 and offsets is not None:
            T, Hv, dv = sv
            B, n = 1, offsets.numel() - 1
            nseq = n
            same = (sk[0] == T and gate == (T, Hv) and n >= 0 and offsets.dim() == 1 and offsets.dtype is torch.int32
                    and offsets.get_device() == dev and offsets.is_contiguous())
        else:
            return None
        Hk, dk = sk[-2], sk[-1]
        if not (same and dev >= 0 and dt in _DTYPES and k.dtype is dt and q.dtype is dt and beta.dtype is f32 and q.shape == sk
                and len(sk) == len(sv) and 0 < dk <= 128 and 0 < dv <= 128 and Hk > 0 and 0 < Hv <= _MOST and Hv % Hk == 0
                and B <= _MOST and T <= _MOST
                and q.get_device() == dev and k.get_device() == dev and beta.get_device() == dev
                and v.is_contiguous() and q.is_contiguous() and k.is_contiguous() and beta.is_contiguous()
                and (decay is None or (decay.dtype is f32 and decay.shape == gate and decay.get_device() == dev
                                       and decay.is_contiguous()))
                and ((state is None and not step) or _fine(state, (n, Hv, dk, dv), f32, dev))):
            return None
    except (AttributeError, ValueError, IndexError):
        return None
    rk, rv = Hk * dk, Hv * dv
    rows = _Rows5(q.data_ptr(), T * rk, rk, k.data_ptr(), T * rk, rk, v.data_ptr(), T * rv, rv, beta.data_ptr(), T * Hv, Hv,
                  0 if decay is None else decay.data_ptr(), T * Hv, Hv)
    at = ctypes.addressof(rows)
    return _Delta(dev, rows, at, at + _ROWS, at + 2 * _ROWS, at + 3 * _ROWS, None if decay is None else at + 4 * _ROWS,
                  _DTYPES[dt], B, T, Hk, Hv, dk, dv, n, nseq)


def _delta(q, k, v, beta, decay, state, offsets, step: bool = False) -> _Delta:
    d = _plain_delta(q, k, v, beta, decay, state, offsets, step)
    if d is not None:
        return d
    dev = _gpu(v, "v")
    if v.dtype not in _DTYPES:
        raise ValueError(f"v: unsupported dtype {v.dtype}")
    like = "step" if step else "batch" if offsets is None else "packed"
    if v.dim() != (4 if like == "batch" else 3):
        raise ValueError(f"v has shape {tuple(v.shape)}, expected " +
                         {"step": "(B, Hv, dv)", "batch": "(B, T, Hv, dv)", "packed": "(T, Hv, dv) rows with offsets"}[like])
    lead = v.shape[:-2]
    B, T = (lead[0], 1) if step else lead if offsets is None else (1, lead[0])
    _sizes("v", v.shape, *v.shape)
    rv, Hv = _heads(v, "v", lead, 0, v.dtype, dev, like)
    rk, Hk = _heads(k, "k", lead, 0, v.dtype, dev, like)
    dk, dv = k.shape[-1], v.shape[-1]
    rq, Hq = _heads(q, "q", lead, dk, v.dtype, dev, like)
    if Hq != Hk or Hv % Hk:
        raise ValueError(f"{Hq} query, {Hk} key and {Hv} value heads: as many queries as keys, and values a multiple of them")
    if not 0 < dk <= 128 or not 0 < dv <= 128:
        raise ValueError(f"heads of {dk} and {dv}: widths of 1 to 128 are taken")
    rb = _gate_rows(beta, "beta", lead, Hv, dev, like)
    rd = None if decay is None else _gate_rows(decay, "decay", lead, Hv, dev, like)
    n, nseq = B, 0
    if offsets is not None:
        _gpu(offsets, "offsets")
        if offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets must be a tensor of n + 1 row numbers")
        _check(offsets, "offsets", offsets.shape, torch.int32, dev)
        n = nseq = offsets.numel() - 1
    if state is not None or step:
        _check(state, "state", (n, Hv, dk, dv), torch.float32, dev)
    rows = rq, rk, rv, rb, rd
    return _Delta(dev, rows, *(_ref(r) for r in rows), _DTYPES[v.dtype], B, T, Hk, Hv, dk, dv, n, nseq)


def delta_forward(q, k, v, beta, decay=None, state=None, offsets=None, out=None, scale=None, keep=False):
    """:func:`delta_rule` with what its adjoint needs: (y, final state, errors, states), the last two None unless ``keep``."""
    d = _delta(q, k, v, beta, decay, state, offsets)
    packed = offsets is not None
    if out is None:
        y = _new(v)
    else:
        y = _check(out, "out", v.shape, v.dtype, d.dev)
    final = v.new_empty((d.n, d.Hv, d.dk, d.dv), dtype=torch.float32)
    lib = _lib.load()
    errors = states = None
    if keep:
        errors = v.new_empty(v.shape, dtype=torch.float32)
        states = v.new_empty((lib.cssm_delta_rule_segments(d.B, d.T, d.nseq, int(packed)), d.Hv, d.dk, d.dv), dtype=torch.float32)
    if d.n:
        need = lib.cssm_delta_rule_workspace_size(d.B, d.T, d.Hv, d.dk, d.dv, d.nseq, int(packed))
        work = v.new_empty(need, dtype=torch.uint8)
        _call(d.dev, "cssm_delta_rule", d.q, d.k, d.v, d.dtype, d.beta, d.decay, d.B, d.T, d.Hk, d.Hv, d.dk, d.dv,
              d.dk ** -0.5 if scale is None else float(scale), _ptr(state), _ptr(offsets), d.nseq, y.data_ptr(), int(packed and out is None), final.data_ptr(), _ptr(errors), _ptr(states), work.data_ptr(), need)
    elif packed and out is None:
        y.zero_()
    return y, final, errors, states


def delta_backward(q, k, beta, decay, offsets, errors, states, dy, dfinal, scale=None):
    """Adjoint of :func:`delta_rule` (cssm_delta_rule_bwd): (dq, dk, dv, dbeta, ddecay, dstate), ddecay None without decay."""
    d = _delta(q, k, dy, beta, decay, dfinal, offsets)
    packed = offsets is not None
    lib = _lib.load()
    _check(errors, "errors", dy.shape, torch.float32, d.dev)
    _check(states, "states", (lib.cssm_delta_rule_segments(d.B, d.T, d.nseq, int(packed)), d.Hv, d.dk, d.dv), torch.float32, d.dev)
    dq, dk, dv, db, dg = _new(q), _new(k), _new(dy), _new(beta), None if decay is None else _new(decay)
    dh0 = dy.new_empty((d.n, d.Hv, d.dk, d.dv), dtype=torch.float32)
    if d.n:
        need = lib.cssm_delta_rule_bwd_workspace_size(d.B, d.T, d.Hk, d.Hv, d.dk, d.dv, d.nseq, int(packed))
        work = dy.new_empty(need, dtype=torch.uint8)
        _call(d.dev, "cssm_delta_rule_bwd", d.q, d.k, d.dtype, d.beta, d.decay, d.v, d.B, d.T, d.Hk, d.Hv, d.dk, d.dv,
              d.dk ** -0.5 if scale is None else float(scale), _ptr(offsets), d.nseq, errors.data_ptr(), states.data_ptr(), _ptr(dfinal), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
              db.data_ptr(), _ptr(dg), dh0.data_ptr(), work.data_ptr(), need)
    else:
        for t in (dq, dk, dv, db) if dg is None else (dq, dk, dv, db, dg):
            t.zero_()
    return dq, dk, dv, db, dg, dh0


def delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, beta: torch.Tensor, decay: Optional[torch.Tensor] = None,
               state: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gated delta rule over whole sequences: (y, final state).  For each value head, S (dk, dv) its state:

        e_t = v_t - a_t S_{t-1}^T k_t,  S_t = a_t S_{t-1} + k_t (beta_t e_t)^T,  y_t = scale S_t^T q_t,  a = exp(decay)

    ``q``, ``k`` (B, T, Hk, dk) and ``v`` (B, T, Hv, dv), float32 or bfloat16 and alike, widths to 128, the heads side by
    side (slices of one projection's output will do); Hv / Hk value heads next to each other share a query and key head.
    ``beta``, ``decay`` (B, T, Hv) float32, decay <= 0 (None: 0, no decay; -inf clears the state).  The rule is stable for
    keys of at most unit length and 0 <= beta <= 2; nothing checks that.  A row with beta = 0 and decay = 0 leaves the state:
    that masks it, its values and the products of its key and query with others being finite (zeros, not the type's lowest
    value).  ``state`` (B, Hv, dk, dv) float32 before the first
    row (None: zeros); ``scale`` dk^-0.5 unless given.  ``offsets`` and ``out`` as in :func:`token_scan`: packed rows
    (T, H, width), states (n, Hv, dk, dv).  Rows are taken 32 at a time, and a value that is not finite spoils its sequence
    from the 32 rows on in which it stands.  Not differentiable: see :func:`cssm_amd.training.delta_rule_train`.
    """
    return delta_forward(q, k, v, beta, decay, state, offsets, out, scale)[:2]


def delta_rule_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, beta: torch.Tensor, state: torch.Tensor,
                    decay: Optional[torch.Tensor] = None, out_state: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token for each sequence: (y, state) from ``q``, ``k`` (B, Hk, dk), ``v`` (B, Hv, dv), ``beta``, ``decay`` (B, Hv)
    and ``state`` (B, Hv, dk, dv) float32, which ``out_state=state`` updates in place."""
    d = _delta(q, k, v, beta, decay, state, None, step=True)
    if out_state is None:
        out_state = torch.empty_like(state)
    elif out_state is not state:
        _check(out_state, "out_state", state.shape, torch.float32, d.dev)
    y = _new(v)
    if d.B:
        _call(d.dev, "cssm_delta_rule_step", d.q, d.k, d.v, d.dtype, d.beta, d.decay, d.B, d.Hk, d.Hv, d.dk, d.dv,
              d.dk ** -0.5 if scale is None else float(scale), state.data_ptr(), y.data_ptr(), out_state.data_ptr())
    return y, out_state


class RotaryTable(NamedTuple):
    """How the pairs of a head turn: ``frequencies`` (P,) float64 radians a position, ``axes`` (P,) int32, the axis of the
    positions that each turns with."""
    frequencies: torch.Tensor
    axes: torch.Tensor


def rotary_table(sections, base: float = 10000.0, device="cuda", shared: bool = False) -> RotaryTable:
    """The usual table: ``sections[i]`` pairs turn with axis i (time, height, width; one number: plain positions).  Each axis
    has a geometric row of frequencies base^(-j / n) of its own, j < n its pairs; with ``shared`` one row runs over all
    pairs.  Laid out once for a model."""
    sections = [int(n) for n in sections]
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or not sum(sections):
        raise ValueError(f"sections={sections}: 1 to 4 numbers of pairs")
    if not base > 0:
        raise ValueError(f"base={base} must be positive")
    total = sum(sections)
    freq = [base ** (-j / n) for n in sections for j in range(n)] if not shared else [base ** (-j / total) for j in range(total)]
    return RotaryTable(torch.tensor(freq, dtype=torch.float64, device=device),
                       torch.tensor([i for i, n in enumerate(sections) for _ in range(n)], dtype=torch.int32, device=device))


_HEAD_NORMS = {"rms": 0, "l2": 1, "none": 2}
_PAIRS = {"neighbours": 0, "halves": 1}


class _Rotary(NamedTuple):
    """Checked arguments of the head rotation."""
    dev: int
    rows: object     # what q and k are the addresses in
    q: int
    k: Optional[int]
    head: tuple      # dtype, B, T, Hq, Hk, D
    rest: tuple      # weights, norm, eps, positions, axes, frequencies, axis, P, halves


def _rotary(q, k, positions, table, q_weight, k_weight, norm, eps, pairs) -> _Rotary:
    dev = _gpu(q, "q")
    if q.dtype not in _DTYPES:
        raise ValueError(f"q: unsupported dtype {q.dtype}")
    if q.dim() not in (3, 4):
        raise ValueError(f"q has shape {tuple(q.shape)}, expected (B, T, H, D) or (M, H, D)")
    if norm not in _HEAD_NORMS:
        raise ValueError(f"norm={norm!r}: one of {sorted(_HEAD_NORMS)}")
    if pairs not in _PAIRS:
        raise ValueError(f"pairs={pairs!r}: one of {sorted(_PAIRS)}")
    lead, (Hq, D) = q.shape[:-2], q.shape[-2:]
    B, T = lead if len(lead) == 2 else (1, lead[0])
    if D % 2 or not 0 < D <= 512:
        raise ValueError(f"heads of {D}: even widths to 512 are taken")
    sk = None if k is None else k.shape
    if (Hq and q.is_contiguous() and (k is None or (k.get_device() == dev and k.dtype is q.dtype and len(sk) == len(lead) + 2 and
                                                    sk[:-2] == lead and sk[-2] and sk[-1] == D and k.is_contiguous()))):
        Hk = 0 if k is None else sk[-2]     # contiguous, as usual
        rows = _Rows2(q.data_ptr(), T * Hq * D, Hq * D, 0 if k is None else k.data_ptr(), T * Hk * D, Hk * D)
        rq, rk = ctypes.addressof(rows), None if k is None else ctypes.addressof(rows) + _ROWS
    else:
        like = "batch" if len(lead) == 2 else "packed"
        tq, Hq = _heads(q, "q", lead, D, q.dtype, dev, like)
        tk, Hk = (None, 0) if k is None else _heads(k, "k", lead, D, q.dtype, dev, like)
        rows, rq, rk = (tq, tk), _ref(tq), _ref(tk)
    _sizes("q", q.shape, B, T, Hq, Hk)
    if q_weight is not None and not _fine(q_weight, (D,), torch.float32, dev):
        _check(q_weight, "q_weight", (D,), torch.float32, dev)
    if k_weight is not None and not _fine(k_weight, (D,), torch.float32, dev):
        _check(k_weight, "k_weight", (D,), torch.float32, dev)
    if (positions is None) != (table is None):
        raise ValueError("positions and table go together")
    axes = P = 0
    freq = axis = None
    if table is not None:
        freq, axis = table
        _gpu(freq, "table.frequencies")
        P = freq.numel()
        if not _fine(freq, (P,), torch.float64, dev) or not _fine(axis, (P,), torch.int32, dev):
            _check(freq, "table.frequencies", (P,), torch.float64, dev)
            _check(axis, "table.axes", (P,), torch.int32, dev)
        if 2 * P > D:
            raise ValueError(f"{P} pairs in heads of {D}")
        axes = positions.shape[-1] if isinstance(positions, torch.Tensor) and positions.dim() else 0
        if not _fine(positions, (*lead, axes), torch.int32, dev):
            _check(positions, "positions", (*lead, axes), torch.int32, dev)
        if not 1 <= axes <= 4:
            raise ValueError(f"positions have {axes} axes: 1 to 4 are taken")
    rest = (_ptr(q_weight), _ptr(k_weight), _HEAD_NORMS[norm], float(eps), _ptr(positions), axes, _ptr(freq), _ptr(axis), P,
            _PAIRS[pairs])
    return _Rotary(dev, rows, rq, rk, (_DTYPES[q.dtype], B, T, Hq, Hk, D), rest)


def rotate_heads(q: torch.Tensor, k: Optional[torch.Tensor], positions: Optional[torch.Tensor] = None, table=None,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, norm: str = "rms",
                 eps: float = 1e-6, pairs: str = "halves"):
    """(q', k'): each head's norm and the rotation by its row's positions, in one pass.

    ``q`` (B, T, Hq, D) and ``k`` (B, T, Hk, D) or None, or rows (M, H, D); float32 or bfloat16 and alike, D even and to
    512, the heads side by side (slices of one projection's output will do).  ``norm`` 'rms' (x / sqrt(mean(x^2) + eps)),
    'l2' (x / sqrt(sum(x^2) + eps), unit lengths as :func:`delta_rule` takes its keys) or 'none', then times ``q_weight`` /
    ``k_weight`` (D) float32.  ``positions`` (B, T, A) or (M, A) int32, 1 to 4 axes, negative ones too; ``table`` a
    :class:`RotaryTable` (:func:`rotary_table`) of P <= D / 2 pairs; both None: no rotation.  ``pairs`` 'halves': (j, j + P);
    'neighbours': (2 j, 2 j + 1); values from 2 P on are not turned.  Not differentiable: see
    :func:`cssm_amd.training.rotate_heads_train`.
    """
    r = _rotary(q, k, positions, table, q_weight, k_weight, norm, eps, pairs)
    q_out, k_out = _new(q), None if k is None else _new(k)
    if q.numel():
        _call(r.dev, "cssm_rotate_heads", r.q, r.k, *r.head, *r.rest, q_out.data_ptr(), _ptr(k_out))
    return q_out, k_out


def rotate_heads_backward(q, k, dq_out, dk_out, positions, table, q_weight, k_weight, norm, eps, pairs):
    """Adjoint of :func:`rotate_heads` (cssm_rotate_heads_bwd): (dq, dk, dq_weight, dk_weight), None where there is none."""
    r = _rotary(q, k, positions, table, q_weight, k_weight, norm, eps, pairs)
    if _fine(dq_out, q.shape, q.dtype, r.dev) and (k is None or _fine(dk_out, k.shape, q.dtype, r.dev)):
        _, _, T, Hq, Hk, D = r.head     # contiguous, as usual
        rows = _Rows2(dq_out.data_ptr(), T * Hq * D, Hq * D, 0 if k is None else dk_out.data_ptr(), T * Hk * D, Hk * D)
        gq, gk = ctypes.addressof(rows), None if k is None else ctypes.addressof(rows) + _ROWS
    else:
        like = "batch" if q.dim() == 4 else "packed"
        tq, _ = _heads(dq_out, "dq_out", q.shape[:-2], q.shape[-1], q.dtype, r.dev, like)
        tk = None if k is None else _heads(dk_out, "dk_out", q.shape[:-2], q.shape[-1], q.dtype, r.dev, like)[0]
        if dq_out.shape != q.shape or (k is not None and dk_out.shape != k.shape):
            raise ValueError("the outputs' gradients have the outputs' shapes")
        gq, gk = _ref(tq), _ref(tk)
    dq, dk = _new(q), None if k is None else _new(k)
    dwq, dwk = (None if w is None else torch.empty_like(w) for w in (q_weight, k_weight))
    if q.numel():
        work, need = None, 0
        if dwq is not None or dwk is not None:
            need = _lib.load().cssm_rotate_heads_bwd_workspace_size(q.shape[-1])
            work = q.new_empty(need // 4, dtype=torch.float32)
        _call(r.dev, "cssm_rotate_heads_bwd", r.q, r.k, gq, gk, *r.head, *r.rest, dq.data_ptr(),
              _ptr(dk), _ptr(dwq), _ptr(dwk), _ptr(work), need)
    else:
        for t in (dwq, dwk):
            if t is not None:
                t.zero_()
    return dq, dk, dwq, dwk
