"""Refusals of the token-sequence entry points: arguments are checked before any GPU work, so no GPU is needed."""
import ctypes

import pytest

from cssm_amd import _lib

BUF = ctypes.create_string_buffer(4096)
P = (ctypes.addressof(BUF) + 255) // 256 * 256
ROWS = _lib.TokenRows(P, 64, 8)
R = ctypes.addressof(ROWS)
EMPTY = _lib.TokenRows(None, 64, 8)
BIG = 1 << 30


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def fails(fn, args, status, **change):
    a = dict(args, **change)
    st = fn(*a.values())
    assert st == status, (change, st, _lib.load().cssm_last_error())
    assert _lib.load().cssm_last_error()


def test_scan(lib):
    args = dict(x=R, delta=R, z=R, dtype=0, B=2, T=200, C=8, kappa=P, bias=P, h0=None, offsets=None, nseq=0, y=P,
                zero_tail=0, h_out=P, states=P, kept=None, kept_scales=None, work=P, bytes=BIG, stream=None)
    fn = lib.cssm_token_scan
    for name in ("x", "delta", "kappa", "bias", "y"):
        fails(fn, args, -1, **{name: None})
    fails(fn, args, -1, kept=P, kept_scales=P, states=None)
    fails(fn, args, -1, x=ctypes.addressof(EMPTY))
    fails(fn, args, -1, z=ctypes.addressof(EMPTY))
    fails(fn, args, -1, kept=P)
    fails(fn, args, -1, kept_scales=P)
    fails(fn, args, -4, dtype=2)
    for name in ("B", "T", "C"):
        fails(fn, args, -2, **{name: -1})
    fails(fn, args, -2, offsets=P, nseq=3)            # packed rows are one batch
    fails(fn, args, -2, B=1, offsets=P, nseq=-1)
    fails(fn, args, -4, work=None)
    fails(fn, args, -4, bytes=lib.cssm_token_scan_workspace_size(2, 200, 8, 0) - 1)
    fails(fn, args, -5, work=P + 4)
    fails(fn, args, -3, B=1 << 20, T=1 << 20, C=1 << 10)
    # nothing to do is no error
    assert fn(*dict(args, B=0).values()) == 0 and fn(*dict(args, C=0).values()) == 0


def test_scan_bwd(lib):
    args = dict(x=R, delta=R, z=R, gated=1, dy=R, dtype=1, B=2, T=200, C=8, kappa=P, bias=P, h0=None, offsets=None,
                nseq=0, states=P, kept=None, kept_scales=None, dh=None, dx=P, dd=P, dz=P, dk=P, db=P, dh0=None, work=P,
                bytes=BIG, stream=None)
    fn = lib.cssm_token_scan_bwd
    for name in ("x", "delta", "z", "dy", "kappa", "bias", "states", "dx", "dd", "dz", "dk", "db"):
        fails(fn, args, -1, **{name: None})
    fails(fn, args, -1, kept=P)
    fails(fn, args, -4, dtype=-1)
    fails(fn, args, -2, B=0)
    fails(fn, args, -4, bytes=lib.cssm_token_scan_workspace_size(2, 200, 8, 1) - 1)
    fails(fn, args, -5, work=P + 4)


def test_step(lib):
    args = dict(x=R, delta=R, z=None, dtype=1, B=2, C=8, kappa=P, bias=P, state=P, y=P, out=P, stream=None)
    fn = lib.cssm_token_scan_step
    for name in ("x", "delta", "kappa", "bias", "state", "y", "out"):
        fails(fn, args, -1, **{name: None})
    fails(fn, args, -4, dtype=7)
    fails(fn, args, -2, B=-1)
    assert fn(*dict(args, B=0).values()) == 0


def test_workspace_and_chunks(lib):
    assert [lib.cssm_token_scan_chunks(t) for t in (0, 1, 128, 129, 1000)] == [1, 1, 1, 2, 8]
    assert lib.cssm_token_scan_workspace_size(1, 128, 64, 0) == 0
    for b, t, c in ((0, 5, 5), (5, 5, 0), (-1, 5, 5), (1, -1, 5)):
        assert lib.cssm_token_scan_workspace_size(b, t, c, 1) == 0
    # sizes past 32 bits
    assert lib.cssm_token_scan_workspace_size(64, 1 << 20, 1 << 13, 0) >= 64 * (1 << 13) * (1 << 13) * 8


def test_rms_norm(lib):
    args = dict(x=P, res=P, dtype=1, M=3, C=8, w=P, eps=1e-6, s=P, y=P, scales=None, stream=None)
    fn = lib.cssm_rms_norm
    for name in ("x", "w", "y", "res", "s"):
        fails(fn, args, -1, **{name: None})
    fails(fn, args, -4, dtype=2)
    fails(fn, args, -4, eps=-1.0)
    fails(fn, args, -4, eps=float("nan"))
    fails(fn, args, -2, M=-1)
    fails(fn, args, -2, M=1 << 31)
    fails(fn, args, -5, x=P + 1)
    assert fn(*dict(args, M=0).values()) == 0
    back = dict(dy=P, ds=None, s=P, dtype=0, M=3, C=8, w=P, eps=1e-6, dx=P, dw=P, work=P, bytes=BIG, stream=None)
    fn = lib.cssm_rms_norm_bwd
    for name in ("dy", "s", "w", "dx", "dw"):
        fails(fn, back, -1, **{name: None})
    fails(fn, back, -2, M=0)
    fails(fn, back, -4, work=None)
    fails(fn, back, -4, bytes=lib.cssm_rms_norm_bwd_workspace_size(3, 8) - 1)
    fails(fn, back, -4, eps=-0.5)


def test_quantize_and_product(lib):
    q = dict(x=P, dtype=0, M=3, K=8, q=P, s=P, stream=None)
    for name in ("x", "q", "s"):
        fails(lib.cssm_quantize_rows, q, -1, **{name: None})
    fails(lib.cssm_quantize_rows, q, -4, dtype=3)
    fails(lib.cssm_quantize_rows, q, -2, M=-3)
    w = dict(k=P, K=8, N=8, q=P, s=P, stream=None)
    for name in ("k", "q", "s"):
        fails(lib.cssm_quantize_weight, w, -1, **{name: None})
    fails(lib.cssm_quantize_weight, w, -2, N=0)
    args = dict(a=P, sa=P, w=P, sw=P, M=4, N=8, K=32, bias=None, act=0, out=P, dtype=1, stream=None)
    fn = lib.cssm_scaled_matmul
    for name in ("a", "sa", "w", "sw", "out"):
        fails(fn, args, -1, **{name: None})
    fails(fn, args, -3, K=24)
    fails(fn, args, -2, K=0)
    fails(fn, args, -2, N=-8)
    fails(fn, args, -4, act=3)
    fails(fn, args, -4, dtype=2)
    fails(fn, args, -5, a=P + 8)
    fails(fn, args, -5, w=P + 8)
    fails(fn, args, -5, out=P + 1)
    assert fn(*dict(args, M=0).values()) == 0


def test_too_large_for_one_launch(lib):
    """sizes whose launch would pass 2^32 threads, or 32-bit byte offsets"""
    scan = dict(x=R, delta=R, z=R, dtype=0, B=1 << 24, T=1, C=1, kappa=P, bias=P, h0=None, offsets=None, nseq=0, y=P,
                zero_tail=0, h_out=P, states=None, kept=None, kept_scales=None, work=None, bytes=0, stream=None)
    fails(lib.cssm_token_scan, scan, -3)
    fails(lib.cssm_token_scan, scan, -3, B=1, C=1 << 26)
    step = dict(x=R, delta=R, z=None, dtype=1, B=1 << 24, C=8, kappa=P, bias=P, state=P, y=P, out=P, stream=None)
    fails(lib.cssm_token_scan_step, step, -3)
    M = 1 << 24
    fails(lib.cssm_rms_norm, dict(x=P, r=None, dtype=0, M=M, C=8, w=P, eps=1e-6, s=None, y=P, sc=None, st=None), -3)
    bwd = dict(dy=P, ds=None, s=P, dtype=0, M=M, C=8, w=P, eps=1e-6, dx=P, dw=P, work=P, bytes=1 << 50, st=None)
    fails(lib.cssm_rms_norm_bwd, bwd, -3)
    fails(lib.cssm_rms_norm_bwd, bwd, -3, M=4, C=1 << 24)
    fails(lib.cssm_quantize_rows, dict(x=P, dtype=0, M=1 << 26, K=8, q=P, s=P, st=None), -3)
    fails(lib.cssm_quantize_weight, dict(w=P, K=1 << 20, N=1 << 20, q=P, s=P, st=None), -3)
    prod = dict(a=P, sa=P, w=P, sw=P, M=4, N=8, K=1 << 24, bias=None, act=0, out=P, dtype=1, st=None)
    fails(lib.cssm_scaled_matmul, prod, -3)
    fails(lib.cssm_scaled_matmul, prod, -3, M=1 << 30, N=1 << 20, K=16)
    fails(lib.cssm_scaled_matmul, prod, -3, M=4, N=1 << 28, K=16)


def test_misaligned(lib):
    bwd = dict(dy=P, ds=None, s=P, dtype=0, M=4, C=8, w=P, eps=1e-6, dx=P, dw=P, work=P, bytes=1 << 20, st=None)
    for name in ("dy", "s", "dx", "w", "dw"):
        fails(lib.cssm_rms_norm_bwd, bwd, -5, **{name: P + 2})
    norm = dict(x=P, r=P, dtype=0, M=4, C=8, w=P, eps=1e-6, s=P, y=P, sc=None, st=None)
    for name in ("x", "r", "s", "y", "w"):
        fails(lib.cssm_rms_norm, norm, -5, **{name: P + 2})


def test_longest_sequences(lib):
    """rows up to 2^31 - 1: the tiles are counted without overflow, and what has 2^24 of them or more is refused"""
    most = (1 << 31) - 1
    assert [lib.cssm_token_scan_chunks(most - k) for k in (0, 126, 127, 128)] == [1 << 24, 1 << 24, (1 << 24) - 1, (1 << 24) - 1]
    n = 1 << 24
    assert lib.cssm_token_scan_workspace_size(1, most, 1, 0) == 8 * (1 + n + n // 8)
    scan = dict(x=R, delta=R, z=None, dtype=1, B=1, T=most, C=1, kappa=P, bias=P, h0=None, offsets=None, nseq=0, y=P,
                zero_tail=0, h_out=P, states=None, kept=None, kept_scales=None, work=P, bytes=1 << 62, stream=None)
    fails(lib.cssm_token_scan, scan, -3)
    fails(lib.cssm_token_scan, scan, -3, T=most - 126)


def test_longest_rows(lib):
    """row lengths whose end, rounded up to a block or a workgroup's step, passes 2^31"""
    for n in ((1 << 31) - 1, (1 << 31) - 512):
        fails(lib.cssm_rms_norm, dict(x=P, r=None, dtype=1, M=1, C=n, w=P, eps=1e-6, s=None, y=P, sc=None, st=None), -3)
        fails(lib.cssm_quantize_rows, dict(x=P, dtype=1, M=1, K=n, q=P, s=P, st=None), -3)


@pytest.mark.parametrize("dtype", [0, 1])
def test_scan_misaligned(lib, dtype):
    """rows and outputs to their type's size, the float32 and offset arguments to 4 bytes"""
    off = _lib.TokenRows(P + (2 if dtype == 0 else 1), 64, 8)
    bad, plain = ctypes.addressof(off), P + (2 if dtype == 0 else 1)
    scan = dict(x=R, delta=R, z=R, dtype=dtype, B=1, T=200, C=8, kappa=P, bias=P, h0=P, offsets=P, nseq=3, y=P, zero_tail=0,
                h_out=P, states=P, kept=None, kept_scales=None, work=P, bytes=BIG, stream=None)
    for name in ("x", "delta", "z"):
        fails(lib.cssm_token_scan, scan, -5, **{name: bad})
    fails(lib.cssm_token_scan, scan, -5, y=plain)
    for name in ("kappa", "bias", "h0", "offsets", "h_out", "states"):
        fails(lib.cssm_token_scan, scan, -5, **{name: P + 2})
    back = dict(x=R, delta=R, z=R, gated=1, dy=R, dtype=dtype, B=1, T=200, C=8, kappa=P, bias=P, h0=P, offsets=P, nseq=3,
                states=P, kept=None, kept_scales=None, dh=P, dx=P, dd=P, dz=P, dk=P, db=P, dh0=P, work=P, bytes=BIG, stream=None)
    for name in ("x", "delta", "z", "dy"):
        fails(lib.cssm_token_scan_bwd, back, -5, **{name: bad})
    for name in ("dx", "dd", "dz"):
        fails(lib.cssm_token_scan_bwd, back, -5, **{name: plain})
    for name in ("kappa", "bias", "h0", "offsets", "states", "dh", "dk", "db", "dh0"):
        fails(lib.cssm_token_scan_bwd, back, -5, **{name: P + 2})
    step = dict(x=R, delta=R, z=R, dtype=dtype, B=2, C=8, kappa=P, bias=P, state=P, y=P, out=P, stream=None)
    for name in ("x", "delta", "z"):
        fails(lib.cssm_token_scan_step, step, -5, **{name: bad})
    fails(lib.cssm_token_scan_step, step, -5, y=plain)
    for name in ("kappa", "bias", "state", "out"):
        fails(lib.cssm_token_scan_step, step, -5, **{name: P + 2})


def test_rows_upwards(lib):
    """a negative row stride is refused (that of the step is not used, and rows that are not read are not looked at)"""
    down = _lib.TokenRows(P, 64, -8)
    bad = ctypes.addressof(down)
    scan = dict(x=R, delta=R, z=R, dtype=0, B=1, T=200, C=8, kappa=P, bias=P, h0=P, offsets=None, nseq=0, y=P, zero_tail=0,
                h_out=P, states=P, kept=None, kept_scales=None, work=P, bytes=BIG, stream=None)
    for name in ("x", "delta", "z"):
        fails(lib.cssm_token_scan, scan, -4, **{name: bad})
    back = dict(x=R, delta=R, z=R, gated=1, dy=R, dtype=0, B=1, T=200, C=8, kappa=P, bias=P, h0=P, offsets=None, nseq=0,
                states=P, kept=None, kept_scales=None, dh=P, dx=P, dd=P, dz=P, dk=P, db=P, dh0=P, work=P, bytes=BIG, stream=None)
    for name in ("x", "delta", "z", "dy"):
        fails(lib.cssm_token_scan_bwd, back, -4, **{name: bad})
