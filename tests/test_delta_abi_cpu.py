"""Refusals of the delta rule's and the head rotation's entry points: arguments are checked before any GPU work, so no GPU
is needed."""
import ctypes

import pytest

from cssm_amd import _lib

BUF = ctypes.create_string_buffer(8192)
P = (ctypes.addressof(BUF) + 255) // 256 * 256
ROWS = _lib.TokenRows(P, 1 << 12, 64)
R = ctypes.addressof(ROWS)
EMPTY, DOWN, WIDE, OFF = (_lib.TokenRows(*a) for a in ((None, 64, 8), (P, 64, -8), (P, 64, (1 << 24) + 8), (P + 1, 64, 8)))
BIG = 1 << 40

RULE = dict(q=R, k=R, v=R, dtype=1, beta=R, decay=R, B=2, T=200, Hk=2, Hv=4, dk=16, dv=8, scale=1.0, h0=None, offsets=None,
            nseq=0, y=P, zero_tail=0, h_out=None, errors=None, states=None, work=P, bytes=BIG, stream=None)
BWD = dict(q=R, k=R, dtype=0, beta=R, decay=R, dy=R, B=2, T=200, Hk=2, Hv=4, dk=16, dv=8, scale=1.0, offsets=None, nseq=0,
           errors=P, states=P, dh=None, dq=P, dkey=P, dval=P, dbeta=P, ddecay=P, dh0=None, work=P, bytes=BIG, stream=None)
STEP = dict(q=R, k=R, v=R, dtype=1, beta=R, decay=None, B=2, Hk=2, Hv=4, dk=16, dv=8, scale=1.0, state=P, y=P, out=P, stream=None)
TURN = dict(q=R, k=R, dtype=1, B=2, T=5, Hq=2, Hk=1, D=16, wq=P, wk=P, norm=0, eps=1e-6, positions=P, axes=2, freq=P, axis=P,
            P=8, halves=1, qo=P, ko=P, stream=None)
TURN_BWD = dict(q=R, k=R, dqo=R, dko=R, dtype=1, B=2, T=5, Hq=2, Hk=1, D=16, wq=P, wk=P, norm=0, eps=1e-6, positions=P, axes=2,
                freq=P, axis=P, P=8, halves=1, dq=P, dk=P, dwq=P, dwk=P, work=P, bytes=BIG, stream=None)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def fails(fn, args, status, **change):
    st = fn(*dict(args, **change).values())
    assert st == status, (change, st, _lib.load().cssm_last_error())
    assert _lib.load().cssm_last_error()


def of(rows):
    return ctypes.addressof(rows)


def test_rule(lib):
    fn = lib.cssm_delta_rule
    for name in ("q", "k", "v", "beta", "y"):
        fails(fn, RULE, -1, **{name: None})
    for name in ("q", "k", "v", "beta", "decay"):
        fails(fn, RULE, -1, **{name: of(EMPTY)})
        fails(fn, RULE, -4, **{name: of(DOWN)})
    for name in ("q", "k", "v"):
        fails(fn, RULE, -3, **{name: of(WIDE)})
        fails(fn, RULE, -5, **{name: of(OFF)})
    fails(fn, RULE, -1, errors=P)
    fails(fn, RULE, -1, states=P)
    fails(fn, RULE, -4, dtype=2)
    for name in ("B", "T"):
        fails(fn, RULE, -2, **{name: -1})
    for name in ("Hk", "Hv", "dk", "dv"):
        fails(fn, RULE, -2, **{name: 0})
    fails(fn, RULE, -2, Hk=3)
    fails(fn, RULE, -2, offsets=P, nseq=3)            # packed rows are one batch
    fails(fn, RULE, -2, B=1, offsets=P, nseq=0)
    fails(fn, RULE, -3, dk=129)
    fails(fn, RULE, -3, dv=129)
    fails(fn, RULE, -3, Hv=1 << 17)
    fails(fn, RULE, -3, B=1 << 20)
    fails(fn, RULE, -3, B=1, T=(1 << 31) - 1)
    fails(fn, RULE, -4, work=None)
    fails(fn, RULE, -4, bytes=lib.cssm_delta_rule_workspace_size(2, 200, 4, 16, 8, 0, 0) - 1)
    fails(fn, RULE, -5, work=P + 8)
    for name in ("h0", "h_out", "y"):
        fails(fn, RULE, -5, **{name: P + 1})
    fails(fn, RULE, -5, beta=of(OFF))
    assert fn(*dict(RULE, B=0).values()) == 0


def test_rule_bwd(lib):
    fn = lib.cssm_delta_rule_bwd
    for name in ("q", "k", "beta", "dy", "errors", "states", "dq", "dkey", "dval", "dbeta", "ddecay"):
        fails(fn, BWD, -1, **{name: None})
    fails(fn, BWD, -1, decay=None)                    # ddecay and decay go together
    fails(fn, BWD, -4, dtype=3)
    fails(fn, BWD, -3, dk=200)
    fails(fn, BWD, -3, dy=of(WIDE))
    fails(fn, BWD, -4, bytes=lib.cssm_delta_rule_bwd_workspace_size(2, 200, 2, 4, 16, 8, 0, 0) - 1)
    fails(fn, BWD, -5, work=P + 4)
    for name in ("dh", "dh0", "dbeta", "ddecay", "errors", "states", "dq", "dkey", "dval"):
        fails(fn, BWD, -5, **{name: P + 1})
    assert fn(*dict(BWD, B=0).values()) == 0


def test_step(lib):
    fn = lib.cssm_delta_rule_step
    for name in ("q", "k", "v", "beta", "state", "y", "out"):
        fails(fn, STEP, -1, **{name: None})
    fails(fn, STEP, -2, Hv=3)
    fails(fn, STEP, -3, dv=256)
    fails(fn, STEP, -4, dtype=-1)
    fails(fn, STEP, -5, state=P + 2)
    fails(fn, STEP, -5, out=P + 2)
    assert fn(*dict(STEP, B=0).values()) == 0


def test_sizes(lib):
    assert [lib.cssm_delta_rule_segments(1, t, 0, 0) for t in (0, 1, 128, 129)] == [0, 1, 1, 2]
    assert lib.cssm_delta_rule_segments(3, 200, 0, 0) == 6 and lib.cssm_delta_rule_segments(1, 300, 5, 1) == 7
    assert lib.cssm_delta_rule_segments(0, 5, 0, 0) == lib.cssm_delta_rule_segments(1, -1, 0, 0) == 0
    for a in ((0, 5, 1, 1, 1, 0, 0), (1, -1, 1, 1, 1, 0, 0), (1, 5, 0, 1, 1, 0, 0), (1, 5, 1, 0, 1, 0, 0)):
        assert lib.cssm_delta_rule_workspace_size(*a) == 0
    assert lib.cssm_delta_rule_segments(1 << 30, 1 << 30, 0, 0) == (1 << 31) - 1
    # sizes past 32 bits
    assert lib.cssm_delta_rule_workspace_size(1 << 20, 1 << 20, 1, 8, 8, 0, 0) > 1 << 45
    assert lib.cssm_delta_rule_workspace_size(64, 1 << 16, 32, 128, 128, 0, 0) > 1 << 32
    assert lib.cssm_delta_rule_bwd_workspace_size(64, 1 << 16, 32, 32, 128, 128, 0, 0) > 1 << 34


def test_rotate(lib):
    fn = lib.cssm_rotate_heads
    for name in ("q", "k", "positions", "freq", "axis", "qo", "ko"):
        fails(fn, TURN, -1, **{name: None})
    fails(fn, TURN, -4, q=of(DOWN))
    fails(fn, TURN, -5, q=of(OFF))
    fails(fn, TURN, -5, freq=P + 4)
    for name in ("wq", "wk", "positions", "axis"):
        fails(fn, TURN, -5, **{name: P + 2})
    fails(fn, TURN, -4, dtype=2)
    fails(fn, TURN, -4, norm=3)
    fails(fn, TURN, -4, eps=-1.0)
    fails(fn, TURN, -4, eps=float("nan"))
    for change in (dict(B=-1), dict(T=-1), dict(Hq=0), dict(Hk=-1), dict(D=15), dict(D=0), dict(P=9), dict(P=-1)):
        fails(fn, TURN, -2, **change)
    for change in (dict(D=514), dict(axes=0), dict(axes=5), dict(B=1 << 16, T=1 << 16), dict(Hq=1 << 24)):
        fails(fn, TURN, -3, **change)
    assert fn(*dict(TURN, B=0).values()) == 0
    fn = lib.cssm_rotate_heads_bwd
    for name in ("q", "k", "dqo", "dko", "dq", "dk"):
        fails(fn, TURN_BWD, -1, **{name: None})
    fails(fn, TURN_BWD, -2, T=0)
    fails(fn, TURN_BWD, -4, work=None)
    fails(fn, TURN_BWD, -4, bytes=lib.cssm_rotate_heads_bwd_workspace_size(16) - 1)
    fails(fn, TURN_BWD, -5, work=P + 2)
    fails(fn, TURN_BWD, -5, dq=P + 1)


def test_wide_tensors(monkeypatch):
    """sizes that the 32-bit arguments would cut are refused before the call; tensors without memory stand for the GPU's"""
    torch = pytest.importorskip("torch")
    from cssm_amd import sequence as Q
    got, far = [], (1 << 32) + 16
    monkeypatch.setattr(Q, "_gpu", lambda x, name: 0)
    monkeypatch.setattr(Q, "_call", lambda dev, name, *args: got.append(name))

    def t(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        Q.delta_rule(t(1, far, 1, 8), t(1, far, 1, 8), t(1, far, 1, 8), t(1, far, 1))
    with pytest.raises(ValueError, match="2\\^31"):
        Q.delta_rule_step(t(far, 1, 8), t(far, 1, 8), t(far, 1, 8), t(far, 1), t(far, 1, 8, 8))
    with pytest.raises(ValueError, match="2\\^31"):
        Q.rotate_heads(t(far, 1, 8), None)
    assert not got
    Q.delta_rule(t(1, 9, 1, 8), t(1, 9, 1, 8), t(1, 9, 1, 8), t(1, 9, 1))
    Q.delta_rule_step(t(2, 1, 8), t(2, 1, 8), t(2, 1, 8), t(2, 1), t(2, 1, 8, 8))
    Q.rotate_heads(t(3, 1, 8), None)
    assert got == ["cssm_delta_rule", "cssm_delta_rule_step", "cssm_rotate_heads"]
