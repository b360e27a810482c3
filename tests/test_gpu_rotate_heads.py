"""Norm and rotation of heads by positions on several axes, and its adjoint, against float64.

Bounds, u = 2^-24: the sum of squares is 16 terms a lane in a row and 6 exchanges, which moves r by half of 22 u, and r
itself, cosine, sine (an ulp or two each, and the rounding of the reduced angle, 2 pi 2^-26) and four products and a sum add
under 16 u more: 32 u of the pair's length.  An adjoint has such an error in each of its two terms, and its dot product 22 u
of the sum of magnitudes: 64 u of all.  A weight's gradient adds up at most 128 rows and heads in a lane one behind the
other before they are joined: 128 + 64 u of the sum of magnitudes.  A bfloat16 result adds half its step, eps / 2."""
import math

import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
BF16, F32, U = torch.bfloat16, torch.float32, 2.0 ** -24


@pytest.fixture(scope="module")
def Q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import sequence
    return sequence


@pytest.fixture(scope="module")
def T():
    from cssm_amd import training
    return training


def swap(x, P, pairs):
    """each value's partner with the sign that the rotation gives it (0 where nothing turns)"""
    out = torch.zeros_like(x)
    if pairs == "halves":
        out[..., :P], out[..., P:2 * P] = -x[..., P:2 * P], x[..., :P]
    else:
        out[..., 0:2 * P:2], out[..., 1:2 * P:2] = -x[..., 1:2 * P:2], x[..., 0:2 * P:2]
    return out


def plain(x, w, positions, table, norm, eps, pairs, dy=None):
    """dict of y and with dy of dx, dw in float64, and bounds as name + '_err' (before the output's own rounding)"""
    x = x.detach().double().cpu()
    D = x.shape[-1]
    w = torch.ones(D, dtype=torch.float64) if w is None else w.detach().double().cpu()
    c, s, P = torch.ones(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64), 0
    if table is not None:
        f, ax = table[0].double().cpu(), table[1].long().cpu()
        P = f.numel()
        a = (positions.cpu().double()[..., ax] * f)[..., None, :]
        one = torch.ones((*a.shape[:-1], D - 2 * P), dtype=torch.float64)
        if pairs == "halves":
            c, s = torch.cat([a.cos(), a.cos(), one], -1), torch.cat([a.sin(), a.sin(), 0 * one], -1)
        else:
            c = torch.cat([a.cos().repeat_interleave(2, -1), one], -1)
            s = torch.cat([a.sin().repeat_interleave(2, -1), 0 * one], -1)
    n = {"rms": D, "l2": 1}.get(norm)
    r = 1.0 if n is None else 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / n + eps)
    v = x * r * w
    out = {"y": v * c + swap(v, P, pairs) * s}
    out["y_err"] = 32 * U * (v.square() + swap(v, P, pairs).square()).sqrt()
    if dy is None:
        return out
    dy = dy.detach().double().cpu()
    g = dy * c - swap(dy, P, pairs) * s
    length = (dy.square() + swap(dy, P, pairs).square()).sqrt()
    t, tl = g * w, length * w.abs()
    share = 0.0 if n is None else r ** 3 / n * (t * x).sum(-1, keepdim=True)
    out["dx"] = r * t - share * x
    out["dx_err"] = 64 * U * (r * tl + (0.0 if n is None else r ** 3 / n * (tl * x.abs()).sum(-1, keepdim=True) * x.abs()))
    out["dw"] = (g * x * r).flatten(0, -2).sum(0)
    out["dw_err"] = 192 * U * (length * (x * r).abs()).flatten(0, -2).sum(0)
    return out


def off(got, want, err):
    got = got.detach()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else U
    d = (got.double().cpu() - want).abs()
    assert got.shape == want.shape and torch.isfinite(got).all()
    return float((d / (err * (1 + 2 * half) + half * want.abs() + 1e-37)).max()) if d.numel() else 0.0


# lead, Hq, Hk, D, sections (None: no rotation)
CASES = [((5,), 3, 1, 64, [32]), ((2, 9), 4, 2, 128, [24, 20, 20]), ((1,), 1, 1, 2, [1]), ((33,), 6, 6, 72, [18, 18]),
         ((7,), 2, 5, 96, [16, 16]), ((3, 4), 2, 1, 50, [10, 5, 3, 7]), ((130,), 5, 5, 256, [40, 30, 10]), ((4,), 2, 2, 512, [256]),
         ((300,), 1, 1, 16, [3, 2]), ((6,), 3, 3, 40, None), ((1200,), 16, 4, 128, [64])]


def make(Q, lead, Hq, Hk, D, sections, dtype, weights, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(s, generator=gen, device="cuda")
    q, k = ((r(*lead, H, D) * (0.1 + r(*lead, H, 1).abs())).to(dtype) for H in (Hq, Hk))
    w = [1 + 0.3 * r(D), 1 + 0.3 * r(D)] if weights else [None, None]
    table = positions = None
    if sections:
        table = Q.rotary_table(sections)
        positions = torch.randint(-50, 1 << 20, (*lead, len(sections)), generator=gen, device="cuda", dtype=torch.int32)
    return q, k, positions, table, w


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("norm,pairs,weights", [("rms", "halves", True), ("l2", "neighbours", False), ("none", "halves", True),
                                                ("rms", "neighbours", True), ("none", "neighbours", False)])
@pytest.mark.parametrize("lead,Hq,Hk,D,sections", CASES)
def test_forward_and_adjoint(Q, T, lead, Hq, Hk, D, sections, norm, pairs, weights, dtype):
    print_case(test="rotate heads", lead=lead, Hq=Hq, Hk=Hk, D=D, sections=sections, norm=norm, pairs=pairs, dtype=str(dtype))
    q, k, positions, table, (wq, wk) = make(Q, lead, Hq, Hk, D, sections, dtype, weights, D + Hq)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk) if t is not None]
    yq, yk = T.rotate_heads_train(q, k, positions, table, wq, wk, norm, 1e-5, pairs)
    with torch.no_grad():
        same = Q.rotate_heads(q, k, positions, table, wq, wk, norm, 1e-5, pairs)
    assert torch.equal(same[0], yq) and torch.equal(same[1], yk)
    gq, gk = torch.randn_like(yq), torch.randn_like(yk)
    grads = dict(zip([n for n, t in zip(("q", "k", "wq", "wk"), (q, k, wq, wk)) if t is not None],
                     torch.autograd.grad((yq, yk), leaves, (gq, gk))))
    for x, w, y, g, n in ((q, wq, yq, gq, "q"), (k, wk, yk, gk, "k")):
        want = plain(x, w, positions, table, norm, 1e-5, pairs, g)
        assert off(y, want["y"], want["y_err"]) <= 1
        assert off(grads[n], want["dx"], want["dx_err"]) <= 1
        if w is not None:
            assert off(grads["w" + n], want["dw"], want["dw_err"]) <= 1


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_far_positions(Q, dtype):
    """angles of positions up to 2^31: those of the definition, not of their float32 neighbours"""
    q, k, _, table, _ = make(Q, (64,), 2, 2, 64, [16, 16], dtype, False, 3)
    positions = torch.randint(-(1 << 31), (1 << 31) - 1, (64, 2), device="cuda", dtype=torch.int32)
    positions[0] = (1 << 31) - 1
    yq, yk = Q.rotate_heads(q, k, positions, table)
    for x, y in ((q, yq), (k, yk)):
        want = plain(x, None, positions, table, "rms", 1e-6, "halves")
        # float64 angles of 2^31 on either side are off by 2^-22 themselves
        assert off(y, want["y"], want["y_err"] + 2.0 ** -21 * want["y_err"] / (32 * U)) <= 1


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1])
def test_strided(Q, T, dtype, shift):
    """q and k as slices of one projection, on and off the vector width; a gradient that is one number for all"""
    B, L, H, D = 2, 11, 3, 32
    rows = torch.randn((B, L, 3 * H * D + shift), device="cuda").to(dtype)[..., shift:]
    q, k, _ = (t.unflatten(-1, (H, D)) for t in rows.split(H * D, -1))
    positions = torch.arange(L, device="cuda", dtype=torch.int32).expand(B, L)[..., None].contiguous()
    table = Q.rotary_table([16])
    got = Q.rotate_heads(q, k, positions, table)
    for x, y in zip((q, k), got):
        want = plain(x, None, positions, table, "rms", 1e-6, "halves")
        assert off(y, want["y"], want["y_err"]) <= 1
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    yq, yk = T.rotate_heads_train(q, k, positions, table)
    one = torch.ones((), device="cuda", dtype=dtype).expand_as(yq)
    for g, x in zip(torch.autograd.grad((yq, yk), (q, k), (one, one)), (q, k)):
        want = plain(x, None, positions, table, "rms", 1e-6, "halves", one)
        assert off(g, want["dx"], want["dx_err"]) <= 1


def test_queries_alone(Q, T):
    q, _, positions, table, (w, _) = make(Q, (9,), 4, 1, 64, [32], BF16, True, 5)
    y, none = Q.rotate_heads(q, None, positions, table, q_weight=w)
    want = plain(q, w, positions, table, "rms", 1e-6, "halves")
    assert none is None and off(y, want["y"], want["y_err"]) <= 1
    q.requires_grad_(), w.requires_grad_()
    y, none = T.rotate_heads_train(q, None, positions, table, q_weight=w)
    g = torch.randn_like(y)
    dq, dw = torch.autograd.grad(y, (q, w), g)
    want = plain(q, w, positions, table, "rms", 1e-6, "halves", g)
    assert none is None and off(dq, want["dx"], want["dx_err"]) <= 1 and off(dw, want["dw"], want["dw_err"]) <= 1


def test_one_output_used(Q, T):
    q, k, positions, table, (wq, wk) = make(Q, (20,), 2, 2, 64, [32], F32, True, 6)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = T.rotate_heads_train(q, k, positions, table, wq, wk)
    g = torch.randn_like(yq)
    dq, dk, dwq, dwk = torch.autograd.grad(yq, leaves, g, allow_unused=True)
    want = plain(q, wq, positions, table, "rms", 1e-6, "halves", g)
    assert off(dq, want["dx"], want["dx_err"]) <= 1 and off(dwq, want["dw"], want["dw_err"]) <= 1
    assert not dk.any() and not dwk.any()


def test_zero_heads_and_no_rows(Q, T):
    """heads of zeros give zeros; no rows give no rows, and weights a gradient of zero"""
    q = torch.zeros((3, 2, 64), device="cuda")
    y, _ = Q.rotate_heads(q, None, norm="l2")
    assert not y.any()
    q, k, w = (torch.zeros(s, device="cuda").requires_grad_() for s in ((0, 2, 64), (0, 1, 64), (64,)))
    yq, yk = T.rotate_heads_train(q, k, q_weight=w)
    assert yq.shape == q.shape and yk.shape == k.shape
    assert not torch.autograd.grad(yq.sum() + yk.sum(), w)[0].any()


def test_table(Q):
    t = Q.rotary_table([2, 3], base=100.0)
    assert torch.allclose(t.frequencies.cpu(), torch.tensor([1, 0.1, 1, 100 ** (-1 / 3), 100 ** (-2 / 3)], dtype=torch.float64))
    assert t.axes.tolist() == [0, 0, 1, 1, 1]
    t = Q.rotary_table([2, 2], base=16.0, shared=True)
    assert torch.allclose(t.frequencies.cpu(), torch.tensor([1, 0.5, 0.25, 0.125], dtype=torch.float64))
    for bad in ([], [0], [1] * 5, [4, -1]):
        with pytest.raises(ValueError):
            Q.rotary_table(bad)


def test_captured(Q, T):
    """forward and backward in a graph, replayed between eager work"""
    q, k, positions, table, (wq, wk) = make(Q, (2, 50), 4, 2, 64, [16, 16], BF16, True, 8)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    gq, gk = torch.randn_like(q), torch.randn_like(k)

    def run(a):
        yq, yk = T.rotate_heads_train(a[0], a[1], positions, table, a[2], a[3])
        return (yq.detach(), yk.detach(), *torch.autograd.grad((yq, yk), a, (gq, gk)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(leaves)
    for i in range(4):
        with torch.no_grad():
            q.mul_(1 + i), positions.add_(i)
        want = run([t.detach().requires_grad_() for t in leaves])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_refusals(Q):
    q, k, positions, table, (w, _) = make(Q, (2, 5), 2, 1, 64, [16, 16], BF16, True, 9)
    for args, kw in [((q.cpu(), k, positions, table), {}), ((q, k.float(), positions, table), {}), ((q, k[:, :4], positions, table), {}),
                     ((q, k, positions.long(), table), {}), ((q, k, positions[:, :4], table), {}), ((q, k, positions, None), {}),
                     ((q, k, None, table), {}), ((q, k, positions, (table[0].float(), table[1])), {}),
                     ((q, k, positions, (table[0], table[1][:4])), {}), ((q, k, positions, table), dict(q_weight=w[:4])),
                     ((q, k, positions, table), dict(norm="layer")), ((q, k, positions, table), dict(pairs="thirds")),
                     ((q[..., :63], k[..., :63], positions, table), {}), ((q.transpose(-1, -2), k, positions, table), {}),
                     ((q[..., :32], k[..., :32], positions, Q.rotary_table([20])), {}), ((q.double(), None, positions, table), {}),
                     ((q, k, positions.repeat(1, 1, 3), table), {})]:
        with pytest.raises(ValueError):
            Q.rotate_heads(*args, **kw)
    from cssm_amd._lib import CssmError
    with pytest.raises(CssmError):
        Q.rotate_heads(q, k, positions, table, eps=-1.0)
    assert math.isfinite(float(Q.rotate_heads(q, k, positions, table, eps=0.0)[0].sum()))
