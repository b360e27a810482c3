"""Gradients of the gated delta rule over token sequences against float64 differentiation, token by token."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import delta_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NAMES = ("q", "k", "v", "beta", "decay", "state")


@pytest.fixture(scope="module")
def T():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import training
    return training


def check(T, args, offsets=None, dy=True, dfinal=True, scale=None):
    args = [None if t is None else t.requires_grad_() for t in args]
    y, final = T.delta_rule_train(*args[:4], decay=args[4], state=args[5], offsets=offsets, scale=scale)
    gen = torch.Generator(device="cuda").manual_seed(1)
    gy = torch.randn(y.shape, generator=gen, device="cuda").to(y.dtype) if dy else None
    gf = torch.randn(final.shape, generator=gen, device="cuda") if dfinal else None
    if offsets is not None and dy:
        gy[int(offsets[-1]):] = float("nan")       # not read
    leaves = [t for t in args if t is not None]
    grads = torch.autograd.grad([t for t, g in ((y, gy), (final, gf)) if g is not None], leaves,
                                [g for g in (gy, gf) if g is not None])
    if offsets is not None and dy:
        gy = torch.nan_to_num(gy)
    want = R.whole(*args, offsets=offsets, scale=scale, dy=gy, dfinal=gf)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1
    for name, got in zip([n for n, t in zip(NAMES, args) if t is not None], grads):
        assert R.off(got, want["d" + name]) <= 1, (name, R.off(got, want["d" + name]))
    return grads


SIZES = [(1, 1, 1, 1, 1, 1), (2, 31, 1, 2, 16, 16), (1, 32, 2, 2, 64, 64), (2, 33, 1, 1, 128, 128), (1, 128, 3, 3, 40, 50),
         (2, 129, 1, 3, 65, 100), (1, 300, 1, 2, 5, 33), (1, 257, 2, 2, 128, 64), (1, 160, 1, 1, 32, 128)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T_,Hk,Hv,dk,dv", SIZES)
def test_sequences(T, B, T_, Hk, Hv, dk, dv, dtype):
    print_case(test="delta rule gradients", B=B, T=T_, Hk=Hk, Hv=Hv, dk=dk, dv=dv, dtype=str(dtype))
    check(T, R.inputs(B, T_, Hk, Hv, dk, dv, dtype, B * T_ + dk))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long(T, dtype):
    """few heads of a long sequence, which the forward walks in parts"""
    check(T, R.inputs(1, 1500, 1, 2, 48, 32, dtype, 5))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dy,dfinal", [(True, False), (False, True)])
def test_one_gradient(T, dy, dfinal, dtype):
    """no decay, no state, another scale; one of the two outputs used"""
    a = R.inputs(2, 150, 2, 4, 48, 24, dtype, 3)
    check(T, [*a[:4], None, None], dy=dy, dfinal=dfinal, scale=0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_correlated_keys(T, dtype):
    check(T, R.inputs(1, 200, 1, 2, 64, 64, dtype, 6, correlated=True))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offsets,tail", [([0, 5, 5, 40, 104, 290], 9), ([0, 0, 0, 1, 2, 34, 180, 180], 0), ([0, 128, 256], 50),
                                          ([0, 0], 7)])
def test_packed(T, offsets, tail, dtype):
    n, rows = len(offsets) - 1, offsets[-1] + tail
    print_case(test="delta rule gradients packed", offsets=offsets, tail=tail, dtype=str(dtype))
    a = R.inputs(1, rows, 2, 4, 40, 24, dtype, rows + n, n=n)
    for t in a[:5]:
        t[offsets[-1]:] = float("nan")             # not read
    a[0][offsets[-1]:], a[1][offsets[-1]:], a[2][offsets[-1]:] = 0, 0, float("nan")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    # the float64 side multiplies what lies behind by zero: it gets the rows up to there
    args = [t.requires_grad_() for t in a]
    y, final = T.delta_rule_train(*args[:4], decay=args[4], state=args[5], offsets=off)
    gy, gf = torch.randn_like(y), torch.randn_like(final)
    grads = torch.autograd.grad((y, final), args, (gy, gf))
    end = offsets[-1]
    want = R.whole(*(t[:end] for t in args[:5]), args[5], off, dy=gy[:end], dfinal=gf)
    assert R.off(y[:end], want["y"]) <= 1 and R.off(final, want["final"]) <= 1 and not y[end:].any()
    for name, got in zip(NAMES, grads):
        if name != "state":
            assert not got[end:].any()
            got = got[:end]
        assert R.off(got, want["d" + name]) <= 1, name


def test_masked_rows(T):
    """beta = 0 and decay = 0 in places; decay = -inf, whose own gradient is none up to rounding"""
    q, k, v, beta, decay, state = R.inputs(2, 190, 1, 2, 32, 32, F32, 11)
    beta[:, 20:50], decay[:, 20:50] = 0.0, 0.0
    decay[0, 70], decay[1, 133] = float("-inf"), float("-inf")
    args = [t.requires_grad_() for t in (q, k, v, beta, decay, state)]
    y, final = T.delta_rule_train(*args[:4], decay=args[4], state=args[5])
    gy, gf = torch.randn_like(y), torch.randn_like(final)
    grads = torch.autograd.grad((y, final), args, (gy, gf))
    want = R.whole(*args, dy=gy, dfinal=gf)
    want["ddecay"] = torch.nan_to_num(want["ddecay"], nan=0.0)
    for name, got in zip(NAMES, grads):
        assert R.off(got, want["d" + name]) <= 1, name


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided(T, dtype):
    """slices of one projection's rows, and a gradient that is a slice or one number for all"""
    B, T_, H, d = 2, 75, 2, 32
    rows = torch.randn((B, T_, 3 * H * d), device="cuda")
    rows[..., H * d:2 * H * d] = torch.nn.functional.normalize(rows[..., H * d:2 * H * d].unflatten(-1, (H, d)), dim=-1).flatten(-2)
    rows = rows.to(dtype).requires_grad_()
    gates = torch.rand((B, T_, 2 * H), device="cuda").requires_grad_()

    def parts():
        q, k, v = (t.unflatten(-1, (H, d)) for t in rows.split(H * d, -1))
        return q, k, v, gates[..., :H], -gates[..., H:]
    for grad in (torch.randn((B, T_, 2 * H, d), device="cuda").to(dtype)[..., 1:1 + H, :], torch.ones((), device="cuda", dtype=dtype).expand(B, T_, H, d)):
        q, k, v, beta, decay = parts()
        y, _ = T.delta_rule_train(q, k, v, beta, decay)
        got = torch.autograd.grad(y, (rows, gates), grad)
        want = R.whole(q, k, v, beta, decay, dy=grad)
        each = torch.cat([want[n].flatten(-2) for n in ("dq", "dk", "dv")], -1)
        assert R.off(got[0], each) <= 1
        assert R.off(got[1], torch.cat([want["dbeta"], -want["ddecay"]], -1)) <= 1


def test_same_tensor_twice(T):
    """one tensor as q, k and v: its gradients add up"""
    x = torch.nn.functional.normalize(torch.randn((1, 100, 2, 32), device="cuda"), dim=-1).requires_grad_()
    beta = torch.rand((1, 100, 2), device="cuda")
    y, _ = T.delta_rule_train(x, x, x, beta)
    g = torch.randn_like(y)
    got, = torch.autograd.grad(y, x, g)
    want = R.whole(x, x, x, beta, dy=g)
    assert R.off(got, want["dq"] + want["dk"] + want["dv"]) <= 1


def test_differences(T):
    """the gradients' sum along a direction, against a difference of the kernel's own outputs: y is a polynomial in beta and
    v, so central differences of step h are off by h^2 of it, and by 2^-24 / h of rounding: 2^-12 for h = 2^-8"""
    args = [t.requires_grad_() for t in R.inputs(1, 140, 1, 2, 32, 32, F32, 21)]
    gy = torch.randn_like(args[2])
    y, _ = T.delta_rule_train(*args[:4], decay=args[4], state=args[5])
    grads = torch.autograd.grad(y, args, gy)
    h = 2.0 ** -8
    for i, (t, g) in enumerate(zip(args, grads)):
        step = 0.1 * torch.randn_like(t)
        ends = []
        for s in (h, -h):
            moved = [a.detach() for a in args]
            moved[i] = t.detach() + s * step
            y = T.delta_rule_train(*moved[:4], decay=moved[4], state=moved[5])[0]
            ends.append(float((y.double() * gy.double()).sum()))
        along = float((g.double() * step.double()).sum())
        size = float(g.double().norm() * step.double().norm()) / t.numel() ** 0.5
        assert abs((ends[0] - ends[1]) / (2 * h) - along) <= 2.0 ** -12 * (size * t.numel() ** 0.5 + float(gy.norm() * y.norm()))


def test_repeats_and_streams(T):
    sets = [[t.requires_grad_() for t in R.inputs(1, 700, 4, 8, 128, 128, BF16, 20 + i)] for i in range(2)]

    def run(a):
        y, f = T.delta_rule_train(*a[:4], decay=a[4], state=a[5])
        return torch.autograd.grad((y, f), a, (y.detach(), f.detach()))
    want = [run(a) for a in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for x, w in zip(g, want[i]):
                assert torch.equal(x, w)


def test_captured(T):
    """forward and backward in one graph, replayed between eager work"""
    a = [t.requires_grad_() for t in R.inputs(2, 140, 1, 2, 64, 64, BF16, 30)]
    grad = torch.randn_like(a[2])

    def run(a):
        y, f = T.delta_rule_train(*a[:4], decay=a[4], state=a[5])
        return (y.detach(), *torch.autograd.grad((y, f), a, (grad, f.detach())))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(a)
    for i in range(4):
        with torch.no_grad():
            a[2].add_(i), a[5].mul_(0.5)
        want = run([t.detach().requires_grad_() for t in a])
        graph.replay()
        torch.cuda.synchronize()
        for x, w in zip(got, want):
            assert torch.equal(x, w)


def test_second_derivative_refused(T):
    a = [t.requires_grad_() for t in R.inputs(1, 8, 1, 1, 8, 8, F32, 31)]
    y, _ = T.delta_rule_train(*a[:4], decay=a[4], state=a[5])
    g, = torch.autograd.grad(y.sum(), a[0], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_no_rows(T):
    a = [t.requires_grad_() for t in R.inputs(2, 0, 1, 2, 16, 8, BF16, 4)]
    y, f = T.delta_rule_train(*a[:4], decay=a[4], state=a[5])
    g = torch.randn_like(f)
    grads = torch.autograd.grad((f, y), a, (g, torch.ones((), device="cuda", dtype=BF16).expand_as(y)))
    assert torch.equal(grads[5], g) and all(not t.numel() for t in grads[:5])
