"""Gradients of the gated delta rule where the first tests do not look: packed rows whose forward is walked in parts, more
packed sequences than are taken by length, what lies behind the last sequence, and differences along the gradient itself."""
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


def check(T, offsets, tail, Hk, Hv, dk, dv, dtype, seed):
    """whatever is read behind the last sequence would show: it is not a number, in the gradient that comes in too"""
    n, end = len(offsets) - 1, offsets[-1]
    args = R.inputs(1, end + tail, Hk, Hv, dk, dv, dtype, seed, n=n)
    for t in args[:5]:
        t[end:] = float("nan")
    args = [t.requires_grad_() for t in args]
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y, final = T.delta_rule_train(*args[:4], decay=args[4], state=args[5], offsets=off)
    gy, gf = torch.randn_like(y), torch.randn_like(final)
    gy[end:] = float("nan")
    grads = torch.autograd.grad((y, final), args, (gy, gf))
    want = R.whole(*(t[:end] for t in args[:5]), args[5], off, dy=gy[:end], dfinal=gf)
    assert R.off(y[:end], want["y"]) <= 1 and R.off(final, want["final"]) <= 1 and not y[end:].any()
    for name, got in zip(NAMES, grads):
        if name != "state":
            assert not got[end:].any(), name
            got = got[:end]
        assert R.off(got, want["d" + name]) <= 1, (name, R.off(got, want["d" + name]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dk,dv", [(40, 24), (128, 64), (33, 50)])
@pytest.mark.parametrize("offsets,tail", [([0, 5, 5, 40, 104, 290], 9), ([0, 128, 256], 50), ([0, 0], 7), ([0, 31], 1)])
def test_tails(T, offsets, tail, dk, dv, dtype):
    print_case(test="delta rule gradients, tails", offsets=offsets, tail=tail, dk=dk, dv=dv, dtype=str(dtype))
    check(T, offsets, tail, 2, 4, dk, dv, dtype, offsets[-1] + dk)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offsets,tail", [([0, 700, 700, 1800, 3100], 13), ([0, 0, 2100, 2101], 0)])
def test_parts(T, offsets, tail, dtype):
    """few heads of long packed sequences: the forward walks them in parts, with errors and states kept"""
    print_case(test="delta rule gradients, packed in parts", offsets=offsets, tail=tail, dtype=str(dtype))
    check(T, offsets, tail, 1, 2, 40, 24, dtype, 3)


@pytest.mark.parametrize("n", [64, 65, 150])
def test_many(T, n):
    """sequences taken by their length up to 64 of them, in their order from there"""
    cuts = torch.randint(0, 900, (n - 1,), generator=torch.Generator().manual_seed(n)).sort().values.tolist()
    check(T, [0] + cuts + [900], 6, 1, 2, 16, 8, F32, n)


@pytest.mark.parametrize("dtype", [F32])
@pytest.mark.parametrize("name", NAMES)
def test_along_the_gradient(T, name, dtype):
    """The difference of the outputs' product with gy over a step h along the gradient's own direction is its length.

    Central differences, the kernels' float32 outputs summed up in float64, with h such that the product changes by 2^-6 of |y|.
    The outputs' roundings are 2^-18 of their length at most (tests/delta_reference.py) and do not follow gy, whose values have random
    signs and length 1 each: at three deviations 3 x 2^-18 |y| of the product at either end, 3 x 2^-13 of the difference over
    the two ends' 2 x 2^-6 |y|, taken as if they added up.  The third derivative's share of it is 2.1e-5 for decay, the most, in
    float64 arithmetic of the same inputs.  2^-11 bounds both."""
    args = [t.requires_grad_() for t in R.inputs(1, 140, 1, 2, 32, 32, dtype, 21)]
    gy = torch.randn(args[2].shape, generator=torch.Generator("cuda").manual_seed(4), device="cuda")
    y, _ = T.delta_rule_train(*args[:4], decay=args[4], state=args[5])
    g = torch.autograd.grad(y, args, gy)[NAMES.index(name)].double()
    length = float(g.norm())
    h = 2.0 ** -6 * float(y.detach().double().norm()) / length
    ends = []
    for s in (h, -h):
        moved = [a.detach() for a in args]
        i = NAMES.index(name)
        moved[i] = (moved[i].double() + s * g / length).float()
        z = T.delta_rule_train(*moved[:4], decay=moved[4], state=moved[5])[0]
        ends.append(float((z.double() * gy.double()).sum()))
    assert abs((ends[0] - ends[1]) / (2 * h) - length) <= 2.0 ** -11 * length
