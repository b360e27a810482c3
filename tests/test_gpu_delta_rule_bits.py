"""y of the gated delta rule in bfloat16 is rounded once, from float32 sums.

Bounds, u = 2^-24.  Chosen values: |y - want| <= half a step of want (2^-8 of it) and u for each of the sums that a value
goes through (the parts of a product, the chunk's, the state's: 6) of the terms' magnitudes.
Random values: before its rounding y is off by at most 2^-18 of the tensor's root mean square in the mean, the bound of float32
results (tests/delta_reference.py).  A value comes to the other neighbour with the probability of its error over its step,
1 at most.  A normal value's step is 2^-7 of the power of two below it, 0.72 x 2^-7 of |y| in the mean; with c = 2^-18 / (0.72 x
2^-7) = 6.8e-4 that is the mean of min(1, c / |y|) = 0.8 c (1 + ln(1 / c)) = 4.5e-3 of the values."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import delta_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32, U = torch.bfloat16, torch.float32, 2.0 ** -24
LONG = [1.0, 3 * 2.0 ** -10, 2.0 ** -17, 2.0 ** -23]   # their sum has 24 bits, two bfloat16 parts of it are 2^-17 away
LEFT = LONG[2] + LONG[3]                               # of it, when the first two are taken away


@pytest.fixture(scope="module")
def Q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import sequence
    return sequence


def near(y, terms):
    assert y.dtype == BF16
    assert bool(((y.double() - LEFT).abs() <= 2.0 ** -8 * LEFT + 6 * U * terms).all()), y.flatten()[:4]


@pytest.mark.parametrize("width", [8, 50, 64, 128])
def test_state(Q, width):
    """two rows of the state that nearly cancel in the query"""
    T = 70
    q = torch.zeros((1, T, 1, width), dtype=BF16, device="cuda")
    q[..., 1], q[..., width - 1] = 1.0, 1.0
    state = torch.zeros((1, 1, width, width), device="cuda")
    state[:, :, 1], state[:, :, width - 1] = sum(LONG), -sum(LONG[:2])
    v = torch.zeros_like(q)
    y, final = Q.delta_rule(q, v, v, torch.zeros((1, T, 1), device="cuda"), state=state, scale=1.0)
    assert torch.equal(final, state)
    near(y, 2.01)


@pytest.mark.parametrize("width", [8, 50, 64, 128])
@pytest.mark.parametrize("first", [0, 7, 30])
def test_errors(Q, first, width):
    """two rows of a chunk whose shares nearly cancel: the errors have the bits"""
    q, k, v = (torch.zeros((1, 40, 1, width), dtype=BF16, device="cuda") for _ in range(3))
    beta = torch.zeros((1, 40, 1), device="cuda")
    k[:, first, :, 0], k[:, first + 1, :, 1] = 1.0, 1.0
    beta[:, first], beta[:, first + 1] = sum(LONG), sum(LONG[:2])
    v[:, first], v[:, first + 1] = 1.0, -1.0
    q[..., 0], q[..., 1] = 1.0, 1.0
    y, _ = Q.delta_rule(q, k, v, beta, scale=1.0)
    near(y[:, first + 1:], 2.01)


@pytest.mark.parametrize("width", [8, 50, 64, 128])
def test_pairs(Q, width):
    """the same, the products of queries and keys having the bits"""
    q, k, v = (torch.zeros((1, 40, 1, width), dtype=BF16, device="cuda") for _ in range(3))
    beta = torch.zeros((1, 40, 1), device="cuda")
    k[:, 3, :, :4] = torch.tensor(LONG, device="cuda")
    k[:, 4, :, 4:6] = -torch.tensor(LONG[:2], device="cuda")
    beta[:, 3:5], v[:, 3:5] = 1.0, 1.0
    q[..., :6] = 1.0
    y, _ = Q.delta_rule(q, k, v, beta, scale=1.0)
    near(y[:, 4:], 2.01)


@pytest.mark.parametrize("offsets", [None, [0, 300, 300, 411]])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (100, 40)])
def test_rounded_once(Q, dk, dv, offsets):
    T, n = 411, None if offsets is None else len(offsets) - 1
    print_case(test="delta rule rounded once", dk=dk, dv=dv, offsets=offsets)
    q, k, v, beta, decay, state = R.inputs(1, T, 2, 4, dk, dv, BF16, dk + dv, n=n, correlated=True)
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y, _ = Q.delta_rule(q, k, v, beta, decay, state, offsets=off)
    want = R.whole(q, k, v, beta, decay, state, off)["y"].bfloat16()
    assert float((y.cpu() != want).double().mean()) <= 4.5e-3
