"""The decays' gradient of the gated delta rule where decays are strong: against float64, each head by itself.

A decay's gradient is the sum of what crosses its row, every term with the factor exp(decay), so that float32's bound as a
length (2^-18, tests/delta_reference.py) holds for a head whose gradients are small throughout, and where a decay clears the
state its gradient is 0, not a small number."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import delta_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def T():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import training
    return training


def gradients(T, q, k, v, beta, decay, state, offsets=None):
    args = [t.requires_grad_() for t in (q, k, v, beta, decay, state)]
    y, final = T.delta_rule_train(*args[:4], decay=args[4], state=args[5], offsets=offsets)
    gen = torch.Generator(device="cuda").manual_seed(2)
    gy, gf = (torch.randn(t.shape, generator=gen, device="cuda").to(t.dtype) for t in (y, final))
    got = torch.autograd.grad((y, final), args, (gy, gf))
    want = R.whole(*args, offsets, dy=gy, dfinal=gf)
    for name, g in zip(("q", "k", "v", "beta", "state"), (*got[:4], got[5])):
        assert R.off(g, want["d" + name]) <= 1, name
    return got[4], want["ddecay"]


def each_head(got, want):
    for h in range(got.shape[-1]):
        assert R.off(got[..., h], want[..., h]) <= 1, (h, R.off(got[..., h], want[..., h]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T_,dk,dv", [(200, 64, 64), (77, 128, 128), (257, 100, 50)])
@pytest.mark.parametrize("decay", [-0.01, -1.0, -2.0, -4.0, -8.0, -16.0, -30.0])
def test_uniform(T, decay, T_, dk, dv, dtype):
    print_case(test="uniform decays", decay=decay, T=T_, dk=dk, dv=dv, dtype=str(dtype))
    q, k, v, beta, d, state = R.inputs(1, T_, 1, 2, dk, dv, dtype, T_)
    each_head(*gradients(T, q, k, v, beta, torch.full_like(d, decay), state))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("decay", [-4.0, -16.0])
def test_one_strong_row(T, decay, dtype):
    """each head has one strong decay in each 128 rows and none beside it: its gradient against that row's own size"""
    H, T_ = 8, 300
    q, k, v, beta, d, state = R.inputs(1, T_, 4, H, 48, 64, dtype, 7)
    d = torch.zeros_like(d)
    at = [[(17 * h + 5) % 128, 128 + 16 * h, 256 + h] for h in range(H)]
    for h in range(H):
        d[:, at[h], h] = decay
    got, want = gradients(T, q, k, v, beta, d, state)
    each_head(got, want)
    rows = [torch.cat([g[0, at[h], h].double().cpu() for h in range(H)]) for g in (got, want)]
    # three times 8 single numbers, each a sum of terms of both signs: as single values, of their own root mean square
    assert float((rows[0] - rows[1]).abs().max()) <= R.SINGLE * float(rows[1].square().mean().sqrt())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_mixed(T, dtype):
    """from none to underflow, another for each row; heads of their own strength"""
    q, k, v, beta, d, state = R.inputs(2, 190, 2, 4, 64, 40, dtype, 8)
    d = -torch.tensor([0.1, 3.0, 9.0, 40.0], device="cuda") * torch.rand(d.shape, generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    each_head(*gradients(T, q, k, v, beta, d, state))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 96)])
def test_cleared_is_zero(T, dk, dv, dtype):
    """decay = -inf: nothing crosses the row, and its gradient is 0; those beside it are as they should be"""
    q, k, v, beta, d, state = R.inputs(2, 190, 1, 2, dk, dv, dtype, 9)
    rows = [0, 1, 31, 32, 63, 64, 100, 127, 128, 150, 189]
    d[0, rows], d[1, 40, 1], d[1, 129, 0] = float("-inf"), float("-inf"), float("-inf")
    gone = torch.isinf(d)
    got, want = gradients(T, q, k, v, beta, d, state)
    assert not got[gone].any()
    each_head(got, torch.nan_to_num(want, nan=0.0))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed(T, dtype):
    cuts = [0, 0, 5, 137, 138, 330, 458]
    q, k, v, beta, d, state = R.inputs(1, cuts[-1], 1, 3, 64, 128, dtype, 10, n=len(cuts) - 1)
    d = torch.tensor([-6.0, -12.0, -0.2], device="cuda").expand_as(d).contiguous()
    each_head(*gradients(T, q, k, v, beta, d, state, torch.tensor(cuts, dtype=torch.int32, device="cuda")))
