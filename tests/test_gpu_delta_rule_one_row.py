"""Sequences of one row, whose row stride means nothing: any number that it holds gives the bits of the contiguous call."""
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


def apart(t, stride):
    """(B, 1, H, D) with another batch than the contiguous one and this row stride"""
    B, _, H, D = t.shape
    room = torch.zeros((B, H * D + 32), dtype=t.dtype, device=t.device)
    out = room.as_strided((B, 1, H, D), (H * D + 32, stride, D, 1))
    out.copy_(t)
    return out


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("stride", [0, 1, 8, 1 << 28, 1 << 30, 1 << 31, 1 << 32, (1 << 40) + 8])
@pytest.mark.parametrize("Hk,Hv,dk,dv", [(2, 2, 64, 64), (1, 2, 128, 40)])
def test_stride_is_not_used(T, Hk, Hv, dk, dv, stride, dtype):
    print_case(test="delta rule one row", Hk=Hk, Hv=Hv, dk=dk, dv=dv, stride=stride, dtype=str(dtype))
    args = R.inputs(3, 1, Hk, Hv, dk, dv, dtype, 5)
    gy = torch.randn_like(args[2])

    def run(args, gy):
        args = [t.requires_grad_() for t in args]
        y, final = T.delta_rule_train(*args[:4], decay=args[4], state=args[5])
        return (y, final, *torch.autograd.grad(y, args, gy))
    want = run([t.detach() for t in args], gy)
    got = run([*(apart(t.detach(), stride) for t in args[:3]), *(t.detach() for t in args[3:])], apart(gy, stride))
    for g, w in zip(got, want):
        assert torch.equal(g, w)
