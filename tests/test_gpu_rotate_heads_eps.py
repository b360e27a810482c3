"""The heads' norm without eps: lanes that have no head take no part in the weights' gradients (sizes where a wave's heads do
not divide the row's), and eps of any size gives the gradient of the definition."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests.test_gpu_rotate_heads import make, off, plain  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def T():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import training
    return training


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("norm", ["rms", "l2"])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("lead,Hq,Hk,D,sections", [((5,), 3, 1, 64, [32]), ((1,), 1, 1, 16, None), ((9,), 5, 2, 50, [25]), ((40,), 16, 4, 128, [64]),
                                                   ((2, 3), 1, 7, 30, [10, 5])])
def test_weights(T, lead, Hq, Hk, D, sections, eps, norm, dtype):
    from cssm_amd import sequence as Q
    print_case(test="rotate heads eps", lead=lead, Hq=Hq, Hk=Hk, D=D, eps=eps, norm=norm, dtype=str(dtype))
    q, k, positions, table, (wq, wk) = make(Q, lead, Hq, Hk, D, sections, dtype, True, D + Hq)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = T.rotate_heads_train(q, k, positions, table, wq, wk, norm, eps, "halves")
    gq, gk = torch.randn_like(yq), torch.randn_like(yk)
    grads = torch.autograd.grad((yq, yk), leaves, (gq, gk))
    for x, w, y, g, dx, dw in ((q, wq, yq, gq, grads[0], grads[2]), (k, wk, yk, gk, grads[1], grads[3])):
        want = plain(x, w, positions, table, norm, eps, "halves", g)
        assert off(y, want["y"], want["y_err"]) <= 1
        assert off(dx, want["dx"], want["dx_err"]) <= 1
        assert off(dw, want["dw"], want["dw_err"]) <= 1
