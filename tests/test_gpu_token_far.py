"""The gated recurrence over sequences whose first and last rows lie more than 2^32 bytes apart, in the kernels that take
several channels a thread and so count a tile's rows in 32 bits, against float64 row by row."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import token_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def Q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import sequence
    yield sequence
    torch.cuda.empty_cache()


def dbl(*ts):
    return [None if t is None else t.double().cpu() for t in ts]


def params(C, gen):
    return (0.9 + 0.1 * torch.rand((C,), generator=gen, device="cuda"),
            -2.0 + 2.0 * torch.rand((C,), generator=gen, device="cuda"))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,step,T", [(BF16, 1 << 22, 700), (F32, 1 << 22, 400), (BF16, 3 << 20, 800)])
def test_rows_far_apart(Q, dtype, step, T, packed):
    """x, delta, z and dy as slices of rows of 2^22 values, the widest that the vector loads take: forward and adjoint,
    every row of every tile."""
    print_case(test="rows far apart", dtype=dtype, step=step, T=T, packed=packed)
    from cssm_amd import training
    C = 64
    gen = torch.Generator(device="cuda").manual_seed(T)
    buf = torch.empty((T - 1) * step + 4 * C, dtype=dtype, device="cuda")
    part = []
    for i in range(4):
        v = buf.as_strided((1, T, C), (T * step, step, 1), i * C)
        v.copy_((torch.randn((1, T, C), generator=gen, device="cuda") - (1.0 if i == 1 else 0.0)).to(dtype))
        part.append(v)
    assert (T - 1) * step * buf.element_size() >= 1 << 32
    kap, bias = params(C, gen)
    lens = [37, 0, T - 37 - 5] if packed else [T]
    h0 = torch.randn((len(lens), C), generator=gen, device="cuda")
    df = torch.randn((len(lens), C), generator=gen, device="cuda")
    off = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32) if packed else None
    x, d, z, dy = ([v[0] for v in part] if packed else part)
    leaves = [t.detach().requires_grad_(True) for t in (x, d, z, h0)]
    y, final = training.token_scan_train(leaves[0], leaves[1], kap, bias, z=leaves[2], state=leaves[3], offsets=off)
    g = torch.autograd.grad((y, final), leaves, (dy, df))
    at = 0
    for i, n in enumerate(lens):
        rows = [(v[at:at + n][None] if packed else v) for v in (x, d, z, dy, y, g[0], g[1], g[2])]
        xs, ds, zs, dys = dbl(*rows[:4])
        w = R.scan(xs, ds, *dbl(kap, bias), zs, *dbl(h0[i:i + 1]), dys, *dbl(df[i:i + 1]))
        for got, name in zip(rows[4:], ("y", "dx", "ddelta", "dz")):
            assert R.off(got, w[name], w[name + "_err"], dtype) <= 1, (i, name)
        assert R.off(final[i:i + 1], w["final"], w["final_err"]) <= 1
        assert R.off(g[3][i:i + 1], w["dstate"], w["dstate_err"]) <= 1
        at += n


def test_long_checkpoint(Q):
    """2^20 + 64 rows of 4096 channels: the planes of the 8-bit checkpoint have more than 2^32 values each.  The first
    tile, the one whose last rows a wrapped end would take from the wrong place, against float64; only its rows have a
    gradient of y, so that nothing comes from behind."""
    C, T, n = 4096, (1 << 20) + 64, 128
    print_case(test="long checkpoint", C=C, T=T)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((1, 1, C), generator=gen, device="cuda").to(BF16).expand(1, T, C)
    d = torch.empty((1, T, C), dtype=BF16, device="cuda").normal_(-1.0, 1.0, generator=gen)
    kap, bias = params(C, gen)
    y, final, states, kept, sc = Q.scan_forward(x, d, kap, bias, keep_states=True, keep_e4m3=True)
    w = R.scan(*dbl(x[:, :n], d[:, :n], kap, bias))
    assert R.off(y[:, :n], w["y"], w["y_err"], BF16) <= 1
    del y
    dy = torch.zeros((1, T, C), dtype=BF16, device="cuda")
    dy[:, :n] = torch.randn((1, n, C), generator=gen, device="cuda").to(BF16)
    dx, dd, _, dk, db, dh0 = Q.scan_backward(None, None, kap, bias, None, None, None, states, kept, sc, dy, None, False)
    k8 = [R.e4m3_blocks(t[:, :n].double().cpu(), 8, 16)[0] for t in (x, d)]
    w = R.scan(*dbl(x[:, :n], d[:, :n], kap, bias), dy=dy[:, :n].double().cpu(), kept=[*k8, None])
    for got, name in ((dx[:, :n], "dx"), (dd[:, :n], "ddelta")):
        assert R.off(got, w[name], w[name + "_err"], BF16) <= 1, name
    assert not dx[:, n:].any() and not dd[:, n:].any()
    assert R.off(dk, w["dkappa"], w["dkappa_err"]) <= 1 and R.off(db, w["dbias"], w["dbias_err"]) <= 1
    assert R.off(dh0, w["dstate"], w["dstate_err"]) <= 1
