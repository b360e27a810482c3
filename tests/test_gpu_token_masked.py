"""Masked rows of the gated recurrence under 8-bit checkpoints: delta at -inf, at the type's lowest value or far below
where softplus is nil, with anything finite in x there, beside rows that are not masked."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import token_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")


@pytest.fixture(scope="module")
def T():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import training
    return training


def make(B, n, C, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 7 * n + C)

    def r(*s, scale=1.0, shift=0.0):
        return shift + scale * torch.randn(s, generator=gen, device="cuda")
    rows = (r(B, n, C).to(dtype), r(B, n, C, shift=-1.0).to(dtype), r(B, n, C).to(dtype), r(B, n, C).to(dtype))
    return (*rows, 0.9 + 0.1 * torch.rand((C,), generator=gen, device="cuda"),
            -2.0 + 2.0 * torch.rand((C,), generator=gen, device="cuda"), r(B, C), r(B, C), gen)


def kept(t, gone):
    """What the checkpoint stands for: the values that are there under their block's exponent, zero in the others' place."""
    return R.e4m3_blocks(torch.where(gone, torch.zeros_like(t), t), 8, 16)[0]


def grads(T, x, d, z, kap, bias, h0, dy, df, **kw):
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, d, z, kap, bias, h0)]
    y, final = T.token_scan_train(leaves[0], leaves[1], leaves[3], leaves[4], z=leaves[2], state=leaves[5], checkpoint="e4m3", **kw)
    return y, final, dict(zip(("dx", "ddelta", "dz", "dkappa", "dbias", "dstate"), torch.autograd.grad((y, final), leaves, (dy, df))))


# a mask by rows, by single values, over whole blocks and whole tiles, and everything
def places(kind, B, n, C, gen):
    m = torch.zeros((B, n, C), dtype=torch.bool, device="cuda")
    if kind == "rows":
        m |= torch.rand((B, n, 1), generator=gen, device="cuda") < 0.3
    elif kind == "values":
        m |= torch.rand((B, n, C), generator=gen, device="cuda") < 0.2
    elif kind == "tail":
        m[0, n // 3:] = True          # a padded batch
        m[-1, : n // 2] = True
    else:
        m[:] = True
    return m


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["rows", "values", "tail", "all"])
@pytest.mark.parametrize("B,n,C", [(2, 300, 36), (1, 40, 7), (3, 131, 64)])
def test_gradients(T, B, n, C, kind, dtype):
    print_case(test="masked rows", B=B, T=n, C=C, kind=kind, dtype=dtype)
    x, d, z, dy, kap, bias, h0, df, gen = make(B, n, C, dtype)
    gone = places(kind, B, n, C, gen)
    low = torch.tensor([-INF, torch.finfo(dtype).min, -1e4, -120.0], device="cuda").to(dtype)
    pick = torch.randint(0, 4, gone.shape, generator=gen, device="cuda")
    d = torch.where(gone, low[pick], d)
    x = torch.where(gone & (pick % 2 == 0), torch.full_like(x, 1e30), x)      # what lies in padding
    y, final, g = grads(T, x, d, z, kap, bias, h0, dy, df)
    x6, d6, z6, dy6, k6, b6, h6, f6 = (t.double().cpu() for t in (x, d, z, dy, kap, bias, h0, df))
    gone = gone.cpu()
    # a masked value has a gain of zero whatever x is: as -inf and 0 there
    x6, d6 = torch.where(gone, 0.0, x6), torch.where(gone, -INF, d6)
    k8 = [kept(x6, gone), torch.where(gone, -INF, kept(d6, gone)), R.e4m3_blocks(z6, 8, 16)[0]]
    w = R.scan(x6, d6, k6, b6, z6, h6, dy6, f6, kept=k8)
    assert R.off(y, w["y"], w["y_err"], dtype) <= 1 and R.off(final, w["final"], w["final_err"]) <= 1
    for name, got in g.items():
        assert R.off(got, w[name], w[name + "_err"], dtype if got.dim() == 3 else F32) <= 1, name


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_packed(T, dtype):
    """masked rows at the starts and ends of packed sequences"""
    lens, C = [70, 0, 9, 130, 41], 20
    x, d, z, dy, kap, bias, _, _, gen = make(1, sum(lens) + 6, C, dtype)
    h0, df = (torch.randn((len(lens), C), generator=gen, device="cuda") for _ in range(2))
    off = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    gone = torch.zeros_like(d, dtype=torch.bool)
    gone[0, off[:-1].long().clamp(max=sum(lens) - 1)] = True
    gone[0, (off[1:].long() - 1)] = True
    gone[0, 75:100] = True
    d = torch.where(gone, torch.full_like(d, -INF), d)
    y, final, g = grads(T, x[0], d[0], z[0], kap, bias, h0, dy[0], df, offsets=off)
    end = sum(lens)
    x6, d6, z6, dy6 = (t[0, :end].double().cpu() for t in (x, d, z, dy))
    m = gone[0, :end].cpu()
    x6 = torch.where(m, 0.0, x6)
    k8 = [kept(x6, m), torch.where(m, -INF, kept(d6, m)), R.e4m3_blocks(z6, 8, 16)[0]]
    at = 0
    for i, n in enumerate(lens):
        s = slice(at, at + n)
        w = R.scan(x6[None, s], d6[None, s], kap.double().cpu(), bias.double().cpu(), z6[None, s], h0[i:i + 1].double().cpu(),
                   dy6[None, s], df[i:i + 1].double().cpu(), kept=[v[None, s] for v in k8], row0=at)
        for name in ("dx", "ddelta", "dz"):
            assert R.off(g[name][None, s], w[name], w[name + "_err"], dtype) <= 1, (i, name)
        assert R.off(g["dstate"][i:i + 1], w["dstate"], w["dstate_err"]) <= 1
        at += n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bias0", [0.0, 150.0, -150.0])
def test_border(T, dtype, bias0):
    """It is delta + bias that decides: values that only the bias masks, or does not, keep their gradients; a value of
    -100 is an ordinary one."""
    B, n, C = 1, 33, 24
    x, d, z, dy, kap, bias, h0, df, gen = make(B, n, C, dtype)
    d = (d.float() - bias0).to(dtype)
    d[:, ::3] = torch.tensor(-100.0 - bias0, dtype=dtype)
    bias = bias + bias0
    u = d.float() + bias
    assert bool((u > -104).all())
    _, _, g = grads(T, x, d, z, kap, bias, h0, dy, df)
    x6, d6, z6, dy6, k6, b6, h6, f6 = (t.double().cpu() for t in (x, d, z, dy, kap, bias, h0, df))
    w = R.scan(x6, d6, k6, b6, z6, h6, dy6, f6, kept=[R.e4m3_blocks(t, 8, 16)[0] for t in (x6, d6, z6)])
    for name, got in g.items():
        assert R.off(got, w[name], w[name + "_err"], dtype if got.dim() == 3 else F32) <= 1, name


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("C", [5, 16])
def test_not_a_number_is_no_mask(T, C, dtype):
    """NaN of either sign and +inf in delta stay not a number in the gradients, beside masked rows; so does an infinite x
    where delta masks it."""
    x, d, z, dy, kap, bias, h0, df, _ = make(4, 24, C, dtype)
    nan = torch.tensor([float("nan")]).to(dtype)
    word = nan.view(torch.int16 if dtype == BF16 else torch.int32)
    signed = (word | torch.iinfo(word.dtype).min).view(dtype)
    assert bool(torch.isnan(signed).all()) and bool(torch.signbit(signed).all())
    d[:, 3] = -INF
    d[0, 10], d[1, 10], d[2, 10] = nan.cuda(), signed.cuda(), INF
    d[3, 10], x[3, 10] = -INF, INF
    _, _, g = grads(T, x, d, z, kap, bias, h0, dy, df)
    assert bool(torch.isnan(g["ddelta"][:, 10]).all()) and bool(torch.isnan(g["dstate"][:2]).all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("checkpoint", ["none", "e4m3"])
@pytest.mark.parametrize("C", [7, 32])
def test_largest_x_under_the_mask(T, C, checkpoint, dtype):
    """x at the type's largest value where delta masks it, with gradients above 1: as with 0 there, in every output"""
    x, d, z, dy, kap, bias, h0, df, gen = make(2, 150, C, dtype, seed=2)
    dy, df = 100 * dy, 100 * df
    gone = places("rows", 2, 150, C, gen)
    gone[:, 3:9] = True
    d = torch.where(gone, torch.full_like(d, -INF), d)
    got = []
    for fill in (torch.finfo(dtype).max, 0.0):
        leaves = [t.detach().clone().requires_grad_(True) for t in (torch.where(gone, torch.full_like(x, fill), x), d, z, kap, bias, h0)]
        y, final = T.token_scan_train(leaves[0], leaves[1], leaves[3], leaves[4], z=leaves[2], state=leaves[5], checkpoint=checkpoint)
        got.append((y, final, *torch.autograd.grad((y, final), leaves, (dy, df))))
    assert not got[0][3][gone].any()
    for a, b in zip(*got):
        assert bool(torch.isfinite(a).all()) and bool((a == b).all())
