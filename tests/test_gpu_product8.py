"""The product of 8-bit rows and an 8-bit weight (cssm_scaled_matmul) against float64 of the values they stand for."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import token_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


@pytest.fixture(scope="module")
def Q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import sequence
    return sequence


def make(Q, M, N, K, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + M + 3 * N + 7 * K)
    a = torch.randn((M, K), generator=gen, device="cuda") * torch.exp2(torch.randint(-6, 7, (M, -(-K // 128)), generator=gen,
                    device="cuda").float()).repeat_interleave(128, 1)[:, :K]      # blocks of very different scales
    w = torch.randn((K, N), generator=gen, device="cuda") / K ** 0.5
    return Q.quantize_rows(a), Q.quantize_weight(w), torch.randn((N,), generator=gen, device="cuda")


def values(b, rows):
    M, K = b.values.shape
    return b.values.double() * b.scales.float().double().repeat_interleave(rows, 0)[:M].repeat_interleave(128, 1)[:, :K]


def check(Q, a, w, bias, act, dtype, got=None):
    A, W = values(a, 1), values(w, 128)
    got = Q.scaled_matmul(a, w, bias=bias, act=act, out_dtype=dtype) if got is None else got
    c, mag = A @ W.t(), A.abs() @ W.abs().t()
    if bias is not None:
        c, mag = c + bias.double(), mag + bias.double().abs()
    # exact products (8 mantissa bits), float32 sums: at most one rounding of the running magnitude for each of the
    # K / 4 additions that an instruction may do in turn, and for each 128.  With a bfloat16 output the 8-bit
    # instruction drops what lies 13 bits below the largest of up to 8 products that it adds at once
    K = a.values.shape[1]
    err = (K / 4 + 8) * U * mag + (0 if dtype == F32 else 2.0 ** -10 * mag)
    if act == "silu":
        want = c * torch.sigmoid(c)
    elif act == "gelu":
        want = torch.nn.functional.gelu(c, approximate="tanh")
    else:
        want = c
    if act != "none":
        # slopes are at most 1.13; the sigmoid's exponential carries its argument's error, up to 2 |c| (1 + c^2 / 8) u
        err = 1.13 * err + U * want.abs() * (12 + 4 * c.abs().clamp(max=90) * (1 + c.abs().clamp(max=30) ** 2 / 8))
    assert got.dtype == dtype and got.shape == want.shape
    assert R.off(got, want, err + 1e-30, dtype) <= 1


# part tiles every way; one row and one column; K inside a block, over one, many
SIZES = [(1, 1, 16), (1, 128, 128), (3, 5, 48), (16, 64, 1024), (17, 130, 144), (128, 128, 256), (129, 127, 272),
         (200, 516, 400), (33, 1000, 128), (300, 260, 2048), (1, 4096, 4096), (64, 96, 112), (513, 640, 512)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("act,bias", [("none", False), ("silu", True), ("gelu", True)])
def test_product(Q, M, N, K, dtype, act, bias):
    print_case(test="scaled_matmul", M=M, N=N, K=K, dtype=dtype, act=act)
    a, w, b = make(Q, M, N, K)
    check(Q, a, w, b if bias else None, act, dtype)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 31, 32, 33, 48, 63, 64, 65, 96])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_few_rows(Q, M, dtype):
    a, w, b = make(Q, M, 384, 1152)
    check(Q, a, w, b, "none", dtype)


def test_each_row_alone(Q):
    """A row's result does not depend on the rows beside it, within a launch of one kind."""
    a, w, b = make(Q, 200, 256, 640)
    whole = Q.scaled_matmul(a, w, bias=b, out_dtype=F32)
    part = Q.scaled_matmul(Q.Blocks8(a.values[70:], a.scales[70:]), w, bias=b, out_dtype=F32)
    assert torch.equal(whole[70:], part)


def test_lead_axes_and_odd_output(Q):
    a, w, b = make(Q, 12, 37, 160)
    got = Q.scaled_matmul(Q.Blocks8(a.values.view(3, 4, 160), a.scales.view(3, 4, 2)), w, bias=b, out_dtype=F32)
    assert got.shape == (3, 4, 37)
    check(Q, a, w, b, "none", F32, got.view(12, 37))
    z = Q.scaled_matmul(Q.Blocks8(a.values[:0], a.scales[:0]), w)
    assert z.shape == (0, 37)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_poison_stays_in_its_row_and_column(Q, dtype):
    a, w, _ = make(Q, 140, 140, 256)
    ref = Q.scaled_matmul(a, w, out_dtype=dtype)
    av, wv = a.values.clone(), w.values.clone()
    av.view(torch.uint8)[3, 40] = 0x7f
    wv.view(torch.uint8)[131, 200] = 0xff
    got = Q.scaled_matmul(Q.Blocks8(av, a.scales), Q.Blocks8(wv, w.scales), out_dtype=dtype)
    bad = torch.isnan(got)
    assert bool(bad[3].all()) and bool(bad[:, 131].all())
    keep = torch.ones_like(bad)
    keep[3], keep[:, 131] = False, False
    assert torch.equal(got[keep], ref[keep])


def test_scales_at_the_ends(Q):
    """Exponents from the least to the largest a block can have."""
    a, w, _ = make(Q, 4, 8, 256)
    sa = a.scales.clone()
    sa.view(torch.uint8)[0] = 1          # 2^-126
    sa.view(torch.uint8)[1] = 246
    sw = w.scales.clone()
    sw.view(torch.uint8)[:] = 100
    for dtype in (F32, BF16):
        check(Q, Q.Blocks8(a.values, sa), Q.Blocks8(w.values, sw), None, "none", dtype)


def test_refusals(Q):
    a, w, b = make(Q, 4, 8, 32)
    for args, kw in (((Q.Blocks8(a.values.float(), a.scales), w), {}), ((Q.Blocks8(a.values, a.scales.float()), w), {}),
                     ((Q.Blocks8(a.values[:, :16].contiguous(), a.scales), w), {}), ((a, w), dict(bias=b[:4])),
                     ((a, w), dict(act="tanh")), ((a, w), dict(out_dtype=torch.float16)),
                     ((Q.Blocks8(a.values.cpu(), a.scales), w), {}), ((Q.Blocks8(a.values[:2], a.scales), w), {})):
        with pytest.raises(ValueError):
            Q.scaled_matmul(*args, **kw)
    from cssm_amd._lib import CssmError
    a, w, b = make(Q, 4, 8, 24)
    with pytest.raises(CssmError):
        Q.scaled_matmul(a, w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,K,shift", [(1, 8, 0), (3, 120, 0), (5, 136, 0), (33, 1000, 0), (7, 256, 1), (4, 300, 0)])
def test_quantize_rows_forms(M, K, shift, dtype):
    """8 values a thread where rows are aligned for it, 2 where they are not: the same bytes as the definition"""
    from cssm_amd import sequence as Q
    from tests import token_reference as R
    gen = torch.Generator(device="cuda").manual_seed(M + K)
    flat = torch.randn(M * K + shift, generator=gen, device="cuda") * torch.exp2(
        torch.randint(-40, 40, (M * K + shift,), generator=gen, device="cuda").float())
    x = flat.to(dtype)[shift:].view(M, K)
    if K > 100:
        x[0, 3], x[-1, K - 1] = float("inf"), float("nan")
    q = Q.quantize_rows(x)
    want, e = R.e4m3_blocks(x.double().cpu(), 1, 128)
    got_e = q.scales.view(torch.uint8).cpu().double() - 127
    assert torch.equal(got_e, e.reshape(got_e.shape).double())
    got = q.values.float().double().cpu() * torch.exp2(got_e).repeat_interleave(128, -1)[:, :K]
    assert torch.equal(torch.nan_to_num(got, nan=1e300), torch.nan_to_num(want, nan=1e300))
