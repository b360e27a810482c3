"""More of the product of 8-bit rows and an 8-bit weight: sizes that reach every kernel it is launched as, in integers and
so exactly; inner sizes of zero."""
import pytest

from tests.gpu_util import print_case
from tests.test_gpu_product8 import check, make

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def Q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import sequence
    return sequence


def test_inner_size_of_zero(Q):
    """refused by the entry point as any K it does not take, not by a division"""
    from cssm_amd._lib import CssmError
    a = Q.quantize_rows(torch.empty((4, 0), device="cuda"))
    assert a.values.shape == (4, 0) and a.scales.shape == (4, 0)
    w = Q.Blocks8(torch.empty((8, 0), dtype=torch.float8_e4m3fn, device="cuda"),
                  torch.empty((1, 0), dtype=torch.float8_e8m0fnu, device="cuda"))
    with pytest.raises(CssmError):
        Q.scaled_matmul(a, w)


def over(n, d):
    return -(-n // d)


def form(M, N):
    """the kernel by its launch rule: few rows (16, 32 columns a workgroup), tiles of 256 or 128"""
    if M <= 64 or (M <= 128 and over(N, 128) < 64):
        return "16 rows" if M <= 16 and N < 8192 else "16 rows wide" if M <= 16 else "32 rows" if M <= 32 else "64 rows"
    return "256 tiles" if over(M, 256) * over(N, 256) >= 192 else "128 tiles"


# both sides of each border of the launch rule; part tiles both ways, whole 16-byte pieces of the output and not; K under and
# over a block, and past the 64 blocks whose exponents a tile holds at a time, with a part block behind them
SIZES = [(3100, 4100, 272, "256 tiles"), (3300, 3848, 144, "256 tiles"), (3073, 4096, 128, "256 tiles"),
         (257, 24500, 400, "256 tiles"), (2900, 3900, 8336, "256 tiles"), (130, 140, 8336, "128 tiles"), (300, 264, 16400, "128 tiles"),
         (129, 4097, 8192, "128 tiles"), (100, 8200, 272, "128 tiles"), (100, 8000, 144, "64 rows"), (65, 130, 8336, "64 rows"),
         (64, 8193, 48, "64 rows"), (33, 70, 272, "64 rows"), (32, 8200, 400, "32 rows"), (17, 50, 8336, "32 rows"),
         (16, 8192, 144, "16 rows wide"), (5, 8200, 400, "16 rows wide"), (1, 8223, 8336, "16 rows wide"),
         (16, 8191, 144, "16 rows"), (7, 33, 16400, "16 rows")]


def test_every_form_is_reached():
    assert {k for *_, k in SIZES} == {"16 rows", "16 rows wide", "32 rows", "64 rows", "128 tiles", "256 tiles"}
    for M, N, K, k in SIZES:
        assert form(M, N) == k and K % 16 == 0


def integers(M, N, K):
    """Values in -2 .. 2 and powers of two from 1 to 8, another one for each block: every product, and every sum of them up
    to 2^24, is exact in any order, and none is 13 bits below another of its block."""
    gen = torch.Generator(device="cuda").manual_seed(M + 3 * N + 7 * K)

    def draw(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda")
    nk = over(K, 128)
    a, w = draw(-2, 3, M, K).float(), draw(-2, 3, N, K).float()
    sa, sw = torch.exp2(draw(0, 4, M, nk).float()), torch.exp2(draw(0, 4, over(N, 128), nk).float())
    A = a * sa.repeat_interleave(128, 1)[:, :K]
    W = w * sw.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    assert 4 * K * 64 < 1 << 24
    return a, sa, w, sw, A.double() @ W.double().t()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,kind", SIZES)
def test_integers(Q, M, N, K, kind, dtype):
    """exact, and so equal: every row, column, block and exponent in its place"""
    print_case(test="scaled_matmul integers", M=M, N=N, K=K, kind=kind, dtype=dtype)
    a, sa, w, sw, want = integers(M, N, K)
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    assert float(want.abs().max()) < 1 << 24
    got = Q.scaled_matmul(Q.Blocks8(a.to(f8), sa.to(e8)), Q.Blocks8(w.to(f8), sw.to(e8)), out_dtype=dtype)
    assert torch.equal(got, want.float().to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(3100, 4100, 272), (16, 8200, 400), (130, 140, 8336)])
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_normal_values(Q, M, N, K, act, dtype):
    print_case(test="scaled_matmul large", M=M, N=N, K=K, act=act, dtype=dtype)
    a, w, b = make(Q, M, N, K)
    check(Q, a, w, b, act, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(16, 40, 688), (40, 140, 688), (150, 260, 688)])
def test_each_block_alone(Q, M, N, K, dtype):
    """One block of 128 at a time, zeros in the others under exponents of their own, so that the bound is of that block's
    products: float32 roundings of 128 of them and, in bfloat16, what the instruction drops (2^-13 of the largest of up to
    8 that it adds at once, for each: under 2^-10 of their sum of magnitudes) and the output's half step."""
    print_case(test="scaled_matmul blocks", M=M, N=N, K=K, dtype=dtype)
    gen = torch.Generator(device="cuda").manual_seed(K)
    nk = over(K, 128)
    a, w = (torch.randn((n, K), generator=gen, device="cuda").to(torch.float8_e4m3fn) for n in (M, N))
    sa, sw = (torch.randint(100, 150, (n, nk), generator=gen, device="cuda").to(torch.uint8) for n in (M, over(N, 128)))
    W = w.double() * torch.exp2(sw.double() - 127).repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    for b in range(nk):
        one = torch.zeros((M, K), device="cuda")
        one[:, b * 128:(b + 1) * 128] = a.float()[:, b * 128:(b + 1) * 128]
        A = one.double() * torch.exp2(sa.double() - 127).repeat_interleave(128, 1)[:, :K]
        want, mag = A @ W.t(), A.abs() @ W.abs().t()
        got = Q.scaled_matmul(Q.Blocks8(one.to(torch.float8_e4m3fn), sa.view(torch.float8_e8m0fnu)),
                              Q.Blocks8(w, sw.view(torch.float8_e8m0fnu)), out_dtype=dtype)
        u = 2.0 ** -24
        lim = 128 * u * mag + (0 if dtype == F32 else 2.0 ** -10 * mag * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs())
        assert bool(((got.double() - want).abs() <= lim).all()), b


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(3, 40, 16400), (20, 8200, 8336), (40, 140, 16400), (150, 260, 16400), (3100, 4100, 2064)])
def test_large_sums(Q, M, N, K, dtype):
    """Sums near 2^20 of products down to 1, taken away again by the bias: what the accumulator holds is float32, whatever
    the instruction drops among the products that it adds at once."""
    print_case(test="scaled_matmul large sums", M=M, N=N, K=K, dtype=dtype)
    gen = torch.Generator(device="cuda").manual_seed(N + K)
    nk = over(K, 128)
    a, w = (torch.randint(1, 5, (n, K), generator=gen, device="cuda").float() for n in (1, N))
    sa, sw = (torch.exp2(torch.randint(0, 3, (n, nk), generator=gen, device="cuda").float()) for n in (1, over(N, 128)))
    want = ((a * sa.repeat_interleave(128, 1)[:, :K]).double()
            @ (w * sw.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]).double().t())
    assert float(want.max()) < 1 << 24
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    got = Q.scaled_matmul(Q.Blocks8(a.expand(M, K).contiguous().to(f8), sa.expand(M, nk).contiguous().to(e8)),
                          Q.Blocks8(w.to(f8), sw.to(e8)), bias=-want[0].float(), out_dtype=dtype)
    assert not got.any()
