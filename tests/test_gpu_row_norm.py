"""The root-mean-square norm with the residual's addition and 8-bit output (cssm_rms_norm, _bwd) and the 8-bit operands
(cssm_quantize_rows, cssm_quantize_weight) against float64."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import token_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
EPS, U = 1e-6, 2.0 ** -24


@pytest.fixture(scope="module")
def Q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import sequence
    return sequence


def make(M, C, dtype, residual, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(M + 3 * C)

    def rows():
        t = torch.randn((M * C + offset,), generator=gen, device="cuda") * 3.0
        return t.to(dtype)[offset:].view(M, C)
    return rows(), 1.0 + 0.5 * torch.randn((C,), generator=gen, device="cuda"), rows() if residual else None


def exact(x, w, r):
    s = x if r is None else (x.float() + r.float()).to(x.dtype)
    v = s.double()
    n = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    return s, n, n * w.double()


# one lane, part rows, every register kernel's smallest and largest width, the looped kernel; off a vector boundary
WIDTHS = [(1, 1, 0), (5, 7, 0), (3, 8, 0), (9, 64, 0), (77, 130, 0), (6, 512, 1), (5, 520, 0), (4, 1024, 0), (3, 2040, 0),
          (3, 2056, 0), (2, 4096, 0), (2, 8192, 0), (2, 8200, 0), (1, 10007, 0), (1030, 96, 0), (4200, 32, 0)]


@pytest.mark.parametrize("M,C,offset", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("residual", [True, False])
def test_forward(Q, M, C, offset, dtype, residual):
    print_case(test="rms_norm", M=M, C=C, offset=offset, dtype=dtype, residual=residual)
    x, w, r = make(M, C, dtype, residual, offset)
    s, _, want = exact(x, w, r)
    y, s1 = Q.rms_norm(x, w, residual=r, eps=EPS)
    assert torch.equal(s, s1)          # one rounding of an exact sum
    # the squares' sum (64 in a row, then lanes), the root and two products: C is at most 2^14, half the sum's error
    assert R.off(y, want, 24 * U * want.abs(), dtype) <= 1
    q, s2 = Q.rms_norm(x, w, residual=r, eps=EPS, out="e4m3")
    assert torch.equal(s, s2) and q.values.shape == x.shape and q.scales.shape == (M, -(-C // 128))
    got = q.values.double() * q.scales.float().double().repeat_interleave(128, 1)[:, :C]
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the block's power of two below 2^-6 of it
    lim = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * q.scales.float().double().repeat_interleave(128, 1)[:, :C])
    assert bool(((got - want).abs() <= lim * (1 + 2.0 ** -10)).all())
    top = torch.nn.functional.pad(want.abs(), (0, -C % 128)).view(M, -1, 128).amax(-1)
    sc = q.scales.float().double()
    assert bool(((top <= 448 * sc * (1 + 24 * U)) & ((top > 224 * sc * (1 - 24 * U)) | (top == 0))).all())


@pytest.mark.parametrize("M,C,offset", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("residual", [True, False])
def test_gradients(Q, M, C, offset, dtype, residual):
    from cssm_amd import training
    print_case(test="rms_norm_train", M=M, C=C, offset=offset, dtype=dtype, residual=residual)
    x, w, r = make(M, C, dtype, residual, offset)
    gen = torch.Generator(device="cuda").manual_seed(1)
    dy, ds = (torch.randn((M, C), generator=gen, device="cuda").to(dtype) for _ in range(2))
    s, n, want = exact(x, w, r)
    leaves = [t.requires_grad_(True) for t in (x, w, r) if t is not None]
    y, s1 = training.rms_norm_train(x, w, residual=r, eps=EPS)
    g = torch.autograd.grad((y, s1) if residual else y, leaves, (dy, ds) if residual else dy)
    assert R.off(y, want, 24 * U * want.abs(), dtype) <= 1
    t = dy.double() * w.detach().double()
    rstd = 1 / torch.sqrt((s.detach().double() ** 2).mean(-1, keepdim=True) + EPS)
    mean = (t * n).mean(-1, keepdim=True)
    dx = rstd * (t - n * mean)
    # two sums over a row, each off by at most 24 roundings of the sum of its terms' magnitudes (64 in order, then a tree)
    err = 32 * U * rstd * (t.abs() + n.abs() * (t * n).abs().mean(-1, keepdim=True) * 2)
    if residual:
        dx, err = dx + ds.double(), err + U * ds.double().abs()
        assert torch.equal(g[0], g[2])
    assert R.off(g[0], dx, err, dtype) <= 1
    dw = (dy.double() * n).sum(0)
    # a workgroup's rows in order (at most 8 of these sizes), then float64
    assert R.off(g[1], dw, 48 * U * (dy.double() * n).abs().sum(0)) <= 1


def test_gradient_against_differences(Q):
    from cssm_amd import training
    x, w, r = make(6, 40, F32, True)
    way = [torch.randn_like(t).double() for t in (x, w, r)]
    dy, ds = torch.randn_like(x), torch.randn_like(x)
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    y, s = training.rms_norm_train(*leaves[:2], residual=r, eps=EPS)
    g = torch.autograd.grad((y, s), leaves, (dy, ds))

    def loss(p):
        v = p[0] + p[2]
        n = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * p[1]
        return float((n * dy.double()).sum() + (v * ds.double()).sum())
    base = [t.detach().double() for t in (x, w, r)]
    for i in range(3):
        up, dn = ([b + c * 1e-5 * way[i] if j == i else b for j, b in enumerate(base)] for c in (1, -1))
        num = (loss(up) - loss(dn)) / 2e-5
        terms = g[i].double() * way[i]
        assert abs(num - float(terms.sum())) <= 1e-5 * float(terms.abs().sum())


@pytest.mark.parametrize("M", [1, 1023, 1025, 5000])
def test_many_rows(Q, M):
    """dweight over more rows than workgroups; the same bits twice."""
    x, w, _ = make(M, 24, F32, False)
    dy = torch.ones_like(x)
    _, n, _ = exact(x, w, None)
    dx, dw = Q.rms_norm_backward(dy, None, x, w, EPS)
    assert R.off(dw, n.sum(0), 64 * U * n.abs().sum(0)) <= 1
    dx2, dw2 = Q.rms_norm_backward(dy, None, x, w, EPS)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


def test_rows_of_zeros_and_poison(Q):
    """A row of zeros is zeros (scale 1); a row with a NaN or an infinity is not a number where it has to be, and
    leaves the others alone."""
    for C in (64, 130, 8200):
        x, w, _ = make(4, C, F32, False)
        ref, _ = Q.rms_norm(x, w, eps=EPS, out="e4m3")
        p = x.clone()
        p[0] = 0.0
        p[1, 3] = float("nan")
        p[2, 5] = float("inf")
        q, _ = Q.rms_norm(p, w, eps=EPS, out="e4m3")
        v, sc = q.values.float(), q.scales.float()
        assert not v[0].any() and bool((sc[0] == 1).all())
        assert bool(torch.isnan(v[1]).all())
        assert bool(torch.isnan(v[2, 5])) and not v[2, :5].any()
        assert torch.equal(v[3], ref.values.float()[3]) and torch.equal(sc[3], ref.scales.float()[3])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 127), (7, 128), (2, 129), (5, 1000)])
def test_quantize_rows(Q, M, K, dtype):
    gen = torch.Generator(device="cuda").manual_seed(K)
    x = (torch.randn((M, K), generator=gen, device="cuda") * torch.exp2(torch.randint(-40, 40, (M, 1), generator=gen, device="cuda").float())).to(dtype)
    x[0, 0] = 0.0
    q = Q.quantize_rows(x)
    want, e = R.e4m3_blocks(x.double().cpu(), 1, 128)
    assert torch.equal(q.scales.float().double().cpu(), torch.exp2(e.double()))
    got = q.values.float().double().cpu() * torch.exp2(e.double()).repeat_interleave(128, 1)[:, :K]
    assert torch.equal(got, want)


def test_quantize_special_values(Q):
    """Extremes of the range, blocks of zeros, NaN and infinities beside finite values."""
    x = torch.zeros((6, 128), device="cuda")
    x[0, :3] = torch.tensor([3.4e38, -1.0, float("inf")])
    x[1, :2] = torch.tensor([1e-45, float("nan")])
    x[2, :2] = torch.tensor([2.0 ** -126, -2.0 ** -130])
    x[3, :3] = torch.tensor([448.0, 1.0, -0.0])
    x[4, :3] = torch.tensor([448.0001, 1.0, float("-inf")])
    q = Q.quantize_rows(x)
    want, e = R.e4m3_blocks(x.double().cpu(), 1, 128)
    assert torch.equal(q.scales.float().double().cpu(), torch.exp2(e.double()))
    got = q.values.float().double().cpu() * torch.exp2(e.double())
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("K,N", [(1, 1), (16, 5), (128, 128), (130, 257), (400, 96)])
def test_quantize_weight(Q, K, N):
    gen = torch.Generator(device="cuda").manual_seed(K + N)
    w = torch.randn((K, N), generator=gen, device="cuda") * 0.02
    q = Q.quantize_weight(w)
    want, e = R.e4m3_blocks(w.t().double().cpu(), 128, 128)
    sc = torch.exp2(e.double())
    assert torch.equal(q.scales.float().double().cpu(), sc)
    got = q.values.float().double().cpu() * sc.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    assert torch.equal(got, want)


def test_sizes_of_zero(Q):
    w = torch.ones(8, device="cuda")
    y, s = Q.rms_norm(torch.empty((0, 8), device="cuda"), w)
    assert y.shape == (0, 8)
    dx, dw = Q.rms_norm_backward(y, None, y, w, EPS)
    assert dx.shape == (0, 8) and not dw.any()
    assert Q.quantize_rows(y).scales.shape == (0, 1)


def test_refusals(Q):
    x, w, r = make(4, 8, F32, True)
    for args, kw in (((x.cpu(), w), {}), ((x.half(), w), {}), ((x, w[:4]), {}), ((x, w.bfloat16()), {}),
                     ((x[:, ::2], w[::2].contiguous()), {}), ((x, w), dict(residual=r[:2])),
                     ((x, w), dict(residual=r.bfloat16())), ((x, w), dict(out="int8"))):
        with pytest.raises(ValueError):
            Q.rms_norm(*args, **kw)
    from cssm_amd._lib import CssmError
    with pytest.raises(CssmError):
        Q.rms_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError):
        Q.quantize_rows(x.half())
    with pytest.raises(ValueError):
        Q.quantize_weight(x.t())
    with pytest.raises(ValueError):
        Q.quantize_weight(x.bfloat16())
