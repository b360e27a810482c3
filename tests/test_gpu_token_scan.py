"""The gated recurrence over token sequences (cssm_token_scan, _bwd, _step) against float64 row by row."""
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
    return sequence


def make(B, T, C, dtype, gated=True, state=True, layout="plain", seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 7 * T + C)

    def rows(scale=1.0, shift=0.0):
        return (shift + scale * torch.randn((B, T, C), generator=gen, device="cuda")).to(dtype)
    x, d, z = rows(), rows(1.0, -1.0), rows(1.5)
    if layout == "slices":          # parts of one projection's output, in another order
        p = torch.cat([z, x, d], dim=2)
        z, x, d = p[..., :C], p[..., C:2 * C], p[..., 2 * C:]
    elif layout == "time first":
        x, d, z = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, d, z))
    elif layout == "off by one":    # rows that start off every vector boundary
        x, d, z = (torch.nn.functional.pad(t, (1, 2))[..., 1:-2] for t in (x, d, z))
    kap = 0.9 + 0.1 * torch.rand((C,), generator=gen, device="cuda")
    kap[::5] *= -1.0
    bias = -2.0 + 2.0 * torch.rand((C,), generator=gen, device="cuda")
    h0 = torch.randn((B, C), generator=gen, device="cuda") if state else None
    return x, d, kap, bias, z if gated else None, h0


def dbl(*ts):
    return [None if t is None else t.double().cpu() for t in ts]


# around every border: a row group (8), a tile (128), several; channels with and without vector loads, one lane, a part tile
SIZES = [(1, 1, 1), (2, 7, 3), (3, 8, 64), (1, 9, 16), (2, 127, 20), (1, 128, 130), (2, 129, 68), (1, 1000, 100),
         (3, 260, 33), (1, 2500, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,T,C", SIZES)
@pytest.mark.parametrize("gated,state", [(True, True), (False, False)])
def test_forward(Q, B, T, C, gated, state, dtype):
    print_case(test="token_scan", B=B, T=T, C=C, gated=gated, state=state, dtype=dtype)
    a = make(B, T, C, dtype, gated, state)
    y, final = Q.token_scan(*a[:4], z=a[4], state=a[5])
    w = R.scan(*dbl(*a))
    assert y.dtype == dtype and R.off(y, w["y"], w["y_err"], dtype) <= 1
    assert R.off(final, w["final"], w["final_err"]) <= 1


@pytest.mark.parametrize("layout", ["slices", "time first", "off by one"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,T,C", [(2, 150, 24), (3, 20, 7)])
def test_strides(Q, B, T, C, dtype, layout):
    """Any batch and row strides give the contiguous result: the same values in the same order of operations."""
    print_case(test="token_scan_strides", B=B, T=T, C=C, layout=layout, dtype=dtype)
    a = make(B, T, C, dtype, layout=layout)
    y, final = Q.token_scan(*a[:4], z=a[4], state=a[5])
    c = [t.contiguous() for t in a]
    y2, final2 = Q.token_scan(*c[:4], z=c[4], state=c[5])
    assert torch.equal(y, y2) and torch.equal(final, final2)
    e = [t[:, :1].expand(B, T, C) for t in (a[0], a[1], a[4])]      # one row for every step: stride 0
    y, _ = Q.token_scan(e[0], e[1], *a[2:4], z=e[2], state=a[5])
    y2, _ = Q.token_scan(e[0].contiguous(), e[1].contiguous(), *a[2:4], z=e[2].contiguous(), state=a[5])
    assert torch.equal(y, y2)


def grads_of(fn, inputs, outs):
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in inputs]
    y, final = fn(*leaves)
    return y, final, torch.autograd.grad((y, final), [t for t in leaves if t is not None], outs)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("checkpoint", ["none", "e4m3"])
@pytest.mark.parametrize("B,T,C", SIZES)
@pytest.mark.parametrize("gated,state", [(True, True), (False, False)])
def test_gradients(Q, B, T, C, gated, state, checkpoint, dtype):
    from cssm_amd import training
    print_case(test="token_scan_train", B=B, T=T, C=C, gated=gated, state=state, dtype=dtype, checkpoint=checkpoint)
    a = make(B, T, C, dtype, gated, state)
    gen = torch.Generator(device="cuda").manual_seed(3)
    dy = torch.randn((B, T, C), generator=gen, device="cuda").to(dtype)
    df = torch.randn((B, C), generator=gen, device="cuda")
    y, final, g = grads_of(lambda x, d, k, b, z, h: training.token_scan_train(x, d, k, b, z=z, state=h,
                                                                                checkpoint=checkpoint), a, (dy, df))
    kept = None
    if checkpoint == "e4m3":
        kept = [None if t is None else R.e4m3_blocks(t.double().cpu(), 8, 16)[0] for t in (a[0], a[1], a[4])]
    w = R.scan(*dbl(*a), *dbl(dy, df), kept=kept)
    assert R.off(y, w["y"], w["y_err"], dtype) <= 1
    names = ["dx", "ddelta", "dkappa", "dbias"] + (["dz"] if gated else []) + (["dstate"] if state else [])
    for name, got in zip(names, g):
        assert R.off(got, w[name], w[name + "_err"], dtype if got.dim() == 3 else F32) <= 1, name


def test_gradients_against_differences(Q):
    """Central differences of the float64 recurrence along random directions, against the kernels' gradients."""
    from cssm_amd import training
    a = make(2, 140, 12, F32)
    gen = torch.Generator(device="cuda").manual_seed(4)
    dy, df = torch.randn((2, 140, 12), generator=gen, device="cuda"), torch.randn((2, 12), generator=gen, device="cuda")
    _, _, g = grads_of(lambda x, d, k, b, z, h: training.token_scan_train(x, d, k, b, z=z, state=h), a, (dy, df))
    v = dbl(*a)
    order = [0, 1, 2, 3, 4, 5]

    def loss(p):
        w = R.scan(*p)
        return float((w["y"] * dy.double().cpu()).sum() + (w["final"] * df.double().cpu()).sum())
    for i, got in zip(order, g):
        way = torch.randn(v[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        h = 1e-5
        up, dn = [[t + s * h * way if j == i else t for j, t in enumerate(v)] for s in (1, -1)]
        num = (loss(up) - loss(dn)) / (2 * h)
        ana = float((got.double().cpu() * way).sum())
        # h^2 of the third derivative and 1e-16 / h of the rounding, with the float32 gradient's 1e-5
        assert abs(num - ana) <= 3e-5 * float((got.double().cpu() * way).abs().sum()), i


PACKS = [[5], [0, 0, 3], [1, 1, 1, 0, 2], [127, 1, 128, 0, 130, 7], [300, 0, 0, 41], [64] * 9, [0, 128, 128, 0]]


def packed(lens, tail, C, dtype, gated=True, seed=0):
    a = make(1, sum(lens) + tail, C, dtype, gated, False, seed=seed)
    gen = torch.Generator(device="cuda").manual_seed(5)
    h0 = torch.randn((len(lens), C), generator=gen, device="cuda")
    off = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    return [None if t is None else (t[0] if t.dim() == 3 else t) for t in a[:5]] + [h0], off


@pytest.mark.parametrize("lens", PACKS, ids=str)
@pytest.mark.parametrize("tail,C,dtype", [(0, 20, F32), (3, 64, BF16), (140, 5, F32)])
def test_packed(Q, lens, tail, C, dtype):
    """Sequences one behind the other give what each gives alone; empty ones hand their state through."""
    print_case(test="token_scan_packed", lens=lens, tail=tail, C=C, dtype=dtype)
    from cssm_amd import training
    a, off = packed(lens, tail, C, dtype)
    gen = torch.Generator(device="cuda").manual_seed(6)
    dy = torch.randn(a[0].shape, generator=gen, device="cuda").to(dtype)
    df = torch.randn((len(lens), C), generator=gen, device="cuda")
    y, final, g = grads_of(lambda x, d, k, b, z, h: training.token_scan_train(x, d, k, b, z=z, state=h, offsets=off),
                           a, (dy, df))
    end = sum(lens)
    for t in (y, g[0], g[1], g[4]):
        assert not t[end:].any()
    buf = torch.full_like(y, 7.0)
    y2, final2 = Q.token_scan(*a[:4], z=a[4], state=a[5], offsets=off, out=buf)
    assert y2 is buf and torch.equal(buf[:end], y[:end]) and bool((buf[end:] == 7.0).all()) and torch.equal(final, final2)
    dk, db = torch.zeros(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64)
    ek, eb = torch.zeros_like(dk), torch.zeros_like(db)
    at = 0
    for i, n in enumerate(lens):
        part = [t[None, at:at + n] if t is not None and t.dim() == 2 else t for t in a[:5]] + [a[5][i:i + 1]]
        w = R.scan(*dbl(*part), *dbl(dy[None, at:at + n], df[i:i + 1]))
        for got, name in ((y, "y"), (g[0], "dx"), (g[1], "ddelta"), (g[4], "dz")):
            assert R.off(got[None, at:at + n], w[name], w[name + "_err"], dtype) <= 1, (i, name)
        assert R.off(final[i:i + 1], w["final"], w["final_err"]) <= 1
        assert R.off(g[5][i:i + 1], w["dstate"], w["dstate_err"]) <= 1
        dk += w["dkappa"]
        db += w["dbias"]
        ek += w["dkappa_err"]
        eb += w["dbias_err"]
        at += n
    # the sequences' sums are sums of the same terms: their bounds add
    assert R.off(g[2], dk, ek + 1e-30) <= 1 and R.off(g[3], db, eb + 1e-30) <= 1


def test_packed_checkpoint(Q):
    """8-bit checkpoints of packed rows: blocks and segments count rows of the whole axis, whatever sequence they are of."""
    from cssm_amd import training
    lens, tail, C = [100, 0, 61, 3, 200], 20, 36
    a, off = packed(lens, tail, C, F32)
    a[0][sum(lens):], a[1][sum(lens):] = float("nan"), 1e30     # what lies behind the last sequence is not looked at
    gen = torch.Generator(device="cuda").manual_seed(8)
    dy = torch.randn(a[0].shape, generator=gen, device="cuda")
    df = torch.randn((len(lens), C), generator=gen, device="cuda")
    _, _, g = grads_of(lambda x, d, k, b, z, h: training.token_scan_train(x, d, k, b, z=z, state=h, offsets=off,
                                                                          checkpoint="e4m3"), a, (dy, df))
    end = sum(lens)
    x, d, k, b, z, h0 = dbl(*a)
    kx, kd, kz = (R.e4m3_blocks(t[:end], 8, 16)[0] for t in (x, d, z))
    at = 0
    for i, n in enumerate(lens):
        w = R.scan(x[None, at:at + n], d[None, at:at + n], k, b, z[None, at:at + n], h0[i:i + 1],
                   dy[None, at:at + n].double().cpu(), df[i:i + 1].double().cpu(),
                   kept=[v[None, at:at + n] for v in (kx, kd, kz)], row0=at)
        for got, name in ((g[0], "dx"), (g[1], "ddelta"), (g[4], "dz")):
            assert R.off(got[None, at:at + n], w[name], w[name + "_err"]) <= 1, (i, name)
        assert R.off(g[5][i:i + 1], w["dstate"], w["dstate_err"]) <= 1
        at += n


def test_poison_stays_in_its_sequence(Q):
    """A sequence of NaN and infinities between others leaves them as they are alone, in both directions."""
    from cssm_amd import training
    lens, C = [70, 90, 200], 16
    a, off = packed(lens, 0, C, F32)
    ref = [t.clone() for t in a]
    a[0][70:160] = float("nan")
    a[0][80] = float("inf")
    a[5][1] = float("-inf")
    dy = torch.ones_like(a[0])
    dyb = dy.clone()
    dyb[100] = float("nan")
    df = torch.ones((3, C), device="cuda")

    def fn(x, d, k, b, z, h):
        return training.token_scan_train(x, d, k, b, z=z, state=h, offsets=off)
    y, f, g = grads_of(fn, a, (dyb, df))
    y0, f0, g0 = grads_of(fn, ref, (dy, df))
    keep = torch.ones(360, dtype=torch.bool)
    keep[70:160] = False
    for got, want in ((y, y0), (g[0], g0[0]), (g[1], g0[1]), (g[4], g0[4])):
        assert torch.equal(got[keep], want[keep])
    assert torch.equal(f[[0, 2]], f0[[0, 2]]) and torch.equal(g[5][[0, 2]], g0[5][[0, 2]])


def test_masked_rows(Q):
    """delta = -inf hands the state on times kappa; the type's lowest value does the same."""
    a = list(make(2, 300, 12, BF16, gated=False))
    a[2] = torch.ones_like(a[2])
    a[1][0, 100:220] = float("-inf")
    a[1][1] = torch.finfo(BF16).min
    y, final = Q.token_scan(*a[:4], state=a[5])
    assert torch.equal(y[0, 100:220], y[0, 99:100].expand(120, 12))
    assert torch.equal(final[1], a[5][1])
    from cssm_amd import training
    _, _, g = grads_of(lambda x, d, k, b, z, h: training.token_scan_train(x, d, k, b, z=z, state=h), a,
                       (torch.ones_like(y), torch.ones_like(final)))
    assert not g[0][0, 100:220].any() and not g[1][0, 100:220].any() and not g[0][1].any()
    assert torch.equal(g[4][1], torch.full((12,), 301.0, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,C,gated", [(1, 1, True), (3, 7, False), (16, 1024, True), (130, 36, True)])
def test_step(Q, B, C, gated, dtype):
    """The same bits as a sequence of one row; in place, from slices, over many tokens."""
    print_case(test="token_scan_step", B=B, C=C, gated=gated, dtype=dtype)
    a = make(B, 5, C, dtype, gated, layout="slices")
    state = a[5].clone()
    for t in range(5):
        row = [None if v is None else v[:, t] for v in (a[0], a[1], a[4])]
        one, f1 = Q.token_scan(row[0][:, None], row[1][:, None], *a[2:4], z=None if row[2] is None else row[2][:, None],
                               state=state)
        y, new = Q.token_scan_step(row[0], row[1], *a[2:4], state, z=row[2])
        assert torch.equal(y, one[:, 0]) and torch.equal(new, f1) and new is not state
        y2, same = Q.token_scan_step(row[0], row[1], *a[2:4], state, z=row[2], out_state=state)
        assert same is state and torch.equal(state, new) and torch.equal(y2, y)
    whole, f = Q.token_scan(*a[:4], z=a[4], state=a[5])
    assert torch.equal(f, state) and torch.equal(whole[:, -1], y)


def test_sizes_of_zero(Q):
    from cssm_amd import training
    a = make(2, 0, 6, F32)
    y, f = Q.token_scan(*a[:4], z=a[4], state=a[5])
    assert y.shape == (2, 0, 6) and torch.equal(f, a[5])
    _, _, g = grads_of(lambda x, d, k, b, z, h: training.token_scan_train(x, d, k, b, z=z, state=h, checkpoint="e4m3"),
                       a, (y, f))
    assert torch.equal(g[5], f) and not g[2].any() and not g[3].any()
    for shape in ((0, 9, 6), (2, 9, 0)):
        a = make(*shape, F32)
        y, f = Q.token_scan(*a[:4], z=a[4], state=a[5])
        assert y.shape == shape and f.shape == (shape[0], shape[2])
        _, _, g = grads_of(lambda x, d, k, b, z, h: training.token_scan_train(x, d, k, b, z=z, state=h), a, (y, f))
        assert not g[2].any()
    x = torch.zeros((4, 6), device="cuda")
    y, f = Q.token_scan(x, x, x[0], x[0], offsets=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert not y.any() and f.shape == (0, 6)
    y, _ = Q.token_scan_step(x[:0], x[:0], x[0], x[0], x[:0])
    assert y.shape == (0, 6)


def test_same_bits_twice_and_on_another_stream(Q):
    from cssm_amd import training
    a = make(2, 3000, 48, BF16)
    dy, df = torch.ones_like(a[0]), torch.ones_like(a[5])

    def fn(x, d, k, b, z, h):
        return training.token_scan_train(x, d, k, b, z=z, state=h, checkpoint="e4m3")
    first = grads_of(fn, a, (dy, df))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = grads_of(fn, a, (dy, df))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p, q in zip((*first[:2], *first[2]), (*again[:2], *again[2])):
        assert torch.equal(p, q)


def test_offsets_past_32_bits(Q):
    """Rows that lie more than 2^31 elements apart."""
    step = (1 << 30) + 64
    n = 3
    big = torch.empty(step * (n - 1) + 64, dtype=BF16, device="cuda")
    x = big.as_strided((1, n, 64), (0, step, 1))
    a = make(1, n, 64, BF16)
    x.copy_(a[0])
    y, f = Q.token_scan(x, *a[1:4], z=a[4], state=a[5])
    y2, f2 = Q.token_scan(*a[:4], z=a[4], state=a[5])
    assert torch.equal(y, y2) and torch.equal(f, f2)


def test_graph_of_a_training_pass(Q):
    """Forward and adjoint captured together replay to the eager bits, with eager passes between the replays."""
    sets = [make(2, 700, 32, BF16, seed=s) for s in range(3)]
    offs = None
    dys = [torch.randn((2, 700, 32), device="cuda").to(BF16) for _ in sets]
    static = [t.clone() for t in sets[0]]
    sdy = dys[0].clone()

    def both(a, dy):
        x, d, k, b, z, h = a
        y, f, states, kept, sc = Q.scan_forward(x, d, k, b, z, h, offs, keep_states=True, keep_e4m3=True)
        return (y, f, *Q.scan_backward(None, None, k, b, None, h, offs, states, kept, sc, dy, f, True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(static, sdy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(static, sdy)
    for i in (0, 1, 2, 1, 0):
        want = both(sets[i], dys[i])
        torch.cuda.synchronize()
        for t, v in zip((*static, sdy), (*sets[i], dys[i])):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q), i


def test_kept_values(Q):
    """What the 8-bit checkpoint holds: every bfloat16 value, ties and subnormals among them, zeros, NaN and infinities."""
    v = torch.arange(1 << 16, device="cuda", dtype=torch.int32).to(torch.int16).view(BF16).view(1, 4096, 16)
    v = v[:, torch.randperm(4096, generator=torch.Generator().manual_seed(0)).to("cuda")].contiguous()
    v[:, :8] = 0.0
    flat = torch.zeros_like(v)
    k = torch.ones(16, device="cuda")
    _, _, _, kept, sc = Q.scan_forward(v, flat, k, k, keep_e4m3=True)
    want, e = R.e4m3_blocks(v[0].double().cpu(), 8, 16)
    assert torch.equal(sc[0, 0].cpu().int() - 127, e.int())
    got = kept[0, 0].view(torch.float8_e4m3fn).float().double().cpu() * torch.exp2(e.double()).repeat_interleave(8, 0).repeat_interleave(16, 1)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_refusals(Q):
    a = make(2, 6, 8, F32)
    x, d, k, b, z, h = a

    def bad(*args, **kw):
        with pytest.raises(ValueError):
            Q.token_scan(*args, **kw)
    bad(x.cpu(), d, k, b)
    bad(x[0], d[0], k, b)
    bad(x, d[:, :5], k, b)
    bad(x, d.bfloat16(), k, b)
    bad(x.half(), d.half(), k, b)
    bad(x.transpose(1, 2).contiguous().transpose(1, 2), d, k, b)
    bad(x, d, k[:7], b)
    bad(x, d, k.bfloat16(), b)
    bad(x, d, k, b, state=h[:1])
    bad(x, d, k, b, z=z[..., :4])
    bad(x, d, k, b, out=torch.empty_like(x[:, :3]))
    bad(x, d, k, b, offsets=torch.zeros(2, dtype=torch.int32, device="cuda"))
    bad(x[0], d[0], k, b, offsets=torch.zeros(2, dtype=torch.int64, device="cuda"))
    bad(x[0], d[0], k, b, offsets=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        Q.token_scan_step(x, d, k, b, h)
    with pytest.raises(ValueError):
        Q.token_scan_step(x[0], d[0], k, b, h[:1])
    from cssm_amd import training
    with pytest.raises(ValueError):
        training.token_scan_train(x, d, k, b, checkpoint="int8")
