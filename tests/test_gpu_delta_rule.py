"""The gated delta rule over token sequences against float64, token by token: lengths and widths off every block, shared
heads, packed and strided rows, masked rows, single tokens, other streams and captured calls."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import delta_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def Q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import sequence
    return sequence


SIZES = [(1, 1, 1, 1, 1, 1), (2, 31, 1, 2, 16, 16), (1, 32, 2, 2, 64, 64), (2, 33, 1, 1, 128, 128), (1, 64, 3, 3, 40, 50),
         (3, 65, 2, 4, 65, 100), (1, 127, 1, 3, 5, 33), (2, 200, 2, 2, 128, 128), (1, 130, 1, 1, 127, 1), (1, 129, 2, 6, 32, 128)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,Hk,Hv,dk,dv", SIZES)
def test_sequences(Q, B, T, Hk, Hv, dk, dv, dtype):
    print_case(test="delta rule", B=B, T=T, Hk=Hk, Hv=Hv, dk=dk, dv=dv, dtype=str(dtype))
    q, k, v, beta, decay, state = R.inputs(B, T, Hk, Hv, dk, dv, dtype, B * T + dk)
    y, final = Q.delta_rule(q, k, v, beta, decay, state)
    want = R.whole(q, k, v, beta, decay, state)
    assert y.dtype == dtype and R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_defaults(Q, dtype):
    """no decay, no state, another scale"""
    q, k, v, beta, _, _ = R.inputs(2, 70, 2, 4, 48, 24, dtype, 3)
    y, final = Q.delta_rule(q, k, v, beta, scale=0.5)
    want = R.whole(q, k, v, beta, scale=0.5)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_rows(Q, dtype):
    q, k, v, beta, decay, state = R.inputs(2, 0, 1, 2, 16, 8, dtype, 4)
    y, final = Q.delta_rule(q, k, v, beta, decay, state)
    assert y.shape == v.shape and torch.equal(final, state)
    assert not Q.delta_rule(q, k, v, beta, decay)[1].any()
    q, k, v, beta, decay, state = R.inputs(0, 9, 1, 2, 16, 8, dtype, 4)
    y, final = Q.delta_rule(q, k, v, beta, decay, state)
    assert y.shape == v.shape and final.shape == state.shape


@pytest.mark.parametrize("beta", [1.0, 2.0])
def test_equal_keys(Q, beta):
    """every key the same: with beta = 1 each row replaces what the one before wrote, with 2 it reflects.  There the rows'
    errors are not independent, as the tolerance has it: k.k is the same number in all of them, with the same rounding of u =
    2^-24 at least, and nothing damps the state along k.  A reflection 1 - 2 k.k is off by 2 u of it, 100 rows by 200 u."""
    q, k, v, b, decay, state = R.inputs(1, 100, 1, 1, 64, 32, F32, 5)
    k = k[:, :1].expand_as(k).contiguous()
    b = torch.full_like(b, beta)
    y, final = Q.delta_rule(q, k, v, b, None, state)
    want = R.whole(q, k, v, b, None, state)
    more = 200 * 2.0 ** -24 / R.LENGTH if beta == 2 else 1
    assert R.off(y, want["y"]) <= more and R.off(final, want["final"]) <= more


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_correlated_keys(Q, dtype):
    q, k, v, b, decay, state = R.inputs(1, 260, 1, 2, 128, 64, dtype, 6, correlated=True)
    y, final = Q.delta_rule(q, k, v, b, decay, state)
    want = R.whole(q, k, v, b, decay, state)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1


OFFSETS = [[0, 5, 5, 40, 104, 150], [0, 0, 0, 1, 2, 34, 98, 98], [0, 32, 64, 96], [0, 150], [0, 0]]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offsets", OFFSETS)
@pytest.mark.parametrize("tail", [0, 7, 50])
def test_packed(Q, offsets, tail, dtype):
    T, n = offsets[-1] + tail, len(offsets) - 1
    print_case(test="delta rule packed", offsets=offsets, tail=tail, dtype=str(dtype))
    q, k, v, beta, decay, state = R.inputs(1, T, 2, 4, 40, 24, dtype, T + n, n=n)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    # what lies behind the last sequence is not read
    for t in (q, k, v, beta, decay):
        t[offsets[-1]:] = float("nan")
    want = R.whole(q, k, v, beta, decay, state, off)
    y, final = Q.delta_rule(q, k, v, beta, decay, state, offsets=off)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1
    assert not y[offsets[-1]:].any()
    out = torch.full_like(v, 7.0)
    y2, _ = Q.delta_rule(q, k, v, beta, decay, state, offsets=off, out=out)
    assert y2 is out and torch.equal(out[:offsets[-1]], y[:offsets[-1]]) and bool((out[offsets[-1]:] == 7).all())


@pytest.mark.parametrize("n", [63, 64, 65, 200])
def test_many_packed(Q, n):
    """sequences taken by their length up to 64 of them, in their order from there"""
    gen = torch.Generator().manual_seed(n)
    cuts = torch.randint(0, 700, (n - 1,), generator=gen).sort().values.tolist()
    off = torch.tensor([0] + cuts + [700], dtype=torch.int32, device="cuda")
    q, k, v, beta, decay, state = R.inputs(1, 705, 1, 2, 16, 8, F32, n, n=n)
    want = R.whole(q, k, v, beta, decay, state, off)
    y, final = Q.delta_rule(q, k, v, beta, decay, state, offsets=off)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1


def test_packed_as_alone(Q):
    """each packed sequence as it is by itself, bit for bit"""
    q, k, v, beta, decay, state = R.inputs(1, 300, 1, 2, 64, 64, BF16, 8, n=4)
    cuts = [0, 70, 70, 203, 300]
    off = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    y, final = Q.delta_rule(q, k, v, beta, decay, state, offsets=off)
    for i in range(4):
        r = slice(cuts[i], cuts[i + 1])
        yi, fi = Q.delta_rule(*(t[None, r] for t in (q, k, v, beta, decay)), state[i:i + 1])
        assert torch.equal(yi[0], y[r]) and torch.equal(fi[0], final[i])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,Hk,Hv,dk,dv", [(1, 1400, 1, 1, 64, 48), (1, 3000, 1, 2, 128, 128), (2, 2049, 1, 1, 100, 72),
                                             (1, 6001, 1, 1, 32, 16)])
def test_long(Q, B, T, Hk, Hv, dk, dv, dtype):
    """few heads of long sequences, which are walked in parts"""
    print_case(test="delta rule long", B=B, T=T, Hk=Hk, Hv=Hv, dk=dk, dv=dv, dtype=str(dtype))
    q, k, v, beta, decay, state = R.inputs(B, T, Hk, Hv, dk, dv, dtype, T, correlated=True)
    want = R.whole(q, k, v, beta, decay, state)
    y, final = Q.delta_rule(q, k, v, beta, decay, state)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1
    again = Q.delta_rule(q, k, v, beta, decay, state)
    assert torch.equal(y, again[0]) and torch.equal(final, again[1])
    y, final = Q.delta_rule(q, k, v, beta)
    want = R.whole(q, k, v, beta)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offsets,tail", [([0, 700, 700, 1800, 3100], 13), ([0, 0, 2100, 2101], 0), ([0, 5, 3000], 200),
                                          ([0, 2048], 900)])
def test_long_packed(Q, offsets, tail, dtype):
    T, n = offsets[-1] + tail, len(offsets) - 1
    print_case(test="delta rule long packed", offsets=offsets, tail=tail, dtype=str(dtype))
    q, k, v, beta, decay, state = R.inputs(1, T, 1, 2, 40, 24, dtype, T + n, n=n)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    for t in (q, k, v, beta, decay):
        t[offsets[-1]:] = float("nan")
    want = R.whole(q, k, v, beta, decay, state, off)
    y, final = Q.delta_rule(q, k, v, beta, decay, state, offsets=off)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1
    assert not y[offsets[-1]:].any()
    for bad in ([0, 1 << 30], [-5, 50], [0, 1 << 30, 20], [900, 10, 3000]):
        Q.delta_rule(q, k, v, beta, decay, offsets=torch.tensor(bad, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


def test_no_sequences(Q):
    q, k, v, beta, decay, state = R.inputs(1, 9, 1, 2, 16, 8, BF16, 9, n=0)
    off = torch.zeros(1, dtype=torch.int32, device="cuda")
    y, final = Q.delta_rule(q, k, v, beta, decay, state, offsets=off)
    assert not y.any() and final.shape == state.shape


def test_bad_offsets_stay_inside(Q):
    """offsets outside the rows: which rows belong together is not defined, but nothing outside is touched"""
    q, k, v, beta, decay, _ = R.inputs(1, 100, 1, 2, 16, 8, BF16, 10, n=1)
    for bad in ([0, 1 << 30], [-5, 50], [0, 1 << 30, 20], [90, 10, 200]):
        off = torch.tensor(bad, dtype=torch.int32, device="cuda")
        Q.delta_rule(q, k, v, beta, decay, offsets=off)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1])
def test_strided(Q, dtype, shift):
    """slices of one projection's rows, on and off the vector width; gates as slices too"""
    B, T, H, d = 2, 75, 2, 32
    rows = torch.randn((B, T, 3 * H * d + shift), device="cuda").to(dtype)[..., shift:]
    q, k, v = (t.unflatten(-1, (H, d)) for t in rows.split(H * d, -1))
    k = torch.nn.functional.normalize(k.float(), dim=-1).to(dtype)
    rows[..., H * d:2 * H * d] = k.flatten(-2)
    q, k, v = (t.unflatten(-1, (H, d)) for t in rows.split(H * d, -1))
    gates = torch.rand((B, T, 2 * H + 1), device="cuda")
    beta, decay = gates[..., :H], gates[..., H + 1:]
    decay.neg_()
    y, final = Q.delta_rule(q, k, v, beta, decay)
    want = R.whole(q, k, v, beta, decay)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1
    same = Q.delta_rule(*(t.contiguous() for t in (q, k, v, beta, decay)))
    assert torch.equal(y, same[0]) and torch.equal(final, same[1])


def test_masked_rows(Q):
    """beta = 0 and decay = 0 leave the state; decay = -inf clears it, whatever it held"""
    q, k, v, beta, decay, state = R.inputs(2, 90, 1, 2, 32, 32, F32, 11)
    beta[:, 20:50], decay[:, 20:50] = 0.0, 0.0
    decay[0, 70], decay[1, 33] = float("-inf"), float("-inf")
    y, final = Q.delta_rule(q, k, v, beta, decay, state)
    want = R.whole(q, k, v, beta, decay, state)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1
    cleared = Q.delta_rule(*(t[:1, 70:] for t in (q, k, v, beta, decay)))
    assert R.off(final[:1], cleared[1]) <= 1
    kept = Q.delta_rule(*(t[:1, 20:50] for t in (q, k, v, beta, decay)), state[:1])[1]
    assert torch.equal(kept, state[:1])


def test_strong_decay(Q):
    """decays that underflow within a chunk"""
    q, k, v, beta, _, state = R.inputs(1, 100, 1, 2, 32, 32, F32, 12)
    decay = -40.0 * torch.rand((1, 100, 2), device="cuda")
    y, final = Q.delta_rule(q, k, v, beta, decay, state)
    want = R.whole(q, k, v, beta, decay, state)
    assert R.off(y, want["y"]) <= 1 and R.off(final, want["final"]) <= 1


@pytest.mark.parametrize("scale", [1e-25, 1e20])
def test_range(Q, scale):
    """values far from 1: the rule is linear in v and the state"""
    q, k, v, beta, decay, state = R.inputs(1, 70, 1, 1, 64, 64, F32, 13)
    y, final = Q.delta_rule(q, k, v * scale, beta, decay, state * scale)
    want = R.whole(q, k, v * scale, beta, decay, state * scale)
    assert R.off(y / scale, want["y"] / scale) <= 1 and R.off(final / scale, want["final"] / scale) <= 1


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Hk,Hv,dk,dv", [(1, 1, 1, 1, 1), (3, 2, 4, 64, 64), (5, 1, 3, 33, 50), (2, 2, 2, 128, 128), (7, 1, 1, 100, 4)])
def test_step(Q, B, Hk, Hv, dk, dv, dtype):
    print_case(test="delta rule step", B=B, Hk=Hk, Hv=Hv, dk=dk, dv=dv, dtype=str(dtype))
    q, k, v, beta, decay, state = R.inputs(B, 3, Hk, Hv, dk, dv, dtype, B + dk)
    want = R.whole(q, k, v, beta, decay, state)
    held = state.clone()
    for t in range(3):
        y, held2 = Q.delta_rule_step(q[:, t], k[:, t], v[:, t], beta[:, t], held, decay=decay[:, t],
                                     out_state=held if t else None)
        assert (held2 is held) == (t > 0)
        held = held2
        assert R.off(y, want["y"][:, t]) <= 1
    assert R.off(held, want["final"]) <= 1
    y, s = Q.delta_rule_step(q[:, 0], k[:, 0], v[:, 0], beta[:, 0], state, scale=2.0)
    one = R.whole(q[:, :1], k[:, :1], v[:, :1], beta[:, :1], None, state, scale=2.0)
    assert R.off(y, one["y"][:, 0]) <= 1 and R.off(s, one["final"]) <= 1


def test_repeats_and_streams(Q):
    """the same bits again, alone and on two streams at once"""
    sets = [R.inputs(1, 700, 4, 8, 128, 128, BF16, 20 + i) for i in range(2)]
    want = [Q.delta_rule(*a) for a in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(Q.delta_rule(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g[0], want[i][0]) and torch.equal(g[1], want[i][1])


def test_captured(Q):
    """a prompt and its next tokens in one graph, replayed between eager work"""
    q, k, v, beta, decay, state = R.inputs(2, 101, 2, 4, 64, 64, BF16, 30)
    held = state.clone()

    def run():
        y, s = Q.delta_rule(q[:, :100], k[:, :100], v[:, :100], beta[:, :100], decay[:, :100], state)
        held.copy_(s)
        y1, _ = Q.delta_rule_step(q[:, 100], k[:, 100], v[:, 100], beta[:, 100], held, decay=decay[:, 100], out_state=held)
        return y, y1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(4):
        v.add_(i), state.mul_(0.5)
        want = [t.clone() for t in (*run(), held)]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*got, held), want):
            assert torch.equal(a, b)


def test_refusals(Q):
    q, k, v, beta, decay, state = R.inputs(2, 8, 1, 2, 16, 8, BF16, 40)
    off = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda")
    wide = torch.zeros((2, 8, 2, 129), dtype=BF16, device="cuda")
    for args, kw in [((q.cpu(), k, v, beta), {}), ((q, k.float(), v, beta), {}), ((q, k[:, :7], v, beta), {}),
                     ((q, k, v, beta.double()), {}), ((q, k, v, beta[..., :1]), {}), ((q, k, v.double(), beta), {}),
                     ((q, k, v, beta, decay.bfloat16()), {}), ((q, k, v, beta, decay, state[:1]), {}),
                     ((q, k, v, beta, decay, state.bfloat16()), {}), ((q, k, v, beta), dict(offsets=off)),
                     ((q.transpose(-1, -2), k, v, beta), {}), ((q, k, wide, beta), {}),
                     ((wide[..., :1, :], wide[..., :1, :], v, beta), {}),
                     ((q[0], k[0], v[0], beta[0]), dict(offsets=off.long())), ((q[0], k[0], v[0], beta[0]), {}),
                     ((q.expand(2, 8, 3, 16), k.expand(2, 8, 3, 16), v, beta), {}), ((q, k, v, beta), dict(out=v.float())),
                     ((q[:, :, :0], k[:, :, :0], v, beta), {})]:
        with pytest.raises(ValueError):
            Q.delta_rule(*args, **kw)
    with pytest.raises(ValueError):
        Q.delta_rule_step(q, k, v, beta, state)
    with pytest.raises(ValueError):
        Q.delta_rule_step(q[:, 0], k[:, 0], v[:, 0], beta[:, 0], state[:, :, :, :4])
    with pytest.raises(ValueError):
        Q.delta_rule_step(q[:, 0], k[:, 0], v[:, 0], beta[:, 0], None)
