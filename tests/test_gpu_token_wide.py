"""The gated recurrence where there are tiles enough for the forward of 32 threads across, which the large sizes run: batches
and packed rows over many tiles and off every border, against float64 row by row."""
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


def over(n, d):
    return -(-n // d)


def wide(B, T, C, dtype):
    """tiles of 128 rows x 32 threads of 4 (bf16) or 2 (float32) channels; 256 of them select the kernel"""
    v = 4 if dtype == BF16 else 2
    return C % v == 0 and B * over(T, 128) * over(C, 32 * v) >= 256


def make(B, T, C, dtype, gated=True, slices=False):
    gen = torch.Generator(device="cuda").manual_seed(T + C)

    def r(*s, scale=1.0, shift=0.0):
        return shift + scale * torch.randn(s, generator=gen, device="cuda")
    x, d, z = r(B, T, C).to(dtype), r(B, T, C, shift=-1.0).to(dtype), r(B, T, C, scale=1.5).to(dtype)
    if slices:
        p = torch.cat([z, x, d], dim=2)
        z, x, d = p.chunk(3, dim=2)
    kap = 0.9 + 0.1 * torch.rand((C,), generator=gen, device="cuda")
    kap[::5] *= -1.0
    return x, d, kap, -2.0 + 2.0 * torch.rand((C,), generator=gen, device="cuda"), z if gated else None, gen


def dbl(*ts):
    return [None if t is None else t.double() for t in ts]


# (the float64 recurrence runs on the GPU: elementwise operations only)
@pytest.mark.parametrize("B,T,C,dtype,slices", [(2, 1100, 2052, BF16, False), (1, 2100, 1030, F32, False), (3, 1025, 1284, BF16, True),
                                                (40, 130, 516, BF16, False), (130, 1, 260, F32, True), (256, 5, 12, BF16, False)])
@pytest.mark.parametrize("gated,state", [(True, True), (False, False)])
def test_batch(Q, B, T, C, dtype, slices, gated, state):
    print_case(test="token_scan wide", B=B, T=T, C=C, dtype=dtype, slices=slices, gated=gated)
    assert wide(B, T, C, dtype)
    x, d, kap, bias, z, gen = make(B, T, C, dtype, gated, slices)
    h0 = torch.randn((B, C), generator=gen, device="cuda") if state else None
    y, final = Q.token_scan(x, d, kap, bias, z=z, state=h0)
    w = R.scan(*dbl(x, d, kap, bias, z, h0))
    assert R.off(y, w["y"], w["y_err"], dtype) <= 1 and R.off(final, w["final"], w["final_err"]) <= 1
    # the same bits again, and the states that a training pass keeps are those between the rows
    y2, f2, states, _, _ = Q.scan_forward(x, d, kap, bias, z, h0, None, keep_states=True)
    assert torch.equal(y, y2) and torch.equal(final, f2) and states.shape == (B, over(T, 128), C)
    for k in range(1, states.shape[1]):
        _, part = Q.token_scan(x[:, :128 * k], d[:, :128 * k], kap, bias, state=h0)
        ref = R.scan(*dbl(x[:, :128 * k], d[:, :128 * k], kap, bias, None, h0))
        assert R.off(states[:, k], ref["final"], ref["final_err"]) <= 1 and R.off(part, ref["final"], ref["final_err"]) <= 1
        if k == 2:
            break


# starts and ends on borders of tiles, of spans of 8 tiles and of row groups, and off them; empty ones in every place
LENS = [[0, 128, 0, 896, 1, 127, 1024, 0, 0, 37, 300, 0], [3, 0, 2040, 5, 200, 64, 64], [2500]]


@pytest.mark.parametrize("lens", LENS, ids=lambda v: str(len(v)))
@pytest.mark.parametrize("tail", [0, 140])
@pytest.mark.parametrize("C,dtype,gated", [(2052, BF16, True), (1030, F32, True), (1800, BF16, False)])
def test_packed(Q, lens, tail, C, dtype, gated):
    print_case(test="token_scan wide packed", lens=lens, tail=tail, C=C, dtype=dtype, gated=gated)
    end = sum(lens)
    assert wide(1, end + tail, C, dtype)
    x, d, kap, bias, z, gen = make(1, end + tail, C, dtype, gated, slices=True)
    x, d, z = x[0], d[0], None if z is None else z[0]
    x[end:], d[end:] = float("nan"), float("nan")       # what lies behind the last sequence is not looked at
    h0 = torch.randn((len(lens), C), generator=gen, device="cuda")
    off = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    buf = torch.full((end + tail, C), 7.0, dtype=dtype, device="cuda")
    y, final = Q.token_scan(x, d, kap, bias, z=z, state=h0, offsets=off)
    y2, final2 = Q.token_scan(x, d, kap, bias, z=z, state=h0, offsets=off, out=buf)
    assert torch.equal(y[:end], y2[:end]) and torch.equal(final, final2)
    assert not y[end:].any() and bool((buf[end:] == 7.0).all())
    at = 0
    for i, n in enumerate(lens):
        part = [t[None, at:at + n] if t is not None else None for t in (x, d, z)]
        w = R.scan(*dbl(part[0], part[1], kap, bias, part[2], h0[i:i + 1]))
        assert R.off(y[None, at:at + n], w["y"], w["y_err"], dtype) <= 1, i
        assert R.off(final[i:i + 1], w["final"], w["final_err"]) <= 1, i
        at += n


def test_many_short_sequences(Q):
    """Thousands of sequences of 0 to 12 rows: what the same rows give as a padded batch, whose rows behind each sequence
    delta = -inf and kappa = 1 make idle."""
    n, C = 3000, 260
    gen = torch.Generator(device="cuda").manual_seed(3)
    lens = torch.randint(0, 13, (n,), generator=gen, device="cuda")
    off = torch.cat([lens.new_zeros(1), lens.cumsum(0)]).to(torch.int32)
    T = int(off[-1])
    assert wide(1, T, C, BF16)
    x, d, _, bias, z, _ = make(1, T, C, BF16)
    x, d, z = x[0], d[0], z[0]
    one = torch.ones(C, device="cuda")
    h0 = torch.randn((n, C), generator=gen, device="cuda")
    y, final = Q.token_scan(x, d, one, bias, z=z, state=h0, offsets=off)
    row = torch.arange(12, device="cuda")[None] + off[:-1, None]
    there = torch.arange(12, device="cuda")[None] < lens[:, None]
    px, pd, pz = (t[row.clamp(max=T - 1)] for t in (x, d, z))
    px, pd = torch.where(there[..., None], px, 0.0), torch.where(there[..., None], pd, float("-inf"))
    w = R.scan(*dbl(px, pd, one, bias, pz, h0))
    assert R.off(final, w["final"], w["final_err"]) <= 1
    assert R.off(y, w["y"][there], w["y_err"][there], BF16) <= 1
