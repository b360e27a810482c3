"""Packed rows of the gated recurrence in training without a gate, without states, with either gradient alone, from either
checkpoint, and packs without a row."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import token_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def T():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import training
    return training


def make(lens, tail, C, dtype):
    gen = torch.Generator(device="cuda").manual_seed(sum(lens) + C)

    def r(*s, shift=0.0):
        return shift + torch.randn(s, generator=gen, device="cuda")
    n = sum(lens) + tail
    off = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    return (r(n, C).to(dtype), r(n, C, shift=-1.0).to(dtype), 0.9 + 0.1 * torch.rand((C,), generator=gen, device="cuda"),
            r(C, shift=-1.0), r(n, C).to(dtype), r(len(lens), C), r(n, C).to(dtype), r(len(lens), C), off)


@pytest.mark.parametrize("lens,tail", [([130, 0, 7, 300], 9), ([0, 0], 140), ([1] * 40, 0)])
@pytest.mark.parametrize("gated,state,with_dy,with_df", [(False, False, True, True), (True, False, True, False), (False, True, False, True)])
@pytest.mark.parametrize("checkpoint", ["none", "e4m3"])
@pytest.mark.parametrize("dtype,C", [(F32, 13), (BF16, 72)])
def test_gradients(T, lens, tail, gated, state, with_dy, with_df, checkpoint, dtype, C):
    print_case(test="packed training", lens=lens, tail=tail, gated=gated, state=state, dy=with_dy, df=with_df,
               checkpoint=checkpoint, dtype=dtype, C=C)
    x, d, kap, bias, z, h0, dy, df, off = make(lens, tail, C, dtype)
    z, h0 = z if gated else None, h0 if state else None
    names = ["dx", "ddelta", "dkappa", "dbias"] + ["dz"] * gated + ["dstate"] * state
    leaves = [t.requires_grad_(True) for t in (x, d, kap, bias, z, h0) if t is not None]
    y, final = T.token_scan_train(x, d, kap, bias, z=z, state=h0, offsets=off, checkpoint=checkpoint)
    outs = ([(y, dy)] if with_dy else []) + ([(final, df)] if with_df else [])
    g = dict(zip(names, torch.autograd.grad([o for o, _ in outs], leaves, [v for _, v in outs])))
    end = sum(lens)
    k8 = None
    if checkpoint == "e4m3":
        k8 = [None if t is None else R.e4m3_blocks(t.detach()[:end].double().cpu(), 8, 16)[0] if end else t.detach()[:0].double().cpu()
              for t in (x, d, z)]
    x6, d6, z6, k6, b6, h6 = (None if t is None else t.detach().double().cpu() for t in (x, d, z, kap, bias, h0))
    dy6 = dy.double().cpu() if with_dy else torch.zeros((end + tail, C), dtype=torch.float64)
    f6 = df.double().cpu() if with_df else torch.zeros((len(lens), C), dtype=torch.float64)
    sums = {k: torch.zeros(C, dtype=torch.float64) for k in ("dkappa", "dkappa_err", "dbias", "dbias_err")}
    at = 0
    for i, n in enumerate(lens):
        s = slice(at, at + n)
        part = [None if t is None else t[None, s] for t in (x6, d6, z6)]
        w = R.scan(part[0], part[1], k6, b6, part[2], None if h6 is None else h6[i:i + 1], dy6[None, s], f6[i:i + 1],
                   kept=None if k8 is None else [None if v is None else v[None, s] for v in k8], row0=at)
        assert R.off(y[None, s], w["y"], w["y_err"], dtype) <= 1 and R.off(final[i:i + 1], w["final"], w["final_err"]) <= 1
        for name in ["dx", "ddelta"] + ["dz"] * gated:
            assert R.off(g[name][None, s], w[name], w[name + "_err"], dtype) <= 1, (i, name)
        if state:
            assert R.off(g["dstate"][i:i + 1], w["dstate"], w["dstate_err"]) <= 1
        for k in sums:
            sums[k] += w[k]
        at += n
    for k in ("dkappa", "dbias"):
        assert R.off(g[k], sums[k], sums[k + "_err"] + 1e-30) <= 1
    for t in [y] + [g[k] for k in ("dx", "ddelta") + ("dz",) * gated]:
        assert not t[end:].any()


@pytest.mark.parametrize("checkpoint", ["none", "e4m3"])
def test_no_rows_at_all(T, checkpoint):
    """three empty sequences, no row: states and their gradients go through"""
    x, d, kap, bias, z, h0, dy, df, off = make([0, 0, 0], 0, 20, BF16)
    leaves = [t.requires_grad_(True) for t in (x, d, kap, bias, z, h0)]
    y, final = T.token_scan_train(x, d, kap, bias, z=z, state=h0, offsets=off, checkpoint=checkpoint)
    assert y.shape == (0, 20) and torch.equal(final, h0)
    g = torch.autograd.grad((y, final), leaves, (dy, df))
    assert torch.equal(g[5], df) and not g[2].any() and not g[3].any() and g[0].shape == (0, 20)
