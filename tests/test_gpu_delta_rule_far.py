"""The gated delta rule over rows whose elements pass 2^31: the last rows, forward and backward, have the bits that they have as a
short sequence from the state before them (a whole number of the kernels' 128 rows lies before), and the first ones theirs."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("packed", [False, True])
def test_past_32_bits(packed):
    if torch.cuda.get_device_properties(0).total_memory < 200 << 30:
        pytest.skip("needs 100 GB")
    from cssm_amd import training
    head, last, Hk, Hv, dk, dv = 128 * 1093, 64, 2, 128, 16, 128
    T = head + last
    assert T * Hv * dv > 1 << 31
    print_case(test="delta rule past 32 bits", T=T, Hv=Hv, dv=dv, packed=packed)
    gen = torch.Generator("cuda").manual_seed(1)

    def normal(*s, dtype=torch.bfloat16):
        return torch.randn(s, generator=gen, device="cuda", dtype=dtype)
    lead = (T,) if packed else (1, T)
    q, k = (torch.nn.functional.normalize(normal(*lead, Hk, dk).float(), dim=-1).bfloat16() for _ in range(2))
    v = normal(*lead, Hv, dv)
    beta = torch.rand((*lead, Hv), generator=gen, device="cuda")
    decay = -0.1 * torch.rand((*lead, Hv), generator=gen, device="cuda")
    off = torch.tensor([0, T], dtype=torch.int32, device="cuda") if packed else None
    grad = normal(*lead[:-1], last, Hv, dv)
    gy = torch.zeros_like(v)
    rows = (slice(head, T),) if packed else (slice(None), slice(head, T))
    gy[rows] = grad

    def run(args, state, offsets, gy):
        args = [t.detach().requires_grad_() for t in args]
        y, final = training.delta_rule_train(*args[:4], decay=args[4], state=state, offsets=offsets)
        grads = torch.autograd.grad(y, args, gy)
        return y.detach(), final.detach(), grads
    y, final, grads = run((q, k, v, beta, decay), None, off, gy)
    del gy
    assert all(bool(torch.isfinite(g.sum()).all()) for g in grads)
    before = (slice(0, head),) if packed else (slice(None), slice(0, head))
    from cssm_amd import sequence
    off_head = torch.tensor([0, head], dtype=torch.int32, device="cuda") if packed else None
    y_head, state = sequence.delta_rule(*(t[before] for t in (q, k, v, beta, decay)), offsets=off_head)
    assert torch.equal(y[before], y_head)
    del y_head
    off_last = torch.tensor([0, last], dtype=torch.int32, device="cuda") if packed else None
    y1, final1, grads1 = run([t[rows].contiguous() for t in (q, k, v, beta, decay)], state, off_last, grad)
    assert torch.equal(y[rows], y1) and torch.equal(final, final1)
    for g, g1 in zip(grads, grads1):
        assert torch.equal(g[rows], g1)
    few = (slice(0, 200),) if packed else (slice(None), slice(0, 200))
    off_few = torch.tensor([0, 200], dtype=torch.int32, device="cuda") if packed else None
    y2, _ = sequence.delta_rule(*(t[few].contiguous() for t in (q, k, v, beta, decay)), offsets=off_few)
    assert torch.equal(y[few], y2)
