"""The token-sequence operators one behind the other, as a layer uses them: norm with the residual's addition, 8-bit
product, recurrence on slices of its output - a prompt, then single tokens, captured too - and a training pass."""
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


def plain(b):
    """The float64 values that 8-bit blocks stand for (128 of a row, or 128 x 128)."""
    v, e = b.values.float().double().cpu(), b.scales.view(torch.uint8).cpu().double() - 127
    rows = 128 if b.scales.shape[:-1] != b.values.shape[:-1] else 1
    e = e.repeat_interleave(128, -1)[..., :v.shape[-1]]
    if rows > 1:
        e = e.repeat_interleave(rows, 0)[:v.shape[0]]
    return v * 2.0 ** e


def layer(K, C, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s, scale=1.0, shift=0.0):
        return shift + scale * torch.randn(s, generator=gen, device="cuda")
    return dict(w=r(K, scale=0.1, shift=1.0), kernel=r(K, 3 * C, scale=K ** -0.5), b=r(3 * C, scale=0.1),
                kappa=0.9 + 0.1 * torch.rand(C, generator=gen, device="cuda"), bias=r(C, scale=0.5, shift=-1.0)), r


def check_product(p, a8, w8, b):
    """half a bf16 step, what the 8-bit instruction drops (2^-13 of the largest product for each of its additions, of
    which 128 values take 4: under 2^-11 of the sum of magnitudes) and float32 sums"""
    a, w = plain(a8), plain(w8)
    want, mag = a @ w.T + b.double().cpu(), a.abs() @ w.abs().T + b.double().cpu().abs()
    lim = 2.0 ** -8 * want.abs() + 2.0 ** -11 * mag
    assert float(((p.double().cpu() - want).abs() / lim).max()) <= 1


def check_scan(y, final, x, d, kap, bias, z, state):
    w = R.scan(*(None if t is None else t.double().cpu() for t in (x, d, kap, bias, z, state)))
    assert R.off(y, w["y"], w["y_err"], y.dtype) <= 1 and R.off(final, w["final"], w["final_err"]) <= 1


@pytest.mark.parametrize("B,T,K,C", [(2, 150, 128, 64), (3, 33, 208, 20), (1, 300, 256, 130)])
def test_prompt_then_tokens(Q, B, T, K, C):
    print_case(test="prompt then tokens", B=B, T=T, K=K, C=C)
    L, r = layer(K, C, 3)
    w8 = Q.quantize_weight(L["kernel"])
    x, res = r(B, T, K).bfloat16(), r(B, T, K).bfloat16()

    def front(x, res):
        y8, s = Q.rms_norm(x, L["w"], res, out="e4m3")
        return y8, s, Q.scaled_matmul(y8, w8, L["b"])
    y8, s, p = front(x, res)
    sd = (x.double() + res.double()).bfloat16()
    assert torch.equal(s, sd)
    check_product(p, y8, w8, L["b"])
    z, xs, d = p.chunk(3, dim=-1)
    P = T - 5
    y, h = Q.token_scan(xs[:, :P], d[:, :P], L["kappa"], L["bias"], z=z[:, :P])
    check_scan(y, h, xs[:, :P], d[:, :P], L["kappa"], L["bias"], z[:, :P], None)

    # the last tokens one by one, from the prompt's state
    def token(x, res, h, out_state):
        y8, _, p = front(x, res)
        z, xs, d = p.chunk(3, dim=-1)
        return (*Q.token_scan_step(xs, d, L["kappa"], L["bias"], h, z=z, out_state=out_state), y8, p)
    h1, eager = h.clone(), []
    for t in range(P, T):
        before = h1.clone()
        yt, h1, t8, pt = token(x[:, t].contiguous(), res[:, t].contiguous(), h1, h1)
        assert torch.equal(t8.values.view(torch.uint8), y8.values[:, t].view(torch.uint8))      # a row's own
        assert torch.equal(t8.scales.view(torch.uint8), y8.scales[:, t].view(torch.uint8))
        check_product(pt, t8, w8, L["b"])
        q = [v[:, None] for v in pt.chunk(3, dim=-1)]
        check_scan(yt[:, None], h1, q[1], q[2], L["kappa"], L["bias"], q[0], before)
        eager.append((yt, h1.clone()))

    # captured on another stream, replayed for each token
    sx, sr, sh = x[:, 0].contiguous(), res[:, 0].contiguous(), h.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token(sx, sr, sh, sh)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gy = token(sx, sr, sh, sh)[0]
    sh.copy_(h)
    for t in range(P, T):
        sx.copy_(x[:, t]), sr.copy_(res[:, t])
        graph.replay()
        assert torch.equal(gy, eager[t - P][0]) and torch.equal(sh, eager[t - P][1])
        torch.cuda.synchronize()
        front(x, res)          # the program's own eager work in between


def test_captured_prompt(Q):
    """norm, product and recurrence of a prompt over several tiles in one graph: every replay as the eager call"""
    L, r = layer(256, 96, 5)
    w8 = Q.quantize_weight(L["kernel"])
    x, res = r(2, 700, 256).bfloat16(), r(2, 700, 256).bfloat16()

    def run():
        y8, s = Q.rms_norm(x, L["w"], res, out="e4m3")
        z, xs, d = Q.scaled_matmul(y8, w8, L["b"], act="none").chunk(3, dim=-1)
        y, h = Q.token_scan(xs, d, L["kappa"], L["bias"], z=z)
        return s, y, h
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(4):
        x.add_(i), res.mul_(0.5)
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("checkpoint", ["none", "e4m3"])
@pytest.mark.parametrize("B,T,K,C", [(2, 40, 64, 32), (1, 140, 48, 20)])
def test_training_pass(Q, B, T, K, C, checkpoint):
    """norm -> projection -> recurrence -> loss: the recurrence's gradients within its bounds at the projection's outputs,
    the norm's and the projection's against float64 from there (sums of at most 2^10 float32 terms, 2^-24 each rounding:
    2^-13 of the gradient's length)."""
    print_case(test="training pass", B=B, T=T, K=K, C=C, checkpoint=checkpoint)
    from cssm_amd import training
    L, r = layer(K, C, 7)
    x, res, w, kernel = [t.requires_grad_() for t in (r(B, T, K), r(B, T, K), L["w"], L["kernel"])]
    kap, bias = L["kappa"].requires_grad_(), L["bias"].requires_grad_()
    gy, gs = r(B, T, C), r(B, T, K)
    n, s = training.rms_norm_train(x, w, residual=res)
    p = torch.matmul(n, kernel) + L["b"]
    p.retain_grad()
    z, xs, d = p.chunk(3, dim=-1)
    y, final = training.token_scan_train(xs, d, kap, bias, z=z, checkpoint=checkpoint)
    ((y * gy).sum() + (s * gs).sum()).backward()
    D = [t.detach().double().cpu() for t in (xs, d, kap, bias, z)]
    kept = None
    if checkpoint == "e4m3":
        kept = [R.e4m3_blocks(D[i], 8, 16)[0] for i in (0, 1, 4)]
    want = R.scan(*D, dy=gy.double().cpu(), kept=kept)
    assert R.off(y, want["y"], want["y_err"]) <= 1
    for got, name in zip(p.grad.chunk(3, dim=-1), ("dz", "dx", "ddelta")):
        assert R.off(got, want[name], want[name + "_err"]) <= 1, name
    assert R.off(kap.grad, want["dkappa"], want["dkappa_err"]) <= 1
    assert R.off(bias.grad, want["dbias"], want["dbias_err"]) <= 1
    x6, r6, w6, k6 = [t.detach().double().cpu().requires_grad_() for t in (x, res, w, kernel)]
    s6 = x6 + r6
    n6 = s6 * torch.rsqrt(s6.square().mean(-1, keepdim=True) + 1e-6) * w6
    ((n6 @ k6) * p.grad.double().cpu()).sum().add((s6 * gs.double().cpu()).sum()).backward()
    for got, ref in ((x, x6), (res, r6), (w, w6), (kernel, k6)):
        assert float((got.grad.double().cpu() - ref.grad).norm() / ref.grad.norm()) <= 2.0 ** -13


def test_two_streams_at_once(Q):
    """Two recurrences of many tiles, and their adjoints, side by side on two streams: each as it is alone."""
    _, r = layer(16, 16, 9)
    sets = [(r(1, 20000, 128).bfloat16(), r(1, 20000, 128).bfloat16(), 0.9 + 0.01 * r(128), r(128) - 2,
             r(1, 20000, 128).bfloat16()) for _ in range(2)]

    def run(a):
        x, d, k, b, z = a
        y, h, st, _, _ = Q.scan_forward(x, d, k, b, z, None, None, keep_states=True)
        return (y, h, *Q.scan_backward(x, d, k, b, z, None, None, st, None, None, y, None, True))
    want = [run(a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for a, b in zip(g, want[i]):
                assert torch.equal(a, b)


def test_same_tensor_twice(Q):
    """one tensor as x, delta and z, and as x and its own residual, with gradients that add up"""
    from cssm_amd import training
    L, r = layer(64, 64, 11)
    v = r(2, 50, 64).requires_grad_()
    g = r(2, 50, 64)
    y, _ = training.token_scan_train(v, v, L["kappa"], L["bias"], z=v)
    y.backward(g)
    D = [t.detach().double().cpu() for t in (v, v, L["kappa"], L["bias"], v)]
    w = R.scan(*D, dy=g.double().cpu())
    err = sum(w[n + "_err"] + 4 * R.U * w[n].abs() for n in ("dx", "ddelta", "dz"))
    assert R.off(v.grad, w["dx"] + w["ddelta"] + w["dz"], err) <= 1
    u = r(5, 64).requires_grad_()
    n, s = training.rms_norm_train(u, L["w"], residual=u)
    gn, gs = r(5, 64), r(5, 64)
    torch.autograd.backward([n, s], [gn, gs])
    u6 = u.detach().double().cpu().requires_grad_()
    s6 = u6 + u6
    n6 = s6 * torch.rsqrt(s6.square().mean(-1, keepdim=True) + 1e-6) * L["w"].double().cpu()
    torch.autograd.backward([n6, s6], [gn.double().cpu(), gs.double().cpu()])
    # 64 terms and a handful of operations, each 2^-24: under 2^-17 of the gradient's length
    assert float((u.grad.double().cpu() - u6.grad).norm() / u6.grad.norm()) <= 2.0 ** -17
