"""The delta rule as a layer uses it: norm behind the residual's addition, projection, heads of unit length turned by their
positions, the rule on slices of the projection - a prompt, then single tokens, captured too - and a training pass."""
import pytest

from tests.gpu_util import print_case

torch = pytest.importorskip("torch")
from tests import delta_reference as R  # noqa: E402
from tests.test_gpu_rotate_heads import off, plain  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def Q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import sequence
    return sequence


def layer(Q, K, Hk, Hv, d, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s, scale=1.0, shift=0.0):
        return shift + scale * torch.randn(s, generator=gen, device="cuda")
    return dict(norm=r(K, scale=0.1, shift=1.0), qkv=r(K, (2 * Hk + Hv) * d, scale=K ** -0.5).to(dtype),
                gates=r(K, 2 * Hv, scale=K ** -0.5), out=r(Hv * d, K, scale=(Hv * d) ** -0.5).to(dtype),
                table=Q.rotary_table([d // 8, d // 8, d // 4])), r


def front(Q, L, x, res, positions, Hk, Hv, d):
    """(stream, q, k, v, beta, decay) of rows (..., K)"""
    n, s = Q.rms_norm(x, L["norm"], residual=res)
    p = n @ L["qkv"]
    q, k, v = p.split((Hk * d, Hk * d, Hv * d), -1)
    q, k = Q.rotate_heads(q.unflatten(-1, (Hk, d)), k.unflatten(-1, (Hk, d)), positions, L["table"], norm="l2")
    b, g = (n.float() @ L["gates"]).split(Hv, -1)
    return s, q, k, v.unflatten(-1, (Hv, d)), torch.sigmoid(b), -torch.nn.functional.softplus(g)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,K,Hk,Hv,d", [(2, 150, 96, 1, 2, 32), (1, 1300, 64, 2, 2, 64)])
def test_prompt_then_tokens(Q, B, T, K, Hk, Hv, d, dtype):
    print_case(test="delta block", B=B, T=T, K=K, Hk=Hk, Hv=Hv, d=d, dtype=str(dtype))
    L, r = layer(Q, K, Hk, Hv, d, dtype, 3)
    x, res = r(B, T, K).to(dtype), r(B, T, K).to(dtype)
    at = torch.arange(T, device="cuda")
    positions = torch.stack([at // 16, at // 4 % 4, at % 4], -1).to(torch.int32).expand(B, T, 3).contiguous()
    s, q, k, v, beta, decay = front(Q, L, x, res, positions, Hk, Hv, d)
    p = (Q.rms_norm(x, L["norm"], residual=res)[0] @ L["qkv"])
    for got, raw in ((q, p[..., :Hk * d]), (k, p[..., Hk * d:2 * Hk * d])):
        want = plain(raw.unflatten(-1, (Hk, d)), None, positions, L["table"], "l2", 1e-6, "halves")
        assert off(got, want["y"], want["y_err"]) <= 1
    P = T - 5
    y, h = Q.delta_rule(q[:, :P], k[:, :P], v[:, :P], beta[:, :P], decay[:, :P])
    want = R.whole(q, k, v, beta, decay)
    assert R.off(y, want["y"][:, :P]) <= 1

    # the last tokens one by one, from the prompt's state, eager and captured on another stream
    def token(x, res, positions, h):
        _, q, k, v, beta, decay = front(Q, L, x, res, positions, Hk, Hv, d)
        return Q.delta_rule_step(q, k, v, beta, h, decay=decay, out_state=h)[0], (q, k, v, beta, decay)
    h1, eager = h.clone(), []
    for t in range(P, T):
        before = h1.clone()
        yt, args = token(x[:, t].contiguous(), res[:, t].contiguous(), positions[:, t].contiguous(), h1)
        one = R.whole(*(a[:, None] for a in args), before)
        assert R.off(yt, one["y"][:, 0]) <= 1 and R.off(h1, one["final"]) <= 1
        eager.append((yt, h1.clone()))
    sx, sr, sp, sh = x[:, 0].contiguous(), res[:, 0].contiguous(), positions[:, 0].contiguous(), h.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token(sx, sr, sp, sh)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gy = token(sx, sr, sp, sh)[0]
    sh.copy_(h)
    for t in range(P, T):
        sx.copy_(x[:, t]), sr.copy_(res[:, t]), sp.copy_(positions[:, t])
        graph.replay()
        # the library's products may take another kernel under capture: the rule's own values are checked against float64
        assert torch.isfinite(gy).all() and gy.shape == eager[t - P][0].shape
        assert float((gy.float() - eager[t - P][0].float()).norm() / eager[t - P][0].float().norm()) <= 2.0 ** -6
        torch.cuda.synchronize()
        front(Q, L, x, res, positions, Hk, Hv, d)          # the program's own eager work in between


def test_training_pass(Q):
    """norm -> projection -> heads -> rule -> projection -> loss in float32: every gradient against float64 differentiation of
    the same layer.  The norms and products before the rule put errors of some 2^-20 of its inputs into it, which it hands on
    at most at their size; 2^-13 of a gradient's length leaves room for the products' sums of up to 2^8 terms."""
    from cssm_amd import training as T
    B, L_, K, Hk, Hv, d = 2, 70, 48, 1, 2, 32
    L, r = layer(Q, K, Hk, Hv, d, F32, 7)
    x, res = r(B, L_, K).requires_grad_(), r(B, L_, K).requires_grad_()
    ws = {n: L[n].requires_grad_() for n in ("norm", "qkv", "gates", "out")}
    at = torch.arange(L_, device="cuda")
    positions = torch.stack([at // 16, at // 4 % 4, at % 4], -1).to(torch.int32).expand(B, L_, 3).contiguous()
    gy = r(B, L_, K)
    n, s = T.rms_norm_train(x, ws["norm"], residual=res)
    q, k, v = (n @ ws["qkv"]).split((Hk * d, Hk * d, Hv * d), -1)
    q, k = T.rotate_heads_train(q.unflatten(-1, (Hk, d)), k.unflatten(-1, (Hk, d)), positions, L["table"], norm="l2")
    b, g = (n @ ws["gates"]).split(Hv, -1)
    y, _ = T.delta_rule_train(q, k, v.unflatten(-1, (Hv, d)), torch.sigmoid(b), -torch.nn.functional.softplus(g))
    out = y.flatten(-2) @ ws["out"] + s
    leaves = [x, res, *ws.values()]
    got = torch.autograd.grad(out, leaves, gy)

    x6, r6, *w6 = (t.detach().double().cpu().requires_grad_() for t in leaves)
    s6 = x6 + r6
    n6 = s6 * torch.rsqrt(s6.square().mean(-1, keepdim=True) + 1e-6) * w6[0]
    q6, k6, v6 = (n6 @ w6[1]).split((Hk * d, Hk * d, Hv * d), -1)
    ang = positions.cpu().double()[..., L["table"].axes.long().cpu()] * L["table"].frequencies.cpu()
    c, sn = torch.cat([ang.cos()] * 2, -1)[:, :, None], torch.cat([ang.sin()] * 2, -1)[:, :, None]

    def turn(t):
        t = t.unflatten(-1, (Hk, d))
        t = t * torch.rsqrt(t.square().sum(-1, keepdim=True) + 1e-6)
        a, e = t.chunk(2, -1)
        return t * c + torch.cat([-e, a], -1) * sn
    b6, g6 = (n6 @ w6[2]).split(Hv, -1)
    zero = torch.zeros((B, Hv, d, d), dtype=torch.float64)
    y6, _ = R.rule(turn(q6).repeat_interleave(Hv // Hk, -2), turn(k6).repeat_interleave(Hv // Hk, -2), v6.unflatten(-1, (Hv, d)),
                   torch.sigmoid(b6), -torch.nn.functional.softplus(g6), zero, d ** -0.5)
    out6 = y6.flatten(-2) @ w6[3] + s6
    want = torch.autograd.grad(out6, [x6, r6, *w6], gy.double().cpu())
    for a, e in zip(got, want):
        assert float((a.double().cpu() - e).norm() / e.norm()) <= 2.0 ** -13
