"""The gated delta rule in float64, token by token, with its gradients by torch's differentiation (not collected by
pytest), and how far float32 arithmetic may be from it.

Tolerance of float32 results, as lengths (2-norms over the whole tensor): u = 2^-24.  A result is three products in a row
(with the state, within the chunk, with the state again), each a sum of at most 128 + 32 terms whose roundings are
independent: about sqrt(160) u / sqrt(3) = 7.3 u of the terms' own length, which is up to 3 times the result's where keys
are correlated.  The recurrence itself does not enlarge an error (|1 - beta k k^T| <= 1 for unit keys and beta in 0 .. 2), and
those of different chunks are independent.  3 x 7.3 x 3 = 66 u, taken as 64 u = 2^-18.  Single values: up to 6 deviations
among a million, and the gradients of decay add two sums over 128 rows: 16 times that, of the tensor's root mean square.
A bfloat16 result adds half its step, eps / 2 of the value, and its own two parts of 2^-17 each are within the same 2^-14.
"""
import torch

LENGTH, SINGLE = 2.0 ** -18, 2.0 ** -14


def rule(q, k, v, beta, decay, state, scale):
    """(y, final state) of (B, T, H, width) float64 tensors with as many key as value heads."""
    S, ys = state, []
    for t in range(v.shape[1]):
        if decay is not None:
            S = torch.exp(decay[:, t])[..., None, None] * S
        kt = k[:, t][..., None]
        e = v[:, t] - (kt * S).sum(-2)
        S = S + kt * (beta[:, t][..., None] * e)[..., None, :]
        ys.append(scale * (q[:, t][..., None] * S).sum(-2))
    return (torch.stack(ys, 1) if ys else torch.zeros_like(v)), S


def whole(q, k, v, beta, decay=None, state=None, offsets=None, scale=None, dy=None, dfinal=None):
    """As cssm_amd.sequence.delta_rule, in float64 on the CPU: a dict of y, final and, with dy or dfinal, the gradients."""
    ts = {n: None if t is None else t.detach().double().cpu().requires_grad_() for n, t in
          dict(q=q, k=k, v=v, beta=beta, decay=decay, state=state).items()}
    G, dk = v.shape[-2] // k.shape[-2], k.shape[-1]
    scale = dk ** -0.5 if scale is None else scale
    qq, kk = (ts[n].repeat_interleave(G, -2) for n in "qk")
    n = v.shape[0] if offsets is None else offsets.numel() - 1
    S = ts["state"] if state is not None else torch.zeros((n, v.shape[-2], dk, v.shape[-1]), dtype=torch.float64)
    if offsets is None:
        y, final = rule(qq, kk, ts["v"], ts["beta"], ts["decay"], S, scale)
    else:
        off, ys, finals = offsets.tolist(), [], []
        for i in range(n):
            r = slice(off[i], off[i + 1])
            yi, f = rule(qq[None, r], kk[None, r], ts["v"][None, r], ts["beta"][None, r],
                         None if decay is None else ts["decay"][None, r], S[i:i + 1], scale)
            ys.append(yi[0]), finals.append(f)
        y = torch.cat(ys + [torch.zeros((v.shape[0] - off[-1], *v.shape[1:]), dtype=torch.float64)])
        final = torch.cat(finals) if finals else S
    got = {"y": y.detach(), "final": final.detach()}
    if dy is not None or dfinal is not None:
        loss = 0.0
        if dy is not None:
            loss = loss + (y * dy.double().cpu()).sum()
        if dfinal is not None:
            loss = loss + (final * dfinal.double().cpu()).sum()
        names = [m for m, t in ts.items() if t is not None]
        grads = torch.autograd.grad(loss, [ts[m] for m in names], allow_unused=True)
        got.update({"d" + m: torch.zeros_like(ts[m]) if g is None else g for m, g in zip(names, grads)})
    return got


def off(got, want):
    """The larger of the error's length and of its largest value over what each may be."""
    got, want = got.detach(), want.detach().double().cpu()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all()
    if not want.numel():
        return 0.0
    d = (got - want).abs()
    rms = want.square().mean().sqrt() + 1e-30
    single = float((d / (half * (1 + SINGLE) * want.abs() + SINGLE * (rms + want.abs()))).max())
    if half:
        return single
    return max(single, float(d.square().mean().sqrt() / (LENGTH * rms)))


def inputs(B, T, Hk, Hv, dk, dv, dtype, seed, n=None, device="cuda", correlated=False):
    """q, k (unit lengths), v, beta, decay, state as a layer has them; n: packed rows (T, ...) of n sequences."""
    gen = torch.Generator(device="cpu").manual_seed(seed)

    def r(*s):
        return torch.randn(s, generator=gen)
    lead = (T,) if n is not None else (B, T)
    q, k = r(*lead, Hk, dk), r(*lead, Hk, dk)
    if correlated:
        k = 0.3 * k + r(Hk, dk)
    q, k = (t / t.norm(dim=-1, keepdim=True).clamp(min=1e-6) for t in (q, k))
    rate = torch.exp(-5.0 + 5.0 * torch.rand(Hv, generator=gen))
    out = [q.to(dtype), k.to(dtype), r(*lead, Hv, dv).to(dtype), torch.sigmoid(2 * r(*lead, Hv)),
           -rate * torch.nn.functional.softplus(r(*lead, Hv)), r(B if n is None else n, Hv, dk, dv)]
    return [t.to(device) for t in out]
