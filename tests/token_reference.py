"""The gated recurrence over token sequences in float64, row by row, with its gradients and how far float32 arithmetic
may be from them (not collected by pytest).

Bounds: u = 2^-24 is half a float32 step.  A gain (softplus or sigmoid of v = delta + bias) is off by at most
``k`` roundings, k = 2 max|v| + 8: v's own rounding and the exponential's argument each move ln(gain) by |v| u, the
exponential, logarithm, reciprocal, products and sums by an ulp or so each.  A state is a sum of terms that were
multiplied once for each row since: with H_t = |a_t| H_{t-1} + |D_t x_t| the sum of the terms' magnitudes and
J_t = |a_t| (J_{t-1} + H_{t-1}) the same weighted with the rows since, it is off by at most k u (H_t + J_t), in any order
of the joins (a join adds one rounding, the k has room for it).  The gradients' chain runs backwards likewise, and
products of the two carry both errors.  Column sums add 64 u of the sum of magnitudes (8 rows, 16 groups in order).
"""
import torch

U = 2.0 ** -24


def gains(v):
    """softplus(v), sigmoid(-v), sigmoid(v); -inf gives 0, 1, 0."""
    e = torch.exp(-v.abs())
    return v.clamp(min=0) + torch.log1p(e), torch.where(v > 0, e / (1 + e), 1 / (1 + e)), torch.where(v > 0, 1 / (1 + e), e / (1 + e))


def silu(z):
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


def scan(x, delta, kappa, bias, z=None, state=None, dy=None, dfinal=None, kept=None, row0=0):
    """One batch of equal lengths (B, T, C), everything float64.  A dict of y, final, and with dy the gradients; beside each
    value v its bound as v + '_err'.  kept: (x, delta, z) as the 8-bit checkpoint stands for them, which the gradients
    are taken at, from the forward's states before every 128th row (the first one here being row row0)."""
    B, T, C = x.shape
    out = {}

    def forward(x, delta, z, states=None):
        v = delta + bias
        k = 2 * float(v[torch.isfinite(v)].abs().max()) + 8 if v.numel() and torch.isfinite(v).any() else 8
        D, keep, gate = gains(v)
        a = kappa * keep
        h = torch.zeros((B, C), dtype=x.dtype, device=x.device) if state is None else state
        H, J = h.abs(), torch.zeros_like(h)
        hs, Hs, Js, before = [], [], [], []
        for t in range(T):
            if states is not None and t and (row0 + t) % 128 == 0:
                h, H, J = states[t]
            before.append((h, H, J))
            J = a[:, t].abs() * (J + H)
            H = a[:, t].abs() * H + (D[:, t] * x[:, t]).abs()
            h = a[:, t] * h + D[:, t] * x[:, t]
            hs.append(h), Hs.append(H), Js.append(J)
        return D, keep, gate, a, k, hs, Hs, Js, before, h

    D, keep, gate, a, k, hs, Hs, Js, before, h = forward(x, delta, z)

    def cat(v):
        return torch.stack(v, 1) if v else torch.zeros((B, 0, C), dtype=x.dtype, device=x.device)
    Eh = k * U * (cat(Hs) + cat(Js))
    sz = 1.0 if z is None else silu(z)[0]
    out["y"] = cat(hs) * sz
    out["y_err"] = Eh * (sz.abs() if z is not None else 1.0) + (8 + (0 if z is None else z.abs())) * U * out["y"].abs()
    out["final"] = h
    out["final_err"] = Eh[:, -1] if T else torch.zeros_like(h)
    if dy is None:
        return out
    if kept is not None:
        x, delta, z = kept
        k1 = k
        D, keep, gate, a, k, hs, Hs, Js, before, _ = forward(x, delta, z, before)
        k = max(k, k1)
        Eh = k * U * (cat(Hs) + cat(Js))
    hb, Hb, Jb = (cat([b[i] for b in before]) for i in range(3))
    Eb = k * U * (Hb + Jb)
    s, ds = (None, None) if z is None else silu(z)
    p = dy if z is None else dy * s
    Gn = torch.zeros((B, C), dtype=x.dtype, device=x.device) if dfinal is None else dfinal
    A, W = Gn.abs(), torch.zeros_like(Gn)
    g, ga, gw = [None] * T, [None] * T, [None] * T
    zz = 0.0 if z is None else z.abs()
    for t in range(T - 1, -1, -1):
        g[t] = p[:, t] + Gn
        ga[t], gw[t] = p[:, t].abs() + A, W + (0.0 if z is None else zz[:, t] * p[:, t].abs())
        Gn = a[:, t] * g[t]
        W = a[:, t].abs() * (gw[t] + ga[t])
        A = a[:, t].abs() * ga[t]
    g, ga = cat(g), cat(ga)
    Eg = k * U * (ga + cat(gw))
    m = x.abs() + a.abs() * Hb
    out["dx"], out["dx_err"] = D * g, D * (Eg + k * U * ga)
    out["ddelta"] = gate * g * (x - a * hb)
    out["ddelta_err"] = gate * (Eg * m + ga * (a.abs() * Eb + 2 * k * U * m))
    if z is not None:
        out["dz"] = dy * cat(hs) * ds
        out["dz_err"] = dy.abs() * (1.1 * Eh + cat(Hs) * (1 + zz) ** 2 * 12 * U)
    q = g * keep * hb
    qe = keep * (Eg * Hb + ga * (Eb + 2 * k * U * Hb))
    out["dkappa"], out["dkappa_err"] = q.sum((0, 1)), (qe + 64 * U * q.abs()).sum((0, 1))
    out["dbias"] = out["ddelta"].sum((0, 1))
    out["dbias_err"] = (out["ddelta_err"] + 64 * U * out["ddelta"].abs()).sum((0, 1))
    out["dstate"], out["dstate_err"] = Gn, k * U * (A + W)
    return out


def off(got, want, err, dtype=torch.float32):
    """The largest of |got - want| over its bound: the float32 arithmetic's, and half a step of a 16-bit output.  Not a
    number and infinities have to be where they are wanted."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    lim = err.double().cpu().expand_as(want) + 1e-37
    if dtype != torch.float32:
        lim = lim * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).eps / 2 * want.abs()
    else:
        lim = lim + U * want.abs()
    r = ((got - want).abs() / lim)[fine]
    return float(r.max()) if r.numel() else 0.0


def e4m3_blocks(v, rows, cols):
    """(..., M, K) float64 -> what each block of rows x cols keeps of it in e4m3 under its power of two, and the exponents;
    NaN and infinities become NaN."""
    *lead, M, K = v.shape
    m, k = -(-M // rows), -(-K // cols)
    p = torch.nn.functional.pad(v, (0, k * cols - K, 0, m * rows - M)).reshape(*lead, m, rows, k, cols)
    bad = ~torch.isfinite(p)
    p = torch.where(bad, torch.zeros_like(p), p)
    top = p.abs().amax(dim=(-3, -1), keepdim=True)
    f, e = torch.frexp(top)                                       # top = f 2^e, f in [0.5, 1); 448 = 0.875 2^9
    e = torch.where(top > 0, torch.where(f > 0.875, e - 8, e - 9), torch.zeros_like(e)).clamp(min=-126)
    t = torch.ldexp(p, -e)
    step = torch.ldexp(torch.ones_like(t), torch.frexp(t.abs().clamp(min=2.0 ** -6))[1] - 4)
    q = torch.ldexp(torch.round(t / step) * step, e)
    q = torch.where(bad, torch.full_like(q, float("nan")), q)
    return q.reshape(*lead, m * rows, k * cols)[..., :M, :K], e[..., :, 0, :, 0]
