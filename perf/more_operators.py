"""The delta rule over token sequences and the operator that prepares its queries and keys, as this framework is timed on
them through its public entry points.

A case's ``op`` names one:
  step      one token of the gated delta rule for each sequence of a batch, with its state
  rule      the gated delta rule over whole sequences: a (B, T) batch, or rows packed one sequence behind the other
  train     the same forward and backward
  rotate    norm of each head's queries and keys and the rotation by their positions on several axes
  rtrain    the same forward and backward

The delta rule, for each value head (G of them share one query and key head), with S (dk, dv) the state:
e_t = v_t - a_t S_{t-1}^T k_t, S_t = a_t S_{t-1} + k_t (b_t e_t)^T and y_t = scale S_t^T q_t, a = exp(decay).
The rotation: n = x / norm(x) * weight for each head, then the pair j turned by the angle freq_j position_{axis j}.
Where ``own`` is false ``run`` computes these in elementary torch operations.
"""
import math

import torch

own = False

CHUNK = 64             # rows that the plain form takes at once
EPS = 1e-6


def listed():
    return [
        # serving: one token for a small batch, the smallest call
        dict(name="step_4", op="step", B=4, Hk=4, Hv=4, dk=64, dv=64, io="bf16"),
        # one token for many sequences, two value heads for each key head: the states' bytes
        dict(name="step_128", op="step", B=128, Hk=8, Hv=16, dk=128, dv=128, io="bf16"),
        # the tokens of a few small images in odd sizes, continued from a state
        dict(name="rule_odd", op="rule", B=3, T=197, Hk=3, Hv=3, dk=40, dv=50, N=0, tail=0, io="f32"),
        # a prefill of a batch of equal lengths
        dict(name="rule_prefill", op="rule", B=8, T=2048, Hk=16, Hv=16, dk=128, dv=128, N=0, tail=0, io="bf16"),
        # one very long sequence, where only the time axis offers parallel work
        dict(name="rule_long", op="rule", B=1, T=65536, Hk=8, Hv=8, dk=128, dv=128, N=0, tail=0, io="bf16"),
        # a serving prefill: ragged sequences packed behind each other, some empty, padding rows behind the last
        dict(name="rule_packed", op="rule", B=1, T=16001, Hk=8, Hv=16, dk=128, dv=128, N=23, tail=77, io="bf16"),
        # a training step on long sequences
        dict(name="train_4096", op="train", B=4, T=4096, Hk=16, Hv=16, dk=128, dv=128, N=0, tail=0, io="bf16"),
        # a small float32 training step at sizes off every block, two value heads for each key head
        dict(name="train_odd", op="train", B=2, T=501, Hk=2, Hv=4, dk=64, dv=72, N=0, tail=0, io="f32"),
        # queries and keys of one serving step, plain positions
        dict(name="rotate_token", op="rotate", M=16, Hq=16, Hk=4, D=128, axes=1, norm="rms", pairs="halves", io="bf16"),
        # queries and keys of a batch of clips: time, height and width
        dict(name="rotate_video", op="rotate", M=16384, Hq=16, Hk=16, D=128, axes=3, norm="rms", pairs="halves", io="bf16"),
        # the same in training
        dict(name="rtrain_video", op="rtrain", M=16384, Hq=16, Hk=16, D=128, axes=3, norm="rms", pairs="halves", io="bf16"),
        # training on images in float32: two axes, neighbours paired, unit lengths as the delta rule takes them
        dict(name="rtrain_image", op="rtrain", M=3137, Hq=6, Hk=6, D=72, axes=2, norm="l2", pairs="neighbours", io="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["step", "rule", "rule", "train", "train", "rotate", "rtrain"])
    io = rng.choice(["bf16", "bf16", "f32"])
    if op in ("step", "rule", "train"):
        G = rng.choice([1, 1, 2, 4])
        Hk = _log(rng, 1, 16)
        Hv = min(32, G * Hk) if op == "step" else G * Hk if G * Hk <= 16 else Hk
        Hv -= Hv % Hk
        dk, dv = [rng.choice([128, 64, rng.randint(9, 128)]) for _ in range(2)]
        if op == "step":
            return dict(op=op, B=_log(rng, 1, 128), Hk=Hk, Hv=Hv, dk=dk, dv=dv, io=io)
        T = _log(rng, 1, 32768 if op == "rule" else 4096)
        packed = rng.random() < 0.4
        B = 1 if packed else _log(rng, 1, 8)
        most = (1 << 18) if op == "rule" else (1 << 17) if io == "bf16" else (1 << 16)
        while B * T * Hv > most:
            B, T = max(1, B // 2), max(1, T - T // 3)
        return dict(op=op, B=B, T=T, Hk=Hk, Hv=Hv, dk=dk, dv=dv, N=rng.randint(1, 30) if packed else 0,
                    tail=min(T - 1, rng.choice([0, 0, 5, 130])) if packed else 0, io=io)
    D = rng.choice([128, 64, 2 * rng.randint(8, 128)])
    M, Hq = _log(rng, 1, 16384), _log(rng, 1, 32)
    while M * Hq * D > (1 << 25):
        M = M - M // 3
    return dict(op=op, M=M, Hq=Hq, Hk=max(1, Hq // rng.choice([1, 1, 4])), D=D, axes=rng.choice([1, 2, 3]),
                norm=rng.choice(["rms", "rms", "l2"]), pairs=rng.choice(["halves", "halves", "neighbours"]), io=io)


def _dtype(io):
    return torch.float32 if io == "f32" else torch.bfloat16


def _sections(case):
    """Pairs that turn with each axis: all of a head's, the odd ones to the first."""
    n, P = case["axes"], case["D"] // 2
    return [P - (n - 1) * (P // n)] + [P // n] * (n - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")
    op, dt = case["op"], _dtype(case["io"])
    s = {"case": case}
    if op in ("step", "rule", "train"):
        B, Hk, Hv, dk, dv = (case[k] for k in ("B", "Hk", "Hv", "dk", "dv"))
        # a packed call has one row axis, a batch its sequences
        lead = (B,) if op == "step" else (case["T"],) if case["N"] else (B, case["T"])
        q, k = normal(*lead, Hk, dk), normal(*lead, Hk, dk) + normal(Hk, dk)      # keys have a mean of their own
        s["q"] = (q / q.norm(dim=-1, keepdim=True)).to(dt)
        s["k"] = (k / k.norm(dim=-1, keepdim=True)).to(dt)
        s["v"] = normal(*lead, Hv, dv).to(dt)
        s["beta"] = torch.sigmoid(normal(*lead, Hv))
        # decay times from one to some hundreds of tokens
        rate = torch.exp(-5.5 + 5.0 * uniform(Hv))
        s["decay"] = -rate * torch.nn.functional.softplus(normal(*lead, Hv) + 1.0)
        s["offsets"] = None
        n = B
        if op != "step" and case["N"]:
            n = case["N"]
            end = case["T"] - case["tail"]
            cuts = torch.randint(0, end + 1, (n - 1,), generator=gen, device="cuda").sort().values
            off = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), end)])
            s["offsets"] = off.to(torch.int32)
        s["state"] = normal(n, Hv, dk, dv)
        if op == "rule":
            s["out"] = torch.zeros_like(s["v"])      # rows behind the last sequence stay as they are
        if op == "train":
            s["dy"] = normal(*lead, Hv, dv).to(dt)
            s["dstate"] = 0.1 * normal(n, Hv, dk, dv)
            for name in ("q", "k", "v", "beta", "decay", "state"):
                s[name].requires_grad_(True)
        return s
    M, Hq, Hk, D = (case[k] for k in ("M", "Hq", "Hk", "D"))
    s["q"] = (normal(M, Hq, D) * (0.25 + normal(M, Hq, 1).abs())).to(dt)
    s["k"] = (normal(M, Hk, D) * (0.25 + normal(M, Hk, 1).abs())).to(dt)
    s["wq"], s["wk"] = (1.0 + 0.2 * normal(D), 1.0 + 0.2 * normal(D)) if case["norm"] == "rms" else (None, None)
    # frames of 32 x 32 places, or tokens from far into a sequence
    at = torch.arange(M, device="cuda") + torch.randint(0, 1 << 18, (1,), generator=gen, device="cuda")
    s["positions"] = torch.stack({1: [at], 2: [at // 32 % 32, at % 32], 3: [at // 1024, at // 32 % 32, at % 32]}[case["axes"]],
                                 -1).to(torch.int32)
    # radians a position for each pair, a geometric row of them for each axis, and the axis it turns with
    secs = _sections(case)
    s["freq"] = torch.tensor([10000.0 ** (-j / n) for n in secs for j in range(n)], dtype=torch.float64, device="cuda")
    s["axis"] = torch.tensor([i for i, n in enumerate(secs) for _ in range(n)], dtype=torch.int32, device="cuda")
    if op == "rtrain":
        s["dq"], s["dk"] = normal(M, Hq, D).to(dt), normal(M, Hk, D).to(dt)
        for name in ("q", "k", "wq", "wk"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------ plain forms

def _unit_lower_inverse(m):
    """Inverse of (..., n, n) unit lower triangular matrices, n a power of two: twice as large blocks each time."""
    n = m.shape[-1]
    inv, w = torch.ones((*m.shape[:-1], 1), device=m.device, dtype=m.dtype)[..., None], 1
    while w < n:
        low = torch.stack([m[..., i + w:i + 2 * w, i:i + w] for i in range(0, n, 2 * w)], -3)
        a, c = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        b = -(c @ (low @ a))
        inv = torch.cat([torch.cat([a, torch.zeros_like(a)], -1), torch.cat([b, c], -1)], -2)
        w *= 2
    return inv[..., 0, :, :]


def _padded(s):
    """(rows, lengths): for each sequence and place the row of it, sequences padded to whole chunks of the longest."""
    case = s["case"]
    if s["offsets"] is None:
        B, T = case["B"], case["T"]
        first, length, most = torch.arange(B, device="cuda") * T, torch.full((B,), T, device="cuda"), T
    else:
        off = s["offsets"].long()
        first, length = off[:-1], off[1:] - off[:-1]
        most = int(length.max())
    at = torch.arange(max(1, -(-most // CHUNK)) * CHUNK, device="cuda")
    return first[:, None] + at, at < length[:, None]


def _plain_rule(s, q, k, v, beta, decay, state):
    """(y rows in place, final state) from float32 inputs, CHUNK rows at once."""
    case = s["case"]
    Hv, dk, dv = case["Hv"], case["dk"], case["dv"]
    G, scale = Hv // case["Hk"], dk ** -0.5
    rows, live = _padded(s)
    n, C = rows.shape[0], rows.shape[1] // CHUNK
    idx = torch.where(live, rows, torch.zeros_like(rows)).view(-1)

    def lay(t, heads):                # (n, heads, chunks, CHUNK, width), zero where a sequence has no row
        t = t.reshape(-1, *t.shape[-(2 if t.dim() > beta.dim() else 1):])
        t = t[idx].view(n, C, CHUNK, heads, -1) * live.view(n, C, CHUNK, 1, 1)
        return t.permute(0, 3, 1, 2, 4).contiguous()
    Q, K, V = lay(q, case["Hk"]), lay(k, case["Hk"]), lay(v, Hv)
    Q, K = Q.repeat_interleave(G, 1), K.repeat_interleave(G, 1)
    b, g = lay(beta, Hv), lay(decay, Hv)[..., 0].double().cumsum(-1)
    low = torch.ones((CHUNK, CHUNK), dtype=torch.bool, device="cuda").tril()
    D = torch.where(low, torch.exp(torch.where(low, g[..., :, None] - g[..., None, :], 0.0)), 0.0).float()
    to_start, to_end = torch.exp(g).float()[..., None], torch.exp(g[..., -1:] - g).float()[..., None]
    Kt = K.transpose(-1, -2).contiguous()
    A = (K @ Kt) * D * b
    inv = _unit_lower_inverse(A.tril(-1) + torch.eye(CHUNK, device="cuda"))
    P = (Q @ Kt) * (D * scale)
    W, X = inv @ (b * to_start * K), inv @ (b * V)
    Qs, Ke, whole = Q * to_start * scale, (Kt * to_end.transpose(-1, -2)).contiguous(), to_start[..., -1:, :]
    S, ys = state, []
    for c in range(C):
        U = X[:, :, c] - W[:, :, c] @ S
        ys.append(Qs[:, :, c] @ S + P[:, :, c] @ U)
        S = whole[:, :, c] * S + Ke[:, :, c] @ U
    y = torch.stack(ys, 2).permute(0, 2, 3, 1, 4).reshape(n * C * CHUNK, Hv, dv)
    keep = live.view(-1)
    out = torch.zeros((v.numel() // (Hv * dv), Hv, dv), device="cuda")
    return out.index_copy(0, rows.view(-1)[keep], y[keep]).view(v.shape), S


def _angles(s):
    """cos and sin (M, 1, D / 2) of each row's pairs, from angles in 64 bits."""
    a = s["positions"].double()[:, s["axis"].long()] * s["freq"]
    return torch.cos(a)[:, None], torch.sin(a)[:, None]


def _turn(x, cos, sin, pairs):
    if pairs == "halves":
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)


def _plain_rotate(s):
    case = s["case"]
    cos, sin = (t.float() for t in _angles(s))
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        v = x.float()
        sq = (v * v).mean(-1, keepdim=True) if case["norm"] == "rms" else (v * v).sum(-1, keepdim=True)
        v = v * torch.rsqrt(sq + EPS)
        out.append(_turn(v if w is None else v * w, cos, sin, case["pairs"]).to(x.dtype))
    return out


def run(s):
    case, op = s["case"], s["case"]["op"]
    if own:
        from cssm_amd import sequence, training
        if op == "step":
            y, state = sequence.delta_rule_step(s["q"], s["k"], s["v"], s["beta"], s["state"], decay=s["decay"])
            return {"y": y, "state": state}
        if op == "rule":
            y, state = sequence.delta_rule(s["q"], s["k"], s["v"], s["beta"], decay=s["decay"], state=s["state"],
                                           offsets=s["offsets"], out=s["out"])
            return {"y": y, "state": state}
        if op == "train":
            y, state = training.delta_rule_train(s["q"], s["k"], s["v"], s["beta"], decay=s["decay"], state=s["state"],
                                                 offsets=s["offsets"])
        elif op == "rotate":
            q, k = sequence.rotate_heads(s["q"], s["k"], s["positions"], (s["freq"], s["axis"]), q_weight=s["wq"], k_weight=s["wk"],
                                         norm=case["norm"], eps=EPS, pairs=case["pairs"])
            return {"q": q, "k": k}
        else:
            q, k = training.rotate_heads_train(s["q"], s["k"], s["positions"], (s["freq"], s["axis"]), q_weight=s["wq"],
                                               k_weight=s["wk"], norm=case["norm"], eps=EPS, pairs=case["pairs"])
    elif op == "step":
        G = case["Hv"] // case["Hk"]
        q, k = (s[n].float().repeat_interleave(G, 1) for n in ("q", "k"))
        S = torch.exp(s["decay"])[..., None, None] * s["state"]
        e = s["v"].float() - (k[..., None] * S).sum(-2)
        S = S + k[..., None] * (s["beta"][..., None] * e)[..., None, :]
        return {"y": ((q * case["dk"] ** -0.5)[..., None] * S).sum(-2).to(s["v"].dtype), "state": S}
    elif op == "rule":
        y, state = _plain_rule(s, *(s[n].float() for n in ("q", "k", "v", "beta", "decay", "state")))
        out = s["out"].clone()
        end = y.shape[0] - case["tail"] if case["N"] else None
        out[:end] = y[:end].to(out.dtype)
        return {"y": out, "state": state}
    elif op == "train":
        y, state = _plain_rule(s, *(s[n].float() for n in ("q", "k", "v", "beta", "decay", "state")))
        y = y.to(s["v"].dtype)
    elif op == "rotate":
        q, k = _plain_rotate(s)
        return {"q": q, "k": k}
    else:
        q, k = _plain_rotate(s)
    if op == "train":
        names = ["q", "k", "v", "beta", "decay", "state"]
        grads = torch.autograd.grad((y, state), [s[n] for n in names], (s["dy"], s["dstate"]))
        return {"y": y.detach(), "state": state.detach(), **{"d" + n: g for n, g in zip(names, grads)}}
    names = [n for n in ("q", "k", "wq", "wk") if s[n] is not None]
    grads = torch.autograd.grad((q, k), [s[n] for n in names], (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def work(case):
    op, size = case["op"], 4 if case["io"] == "f32" else 2
    if op in ("rotate", "rtrain"):
        el = case["M"] * (case["Hq"] + case["Hk"]) * case["D"]
        ends = case["M"] * case["axes"] * 4
        # rotate: x in, y out; training also dy in and dx out
        return {"bytes": (4 if op == "rtrain" else 2) * size * el + ends, "flops": (24 if op == "rtrain" else 10) * el}
    Hk, Hv, dk, dv = (case[k] for k in ("Hk", "Hv", "dk", "dv"))
    rows = case["B"] * (case["T"] - case["tail"] if op != "step" else 1)
    n = case["N"] or case["B"] if op != "step" else case["B"]
    qk, vo, gates, states = rows * Hk * dk * 2 * size, rows * Hv * dv * 2 * size, rows * Hv * 8, n * Hv * dk * dv * 8
    # a token's products with the state: read by the key, written by the key, read by the query
    flops = 6 * rows * Hv * dk * dv
    if op == "train":
        # q, k, v and dy in, y and the gradients out; the adjoint has two products for each of the forward's
        return {"bytes": 2 * qk + 2 * vo + 2 * gates + 2 * states, "flops": 3 * flops}
    return {"bytes": qk + vo + gates + states, "flops": flops}


# ------------------------------------------------------------------ 64 bits, token by token

def _exact_rule(case, d, off):
    B, T, Hk, Hv = case["B"], case["T"], case["Hk"], case["Hv"]
    G, scale, flat = Hv // Hk, case["dk"] ** -0.5, off is not None
    lengths = [b - a for a, b in zip(off, off[1:])] if flat else [T] * B
    firsts = off[:-1] if flat else [i * T for i in range(B)]
    order = sorted(range(len(lengths)), key=lambda i: -lengths[i])       # the longest first: those alive are a prefix
    dev = d["v"].device
    start = torch.tensor([firsts[i] for i in order], device=dev)
    alive = [sum(l > t for l in lengths) for t in range(max(lengths) if lengths else 0)]
    flatten = {n: d[n].reshape(-1, *d[n].shape[(1 if flat else 2):]) for n in ("q", "k", "v", "beta", "decay")}
    perm = torch.tensor(order, device=dev)

    def token(t):
        r = start[:alive[t]] + t
        q, k = (flatten[n][r].repeat_interleave(G, 1)[..., None] for n in ("q", "k"))
        return r, q, k, flatten["v"][r], flatten["beta"][r][..., None], torch.exp(flatten["decay"][r])[..., None, None]

    def advance(S, t):
        r, q, k, v, b, a = token(t)
        Z = a * S[:alive[t]]
        e = v - (k * Z).sum(-2)
        return r, q, k, b, a, Z, e, Z + k * (b * e)[..., None, :]
    S, y, kept, every = d["state"][perm].clone(), torch.zeros_like(flatten["v"]), [], 64
    for t in range(len(alive)):
        if t % every == 0:
            kept.append(S.clone())
        r, q, _, _, _, _, _, new = advance(S, t)
        S[:alive[t]] = new
        y[r] = scale * (q * new).sum(-2)
    back = torch.empty_like(perm)
    back[perm] = torch.arange(len(order), device=dev)
    got = {"y": y.view(d["v"].shape), "state": S[back]}
    if "dy" not in d:
        return got
    dy = d["dy"].reshape(flatten["v"].shape)
    grads = {n: torch.zeros_like(flatten[n]) for n in flatten}
    D = d["dstate"][perm].clone()

    def group(x):                       # the value heads' shares of one key head
        return x.view(x.shape[0], Hk, G, -1).sum(2)
    for c in range(len(kept) - 1, -1, -1):
        S, steps = kept[c], []
        for t in range(c * every, min((c + 1) * every, len(alive))):
            steps.append(advance(S, t))
            S = torch.cat([steps[-1][-1], S[alive[t]:]])
        for t in range(min((c + 1) * every, len(alive)) - 1, c * every - 1, -1):
            r, q, k, b, a, Z, e, new = steps[t - c * every]
            g = dy[r][..., None, :]
            H = D[:alive[t]] + scale * q * g
            grads["q"][r] = group(scale * (new * g).sum(-1))
            du = (H * k).sum(-2)
            de = b * du
            grads["beta"][r] = (du * e).sum(-1)
            grads["v"][r] = de
            dZ = H - k * de[..., None, :]
            grads["k"][r] = group((H * (b * e)[..., None, :]).sum(-1) - (Z * de[..., None, :]).sum(-1))
            grads["decay"][r] = (dZ * Z).sum((-1, -2))
            D[:alive[t]] = a * dZ
    got.update({"d" + n: grads[n].view(d[n].shape) for n in grads})
    got["dstate"] = D[back]
    return got


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if op == "step":
        G = case["Hv"] // case["Hk"]
        q, k = (d[n].repeat_interleave(G, 1) for n in ("q", "k"))
        Z = torch.exp(d["decay"])[..., None, None] * d["state"]
        e = d["v"] - torch.matmul(k[..., None, :], Z)[..., 0, :]
        S = Z + torch.matmul(k[..., None], (d["beta"][..., None] * e)[..., None, :])
        return {"y": torch.matmul(q[..., None, :], S)[..., 0, :] / math.sqrt(case["dk"]), "state": S}
    if op in ("rule", "train"):
        return _exact_rule(case, d, None if s["offsets"] is None else s["offsets"].tolist())
    M, D = case["M"], case["D"]
    angle = torch.empty((M, D // 2), dtype=torch.float64, device="cuda")
    at = 0
    for i, n in enumerate(_sections(case)):
        for j in range(n):
            angle[:, at + j] = s["positions"][:, i].double() * math.exp(-math.log(10000.0) * j / n)
        at += n
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    half = case["pairs"] == "halves"

    def paired(x):
        return torch.complex(x[..., :D // 2], x[..., D // 2:]) if half else torch.view_as_complex(
            x.reshape(*x.shape[:-1], D // 2, 2).contiguous())

    def apart(z):
        return torch.cat([z.real, z.imag], -1) if half else torch.view_as_real(z).flatten(-2)
    got = {}
    for name, w in (("q", "wq"), ("k", "wk")):
        x = d[name]
        count = D if case["norm"] == "rms" else 1
        r = 1.0 / torch.sqrt((x ** 2).sum(-1, keepdim=True) / count + EPS)
        wt = d.get(w, torch.ones(D, dtype=torch.float64, device="cuda"))
        got[name] = apart(paired(x * r * wt) * turn)
        if op == "rtrain":
            back = apart(paired(d["d" + name]) * turn.conj())
            t = back * wt
            got["d" + name] = r * t - x * r ** 3 / count * (t * x).sum(-1, keepdim=True)
            if w in d:
                got["d" + w] = (back * x * r).sum((0, 1))
    return got
