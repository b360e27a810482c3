"""The operators over token sequences that this framework is timed on, through its public entry points.

A case's ``op`` names one:
  step      one token of the gated recurrence for each sequence of a batch, with its state
  scan      the gated recurrence over whole sequences: a (B, T, C) batch, or rows packed one sequence behind the other
  train     the recurrence forward and backward, on its inputs or on checkpoints in 8 bits
  norm      root-mean-square norm of x + residual with the output in 8 bits and a scale for each 128 of a row
  ntrain    the norm forward and backward, in the inputs' type
  product   matrix product of 8-bit rows and an 8-bit weight with a scale for each block of 128

The recurrence, for each channel: D = softplus(delta + bias), h_t = kappa exp(-D_t) h_{t-1} + D_t x_t and
y_t = h_t SiLU(z_t).  Where ``own`` is false ``run`` computes these in elementary torch operations.
"""
import torch

own = False

SEGMENT = 128          # rows between the states that a checkpoint keeps
EPS = 1e-6


def listed():
    return [
        # serving: one token for a small batch, the smallest call
        dict(name="step_16", op="step", B=16, C=1024, io="bf16", gate=True),
        # the tokens of a few small images in odd sizes, continued from a state, without the readout gate
        dict(name="scan_odd", op="scan", B=3, T=197, C=100, N=0, tail=0, io="f32", gate=False),
        # one very long sequence, where only the time axis offers parallel work
        dict(name="scan_long", op="scan", B=1, T=65536, C=1024, N=0, tail=0, io="bf16", gate=True),
        # a serving prefill: ragged sequences packed behind each other, some empty, padding rows behind the last
        dict(name="scan_packed", op="scan", B=1, T=16001, C=2048, N=23, tail=77, io="bf16", gate=True),
        # a training step on long sequences
        dict(name="train_4096", op="train", B=8, T=4096, C=1024, N=0, tail=0, io="bf16", gate=True, bits=16),
        # the same step keeping its activations in 8 bits
        dict(name="train_4096_e4m3", op="train", B=8, T=4096, C=1024, N=0, tail=0, io="bf16", gate=True, bits=8),
        # a small float32 training step with 8-bit checkpoints at sizes off every block
        dict(name="train_odd_e4m3", op="train", B=2, T=1001, C=228, N=0, tail=0, io="f32", gate=True, bits=8),
        # the norm before an 8-bit projection in a large prefill
        dict(name="norm_prefill", op="norm", M=16384, C=4096, io="bf16", residual=True),
        # the same for the tokens of one serving step
        dict(name="norm_token", op="norm", M=16, C=1024, io="bf16", residual=True),
        # the norm in training
        dict(name="ntrain_32768", op="ntrain", M=32768, C=1024, io="bf16", residual=True),
        # a projection of a large prefill: the matrix cores' rate
        dict(name="product_prefill", op="product", M=8192, N=8192, K=4096, out="bf16", act="none"),
        # the same projection for the tokens of one serving step: the weight's bytes
        dict(name="product_token", op="product", M=16, N=8192, K=4096, out="bf16", act="silu"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "train", "train", "norm", "ntrain", "product", "product"])
    io = rng.choice(["bf16", "bf16", "f32"])
    if op == "step":
        return dict(op=op, B=_log(rng, 1, 512), C=_log(rng, 32, 8192), io=io, gate=rng.random() < 0.7)
    if op in ("scan", "train"):
        most = (1 << 25) if op == "scan" else (1 << 24)
        C = _log(rng, 17, 4096) if rng.random() < 0.5 else 8 * _log(rng, 4, 512)
        T = _log(rng, 1, 65536)
        packed = rng.random() < 0.4
        B = 1 if packed else _log(rng, 1, 32)
        while B * T * C > most:
            B, T = max(1, B // 2), max(1, T - T // 3)
        case = dict(op=op, B=B, T=T, C=C, N=rng.randint(1, 40) if packed else 0,
                    tail=min(T - 1, rng.choice([0, 0, 5, 130])) if packed else 0, io=io, gate=rng.random() < 0.8)
        if op == "train":
            case["bits"] = rng.choice([8, 16])
        return case
    if op in ("norm", "ntrain"):
        M, C = _log(rng, 1, 32768), _log(rng, 16, 8192)
        while M * C > (1 << 24):
            M = M - M // 3
        return dict(op=op, M=M, C=C, io=io, residual=rng.random() < 0.7)
    M, N, K = _log(rng, 1, 8192), _log(rng, 16, 8192), 16 * _log(rng, 4, 512)
    while M * N * K > (1 << 37):
        M = M - M // 3
    return dict(op=op, M=M, N=N, K=K, out=rng.choice(["bf16", "f32"]), act=rng.choice(["none", "silu", "gelu"]))


def _dtype(io):
    return torch.float32 if io == "f32" else torch.bfloat16


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    op = case["op"]
    s = {"case": case}
    if op in ("step", "scan", "train"):
        B, C, dt = case["B"], case["C"], _dtype(case["io"])
        # a packed call has one row axis, a batch its sequences
        lead = (B,) if op == "step" else (case["T"],) if case["N"] else (B, case["T"])
        s["x"] = normal(*lead, C).to(dt)
        # decay times from a few to a few hundred tokens: the bias spreads softplus over two decades
        s["delta"] = (0.5 * normal(*lead, C)).to(dt)
        s["bias"] = -5.0 + 5.0 * torch.rand((C,), generator=gen, device="cuda")
        s["kappa"] = 0.98 + 0.02 * torch.rand((C,), generator=gen, device="cuda")
        s["z"] = normal(*lead, C).to(dt) if case["gate"] else None
        s["starts"] = s["offsets"] = None
        n = B
        if op != "step" and case["N"]:
            n = case["N"]
            end = case["T"] - case["tail"]
            cuts = torch.randint(0, end + 1, (n - 1,), generator=gen, device="cuda").sort().values
            off = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), end)])
            s["offsets"] = off.to(torch.int32)
        s["state"] = normal(n, C)
        if op != "step":
            s["out"] = torch.zeros_like(s["x"])      # rows behind the last sequence stay as they are
        if op == "train":
            s["dy"] = normal(*lead, C).to(dt)
            s["dstate"] = normal(n, C)
            for k in ("x", "delta", "z", "kappa", "bias", "state"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    elif op in ("norm", "ntrain"):
        M, C, dt = case["M"], case["C"], _dtype(case["io"])
        s["x"] = (normal(M, C) * (0.25 + normal(M, 1).abs())).to(dt)
        s["residual"] = normal(M, C).to(dt) if case["residual"] else None
        s["weight"] = 1.0 + 0.2 * normal(C)
        if op == "ntrain":
            s["dy"], s["ds"] = normal(M, C).to(dt), (0.1 * normal(M, C)).to(dt)
            for k in ("x", "residual", "weight"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    else:
        M, N, K = case["M"], case["N"], case["K"]
        s["a"], s["sa"] = _rows8(normal(M, K) * (0.25 + normal(M, 1).abs()))
        s["w"], s["sw"] = _tiles8(normal(N, K) / K ** 0.5)
        s["bias"] = 0.1 * normal(N)
    return s


# ------------------------------------------------------------------ plain forms

def _exponent(top):
    """The least e with top <= 448 * 2^e (0 for a block of zeros), 448 the largest e4m3 value."""
    m, k = torch.frexp(top)                                   # top = m 2^k, m in [0.5, 1)
    e = torch.where(m > 0.875, k - 8, k - 9)
    return torch.where(top > 0, e, torch.zeros_like(e)).clamp(-126, 127)


def _pow2(e):
    return ((e.int() + 127) << 23).view(torch.float32)      # by its bits: ldexp is off by a rounding at some e


def _blocks8(v, rows, cols):
    """(..., M, K) values -> e4m3 of the same shape and the power of two of each rows x cols block."""
    *lead, M, K = v.shape
    m, k = -(-M // rows), -(-K // cols)
    p = torch.nn.functional.pad(v, (0, k * cols - K, 0, m * rows - M)).view(*lead, m, rows, k, cols)
    e = _exponent(p.abs().amax(dim=(-3, -1)))
    q = (p * _pow2(-e)[..., :, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(*lead, m * rows, k * cols)[..., :M, :K].contiguous(), _pow2(e)


def _rows8(v):
    q, s = _blocks8(v, 1, 128)
    return q, s.to(torch.float8_e8m0fnu)


def _tiles8(v):
    q, s = _blocks8(v, 128, 128)
    return q, s.to(torch.float8_e8m0fnu)


def _spread(s, rows, cols, M, K):
    """A block's scale for each of its values."""
    return s.float().repeat_interleave(rows, -2)[..., :M, :].repeat_interleave(cols, -1)[..., :K]


def _kept8(v):
    """(B, T, C) values as their 8-bit checkpoint gives them back: 8 rows x 16 channels share a power of two."""
    q, s = _blocks8(v, 8, 16)
    return q.float() * _spread(s, 8, 16, *v.shape[1:])


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1, h_{-1} = 0: pairs of spans joined, twice as long each time."""
    k, T = 1, a.shape[1]
    while k < T:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _gains(delta, bias):
    """softplus(u) and exp(-softplus(u)) = sigmoid(-u) of u = delta + bias."""
    u = delta + bias
    return u.clamp(min=0.0) + torch.log1p(torch.exp(-u.abs())), torch.sigmoid(-u)


def _silu(z):
    return z * torch.sigmoid(z)


def _layout(s):
    """The sequences as (B, T, C) float32 with the first and last row of each sequence and its number there."""
    case = s["case"]
    three = [None if s[k] is None else s[k].detach().float() for k in ("x", "delta", "z")]
    if s["offsets"] is None:
        B, T = case["B"], case["T"]
        n = torch.arange(B, device="cuda")
        first, last, full = (n, torch.zeros_like(n)), (n, torch.full_like(n, T - 1)), n
    else:
        off = s["offsets"].long()
        full = torch.nonzero(off[1:] > off[:-1])[:, 0]         # sequences that are not empty
        zero = torch.zeros_like(full)
        first, last = (zero, off[:-1][full]), (zero, off[1:][full] - 1)
        end = case["T"] - case["tail"]
        three = [None if t is None else t[None, :end] for t in three]
    return three, first, last, full


def _plain_scan(s):
    (x, delta, z), first, last, full = _layout(s)
    D, sg = _gains(delta, s["bias"].detach())
    h0 = s["state"].detach()
    a, b = s["kappa"].detach() * sg, D * x
    b[first] += a[first] * h0[full]
    a[first] = 0.0
    h = _scan(a, b)
    hT = h0.clone()
    hT[full] = h[last]
    y = h if z is None else h * _silu(z)
    out = s["out"].detach().clone().view(-1, y.shape[-1])
    rows = y.reshape(-1, y.shape[-1])
    out[:rows.shape[0]] = rows.to(out.dtype)
    return out.view(s["out"].shape), hT, h


def _plain_train(s):
    y, hT, h = _plain_scan(s)
    (x, delta, z), first, last, full = _layout(s)
    kappa, bias, h0 = s["kappa"].detach(), s["bias"].detach(), s["state"].detach()
    dy = s["dy"].float()
    dy = dy[None, :x.shape[1]] if s["offsets"] is not None else dy
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    before[first] = h0[full]
    if s["case"]["bits"] == 8:
        x, delta, z = (None if t is None else _kept8(t) for t in (x, delta, z))
    D, sg = _gains(delta, bias)
    a = kappa * sg
    if s["case"]["bits"] == 8:
        # the states between, from those before every 128th row and at the starts
        c, b = a.clone(), D * x
        b[:, ::SEGMENT] += a[:, ::SEGMENT] * before[:, ::SEGMENT]
        c[:, ::SEGMENT] = 0.0
        inner = first[1] % SEGMENT != 0
        at = (first[0][inner], first[1][inner])
        b[at] += a[at] * before[at]
        c[at] = 0.0
        h = _scan(c, b)
        kept = before
        before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
        before[:, ::SEGMENT] = kept[:, ::SEGMENT]
        before[first] = kept[first]
    sz = None if z is None else torch.sigmoid(z)
    u = dy if z is None else dy * (z * sz)
    u = u.clone()
    u[last] += s["dstate"][full]
    nxt = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    nxt[last] = 0.0
    g = _scan(nxt.flip(1), u.flip(1)).flip(1)
    dd = g * (x - a * before) * torch.sigmoid(delta + bias)
    dh0 = s["dstate"].clone()
    dh0[full] = (a * g)[first]

    def back(v):
        out = torch.zeros(s["x"].shape, dtype=s["x"].dtype, device="cuda").view(-1, v.shape[-1])
        out[:v.shape[0] * v.shape[1]] = v.reshape(-1, v.shape[-1]).to(out.dtype)
        return out.view(s["x"].shape)
    return {"y": y, "state": hT, "dx": back(D * g), "ddelta": back(dd),
            "dz": None if z is None else back(dy * h * (sz * (1.0 + z * (1.0 - sz)))),
            "dkappa": (g * sg * before).sum((0, 1)), "dbias": dd.sum((0, 1)), "dstate": dh0}


def _plain_norm(s):
    x = s["x"].detach()
    if s["residual"] is not None:
        x = (x.float() + s["residual"].detach().float()).to(x.dtype)
    v = x.float()
    rstd = torch.rsqrt((v * v).mean(1, keepdim=True) + EPS)
    return x, v, rstd


def run(s):
    case, op = s["case"], s["case"]["op"]
    if own:
        from cssm_amd import sequence, training
        if op == "step":
            y, state = sequence.token_scan_step(s["x"], s["delta"], s["kappa"], s["bias"], s["state"], z=s["z"])
            return {"y": y, "state": state}
        if op == "scan":
            y, state = sequence.token_scan(s["x"], s["delta"], s["kappa"], s["bias"], z=s["z"], state=s["state"],
                                           offsets=s["offsets"], out=s["out"])
            return {"y": y, "state": state}
        if op == "train":
            y, state = training.token_scan_train(s["x"], s["delta"], s["kappa"], s["bias"], z=s["z"],
                                                 state=s["state"], offsets=s["offsets"],
                                                 checkpoint="e4m3" if case["bits"] == 8 else "none")
            names = [k for k in ("x", "delta", "z", "kappa", "bias", "state") if s[k] is not None]
            grads = torch.autograd.grad((y, state), [s[k] for k in names], (s["dy"], s["dstate"]))
            return {"y": y.detach(), "state": state.detach(), **{"d" + k: g for k, g in zip(names, grads)}}
        if op == "norm":
            y, stream = sequence.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, out="e4m3")
            return {"q": y.values, "scales": y.scales, "stream": stream}
        if op == "ntrain":
            y, stream = training.rms_norm_train(s["x"], s["weight"], residual=s["residual"], eps=EPS)
            names = [k for k in ("x", "residual", "weight") if s[k] is not None]
            grads = torch.autograd.grad((y, stream) if s["residual"] is not None else y, [s[k] for k in names],
                                        (s["dy"], s["ds"]) if s["residual"] is not None else s["dy"])
            return {"y": y.detach(), "stream": stream.detach(), **{"d" + k: g for k, g in zip(names, grads)}}
        return sequence.scaled_matmul(sequence.Blocks8(s["a"], s["sa"]), sequence.Blocks8(s["w"], s["sw"]),
                                      bias=s["bias"], act=case["act"], out_dtype=_dtype(case["out"]))
    if op == "step":
        x, delta = s["x"].float(), s["delta"].float()
        D, sg = _gains(delta, s["bias"])
        h = s["kappa"] * sg * s["state"] + D * x
        y = h if s["z"] is None else h * _silu(s["z"].float())
        return {"y": y.to(s["x"].dtype), "state": h}
    if op == "scan":
        y, state, _ = _plain_scan(s)
        return {"y": y, "state": state}
    if op == "train":
        return {k: v for k, v in _plain_train(s).items() if v is not None}
    if op == "norm":
        x, v, rstd = _plain_norm(s)
        q, e = _rows8(v * rstd * s["weight"])
        return {"q": q, "scales": e, "stream": x}
    if op == "ntrain":
        x, v, rstd = _plain_norm(s)
        n = v * rstd
        w, dy = s["weight"].detach(), s["dy"].float()
        t = w * dy
        dx = rstd * (t - n * (t * n).mean(1, keepdim=True))
        if s["residual"] is not None:
            dx = dx + s["ds"].float()
        dx = dx.to(x.dtype)
        got = {"y": (n * w).to(x.dtype), "stream": x, "dx": dx, "dweight": (dy * n).sum(0)}
        return got if s["residual"] is None else {**got, "dresidual": dx}
    M, K = s["a"].shape
    N = s["w"].shape[0]
    c = (s["a"].float() * _spread(s["sa"], 1, 128, M, K)) @ (s["w"].float() * _spread(s["sw"], 128, 128, N, K)).t()
    c = c + s["bias"]
    if case["act"] == "silu":
        c = _silu(c)
    elif case["act"] == "gelu":
        c = 0.5 * c * (1.0 + torch.tanh(0.7978845608028654 * (c + 0.044715 * c * c * c)))
    return c.to(_dtype(case["out"]))


def work(case):
    op = case["op"]
    size = 4 if case.get("io") == "f32" else 2
    if op in ("step", "scan", "train"):
        rows = case["B"] * (case["T"] - case["tail"] if op != "step" else 1)
        el = rows * case["C"]
        n = (case["N"] or case["B"]) if op != "step" else case["B"]
        ends = 8 * n * case["C"] + 8 * case["C"]              # states in and out, kappa and bias
        gate = int(case["gate"])
        if op != "train":
            return {"bytes": (3 + gate) * size * el + ends, "flops": 25 * el}
        # x, delta, z and dy in, y and their gradients out
        return {"bytes": (6 + 2 * gate) * size * el + 2 * ends, "flops": 75 * el}
    if op in ("norm", "ntrain"):
        el = case["M"] * case["C"]
        r = int(case["residual"])
        if op == "norm":
            return {"bytes": (1 + 2 * r) * size * el + el + el // 128, "flops": 8 * el}
        return {"bytes": (4 + 3 * r) * size * el, "flops": 20 * el}
    M, N, K = case["M"], case["N"], case["K"]
    out = 4 if case["out"] == "f32" else 2
    return {"bytes": (M + N) * K + M * N * out + 4 * N, "flops": 2 * M * N * K}


# ------------------------------------------------------------------ 64 bits, row by row

def _two(e):
    """2^e in float64 by its bits (pow is off by a rounding at some exponents)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact8(v, rows, cols):
    """(M, K) float64 -> the nearest values of 3 mantissa bits (ties to even) under the blocks' powers of two."""
    M, K = v.shape
    r = torch.arange(M, device=v.device) // rows
    c = torch.arange(K, device=v.device) // cols
    top = torch.zeros((int(r[-1]) + 1, int(c[-1]) + 1), dtype=v.dtype, device=v.device)
    top.view(-1).scatter_reduce_(0, (r[:, None] * top.shape[1] + c).view(-1), v.abs().reshape(-1), "amax")
    e = torch.ceil(torch.log2((top / 448.0).clamp(min=2.0 ** -126)))
    e = torch.where(448.0 * _two(e - 1) >= top, e - 1, e)      # log2 may land a step high or low
    e = torch.where(448.0 * _two(e) < top, e + 1, e)
    e = torch.where(top > 0, e.clamp(-126, 127), torch.zeros_like(e))
    scale = _two(e)[r][:, c]
    t = v / scale
    step = _two(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(t / step) * step, scale, _two(e)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    d = {k: (v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v)
         for k, v in s.items() if k not in ("a", "w", "sa", "sw")}

    def gains(delta):
        u = delta + d["bias"]
        return torch.clamp(u, min=0) + torch.log1p(torch.exp(-u.abs())), 1.0 / (1.0 + torch.exp(u))
    if op == "step":
        D, sg = gains(d["delta"])
        h = d["kappa"] * sg * d["state"] + D * d["x"]
        return {"y": h if d["z"] is None else h * d["z"] / (1.0 + torch.exp(-d["z"])), "state": h}
    if op in ("scan", "train"):
        C = case["C"]
        flat = d["x"].dim() == 2
        end = case["T"] - case["tail"]
        t3 = [None if d[k] is None else (d[k][None] if flat else d[k]) for k in ("x", "delta", "z")]
        x, delta, z = t3
        off = s["offsets"].tolist() if flat else None
        begins = {}                                          # row -> the sequence that starts there
        ends = {}
        if flat:
            for i in range(case["N"]):
                if off[i + 1] > off[i]:
                    begins[off[i]], ends[off[i + 1] - 1] = i, i

        def forward(D, a, keep=None):
            """States after each row; keep: states before the rows, taken at every 128th."""
            h, hs, was = None, [], []
            for t in range(end):
                if flat and t in begins:
                    h = d["state"][begins[t]][None]
                elif not flat and t == 0:
                    h = d["state"]
                elif keep is not None and t % SEGMENT == 0:
                    h = keep[t]
                was.append(h)
                h = torch.addcmul(D[:, t], a[:, t], h)
                hs.append(h)
            return hs, was
        D, sg = gains(delta)
        hs, was = forward(D * x, d["kappa"] * sg)
        hT = d["state"].clone()
        if flat:
            for t, i in ends.items():
                hT[i] = hs[t][0]
        else:
            hT = hs[-1]
        h = torch.stack(hs, 1)
        rest = torch.zeros((x.shape[0], case["T"] - end, C), dtype=h.dtype, device=h.device)

        def whole(v):
            v = torch.cat([v, rest], 1)
            return v[0] if flat else v
        zz = None if z is None else z[:, :end]
        y = h if z is None else h * zz / (1.0 + torch.exp(-zz))
        got = {"y": whole(y), "state": hT}
        if op == "scan":
            return got
        x, delta = x[:, :end], delta[:, :end]
        dy = (d["dy"][None] if flat else d["dy"])[:, :end]
        if case["bits"] == 8:
            def kept(v):
                return torch.stack([q * sc for q, sc, _ in (_exact8(p, 8, 16) for p in v)])
            x, delta = kept(x), kept(delta)
            zz = None if z is None else kept(zz)
            D, sg = gains(delta)
            hs, was = forward(D * x, d["kappa"] * sg, was)
            h = torch.stack(hs, 1)
        else:
            D, sg = D[:, :end], sg[:, :end]
        was = torch.stack(was, 1)
        a = d["kappa"] * sg
        sz = None if z is None else 1.0 / (1.0 + torch.exp(-zz))
        u = dy if z is None else dy * zz * sz
        g, gs = None, [None] * end
        dh0 = d["dstate"].clone()
        for t in range(end - 1, -1, -1):
            if flat and t in ends:
                g = u[:, t] + d["dstate"][ends[t]][None]
            elif not flat and t == end - 1:
                g = u[:, t] + d["dstate"]
            else:
                g = torch.addcmul(u[:, t], a[:, t + 1], g)
            gs[t] = g
            if flat and t in begins:
                dh0[begins[t]] = (a[:, t] * g)[0]
        g = torch.stack(gs, 1)
        if not flat:
            dh0 = a[:, 0] * g[:, 0]
        dd = g * (x - a * was) / (1.0 + torch.exp(-delta - d["bias"]))
        got.update(dx=whole(D * g), ddelta=whole(dd), dkappa=(g * sg * was).sum((0, 1)), dbias=dd.sum((0, 1)),
                   dstate=dh0)
        if z is not None:
            got["dz"] = whole(dy * h * sz * (1.0 + zz * (1.0 - sz)))
        return got
    if op in ("norm", "ntrain"):
        v = d["x"]
        if d["residual"] is not None:
            v = (d["x"] + d["residual"]).to(s["x"].dtype).double()
        rstd = 1.0 / torch.sqrt((v ** 2).sum(1, keepdim=True) / case["C"] + EPS)
        n = v * rstd
        if op == "norm":
            q, _, e = _exact8(n * d["weight"], 1, 128)
            return {"q": q, "scales": e, "stream": v}
        t = d["dy"] * d["weight"]
        dx = rstd * t - n * rstd * (t * n).sum(1, keepdim=True) / case["C"]
        got = {"y": n * d["weight"], "stream": v, "dweight": (d["dy"] * n).sum(0)}
        if d["residual"] is not None:
            got["dresidual"] = dx + d["ds"]
        return {**got, "dx": dx + d["ds"] if d["residual"] is not None else dx}
    M, N, K = case["M"], case["N"], case["K"]
    at = torch.arange(K, device="cuda") // 128
    A = s["a"].float().double() * s["sa"].float().double()[:, at]
    W = s["w"].float().double() * s["sw"].float().double()[torch.arange(N, device="cuda") // 128][:, at]
    c = A @ W.t() + d["bias"]
    if case["act"] == "silu":
        c = c / (1.0 + torch.exp(-c))
    elif case["act"] == "gelu":
        c = 0.5 * c * (1.0 + torch.tanh((2.0 / torch.pi) ** 0.5 * (c + 0.044715 * c ** 3)))
    return c
