"""Timed work of the sequence operators: rotary positions, differential attention, the gated linear recurrence and group
normalisation with an activation, on time-major (batch, time, channels) tensors.

`own` false: every operator in its plain form, elementary torch operations in 32 bits (angles in 64).  `own` true: the same passes
through this package's entry points (xva_trainer_amd.seq_ops).  `exact` restates each operator in 64 bits, with gradients written
out from the formulas instead of taken by autograd.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
TURN = 2.0 * math.pi


# ------------------------------------------------------------------------------------------------------------------ cases ----
def listed():
    return [
        # one new token of each of 64 streams at far positions, part of each head rotated (interleaved pairs), angles scaled for long contexts
        {"name": "rotary_step", "op": "rotary", "dtype": "float16", "B": 64, "T": 1, "H": 16, "Hk": 4, "D": 96, "rd": 64, "interleaved": True,
         "scaling": "yarn", "factor": 16.0, "first": 40000, "grad": False},
        # queries and keys of a long document, whole heads in the half layout, with the gradient
        {"name": "rotary_long", "op": "rotary", "dtype": "bfloat16", "B": 2, "T": 16384, "H": 16, "Hk": 4, "D": 128, "rd": 128, "interleaved": False,
         "scaling": "none", "factor": 1.0, "first": 0, "grad": True},
        # one new token of each of 16 streams against ragged caches of up to 8192 keys, four query heads to a key head
        {"name": "diff_step", "op": "diff", "dtype": "bfloat16", "B": 16, "Tq": 1, "Tk": 8192, "H": 16, "Hk": 4, "d": 64, "causal": True, "ragged": True,
         "grad": False},
        # training step of a text encoder: 32 texts of up to 150 symbols
        {"name": "diff_text", "op": "diff", "dtype": "bfloat16", "B": 32, "Tq": 150, "Tk": 150, "H": 4, "Hk": 4, "d": 32, "causal": False, "ragged": True,
         "grad": True},
        # training step of a mel decoder: 32 clips of up to 860 frames, heads of 96 (two halves of 48)
        {"name": "diff_frames", "op": "diff", "dtype": "float16", "B": 32, "Tq": 860, "Tk": 860, "H": 4, "Hk": 2, "d": 48, "causal": False, "ragged": True,
         "grad": True},
        # training step on one long causal sequence
        {"name": "diff_long", "op": "diff", "dtype": "bfloat16", "B": 1, "Tq": 8192, "Tk": 8192, "H": 16, "Hk": 4, "d": 64, "causal": True, "ragged": False,
         "grad": True},
        # one new frame of each of 64 streams
        {"name": "recurrence_step", "op": "recurrence", "dtype": "bfloat16", "B": 64, "T": 1, "C": 1024, "reverse": False, "gain": "convex", "ragged": False,
         "grad": False},
        # training step over 32 clips of up to 860 frames
        {"name": "recurrence_frames", "op": "recurrence", "dtype": "bfloat16", "B": 32, "T": 860, "C": 384, "reverse": False, "gain": "convex", "ragged": True,
         "grad": True},
        # training step over long sequences in 32 bits, from the end to the start
        {"name": "recurrence_long", "op": "recurrence", "dtype": "float32", "B": 2, "T": 32768, "C": 1024, "reverse": True, "gain": "convex", "ragged": False,
         "grad": True},
        # each head's output normalised by itself, behind an attention over 32 x 860 frames
        {"name": "norm_heads", "op": "norm", "dtype": "bfloat16", "B": 27520, "T": 1, "C": 512, "G": 8, "act": "none", "ragged": False, "grad": True},
        # a convolution block's norm + activation over 32 clips of up to 860 frames
        {"name": "norm_frames", "op": "norm", "dtype": "bfloat16", "B": 32, "T": 860, "C": 384, "G": 16, "act": "silu", "ragged": True, "grad": True},
        # a vocoder's last stage, 64 segments of 8192 samples
        {"name": "norm_samples", "op": "norm", "dtype": "float32", "B": 64, "T": 8192, "C": 32, "G": 4, "act": "gelu", "ragged": False, "grad": True},
    ]


def _spread(rng, lo, hi):
    """An integer of lo .. hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "diff", "recurrence", "norm"])
    half = rng.choice(["bfloat16", "float16"])
    any_type = rng.choice(["bfloat16", "float16", "float32"])
    grad = rng.random() < 0.6
    if op == "rotary":
        D = 2 * _spread(rng, 8, 96)
        Hk = rng.choice([1, 2, 3, 4, 8])
        H = Hk * rng.choice([1, 1, 2, 4])
        T = 1 if rng.random() < 0.2 else _spread(rng, 2, 16384)
        B = _spread(rng, 1, max(1, min(128, 2 * 16384 * 20 * 128 // (T * (H + Hk) * D) // (2 if any_type == "float32" else 1))))
        return {"op": op, "dtype": any_type, "B": B, "T": T, "H": H, "Hk": Hk, "D": D, "rd": D if rng.random() < 0.5 else 2 * rng.randint(1, D // 2),
                "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "factor": rng.choice([2.0, 4.0, 8.0, 32.0]),
                "first": _spread(rng, 1, 500000) - 1, "grad": grad}
    if op == "diff":
        d = 8 * rng.randint(2, 8)
        Hk = rng.choice([1, 2, 3, 4])
        H = Hk * rng.choice([1, 1, 2, 4])
        cap = 8192 * 8192 * 16 // 2
        if not grad and rng.random() < 0.6:
            Tq, Tk = rng.choice([1, 1, 2, 5]), _spread(rng, 1, 40000)
            B = _spread(rng, 1, max(1, min(64, 16 * 8192 * 4 * 64 // (Tk * Hk * d))))
        else:
            Tq = _spread(rng, 2, 4096)      # (a lone key's weight is 1: gradients that are nothing are not worth comparing)
            Tk = Tq if rng.random() < 0.7 else _spread(rng, 2, 4096)
            B = _spread(rng, 1, max(1, min(48, cap // (Tq * Tk * H), 2 ** 25 // ((Tq * H + Tk * Hk) * d))))
        return {"op": op, "dtype": half, "B": B, "Tq": Tq, "Tk": Tk, "H": H, "Hk": Hk, "d": d, "causal": rng.random() < 0.5, "ragged": rng.random() < 0.6,
                "grad": grad}
    if op == "recurrence":
        C = _spread(rng, 1, 2048)
        T = 1 if rng.random() < 0.15 else _spread(rng, 2, 32768)
        B = _spread(rng, 1, max(1, min(128, 2 ** 25 // (T * C))))
        return {"op": op, "dtype": any_type, "B": B, "T": T, "C": C, "reverse": rng.random() < 0.5, "gain": rng.choice(["convex", "unit"]),
                "ragged": rng.random() < 0.5, "grad": grad}
    G = rng.choice([1, 2, 3, 4, 8, 16, 32])
    T = 1 if rng.random() < 0.2 else _spread(rng, 2, 16384)
    C = G * _spread(rng, -(-16 // T), 1024 // G)      # (groups of 16 values at least: a normalised pair is +-1 whatever it was, its gradient rounding alone)
    B = _spread(rng, 1, max(1, min(30000, 2 ** 24 // (T * C))))
    # (no activation with a kink: of millions of values some lie nearer to it than 32 bits tell, and each moves a whole gradient)
    return {"op": op, "dtype": any_type, "B": B, "T": T, "C": C, "G": G, "act": rng.choice(["none", "silu", "gelu", "tanh"]),
            "ragged": rng.random() < 0.5, "grad": grad}


# ----------------------------------------------------------------------------------------------------------------- inputs ----
def _lengths(B, T, ragged):
    """Ragged lengths of a batch: one whole, most between a half and the whole, and from four items on a short one."""
    if not ragged:
        return [T] * B
    out = [T - (i * 7919) % (T // 2 + 1) for i in range(B)]
    if B >= 4:
        out[B - 1] = T // 16
    return out


def _frequencies(case):
    """Angle per position of each pair in float64, and the factor on cosine and sine."""
    rd, base, factor = case["rd"], 10000.0, case["factor"]
    if case["scaling"] == "ntk" and rd > 2:
        base *= factor ** (rd / (rd - 2.0))
    i = torch.arange(rd // 2, dtype=torch.float64)
    freq = base ** (-2.0 * i / rd)
    if case["scaling"] == "linear":
        return freq / factor, 1.0
    if case["scaling"] == "yarn":
        def pair_of(turns):   # the (fractional) pair that makes `turns` turns over the original length
            return rd * math.log(4096.0 / (turns * TURN)) / (2.0 * math.log(base))
        low, high = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), rd - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return freq * (1.0 - ramp) + freq / factor * ramp, 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0, dtype=dt, leaf=True):
        t = (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(dtype)
        return t.requires_grad_(True) if leaf and case["grad"] else t

    def lengths(B, T):
        """The batch's lengths in an order that the seed picks."""
        order = torch.randperm(B, device="cuda", generator=g)
        return torch.tensor(_lengths(B, T, True), dtype=torch.int32, device="cuda")[order].contiguous()

    s = {"case": case}
    if case["op"] == "rotary":
        B, T, D = case["B"], case["T"], case["D"]
        s["q"], s["k"] = normal(B, T, case["H"], D), normal(B, T, case["Hk"], D)
        s["dq"], s["dk"] = normal(B, T, case["H"], D, leaf=False), normal(B, T, case["Hk"], D, leaf=False)
        start = torch.randint(0, 4096, (B, 1), device="cuda", generator=g) + case["first"]
        s["positions"] = (start + torch.arange(T, device="cuda")).contiguous()
        s["freq"], s["gain"] = _frequencies(case)
        s["freq"] = s["freq"].cuda()
    elif case["op"] == "diff":
        B, Tq, Tk, H, Hk, d = (case[n] for n in ("B", "Tq", "Tk", "H", "Hk", "d"))
        s["q"], s["k"], s["v"] = normal(B, Tq, H, 2, d), normal(B, Tk, Hk, 2, d), normal(B, Tk, Hk, 2 * d)
        s["lam"] = normal(H, mean=0.5, std=0.15)
        s["dout"] = normal(B, Tq, H, 2 * d, leaf=False)
        s["k_lens"] = lengths(B, Tk) if case["ragged"] else None
        s["q_lens"] = s["k_lens"] if case["ragged"] and Tq == Tk else None
    elif case["op"] == "recurrence":
        B, T, C = case["B"], case["T"], case["C"]
        s["x"], s["gate"] = normal(B, T, C), normal(B, T, C, mean=2.0, std=1.5)
        s["h0"] = normal(B, C, dtype=torch.float32)
        s["dh"], s["dlast"] = normal(B, T, C, leaf=False), normal(B, C, dtype=torch.float32, leaf=False)
        s["lens"] = lengths(B, T) if case["ragged"] else None
    else:
        B, T, C = case["B"], case["T"], case["C"]
        s["x"] = normal(B, T, C, mean=0.3)
        s["weight"], s["bias"] = normal(C, mean=1.0, std=0.1, dtype=torch.float32), normal(C, std=0.1, dtype=torch.float32)
        s["dy"] = normal(B, T, C, leaf=False)
        s["lens"] = lengths(B, T) if case["ragged"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from xva_trainer_amd import seq_ops
        s["ops"] = seq_ops
        if case["op"] == "rotary":
            s["plan"] = seq_ops.RotaryPlan(case["rd"], base=10000.0, interleaved=case["interleaved"], scaling=case["scaling"], factor=case["factor"],
                                           original_length=4096, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms ----
def _live(lens, T, device):
    return torch.arange(T, device=device)[None, :] < lens[:, None].long()


def _plain_rotary(x, positions, freq, gain, interleaved):
    angle = positions.double()[:, :, None, None] * freq
    cos, sin = (angle.cos() * gain).float(), (angle.sin() * gain).float()
    rd = 2 * freq.numel()
    xf = x.float()
    head, tail = xf[..., :rd], xf[..., rd:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = head[..., :rd // 2], head[..., rd // 2:]
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((out, tail), dim=-1).to(x.dtype)


def _visible(case, q_lens, k_lens, device):
    """(B or 1, Tq, Tk): which keys a query sees; with `causal` the last live query sees the last live key."""
    Tq, Tk = case["Tq"], case["Tk"]
    i, j = torch.arange(Tq, device=device)[None, :, None], torch.arange(Tk, device=device)[None, None, :]
    ql = q_lens.long()[:, None, None] if q_lens is not None else torch.full((1, 1, 1), Tq, device=device)
    kl = k_lens.long()[:, None, None] if k_lens is not None else torch.full((1, 1, 1), Tk, device=device)
    see = (i < ql) & (j < kl)
    return see & (j <= i + kl - ql) if case["causal"] else see


def _plain_diff(s):
    case = s["case"]
    share = case["H"] // case["Hk"]
    see = _visible(case, s["q_lens"], s["k_lens"], s["q"].device)[:, None, None]
    q = s["q"].float().permute(0, 2, 3, 1, 4)
    k = s["k"].float().permute(0, 2, 3, 1, 4).repeat_interleave(share, dim=1)
    v = s["v"].float().permute(0, 2, 1, 3).repeat_interleave(share, dim=1)
    score = torch.matmul(q, k.transpose(-1, -2)) * (case["d"] ** -0.5)
    score = score.masked_fill(~see, -1e30)
    e = torch.exp(score - score.amax(-1, keepdim=True)) * see
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    p = p[:, :, 0] - s["lam"].float()[None, :, None, None] * p[:, :, 1]
    return torch.matmul(p, v).permute(0, 2, 1, 3).to(s["q"].dtype)


def _plain_recurrence(s):
    case, T = s["case"], s["case"]["T"]
    x, gate = s["x"].float(), s["gate"].float()
    f = torch.sigmoid(gate)
    u = x * torch.sigmoid(-gate) if case["gain"] == "convex" else x
    live = None
    if s["lens"] is not None:
        live = _live(s["lens"], T, x.device)[:, :, None]
        f, u = torch.where(live, f, torch.ones_like(f)), u * live
    if case["reverse"]:
        f, u = f.flip(1), u.flip(1)
    step = 1
    while step < T:      # after each turn an element holds the sums of 2 * step steps
        u = u + f * torch.cat((torch.zeros_like(u[:, :step]), u[:, :-step]), 1)
        f = f * torch.cat((torch.ones_like(f[:, :step]), f[:, :-step]), 1)
        step *= 2
    h = u + f * s["h0"][:, None]
    last = h[:, -1].contiguous()
    h = h.flip(1) if case["reverse"] else h
    return (h * live if live is not None else h).to(s["x"].dtype), last


def _plain_act(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return torch.tanh(z) if act == "tanh" else z


def _plain_norm(s):
    case = s["case"]
    B, T, C, G = (case[n] for n in ("B", "T", "C", "G"))
    x = s["x"].float().view(B, T, G, C // G)
    if s["lens"] is not None:
        live = _live(s["lens"], T, x.device)[:, :, None, None].float()
        count = (s["lens"].float() * (C // G)).clamp_min(1.0)[:, None, None, None]
    else:
        live, count = torch.ones(1, 1, 1, 1, device=x.device), float(T * (C // G))
    mean = (x * live).sum((1, 3), keepdim=True) / count
    off = (x - mean) * live
    rstd = torch.rsqrt((off * off).sum((1, 3), keepdim=True) / count + 1e-5)
    z = (off * rstd).reshape(B, T, C) * s["weight"] + s["bias"]
    return (_plain_act(z, case["act"]) * live[..., 0]).to(s["x"].dtype)


# -------------------------------------------------------------------------------------------------------------------- run ----
def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if op == "rotary":
        if own:
            q, k = s["ops"].rotary(s["plan"], s["q"], s["k"], positions=s["positions"])
        else:
            q, k = (_plain_rotary(s[n], s["positions"], s["freq"], s["gain"], case["interleaved"]) for n in ("q", "k"))
        outs, leaves, grads = (q, k), ("q", "k"), (s["dq"], s["dk"])
    elif op == "diff":
        if own:
            out = s["ops"].differential_attention(s["q"], s["k"], s["v"], s["lam"], causal=case["causal"], q_lens=s["q_lens"], k_lens=s["k_lens"])
        else:
            out = _plain_diff(s)
        outs, leaves, grads = (out,), ("q", "k", "v", "lam"), (s["dout"],)
    elif op == "recurrence":
        if own:
            outs = s["ops"].gated_recurrence(s["x"], s["gate"], s["h0"], lens=s["lens"], reverse=case["reverse"], gain=case["gain"])
        else:
            outs = _plain_recurrence(s)
        leaves, grads = ("x", "gate", "h0"), (s["dh"], s["dlast"])
    else:
        if own:
            out = s["ops"].group_norm_act(s["x"], case["G"], s["weight"], s["bias"], lens=s["lens"], eps=1e-5, act=case["act"])
        else:
            out = _plain_norm(s)
        outs, leaves, grads = (out,), ("x", "weight", "bias"), (s["dy"],)
    if not case["grad"]:
        return list(outs)
    got = torch.autograd.grad(outs, [s[n] for n in leaves], grads)
    return [o.detach() for o in outs] + list(got)


# ------------------------------------------------------------------------------------------------------------------- work ----
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    passes = 2 if case["grad"] else 1
    if case["op"] == "rotary":
        n = case["B"] * case["T"] * (case["H"] + case["Hk"])
        return {"bytes": passes * (2 * n * case["D"] * size + 8 * case["B"] * case["T"]), "flops": passes * 3 * n * case["rd"]}
    if case["op"] == "diff":
        B, Tq, Tk, H, Hk, d = (case[n] for n in ("B", "Tq", "Tk", "H", "Hk", "d"))
        kl = _lengths(B, Tk, case["ragged"])
        ql = kl if case["ragged"] and Tq == Tk else [Tq] * B
        pairs = keys = rows = 0
        for a, b in zip(ql, kl):
            if case["causal"]:      # query i of a sees i + 1 + b - a keys, where that is more than none
                first = max(1 + b - a, 1)
                pairs += (first + b) * (b - first + 1) // 2 if b >= first else 0
            else:
                pairs += a * b
            keys += b
            rows += a
        q_bytes, kv_bytes = rows * H * 2 * d * size, keys * Hk * 4 * d * size
        if not case["grad"]:
            return {"bytes": 2 * q_bytes + kv_bytes, "flops": pairs * H * 12 * d}
        return {"bytes": 4 * q_bytes + 2 * kv_bytes, "flops": pairs * H * 32 * d}
    n = sum(_lengths(case["B"], case["T"], case["ragged"])) * case["C"]
    if case["op"] == "recurrence":
        # forward: x, gate -> h; backward: x, gate, dh -> dx, dgate
        return {"bytes": (8 if case["grad"] else 3) * n * size + (4 if case["grad"] else 2) * 4 * case["B"] * case["C"], "flops": (16 if case["grad"] else 6) * n}
    # forward: x -> y; backward: x, dy -> dx
    return {"bytes": (5 if case["grad"] else 2) * n * size + (4 if case["grad"] else 2) * 4 * case["C"], "flops": (30 if case["grad"] else 12) * n}


# ------------------------------------------------------------------------------------------------------------------ exact ----
def _exact_rotary(s, case):
    rd = case["rd"]
    turn = torch.polar(torch.full((), s["gain"], dtype=torch.float64, device="cuda"), s["positions"].double()[..., None] * s["freq"])[:, :, None]

    def rotate(x, by):
        x = x.detach().double()
        lo, hi = (slice(0, rd, 2), slice(1, rd, 2)) if case["interleaved"] else (slice(0, rd // 2), slice(rd // 2, rd))
        z = torch.complex(x[..., lo].contiguous(), x[..., hi].contiguous()) * by
        x = x.clone()
        x[..., lo], x[..., hi] = z.real, z.imag
        return x
    out = [rotate(s["q"], turn), rotate(s["k"], turn)]
    return out + [rotate(s["dq"], turn.conj()), rotate(s["dk"], turn.conj())] if case["grad"] else out


def _exact_diff(s, case):
    B, Tq, Tk, H, Hk, d = (case[n] for n in ("B", "Tq", "Tk", "H", "Hk", "d"))
    if case["grad"] and B * H * Tq * Tk > 2 ** 31:
        return None
    scale = 1.0 / math.sqrt(d)
    q, k, v, lam, do = (s[n].detach().double() for n in ("q", "k", "v", "lam", "dout"))
    out, dq, dk, dv, dlam = torch.zeros_like(do), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(lam)
    ql = s["q_lens"].tolist() if s["q_lens"] is not None else [Tq] * B
    kl = s["k_lens"].tolist() if s["k_lens"] is not None else [Tk] * B
    for b in range(B):
        nq, nk = ql[b], kl[b]
        skip = max(nq - nk, 0) if case["causal"] else 0      # the first rows see nothing
        if nk == 0 or skip >= nq:
            continue
        hidden = None
        if case["causal"]:
            hidden = torch.ones(nq - skip, nk, dtype=torch.bool, device="cuda").triu(1 + nk - (nq - skip))
        for h in range(H):
            kv = h // (H // Hk)
            maps = []
            for m in (0, 1):
                w = q[b, skip:nq, h, m] @ k[b, :nk, kv, m].T * scale
                if hidden is not None:
                    w = w.masked_fill(hidden, -math.inf)
                maps.append(torch.softmax(w, -1))
            V, g = v[b, :nk, kv], do[b, skip:nq, h]
            both = maps[0] - lam[h] * maps[1]
            out[b, skip:nq, h] = both @ V
            if not case["grad"]:
                continue
            dv[b, :nk, kv] += both.T @ g
            gp = g @ V.T
            dlam[h] -= (gp * maps[1]).sum()
            for m, c in ((0, 1.0), (1, -lam[h])):
                gs = maps[m] * (gp - (gp * maps[m]).sum(-1, keepdim=True)) * (c * scale)
                dq[b, skip:nq, h, m] = gs @ k[b, :nk, kv, m]
                dk[b, :nk, kv, m] += gs.T @ q[b, skip:nq, h, m]
    return [out, dq, dk, dv, dlam] if case["grad"] else [out]


def _exact_recurrence(s, case):
    B, T, C = case["B"], case["T"], case["C"]
    x, gate, h = (s[n].detach().double() for n in ("x", "gate", "h0"))
    f = 1.0 / (1.0 + torch.exp(-gate))
    keep = 1.0 / (1.0 + torch.exp(gate)) if case["gain"] == "convex" else torch.ones_like(f)
    lens = s["lens"].tolist() if s["lens"] is not None else [T] * B
    live = torch.tensor(lens, device="cuda")[:, None] > torch.arange(T, device="cuda")[None]
    order = range(T - 1, -1, -1) if case["reverse"] else range(T)
    f = f.masked_fill(~live[:, :, None], 1.0)
    u = (keep * x).masked_fill(~live[:, :, None], 0.0)
    hs, before = torch.zeros_like(x), torch.zeros_like(x)
    for t in order:
        before[:, t] = h
        h = torch.addcmul(u[:, t], f[:, t], h)
        hs[:, t] = h
    out = [hs * live[:, :, None], h]
    if not case["grad"]:
        return out
    g = s["dlast"].detach().double()
    dh = s["dh"].detach().double() * live[:, :, None]
    total = torch.zeros_like(x)
    for t in reversed(order):
        total[:, t] = g = g + dh[:, t]
        g = g * f[:, t]
    dx = total * keep * live[:, :, None]
    pull = before - x if case["gain"] == "convex" else before
    dgate = total * pull * f * (1.0 / (1.0 + torch.exp(gate))) * live[:, :, None]
    return out + [dx, dgate, g]


def _exact_norm(s, case):
    B, T, C, G = (case[n] for n in ("B", "T", "C", "G"))
    x, w, bias, dy = (s[n].detach().double() for n in ("x", "weight", "bias", "dy"))
    live = torch.ones(B, T, 1, dtype=torch.float64, device="cuda")
    if s["lens"] is not None:
        live = (torch.arange(T, device="cuda") < s["lens"][:, None]).double()[:, :, None]

    def per_group(t):      # mean over a group's live values, spread back over its channels
        total = (t * live).view(B, T, G, C // G).sum(3).sum(1)
        n = live.sum(1).clamp_min(1.0) * (C // G)
        return (total / n).repeat_interleave(C // G, 1)[:, None]
    mu = per_group(x)
    inv = (per_group((x - mu) ** 2) + 1e-5) ** -0.5
    xh = (x - mu) * inv
    z = xh * w + bias
    act = case["act"]
    sig = 1.0 / (1.0 + torch.exp(-z))
    if act == "silu":
        y, slope = z * sig, sig * (1.0 + z * (1.0 - sig))
    elif act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(TURN)
    elif act == "tanh":
        y = torch.tanh(z)
        slope = 1.0 - y * y
    else:
        y, slope = z, torch.ones_like(z)
    if not case["grad"]:
        return [y * live]
    dz = dy * slope * live
    gx = dz * w
    dx = inv * (gx - per_group(gx) - xh * per_group(gx * xh)) * live
    return [y * live, dx, (dz * xh).sum((0, 1)), dz.sum((0, 1))]


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotary": _exact_rotary, "diff": _exact_diff, "recurrence": _exact_recurrence, "norm": _exact_norm}[case["op"]](s, case)
