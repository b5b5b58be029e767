"""Operators of a decoder block that reads an encoder's states: group norm with an activation, rotary positions, cross attention.

`listed()` names the measured cases, `draw()` makes further ones of the same ranges, `run()` is one pass of a case: the
operators' plain form (elementary torch operations in 32 bits) or, with `own` set, the framework's kernels.  `exact()` is the
same pass from the definitions in 64 bits."""
import math

import numpy as np
import torch

own = False

ACTS = {"none": 0, "relu": 1, "silu": 6, "gelu": 7}          # styler_amd.ops.ACT_*
BANDS = {"orig_len": 1024, "low": 1.0, "high": 4.0}           # the frequency bands of the "bands" scaling
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------------- cases
def _gn(name, B, L, C, groups, act, dtype, direction, ragged):
    return dict(name=name, op="groupnorm_act", B=B, L=L, C=C, groups=groups, act=act, dtype=dtype, dir=direction, ragged=ragged)


def _rot(name, B, L, H, D, rot, interleaved, scaling, pos, sliced, dtype, direction):
    return dict(name=name, op="rotary", B=B, L=L, H=H, D=D, rot=rot, interleaved=interleaved, scaling=scaling, pos=pos,
                sliced=sliced, dtype=dtype, dir=direction)


def _att(name, B, Lq, Lk, H, G, D, dtype, direction, ragged, mask):
    return dict(name=name, op="cross_attention", B=B, Lq=Lq, Lk=Lk, H=H, G=G, D=D, dtype=dtype, dir=direction, ragged=ragged,
                mask=mask)


def listed():
    return [
        # one utterance's style sequence through a norm of an audio encoder while serving: latency
        _gn("gn_serve", 1, 60, 320, 20, "relu", "bf16", "fwd", False),
        # a training batch of padded utterances (mel frames, 320 channels in groups of 16), statistics of the valid frames
        _gn("gn_train_ragged", 16, 1000, 320, 20, "silu", "bf16", "train", True),
        # long recordings at full precision: far more than the caches hold
        _gn("gn_train_long", 8, 16384, 512, 32, "gelu", "fp32", "train", False),
        # one token for each of 32 running requests, far into their texts: queries and keys of a fused q|k|v row
        _rot("rotary_token", 32, 1, 10, 64, 64, False, "bands", "far", True, "bf16", "fwd"),
        # a batch of mel frames on the phonemes' time scale (fractional positions), a quarter of the head left as it is
        _rot("rotary_frames", 16, 1000, 4, 64, 48, True, "none", "frames", False, "fp32", "fwd"),
        # training on long texts, positions interpolated, forward and gradient
        _rot("rotary_train_long", 4, 8192, 32, 128, 128, False, "linear", "start", False, "bf16", "train"),
        # one token for each of 32 requests over their encoder states, grouped heads: bound by the reading of keys and values
        _att("attn_token", 32, 1, 1500, 16, 4, 64, "bf16", "fwd", True, False),
        # one token of two requests over a very long encoded document: few rows, a long axis
        _att("attn_token_long", 2, 1, 65537, 8, 8, 128, "bf16", "fwd", False, False),
        # a training batch's mel frames over its phonemes at the model's own sizes
        _att("attn_frames", 48, 1000, 133, 4, 4, 64, "bf16", "train", True, False),
        # a long prompt over a long document, grouped heads: bound by the matrix cores
        _att("attn_prompt", 4, 4096, 4096, 16, 4, 128, "bf16", "fwd", False, False),
        # training over an audio encoder's states, some of them dropped by a key mask
        _att("attn_train", 8, 2048, 1500, 16, 16, 64, "bf16", "train", False, True),
        # the same at full precision, odd lengths
        _att("attn_train_fp32", 8, 1203, 1001, 8, 4, 64, "fp32", "train", True, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["groupnorm_act", "rotary", "cross_attention", "cross_attention"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    direction = rng.choice(["fwd", "train"])
    while True:
        if kind == "groupnorm_act":
            groups, per = rng.choice([1, 2, 3, 4, 5, 8, 16, 20, 32]), rng.choice([1, 2, 3, 4, 8, 10, 16, 24, 32])
            c = _gn(None, rng.randint(1, 16), _log_int(rng, 1, 16384), groups * per, groups,
                    rng.choice(["none", "relu", "silu", "gelu"]), dtype, direction, rng.random() < 0.5)
            fits = 1000 <= c["B"] * c["L"] * c["C"] <= 8 * 16384 * 512
        elif kind == "rotary":
            D = rng.choice([32, 40, 64, 80, 96, 128])
            c = _rot(None, rng.randint(1, 32), _log_int(rng, 1, 8192), rng.choice([1, 2, 4, 5, 8, 10, 16, 32]), D,
                     rng.choice([D, D, D // 2, 2 * rng.randint(2, D // 2)]), rng.random() < 0.5,
                     rng.choice(["none", "linear", "base", "bands"]), rng.choice(["start", "far", "frames"]), rng.random() < 0.5,
                     dtype, direction)
            fits = 1000 <= c["B"] * c["L"] * c["H"] * D <= 4 * 8192 * 32 * 128
        else:
            G = rng.choice([1, 2, 4, 8])
            token = direction == "fwd" and rng.random() < 0.5
            c = _att(None, rng.randint(1, 32), rng.choice([1, 1, 2, 5]) if token else _log_int(rng, 2, 4096),
                     _log_int(rng, 1, 65537 if token else 8192), G * rng.choice([1, 1, 2, 4]), G, rng.choice([32, 64, 64, 80, 128]),
                     dtype, direction, rng.random() < 0.5, rng.random() < 0.3)
            scores = c["B"] * c["H"] * c["Lq"] * c["Lk"]
            kv = c["B"] * c["Lk"] * G * c["D"]
            most = 4 * 16 * 4096 * 4096 if direction == "fwd" and dtype == "bf16" else 8 * 8 * 1203 * 1001
            fits = 100 <= scores <= most and kv <= 1 << 27
        if fits:
            del c["name"]
            return c


def _lengths(n, longest, ragged, least=None):
    """Lengths of a batch: all equal, or spread evenly from a third of the longest to the longest."""
    if not ragged:
        return [longest] * n
    least = max(1, longest // 3) if least is None else least
    return [least + (longest - least) * i // max(1, n - 1) if n > 1 else longest for i in range(n)]


def _shuffled_lengths(n, longest, ragged, seed):
    v = _lengths(n, longest, ragged)
    return [v[i] for i in np.random.default_rng(seed + 7).permutation(n)]


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    train = case["dir"] == "train"
    if case["op"] == "groupnorm_act":
        C, n = case["C"], sum(_lengths(case["B"], case["L"], case["ragged"])) * case["C"]
        full = case["B"] * case["L"] * C
        # x (and dy) of the valid rows in, y (and dx) of all rows out, gamma and beta (and their gradients)
        return {"bytes": es * ((2 * n + 2 * full) if train else (n + full)) + 4 * C * (4 if train else 2),
                "flops": n * (28 if train else 12)}
    if case["op"] == "rotary":
        n = case["B"] * case["L"] * case["H"] * case["D"]
        turned = n // case["D"] * case["rot"]
        rows = case["L"] * (case["B"] if case["pos"] == "far" else 1)
        return {"bytes": es * n * (4 if train else 2) + rows * (4 if case["pos"] == "frames" else 8) + 4 * case["rot"],
                "flops": 3 * turned * (2 if train else 1)}
    kl, ql = _lengths(case["B"], case["Lk"], case["ragged"]), [case["Lq"]] * case["B"]
    if case["ragged"] and case["Lq"] > 8:
        ql = _lengths(case["B"], case["Lq"], True)
    H, G, D = case["H"], case["G"], case["D"]
    # pairs: the i-th longest query sequence meets the i-th longest key sequence (frames follow the text they speak)
    pairs = sum(a * b for a, b in zip(ql, kl))
    q, kv = es * sum(ql) * H * D, es * sum(kl) * G * D
    q_all, kv_all = es * case["B"] * case["Lq"] * H * D, es * case["B"] * case["Lk"] * G * D
    if case["mask"]:
        pairs = pairs * 3 // 4                                # the keys that the mask leaves (one in four is dropped)
        kv = kv * 3 // 4
    if train:
        return {"bytes": 2 * q + 2 * kv + 2 * q_all + 2 * kv_all, "flops": 14 * pairs * H * D}
    return {"bytes": q + 2 * kv + q_all, "flops": 4 * pairs * H * D}


# -------------------------------------------------------------------------------------------------------------------- inputs
def _frequencies(rot, scaling, factor=4.0, base=10000.0):
    """Angle per position of the rot / 2 pairs, in 64 bits."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "bands":
        turns = BANDS["orig_len"] * f / (2 * math.pi)
        keep = ((turns - BANDS["low"]) / (BANDS["high"] - BANDS["low"])).clamp(0, 1)
        f = (1 - keep) * f / factor + keep * f
    return f


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    s = dict(case)
    if case["op"] == "groupnorm_act":
        B, L, C = case["B"], case["L"], case["C"]
        # channels with their own offset and width, as a convolution leaves them
        s["x"] = (randn(B, L, C) * (0.5 + randn(C).abs()) + randn(C)).to(dt)
        s["gamma"], s["beta"] = 1 + 0.1 * randn(C), 0.1 * randn(C)
        s["lens"] = torch.tensor(_shuffled_lengths(B, L, True, seed), device=dev) if case["ragged"] else None
        s["dy"] = randn(B, L, C).to(dt) if case["dir"] == "train" else None
    elif case["op"] == "rotary":
        B, L, H, D, rot = (case[k] for k in ("B", "L", "H", "D", "rot"))
        # a sliced case turns the first H heads of rows that hold more (the queries and keys of a fused projection)
        s["x"] = randn(B, L, H + (2 if case["sliced"] else 0), D).to(dt)[:, :, :H]
        s["dy"] = randn(B, L, H, D).to(dt) if case["dir"] == "train" else None
        if case["pos"] == "start":
            s["pos_of"] = torch.arange(L, device=dev)
        elif case["pos"] == "far":
            s["pos_of"] = torch.randint(1000, 200000, (B, 1), device=dev, generator=g) + torch.arange(L, device=dev)
        else:                                                 # frames on the text's scale: about seven frames a phoneme
            s["pos_of"] = (torch.arange(L, device=dev) / 7.3).float()
        s["gain"] = 1.0 if case["scaling"] != "bands" else 0.1 * math.log(4.0) + 1.0
        if own:
            from styler_amd import ops
            kind = None if case["scaling"] == "none" else case["scaling"]
            s["freqs"] = ops.rotary_freqs(rot, dev, scaling=kind, factor=4.0, **(BANDS if kind == "bands" else {}))
        else:
            s["freqs"] = _frequencies(rot, case["scaling"]).to(dev)
    else:
        B, Lq, Lk, H, G, D = (case[k] for k in ("B", "Lq", "Lk", "H", "G", "D"))
        s["q"] = randn(B, Lq, H, D).to(dt)
        kv = randn(B, Lk, 2, G, D).to(dt)                     # keys and values of one projection of the encoder's states
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        order = np.random.default_rng(seed).permutation(B)
        s["lens"] = s["q_lens"] = s["mask"] = None
        if case["ragged"]:
            lens = _lengths(B, Lk, True)
            s["lens"] = torch.tensor([lens[i] for i in order], device=dev)
            if Lq > 8:
                lens = _lengths(B, Lq, True)
                s["q_lens"] = torch.tensor([lens[i] for i in order], device=dev)
        if case["mask"]:                                      # True: a key that no query sees
            s["mask"] = torch.rand(B, Lk, device=dev, generator=g) < 0.25
        s["dout"] = randn(B, Lq, H, D).to(dt) if case["dir"] == "train" else None
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        t = 1 / (1 + torch.exp(-z))
        return t * (1 + z * (1 - t))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _groupnorm_plain(s):
    B, L, C, G = s["B"], s["L"], s["C"], s["groups"]
    dt = s["x"].dtype
    x = s["x"].float().view(B, L, G, C // G)
    n = torch.full((B,), L, device=x.device) if s["lens"] is None else s["lens"]
    on = (torch.arange(L, device=x.device)[None] < n[:, None]).view(B, L, 1, 1)
    count = (n * (C // G)).clamp_min(1).view(B, 1, 1, 1).float()
    xc = torch.where(on, x - torch.where(on, x, 0).sum((1, 3), keepdim=True) / count, 0)
    rstd = 1 / torch.sqrt((xc * xc).sum((1, 3), keepdim=True) / count + 1e-5)
    xh = xc * rstd
    gamma, beta = s["gamma"].view(1, 1, G, -1), s["beta"].view(1, 1, G, -1)
    z = xh * gamma + beta
    y = torch.where(on, _act(z, s["act"]), 0).view(B, L, C).to(dt)
    if s["dir"] == "fwd":
        return y
    dz = torch.where(on, s["dy"].float().view_as(z) * _act_slope(z, s["act"]), 0)
    dgamma, dbeta = (dz * xh).sum((0, 1)).view(C), dz.sum((0, 1)).view(C)
    d = dz * gamma
    dx = rstd * (d - d.sum((1, 3), keepdim=True) / count - xh * ((d * xh).sum((1, 3), keepdim=True) / count))
    return y, torch.where(on, dx, 0).view(B, L, C).to(dt), dgamma, dbeta


def _rotary_plain(s, x, sign):
    rot = s["rot"]
    angle = s["pos_of"].double()[..., None] * s["freqs"]      # in 64 bits: far positions are many turns
    cos, sin = angle.cos().float() * s["gain"], sign * (angle.sin().float() * s["gain"])
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)           # over the heads
    xf = x.float()
    if s["interleaved"]:
        a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = xf[..., :rot // 2], xf[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, xf[..., rot:]), -1).to(x.dtype)


def _attention_plain(s):
    B, Lq, Lk, H, G, D = (s[k] for k in ("B", "Lq", "Lk", "H", "G", "D"))
    R, dt, dev = H // G, s["q"].dtype, s["q"].device

    def rows(t):                                              # [B, Lq, H, D] -> [B, G, R * Lq, D]: the heads that share keys
        return t.float().view(B, Lq, G, R, D).permute(0, 2, 3, 1, 4).reshape(B, G, R * Lq, D)

    def back(t):
        return t.view(B, G, R, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, H, D).to(dt)

    off = torch.zeros(B, Lk, dtype=torch.bool, device=dev)
    if s["lens"] is not None:
        off = torch.arange(Lk, device=dev)[None] >= s["lens"][:, None]
    if s["mask"] is not None:
        off = off | s["mask"]
    q = rows(s["q"])
    k, v = (s[n].float().permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))
    scale = 1 / math.sqrt(D)
    p = (q @ k.transpose(-1, -2)) * scale
    p = p.masked_fill(off[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1, total)
    live = None
    if s["q_lens"] is not None:
        live = (torch.arange(Lq, device=dev)[None] < s["q_lens"][:, None]).repeat(1, R).view(B, 1, R * Lq, 1)
    o = p @ v
    if live is not None:
        o = torch.where(live, o, 0)
    if s["dir"] == "fwd":
        return back(o)
    do = rows(s["dout"])
    if live is not None:
        do = torch.where(live, do, 0)
    dv = p.transpose(-1, -2) @ do
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * scale
    return (back(o), back(ds @ k), (ds.transpose(-1, -2) @ q).permute(0, 2, 1, 3).to(dt), dv.permute(0, 2, 1, 3).to(dt))


# ------------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    s, train = state, state["dir"] == "train"
    if not own:
        if s["op"] == "groupnorm_act":
            return _groupnorm_plain(s)
        if s["op"] == "rotary":
            y = _rotary_plain(s, s["x"], 1.0)
            return (y, _rotary_plain(s, s["dy"], -1.0)) if train else y
        return _attention_plain(s)
    from styler_amd import ops
    if s["op"] == "groupnorm_act":
        act = ACTS[s["act"]]
        if not train:
            return ops.groupnorm_act(s["x"], s["gamma"], s["beta"], s["groups"], act, lens=s["lens"])
        stats = torch.empty(s["B"], s["groups"], 2, device=s["x"].device, dtype=torch.float32)
        y = ops.groupnorm_act(s["x"], s["gamma"], s["beta"], s["groups"], act, lens=s["lens"], stats=stats)
        return (y, *ops.groupnorm_act_bwd(s["x"], s["dy"], s["gamma"], s["beta"], stats, s["groups"], act, lens=s["lens"]))
    if s["op"] == "rotary":
        y = ops.rotary(s["x"], s["freqs"], s["pos_of"], interleaved=s["interleaved"], gain=s["gain"])
        if not train:
            return y
        return y, ops.rotary(s["dy"], s["freqs"], s["pos_of"], interleaved=s["interleaved"], gain=s["gain"], inverse=True)
    if not train:
        return ops.cross_attention(s["q"], s["k"], s["v"], s["lens"], q_lens=s["q_lens"], mask=s["mask"])
    lse = torch.empty(s["B"], s["H"], s["Lq"], device=s["q"].device, dtype=torch.float32)
    out = ops.cross_attention(s["q"], s["k"], s["v"], s["lens"], q_lens=s["q_lens"], mask=s["mask"], lse=lse)
    return (out, *ops.cross_attention_bwd(s["q"], s["k"], s["v"], out, s["dout"], lse, s["lens"], q_lens=s["q_lens"],
                                          mask=s["mask"]))


# ------------------------------------------------------------------------------------------------------- the definitions, 64 bits
def _exact_groupnorm(s):
    """Item by item and group by group, on the valid rows alone; the gradients by differentiation."""
    B, L, C, G = s["B"], s["L"], s["C"], s["groups"]
    train = s["dir"] == "train"
    gamma, beta = (s[n].double().requires_grad_(train) for n in ("gamma", "beta"))
    y, dx = (torch.zeros(B, L, C, dtype=torch.float64, device=gamma.device) for _ in range(2))
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)
    for b in range(B):
        n = L if s["lens"] is None else int(s["lens"][b])
        if n == 0:
            continue
        x = s["x"][b, :n].double().requires_grad_(train)
        xg = x.reshape(n, G, C // G).transpose(0, 1).reshape(G, -1)
        var, mean = torch.var_mean(xg, 1, correction=0, keepdim=True)
        z = ((xg - mean) * (var + 1e-5).rsqrt()).view(G, n, C // G).transpose(0, 1).reshape(n, C) * gamma + beta
        if s["act"] == "relu":
            z = torch.relu(z)
        elif s["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif s["act"] == "gelu":
            z = z * torch.special.ndtr(z)
        y[b, :n] = z.detach()
        if train:
            d = torch.autograd.grad(z, (x, gamma, beta), s["dy"][b, :n].double())
            dx[b, :n] = d[0]
            dgamma += d[1]
            dbeta += d[2]
    return (y, dx, dgamma.detach(), dbeta.detach()) if train else y


def _exact_rotary(s):
    """Pairs as complex numbers, turned by exp(i angle)."""
    rot = s["rot"]
    angle = s["pos_of"].double()[..., None] * _frequencies(rot, s["scaling"]).to(s["x"].device)
    turn = torch.polar(torch.full_like(angle, s["gain"]), angle).unsqueeze(-2)

    def by(x, w):
        out = x.double().clone()
        head = out[..., :rot]
        c = head.unflatten(-1, (-1, 2)) if s["interleaved"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        r = torch.view_as_real(torch.view_as_complex(c.contiguous()) * w)
        out[..., :rot] = (r if s["interleaved"] else r.transpose(-1, -2)).flatten(-2)
        return out

    y = by(s["x"], turn)
    return (y, by(s["dy"], turn.conj())) if s["dir"] == "train" else y


def _exact_attention(s):
    """Item by item and group of heads by group, over the keys that are seen alone."""
    B, Lq, Lk, H, G, D = (s[k] for k in ("B", "Lq", "Lk", "H", "G", "D"))
    R, dev = H // G, s["q"].device
    o, dq = (torch.zeros(B, Lq, H, D, dtype=torch.float64, device=dev) for _ in range(2))
    dk, dv = (torch.zeros(B, Lk, G, D, dtype=torch.float64, device=dev) for _ in range(2))
    for b in range(B):
        nk = Lk if s["lens"] is None else int(s["lens"][b])
        nq = Lq if s["q_lens"] is None else int(s["q_lens"][b])
        seen = torch.arange(nk, device=dev)
        if s["mask"] is not None:
            seen = seen[~s["mask"][b, :nk]]
        if len(seen) == 0 or nq == 0:
            continue
        for g in range(G):
            heads = slice(g * R, g * R + R)
            q = s["q"][b, :nq, heads].double().transpose(0, 1)
            k, v = s["k"][b, seen, g].double(), s["v"][b, seen, g].double()
            w = torch.softmax(torch.matmul(q, k.t()) / math.sqrt(D), -1)
            o[b, :nq, heads] = torch.matmul(w, v).transpose(0, 1)
            if s["dir"] == "train":
                do = s["dout"][b, :nq, heads].double().transpose(0, 1)
                dv[b, seen, g] = torch.matmul(w.transpose(1, 2), do).sum(0)
                dw = torch.matmul(do, v.t())
                dw = w * (dw - (do * torch.matmul(w, v)).sum(-1, keepdim=True)) / math.sqrt(D)
                dq[b, :nq, heads] = torch.matmul(dw, k).transpose(0, 1)
                dk[b, seen, g] = torch.matmul(dw.transpose(1, 2), q).sum(0)
    return (o, dq, dk, dv) if s["dir"] == "train" else o


def exact(case, seed):
    if case["op"] == "cross_attention" and case["B"] * case["H"] * case["Lq"] * case["Lk"] > 5e9:
        return None
    s = prepare(case, seed)
    return {"groupnorm_act": _exact_groupnorm, "rotary": _exact_rotary, "cross_attention": _exact_attention}[case["op"]](s)
