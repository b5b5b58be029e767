"""Group norm with an activation, rotary positions and cross attention (csrc/groupnorm_act.hip, rotary.hip, cross_attention.hip)
against their definitions in 64 bits; masks, empty rows, strides, sizes of zero and one, refusals, streams and graphs.

Tolerances are bounds: u(t) = finfo(t).eps / 2 for every rounding to the tensor's type, taken with the absolute values that the
rounded terms have in the sum they enter, and a multiple of 2^-24 for the 32-bit sums."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
U32 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def within(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.clamp_min(1e-300)).nan_to_num(1e9).max()):.2f} x its bound"


# ------------------------------------------------------------------------------------------------------------ cross attention
def attention_case(dev, B, Lq, Lk, H, G, D, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed + B * 7 + Lq * 11 + Lk * 13 + H + D)
    q, k, v, do = (torch.randn(*s, generator=g) for s in ((B, Lq, H, D), (B, Lk, G, D), (B, Lk, G, D), (B, Lq, H, D)))
    return [t.to(dtype).to(dev) for t in (q * spread, k, v, do)]


def attention_oracle(q, k, v, do, lens, q_lens, mask, scale, dtype):
    """(out, lse, dq, dk, dv) in 64 bits and the bounds of out, dq, dk, dv."""
    B, Lq, H, D = q.shape
    Lk, G = k.shape[1], k.shape[2]
    R = H // G
    u = half_step(dtype)
    up = u if dtype == torch.bfloat16 else 0.0               # P and dS are rounded between the products in bf16 only
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)
    out, dq, to, tq = z(B, Lq, H, D), z(B, Lq, H, D), z(B, Lq, H, D), z(B, Lq, H, D)
    dk, dv, tk, tv = z(B, Lk, G, D), z(B, Lk, G, D), z(B, Lk, G, D), z(B, Lk, G, D)
    lse = torch.full((B, H, Lq), -math.inf, dtype=torch.float64)
    for b in range(B):
        seen = torch.ones(Lk, dtype=torch.bool)
        if lens is not None:
            seen &= torch.arange(Lk) < int(lens[b])
        if mask is not None:
            seen &= ~mask[b if mask.shape[0] > 1 else 0].cpu()
        nq = Lq if q_lens is None else max(0, min(Lq, int(q_lens[b])))
        j = seen.nonzero()[:, 0]
        if len(j) == 0 or nq == 0:
            continue
        for h in range(H):
            Q, K, V, dO = q[b, :nq, h].cpu().double(), k[b, j, h // R].cpu().double(), v[b, j, h // R].cpu().double(), do[b, :nq, h].cpu().double()
            S = Q @ K.T * scale
            lse[b, h, :nq] = torch.logsumexp(S, 1)
            P = torch.exp(S - lse[b, h, :nq, None])
            O = P @ V
            # relative error of P: 32-bit sums of the scores, the exponent's argument, the sum of P (and lse)
            e = ((D + 4) * U32 * (Q.abs() @ K.abs().T * scale).max() + 4 * U32 * (S.abs().max() + lse[b, h, :nq].abs().max()) + (len(j) + 64) * U32)
            A = P @ V.abs()
            eo = u * O.abs() + (up + 2 * e) * A
            out[b, :nq, h], to[b, :nq, h] = O, eo
            dP = dO @ V.T
            delta = (dO * O).sum(1, keepdim=True)
            dS = P * (dP - delta)
            E = (dO.abs() * eo).sum(1, keepdim=True) + (D + 4) * U32 * (dO.abs() * O.abs()).sum(1, keepdim=True)
            eS = P * (E + (D + 4) * U32 * (dO.abs() @ V.abs().T)) + (up + 2 * e) * dS.abs()
            n = (max(len(j), R * nq) + 16) * U32
            dq[b, :nq, h] = scale * dS @ K
            tq[b, :nq, h] = scale * (eS + n * dS.abs()) @ K.abs()
            dk[b, j, h // R] += scale * dS.T @ Q
            tk[b, j, h // R] += scale * (eS + n * dS.abs()).T @ Q.abs()
            dv[b, j, h // R] += P.T @ dO
            tv[b, j, h // R] += (up + 2 * e + n) * P.T @ dO.abs()
    return (out, lse, dq, dk, dv), (to, tq + u * dq.abs(), tk + u * dk.abs(), tv + u * dv.abs())


def check_attention(q, k, v, do, lens=None, q_lens=None, mask=None, scale=None, oracle=None):
    from styler_amd import ops
    dev = q.device
    B, Lq, H, D = q.shape
    on = lambda t: None if t is None else t.to(dev)
    lse = torch.full((B, H, Lq), 7.0, device=dev)
    out = ops.cross_attention(q, k, v, on(lens), q_lens=on(q_lens), mask=on(mask), scale=scale, lse=lse)
    dq, dk, dv = ops.cross_attention_bwd(q, k, v, out, do, lse, on(lens), q_lens=on(q_lens), mask=on(mask), scale=scale)
    src = oracle or (q, k, v, do)
    ref, tol = attention_oracle(*src, lens, q_lens, mask, 1 / math.sqrt(D) if scale is None else scale, q.dtype)
    got = (out, dq, dk, dv)
    assert all(t.dtype == q.dtype for t in got)
    assert bool((torch.isinf(lse.cpu()) == torch.isinf(ref[1])).all())
    live = torch.isfinite(ref[1])
    if live.any():
        d = (lse.cpu().double() - ref[1])[live].abs().max()
        assert float(d) <= 2e-5 * (1 + float(ref[1][live].abs().max())), float(d)
    for n, a, b, t in zip(("out", "dq", "dk", "dv"), got, (ref[0], ref[2], ref[3], ref[4]), tol):
        within(a.cpu(), b, t + 1e-30, n)
    return got


DT = [torch.bfloat16, torch.float32]


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Lq,Lk,H,G,D", [
    (1, 1, 1, 1, 1, 64),                 # one query, one key
    (2, 1, 300, 8, 2, 64),               # a token of grouped heads, shares of a long axis
    (1, 5, 129, 4, 1, 32),               # 20 rows of one key head, one key past a tile
    (1, 33, 64, 1, 1, 64),               # one row past a wave
    (2, 130, 70, 2, 2, 128),             # odd tiles both ways
    (1, 3, 1000, 1, 1, 128),             # few rows, many keys
    (1, 260, 40, 4, 2, 80),              # a head width inside a tile's
    (3, 17, 33, 2, 1, 8),                # the narrowest head
    (1, 640, 37, 1, 1, 40),              # many rows over few keys: the key gradient's rows are shared out
])
def test_cross_attention_against_definition(dev, B, Lq, Lk, H, G, D, dtype):
    check_attention(*attention_case(dev, B, Lq, Lk, H, G, D, dtype))


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Lq", [1, 45])
def test_cross_attention_masks(dev, dtype, Lq):
    """Lengths of zero, one, all and beyond; whole rows and whole tiles dropped by the mask; queries past their length.  What stands
    in the unseen rows is NaN and infinite."""
    B, Lk, H, G, D = 6, 200, 4, 2, 64
    q, k, v, do = attention_case(dev, B, Lq, Lk, H, G, D, dtype, seed=3)
    lens = torch.tensor([0, 1, 200, 500, 130, 77])
    q_lens = torch.tensor([Lq, Lq, 0, 1, Lq + 9, max(1, Lq - 3)])
    mask = torch.rand(B, Lk, generator=torch.Generator().manual_seed(5)) < 0.4
    mask[3] = True                                            # nothing left
    mask[4, :128] = True                                      # the first tiles empty
    mask[2, 64:128] = True
    seen = (torch.arange(Lk)[None] < lens[:, None]) & ~mask
    dead = torch.arange(Lq)[None] >= q_lens[:, None]
    k2, v2, q2, do2 = k.clone(), v.clone(), q.clone(), do.clone()
    k2[~seen.to(dev)] = math.nan
    v2[~seen.to(dev)] = math.inf
    q2[dead.to(dev)] = math.nan
    do2[dead.to(dev)] = math.nan
    got = check_attention(q2, k2, v2, do2, lens, q_lens, mask, oracle=(q, k, v, do))
    for t in got:
        assert bool(torch.isfinite(t).all())
    assert not got[0][0].any() and not got[0][3].any() and not got[1][0].any()
    assert not got[2][~seen.to(dev)].any() and not got[3][~seen.to(dev)].any()
    # one mask row for all items
    check_attention(q, k, v, do, None, None, mask[5:6])


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Lq,Lk", [(1, 2048), (200, 96), (6, 700)])
def test_cross_attention_layouts(dev, dtype, Lq, Lk):
    """Slices of fused projections, heads before rows, one encoder output shared by all items, a gradient with stride zero, rows
    that a kernel cannot read in place."""
    B, H, G, D = 2, 4, 2, 64
    q, k, v, do = attention_case(dev, B, Lq, Lk, H, G, D, dtype, seed=9)
    from styler_amd import ops
    lse = torch.empty(B, H, Lq, device=dev)
    ref = ops.cross_attention(q, k, v, lse=lse)
    gref = ops.cross_attention_bwd(q, k, v, ref, do, lse)
    kv = torch.stack([k, v], 2)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.randn(B, Lq, H, D + 4, device=dev).to(dtype)
    wide[..., 1:1 + D] = q
    for qq, kk, vv in ((q, kv[:, :, 0], kv[:, :, 1]), (qt, k, v), (wide[..., 1:1 + D], k, v),
                       (q, k.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2), v)):
        l2 = torch.empty_like(lse)
        o2 = ops.cross_attention(qq, kk, vv, lse=l2)
        assert torch.equal(o2, ref) and torch.equal(l2, lse)
        for a, b in zip(ops.cross_attention_bwd(qq, kk, vv, o2, do, l2), gref):
            assert torch.equal(a, b)
    big = torch.zeros(B, Lq, H + 1, D, device=dev, dtype=dtype)      # out = a slice of a wider buffer
    ops.cross_attention(q, k, v, out=big[:, :, 1:])
    assert torch.equal(big[:, :, 1:], ref) and not big[:, :, 0].any()
    shared = check_attention(q, k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1), do)
    assert shared[2].shape == k.shape
    check_attention(q, k, v, do[:, :1, :1].expand(-1, Lq, H, -1))


@gpu
def test_cross_attention_large_scores(dev):
    """Scores of several hundred and a running maximum that keeps moving: nothing overflows, ties of equal keys share."""
    for dtype in DT:
        q, k, v, do = attention_case(dev, 1, 40, 300, 2, 2, 64, dtype, seed=4, spread=30.0)
        k = (k * torch.linspace(0.1, 2, 300, device=dev).view(1, -1, 1, 1)).to(dtype)
        check_attention(q, k, v, do)
        check_attention(q, k, v, do, scale=1e-3)
        same = k[:, :1].expand(-1, 300, -1, -1).contiguous()
        out = check_attention(q, same, v, do)[0]
        within(out.cpu(), v.double().mean(1, keepdim=True).expand(-1, 40, -1, -1).cpu(), 2 * half_step(dtype) * v.double().abs().mean(1, keepdim=True).cpu() + 1e-5, "mean")


@gpu
def test_cross_attention_is_deterministic_and_batch_independent(dev):
    from styler_amd import ops
    q, k, v, do = attention_case(dev, 3, 1, 900, 8, 2, 64, torch.bfloat16, seed=8)
    a = ops.cross_attention(q, k, v)
    assert torch.equal(a, ops.cross_attention(q, k, v))
    lse = torch.empty(3, 8, 1, device=dev)
    o = ops.cross_attention(q, k, v, lse=lse)
    g1, g2 = (ops.cross_attention_bwd(q, k, v, o, do, lse) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(g1, g2))


@gpu
def test_cross_attention_gradient_by_differences(dev):
    """Directional derivatives of sum(out * w) by central differences in 64-bit arithmetic on the 32-bit outputs.  The step h = 2^-6
    leaves an error of h^2 / 6 times the third derivative (of the order of the first for unit-size inputs) and 2^-22 / h of rounding."""
    from styler_amd import ops
    q, k, v, w = attention_case(dev, 2, 9, 70, 4, 2, 32, torch.float32, seed=12)
    lens = torch.tensor([70, 33], device=dev)
    lse = torch.empty(2, 4, 9, device=dev)
    out = ops.cross_attention(q, k, v, lens, lse=lse)
    grads = ops.cross_attention_bwd(q, k, v, out, w, lse, lens)
    f = lambda q, k, v: float((ops.cross_attention(q, k, v, lens).double() * w.double()).sum())
    h = 2.0 ** -6
    for i in range(3):
        d = torch.randn(*(q, k, v)[i].shape, generator=torch.Generator().manual_seed(i)).to(dev)
        d = d / d.norm() * math.sqrt(8.0)
        plus, minus = ([t + s * h * d if j == i else t for j, t in enumerate((q, k, v))] for s in (1, -1))
        num, ana = (f(*plus) - f(*minus)) / (2 * h), float((grads[i].double() * d.double()).sum())
        assert abs(num - ana) <= 2e-3 * float(w.double().norm()), (i, num, ana)


@gpu
def test_cross_attention_empty_sizes(dev):
    from styler_amd import ops
    z = lambda *s: torch.zeros(*s, device=dev)
    lse = z(2, 4, 3)
    out = ops.cross_attention(z(2, 3, 4, 64) + 1, z(2, 0, 2, 64), z(2, 0, 2, 64), lse=lse)
    assert not out.any() and bool((lse == -math.inf).all())
    dq, dk, dv = ops.cross_attention_bwd(z(2, 3, 4, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), out, out, lse)
    assert not dq.any() and dk.numel() == 0
    assert ops.cross_attention(z(0, 3, 4, 64), z(0, 5, 2, 64), z(0, 5, 2, 64)).shape == (0, 3, 4, 64)
    assert ops.cross_attention(z(2, 0, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64)).shape == (2, 0, 4, 64)
    dq, dk, dv = ops.cross_attention_bwd(z(2, 0, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), z(2, 0, 4, 64), z(2, 0, 4, 64), z(2, 4, 0))
    assert dk.shape == (2, 5, 2, 64) and not dk.any()


def test_cross_attention_refusals():
    from styler_amd import ops
    q, k = torch.zeros(2, 3, 4, 64), torch.zeros(2, 5, 2, 64)
    E = ops.StylerHipError
    lens = torch.tensor([1, 2])
    for bad, text in [
        (lambda: ops.cross_attention(q, k, k), "no CPU form"),
        (lambda: ops.cross_attention(q[0], k, k), "expected"),
        (lambda: ops.cross_attention(q, k[0], k[0]), "expected"),
        (lambda: ops.cross_attention(q.half(), k.half(), k.half()), "float32 or bfloat16"),
        (lambda: ops.cross_attention(q, k.bfloat16(), k), "k must be"),
        (lambda: ops.cross_attention(q, k, k[:, :4]), "v must be"),
        (lambda: ops.cross_attention(q[:, :, :3], k, k), "multiple of the key heads"),
        (lambda: ops.cross_attention(q[..., :60], k[..., :60], k[..., :60]), "head width"),
        (lambda: ops.cross_attention(torch.zeros(1, 1, 1, 136), torch.zeros(1, 1, 1, 136), torch.zeros(1, 1, 1, 136)), "head width"),
        (lambda: ops.cross_attention(q, k, k, lens.int()), "lens must be"),
        (lambda: ops.cross_attention(q, k, k, lens[:1]), "lens must be"),
        (lambda: ops.cross_attention(q, k, k, q_lens=lens[:1]), "q_lens must be"),
        (lambda: ops.cross_attention(q, k, k, mask=torch.zeros(2, 5)), "mask must be"),
        (lambda: ops.cross_attention(q, k, k, mask=torch.zeros(2, 4, dtype=torch.bool)), "mask must be"),
        (lambda: ops.cross_attention(q, k, k, scale=0.0), "scale"),
        (lambda: ops.cross_attention(q, k, k, scale=math.nan), "scale"),
        (lambda: ops.cross_attention(q, k, k, lse=torch.zeros(2, 3, 4)), "lse must be"),
        (lambda: ops.cross_attention(q, k, k, out=torch.zeros(2, 3, 4, 32)), "out must be"),
        (lambda: ops.cross_attention(q, k, k, out=torch.zeros(1, 3, 4, 64).expand(2, -1, -1, -1)), "distinct rows"),
        (lambda: ops.cross_attention_bwd(q, k, k, q, q, None), "lse is needed"),
        (lambda: ops.cross_attention_bwd(q, k, k, q, q[:1], torch.zeros(2, 4, 3)), "dout must be"),
    ]:
        with pytest.raises(E, match=text):
            bad()


# ------------------------------------------------------------------------------------------------------------ rotary positions
def rotary_oracle(x, freqs, pos, interleaved, gain, inverse):
    B, L, H, D = x.shape
    rot = 2 * len(freqs)
    pos = torch.arange(L, dtype=torch.float64) if pos is None else pos.cpu().double()
    angle = pos[..., None] * freqs.cpu()
    w = torch.polar(torch.full_like(angle, gain), -angle if inverse else angle).unsqueeze(-2)
    y = x.cpu().double().clone()
    a, b = (y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()) if interleaved else (y[..., :rot // 2].clone(), y[..., rot // 2:rot].clone())
    t = torch.complex(a, b) * w
    size = torch.complex(a, b).abs() * gain
    tol = torch.zeros_like(y)
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = t.real, t.imag
        tol[..., 0:rot:2] = tol[..., 1:rot:2] = size
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = t.real, t.imag
        tol[..., :rot // 2] = tol[..., rot // 2:rot] = size
    # cos, sin (4 half steps), their products with the gain, the two products and their sum; the reduced angle's rounding (2 pi)
    return y, 24 * U32 * tol + half_step(x.dtype) * y.abs()


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,H,D,rot", [
    (1, 1, 1, 2, 2), (2, 7, 3, 64, 64), (3, 5, 10, 128, 32), (1, 300, 2, 96, 34), (2, 3, 9, 17, 6), (1, 2, 1, 130, 130), (2, 33, 5, 40, 40),
])
def test_rotary_against_definition(dev, B, L, H, D, rot, interleaved, dtype):
    from styler_amd import ops
    g = torch.Generator().manual_seed(B + L + H + D)
    x = torch.randn(B, L, H, D, generator=g).to(dtype).to(dev)
    freqs = ops.rotary_freqs(rot, dev)
    far = (torch.randint(0, 1 << 20, (B, 1), generator=g) + torch.arange(L)).to(dev)
    for pos, gain in ((None, 1.0), (far, 1.0), (-far[:1], 1.25), ((torch.arange(L) / 7.3).float().to(dev), 1.0), (far[0], 1.0)):
        for inverse in (False, True):
            y = ops.rotary(x, freqs, pos, interleaved=interleaved, gain=gain, inverse=inverse)
            ref, tol = rotary_oracle(x, freqs, pos, interleaved, gain, inverse)
            within(y.cpu(), ref, tol + 1e-30, (gain, inverse))
            assert torch.equal(y[..., rot:], x[..., rot:])
    # in place, and a slice of wider rows into a slice of wider rows
    z = x.clone()
    ref = ops.rotary(x, freqs, far, interleaved=interleaved)
    assert torch.equal(ops.rotary(z, freqs, far, interleaved=interleaved, out=z), ref) and torch.equal(z, ref)
    wide, into = torch.zeros(B, L, H + 2, D, device=dev, dtype=dtype), torch.zeros(B, L, H + 3, D, device=dev, dtype=dtype)
    wide[:, :, 1:H + 1] = x
    ops.rotary(wide[:, :, 1:H + 1], freqs, far, interleaved=interleaved, out=into[:, :, 2:H + 2])
    assert torch.equal(into[:, :, 2:H + 2], ref) and not into[:, :, :2].any() and not into[:, :, H + 2:].any()
    # features not contiguous; one row for all items
    assert torch.equal(ops.rotary(x.transpose(2, 3).contiguous().transpose(2, 3), freqs, far, interleaved=interleaved), ref)
    e = ops.rotary(x[:1].expand(B, -1, -1, -1), freqs, far, interleaved=interleaved)
    assert torch.equal(e, ops.rotary(x[:1].expand(B, -1, -1, -1).contiguous(), freqs, far, interleaved=interleaved))


@gpu
def test_rotary_turns_back_and_by_differences(dev):
    from styler_amd import ops
    x = torch.randn(2, 50, 4, 64, generator=torch.Generator().manual_seed(1)).to(dev)
    f = ops.rotary_freqs(48, dev, scaling="linear", factor=4.0)
    y = ops.rotary(x, f)
    back = ops.rotary(y, f, inverse=True)
    assert float((back - x).abs().max()) <= 64 * U32 * float(x.abs().max()) * 2
    # linear in x: <w, R d> = <R^T w, d>
    w, d = torch.randn_like(x), torch.randn_like(x)
    a, b = float((w.double() * ops.rotary(d, f).double()).sum()), float((ops.rotary(w, f, inverse=True).double() * d.double()).sum())
    assert abs(a - b) <= 64 * U32 * float(w.double().norm() * d.double().norm())


def test_rotary_freqs_scalings():
    from styler_amd import ops
    f = ops.rotary_freqs(64, "cpu")
    i = torch.arange(32, dtype=torch.float64)
    assert f.dtype == torch.float64 and torch.allclose(f, 10000.0 ** (-i / 32), rtol=1e-14, atol=0)
    assert torch.equal(ops.rotary_freqs(64, "cpu", scaling="linear", factor=8.0), f / 8)
    b = ops.rotary_freqs(64, "cpu", scaling="base", factor=8.0)
    assert abs(float(b[0]) - 1) < 1e-14 and abs(float(b[-1] / f[-1]) - 1 / 8) < 1e-12
    s = ops.rotary_freqs(64, "cpu", scaling="bands", factor=8.0, orig_len=1000, low=1.0, high=4.0)
    turns = 1000 * f / (2 * math.pi)
    assert torch.equal(s[turns > 4], f[turns > 4]) and torch.allclose(s[turns < 1], f[turns < 1] / 8, rtol=1e-14, atol=0)
    assert bool((s <= f).all()) and bool((s >= f / 8 * (1 - 1e-14)).all())
    assert ops.rotary_freqs(2, "cpu", scaling="base", factor=8.0).tolist() == [1.0]


def test_rotary_refusals():
    from styler_amd import ops
    x, f = torch.zeros(2, 3, 4, 64), ops.rotary_freqs(64, "cpu")
    for bad, text in [
        (lambda: ops.rotary(x, f), "no CPU form"),
        (lambda: ops.rotary(x[0], f), "expected"),
        (lambda: ops.rotary(x.half(), f), "float32 or bfloat16"),
        (lambda: ops.rotary(x, f.float()), "freqs must be"),
        (lambda: ops.rotary(x, ops.rotary_freqs(66, "cpu")), "freqs must be"),
        (lambda: ops.rotary(x, f[:0]), "freqs must be"),
        (lambda: ops.rotary(x, f, torch.zeros(3, dtype=torch.int32)), "pos must be"),
        (lambda: ops.rotary(x, f, torch.zeros(4, dtype=torch.int64)), "pos must be"),
        (lambda: ops.rotary(x, f, torch.zeros(3, 3, dtype=torch.int64)), "pos must be"),
        (lambda: ops.rotary(x, f, gain=math.inf), "gain"),
        (lambda: ops.rotary(x, f, out=x[:1].expand(2, -1, -1, -1)), "distinct rows"),
        (lambda: ops.rotary(x, f, out=x.bfloat16()), "out must be"),
        (lambda: ops.rotary_freqs(3, "cpu"), "even"),
        (lambda: ops.rotary_freqs(4, "cpu", base=0.5), "base"),
        (lambda: ops.rotary_freqs(4, "cpu", scaling="other"), "scaling"),
        (lambda: ops.rotary_freqs(4, "cpu", scaling="bands"), "orig_len"),
    ]:
        with pytest.raises(ops.StylerHipError, match=text):
            bad()


# ------------------------------------------------------------------------------------------------------------ group norm
ACTS = {"none": 0, "relu": 1, "silu": 6, "gelu": 7}


def gn_act(z, act):
    return {"none": lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.special.ndtr(z)}[act]()


def gn_case(dev, B, L, C, dtype, seed=0, offset=3.0):
    g = torch.Generator().manual_seed(seed + B + L * 3 + C * 5)
    x = torch.randn(B, L, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + offset * torch.randn(C, generator=g)
    return [t.to(dev) for t in (x.to(dtype), torch.randn(B, L, C, generator=g).to(dtype), 1 + 0.3 * torch.randn(C, generator=g),
                                0.3 * torch.randn(C, generator=g))]


def check_groupnorm(x, dy, gamma, beta, groups, act, lens=None, eps=1e-5, clean=None):
    from styler_amd import ops
    dev = x.device
    B, L, C = x.shape
    stats = torch.full((B, groups, 2), 9.0, device=dev)
    ld = None if lens is None else lens.to(dev)
    y = ops.groupnorm_act(x, gamma, beta, groups, ACTS[act], eps=eps, lens=ld, stats=stats)
    dx, dgamma, dbeta = ops.groupnorm_act_bwd(x, dy, gamma, beta, stats, groups, ACTS[act], lens=ld)
    x0, dy0 = (x, dy) if clean is None else clean
    u, cg = half_step(x.dtype), C // groups
    ga, be = gamma.cpu().double(), beta.cpu().double()
    y_r, dx_r, ty, tx = (torch.zeros(B, L, C, dtype=torch.float64) for _ in range(4))
    dg_r, db_r, tg, tb = (torch.zeros(C, dtype=torch.float64) for _ in range(4))
    rows = 0
    for b in range(B):
        n = L if lens is None else max(0, min(L, int(lens[b])))
        if n == 0:
            continue
        rows += n
        X = x0[b, :n].cpu().double().requires_grad_()
        G_, Bt = ga.clone().requires_grad_(), be.clone().requires_grad_()
        xg = X.view(n, groups, cg)
        mean, var = xg.mean((0, 2), keepdim=True), xg.var((0, 2), correction=0, keepdim=True)
        rstd = (var + eps).rsqrt()
        xh = ((xg - mean) * rstd).reshape(n, C)
        z = xh * G_ + Bt
        yy = gn_act(z, act)
        d = dy0[b, :n].cpu().double()
        gx, gg, gb = torch.autograd.grad(yy, (X, G_, Bt), d)
        with torch.no_grad():
            r, m = rstd.expand(n, groups, cg).reshape(n, C), mean.expand(n, groups, cg).reshape(n, C)
            # error of xh: the values' own size against the spread, and the statistics' (32-bit sums of up to 64 rows a thread, then a tree)
            ex = 8 * U32 * (X.abs() + m.abs()) * r + 96 * U32 * (1 + xh.abs())
            y_r[b, :n], ty[b, :n] = yy, u * yy.abs() + 1.13 * ex * ga.abs() + 16 * U32 * (z.abs() + xh.abs() * ga.abs())
            # dz = dy act'(z): |act''| <= 1 where it exists; a ReLU's kink is kept away from by the caller
            edz = d.abs() * ((0 if act in ("none", "relu") else 1.0) * ga.abs() * ex + 16 * U32 * (1.2 + z.abs()))
            slope = 1.13 if act in ("silu", "gelu") else 1.0
            D = slope * d.abs() * ga.abs()
            gm = lambda t: t.view(n, groups, cg).mean((0, 2), keepdim=True).expand(n, groups, cg).reshape(n, C)
            e1 = gm(edz * ga.abs()) + 128 * U32 * gm(D)
            e2 = gm(edz * ga.abs() * xh.abs() + D * ex) + 128 * U32 * gm(D * xh.abs())
            dx_r[b, :n] = gx
            tx[b, :n] = u * gx.abs() + r * (edz * ga.abs() + e1 + xh.abs() * e2 + ex * gm(D * xh.abs()) + 96 * U32 * (D + gm(D) + xh.abs() * gm(D * xh.abs())))
            dg_r += gg
            db_r += gb
            tg += (edz * xh.abs() + slope * d.abs() * ex).sum(0) + 160 * U32 * (slope * d.abs() * xh.abs()).sum(0)
            tb += edz.sum(0) + 160 * U32 * (slope * d.abs()).sum(0)
    within(y.cpu(), y_r, ty + 1e-30, "y")
    within(dx.cpu(), dx_r, tx + 1e-30, "dx")
    within(dgamma.cpu(), dg_r, tg + 1e-30, "dgamma")
    within(dbeta.cpu(), db_r, tb + 1e-30, "dbeta")
    assert y.dtype == x.dtype and dx.dtype == x.dtype and dgamma.dtype == torch.float32
    return y, dx, dgamma, dbeta


def off_kink(x, gamma, beta, groups, eps=1e-5, lens=None):
    """Moves the values whose pre-activation is within 2^-12 of a ReLU's kink (all of an item's rows are taken together)."""
    x = x.clone()
    for _ in range(4):
        for b in range(x.shape[0]):
            n = x.shape[1] if lens is None else int(lens[b])
            if n == 0:
                continue
            xg = x[b, :n].double().view(n, groups, -1)
            mean, rstd = xg.mean((0, 2), keepdim=True), (xg.var((0, 2), correction=0, keepdim=True) + eps).rsqrt()
            z = ((xg - mean) * rstd).reshape(n, -1) * gamma.double() + beta.double()
            x[b, :n] = torch.where(z.abs() < 2.0 ** -12, (x[b, :n].double() + 2.0 ** -4).to(x.dtype), x[b, :n])
    return x


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,L,C,groups,act", [
    (1, 1, 1, 1, "none"),                # one value: variance zero
    (2, 1, 64, 4, "silu"),               # one row
    (3, 60, 320, 20, "relu"),            # the audio encoder's norm
    (2, 33, 30, 10, "gelu"),             # three channels a group
    (1, 700, 257, 1, "silu"),            # one odd group
    (2, 90, 80, 80, "gelu"),             # a channel a group
    (2, 1500, 96, 3, "silu"),            # too long for one block
    (1, 5000, 40, 5, "relu"),
    (1, 300, 2200, 2, "none"),           # wide groups: several blocks of channels
    (1, 130, 2100, 700, "silu"),
])
def test_groupnorm_act_against_definition(dev, B, L, C, groups, act, dtype):
    x, dy, gamma, beta = gn_case(dev, B, L, C, dtype)
    if act == "relu":
        x = off_kink(x, gamma, beta, groups)
    check_groupnorm(x, dy, gamma, beta, groups, act)


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("L", [50, 1300])
def test_groupnorm_act_lengths(dev, dtype, L):
    """Lengths of zero, one, all and beyond; the rows behind them hold NaN and infinities and come back as zeros."""
    x, dy, gamma, beta = gn_case(dev, 5, L, 64, dtype, seed=2)
    lens = torch.tensor([0, 1, L, L + 7, L // 3])
    dead = (torch.arange(L)[None] >= lens[:, None]).to(dev)
    x2, dy2 = x.clone(), dy.clone()
    x2[dead], dy2[dead] = math.nan, math.inf
    y, dx, _, _ = check_groupnorm(x2, dy2, gamma, beta, 8, "silu", lens, clean=(x, dy))
    assert not y[dead].any() and not dx[dead].any()


@gpu
@pytest.mark.parametrize("L", [40, 4000])
def test_groupnorm_act_large_offset(dev, L):
    """Channels whose offset is 3000 times their spread: the statistics must not cancel."""
    x, dy, gamma, beta = gn_case(dev, 2, L, 32, torch.float32, seed=6, offset=3000.0)
    check_groupnorm(x, dy, gamma, beta, 32, "silu")


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("L", [60, 3000])
def test_groupnorm_act_layouts(dev, dtype, L):
    from styler_amd import ops
    x, dy, gamma, beta = gn_case(dev, 2, L, 48, dtype, seed=7)
    stats = torch.empty(2, 3, 2, device=dev)
    ref = ops.groupnorm_act(x, gamma, beta, 3, stats=stats)
    gref = ops.groupnorm_act_bwd(x, dy, gamma, beta, stats, 3)
    tol = 4 * half_step(dtype) if dtype == torch.bfloat16 else 1e-5     # other vector widths sum in another order
    wide = torch.zeros(2, L, 61, device=dev, dtype=dtype)
    for lo in (0, 5, 8):
        wide.zero_()
        wide[..., lo:lo + 48] = x
        s = wide[..., lo:lo + 48]
        into = torch.full((2, L, 61), 3.0, device=dev, dtype=dtype)
        ops.groupnorm_act(s, gamma, beta, 3, out=into[..., lo:lo + 48])
        assert float((into[..., lo:lo + 48].float() - ref.float()).abs().max()) <= tol * float(ref.float().abs().max())
        assert bool((into[..., :lo] == 3).all()) and bool((into[..., lo + 48:] == 3).all())
        for a, b in zip(ops.groupnorm_act_bwd(s, dy, gamma, beta, stats, 3), gref):
            assert float((a.float() - b.float()).abs().max()) <= tol * float(b.float().abs().max())
    assert torch.equal(ops.groupnorm_act(x.transpose(1, 2).contiguous().transpose(1, 2), gamma, beta, 3), ref)
    z = x.clone()
    assert torch.equal(ops.groupnorm_act(z, gamma, beta, 3, out=z), ref)
    e = dy[:, :1].expand(-1, L, -1)
    for a, b in zip(ops.groupnorm_act_bwd(x, e, gamma, beta, stats, 3), ops.groupnorm_act_bwd(x, e.contiguous(), gamma, beta, stats, 3)):
        assert torch.equal(a, b)
    g2 = ops.groupnorm_act_bwd(x, dy, gamma, beta, stats, 3)
    assert all(torch.equal(a, b) for a, b in zip(gref, g2))


@gpu
def test_groupnorm_act_matches_the_frameworks_norm(dev):
    """16 channels a group and ReLU over the padded length is ops.groupnorm_relu's case."""
    from styler_amd import ops
    x, _, gamma, beta = gn_case(dev, 3, 60, 320, torch.float32, seed=1)
    a, b = ops.groupnorm_act(x, gamma, beta, 20, ops.ACT_RELU), ops.groupnorm_relu(x, gamma, beta, out=torch.empty_like(x))
    assert float((a - b).abs().max()) <= 2e-5


@gpu
def test_groupnorm_act_empty_sizes(dev):
    from styler_amd import ops
    g = torch.ones(8, device=dev)
    assert ops.groupnorm_act(torch.zeros(0, 4, 8, device=dev), g, g, 2).shape == (0, 4, 8)
    x = torch.zeros(2, 0, 8, device=dev)
    assert ops.groupnorm_act(x, g, g, 2).shape == (2, 0, 8)
    dx, dg, db = ops.groupnorm_act_bwd(x, x, g, g, torch.zeros(2, 2, 2, device=dev), 2)
    assert dx.shape == (2, 0, 8) and not dg.any() and not db.any()


def test_groupnorm_act_refusals():
    from styler_amd import ops
    x, g = torch.zeros(2, 5, 8), torch.ones(8)
    s = torch.zeros(2, 2, 2)
    for bad, text in [
        (lambda: ops.groupnorm_act(x, g, g, 2), "no CPU form"),
        (lambda: ops.groupnorm_act(x[0], g, g, 2), "expected"),
        (lambda: ops.groupnorm_act(x.half(), g, g, 2), "float32 or bfloat16"),
        (lambda: ops.groupnorm_act(x, g, g, 3), "groups"),
        (lambda: ops.groupnorm_act(x, g, g, 0), "groups"),
        (lambda: ops.groupnorm_act(x, g[:4], g, 2), "gamma must be"),
        (lambda: ops.groupnorm_act(x, g, g.bfloat16(), 2), "beta must be"),
        (lambda: ops.groupnorm_act(x, g, g, 2, ops.ACT_TANH), "activation"),
        (lambda: ops.groupnorm_act(x, g, g, 2, eps=-1.0), "eps"),
        (lambda: ops.groupnorm_act(x, g, g, 2, lens=torch.zeros(3, dtype=torch.int64)), "lens must be"),
        (lambda: ops.groupnorm_act(x, g, g, 2, stats=s[:1]), "stats must be"),
        (lambda: ops.groupnorm_act_bwd(x, x, g, g, None, 2), "stats are needed"),
    ]:
        with pytest.raises(ops.StylerHipError, match=text):
            bad()


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Lq", [1, 50, 200])
def test_one_seen_key_has_no_score_gradient(dev, dtype, Lq):
    """A query that sees one key gives that key's value, and its scores have no gradient: exactly, not up to a rounding."""
    from styler_amd import ops
    B, H, G, D = 3, 4, 2, 64
    q, k, v, do = attention_case(dev, B, Lq, 90, H, G, D, dtype, seed=21, spread=4.0)
    mask = torch.ones(B, 90, dtype=torch.bool, device=dev)
    for b, j in enumerate((0, 37, 89)):
        mask[b, j] = False
    for kk, vv, m in ((k[:, :1], v[:, :1], None), (k, v, mask)):
        lse = torch.empty(B, H, Lq, device=dev)
        out = ops.cross_attention(q, kk, vv, mask=m, lse=lse)
        ref = vv[:, :1] if m is None else torch.stack([v[b, j] for b, j in enumerate((0, 37, 89))])[:, None]
        assert torch.equal(out, ref.repeat_interleave(H // G, 2).expand(B, Lq, H, D))
        dq, dk, dv = ops.cross_attention_bwd(q, kk, vv, out, do, lse, mask=m)
        assert not dq.any() and not dk.any() and bool(dv.any())


@gpu
@pytest.mark.parametrize("dtype", DT)
def test_groupnorm_act_of_single_values(dev, dtype):
    """A group of one value is its own mean: y = act(beta) and dx = 0 to the last bit."""
    from styler_amd import ops
    x, dy, gamma, beta = gn_case(dev, 8, 1, 128, dtype, seed=13)
    stats = torch.empty(8, 128, 2, device=dev)
    y = ops.groupnorm_act(x, gamma, beta, 128, ops.ACT_NONE, stats=stats)
    assert torch.equal(y, beta.to(dtype).expand(8, 1, 128))
    dx, dgamma, dbeta = ops.groupnorm_act_bwd(x, dy, gamma, beta, stats, 128, ops.ACT_NONE)
    assert not dx.any() and not dgamma.any()
