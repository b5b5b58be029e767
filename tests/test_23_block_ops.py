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
@pytest.mark.parametrize("B,Lq,Lk,H,G,D,lens,q_lens", [
    (3, 530, 500, 2, 1, 32, [500, 3, 260], [530, 530, 100]),              # long ragged items: the most work first
    (4, 600, 450, 1, 1, 128, [17, 0, 450, 450], [600, 1, 0, 599]),
    (5, 520, 510, 2, 2, 80, [510, 64, 65, 1, 509], [1, 520, 519, 520, 0]),
    (4, 1100, 1000, 1, 1, 32, [1000, 33, 0, 999], [1100, 1099, 5, 64]),   # (fp32: through planes from here on)
    (3, 1030, 1020, 2, 2, 64, [1020, 640, 31], [1030, 0, 1]),
    (3, 1, 5000, 4, 1, 64, [5000, 3, 0], None),                           # shares of which some see nothing
    (3, 2, 4097, 16, 4, 128, [4097, 4096, 65], [2, 1, 2]),
    (2, 9, 1500, 8, 1, 32, [1500, 700], None),                            # 72 rows of one key head
    (20, 2, 33, 4, 4, 64, None, None),                                    # many items of few rows
    (300, 130, 5, 2, 1, 8, None, None),                                   # more blocks than the chip holds at once
    (520, 70, 90, 1, 1, 64, [90 - i % 91 for i in range(520)], [i % 71 for i in range(520)]),
    (1, 2500, 33, 2, 1, 64, [32], [2499]),                                # the key gradient's rows shared out, few keys
])
def test_cross_attention_sizes_and_lengths(dev, B, Lq, Lk, H, G, D, lens, q_lens, dtype):
    t = lambda x: None if x is None else torch.tensor(x)
    q, k, v, do = attention_case(dev, B, Lq, Lk, H, G, D, dtype, seed=21)
    got = check_attention(q, k, v, do, t(lens), t(q_lens))
    for b, n in enumerate(lens or []):
        assert not got[2][b, n:].any() and not got[3][b, n:].any()
    for b, n in enumerate(q_lens or []):
        assert not got[0][b, n:].any() and not got[1][b, n:].any()


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
@pytest.mark.parametrize("B,Lq,Lk,H,G,D,shared", [
    (5, 130, 2101, 8, 4, 96, False),         # two blocks of keys in the ordering, few rows: two key groups
    (4, 520, 1203, 4, 2, 64, True),          # one mask for all items
    (3, 1030, 700, 6, 6, 128, False),
    (9, 1100, 4100, 1, 1, 32, False),        # blocks of 128 rows, three blocks of keys
])
def test_cross_attention_long_masks(dev, B, Lq, Lk, H, G, D, shared, dtype):
    """Masks long enough that the seen keys are put in front: every key, none, one, a run, every other, at random; with lengths, and
    what stands in the unseen rows is NaN."""
    q, k, v, do = attention_case(dev, B, Lq, Lk, H, G, D, dtype, seed=31)
    mask = torch.rand(B, Lk + 3, generator=torch.Generator().manual_seed(6))[:, 3:] < 0.4         # rows on odd addresses
    mask[1] = False
    mask[2] = True
    mask[2, Lk - 30] = False
    if B > 3:
        mask[3] = torch.arange(Lk) % 2 == 0
        mask[3, :600] = True
    lens = torch.randint(Lk // 2, Lk + 50, (B,), generator=torch.Generator().manual_seed(7))
    lens[1], lens[2] = Lk, Lk
    if B > 4:
        lens[4] = 0
    if shared:
        mask = mask[:1]
    seen = (torch.arange(Lk)[None] < lens[:, None]) & ~mask
    k2, v2 = k.clone(), v.clone()
    k2[~seen.to(dev)] = math.nan
    v2[~seen.to(dev)] = math.nan
    got = check_attention(q, k2, v2, do, lens, torch.randint(1, Lq + 1, (B,)), mask, oracle=(q, k, v, do))
    assert not got[2][~seen.to(dev)].any() and not got[3][~seen.to(dev)].any()
    check_attention(q, k2, v2, do, lens, None, mask, oracle=(q, k, v, do))


@gpu
@pytest.mark.parametrize("B,Lq,Lk,H,G,D,dtype", [
    (5, 1100, 2101, 16, 8, 32, torch.bfloat16), (16, 2050, 2200, 2, 2, 32, torch.bfloat16),
    (2, 2100, 8200, 4, 4, 32, torch.bfloat16), (2, 2050, 4097, 4, 2, 64, torch.bfloat16), (8, 1030, 1025, 8, 8, 64, torch.bfloat16),
    (2, 1100, 4200, 4, 4, 128, torch.bfloat16), (9, 1000, 530, 8, 8, 80, torch.bfloat16),
    (5, 1100, 2101, 4, 2, 32, torch.float32), (3, 600, 1500, 8, 4, 64, torch.float32), (2, 300, 6000, 2, 2, 72, torch.float32),
])
def test_cross_attention_masked_keys_are_left_out(dev, B, Lq, Lk, H, G, D, dtype):
    """A mask that is put in order gives, bit for bit, what the seen keys give that stand at the front of each item by themselves."""
    from styler_amd import ops
    g = torch.Generator(device=dev).manual_seed(B + Lk)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(dtype)
    q, kv, do = r(B, Lq, H, D), r(B, Lk, 2, G, D), r(B, Lq, H, D)
    mask = torch.rand(B, Lk, generator=g, device=dev) < torch.linspace(0.1, 0.9, B, device=dev)[:, None]
    mask[1] = True                                            # an item without keys
    lens = torch.full((B,), Lk - 5, device=dev)
    seen = ~mask & (torch.arange(Lk, device=dev)[None] < lens[:, None])
    order = torch.argsort((~seen).int(), dim=1, stable=True)
    front = torch.gather(kv, 1, order.view(B, Lk, 1, 1, 1).expand(-1, -1, 2, G, D))
    count = seen.sum(1)

    def both(k, v, n, m):
        lse = torch.empty(B, H, Lq, device=dev)
        out = ops.cross_attention(q, k, v, n, mask=m, lse=lse)
        return out, lse, *ops.cross_attention_bwd(q, k, v, out, do, lse, n, mask=m)

    a, b = both(kv[:, :, 0], kv[:, :, 1], lens, mask), both(front[:, :, 0], front[:, :, 1], count, None)
    assert all(torch.equal(x, y) for x, y in zip(a[:3], b[:3]))
    for x, y in zip(a[3:], b[3:]):
        assert torch.equal(torch.gather(x, 1, order.view(B, Lk, 1, 1).expand(-1, -1, G, D)), y)
        assert not x[~seen].any()


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


# ------------------------------------------------------------------------------------------------------------ together
def test_block_operators_have_schemas_and_fake_kernels():
    import styler_amd.torch_ops as T
    from torch._subclasses.fake_tensor import FakeTensorMode
    assert all(hasattr(torch.ops.styler, n) for n in T.BLOCK_OPS)
    with FakeTensorMode():
        q, k = torch.empty(2, 7, 8, 64, dtype=torch.bfloat16), torch.empty(2, 9, 2, 64, dtype=torch.bfloat16)
        out, lse = torch.ops.styler.cross_attention(q, k, k)
        assert out.shape == q.shape and out.dtype == q.dtype and tuple(lse.shape) == (2, 8, 7) and lse.dtype == torch.float32
        g = torch.ops.styler.cross_attention_bwd(q, k, k, out, out, lse, None, None, None, None)
        assert [tuple(t.shape) for t in g] == [(2, 7, 8, 64), (2, 9, 2, 64), (2, 9, 2, 64)]
        assert torch.ops.styler.rotary(q, torch.empty(32, dtype=torch.float64)).shape == q.shape
        x, w = torch.empty(2, 5, 48, dtype=torch.bfloat16), torch.empty(48)
        y, stats = torch.ops.styler.groupnorm_act(x, w, w, 3, 6)
        assert y.shape == x.shape and tuple(stats.shape) == (2, 3, 2)
        dx, dg, db = torch.ops.styler.groupnorm_act_bwd(x, y, w, w, stats, 3, 6, None)
        assert dx.shape == x.shape and dg.shape == w.shape and dg.dtype == torch.float32


def block_case(dev, dtype, seed=0):
    """A decoder block over an encoder's states: norm -> query projection -> rotary queries and keys -> attention."""
    g = torch.Generator().manual_seed(seed)
    B, Lq, Lk, C, H, G, D = 3, 70, 41, 256, 4, 2, 64
    r = lambda *s: torch.randn(*s, generator=g)
    t = dict(x=r(B, Lq, C).to(dtype), enc=r(B, Lk, 2, G, D).to(dtype), w=(r(H * D, C) / 16), gamma=1 + 0.1 * r(C), beta=0.1 * r(C),
             dout=r(B, Lq, H, D).to(dtype))
    return {k: v.to(dev) for k, v in t.items()}, torch.tensor([70, 1, 33], device=dev), torch.tensor([41, 20, 7], device=dev)


def block_forward(ops_, x, enc, w, gamma, beta, q_lens, lens, freqs, native):
    B, Lq, C = x.shape
    H, G, D = 4, 2, 64
    pos_q = (torch.arange(Lq, device=x.device) / 1.7).float()
    if native:
        y, _ = torch.ops.styler.groupnorm_act(x, gamma, beta, 16, 6, 1e-5, q_lens)
        q = torch.ops.styler.conv_gemm(y.float(), w, None, 0, 0).to(x.dtype).view(B, Lq, H, D)
        q = torch.ops.styler.rotary(q, freqs, pos_q)
        k = torch.ops.styler.rotary(enc[:, :, 0], freqs, None)
        return torch.ops.styler.cross_attention(q, k, enc[:, :, 1], lens, q_lens)[0]
    on = (torch.arange(Lq, device=x.device)[None] < q_lens[:, None])[..., None]
    out = torch.zeros(B, Lq, H, D, dtype=torch.float64, device=x.device)
    turn = lambda t, p: torch.cat([t[..., :32] * p.cos()[:, None] - t[..., 32:] * p.sin()[:, None],
                                   t[..., 32:] * p.cos()[:, None] + t[..., :32] * p.sin()[:, None]], -1)
    for b in range(B):
        n, m = int(q_lens[b]), int(lens[b])
        xb = x[b, :n].view(n, 16, C // 16)
        z = ((xb - xb.mean((0, 2), keepdim=True)) * (xb.var((0, 2), correction=0, keepdim=True) + 1e-5).rsqrt()).reshape(n, C) * gamma + beta
        q = turn((z * torch.sigmoid(z) @ w.T).view(n, H, D), pos_q[:n, None].double() * freqs)
        k = turn(enc[b, :m, 0], torch.arange(m, device=x.device)[:, None].double() * freqs)
        for h in range(H):
            out[b, :n, h] = torch.softmax(q[:, h] @ k[:, h // 2].T / 8, -1) @ enc[b, :m, 1, h // 2]
    return out


@gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 4e-2)])
def test_decoder_block_over_encoder_states(dev, dtype, tol):
    """The operators one after the other through the dispatcher, gradients by the registered formulas, against 64-bit math.  fp32: a
    chain of some thirty 32-bit roundings over sums of up to 256 terms, relative to the largest value; bf16: five roundings to bf16
    on the way (2^-8 each, twice that through the softmax's logits)."""
    import styler_amd.torch_ops  # noqa: F401
    from styler_amd import ops
    t, q_lens, lens = block_case(dev, dtype)
    freqs = ops.rotary_freqs(64, dev)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items() if k != "dout"}
    out = block_forward(ops, *(leaves[k] for k in ("x", "enc", "w", "gamma", "beta")), q_lens, lens, freqs, True)
    grads = torch.autograd.grad(out, list(leaves.values()), t["dout"])
    ref_leaves = {k: v.double().clone().requires_grad_() for k, v in t.items() if k != "dout"}
    ref = block_forward(None, *(ref_leaves[k] for k in ("x", "enc", "w", "gamma", "beta")), q_lens, lens, freqs, False)
    on = (torch.arange(70, device=dev)[None] < q_lens[:, None])[..., None, None]
    ref_grads = torch.autograd.grad(ref, list(ref_leaves.values()), torch.where(on, t["dout"].double(), 0.0))
    assert float((out.double() - ref).detach().abs().max()) <= tol * float(ref.detach().abs().max())
    for (k, _), a, b in zip(leaves.items(), grads, ref_grads):
        assert float((a.double() - b).abs().max()) <= tol * float(b.abs().max()), k


@gpu
def test_block_operators_opcheck(dev):
    import styler_amd.torch_ops  # noqa: F401
    from styler_amd import ops
    q, k, v, do = attention_case(dev, 2, 7, 9, 4, 2, 32, torch.float32)
    lens = torch.tensor([9, 4], device=dev)
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(torch.ops.styler.cross_attention, (q.requires_grad_(), k.requires_grad_(), v.requires_grad_(), lens), test_utils=tests)
    torch.library.opcheck(torch.ops.styler.rotary, (torch.randn(2, 5, 3, 64, device=dev, requires_grad=True), ops.rotary_freqs(32, dev)), test_utils=tests)
    x, dy, gamma, beta = gn_case(dev, 2, 9, 32, torch.float32)
    torch.library.opcheck(torch.ops.styler.groupnorm_act, (x.requires_grad_(), gamma.requires_grad_(), beta.requires_grad_(), 4, 6), test_utils=tests)


@gpu
def test_block_operators_refuse_gradients_they_do_not_have(dev):
    import styler_amd.torch_ops  # noqa: F401
    from styler_amd import ops
    q, k, v, do = attention_case(dev, 1, 7, 9, 2, 2, 32, torch.float32)
    out, lse = torch.ops.styler.cross_attention(q.requires_grad_(), k, v)
    with pytest.raises(ops.StylerHipError, match="no gradient"):
        (out.sum() + lse.sum()).backward()
    x, dy, gamma, beta = gn_case(dev, 2, 9, 32, torch.float32)
    y, stats = torch.ops.styler.groupnorm_act(x.requires_grad_(), gamma, beta, 4, 6)
    with pytest.raises(ops.StylerHipError, match="no gradient"):
        stats.sum().backward()


@gpu
def test_block_operators_gradients_of_broadcast_inputs(dev):
    """Keys that a batch shares, a channel-expanded gradient (a sum's) and an expanded x: autograd sums what broadcasting spread."""
    import styler_amd.torch_ops  # noqa: F401
    from styler_amd import ops
    q, k, v, _ = attention_case(dev, 3, 20, 50, 4, 2, 32, torch.float32)
    k1, v1 = (t[:1].clone().requires_grad_() for t in (k, v))
    torch.ops.styler.cross_attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1))[0].sum().backward()
    k2, v2 = (t[:1].expand(3, -1, -1, -1).contiguous() for t in (k, v))
    lse = torch.empty(3, 4, 20, device=dev)
    out = ops.cross_attention(q, k2, v2, lse=lse)
    _, dk, dv = ops.cross_attention_bwd(q, k2, v2, out, torch.ones_like(out), lse)
    for got, ref in ((k1.grad, dk), (v1.grad, dv)):
        assert float((got - ref.sum(0, keepdim=True)).abs().max()) <= 8 * half_step(torch.float32) * float(ref.abs().sum(0).max())
    x, _, gamma, beta = gn_case(dev, 1, 30, 32, torch.float32)
    x1 = x.clone().requires_grad_()
    torch.ops.styler.groupnorm_act(x1.expand(4, -1, -1), gamma, beta, 4, 6)[0][:, 3:].sum().backward()
    x2 = x.clone().requires_grad_()
    (4 * torch.ops.styler.groupnorm_act(x2, gamma, beta, 4, 6)[0][:, 3:]).sum().backward()
    assert float((x1.grad - x2.grad).abs().max()) <= 64 * half_step(torch.float32) * float(x2.grad.abs().max())
    f = ops.rotary_freqs(32, dev)
    x1 = torch.randn(1, 9, 1, 32, device=dev, requires_grad=True)
    torch.ops.styler.rotary(x1.expand(2, 9, 3, 32), f).sum().backward()
    one = ops.rotary(torch.ones(1, 9, 1, 32, device=dev), f, inverse=True)
    assert float((x1.grad - 6 * one).abs().max()) <= 6 * 8 * half_step(torch.float32) * 2


@gpu
def test_groupnorm_act_gradient_by_differences(dev):
    """Central differences of sum(y dy) in fp32 on a few directions.  With a step of h the quotient is off by the third derivative's
    h^2 / 6 and by y's rounding over 2 h: 600 values of about 2^-24 each add up to less than 1e-5, so h = 1e-2 leaves 1e-3; both are far below
    the 2e-2 allowed of derivatives around 1."""
    from styler_amd import ops
    for act in (ops.ACT_NONE, ops.ACT_SILU, ops.ACT_GELU):
        x, dy, gamma, beta = gn_case(dev, 2, 10, 30, torch.float32, offset=0.5)
        lens = torch.tensor([10, 6], device=dev)
        stats = torch.empty(2, 3, 2, device=dev)
        f = lambda x, g, b: float((ops.groupnorm_act(x, g, b, 3, act, lens=lens, stats=stats).double() * dy.double()).sum())
        f(x, gamma, beta)
        grads = ops.groupnorm_act_bwd(x, dy, gamma, beta, stats.clone(), 3, act, lens=lens)
        gen = torch.Generator().manual_seed(5)
        for i in range(3):
            t = [x, gamma, beta]
            d = torch.randn(t[i].shape, generator=gen).to(dev)
            d /= d.norm()
            up, down = list(t), list(t)
            up[i], down[i] = t[i] + 1e-2 * d, t[i] - 1e-2 * d
            assert abs((f(*up) - f(*down)) / 2e-2 - float((grads[i].double() * d).sum())) < 2e-2, (act, i)


@gpu
def test_block_operators_in_a_graph(dev):
    """Captured once, replayed with new inputs in the same buffers and eager calls of the same operators in between; two graphs that
    share a pool are replayed in turn.  Every replay equals the eager result."""
    from styler_amd import ops
    freqs = ops.rotary_freqs(64, dev)
    lens = torch.tensor([300, 120], device=dev)

    def make(Lq, dtype):
        q, k, v, do = attention_case(dev, 2, Lq, 300, 4, 2, 64, dtype, seed=Lq)
        x, dy, gamma, beta = gn_case(dev, 2, 900 + Lq, 64, dtype, seed=Lq)
        bufs = [q, k, v, do, x, dy]

        def step():
            qr, kr = ops.rotary(q, freqs), ops.rotary(k, freqs)
            lse = torch.empty(2, 4, Lq, device=dev)
            out = ops.cross_attention(qr, kr, v, lens, lse=lse)
            g = ops.cross_attention_bwd(qr, kr, v, out, do, lse, lens)
            stats = torch.empty(2, 4, 2, device=dev)
            y = ops.groupnorm_act(x, gamma, beta, 4, stats=stats)
            return [out, *g, ops.rotary(g[0], freqs, inverse=True), y, *ops.groupnorm_act_bwd(x, dy, gamma, beta, stats, 4)]
        return bufs, step

    sets = [make(1, torch.bfloat16), make(70, torch.float32), make(150, torch.bfloat16)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _, step in sets:
            step()
    torch.cuda.current_stream().wait_stream(side)
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for bufs, step in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            got = step()
        graphs.append((g, got, bufs, step))
    gen = torch.Generator().manual_seed(99)
    for turn in range(4):
        for g, got, bufs, step in graphs:
            for t in bufs:
                t.copy_(torch.randn(t.shape, generator=gen).to(t.dtype))
            want = [t.clone() for t in step()]
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b), turn


@gpu
def test_block_operators_on_another_stream(dev):
    """Two streams at once, each with its own workspaces: the results of either are those of one alone."""
    from styler_amd import ops
    cases = [attention_case(dev, 2, Lq, 4000, 8, 2, 64, dt, seed=s) for s, (Lq, dt) in enumerate([(1, torch.bfloat16), (90, torch.float32)])]

    def step(q, k, v, do):
        lse = torch.empty(2, 8, q.shape[1], device=dev)
        out = ops.cross_attention(q, k, v, lse=lse)
        return [out, *ops.cross_attention_bwd(q, k, v, out, do, lse)]

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(step(*c))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i % 2]))


@gpu
def test_block_operators_make_their_device_current(dev, monkeypatch):
    """Called with another device current: the call is made again with the tensors' own, with every argument."""
    from styler_amd import ops
    q, k, v, do = attention_case(dev, 2, 20, 30, 4, 2, 64, torch.float32)
    x, dy, gamma, beta = gn_case(dev, 2, 40, 64, torch.float32)
    lens, q_lens, gl = (torch.tensor(t, device=dev) for t in ([30, 11], [7, 20], [33, 40]))
    mask = torch.arange(30, device=dev)[None] == 4
    f = ops.rotary_freqs(64, dev)
    pos = torch.arange(20, device=dev).float() * 0.7

    def calls():
        lse, stats = torch.empty(2, 4, 20, device=dev), torch.empty(2, 4, 2, device=dev)
        out = ops.cross_attention(q, k, v, lens, q_lens=q_lens, mask=mask, scale=0.2, out=torch.empty_like(q), lse=lse)
        return [out, lse, *ops.cross_attention_bwd(q, k, v, out, do, lse, lens, q_lens=q_lens, mask=mask, scale=0.2),
                ops.rotary(q, f, pos, interleaved=True, gain=1.5, inverse=True, out=torch.empty_like(q)),
                ops.groupnorm_act(x, gamma, beta, 4, ops.ACT_GELU, eps=0.1, lens=gl, out=torch.empty_like(x), stats=stats), stats,
                *ops.groupnorm_act_bwd(x, dy, gamma, beta, stats, 4, ops.ACT_GELU, lens=gl)]

    want, real, turn = calls(), ops._current_device, [0]

    def other_first():
        turn[0] += 1
        return -1 if turn[0] % 2 else real()

    monkeypatch.setattr(ops, "_current_device", other_first)
    got = calls()
    assert turn[0] == 10 and all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
def test_block_operators_past_32_bit_offsets(dev):
    """Tensors of more than 2^31 elements: what stands at their end is what is read and written."""
    from styler_amd import ops
    Lk = (1 << 21) + 77
    k, v = (torch.zeros(1, Lk, 8, 128, device=dev, dtype=torch.bfloat16) for _ in range(2))
    assert k.numel() > 1 << 31
    q, kt, vt, _ = attention_case(dev, 1, 2, 100, 16, 8, 128, torch.bfloat16, seed=2)
    k[:, -100:], v[:, -100:] = kt, vt
    mask = torch.ones(1, Lk, dtype=torch.bool, device=dev)
    mask[:, -100:] = False
    a, b = ops.cross_attention(q, k, v, mask=mask), ops.cross_attention(q, kt, vt)
    assert float((a.float() - b.float()).abs().max()) <= 2 * half_step(torch.bfloat16) * float(b.float().abs().max())
    x = k.view(1, Lk, 8, 128)
    f = ops.rotary_freqs(128, dev)
    pos = torch.arange(Lk, device=dev)
    y = ops.rotary(x, f, pos, out=v)
    assert torch.equal(y[:, -100:], ops.rotary(kt, f, pos[-100:])) and not y[:, :-100].any()
    y.zero_()
    rows = x.view(1, Lk, 1024)
    w = torch.ones(1024, device=dev)
    ops.groupnorm_act(rows, w, 0 * w, 8, ops.ACT_NONE, out=y.view(1, Lk, 1024))
    t = kt.double().view(100, 8, 128)
    mean = t.sum((0, 2)) / (Lk * 128)
    var = (t ** 2).sum((0, 2)) / (Lk * 128) - mean ** 2
    ref = ((t - mean[:, None]) * (var[:, None] + 1e-5).rsqrt()).view(1, 100, 1024)
    assert float((y.view(1, Lk, 1024)[:, -100:].double() - ref).abs().max()) <= 2 * half_step(torch.bfloat16) * float(ref.abs().max())


def test_block_operators_refuse_shared_outputs():
    """An output in an input's place would be read after it was written; only the elementwise operators work in place, in one layout."""
    from styler_amd import ops
    q, k = torch.zeros(2, 4, 4, 32), torch.zeros(2, 4, 4, 32)
    for out in (q, k):
        with pytest.raises(ops.StylerHipError, match="shares memory"):
            ops.cross_attention(q, k, k, out=out)
    with pytest.raises(ops.StylerHipError, match="shares memory"):
        ops.rotary(q, ops.rotary_freqs(32, "cpu"), out=q.transpose(1, 2))
    with pytest.raises(ops.StylerHipError, match="no CPU form"):
        ops.rotary(q, ops.rotary_freqs(32, "cpu"), out=q)
    x, w = torch.zeros(4, 4, 32), torch.ones(32)
    with pytest.raises(ops.StylerHipError, match="shares memory"):
        ops.groupnorm_act(x, w, w, 4, out=x.transpose(0, 1))
    with pytest.raises(ops.StylerHipError, match="no CPU form"):
        ops.groupnorm_act(x, w, w, 4, out=x)


@gpu
def test_groupnorm_act_of_many_items(dev):
    """More items than a grid's third axis holds, in both forms; items are alike, so each must equal a small batch's."""
    from styler_amd import ops
    for L, C, G in ((1, 16, 4), (2, 2056, 1), (130, 64, 64)):
        B, n = 70001, 7
        x, dy, gamma, beta = gn_case(dev, n, L, C, torch.bfloat16, seed=6)
        at = torch.arange(B, device=dev) % n
        xs, dys = x[at], dy[at]
        lens = torch.tensor([L, L, 0, 1, L, (L + 1) // 2, L], device=dev)
        s1, s2 = torch.empty(n, G, 2, device=dev), torch.empty(B, G, 2, device=dev)
        y1, y2 = ops.groupnorm_act(x, gamma, beta, G, lens=lens, stats=s1), ops.groupnorm_act(xs, gamma, beta, G, lens=lens[at], stats=s2)
        assert float((y1[at].float() - y2.float()).abs().max()) <= 4 * half_step(torch.bfloat16) * float(y1.float().abs().max())
        assert float((s1[at] - s2).abs().max()) <= 1e-5 * float(s1.abs().max())
        g1, g2 = ops.groupnorm_act_bwd(x, dy, gamma, beta, s1, G, lens=lens), ops.groupnorm_act_bwd(xs, dys, gamma, beta, s2, G, lens=lens[at])
        assert float((g1[0][at].float() - g2[0].float()).abs().max()) <= 4 * half_step(torch.bfloat16) * float(g1[0].float().abs().max())
        # the parameters' gradients add B / n of each item, in 32 bits one after the other: B steps of half a unit at most
        w = torch.bincount(at, minlength=n).double()
        each = [ops.groupnorm_act_bwd(x[i:i + 1], dy[i:i + 1], gamma, beta, s1[i:i + 1], G, lens=lens[i:i + 1])[1:] for i in range(n)]
        for j, got in enumerate(g2[1:]):
            ref = sum(w[i] * e[j].double() for i, e in enumerate(each))
            size = sum(w[i] * e[j].double().abs() for i, e in enumerate(each))
            assert float(((got.double() - ref).abs() / (size + 1e-3)).max()) <= B * half_step(torch.float32) * 0.5


# ------------------------------------------------------------------------------------------------------------ values that are not finite
@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("L", [60, 3000])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_groupnorm_act_shows_values_that_are_not_finite(dev, act, L, dtype):
    """A NaN or an infinity among a group's valid rows makes the group NaN, forward and backward, whatever the activation; the other
    groups and items are what they are without it."""
    from styler_amd import ops
    x, dy, gamma, beta = gn_case(dev, 3, L, 64, dtype, seed=17)
    lens = torch.tensor([L, L - 7, L], device=dev)

    def both(x):
        stats = torch.empty(3, 4, 2, device=dev)
        y = ops.groupnorm_act(x, gamma, beta, 4, ACTS[act], lens=lens, stats=stats)
        return (y, *ops.groupnorm_act_bwd(x, dy, gamma, beta, stats, 4, ACTS[act], lens=lens))

    ref = both(x)
    for bad in (math.nan, math.inf, -math.inf):
        x2 = x.clone()
        x2[1, L // 3, 21] = bad                               # group 1 of item 1
        got = both(x2)
        for a, b in zip(got[:2], ref[:2]):
            a = a.clone()
            assert bool(a[1, :L - 7, 16:32].isnan().all()), (bad, act)
            a[1, :L - 7, 16:32] = b[1, :L - 7, 16:32]
            assert torch.equal(a, b)
        assert bool(got[2][16:32].isnan().all())              # dgamma
        for a, b in zip(got[2:], ref[2:]):
            assert torch.equal(a[:16], b[:16]) and torch.equal(a[32:], b[32:])


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("L", [60, 3000])
@pytest.mark.parametrize("groups", [4, 64])
def test_groupnorm_act_of_a_variance_past_the_range(dev, groups, L, dtype):
    """Squares that leave the range of 32 bits make the variance infinite: 1 / sqrt(inf) = 0, so y = act(beta) and dx = 0."""
    from styler_amd import ops
    C, cg = 64, 64 // groups
    x, dy, gamma, beta = gn_case(dev, 2, L, C, dtype, seed=18)
    g = torch.Generator().manual_seed(1)
    x2 = x.clone()
    x2[1, :, :cg] = (1e20 * torch.randn(L, cg, generator=g)).to(dtype).to(dev)
    stats, clean = (torch.empty(2, groups, 2, device=dev) for _ in range(2))
    y, ref = ops.groupnorm_act(x2, gamma, beta, groups, stats=stats), ops.groupnorm_act(x, gamma, beta, groups, stats=clean)
    assert not stats[1, 0, 1].any() and torch.equal(stats[1, 1:], clean[1, 1:]) and torch.equal(stats[0], clean[0])
    want = beta[:cg].double() * torch.sigmoid(beta[:cg].double())
    within(y[1, :, :cg].cpu(), want.cpu().expand(L, cg), (half_step(dtype) + 8 * U32) * want.abs().cpu().expand(L, cg) + 1e-30, "y")
    assert torch.equal(y[1, :, cg:], ref[1, :, cg:]) and torch.equal(y[0], ref[0])
    dx, dgamma, dbeta = ops.groupnorm_act_bwd(x2, dy, gamma, beta, stats, groups)
    assert not dx[1, :, :cg].any() and bool(dgamma.isfinite().all()) and bool(dbeta.isfinite().all())


# ------------------------------------------------------------------------------------------------------------ few seen keys
def score_gradient_oracle(q, k, v, do, seen, scale):
    """(dq, dk) in 64 bits over the seen keys [B, Lk], and bounds that leave the rounding of the stored output out of the rows'
    delta = sum_j P_j (do . v_j): P's relative error e, the 32-bit sums, the roundings of dS and of the result."""
    B, Lq, H, D = q.shape
    Lk, G = k.shape[1:3]
    R, u = H // G, half_step(q.dtype)
    dq, tq = (torch.zeros(B, Lq, H, D, dtype=torch.float64) for _ in range(2))
    dk, tk = (torch.zeros(B, Lk, G, D, dtype=torch.float64) for _ in range(2))
    q, k, v, do = (t.cpu().double() for t in (q, k, v, do))
    for b in range(B):
        j = seen[b].nonzero()[:, 0]
        for h in range(H if len(j) else 0):
            Q, K, V, dO = q[b, :, h], k[b, j, h // R], v[b, j, h // R], do[b, :, h]
            S = Q @ K.T * scale
            lse = torch.logsumexp(S, 1, keepdim=True)
            P = torch.exp(S - lse)
            e = (D + 4) * U32 * (Q.abs() @ K.abs().T * scale).max() + 4 * U32 * (S.abs().max() + lse.abs().max()) + (len(j) + 64) * U32
            O, dP = P @ V, dO @ V.T
            delta = (dO * O).sum(1, keepdim=True)
            A = dO.abs() @ V.abs().T                             # what the 32-bit sums of dP go by
            # delta = dl + sum P (dP - dl): dl (off by the rounding of o) enters with sum P - 1, i.e. e; then the sums
            dl = (dO.abs() * (1 + u) * O.abs()).sum(1, keepdim=True)
            E = 2 * e * (dl + (P * dP.abs()).sum(1, keepdim=True)) + (D + len(j) + 40) * U32 * ((P * A).sum(1, keepdim=True) + dl)
            dS = P * (dP - delta)
            eS = P * (E + (D + 4) * U32 * A) + (u + 2 * e) * dS.abs()
            n = (max(len(j), R * Lq) + 16) * U32
            dq[b, :, h], tq[b, :, h] = scale * dS @ K, scale * (eS + n * dS.abs()) @ K.abs()
            dk[b, j, h // R] += scale * dS.T @ Q
            tk[b, j, h // R] += scale * (eS + n * dS.abs()).T @ Q.abs()
    return dq, tq + u * dq.abs() + 1e-30, dk, tk + u * dk.abs() + 1e-30


@gpu
@pytest.mark.parametrize("by", ["length", "mask", "both"])
@pytest.mark.parametrize("B,Lq,Lk,H,G,D", [
    (4, 5, 256, 4, 2, 64),               # a few rows: four key groups
    (4, 40, 256, 4, 2, 64),              # two key groups
    (4, 33, 200, 2, 1, 96),
    (2, 9, 1000, 3, 3, 128),
    (3, 70, 700, 2, 2, 8),
    (1, 3, 5000, 4, 2, 64),              # shares of a long axis, most of which see nothing
    (1, 200, 2000, 2, 2, 40),
    (64, 130, 300, 4, 4, 32),            # one key group
    (64, 130, 129, 4, 4, 128),
])
def test_cross_attention_score_gradients_over_few_keys(dev, B, Lq, Lk, H, G, D, by):
    """Values that share an offset of a hundred: the scores' gradients are differences of the offset's size, and the rounding of
    a stored bf16 output would be as large as they are.  Two to 32 keys are seen, by a length, by a mask, by both."""
    from styler_amd import ops
    q, k, v, do = attention_case(dev, B, Lq, Lk, H, G, D, torch.bfloat16, seed=41)
    v = (v + 100.0).to(torch.bfloat16)
    g = torch.Generator().manual_seed(B + Lk)
    count = [(2, 3, 32, 17, 31, 5)[b % 6] for b in range(B)]
    if B == 64:                                               # (the oracle's time: three items see keys)
        count = [c if b in (0, 20, 63) else 0 for b, c in enumerate(count)]
    masked = torch.ones(B, Lk, dtype=torch.bool)
    for b, n in enumerate(count):
        masked[b, torch.randperm(Lk, generator=g)[:n]] = False
    lens = {"length": torch.tensor(count), "mask": None, "both": torch.full((B,), Lk // 2)}[by]
    mask = None if by == "length" else masked
    seen = torch.arange(Lk)[None] < (torch.full((B,), Lk) if lens is None else lens)[:, None]
    seen = seen if mask is None else seen & ~mask
    on = lambda t: None if t is None else t.to(dev)
    lse = torch.empty(B, H, Lq, device=dev)
    out = ops.cross_attention(q, k, v, on(lens), mask=on(mask), lse=lse)
    dq, dk, _ = ops.cross_attention_bwd(q, k, v, out, do, lse, on(lens), mask=on(mask))
    rq, tq, rk, tk = score_gradient_oracle(q, k, v, do, seen, D ** -0.5)
    within(dq.cpu(), rq, tq, "dq")
    within(dk.cpu(), rk, tk, "dk")


# ------------------------------------------------------------------------------------------------------------ gradients that are not there
@pytest.mark.parametrize("leaf", ["pos", "freqs"])
def test_rotary_refuses_the_gradient_of_positions_and_angles(leaf):
    """Fractional positions may come from predicted durations, angles may be a parameter: their gradients are not formed, and a
    backward pass that would drop them says so."""
    import styler_amd.torch_ops  # noqa: F401
    from styler_amd import ops
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 5, 3, 64, requires_grad=True)
        pos, freqs = torch.empty(5, requires_grad=leaf == "pos"), torch.empty(32, dtype=torch.float64, requires_grad=leaf == "freqs")
        with pytest.raises(ops.StylerHipError, match="no gradient"):
            torch.ops.styler.rotary(x, freqs, pos).sum().backward()
        torch.ops.styler.rotary(x, freqs.detach(), pos.detach()).sum().backward()
        assert x.grad.shape == x.shape
        torch.ops.styler.rotary(x, freqs.detach()).sum().backward()          # (without positions)


@gpu
@pytest.mark.parametrize("Lq,Lk", [(3, 40), (300, 2000)])
def test_cross_attention_fp32_to_the_ends_of_the_range(dev, Lq, Lk):
    """fp32 values up to the largest, in both arithmetics (few rows; many): what rounds to infinity in bf16 is finite here.  A key of
    infinite distance (a score of -inf) is a key that is not seen."""
    from styler_amd import ops
    B, H, G, D = 2, 8, 4, 64
    q, k, v, do = attention_case(dev, B, Lq, Lk, H, G, D, torch.float32, seed=51)
    top = torch.finfo(torch.float32).max
    v2 = v.clone()
    v2[:, 7, :, 3], v2[:, 11, :, 5] = top, -top
    got, ref = ops.cross_attention(q, k, v2), ops.cross_attention(q, k, v)
    s = torch.matmul(q.double().transpose(1, 2), k.double().repeat_interleave(H // G, 2).permute(0, 2, 3, 1).contiguous()) / 8
    p = torch.softmax(s, -1)
    for d in (3, 5):
        w = torch.matmul(p, v2[..., d].double().repeat_interleave(H // G, 2).transpose(1, 2)[..., None].contiguous())[..., 0].transpose(1, 2)
        a = torch.matmul(p, v2[..., d].double().abs().repeat_interleave(H // G, 2).transpose(1, 2)[..., None].contiguous())[..., 0].transpose(1, 2)
        # P's relative error: the scores' sums, the exponent's argument, the sum (as in attention_oracle, with its largest terms)
        e = (D + 4) * U32 * 64 + 8 * U32 * float(s.abs().max()) + (Lk + 64) * U32
        within(got[..., d].cpu(), w.cpu(), (2 * e * a).cpu(), d)
    rest = [d for d in range(D) if d not in (3, 5)]
    assert torch.equal(got[..., rest], ref[..., rest])
    k3, mask = k.clone(), torch.zeros(B, Lk, dtype=torch.bool, device=dev)
    q3 = q.clone()
    q3[..., 0] = q3[..., 0].abs() + 1e-3
    k3[:, 5, :, 0] = -math.inf
    mask[:, 5] = True
    a, b = ops.cross_attention(q3, k3, v), ops.cross_attention(q3, k, v, mask=mask)
    assert bool(a.isfinite().all())
    assert float((a - b).abs().max()) <= 2 * ((D + 4) * U32 * 64 + 8 * U32 * float(s.abs().max() + 8) + (Lk + 64) * U32) * float(v.abs().max())


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Lq,Lk", [(1, 700), (45, 200), (300, 2000)])
def test_cross_attention_shows_a_seen_nan(dev, Lq, Lk, dtype):
    """A NaN among what is seen shows in everything that depends on it and in nothing else."""
    from styler_amd import ops
    B, H, G, D = 3, 4, 2, 64
    q, k, v, do = attention_case(dev, B, Lq, Lk, H, G, D, dtype, seed=52)

    def both(q, k, v, do):
        lse = torch.empty(B, H, Lq, device=dev)
        out = ops.cross_attention(q, k, v, lse=lse)
        return (out, *ops.cross_attention_bwd(q, k, v, out, do, lse))

    ref = both(q, k, v, do)
    for i in range(4):
        t = [q.clone(), k.clone(), v.clone(), do.clone()]
        t[i][1, 0 if i in (0, 3) else Lk - 3, 1, 17] = math.nan              # query head 1 and key head 1: the key heads 0 and 1
        got = both(*t)
        g = 0 if i in (0, 3) else 1
        heads = [1] if i in (0, 3) else [2, 3]
        nan = [a.isnan() for a in got]
        if i == 0:
            assert bool(nan[0][1, 0, 1].all()) and not nan[0][1, 1:].any()
        elif i == 1:
            assert bool(nan[0][1][:, heads].all())
        elif i == 2:
            assert bool(nan[0][1][:, heads][..., 17].all()) and not nan[0][1][:, heads][..., :17].any()
        if i == 3:
            assert not nan[0].any()
        assert bool(nan[1][1, 0, heads].any()) and bool(nan[2][1, :, g].any())
        for a, b, own in zip(got, ref, (heads, heads, [g], [g])):
            other = [h for h in range(a.shape[2]) if h not in own]
            assert torch.equal(a[[0, 2]], b[[0, 2]]) and torch.equal(a[1][:, other], b[1][:, other])


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_shows_values_that_are_not_finite(dev, interleaved):
    from styler_amd import ops
    f = ops.rotary_freqs(48, dev)
    for dtype in DT:
        x = torch.randn(2, 9, 3, 64, generator=torch.Generator().manual_seed(3)).to(dtype).to(dev)
        ref = ops.rotary(x, f, interleaved=interleaved)
        x2 = x.clone()
        x2[1, 4, 2, 6], x2[0, 3, 0, 60] = math.nan, math.inf                  # one of a pair; a feature that passes through
        got = ops.rotary(x2, f, interleaved=interleaved)
        pair = (6, 7) if interleaved else (6, 30)
        assert all(bool(got[1, 4, 2, d].isnan()) for d in pair) and float(got[0, 3, 0, 60]) == math.inf
        for d in pair:
            got[1, 4, 2, d] = ref[1, 4, 2, d]
        got[0, 3, 0, 60] = ref[0, 3, 0, 60]
        assert torch.equal(got, ref)
        pos = torch.arange(9, device=dev).float()
        pos[5] = math.nan
        got = ops.rotary(x, f, pos, interleaved=interleaved)
        assert bool(got[:, 5, :, :48].isnan().all()) and bool(got[:, :5].isfinite().all()) and bool(got[:, 6:].isfinite().all())


def test_block_operators_refuse_overlapping_outputs():
    """Outputs that share some elements with an input, or rows with themselves; alternating slices of one buffer share none."""
    from styler_amd import ops
    f = ops.rotary_freqs(32, "cpu")
    w = torch.ones(32)
    buf = torch.zeros(2, 6, 12, 32)
    q, k, v, o = buf[:, :, :4], buf[:, :, 4:6], buf[:, :, 6:8], buf[:, :, 8:]
    for out in (buf[:, :, 3:7], buf[:, :, 5:9], buf[:, :, 7:11]):           # one head of q; of k and v; of v
        with pytest.raises(ops.StylerHipError, match="shares memory"):
            ops.cross_attention(q, k, v, out=out)
    with pytest.raises(ops.StylerHipError, match="shares memory"):
        ops.rotary(q, f, out=buf[:, :, 1:5])
    rows = torch.zeros(2, 9, 32)
    with pytest.raises(ops.StylerHipError, match="shares memory"):
        ops.groupnorm_act(rows[:, 1:], w, w, 4, out=rows[:, :-1])           # the next row's place
    flat = torch.zeros(1000)
    twice = flat.as_strided((2, 4, 32), (130, 16, 1))                       # every row over half of the next
    for bad in (lambda: ops.rotary(q, f, out=flat.as_strided(q.shape, (96, 16, 48, 1))),
                lambda: ops.cross_attention(q, k, v, out=flat.as_strided(q.shape, (96, 16, 32, 1)))):
        with pytest.raises(ops.StylerHipError, match="distinct rows"):
            bad()
    assert not ops._rows_ok(twice.shape, twice.stride())
    assert ops._rows_ok((2, 4, 32), (32, 64, 1))                            # rows of the items in turn
    assert ops._rows_ok((3, 2, 32), (64, 96, 1)) and not ops._rows_ok((4, 3, 32), (64, 96, 1))       # (0 64 128 96 160 224; 192 twice)
    # what shares nothing, and what works in place, goes on to the next check
    for fine in (lambda: ops.cross_attention(q, k, v, out=o), lambda: ops.rotary(q, f, out=o), lambda: ops.rotary(q, f, out=q),
                 lambda: ops.groupnorm_act(rows[:, 1:], w, w, 4, out=rows[:, 1:]),
                 lambda: ops.groupnorm_act(torch.zeros(1, 6, 64)[..., :32], w, w, 4, out=torch.zeros(1, 6, 64)[..., 32:])):
        with pytest.raises(ops.StylerHipError, match="no CPU form"):
            fine()
    one = torch.zeros(1, 4, 2, 32)                                          # a batch of one: its item stride is not used
    with pytest.raises(ops.StylerHipError, match="no CPU form"):
        ops.rotary(one, f, out=one.as_strided(one.shape, (7, 64, 32, 1)))


def test_block_operators_refuse_sizes_and_numbers_past_32_bits():
    """What the packed arguments cannot hold is refused like any other argument (no memory behind these: one element, expanded)."""
    from styler_amd import ops
    z, f, w = torch.zeros(1), ops.rotary_freqs(2, "cpu"), torch.ones(1)
    wide = lambda *s: z.expand(*s)
    n = (1 << 31) + 5
    x = torch.zeros(2, 3, 1, 8)
    for bad, text in [
        (lambda: ops.cross_attention(wide(1, n, 1, 8), wide(1, 4, 1, 8), wide(1, 4, 1, 8)), "sizes up to"),
        (lambda: ops.cross_attention(wide(1, 4, 1, 8), wide(1, n, 1, 8), wide(1, n, 1, 8)), "sizes up to"),
        (lambda: ops.cross_attention(wide(n, 4, 1, 8), wide(n, 4, 1, 8), wide(n, 4, 1, 8)), "sizes up to"),
        (lambda: ops.rotary(wide(1, n, 1, 2), f), "sizes up to"),
        (lambda: ops.rotary(wide(1, 1, n, 2), f), "sizes up to"),
        (lambda: ops.groupnorm_act(wide(1, n, 1), w, w, 1), "sizes up to"),
        (lambda: ops.groupnorm_act(wide(n, 1, 1), w, w, 1), "sizes up to"),
        (lambda: ops.groupnorm_act_bwd(wide(1, n, 1), wide(1, n, 1), w, w, torch.zeros(1, 1, 2), 1), "sizes up to"),
        (lambda: ops.rotary(x, f, gain=1e39), "gain"),
        (lambda: ops.rotary(x, f, gain=-math.inf), "gain"),
        (lambda: ops.groupnorm_act(torch.zeros(2, 3, 8), torch.ones(8), torch.ones(8), 2, eps=1e39), "eps"),
        (lambda: ops.cross_attention(x, x, x, scale=1e39), "scale"),
    ]:
        with pytest.raises(ops.StylerHipError, match=text):
            bad()


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Lq,Lk,H,G,D", [(40, 1, 900, 8, 2, 64), (16, 140, 520, 4, 4, 64), (24, 70, 300, 2, 1, 32)])
def test_cross_attention_of_an_item_alone_and_in_a_batch(dev, B, Lq, Lk, H, G, D, dtype):
    """The batch around an item decides how its keys are shared out (and, in fp32, by which instructions they are multiplied): its
    results may change in the roundings, not by more."""
    from styler_amd import ops
    q, k, v, do = attention_case(dev, B, Lq, Lk, H, G, D, dtype, seed=61)
    lens = torch.randint(1, Lk + 1, (B,), generator=torch.Generator().manual_seed(4))

    def both(s):
        n = lens[s].to(dev)
        lse = torch.empty(len(n), H, Lq, device=dev)
        out = ops.cross_attention(q[s], k[s], v[s], n, lse=lse)
        return (out, *ops.cross_attention_bwd(q[s], k[s], v[s], out, do[s], lse, n))

    whole = both(slice(0, B))
    for b in (0, B // 2, B - 1):
        s = slice(b, b + 1)
        ref, tol = attention_oracle(q[s], k[s], v[s], do[s], lens[s], None, None, D ** -0.5, dtype)
        for n, a, w, r, t in zip(("out", "dq", "dk", "dv"), both(s), whole, (ref[0], ref[2], ref[3], ref[4]), tol):
            within(a.cpu(), r, t + 1e-30, n)
            within(w[s].cpu(), r, t + 1e-30, n)


@gpu
@pytest.mark.parametrize("B,Lq,Lk,H,G,D", [(32, 1, 1500, 16, 4, 64), (2, 1, 8197, 8, 8, 128), (3, 5, 129, 6, 2, 96), (5, 2, 31, 8, 1, 40),
                                           (40, 1, 700, 4, 4, 32), (2, 8, 5000, 4, 1, 80)])
def test_cross_attention_tokens_are_rounded_once(dev, B, Lq, Lk, H, G, D):
    """Up to 32 rows a key head, bf16: the probabilities keep 16 bits (two bf16 operands, 2^-17 left) between the two products, so
    that the result is off by its own rounding and by 32-bit arithmetic."""
    from styler_amd import ops
    q, k, v, _ = attention_case(dev, B, Lq, Lk, H, G, D, torch.bfloat16, seed=71)
    lens = torch.randint(0, Lk + 1, (B,), generator=torch.Generator().manual_seed(Lk))
    lens[0] = Lk
    out = ops.cross_attention(q, k, v, lens.to(dev)).cpu()
    q, k, v = (t.cpu().double() for t in (q, k, v))
    for b in range(B):
        n = int(lens[b])
        for h in range(H):
            if n == 0:
                assert not out[b, :, h].any()
                continue
            Q, K, V = q[b, :, h], k[b, :n, h // (H // G)], v[b, :n, h // (H // G)]
            S = Q @ K.T * D ** -0.5
            P = torch.softmax(S, -1)
            lse = torch.logsumexp(S, 1)
            e = (D + 4) * U32 * (Q.abs() @ K.abs().T * D ** -0.5).max() + 4 * U32 * (S.abs().max() + lse.abs().max()) + (n + 64) * U32
            within(out[b, :, h], P @ V, half_step(torch.bfloat16) * (P @ V).abs() + (2.0 ** -17 + 2 * e) * (P @ V.abs()), (b, h))


@gpu
@pytest.mark.parametrize("dtype", DT)
def test_block_operators_with_gradients_in_a_graph(dev, dtype):
    """Norm, rotary positions, attention and the gradients of all of them through the dispatcher, captured once and replayed with new
    inputs and lengths; every replay equals the eager pass over leaves of its own."""
    import styler_amd.torch_ops  # noqa: F401
    from styler_amd import ops
    B, Lq, Lk, H, G, D = 3, 70, 41, 4, 2, 64
    gen = torch.Generator().manual_seed(77)
    r = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(dev)
    shapes = [(B, Lq, H * D), (B, Lk, 2, G, D), (B, Lq, H, D)]
    x, enc, dout = bufs = [r(*s) for s in shapes]
    gamma, beta = (torch.randn(H * D, generator=gen).to(dev) for _ in range(2))
    q_lens, lens = torch.tensor([70, 1, 33], device=dev), torch.tensor([41, 20, 7], device=dev)
    freqs = ops.rotary_freqs(D, dev)

    def step(x, enc, gamma, beta, dout):
        x, enc, gamma, beta = leaves = [t.detach().requires_grad_() for t in (x, enc, gamma, beta)]
        y, _ = torch.ops.styler.groupnorm_act(x, gamma, beta, 16, 6, 1e-5, q_lens)
        q, k = torch.ops.styler.rotary(y.view(B, Lq, H, D), freqs), torch.ops.styler.rotary(enc[:, :, 0], freqs)
        out = torch.ops.styler.cross_attention(q, k, enc[:, :, 1], lens, q_lens)[0]
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, enc, gamma, beta, dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, enc, gamma, beta, dout)
    for turn in range(4):
        for t in bufs:
            t.copy_(torch.randn(t.shape, generator=gen).to(t.dtype))
        q_lens.copy_(torch.randint(0, Lq + 1, (B,), generator=gen))
        lens.copy_(torch.randint(0, Lk + 1, (B,), generator=gen))
        want = [t.clone() for t in step(x.clone(), enc.clone(), gamma.clone(), beta.clone(), dout)]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), turn


# ------------------------------------------------------------------------------------------------------------ the C entries
def test_block_entry_points_refuse_before_any_launch():
    """Every refusal of the C entry points comes before a HIP call: these run without a GPU.  (Addresses are never followed.)"""
    from styler_amd._lib import GN, ROTARY, XATTN, lib
    EINVAL, EALIGN = -1, -2
    P = 4096

    def xattn(bwd=False, ws=P, nbytes=1 << 40, **kw):
        f = dict(q=P, k=P, v=P, out=P, dout=P, dq=P, dk=P, dv=P, lse=P, len=0, q_len=0, mask=0, qb=512, ql=256, qh=64, kb=512, kl=128, kh=64,
                 vb=512, vl=128, vh=64, ob=512, ol=256, oh=64, gb=512, gl=256, gh=64, maskb=0, B=2, Lq=2, Lk=4, H=4, G=2, D=64, bf16=1,
                 scale=0.125)
        f.update(kw)
        fn = lib.styler_cross_attention_bwd if bwd else lib.styler_cross_attention
        return fn(XATTN.pack(*f.values()), ws, nbytes, None)

    for kw in (dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(B=0), dict(Lq=0), dict(Lk=-1), dict(H=3), dict(G=0), dict(D=60), dict(D=136),
               dict(scale=0.0), dict(scale=math.nan), dict(scale=-1.0), dict(ql=1 << 23), dict(kl=1 << 23), dict(B=1 << 23)):
        assert xattn(**kw) == EINVAL, kw
    for kw in (dict(q=P + 2), dict(ql=250), dict(kh=4), dict(vb=-64), dict(out=P + 8)):
        assert xattn(**kw) == EALIGN, kw
    for kw in (dict(dout=0), dict(dq=0), dict(dk=0), dict(dv=0), dict(lse=0), dict(ws=0), dict(nbytes=8), dict(ws=P + 4)):
        assert xattn(bwd=True, **kw) == EINVAL, kw
    assert xattn(bwd=True, gl=12) == EALIGN
    assert xattn(Lk=100000, kb=0, vb=0, ws=0) == EINVAL                      # shares of a long axis need their workspace
    assert lib.styler_cross_attention(None, None, 0, None) == EINVAL

    def rotary(**kw):
        f = dict(x=P, y=P, freqs=P, pos=0, xb=64, xl=64, xh=64, yb=64, yl=64, yh=64, posb=0, B=1, L=1, H=1, D=64, rot=64, pos_kind=0,
                 interleaved=0, inverse=0, bf16=1, gain=1.0)
        f.update(kw)
        return lib.styler_rotary(ROTARY.pack(*f.values()), None)

    for kw in (dict(x=0), dict(y=0), dict(freqs=0), dict(B=0), dict(H=0), dict(rot=0), dict(rot=3), dict(rot=66), dict(D=16384, rot=2),
               dict(pos_kind=3), dict(pos_kind=1), dict(B=1 << 20, L=1 << 12)):
        assert rotary(**kw) == EINVAL, kw
    assert rotary(x=P + 1) == EALIGN
    assert lib.styler_rotary(None, None) == EINVAL

    def gn(bwd=False, ws=P, nbytes=1 << 40, **kw):
        f = dict(x=P, dy=P, out=P, gamma=P, beta=P, stats=P, dgamma=P, dbeta=P, len=0, xb=640, xl=64, db=640, dl=64, ob=640, ol=64, B=2, L=10,
                 C=64, G=4, act=6, bf16=0, eps=1e-5)
        f.update(kw)
        return (lib.styler_groupnorm_act_bwd if bwd else lib.styler_groupnorm_act)(GN.pack(*f.values()), ws, nbytes, None)

    for kw in (dict(x=0), dict(out=0), dict(gamma=0), dict(beta=0), dict(B=0), dict(L=0), dict(C=0), dict(G=0), dict(G=3), dict(act=2),
               dict(act=99), dict(eps=-1.0), dict(eps=math.nan), dict(L=1 << 30 | 1)):
        assert gn(**kw) == EINVAL, kw
    for kw in (dict(dy=0), dict(stats=0), dict(dgamma=0), dict(dbeta=0), dict(ws=0), dict(nbytes=16)):
        assert gn(bwd=True, **kw) == EINVAL, kw
    assert gn(x=P + 2) == EALIGN
    assert gn(L=1 << 20, xb=0, ob=0, ws=0) == EINVAL
    assert lib.styler_groupnorm_act(None, None, 0, None) == EINVAL
