"""The mixture-of-experts operators against their plain 64-bit forms."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from moe_ref import ACT, DEV, Q4_0, Q4_K, Q6_K, Q8_0, Q8_K, TYPES, UNIT, Experts, product, rounding, route  # noqa: E402


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


# ---------------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("rows,n,act", [(1, 4096, Q8_0), (1, 32, Q8_0), (3, 4, None), (5, 256, Q8_K), (37, 1056, Q8_0), (2, 4352, Q8_K),
                                        (130, 2048, Q8_0), (1, 14336, Q8_K), (300, 512, Q8_K), (1025, 96, Q8_0), (33, 20, None), (3, 33024, Q8_0)])
@pytest.mark.parametrize("with_w", [True, False])
def test_norm(rows, n, act, with_w):
    from ameva_compute_amd import ops
    g = gen(rows + n)
    x, r = torch.randn(rows, n, generator=g, device=DEV), 3 * torch.randn(rows, n, generator=g, device=DEV)
    w = torch.randn(n, generator=g, device=DEV) if with_w else None
    if rows > 2:
        x[1], r[1] = 0.0, 0.0  # a row of nothing
    s, o, a = ops.add_rms_norm(x, r, 1e-5, w, act_type=act)
    assert torch.equal(s, x + r)
    z = s.double()
    ref = z / (z.square().mean(-1, keepdim=True) + 1e-5).sqrt() * (1 if w is None else w.double())
    # squares, mean, eps, root, quotient, and the two products, each half a step: the squares' and mean's halve in the root
    assert bool(((o - ref).abs() <= 5.5 * 2.0 ** -24 * ref.abs()).all())
    if act is not None:
        assert torch.equal(a, ops.quantize_act(o, act)[0])
        v = ops.act_values(a, act, rows, n, torch.float32)
        assert torch.equal(ops.act_values(a, act, rows, n), v.half())
        big = o.view(rows, -1, 32 if act == Q8_0 else 256).abs().amax(-1, keepdim=True).double() / 127
        # half a step of the integers, and the scale's own rounding (f16 for Q8_0) times up to 127 of them
        lim = (0.5 + 127 * 2.0 ** (-11 if act == Q8_0 else -23)) * big * (1 + 2.0 ** -20) + 127 * 2.0 ** -25
        assert bool(((v - o).double().abs().view(rows, big.shape[1], -1) <= lim).all())
    y, none, b = ops.add_rms_norm(x, r, 1e-5, w, act_type=act, out=r, normed=False)  # in place
    assert y is r and none is None and torch.equal(r, s) and (act is None or torch.equal(a, b))


@pytest.mark.parametrize("act", [Q8_0, Q8_K])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_norm_of_no_number_stays_in_its_row(act, bad):
    from ameva_compute_amd import ops
    x, r = torch.randn(4, 512, generator=gen(1), device=DEV), torch.zeros(4, 512, device=DEV)
    good = ops.add_rms_norm(x, r, 1e-5, act_type=act)
    x[2, 100] = bad
    s, o, a = ops.add_rms_norm(x, r, 1e-5, act_type=act)
    v, w = (ops.act_values(q, act, 4, 512, torch.float32) for q in (a, good[2]))
    keep = torch.tensor([0, 1, 3], device=DEV)
    assert torch.equal(o[keep], good[1][keep]) and torch.equal(v[keep], w[keep])
    assert bool(o[2, 100].isnan()) and bool(v[2, 96:128].isnan().all())
    if math.isnan(bad):
        assert bool(o[2].isnan().all()) and bool(v[2].isnan().all())


# ---------------------------------------------------------------------------------------------------- routing
def check_route(logits, n_used, **more):
    from ameva_compute_amd import ops
    ids, w = ops.moe_route(logits, n_used, **more)
    rids, rw = route(logits, n_used, **more)
    assert torch.equal(ids.cpu(), rids)
    w, nan = w.double().cpu(), rw.isnan()
    assert torch.equal(w.isnan(), nan)
    # one rounding to 32 bits of what 64 bits hold
    assert bool(((w - rw).abs()[~nan] <= 2.0 ** -24 * 1.001 * rw.abs()[~nan] + 1e-40).all())
    return ids, w


@pytest.mark.parametrize("n,used", [(1, 1), (8, 2), (60, 4), (64, 64), (65, 3), (128, 8), (160, 6), (256, 8), (500, 10), (1024, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(n, used, score):
    g = gen(n)
    for t in (1, 7, 70):
        z = 2 * torch.randn(t, n, generator=g, device=DEV)
        bias = 0.2 * torch.randn(n, generator=g, device=DEV)
        check_route(z, used, score=score)
        check_route(z, used, score=score, renorm=False, scale=2.5)
        check_route(z, used, score=score, bias=bias)
        check_route(z.half().float() * 0 + torch.randint(-2, 3, (t, n), generator=g, device=DEV), used, score=score)  # many equal ones
        check_route(torch.cat([z, z], 1)[:, :n] if t == 1 else torch.cat([z, z], 1)[:, n // 2:n // 2 + n], used, score=score)  # other strides


@pytest.mark.parametrize("n,groups,top,used", [(16, 4, 1, 2), (64, 8, 3, 6), (256, 8, 4, 8), (160, 8, 3, 6), (60, 6, 2, 5), (320, 64, 40, 9)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups(n, groups, top, used, best, score):
    g = gen(n + top)
    z = 2 * torch.randn(50, n, generator=g, device=DEV)
    for bias in (None, torch.randn(n, generator=g, device=DEV)):
        for x in (z, z.round()):
            check_route(x, used, score=score, bias=bias, n_group=groups, top_group=top, group_best=best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [(1, 1), (4, 2)])
def test_route_masks(score, groups):
    """Experts that are masked, rows that leave nothing, values of the type's ends, and no numbers."""
    n, inf, nan = 32, math.inf, math.nan
    z = torch.randn(14, n, generator=gen(5), device=DEV)
    z[0, 3:] = -inf
    z[1] = -inf
    z[2, ::2] = torch.finfo(torch.float32).min
    z[3] = torch.finfo(torch.float32).min
    z[4, 5] = inf
    z[5, 5], z[5, 9] = inf, inf
    z[6, 7] = nan
    z[7] = nan
    z[8, :20], z[8, 25] = -inf, nan
    z[9] = torch.finfo(torch.float32).max
    z[10] = 0.0
    z[10, 4] = -0.0
    z[11] = -800.0
    z[12] = torch.linspace(-1000, 1000, n, device=DEV)
    z[13, 1:] = -inf
    bias = 0.1 * torch.randn(n, generator=gen(6), device=DEV)
    hidden = bias.clone()
    hidden[4:28] = -inf
    hidden[2] = nan
    kw = dict(score=score, n_group=groups[0], top_group=groups[1])
    for b in (None, bias, hidden):
        for best in (1, 2):
            for used in (1, 6):
                check_route(z, used, bias=b, group_best=best, **kw)
                check_route(z, used, bias=b, group_best=best, renorm=False, **kw)


# ---------------------------------------------------------------------------------------------------- products
def ids_for(g, t, used, n, kind="skewed"):
    if kind == "one":  # every token to the same expert
        return torch.full((t, used), n - 1, dtype=torch.int32, device=DEV)
    z = torch.randn(t, n, generator=g, device=DEV) + 2 * torch.randn(n, generator=g, device=DEV)
    ids = z.topk(used, dim=1)[1].int()
    if kind == "holes":  # tokens of a padded batch, single pairs without an expert, an expert twice, ids out of range
        ids[t - t // 4:] = -1
        ids[0, 0] = n
        ids[t // 2, 0] = -(2 ** 31)
        ids[t // 3] = ids[t // 3, :1]
    return ids.contiguous()


SHAPES = [  # tokens, experts, used, rows, k in blocks, kind
    (1, 4, 2, 32, 1, "skewed"), (1, 8, 8, 96, 5, "skewed"), (1, 3, 1, 256, 3, "holes"), (2, 8, 2, 64, 2, "skewed"), (3, 40, 4, 32, 9, "skewed"),
    (6, 5, 3, 288, 4, "holes"), (17, 3, 1, 64, 7, "one"), (40, 16, 2, 160, 6, "holes"), (65, 2, 2, 32, 33, "skewed"), (200, 3, 2, 96, 5, "holes"),
    (333, 60, 4, 64, 2, "skewed"), (9, 4, 2, 96, 57, "holes"), (130, 2, 1, 352, 17, "one"), (1100, 7, 4, 32, 1, "holes"), (700, 5, 1, 544, 3, "skewed"),
    # more experts a token than a workgroup has waves; a plan of more than 4096 pairs with few of them an expert
    (1, 70, 20, 64, 3, "skewed"), (1, 64, 64, 32, 6, "skewed"), (3, 70, 64, 32, 2, "skewed"), (700, 1024, 8, 32, 1, "holes"),
    # the most of a tile's rows that LDS holds at once
    (13, 4, 2, 96, 14, "holes"),
    # a k that fills the lanes, one to a few rows an expert
    (5, 4, 2, 96, 64, "holes"), (17, 10, 4, 160, 64, "skewed"), (6, 12, 3, 32, 64, "skewed"), (7, 3, 1, 288, 64, "one")]


def make(t, shape, seed=0):
    tok, n, used, rows, kb, kind = shape
    k = kb * (32 if t in (Q4_0, Q8_0) else 256)
    if kb == 14:
        k = 3584
    if kb == 64:
        k = 2048
    if kb == 57:  # longer than what LDS holds of a tile's rows: parts of it, the last one not whole
        k = 7264 if t in (Q4_0, Q8_0) else 7424
    g = gen(seed + tok + rows)
    return ids_for(g, tok, used, n, kind), k, g


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("t", TYPES)
def test_gate_up(t, shape):
    from ameva_compute_amd import ops
    tok, n, used, rows, _, _ = shape
    ids, k, g = make(t, shape)
    gate, up = Experts(t, n, rows, k, 1), Experts(t, n, rows, k, 2)
    x = torch.randn(tok, k, generator=g, device=DEV)
    act = ops.quantize_act(x, ACT[t])[0]
    a = ops.act_values(act, ACT[t], tok, k, torch.float32).double().repeat_interleave(used, 0)
    flat = ids.flatten()
    (yg, sg), (yu, su) = product(a, gate, flat), product(a, up, flat)
    ref = yg * torch.sigmoid(yg) * yu
    plan = ops.moe_plan(ids, n)
    out, h = ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=Q8_0, eout=True)
    # the products' errors through the derivatives (that of silu is at most 1.1), and four roundings and the exponential's of the value itself
    lim = rounding(gate) * (1.1 * sg * yu.abs() + (yg * torch.sigmoid(yg)).abs() * su + 1.1 * sg * su * rounding(gate)) + 8 * 2.0 ** -24 * ref.abs() + 1e-30
    assert bool(((h.double() - ref).abs() <= lim).all())
    none = (flat < 0) | (flat >= n)
    assert bool((h[none] == 0).all())
    assert torch.equal(out, ops.quantize_act(h, Q8_0)[0])
    assert torch.equal(ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=Q8_0), out)
    assert torch.equal(ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=None), h)
    arm = ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=Q8_0, rule=ops.Q8_ARM)
    assert torch.equal(arm, ops.quantize_act(h, Q8_0, ops.Q8_ARM)[0])
    if rows % 256 == 0:
        assert torch.equal(ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=Q8_K), ops.quantize_act(h, Q8_K)[0])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("t", TYPES)
def test_down(t, shape):
    from ameva_compute_amd import ops
    tok, n, used, rows, _, _ = shape
    ids, k, g = make(t, shape, 7)
    down = Experts(t, n, rows, k, 3)
    act = ops.quantize_act(torch.randn(tok * used, k, generator=g, device=DEV), ACT[t])[0]
    a = ops.act_values(act, ACT[t], tok * used, k, torch.float32).double()
    weights, add = torch.rand(tok, used, generator=g, device=DEV) * 2 - 0.5, torch.randn(tok, rows, generator=g, device=DEV)
    y, size = (v.view(tok, used, rows) for v in product(a, down, ids.flatten()))
    w = weights.double()[..., None]
    plan = ops.moe_plan(ids, n)
    for extra in (None, add):
        out = ops.moe_down(down.gpu, act, plan, weights, add=extra)
        base = 0 if extra is None else extra.double()
        ref, parts = base + (w * y).sum(1), (w * y).abs().sum(1) + (0 if extra is None else base.abs())
        lim = rounding(down) * (w.abs() * size).sum(1) + used * 2.0 ** -24 * parts * 1.01 + 1e-30
        assert bool(((out.double() - ref).abs() <= lim).all())
    gone = ((ids < 0) | (ids >= n)).all(1)
    assert torch.equal(out[gone], add[gone])
    again = add.clone()
    assert ops.moe_down(down.gpu, act, plan, weights, add=again, out=again) is again and torch.equal(again, out)


@pytest.mark.parametrize("t", TYPES)
def test_tokens_without_a_plan(t):
    """Several tokens through the products that need no plan (the C entries' plan NULL), as bounded as with one."""
    from ameva_compute_amd import ops
    shape = (7, 9, 3, 64, 5, "holes")
    tok, n, used, rows, _, _ = shape
    ids, k, g = make(t, shape, 3)
    gate, up, down = Experts(t, n, rows, k, 1), Experts(t, n, rows, k, 2), Experts(t, n, rows, k, 3)
    act = ops.quantize_act(torch.randn(tok, k, generator=g, device=DEV), ACT[t])[0]
    a = ops.act_values(act, ACT[t], tok, k, torch.float32).double().repeat_interleave(used, 0)
    flat, plan = ids.flatten(), ops.MoePlan(ids, n, None)
    (yg, sg), (yu, su) = product(a, gate, flat), product(a, up, flat)
    ref = yg * torch.sigmoid(yg) * yu
    h = ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=None)
    # as in test_gate_up and test_down
    lim = rounding(gate) * (1.1 * sg * yu.abs() + (yg * torch.sigmoid(yg)).abs() * su + 1.1 * sg * su * rounding(gate)) + 8 * 2.0 ** -24 * ref.abs() + 1e-30
    assert bool(((h.double() - ref).abs() <= lim).all())
    hact = ops.quantize_act(torch.randn(tok * used, k, generator=g, device=DEV), ACT[t])[0]
    weights, add = torch.rand(tok, used, generator=g, device=DEV) * 2 - 0.5, torch.randn(tok, rows, generator=g, device=DEV)
    y, size = (v.view(tok, used, rows) for v in product(ops.act_values(hact, ACT[t], tok * used, k, torch.float32).double(), down, flat))
    w = weights.double()[..., None]
    out = ops.moe_down(down.gpu, hact, plan, weights, add=add)
    ref, parts = add.double() + (w * y).sum(1), (w * y).abs().sum(1) + add.double().abs()
    assert bool(((out.double() - ref).abs() <= rounding(down) * (w.abs() * size).sum(1) + used * 2.0 ** -24 * parts * 1.01 + 1e-30).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tok,k", [(1, 512), (9, 512), (150, 512), (1, 2048), (5, 2048)])
def test_what_no_token_reads_does_not_matter(t, tok, k):
    """Experts without tokens hold no numbers at all; rows and weights of pairs without an expert neither; a token with an infinite or
    absent number keeps it to itself."""
    from ameva_compute_amd import ops
    n, used, rows = 6, 2, 64
    g = gen(tok)
    ids = torch.stack([torch.randint(1, 3, (tok,), generator=g, device=DEV), torch.randint(3, 5, (tok,), generator=g, device=DEV)], 1).int()
    ids[tok // 2, 1] = -1
    gate, up, down = (Experts(t, n, rows, k, s) for s in (1, 2, 3))
    act = ops.quantize_act(torch.randn(tok, k, generator=g, device=DEV), ACT[t])[0]
    x2 = torch.randn(tok * used, k, generator=g, device=DEV)
    hact, weights = ops.quantize_act(x2, ACT[t])[0], torch.rand(tok, used, generator=g, device=DEV)
    plan = ops.moe_plan(ids, n)
    h, y = ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=None), ops.moe_down(down.gpu, hact, plan, weights)
    for e in (gate, up, down):
        e.gpu.data[0], e.gpu.data[5] = 255, 255
    x2[tok // 2 * used + 1] = math.nan
    hact2, _, _ = None, None, None
    _, _, hact2 = ops.add_rms_norm(x2, torch.zeros_like(x2), 0.0, act_type=ACT[t])
    h2 = ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=None)
    assert torch.equal(h, h2)
    w2 = weights.clone()
    w2[tok // 2, 1] = math.nan
    assert torch.equal(ops.moe_down(down.gpu, hact, plan, w2), y)
    y2 = ops.moe_down(down.gpu, hact2, plan, w2)
    assert bool(y2.isfinite().all())
    # a row that is no number, seen by its own token alone
    xn = torch.randn(tok, k, generator=gen(99), device=DEV)
    zero = torch.zeros_like(xn)
    clean = ops.add_rms_norm(xn, zero, 1e-5, act_type=ACT[t])[2]
    xn[0, 3] = math.nan
    dirty = ops.add_rms_norm(xn, zero, 1e-5, act_type=ACT[t])[2]
    a, b = (ops.moe_gate_up(gate.gpu, up.gpu, v, plan, act_type=None).view(tok, used, rows) for v in (clean, dirty))
    assert torch.equal(a[1:], b[1:]) and bool(b[0, 0].isnan().all())
    v = ops.act_values(ops.moe_gate_up(gate.gpu, up.gpu, dirty, plan, act_type=Q8_0), Q8_0, tok * used, rows).view(tok, used, rows)
    assert bool(v[0, 0].isnan().all()) and bool(v[1:].isfinite().all())
    z = ops.moe_down(down.gpu, hact, plan, torch.where(torch.arange(tok, device=DEV)[:, None] == 0, math.inf, weights))
    assert torch.equal(z[1:], y[1:]) and not bool(z[0].isfinite().any())


def test_no_tokens():
    from ameva_compute_amd import ops
    e = Experts(Q4_0, 2, 32, 32, 1)
    empty = torch.empty(0, dtype=torch.uint8, device=DEV)
    s, o, a = ops.add_rms_norm(torch.empty(0, 64, device=DEV), torch.empty(0, 64, device=DEV), 1e-5, act_type=Q8_0)
    assert s.shape == o.shape == (0, 64) and a.numel() == 0
    ids, w = ops.moe_route(torch.empty(0, 2, device=DEV), 1)
    plan = ops.moe_plan(ids, 2)
    assert ops.moe_gate_up(e.gpu, e.gpu, empty, plan).numel() == 0
    assert ops.moe_down(e.gpu, empty, plan, w).shape == (0, 32)


# ---------------------------------------------------------------------------------------------------- together
def layer(ops, s, x, r, router, norm_w):
    total, y, act = ops.add_rms_norm(x, r, 1e-5, norm_w, act_type=ACT[s["t"]])
    ids, w = ops.moe_route(ops.mul_mat(router, y), s["used"], score=s["score"], bias=s["bias"])
    plan = ops.moe_plan(ids, s["n"])
    h = ops.moe_gate_up(s["gate"].gpu, s["up"].gpu, act, plan, act_type=ACT[s["t2"]])
    return ops.moe_down(s["down"].gpu, h, plan, w, add=total), ids, w, total, act, h


def setup(t, t2, n=12, used=3, E=512, F=256, score="softmax", seed=4):
    from ameva_compute_amd import ops
    g = gen(seed)
    s = dict(t=t, t2=t2, n=n, used=used, score=score, bias=0.1 * torch.randn(n, generator=g, device=DEV) if score == "sigmoid" else None,
             gate=Experts(t, n, F, E, 1), up=Experts(t, n, F, E, 2), down=Experts(t2, n, E, F, 3))
    router = ops.QWeight.from_ggml(Q8_0, torch.from_numpy(np.ascontiguousarray(
        __import__("oracle").quantize_q8_0(np.random.default_rng(seed).standard_normal((n, E)).astype(np.float32)))).to(DEV), n, E)
    return s, router, 1 + 0.1 * torch.randn(E, generator=g, device=DEV)


@pytest.mark.parametrize("t,t2", [(Q4_0, Q4_0), (Q4_K, Q6_K), (Q8_0, Q4_K), (Q6_K, Q8_0)])
@pytest.mark.parametrize("tok", [1, 5, 90])
def test_layer(t, t2, tok):
    """The operators as a layer uses them, each step against 64 bits from what the step before gave."""
    from ameva_compute_amd import ops
    s, router, nw = setup(t, t2, score="sigmoid" if tok == 5 else "softmax")
    g = gen(tok)
    x, r = torch.randn(tok, 512, generator=g, device=DEV), torch.randn(tok, 512, generator=g, device=DEV)
    y, ids, w, total, act, h = layer(ops, s, x, r, router, nw)
    assert torch.equal(total, x + r)
    o = ops.add_rms_norm(x, r, 1e-5, nw)[1]
    assert torch.equal(act, ops.quantize_act(o, ACT[t])[0])
    rids, rw = route(ops.mul_mat(router, o), s["used"], score=s["score"], bias=s["bias"])
    assert torch.equal(ids.cpu(), rids)
    a = ops.act_values(act, ACT[t], tok, 512, torch.float32).double().repeat_interleave(s["used"], 0)
    (yg, _), (yu, _) = product(a, s["gate"], ids.flatten()), product(a, s["up"], ids.flatten())
    hv = ops.act_values(h, ACT[t2], tok * s["used"], 256, torch.float32).double()
    ref = yg * torch.sigmoid(yg) * yu
    # an 8-bit block is off by half a step of 1 / 127 of its largest (and Q8_0's scale by 2^-11), and no more than 0.02 % from elsewhere
    big = ref.view(hv.shape[0], -1, 32 if ACT[t2] == Q8_0 else 256).abs().amax(-1, keepdim=True)
    assert bool(((hv - ref).abs().view(hv.shape[0], big.shape[1], -1) <= (0.5 / 127 + 2.0 ** -11 + 2e-4) * big + 1e-9).all())
    z, size = (v.view(tok, s["used"], 512) for v in product(hv, s["down"], ids.flatten()))
    wd = w.double()[..., None]
    ref = total.double() + (wd * z).sum(1)
    lim = rounding(s["down"]) * (wd * size).sum(1) + 4 * 2.0 ** -24 * (total.double().abs() + (wd * z).abs().sum(1)) + 1e-30
    assert bool(((y.double() - ref).abs() <= lim).all())


@pytest.mark.parametrize("tok", [1, 2, 4, 70])
def test_captured_layer(tok):
    """A captured layer replayed over other inputs, another stream beside it, against the eager calls."""
    from ameva_compute_amd import ops
    s, router, nw = setup(Q4_0, Q4_K)
    x, r = torch.zeros(tok, 512, device=DEV), torch.zeros(tok, 512, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        layer(ops, s, x, r, router, nw)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(ops, s, x, r, router, nw)[:3]
        graphs.append((graph, out))
    for i in range(4):
        x.copy_(torch.randn(tok, 512, generator=gen(i), device=DEV))
        r.copy_(torch.randn(tok, 512, generator=gen(50 + i), device=DEV))
        for graph, out in graphs:
            graph.replay()
        eager = layer(ops, s, x, r, router, nw)[:3]
        torch.zeros(1000, device=DEV).sum()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
    with torch.cuda.stream(side):
        other = layer(ops, s, x, r, router, nw)[:3]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, eager))


def test_experts_apart_and_back():
    """Experts with gaps between them (a part of a larger allocation) give what tight ones do; unequal ones are refused."""
    from ameva_compute_amd import ops
    e = Experts(Q4_K, 5, 64, 512, 9)
    need = e.gpu.data.shape[1]
    wide = torch.full((5, need + 48), 255, dtype=torch.uint8, device=DEV)
    wide[:, :need] = e.gpu.data
    far = ops.QExperts(Q4_K, 5, 64, 512, wide)
    ids = torch.tensor([[0, 4], [2, 3], [4, 1]], dtype=torch.int32, device=DEV)
    act = ops.quantize_act(torch.randn(3, 512, generator=gen(3), device=DEV), Q8_K)[0]
    for i in (ids, ids[:1].contiguous()):
        plan, m = ops.moe_plan(i, 5), i.shape[0]
        a = ops.quantize_act(torch.randn(m, 512, generator=gen(3), device=DEV), Q8_K)[0]
        assert torch.equal(ops.moe_gate_up(e.gpu, e.gpu, a, plan, act_type=None), ops.moe_gate_up(far, far, a, plan, act_type=None))
    with pytest.raises(ValueError, match="differ"):
        ops.moe_gate_up(e.gpu, far, act, ops.moe_plan(ids, 5))


# ---------------------------------------------------------------------------------------------------- ends of the ranges
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tok", [1, 30, 300])
def test_largest_integers(t, tok):
    """Weights and activations whose integers and scales are all at their ends, one sign or in turn: no sum of a block or super-block
    leaves what the kernels hold it in."""
    import oracle
    from ameva_compute_amd import ops
    n, used, rows, k = 3, 2, 64, 1024
    d = np.float16(0.01).tobytes()
    block = {Q8_0: d + b"\x80" * 32, Q4_0: d + b"\x00" * 16, Q4_K: d + d + b"\xff" * 140, Q6_K: b"\x00" * 192 + b"\x80" * 16 + d}[t]
    raw = np.frombuffer(block * (n * rows * k // UNIT[t]), dtype=np.uint8).copy()
    e = Experts(t, n, rows, k, 1)
    e.gpu = ops.QExperts.from_ggml(t, torch.from_numpy(raw).to(DEV), n, rows, k)
    e.w = torch.from_numpy(oracle.dequantize(t, raw, k).reshape(n, rows, k).astype(np.float64)).to(DEV)
    e.size = e.w.abs() * (1.15 if t == Q4_K else 1)  # (63 * 15 - 63 of the parts 63 * 15 + 63)
    x = torch.ones(tok * used, k, device=DEV)
    x[1::2, 1::2] = -1
    ids = torch.tensor([[0, 2]], dtype=torch.int32, device=DEV).repeat(tok, 1)
    act = ops.quantize_act(x, ACT[t])[0]
    a = ops.act_values(act, ACT[t], tok * used, k, torch.float32).double()
    weights = torch.ones(tok, used, device=DEV)
    y, size = (v.view(tok, used, rows) for v in product(a, e, ids.flatten()))
    plan = ops.moe_plan(ids, n)
    out = ops.moe_down(e.gpu, act, plan, weights)
    assert bool(((out.double() - y.sum(1)).abs() <= rounding(e) * size.sum(1) + used * 2.0 ** -24 * y.abs().sum(1) * 1.01).all())
    one = x[:tok].contiguous()
    act = ops.quantize_act(one, ACT[t])[0]
    yg, sg = product(ops.act_values(act, ACT[t], tok, k, torch.float32).double().repeat_interleave(used, 0), e, ids.flatten())
    h = ops.moe_gate_up(e.gpu, e.gpu, act, plan, act_type=None)
    ref = yg * torch.sigmoid(yg) * yg
    # as in test_gate_up, with one product twice
    lim = rounding(e) * sg * (1.1 * yg.abs() + (yg * torch.sigmoid(yg)).abs() + 1.1 * sg * rounding(e)) + 8 * 2.0 ** -24 * ref.abs() + 1e-30
    assert bool(((h.double() - ref).abs() <= lim).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tok", [1, 20, 400])
def test_experts_beyond_32_bits(t, tok):
    """Experts 2.2 GB apart (all but their own bytes never written) give what they give side by side."""
    from ameva_compute_amd import ops
    n, used, rows, k = 4, 2, 64, 512
    e = Experts(t, n, rows, k, 3)
    need = e.gpu.data.shape[1]
    wide = torch.empty((n, 2200000000 // 16 * 16), dtype=torch.uint8, device=DEV)
    wide[:, :need] = e.gpu.data
    far = ops.QExperts(t, n, rows, k, wide)
    g = gen(tok)
    ids = torch.stack([torch.randint(0, 2, (tok,), generator=g, device=DEV), torch.randint(2, 4, (tok,), generator=g, device=DEV)], 1).int()
    plan, weights = ops.moe_plan(ids, n), torch.rand(tok, used, generator=g, device=DEV)
    act = ops.quantize_act(torch.randn(tok, k, generator=g, device=DEV), ACT[t])[0]
    hact = ops.quantize_act(torch.randn(tok * used, k, generator=g, device=DEV), ACT[t])[0]
    assert torch.equal(ops.moe_gate_up(far, far, act, plan, act_type=None), ops.moe_gate_up(e.gpu, e.gpu, act, plan, act_type=None))
    assert torch.equal(ops.moe_down(far, hact, plan, weights), ops.moe_down(e.gpu, hact, plan, weights))


def test_outputs_beyond_32_bits():
    """2^20 pairs of 1088 columns (4.6 GB of products) and of 4064 k (4.3 GB of activations): the last tokens' results are what the same
    tokens get by themselves, within the roundings."""
    from ameva_compute_amd import ops
    tok, n, used, last = 1 << 17, 8, 8, 16
    g = gen(8)
    ids = torch.randint(0, n, (tok, used), generator=g, device=DEV).int()
    gate, up = Experts(Q8_0, n, 1088, 32, 1), Experts(Q8_0, n, 1088, 32, 2)
    x = torch.randn(tok, 32, generator=g, device=DEV)
    act, tail = ops.quantize_act(x, Q8_0)[0], ops.quantize_act(x[-last:].contiguous(), Q8_0)[0]
    plan, few = ops.moe_plan(ids, n), ops.moe_plan(ids[-last:].contiguous(), n)
    h = ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=None)[-last * used:].double()
    ref = ops.moe_gate_up(gate.gpu, up.gpu, tail, few, act_type=None).double()
    a, flat = ops.act_values(tail, Q8_0, last, 32, torch.float32).double().repeat_interleave(used, 0), ids[-last:].flatten()
    (yg, sg), (yu, su) = product(a, gate, flat), product(a, up, flat)
    r = rounding(gate)
    lim = 2 * (r * (1.1 * sg * yu.abs() + (yg * torch.sigmoid(yg)).abs() * su + 1.1 * sg * su * r) + 8 * 2.0 ** -24 * ref.abs() + 1e-30)
    assert bool(((h - ref).abs() <= lim).all())
    del h, act, x
    # the down product's rows: zeros but for the last tokens'
    k, rows, pairs = 4064, 32, tok * used
    down = Experts(Q8_0, n, rows, k, 3)
    small = ops.quantize_act(torch.randn(last * used, k, generator=g, device=DEV), Q8_0)[0]
    big = torch.zeros(pairs * k + pairs * k // 32 * 8, dtype=torch.uint8, device=DEV)
    q, m = last * used * k, last * used * k // 32 * 8
    big[pairs * k - q:pairs * k], big[-m:] = small[:q], small[q:q + m]
    weights = torch.rand(tok, used, generator=g, device=DEV)
    y = ops.moe_down(down.gpu, big, plan, weights)
    assert not bool(y[:-last].any())
    p, size = (v.view(last, used, rows) for v in product(ops.act_values(small, Q8_0, last * used, k, torch.float32).double(), down, flat))
    w = weights[-last:].double()[..., None]
    lim = rounding(down) * (w * size).sum(1) + used * 2.0 ** -24 * (w * p).abs().sum(1) * 1.01 + 1e-30
    assert bool(((y[-last:].double() - (w * p).sum(1)).abs() <= lim).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tok", [2, 5, 17, 18, 20, 35, 66, 130])
def test_a_row_s_place_changes_nothing(t, tok):
    """Equal rows of one expert come out equal, bit for bit, wherever the plan (whose order within an expert is any) puts them."""
    from ameva_compute_amd import ops
    n, rows, k = 3, 96, 2048
    gate, up, down = (Experts(t, n, rows, k, s) for s in (1, 2, 3))
    ids = torch.full((tok, 1), 1, dtype=torch.int32, device=DEV)
    act = ops.quantize_act(torch.randn(1, k, generator=gen(tok), device=DEV).repeat(tok, 1).contiguous(), ACT[t])[0]
    plan = ops.moe_plan(ids, n)
    h = ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=None)
    y = ops.moe_down(down.gpu, act, plan, torch.ones(tok, 1, device=DEV))
    assert torch.equal(h, h[:1].expand_as(h)) and torch.equal(y, y[:1].expand_as(y))
