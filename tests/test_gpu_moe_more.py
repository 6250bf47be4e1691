"""The mixture-of-experts operators: what their header says of masks and of numbers that are none, the norm of prompts, and the products'
8-bit rows of 256."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from moe_ref import ACT, DEV, Q8_0, Q8_K, TYPES, Experts  # noqa: E402


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


# ---------------------------------------------------------------------------------------------------- routing
@pytest.mark.parametrize("renorm", [True, False])
def test_route_of_infinite_logits_and_of_no_numbers(renorm):
    """Softmax: minus infinity masks an expert alone; plus infinity or no number makes the scores none, which the weights show where
    the logits order the row, and which leaves nothing to choose where the scores do. Sigmoid: each expert by itself."""
    from ameva_compute_amd import ops
    n, used = 16, 4
    z = torch.randn(3, n, generator=gen(1), device=DEV)
    z[0, 2:9], z[1, 3], z[2, 5] = -math.inf, math.inf, math.nan
    zero = torch.zeros(n, device=DEV)
    by_logits = [dict(), dict(n_group=4, top_group=2), dict(n_group=4, top_group=4, group_best=2)]
    by_scores = [dict(bias=zero), dict(bias=zero, n_group=4, top_group=2), dict(n_group=4, top_group=2, group_best=2)]
    for i, kw in enumerate(by_logits + by_scores):
        ids, w = ops.moe_route(z, used, renorm=renorm, **kw)
        assert bool((ids[0] >= 0).all()) and bool(w[0].isfinite().all()) and bool((w[0] > 0).all())
        assert not bool(((ids[0] >= 2) & (ids[0] < 9)).any())
        if i < len(by_logits):
            assert bool((ids[1:] >= 0).all()) and bool(w[1:].isnan().all()) and int(ids[1, 0]) == 3 and 5 not in ids[2].tolist()
        else:
            assert bool((ids[1:] == -1).all()) and not bool(w[1:].any())
    for kw in by_logits + by_scores:
        ids, w = ops.moe_route(z, used, score="sigmoid", renorm=renorm, **kw)
        assert bool((ids >= 0).all()) and bool(w.isfinite().all()) and int(ids[1, 0]) == 3 and 5 not in ids[2].tolist()


# ---------------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("rows,n,act", [(1024, 1028, None), (1025, 1056, Q8_0), (1024, 2048, Q8_K), (1024, 2052, None), (1100, 2304, Q8_K),
                                        (1024, 4064, Q8_0), (1030, 4096, Q8_K), (1024, 4100, None)])
@pytest.mark.parametrize("with_w", [True, False])
def test_norm_of_a_prompt(rows, n, act, with_w):
    """From 1024 rows on of up to 4096 elements, 256 threads a row: both of their forms, at the ends of their lengths and past them."""
    from ameva_compute_amd import ops
    g = gen(rows + n)
    x, r = torch.randn(rows, n, generator=g, device=DEV), 3 * torch.randn(rows, n, generator=g, device=DEV)
    w = torch.randn(n, generator=g, device=DEV) if with_w else None
    x[1], r[1] = 0.0, 0.0  # a row of nothing
    s, o, a = ops.add_rms_norm(x, r, 1e-5, w, act_type=act)
    assert torch.equal(s, x + r)
    z = s.double()
    ref = z / (z.square().mean(-1, keepdim=True) + 1e-5).sqrt() * (1 if w is None else w.double())
    # squares, mean, eps, root, quotient, and the two products, each half a step: the squares' and mean's halve in the root
    assert bool(((o - ref).abs() <= 5.5 * 2.0 ** -24 * ref.abs()).all())
    assert act is None or torch.equal(a, ops.quantize_act(o, act)[0])
    # among few rows a row's squares are added in another order; both results keep the bound above, so they are within twice that
    few = ops.add_rms_norm(x[:40].contiguous(), r[:40].contiguous(), 1e-5, w)[1]
    assert bool(((few - o[:40]).double().abs() <= 11 * 2.0 ** -24 * ref[:40].abs()).all())
    x[7, n // 2] = math.nan
    s2, o2, a2 = ops.add_rms_norm(x, r, 1e-5, w, act_type=act)
    keep = torch.arange(rows, device=DEV) != 7
    assert torch.equal(o2[keep], o[keep]) and bool(o2[7].isnan().all())
    if act is not None:
        v, v2 = (ops.act_values(q, act, rows, n, torch.float32) for q in (a, a2))
        assert torch.equal(v2[keep], v[keep]) and bool(v2[7].isnan().all())
    x[7, n // 2] = 0.0
    x[7], r[7] = s[7], 0.0
    y, none, b = ops.add_rms_norm(x, r, 1e-5, w, act_type=act, out=r, normed=False)  # in place
    assert y is r and none is None and torch.equal(r, s) and (act is None or torch.equal(a, b))


# ---------------------------------------------------------------------------------------------------- Q8_K from the products
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tok,n,used,rows", [(1, 4, 3, 512), (2, 30, 3, 256), (7, 5, 3, 768), (40, 16, 2, 256), (48, 12, 4, 512), (200, 3, 2, 512),
                                             (700, 5, 2, 256), (1100, 6, 4, 256)])
def test_gate_up_to_blocks_of_256(t, tok, n, used, rows):
    """The Q8_K rows are those of the f32 values, byte for byte, from each of the products (no plan, few and many pairs an expert, plans of
    more than 4096 pairs), with the values asked for and without; pairs without an expert are zeros, blocks with a number that is none
    have a scale that is none."""
    from ameva_compute_amd import ops
    k, g = 512, gen(tok + rows)
    gate, up = Experts(t, n, rows, k, 1), Experts(t, n, rows, k, 2)
    ids = torch.rand(tok, n, generator=g, device=DEV).topk(used, dim=1)[1].int()
    ids[tok // 2:tok // 2 + max(1, tok // 4), 0] = -1
    ids[tok - tok // 5:] = n
    if tok > 1:
        ids[tok // 3] = ids[tok // 3, :1]
    flat, plan, pairs = ids.flatten(), ops.moe_plan(ids.contiguous(), n), tok * used
    x = torch.randn(tok, k, generator=g, device=DEV)
    act = ops.quantize_act(x, ACT[t])[0]
    h = ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=None)
    want = ops.quantize_act(h, Q8_K)[0]
    for _ in range(2):  # (the workspace holds what the call before left there)
        assert torch.equal(ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=Q8_K), want)
        out, values = ops.moe_gate_up(gate.gpu, up.gpu, act, plan, act_type=Q8_K, eout=True)
        assert torch.equal(out, want) and torch.equal(values, h)
    v = ops.act_values(want, Q8_K, pairs, rows, torch.float32)
    none = (flat < 0) | (flat >= n)
    assert bool(none.any()) and not bool(none.all()) and not bool(v[none].any()) and not bool(h[none].any()) and bool((v[~none] != 0).any(1).all())
    x[0, 3] = math.nan
    bad = ops.add_rms_norm(x, torch.zeros_like(x), 1e-5, act_type=ACT[t])[2]
    good = ops.add_rms_norm(x.nan_to_num(), torch.zeros_like(x), 1e-5, act_type=ACT[t])[2]
    a, b = (ops.act_values(ops.moe_gate_up(gate.gpu, up.gpu, z, plan, act_type=Q8_K), Q8_K, pairs, rows, torch.float32) for z in (bad, good))
    mine = (torch.arange(pairs, device=DEV) < used) & ~none
    assert bool(mine.any())
    assert torch.equal(a[~mine], b[~mine]) and bool(a[mine].isnan().view(-1, rows).any(1).all())
