"""The mixture-of-experts calls at the ends of their sizes, through ops: what is computed there, and what is refused with a message."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from moe_ref import DEV, Q4_0, Q8_0, Q8_K, Experts, product, rounding  # noqa: E402


def test_more_pairs_than_the_products_take():
    """2^22 pairs of 1024 columns are one too many: refused by name, with and without a workspace."""
    from ameva_compute_amd import ops
    from ameva_compute_amd._lib import AmevaError
    tok, used, n, rows = 1 << 19, 8, 8, 1024
    ids = torch.full((tok, used), -1, dtype=torch.int32, device=DEV)
    plan = ops.moe_plan(ids, n)
    experts = lambda k: ops.QExperts(Q4_0, n, rows, k, torch.zeros(n, rows * k // 32 * 18, dtype=torch.uint8, device=DEV))  # noqa: E731
    act = torch.zeros(tok * 40, dtype=torch.uint8, device=DEV)
    for at in (Q8_0, Q8_K):
        with pytest.raises(AmevaError, match="pairs of"):
            ops.moe_gate_up(experts(32), experts(32), act, plan, act_type=at)
    with pytest.raises(AmevaError, match="pairs of"):
        ops.moe_down(experts(32), torch.zeros(tok * used * 40, dtype=torch.uint8, device=DEV), plan, torch.zeros(tok, used, device=DEV))


@pytest.mark.parametrize("tok,used,n,rows", [(1, 64, 2, (1 << 20) - 32), (1, 64, 2, 1 << 20), (6, 64, 1024, 174784)])
def test_few_tokens_of_many_columns(tok, used, n, rows):
    """As many columns as the products without a plan hold, and more: moe_plan makes none for so few tokens, the products see to it."""
    from ameva_compute_amd import ops
    k, live = 32, torch.tensor([0, n - 1] if n == 2 else [0, 511, 1000, n - 1], device=DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(rows)
    pick = torch.randint(0, live.numel(), (tok, used), generator=g, device=DEV)
    pick[0, 3] = -1
    ids = torch.where(pick < 0, -1, live[pick.clamp(min=0)]).int().contiguous()
    e = Experts(Q4_0, live.numel(), rows, k, 1)
    data = torch.zeros(n, e.gpu.data.shape[1], dtype=torch.uint8, device=DEV)
    data[live] = e.gpu.data
    w, plan = ops.QExperts(Q4_0, n, rows, k, data), ops.moe_plan(ids, n)
    act = ops.quantize_act(torch.randn(tok, k, generator=g, device=DEV), Q8_0)[0]
    a = ops.act_values(act, Q8_0, tok, k, torch.float32).double().repeat_interleave(used, 0)
    y, size = product(a, e, pick.flatten())
    h = ops.moe_gate_up(w, w, act, plan, act_type=None)
    r = rounding(e)
    at = 1 << 14  # (columns at a time)
    for c in range(0, rows, at):
        yc, sc, hc = y[:, c:c + at], size[:, c:c + at], h[:, c:c + at].double()
        ref = yc * torch.sigmoid(yc) * yc
        # the products' errors through the derivatives (that of silu is at most 1.1), four roundings and the exponential's of the value itself
        lim = r * sc * (1.1 * yc.abs() + (yc * torch.sigmoid(yc)).abs() + 1.1 * sc * r) + 8 * 2.0 ** -24 * ref.abs() + 1e-30
        assert bool(((hc - ref).abs() <= lim).all())
    del h, y, size
    hact = ops.quantize_act(torch.randn(tok * used, k, generator=g, device=DEV), Q8_0)[0]
    weights, add = torch.rand(tok, used, generator=g, device=DEV) * 2 - 0.5, torch.randn(tok, rows, generator=g, device=DEV)
    y, size = (v.view(tok, used, rows) for v in product(ops.act_values(hact, Q8_0, tok * used, k, torch.float32).double(), e, pick.flatten()))
    wd = weights.double()[..., None]
    ref, parts = add.double() + (wd * y).sum(1), (wd * y).abs().sum(1) + add.double().abs()
    out = ops.moe_down(w, hact, plan, weights, add=add)
    assert bool(((out.double() - ref).abs() <= r * (wd.abs() * size).sum(1) + used * 2.0 ** -24 * parts * 1.01 + 1e-30).all())
