"""Counts, sizes and calls at the ends of what the mixture-of-experts entry points take: refused or reckoned on the host (no GPU call is made)."""
import pytest

from ameva_compute_amd._lib import lib
from test_moe_abi import down, gate_up, plan, refused, route


@pytest.mark.parametrize("call", [gate_up, down])
@pytest.mark.parametrize("wrap", [-(1 << 32), 1 << 32, -(1 << 33), 1 << 40, -(1 << 62)])
def test_counts_whose_lower_half_would_do(call, wrap):
    for p in (4096, None):
        refused(call(used=wrap + 2, p=p), "tokens with")
        refused(call(n=wrap + 8, p=p), "tokens with")
        refused(call(used=wrap + 2, n=wrap + 8, p=p), "tokens with")
        refused(call(tok=wrap + 3, p=p), "tokens with" if wrap < 0 else "pairs")
    for bad in (dict(used=wrap + 2), dict(n=wrap + 8)):
        refused(plan(**bad), "tokens with")
    refused(route(used=wrap + 4), "experts a token")
    refused(route(n=wrap + 64, stride=abs(wrap) + 64), "experts (1 to")


def test_workspaces_of_calls_that_are_refused():
    gu, dn = lib().amv_moe_gate_up_workspace_bytes, lib().amv_moe_down_workspace_bytes
    for t in (8, 15):
        for tok, used, rows in ((1 << 62, 4, 256), (1 << 40, 2, 1 << 40), (3, 1 << 62, 256), (3, 65, 256), (3, 2, 1 << 62), (3, 2, (1 << 20) + 32), (1 << 22, 2, 32)):
            assert gu(tok, used, rows, t) == -1 and dn(tok, used, rows) == -1, (tok, used, rows)
    assert gu(1 << 16, 64, 992, 15) == dn(1 << 16, 64, 992) == 4 * (1 << 22) * 992
    assert gu(3, 2, 256, 15) == 6144 and gu(3, 2, 256, 8) == 0 and gu(0, 2, 256, 15) == dn(0, 2, 256) == 0


def test_a_plan_is_made_where_the_products_without_one_end(monkeypatch):
    torch = pytest.importorskip("torch")
    from ameva_compute_amd import ops
    made = []
    monkeypatch.setattr(ops, "_moe_plan_buffer", lambda ids, n, size: made.append((tuple(ids.shape), n)) or "plan")
    ids = torch.zeros(1, 64, dtype=torch.int32)
    few, many = ops.MoePlan(ids, 100, None), ops.MoePlan(ids, 100, "kept")
    assert ops._moe_buffer(few, (1 << 20) - 32) is None and ops._moe_buffer(many, 32) == "kept" and not made
    assert ops._moe_buffer(few, 1 << 20) == "plan" and made == [((1, 64), 100)] and few.buffer is None
    assert ops._moe_buffer(many, 1 << 20) == "kept" and len(made) == 1
    # the kernels refuse from the same number of columns on
    refused(gate_up(tok=1, used=64, rows=1 << 20, k=32, p=None), "without a plan")
    refused(down(tok=1, used=64, rows=1 << 20, k=32, p=None), "without a plan")


def test_values_of_more_blocks_than_a_launch_holds():
    f = lib().amv_act_values
    for t, step in ((8, 32), (15, 256)):
        for values in ((1 << 34) - step, (1 << 34) - 1024 + step):  # whole blocks, in launches of 2^32 threads
            refused(f(t, 4096, values // step, step, 0, 4096, None), "too many")


def test_calls_by_name():
    """Every argument may be given by its name, the first one too."""
    torch = pytest.importorskip("torch")
    from ameva_compute_amd import ops
    x, ids = torch.zeros(2, 64), torch.zeros(2, 2, dtype=torch.int32)
    act, plan = torch.zeros(80, dtype=torch.uint8), ops.MoePlan(ids, 8, None)
    w = ops.QExperts.__new__(ops.QExperts)
    w.index = -1
    for call in (lambda: ops.add_rms_norm(add=x, x=x, eps=1e-5), lambda: ops.moe_route(logits=x, n_used=2), lambda: ops.moe_plan(ids=ids, n_expert=8),
                 lambda: ops.act_values(act=act, act_type=8, m=2, k=32), lambda: ops.moe_gate_up(gate=w, up=w, act=act, plan=plan),
                 lambda: ops.moe_down(down=w, act=act, plan=plan, weights=x)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError, match="logits"):
        ops.moe_route(n_used=2)


@pytest.mark.parametrize("call", [gate_up, down])
def test_sizes_of_the_products(call):
    """The header's limits, at each of them."""
    far = 1 << 40
    for bad in (dict(rows=(1 << 20) + 32, k=32), dict(rows=32, k=(1 << 20) + 32), dict(rows=1 << 16, k=1 << 15)):
        refused(call(tok=1, used=1, stride=far, **bad), "too large")
    refused(call(tok=1 << 16, used=64, rows=1024, k=32, stride=far), "are too many")
    refused(call(tok=1 << 16, used=64, rows=32, k=1024, stride=far), "are too many")
    # tiles of 16 pairs: as many as pairs where they are few, else one of each expert (and of none) beside the whole ones
    refused(call(tok=256, used=4, n=1024, rows=1 << 18, k=32, stride=far), "tiles of")
    refused(call(tok=2048, used=4, n=1024, rows=174656, k=32, stride=far), "tiles of")
    assert (8192 // 16 + 1025) * 174624 < 1 << 28 <= (8192 // 16 + 1025) * 174656
