"""The mixture-of-experts calls at the ends of their sizes, through ops: what is computed there, and what is refused with a message."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from moe_ref import DEV, Q4_0, Q8_0, Q8_K  # noqa: E402


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
