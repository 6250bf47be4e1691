"""The mixture-of-experts operators: what their header says of masks and of numbers that are none."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from moe_ref import DEV  # noqa: E402


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
