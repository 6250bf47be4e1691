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
