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
