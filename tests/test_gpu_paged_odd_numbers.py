"""Infinite bounds, numbers that are none and rows written again in the paged KV cache: what such a key, value or query may reach
and what it may not."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from paged_ref import DEV, F16, Q4_0, Q8_0, World, attend, off  # noqa: E402


def best_pages(w, q, n_sel, n_first, n_last):
    """paged_select by its definition: the largest sum over a group's heads of max(q low, q high), element by element in f64, where an
    infinite bound meets a q of 0 as 0. One token a sequence."""
    G = q.shape[1] // w.g
    sel = torch.full((len(w.n_kv), w.g, n_sel), -1, dtype=torch.int32)
    bounds, table, x = w.cache.bounds.double().cpu(), w.table.long().cpu(), q.double().cpu()
    for s, n_kv in enumerate(w.n_kv):
        n = -(-n_kv // w.page)
        for j in range(w.g):
            b = bounds[table[s, :n], j][:, :, None]                       # [page][low, high][1][d]
            p = (x[s, j * G:(j + 1) * G] * b).masked_fill((x[s, j * G:(j + 1) * G] == 0) & b.isinf(), 0.0)
            score = p.amax(1).sum((1, 2)).tolist()
            must = [i < n_first or i >= n - n_last for i in range(n)]
            order = sorted(range(n), key=lambda i: (not must[i], math.isnan(score[i]), 0.0 if math.isnan(score[i]) else -score[i], i))
            got = sorted(order[:n_sel])
            sel[s, j, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return sel.to(DEV)


@pytest.mark.parametrize("pages,infinite,n_sel,n_first,n_last", [
    (25, [20, 21, 22, 23, 24], 3, 0, 0),               # more pages of an infinite score than places
    (60, [5, 20, 25, 30, 35, 40, 50], 8, 1, 2),        # and the last pages among the places
    (400, list(range(100, 400, 3)), 64, 1, 1),
    (300, [299, 0, 17], 5, 0, 0),                      # fewer
    (90, list(range(90)), 7, 2, 1),                    # nothing else
])
@pytest.mark.parametrize("heads,g", [(8, 2), (4, 4)])
def test_select_among_infinite_scores(pages, infinite, n_sel, n_first, n_last, heads, g):
    from ameva_compute_amd import ops
    w = World(F16, g, 64, 16, [16 * pages - 3], seed=pages, bounds=True)
    q = torch.randn(1, heads, 64, device=DEV)
    q[:, :, 7] = q[:, :, 7].abs() + 0.1
    w.cache.bounds[w.table[0, infinite].long(), :, 1, 7] = math.inf
    sel = ops.paged_select(w.cache, w.batch(), q, n_sel, n_first, n_last)
    assert torch.equal(sel, best_pages(w, q, n_sel, n_first, n_last))
