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


@pytest.mark.parametrize("t", [Q8_0, Q4_0])
@pytest.mark.parametrize("rule,d,at", [(0, 128, (2, 70)), (0, 64, (3, 33)), (1, 128, (0, 127)), (2, 64, (31, 32)), (0, 128, (14, 17))])
def test_append_of_elements_that_are_no_number(t, rule, d, at):
    """A block with such an element gets a scale that is no number, wherever the element stands; all other blocks are as ever, and the
    tokens that see the key or the value get no number where the header says so."""
    from ameva_compute_amd import ops
    a, b, w = (World(t, 2, d, 16, [20, 9], [20, 9], seed=d + rule) for _ in "abw")
    x = w.rand(29, 8, d)
    y = x.clone()
    y[6, 4, at[0]] = math.nan       # a key of KV head 0
    y[6, 7, at[1]] = -math.nan      # a value of KV head 1
    y[25, 4:, at[0]] = math.nan     # all that the second sequence's token 5 stores
    y[25, 4:, at[1]] = math.nan
    q = ops.paged_rope_append(a.cache, a.batch(), x, 4, n_dims=0, rule=rule)
    ops.paged_rope_append(b.cache, b.batch(), y, 4, n_dims=0, rule=rule)
    ni = 16 * d // (1 if t == Q8_0 else 2)
    hit = {(0, 6, "k", 0): at[:1], (0, 6, "v", 1): at[1:], **{(1, 5, p, j): at for p in "kv" for j in range(2)}}
    for p in "kv":
        was, now = getattr(a.cache, p).clone(), getattr(b.cache, p).clone()
        for (s, place, what, j), elements in hit.items():
            if what != p:
                continue
            e, slot = int(w.table[s, place // 16]), place % 16
            for block in {i // 32 for i in elements}:
                c = ni + (slot * (d // 32) + block) * 2
                assert bool(now[e, j, c:c + 2].view(torch.float16).isnan()), (p, s, j, block)
                # (the block's integers do not matter any more)
                row = slice(slot * (ni // 16), (slot + 1) * (ni // 16))
                for pool in (was, now):
                    pool[e, j, c:c + 2] = 0
                    places = pool[e, j, row].view(*((4, d // 32, -1) if p == "k" else (16, d // 32, -1)))
                    places[:, block] = 0
        assert torch.equal(was, now), p
    r = ops.paged_attn(a.cache, a.batch(), q, d ** -0.5)
    z = ops.paged_attn(b.cache, b.batch(), q, d ** -0.5)
    for s, place in ((0, 6), (1, 5)):
        first, hot, end = w.first[s], w.first[s] + place, w.first[s + 1]
        assert off(z[first:hot], r[first:hot].double()) < 2e-5
        assert z[hot:end, :2].isnan().all()  # (heads 0 and 1 are KV head 0's)
        block = at[1] // 32
        assert z[hot:end, 2:, 32 * block:32 * block + 32].isnan().all()


@pytest.mark.parametrize("mode,n_dims", [(0, 64), (2, 64), (2, 32)])
def test_append_of_an_element_that_is_no_number_in_f16(mode, n_dims):
    """F16 pages keep it at its pair's two elements; the bounds are those of the page's other keys there."""
    from ameva_compute_amd import ops
    w = World(F16, 1, 64, 16, [16], [16], seed=3, bounds=True)
    x = w.rand(16, 3, 64)
    x[9, 1, 5] = math.nan
    ops.paged_rope_append(w.cache, w.batch(), x, 1, mode=mode, n_dims=n_dims)
    k = w.cache.k[int(w.table[0, 0]), 0]
    pair = {5, 4} if mode == 0 else {5, 5 + n_dims // 2}
    assert set(torch.nonzero(k.isnan())[:, 1].tolist()) == pair and set(torch.nonzero(k.isnan())[:, 0].tolist()) == {9}
    assert torch.equal(w.cache.bounds[int(w.table[0, 0]), 0],
                       torch.stack([torch.where(k.isnan(), math.inf, k).amin(0), torch.where(k.isnan(), -math.inf, k).amax(0)]))


@pytest.mark.parametrize("heads,g", [(1, 1), (8, 2), (6, 6)])
def test_infinite_bounds_that_no_query_element_meets(heads, g):
    """A bound of infinity where every query of the group has the other sign, or 0, does not enter: the page's score is a number."""
    from ameva_compute_amd import ops
    w = World(F16, g, 64, 16, [16 * 70], seed=heads, bounds=True)
    q = torch.randn(1, heads, 64, device=DEV)
    q[:, :, 3] = -q[:, :, 3].abs()
    q[:, :, 4] = q[:, :, 4].abs()
    q[:, :, 5] = 0.0
    at = w.table[0, 2:60:3].long()
    w.cache.bounds[at, :, 1, 3] = math.inf
    w.cache.bounds[at, :, 0, 4] = -math.inf
    w.cache.bounds[at, :, 0, 5], w.cache.bounds[at, :, 1, 5] = -math.inf, math.inf
    w.cache.bounds[w.table[0, 30].long(), :, 1, 4] = math.inf  # this one's is infinite
    w.cache.bounds[w.table[0, 31].long(), :, :, 9] = math.nan  # and this one's no number
    for n_sel in (1, 9, 69):
        assert torch.equal(ops.paged_select(w.cache, w.batch(), q, n_sel, 0, 0), best_pages(w, q, n_sel, 0, 0))


@pytest.mark.parametrize("t", [Q8_0, Q4_0])
def test_keys_beyond_f16_are_still_selected(t):
    """A quantized key's element above 65504 is an ordinary number, its f16 bound infinite: the page's other elements still count."""
    from ameva_compute_amd import ops
    w = World(t, 1, 64, 16, [16 * 40], [16 * 40], seed=8, bounds=True)
    x = torch.randn(16 * 40, 3, 64, device=DEV)
    x[16 * 25 + 3, 1, 40], x[16 * 25 + 3, 1, :32] = 7e4, 5.0
    ops.paged_rope_append(w.cache, w.batch(), x, 1, n_dims=0)
    page = int(w.table[0, 25])
    assert w.cache.bounds[page, 0, 1, 40] == math.inf and w.cache.bounds[page, 0, 0, 40].isfinite()
    q = torch.ones(1, 1, 64, device=DEV)
    q[0, 0, 40] = -1e-3
    b = ops.PagedBatch(w.n_kv_dev, w.table, 16 * 40)
    assert ops.paged_select(w.cache, b, q, 1, 0, 0).tolist() == [[[25]]]


@pytest.mark.parametrize("t", [F16, Q8_0, Q4_0])
@pytest.mark.parametrize("strange", ["query", "value", "both"])
@pytest.mark.parametrize("prefix,n_kv,n_q", [(0, [700, 300, 64], [300, 90, 64]), (333, [200, 70, 9], [130, 70, 9]), (2100, [5] * 70, [1] * 70)])
def test_rows_that_are_no_number_among_others(t, strange, prefix, n_kv, n_q):
    """One token's query is no number in one head, one sequence's value infinite at a place that some of its tokens do not see: every
    other row is as without them."""
    from ameva_compute_amd import ops
    n_pre = -(-prefix // 16)
    w = World(t, 2, 128, 16, n_kv, n_q, seed=prefix + 17, extra=n_pre)
    pre = w.free[:n_pre].clone()
    q = torch.randn(w.first[-1], 8, 128, device=DEV)
    kv = [x[pre.long()].transpose(0, 1).reshape(2, -1, 128)[:, :prefix] for x in (w.k, w.v)]
    r = attend(w, q, 0.09, prefix=kv)
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    if strange != "value":
        tok = w.first[0] + n_q[0] // 3
        q[tok, 2, 11] = math.nan
        hit[tok, 2] = True
    if strange != "query":
        s = 1
        place = n_kv[s] - 1 - n_q[s] // 2
        e, slot = int(w.table[s, place // 16]), place % 16
        if t == F16:
            w.cache.v[e, 1, slot, 40] = math.inf
        else:
            ni = 16 * 128 // (1 if t == Q8_0 else 2)
            w.cache.v[..., ni:].view(torch.float16).view(-1, 2, 16, 4)[e, 1, slot, 1] = math.inf
        hit[w.first[s + 1] - 1 - n_q[s] // 2:w.first[s + 1], 4:] = True
    b = w.batch()
    y = ops.paged_attn_shared(w.cache, b, q, 0.09, pre, prefix) if prefix else ops.paged_attn(w.cache, b, q, 0.09)
    assert off(y[~hit], r[~hit]) < 1e-5  # (test_gpu_paged_attn.py derives it)
    assert not y[hit].isfinite().all(-1).any()


@pytest.mark.parametrize("t", [F16, Q8_0])
@pytest.mark.parametrize("prefix,n_kv,n_q", [(8192, 64, 1), (0, 1200, 700)])
def test_a_query_that_is_no_number_costs_no_second_pass(t, prefix, n_kv, n_q):
    """The time of a batch with such a row against the same without it (least of several; a second pass over the tile's keys in tiles of
    4 rows took 3 to 7 times as long)."""
    from ameva_compute_amd import ops
    n, n_pre = (64, prefix // 64) if prefix else (2, 0)
    kv = ops.PagedKV.alloc(t, n * -(-n_kv // 64) + n_pre, 64, 8, 128, DEV)
    for x in (kv.k, kv.v):
        x.zero_()
    pages = torch.arange(kv.n_pages, device=DEV).int()
    b = ops.PagedBatch(torch.full((n,), n_kv, device=DEV).int(), pages[n_pre:].view(n, -1).contiguous(), n_kv, n * n_q,
                       cu_q=torch.arange(0, n * n_q + 1, n_q, device=DEV).int(), max_q=n_q)
    q = torch.randn(n * n_q, 32, 128, device=DEV)
    bad = q.clone()
    bad[n * n_q // 3] = math.nan

    def least(x):
        times = []
        for _ in range(6):
            a, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                ops.paged_attn_shared(kv, b, x, 0.1, pages[:n_pre], prefix)
            e.record()
            e.synchronize()
            times.append(a.elapsed_time(e))
        return min(times)
    least(q)
    assert least(bad) < 2 * least(q)


def rows_written_again(w, b, place, x):
    """Appends x at the places from `place` on of a cache that holds one sequence."""
    from ameva_compute_amd import ops
    n = x.shape[0]
    n_kv = torch.tensor([place + n], dtype=torch.int32, device=DEV)
    ops.paged_rope_append(w.cache, ops.PagedBatch(n_kv, w.table, b, n, cu_q=torch.tensor([0, n], dtype=torch.int32, device=DEV), max_q=n),
                          x, 1, n_dims=0)


@pytest.mark.parametrize("t", [F16, Q8_0])
def test_bounds_of_places_written_again(t):
    """Tokens taken back and others appended in their place: the page's bounds hold both, the keys there and those taken back, until
    the page's place 0 is written again; later pages that begin anew have their own."""
    w = World(t, 1, 64, 16, [48], seed=5, bounds=True)
    old, new = w.rand(40, 3, 64), w.rand(14, 3, 64)
    rows_written_again(w, 48, 0, old)
    rows_written_again(w, 48, 20, new)  # 20 .. 33: the rest of page 1, and page 2 from its beginning
    k, k2 = old[:, 1].half(), new[:, 1].half()
    has = lambda *keys: torch.stack([torch.cat(keys).amin(0), torch.cat(keys).amax(0)])
    bounds = w.cache.bounds[w.table[0].long(), 0]
    assert torch.equal(bounds[0], has(k[:16])) and torch.equal(bounds[1], has(k[16:32], k2[:12])) and torch.equal(bounds[2], has(k2[12:]))
    rows_written_again(w, 48, 16, torch.cat([old[16:20], new]))  # the page from its beginning
    bounds = w.cache.bounds[w.table[0].long(), 0]
    assert torch.equal(bounds[1], has(k[16:20], k2[:12])) and torch.equal(bounds[2], has(k2[12:]))


@pytest.mark.parametrize("t", [F16, Q8_0, Q4_0])
@pytest.mark.parametrize("heads,g,n_kv,n_q", [(8, 2, [300, 40], [1, 1]), (8, 2, [300, 40], [2, 1]), (8, 2, [300, 70], [4, 7]),
                                              (32, 2, [90, 64], [2, 1]), (8, 2, [700, 333], [300, 90])])
def test_infinite_keys(t, heads, g, n_kv, n_q):
    """A head's row that sees an infinite key is no number in all elements, or that of the other keys; the rest is as ever."""
    from ameva_compute_amd import ops
    w = World(t, g, 128, 16, n_kv, n_q, seed=31)
    q = torch.randn(w.first[-1], heads, 128, device=DEV)
    r = attend(w, q, 0.09)
    sees = torch.zeros(w.first[-1], dtype=torch.bool, device=DEV)
    there = []
    for s, (n, m) in enumerate(zip(n_kv, n_q)):
        place = n - 1 - m // 2
        e, slot = int(w.table[s, place // 16]), place % 16
        if t == F16:
            w.cache.k[e, 0, slot, 9] = -math.inf if s else math.inf
        else:
            ni = 16 * 128 // (1 if t == Q8_0 else 2)
            w.cache.k[..., ni:].view(torch.float16).view(-1, g, 16, 4)[e, 0, slot, 2] = math.inf
        sees[w.first[s + 1] - 1 - m // 2:w.first[s + 1]] = True
        there.append(torch.arange(n, device=DEV) != place)
    other = attend(w, q, 0.09, see=lambda s, i, j: there[s])
    y, G = ops.paged_attn(w.cache, w.batch(), q, 0.09), heads // g
    assert off(y[~sees], r[~sees]) < 1e-5 and off(y[:, G:], r[:, G:]) < 1e-5
    hit, without = y[sees, :G].flatten(0, 1), other[sees, :G].flatten(0, 1)
    none = hit.isnan().all(-1)
    assert bool(none.any()) and off(hit[~none], without[~none]) < 1e-5


@pytest.mark.parametrize("t", [F16, Q8_0])
@pytest.mark.parametrize("n_q", [1, 2, 4, 100])
def test_queries_of_any_size(t, n_q):
    """|scale log2(e) q| up to 2^117: the key of the largest score has all the weight. From 2^118 on that head's row is no number, and
    the others are as ever."""
    from ameva_compute_amd import ops
    w = World(t, 2, 64, 16, [130], [n_q], seed=n_q)
    q = torch.randn(n_q, 8, 64, device=DEV)
    to = lambda e: 2.0 ** e / (0.125 * math.log2(math.e))
    q[0, 1] *= to(117) / float(q[0, 1].abs().max()) * 0.9
    q[0, 3] *= to(100) / float(q[0, 3].abs().max())
    q[0, 2] *= 2.0 ** -120
    r = attend(w, q, 0.125)
    q[0, 5, 7] = to(118) * 1.01
    y = ops.paged_attn(w.cache, w.batch(), q, 0.125)
    assert y[0, 5].isnan().all()
    y[0, 5] = r[0, 5].float()
    for h in range(8):
        assert off(y[:, h], r[:, h]) < 1e-5, h
