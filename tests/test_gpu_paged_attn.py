"""Attention over the paged KV cache against float64: cache types, head layouts and page sizes; lengths of 0, 1 and around every
tile's end; tokens of one and of many rows, ragged together; a shared prefix; selected pages.

Tolerance: q and the weights go to the matrix cores as two f16, 22 bits together, and everything else is f32. A score of at most 16
sums 128 products in f32: with 2^-24 / sqrt(3) of a partial sum below 16 per rounding and 130 roundings, its rms error is below
6.3e-6, which is the relative error of a weight; the output is a weighted mean of them and shares it at most. 1e-5 holds that
with the splits' 2^-22 and the sums' roundings."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from paged_ref import DEV, F16, Q4_0, Q8_0, World, attend, off  # noqa: E402

TOL = 1e-5


def run(w, heads, seed=1, pad=0, gain=1.0, **kw):
    from ameva_compute_amd import ops
    torch.manual_seed(seed)
    b = w.batch(pad=pad, **kw)
    q = torch.randn(b.n_tok, heads, w.d, device=DEV) * gain
    out = torch.full_like(q, 7.0)
    y = ops.paged_attn(w.cache, b, q, w.d ** -0.5, out=out)
    assert y is out
    n = w.first[-1]
    assert bool((y[n:] == 7.0).all())  # rows behind the last sequence
    return y[:n], attend(w, q[:n], w.d ** -0.5)


@pytest.mark.parametrize("t", [F16, Q8_0, Q4_0])
@pytest.mark.parametrize("heads,g,d,page", [(32, 8, 128, 64), (20, 5, 128, 16), (8, 8, 64, 32), (12, 1, 64, 16), (16, 2, 128, 256),
                                            (40, 2, 64, 128), (66, 2, 128, 1024)])
def test_decode(t, heads, g, d, page):
    w = World(t, g, d, page, [1, 0, 15, 16, 17, 31, 32, 33, 127, 128, 129, 500, 1025], seed=heads)
    y, r = run(w, heads)
    assert off(y, r) < TOL
    assert not y[1].any()


@pytest.mark.parametrize("t", [F16, Q8_0, Q4_0])
@pytest.mark.parametrize("heads,g,d,page,n_kv,n_q", [
    (32, 8, 128, 64, [300, 70, 5, 64], [4, 2, 5, 1]),          # a few tokens each
    (32, 8, 128, 16, [700, 90, 33, 1, 200], [260, 1, 33, 1, 0]),  # a prompt chunk among decode steps, a sequence without tokens
    (20, 5, 128, 32, [129, 64], [129, 64]),                    # prompts without a past
    (8, 8, 64, 128, [1000, 40], [37, 40]),
    (12, 1, 64, 16, [99, 35, 16], [3, 35, 16]),
    (16, 1, 128, 64, [50, 20], [2, 1]),                        # one row more than a tile, and a tile
])
def test_ragged(t, heads, g, d, page, n_kv, n_q):
    w = World(t, g, d, page, n_kv, n_q, seed=sum(n_kv))
    y, r = run(w, heads, pad=3)
    assert off(y, r) < TOL
    for s in range(len(n_kv)):  # no sequence hides in another's norm
        a, e = w.first[s], w.first[s + 1]
        assert off(y[a:e], r[a:e]) < TOL, s


def test_more_tokens_than_keys():
    w = World(F16, 2, 128, 16, [3, 0], [5, 2])
    y, r = run(w, 8)
    assert not y[:2].any() and not y[5:].any() and off(y, r) < TOL  # tokens before place 0 see nothing


@pytest.mark.parametrize("t", [F16, Q8_0])
def test_keys_from_max_kv_on_are_not_seen(t):
    w = World(t, 2, 64, 16, [100, 40], seed=3)
    from ameva_compute_amd import ops
    q = torch.randn(2, 4, 64, device=DEV)
    y = ops.paged_attn(w.cache, w.batch(max_kv=48), q, 0.125)
    w.n_kv = [48, 40]
    assert off(y, attend(w, q, 0.125)) < TOL


def test_pages_outside_the_pool_hold_no_keys():
    from ameva_compute_amd import ops
    w = World(F16, 2, 128, 16, [100, 64], seed=4)
    q = torch.randn(2, 8, 128, device=DEV)
    w.table[0, 2], w.table[0, 3], w.table[1, 0] = 10 ** 9, -5, w.cache.n_pages
    y = ops.paged_attn(w.cache, w.batch(), q, 0.1)
    kept = [torch.tensor([j // 16 not in bad for j in range(n)], device=DEV) for n, bad in ((100, (2, 3)), (64, (0,)))]
    w2 = World(F16, 2, 128, 16, [100, 64], seed=4)
    assert off(y, attend(w2, q, 0.1, see=lambda s, i, j: kept[s])) < TOL
    w.table.fill_(-1)
    assert not ops.paged_attn(w.cache, w.batch(), q, 0.1).any()


@pytest.mark.parametrize("t", [F16, Q8_0, Q4_0])
def test_magnitudes(t):
    """Values far above and below 1, a key that outweighs the others and adds nothing, scores whose differences are large."""
    from ameva_compute_amd import ops
    for k_gain, v_gain, q_gain in ((1e-2, 3e3, 1e2), (50.0, 1e-4, 1e-3), (1.0, 1.0, 0.0)):
        w = World(t, 2, 128, 16, [70, 333], [1, 9], seed=5, k_gain=k_gain, v_gain=v_gain)
        y, r = run(w, 8, gain=q_gain)
        assert off(y, r) < TOL, (k_gain, v_gain, q_gain)
    w = World(t, 1, 128, 16, [600], seed=6)
    q = torch.randn(1, 4, 128, device=DEV)
    from paged_ref import pack
    spike = torch.zeros(1, 1, 16, 128, device=DEV)
    spike[:] = q[0, 0] * 1.3  # scores of about 15 on the first page, whose values are 0
    at = int(w.table[0, 0])
    for of, x in (("k", spike), ("v", torch.zeros_like(spike))):
        pool, value = pack(x, t, of)
        getattr(w.cache, of)[at], getattr(w, of)[at] = pool[0], value[0]
    y = ops.paged_attn(w.cache, w.batch(), q, 128 ** -0.5)
    assert off(y, attend(w, q, 128 ** -0.5)) < 2 * TOL  # (a score of 15 and the sums around it)


@pytest.mark.parametrize("t", [F16, Q4_0])
def test_strided_rows_and_pages_in_a_common_pool(t):
    """q rows inside q/k/v rows; two layers' pages side by side in one allocation."""
    from ameva_compute_amd import ops
    w = World(t, 2, 64, 16, [50, 20, 33], [1, 2, 1], seed=7)
    kv = [torch.empty((w.cache.n_pages, 2, *x.shape[1:]), dtype=x.dtype, device=DEV) for x in (w.cache.k, w.cache.v)]
    kv = [x.view(torch.uint8).fill_(0xFF).view(x.dtype) for x in kv]
    for x, src in zip(kv, (w.cache.k, w.cache.v)):
        x[:, 1] = src
    w.cache = ops.PagedKV(t, kv[0][:, 1], kv[1][:, 1], 16, 2, 64)
    q = torch.randn(4, 12, 64, device=DEV)[:, :8]
    y = ops.paged_attn(w.cache, w.batch(), q, 0.125)
    assert off(y, attend(w, q, 0.125)) < TOL


def test_pool_beyond_4_gib():
    """Pages whose bytes lie behind 2^32 (keys, values and scales)."""
    from ameva_compute_amd import ops
    w = World(Q8_0, 8, 128, 1024, [900, 1100], seed=8)
    n = 4500  # 4500 x 1.1 MB
    k, v = (torch.empty((n, *w.cache.k.shape[1:]), dtype=torch.uint8, device=DEV) for _ in "kv")
    at = torch.arange(n - w.cache.n_pages, n, device=DEV)
    assert at[0].item() * k.stride(0) > 2 ** 32
    k[at], v[at] = w.cache.k, w.cache.v
    q = torch.randn(2, 32, 128, device=DEV)
    r = attend(w, q, 0.08)
    table = torch.where(w.table >= 0, w.table + (n - w.cache.n_pages), w.table)
    y = ops.paged_attn(ops.PagedKV(Q8_0, k, v, 1024, 8, 128), ops.PagedBatch(w.n_kv_dev, table, 1100), q, 0.08)
    assert off(y, r) < TOL


# ------------------------------------------------------------------------------------------------- shared prefix
@pytest.mark.parametrize("t", [F16, Q8_0, Q4_0])
@pytest.mark.parametrize("heads,g,d,page,prefix,n_kv,n_q", [
    (32, 8, 128, 64, 333, [1, 40, 9], [1, 1, 1]),
    (20, 5, 128, 16, 1000, [5] * 40, [1] * 40),              # more rows than a tile, more keys than a part
    (8, 8, 64, 32, 31, [3, 0, 70], [3, 1, 2]),                # a token before its sequence's place 0 sees the prefix
    (12, 1, 64, 16, 1, [20, 1], [1, 1]),
    (32, 8, 128, 64, 500, [90, 1], [90, 1]),                  # a prompt chunk behind the prefix
])
def test_shared_prefix(t, heads, g, d, page, prefix, n_kv, n_q):
    from ameva_compute_amd import ops
    n_pre = -(-prefix // page)
    w = World(t, g, d, page, n_kv, n_q, seed=prefix, extra=n_pre)
    pre = w.free[:n_pre].clone()
    q = torch.randn(w.first[-1] + 2, heads, d, device=DEV)
    out = torch.full_like(q, 7.0)
    y = ops.paged_attn_shared(w.cache, w.batch(pad=2), q, d ** -0.5, pre, prefix, out=out)
    kv = [x[pre.long()].transpose(0, 1).reshape(g, -1, d)[:, :prefix] for x in (w.k, w.v)]
    n = w.first[-1]
    assert off(y[:n], attend(w, q[:n], d ** -0.5, prefix=kv)) < TOL
    assert bool((y[n:] == 7.0).all())
    if prefix > page:  # no prefix is paged_attn
        assert torch.equal(ops.paged_attn_shared(w.cache, w.batch(pad=2), q, d ** -0.5, pre, 0)[:n],
                           ops.paged_attn(w.cache, w.batch(pad=2), q, d ** -0.5)[:n])


# ------------------------------------------------------------------------------------------------- selected pages
def choose(w, q, n_sel, n_first, n_last):
    """paged_select in f64, a token and a KV head at a time."""
    G = q.shape[1] // w.g
    sel = torch.full((q.shape[0], w.g, n_sel), -1, dtype=torch.int32)
    b = w.cache.bounds.double().cpu()
    table, x = w.table.long().cpu(), q.double().cpu()
    for s, (n_kv, n_q) in enumerate(zip(w.n_kv, w.n_q)):
        for i in range(n_q):
            tok, seen = w.first[s] + i, n_kv - n_q + i + 1
            n = -(-seen // w.page) if seen > 0 else 0
            for j in range(w.g):
                got = []
                for p in range(n):
                    e = int(table[s, p])
                    if p < n_first or p >= n - n_last:
                        got.append((-math.inf, p))
                    elif 0 <= e < w.cache.n_pages:
                        y = x[tok, j * G:(j + 1) * G]
                        sc = float((y.clamp(min=0).sum(0) * b[e, j, 1] + y.clamp(max=0).sum(0) * b[e, j, 0]).sum())
                        got.append((1e300 if math.isnan(sc) else -sc, p))
                    else:
                        got.append((1e300, p))
                got = sorted(p for _, p in sorted(got)[:n_sel])
                sel[tok, j, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return sel.to(q.device)


@pytest.mark.parametrize("heads,g,d,page,n_kv,n_q,n_sel,n_first,n_last", [
    (32, 8, 128, 16, [2000, 100, 1, 0, 65], None, 8, 1, 2),
    (8, 8, 64, 32, [999, 3000], [2, 3], 16, 0, 1),
    (20, 5, 128, 64, [6000], None, 5, 0, 0),
    (12, 1, 64, 16, [5000, 300], None, 3, 1, 2),   # nothing is left to choose
    (16, 2, 128, 16, [20000], None, 64, 1, 1),
])
def test_select(heads, g, d, page, n_kv, n_q, n_sel, n_first, n_last):
    from ameva_compute_amd import ops
    w = World(F16, g, d, page, n_kv, n_q, seed=n_sel, bounds=True)
    q = torch.randn(w.first[-1], heads, d, device=DEV)
    sel = ops.paged_select(w.cache, w.batch(), q, n_sel, n_first, n_last)
    assert torch.equal(sel, choose(w, q, n_sel, n_first, n_last))


def test_select_ties_and_numbers_that_are_none():
    from ameva_compute_amd import ops
    w = World(F16, 1, 64, 16, [16 * 400], bounds=True)
    q = torch.randn(1, 4, 64, device=DEV)
    w.cache.bounds[:] = w.cache.bounds[:1]  # all pages alike: the lowest indices
    assert torch.equal(ops.paged_select(w.cache, w.batch(), q, 9, 1, 2)[0, 0], torch.tensor([*range(7), 398, 399], device=DEV).int())
    high = w.table[0, [50, 200, 300]].long()
    w.cache.bounds[high] = w.cache.bounds[high] + 1.0  # three pages above, alike among themselves
    w.cache.bounds[w.table[0, 2].long()] = math.nan
    w.table[0, 3] = -1
    got = ops.paged_select(w.cache, w.batch(), q, 6, 0, 1)
    assert torch.equal(got, choose(w, q, 6, 0, 1))
    assert torch.equal(ops.paged_select(w.cache, w.batch(), q, 399, 0, 0), choose(w, q, 399, 0, 0))  # the page without a score last
    w.cache.bounds.fill_(math.inf)  # no score is a number
    assert torch.equal(ops.paged_select(w.cache, w.batch(), q.abs() + 1, 6, 0, 1), choose(w, q.abs() + 1, 6, 0, 1))


def test_select_most_pages():
    from ameva_compute_amd import ops
    w = World(F16, 1, 64, 16, [16 * 16384], bounds=True)
    q = torch.randn(1, 1, 64, device=DEV)
    sel = ops.paged_select(w.cache, w.batch(), q, 40, 1, 1)
    up, down = q[0, 0].double().clamp(min=0), q[0, 0].double().clamp(max=0)
    b = w.cache.bounds[w.table[0].long(), 0].double()
    score = b[:, 1] @ up + b[:, 0] @ down
    score[0] = score[-1] = math.inf
    assert torch.equal(sel[0, 0].long(), score.topk(40)[1].sort()[0])


@pytest.mark.parametrize("t", [F16, Q8_0, Q4_0])
@pytest.mark.parametrize("heads,g,d,page,n_kv,n_q,n_sel", [
    (32, 8, 128, 64, [2000, 64, 1, 0], None, 9), (20, 5, 128, 16, [900, 333], [3, 1], 7), (8, 8, 64, 32, [4000], None, 40),
    (40, 2, 64, 16, [500, 60], [1, 2], 5)])
def test_sparse(t, heads, g, d, page, n_kv, n_q, n_sel):
    from ameva_compute_amd import ops
    w = World(t, g, d, page, n_kv, n_q, seed=n_sel, bounds=True)
    q = torch.randn(w.first[-1] + 1, heads, d, device=DEV)
    b = w.batch(pad=1)
    sel = ops.paged_select(w.cache, b, q, n_sel, sel=torch.full((b.n_tok, g, n_sel), -1, dtype=torch.int32, device=DEV))
    out = torch.full_like(q, 7.0)
    y = ops.paged_attn_sparse(w.cache, b, q, sel, d ** -0.5, out=out)

    def see(s, i, j):
        n = max(n_kv[s], 0)
        page_of = torch.arange(n, device=DEV) // page
        return torch.isin(page_of, sel[w.first[s] + i, j])
    n = w.first[-1]
    assert off(y[:n], attend(w, q[:n], d ** -0.5, see=see)) < TOL
    assert bool((y[n:] == 7.0).all())
    assert not (bool(sel[n:].ne(-1).any()))


def test_sparse_takes_any_choice():
    """Pages out of order, entries that are no page among them, and rows without one."""
    from ameva_compute_amd import ops
    w = World(F16, 2, 128, 16, [300, 300], seed=9)
    q = torch.randn(2, 8, 128, device=DEV)
    sel = torch.full((2, 2, 9), -1, dtype=torch.int32, device=DEV)
    sel[0, 0] = torch.tensor([7, -1, 3, 10 ** 8, 18, 0, -9, 19, 5], device=DEV)
    sel[0, 1, 4] = 2
    y = ops.paged_attn_sparse(w.cache, w.batch(), q, sel, 0.09)
    page_of = torch.arange(300, device=DEV) // 16
    assert off(y, attend(w, q, 0.09, see=lambda s, i, j: torch.isin(page_of, sel[s, j]))) < TOL
    assert not y[1].any()


def test_all_pages_selected_is_dense():
    from ameva_compute_amd import ops
    w = World(Q8_0, 2, 128, 16, [300, 77], seed=10, bounds=True)
    q = torch.randn(2, 8, 128, device=DEV)
    sel = ops.paged_select(w.cache, w.batch(), q, 30)
    assert off(ops.paged_attn_sparse(w.cache, w.batch(), q, sel, 0.09), ops.paged_attn(w.cache, w.batch(), q, 0.09).double()) < TOL


# ------------------------------------------------------------------------------------------------- what nobody may see
@pytest.mark.parametrize("t", [F16, Q8_0, Q4_0])
@pytest.mark.parametrize("heads,g,d,page,n_kv,n_q", [
    (32, 8, 128, 64, [300, 70, 40], [4, 2, 1]),
    (8, 2, 128, 16, [700, 33, 64], [260, 33, 1]),
    (8, 2, 128, 16, [1300, 33], [260, 33]),
    (6, 2, 64, 32, [1200, 90], [200, 9]),
    (40, 2, 128, 64, [100, 64], [3, 1]),
])
def test_later_tokens_do_not_matter(t, heads, g, d, page, n_kv, n_q):
    """A token whose value is infinite or no number, one whose key is: tokens before it, in the same tile or not, do not see it; what
    those behind it get there is no number, and elements and heads that it does not reach are right."""
    from ameva_compute_amd import ops
    w = World(t, g, d, page, n_kv, n_q, seed=n_kv[0])
    q = torch.randn(w.first[-1], heads, d, device=DEV)
    r = attend(w, q, d ** -0.5)
    for s, (n, m) in enumerate(zip(n_kv, n_q)):
        place = n - 1 - m // 2
        e, slot = int(w.table[s, place // page]), place % page
        if t == F16:
            w.cache.v[e, 0, slot, 5], w.cache.v[e, 0, slot, 40] = math.nan if s & 1 else -math.inf, math.inf
            w.cache.k[e, 1, slot, 3] = math.nan
        else:
            ni = page * d // (1 if t == Q8_0 else 2)
            v, k = (x[..., ni:].view(torch.float16).view(-1, g, page, d // 32) for x in (w.cache.v, w.cache.k))
            v[e, 0, slot, 1] = math.nan if s & 1 else math.inf
            k[e, 1, slot, 0] = math.nan
    y, G = ops.paged_attn(w.cache, w.batch(), q, d ** -0.5), heads // g
    for s, (n, m) in enumerate(zip(n_kv, n_q)):
        a, at, e = w.first[s], w.first[s] + m - 1 - m // 2, w.first[s] + m
        if at > a:
            assert off(y[a:at], r[a:at]) < TOL, s
        hit = [5, 40] if t == F16 else list(range(32, 64))
        assert not y[at:e, :G][..., hit].isfinite().any() and y[at:e, G:2 * G].isnan().all(), s
        if g > 2:
            assert off(y[at:e, 2 * G:], r[at:e, 2 * G:]) < TOL, s
        if m == 1:
            rest = [i for i in range(d) if i not in hit]
            assert off(y[at:e, :G][..., rest], r[at:e, :G][..., rest]) < TOL, s


@pytest.mark.parametrize("t", [F16, Q4_0])
def test_more_sequences_than_lanes(t):
    """150 sequences: steps, a few tokens, prompts, sequences without tokens or without keys, in no order."""
    n_kv = [(37 * i) % 211 for i in range(150)]
    n_q = [min(n, (0, 1, 1, 5, 40)[i * 7 % 5]) for i, n in enumerate(n_kv)]
    w = World(t, 2, 64, 16, n_kv, n_q, seed=11)
    y, r = run(w, 8, pad=2)
    for s in range(150):
        a, e = w.first[s], w.first[s + 1]
        assert off(y[a:e], r[a:e]) < TOL, s


@pytest.mark.parametrize("t", [F16, Q8_0])
@pytest.mark.parametrize("heads,g,d,prefix,n,kv", [(16, 4, 128, 700, 150, 3), (8, 2, 64, 2100, 70, 40), (4, 1, 128, 1500, 40, 300)])
def test_shared_prefix_of_many_sequences(t, heads, g, d, prefix, n, kv):
    """More rows than 128 behind a prefix, whose last tile is not whole."""
    from ameva_compute_amd import ops
    n_kv, n_pre = [(kv * i) % (kv + 1) + 1 for i in range(n)], -(-prefix // 16)
    w = World(t, g, d, 16, n_kv, seed=12, extra=n_pre)
    pre = w.free[:n_pre].clone()
    q = torch.randn(n, heads, d, device=DEV)
    y = ops.paged_attn_shared(w.cache, w.batch(), q, d ** -0.5, pre, prefix)
    kv = [x[pre.long()].transpose(0, 1).reshape(g, -1, d)[:, :prefix] for x in (w.k, w.v)]
    assert off(y, attend(w, q, d ** -0.5, prefix=kv)) < TOL


@pytest.mark.parametrize("t", [F16, Q4_0])
@pytest.mark.parametrize("n,n_q", [(5, 1), (70, 1), (3, 40)])
def test_padding_that_is_no_number(t, n, n_q):
    """q rows behind the last sequence, fewer and more of them than a tile, hold no numbers: nobody reads them."""
    from ameva_compute_amd import ops
    w = World(t, 2, 128, 16, [n_q + 9] * n, [n_q] * n, seed=13, extra=30, bounds=True)
    pre, m = w.free[:30].clone(), n * n_q
    for pad in (3, 200):
        b = w.batch(pad=pad)
        q = torch.randn(m + pad, 8, 128, device=DEV)
        q[m:] = math.nan
        kv = [x[pre.long()].transpose(0, 1).reshape(2, -1, 128)[:, :470] for x in (w.k, w.v)]
        out = torch.full_like(q, 7.0)
        ops.paged_attn_shared(w.cache, b, q, 0.09, pre, 470, out=out)
        assert off(out[:m], attend(w, q[:m], 0.09, prefix=kv)) < TOL and bool((out[m:] == 7.0).all())
        out.fill_(7.0)
        ops.paged_attn(w.cache, b, q, 0.09, out=out)
        assert off(out[:m], attend(w, q[:m], 0.09)) < TOL and bool((out[m:] == 7.0).all())
        sel = ops.paged_select(w.cache, b, q, 2)
        assert torch.equal(sel[:m], choose(w, q[:m], 2, 1, 1))
