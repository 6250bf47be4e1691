"""Keys and values appended to pages: the stored f16 values and ggml blocks bit for bit those of the f64 rotation rounded to f32, the
page bounds, what lies around them untouched, and tokens that cannot be stored counted and left out."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from paged_ref import DEV, F16, Q4_0, Q8_0, World, pack, unpack  # noqa: E402


def rotate(x, pos, n_dims, mode, base=10000.0, scale=1.0, factor=1.0):
    """f64 on the CPU: x [n, heads, d]."""
    x = x.double().cpu()
    ang = pos.double().cpu()[:, None] * scale * base ** (-2.0 * torch.arange(n_dims // 2, dtype=torch.float64) / max(n_dims, 1))
    c, s = ang.cos()[:, None] * factor, ang.sin()[:, None] * factor
    y = x.clone()
    a, b = (slice(0, n_dims // 2), slice(n_dims // 2, n_dims)) if mode == 2 else (slice(0, n_dims, 2), slice(1, n_dims, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y.to(DEV)


def places(w):
    return torch.cat([torch.arange(a - b, a) for a, b in zip(w.n_kv, w.n_q)]).int().to(DEV)


def append_and_check(w, heads, qkv, pos=None, rule=0, stored=None, **rope):
    from ameva_compute_amd import ops
    n, g, d, page = w.first[-1], w.g, w.d, w.page
    kw = {"mode": 0, "n_dims": d, **rope}
    at_all = places(w)
    before = [x.clone() for x in (w.cache.k, w.cache.v)]
    had = None if w.cache.bounds is None else w.cache.bounds.clone()
    y = rotate(qkv[:, :heads + g], at_all if pos is None else pos, kw["n_dims"], kw["mode"], kw.get("freq_base", 1e4),
               kw.get("freq_scale", 1.0), kw.get("attn_factor", 1.0))
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = ops.paged_rope_append(w.cache, w.batch(), qkv, heads, pos=pos, rule=rule, bad=bad, **kw)
    # one rounding to f32 of the f64 value. An angle of a radians is off by up to 4 roundings of 2^-53 a on either side (the
    # frequency, the product, its way into a sine), which moves a value by that times the length of its pair, at most 8 here: at
    # position 1.3e6 by 9e-9, at 300 by 2e-12
    far = 1 + float((at_all if pos is None else pos).abs().max())
    slack = 8 * far * 8 * 2.0 ** -53 * max(1.0, float(qkv.abs().max()) / 8)
    wrong = (q.double() - y[:, :heads]).abs() - y[:, :heads].abs() * 2.0 ** -24
    assert wrong.max().item() <= slack
    seq = torch.cat([torch.full((b,), s) for s, b in enumerate(w.n_q)]).to(DEV)
    stored = torch.ones(n, dtype=torch.bool, device=DEV) if stored is None else stored
    assert int(bad) == int((~stored).sum()) * g
    new = [y[:, heads:].float(), qkv[:, heads + g:].float()]
    want = []
    for of, old, x in zip("kv", before, new):
        full = unpack(old, w.t, of, page, d)  # NaN scales and all: compared as bytes below
        one, _ = pack(x[:, :, None].contiguous(), w.t, of, rule)
        full = old.clone()
        for i in torch.nonzero(stored).flatten().tolist():
            p, r = int(w.table[seq[i], at_all[i] // page]), int(at_all[i]) % page
            if w.t == F16:
                full[p, :, r] = one[i, :, 0]
            else:
                ni = d if w.t == Q8_0 else d // 2
                full[p, :, r * ni:(r + 1) * ni] = one[i, :, :ni]
                full[p, :, page * ni + r * d // 16:page * ni + (r + 1) * d // 16] = one[i, :, ni:]
        want.append(full)
    for of, got, x in zip("kv", (w.cache.k, w.cache.v), want):
        assert torch.equal(got.view(torch.uint8), x.view(torch.uint8)), of
    if had is not None:
        k16 = new[0].half()
        for i in torch.nonzero(stored).flatten().tolist():
            p, r = int(w.table[seq[i], at_all[i] // page]), int(at_all[i]) % page
            if r == 0:
                had[p, :, 0], had[p, :, 1] = k16[i], k16[i]
            had[p, :, 0], had[p, :, 1] = torch.minimum(had[p, :, 0], k16[i]), torch.maximum(had[p, :, 1], k16[i])
        assert torch.equal(w.cache.bounds, had)
    return q


@pytest.mark.parametrize("t", [F16, Q8_0, Q4_0])
@pytest.mark.parametrize("heads,g,d,page,n_kv,n_q,mode,n_dims", [
    (32, 8, 128, 64, [1, 64, 65, 200], [1, 1, 1, 1], 0, 128),
    (20, 5, 128, 16, [40, 16, 33, 5], [40, 3, 18, 0], 2, 128),
    (8, 8, 64, 32, [100, 1], [70, 1], 0, 64),
    (12, 1, 64, 16, [17, 50], [2, 1], 2, 32),       # part of a head rotated
    (4, 2, 128, 128, [300], [299], 0, 96),
    (4, 2, 128, 16, [20], [3], 2, 0),               # none of it
])
def test_append(t, heads, g, d, page, n_kv, n_q, mode, n_dims):
    w = World(t, g, d, page, n_kv, n_q, seed=d + page, bounds=True)
    append_and_check(w, heads, w.rand(w.first[-1], heads + 2 * g, d), mode=mode, n_dims=n_dims)


@pytest.mark.parametrize("rule", [0, 1, 2])
def test_rules_scales_and_odd_values(rule):
    w = World(Q8_0, 2, 64, 16, [30], [20], seed=rule)
    x = w.rand(20, 8, 64)
    x[3] = 0.0
    x[4] *= 1e-6
    x[5] *= 1e4
    append_and_check(w, 4, x, rule=rule, freq_base=500000.0, freq_scale=0.25, attn_factor=1.25)


def test_far_positions():
    """Positions whose angles f32 no longer tells apart."""
    w = World(F16, 1, 128, 16, [40], [40], bounds=True)
    append_and_check(w, 4, w.rand(40, 6, 128), pos=torch.arange(40, device=DEV).int() * 7919 + 1_000_000, mode=2, freq_base=5e5)


def test_in_place_and_strided_rows():
    from ameva_compute_amd import ops
    from ameva_compute_amd._lib import lib
    w, w2 = (World(Q4_0, 2, 64, 16, [30, 9], [20, 1], seed=4) for _ in "ab")
    x = w.rand(21, 14, 64)
    q = ops.paged_rope_append(w2.cache, w2.batch(), x[:, :10], 6)
    y = x.clone()
    b = w.batch()
    rc = lib().amv_paged_rope_append(w.cache._p, b._p, y.data_ptr(), y.stride(0), 6, None, 64, 0, 1e4, 1.0, 1.0, 0, y.data_ptr(),
                                     y.stride(0), None, ops._stream())
    assert rc == 0
    assert torch.equal(y[:, :6], q) and torch.equal(y[:, 6:], x[:, 6:])
    assert torch.equal(w.cache.k, w2.cache.k) and torch.equal(w.cache.v, w2.cache.v)


def test_tokens_that_cannot_be_stored():
    w = World(F16, 2, 64, 16, [3, 40, 33], [5, 20, 1], bounds=True, seed=5)
    seq = torch.cat([torch.full((b,), s) for s, b in enumerate(w.n_q)]).to(DEV)
    at = places(w)
    stored = at >= 0  # two of sequence 0's tokens stand before its beginning
    w.table[1, 1] = 10 ** 6  # places 16 .. 31 of sequence 1
    w.table[2, 2] = -3
    stored &= ~((seq == 1) & (at // 16 == 1)) & (seq != 2)
    append_and_check(w, 4, w.rand(26, 8, 64), stored=stored)


def test_places_from_max_kv_on_are_not_stored():
    from ameva_compute_amd import ops
    w = World(F16, 1, 64, 16, [40], [20], bounds=True)
    x, bad = w.rand(20, 3, 64), torch.zeros(1, dtype=torch.int32, device=DEV)
    k, bounds = w.cache.k.clone(), w.cache.bounds.clone()
    ops.paged_rope_append(w.cache, w.batch(max_kv=24), x, 1, bad=bad)
    assert int(bad) == 16
    p = w.table[0].long()
    assert not torch.equal(w.cache.k[p[1], :, 4:8], k[p[1], :, 4:8])
    assert torch.equal(w.cache.k[p[1], :, 8:].view(torch.uint8), k[p[1], :, 8:].view(torch.uint8))
    assert torch.equal(w.cache.k[p[2]].view(torch.uint8), k[p[2]].view(torch.uint8)) and torch.equal(w.cache.bounds[p[2]], bounds[p[2]])


def test_bounds_grow_token_by_token_as_at_once():
    from ameva_compute_amd import ops
    a, b = (World(F16, 2, 128, 16, [50], [50], seed=6, bounds=True) for _ in "ab")
    x = a.rand(50, 8, 128)
    ops.paged_rope_append(a.cache, a.batch(), x, 4)
    n_kv = torch.ones(1, dtype=torch.int32, device=DEV)
    one = ops.PagedBatch(n_kv, b.table, 50)
    for i in range(50):
        ops.paged_rope_append(b.cache, one, x[i:i + 1], 4)
        n_kv += 1
    assert torch.equal(a.cache.k.view(torch.uint8), b.cache.k.view(torch.uint8)) and torch.equal(a.cache.bounds, b.cache.bounds)
    assert math.isfinite(float(a.cache.bounds[a.table[0].long()].float().abs().max()))
