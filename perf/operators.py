"""The paged KV cache operators, measured over the ranges a server has: keys and values appended to pages with the position
rotation on the way, attention of a ragged batch over its pages, attention of a batch whose sequences share a long prefix,
and attention over the pages that a cheap score selects.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what a program holds before the call, run()
is one pass (own: through ameva_compute_amd.ops, else in elementary torch operations), work() what the pass cannot do
without, exact() its outputs in 64 bits. Pools are made here, in plain torch, in the layout include/ameva_hip.h describes:

  F16         k, v f16 [page][KV head][key][d]
  Q8_0, Q4_0  k, v bytes [page][KV head][integers of all keys | scales of all keys]: integers [key][place] (Q8_0: int8; Q4_0:
              two places a byte, the even one in the low bits, value + 8), scales f16 [key][d / 32]; a key's places hold its
              elements in the order [8-element piece of a block][block][8], a value's in [pair of a block][block][2]
  bounds      f16 [page][KV head][min, max][d] over the keys in the page
"""
import math

import torch

own = False

DEV = "cuda"
F16, Q4_0, Q8_0 = 1, 2, 8
TYPES = {"f16": F16, "q8_0": Q8_0, "q4_0": Q4_0}
EPS = 1e-30


# --------------------------------------------------------------------------------------------------- the cases
# n_seq sequences of up to kv keys each, q of them this call's tokens ("mixed": the first sequence alone has q, the others
# one); heads / kv_heads / d: the head layout; page: keys per page
def _case(name, kind, **more):
    base = {"name": name, "kind": kind, "type": "f16", "heads": 32, "kv_heads": 8, "d": 128, "page": 64, "n_seq": 1, "q": 1,
            "kv": 1, "mixed": False, "prefix": 0, "sel": 0, "pos0": 0, "neox": False}
    return {**base, **more}


def listed():
    return [
        # a decode batch's new keys and values, the page bounds kept for a later selection
        _case("append_decode_48", "append", n_seq=48, kv=700),
        # prompt chunks of several requests that go on far into their documents (positions beyond 100000)
        _case("append_prompt_4500", "append", n_seq=5, q=1300, kv=1800, page=16, pos0=100000, neox=True),
        # a decode step over a quantized cache: append, then attention, one after the other
        _case("step_q8_0_32", "step", type="q8_0", n_seq=32, kv=2048),
        # one chat alone on the card
        _case("attn_single_777", "attn", kv=777, page=16),
        # a server's decode batch of conversations of every length
        _case("attn_decode_64", "attn", n_seq=64, kv=4096, page=16),
        # a few very long documents over a quantized cache
        _case("attn_long_q8_0", "attn", type="q8_0", n_seq=3, kv=65536, page=128),
        # prompt chunks of two requests after a past of their own
        _case("attn_prompt_1024", "attn", n_seq=2, q=1024, kv=3000),
        # one request's prompt chunk between the decode steps of the others
        _case("attn_mixed_31", "attn", n_seq=32, q=509, kv=2048, mixed=True),
        # a handful of requests under one system prompt
        _case("shared_8", "shared", n_seq=8, kv=40, prefix=1500, page=16),
        # many short answers over one long document
        _case("shared_128", "shared", n_seq=128, kv=512, prefix=16384),
        # one long conversation, a small part of its pages read, 4-bit cache
        _case("sparse_one_q4_0", "sparse", type="q4_0", kv=8000, page=32, sel=24),
        # a batch of long documents
        _case("sparse_16", "sparse", n_seq=16, kv=32768, sel=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "step", "attn", "attn", "attn", "attn", "shared", "shared", "sparse", "sparse"])
    heads, kvh, d = rng.choice([(32, 8, 128), (32, 8, 128), (20, 5, 128), (16, 2, 128), (8, 8, 128), (16, 4, 64), (12, 1, 64)])
    c = {"kind": kind, "type": rng.choice(["f16", "f16", "q8_0", "q4_0"]), "heads": heads, "kv_heads": kvh, "d": d,
         "page": rng.choice([16, 32, 64, 128])}
    if kind == "append":
        c["type"] = "f16"
        q = rng.choice([1, _log(rng, 2, 1300)])
        n = _log(rng, 1, 64) if q == 1 else max(1, min(8, 4500 // q))
        c.update(n_seq=n, q=q, kv=q + rng.randrange(600), pos0=rng.choice([0, _log(rng, 10, 200000)]), neox=rng.random() < 0.5)
    elif kind == "step":
        c.update(n_seq=_log(rng, 1, 48), kv=_log(rng, 5, 2048), pos0=rng.choice([0, 1000]))
    elif kind == "attn":
        form = rng.choice(["decode", "decode", "few", "prompt", "mixed"])
        if form == "decode":
            n = _log(rng, 1, 64)
            c.update(n_seq=n, kv=_log(rng, 1, min(65536, 262144 // n)))
        elif form == "few":  # a few tokens a sequence: drafted tokens that are checked together
            c.update(n_seq=_log(rng, 1, 32), q=rng.randrange(2, 9), kv=_log(rng, 10, 4096))
        elif form == "prompt":
            q = _log(rng, 16, 1024)
            c.update(n_seq=rng.choice([1, 2]), q=q, kv=q + rng.choice([0, rng.randrange(1900)]))
        else:
            q = _log(rng, 16, 512)
            c.update(n_seq=_log(rng, 2, 32), q=q, kv=max(q, _log(rng, 64, 2048)), mixed=True)
    elif kind == "shared":
        n = _log(rng, 2, 128)
        c.update(n_seq=n, q=rng.choice([1, 1, 1, 3]), kv=_log(rng, 4, 512), prefix=_log(rng, 100, 16384 if n > 8 else 30000))
    else:
        n = _log(rng, 1, 16)
        c.update(n_seq=n, q=rng.choice([1, 1, 1, 2]), kv=_log(rng, 500, 32768), sel=rng.choice([8, 16, 24, 64]))
    return {k: v for k, v in {**_case("", kind), **c}.items() if k != "name"}


# --------------------------------------------------------------------------------------------------- lengths, by the case alone
def _part(i):
    return math.fmod(0.6180339887 * (i + 1), 1.0)


def _lengths(c):
    """(keys, tokens of this call) of each sequence: the first has the most, the others 25 to 100 percent of it."""
    kv = [c["kv"] if i == 0 else max(1, int(c["kv"] * (0.25 + 0.75 * _part(i)))) for i in range(c["n_seq"])]
    q = [c["q"] if i == 0 else 1 if c["mixed"] else max(1, int(c["q"] * (0.25 + 0.75 * _part(i + 7)))) for i in range(c["n_seq"])]
    return kv, [min(a, b) for a, b in zip(q, kv)]


def _pages(n, page):
    return -(-n // page)


def _row_bytes(c):
    return {"f16": 2 * c["d"], "q8_0": c["d"] + c["d"] // 16, "q4_0": c["d"] // 2 + c["d"] // 16}[c["type"]]


def work(c):
    kv, nq = _lengths(c)
    n_tok, h, g, d = sum(nq), c["heads"], c["kv_heads"], c["d"]
    row = _row_bytes(c)
    keys = c["prefix"] + sum(kv)
    pairs = sum(b * (a + c["prefix"]) - b * (b - 1) // 2 for a, b in zip(kv, nq))  # (token, key it may see)
    bounds, select = 0, 0
    if c["kind"] == "sparse":
        pages = [_pages(a, c["page"]) for a in kv]
        keys = sum(min(p, c["sel"] * b) * c["page"] for p, b in zip(pages, nq))
        pairs = sum(b * min(p, c["sel"]) * c["page"] for p, b in zip(pages, nq))
        bounds, select = sum(pages) * g * d * 4, sum(b * p for p, b in zip(pages, nq)) * g * d * 4
    attn = {"bytes": 2 * keys * g * row + 8 * n_tok * h * d + bounds, "flops": 4 * pairs * h * d + select}
    new = sum(_pages(a, c["page"]) - (a - b) // c["page"] for a, b in zip(kv, nq))  # pages that get tokens
    app = {"bytes": n_tok * ((2 * h + 2 * g) * d * 4 + 2 * g * row) + 2 * new * g * d * 4, "flops": 6 * n_tok * (h + g) * d // 2}
    if c["kind"] == "append":
        return app
    if c["kind"] == "step":
        return {"bytes": app["bytes"] - new * g * d * 8 + attn["bytes"] - 4 * n_tok * h * d, "flops": app["flops"] + attn["flops"]}
    return attn


# --------------------------------------------------------------------------------------------------- pools
def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _places(x, of):
    """Integers [..., block, 32] of keys (of "k") or values as places [..., d]."""
    return x.unflatten(-1, (4, 8) if of == "k" else (16, 2)).transpose(-3, -2).flatten(-3)


def _pack(c, x, of):
    """x f32 [page][KV head][key][d], keys (of "k") or values, as the pool of the case's type."""
    if c["type"] == "f16":
        return x.half()
    p, g, s, d = x.shape
    b = x.view(p, g, s, d // 32, 32)
    if c["type"] == "q8_0":
        big = b.abs().amax(-1)
        scale, inv = big / 127, torch.where(big == 0, big, 127 / big)
        q = (b * inv[..., None]).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
        q = _places(q, of).reshape(p, g, s * d)
    else:
        big = b.gather(-1, b.abs().argmax(-1, keepdim=True))[..., 0]
        scale = big / -8
        inv = torch.where(scale == 0, scale, 1 / scale)
        u = _places((b * inv[..., None] + 8.5).to(torch.int32).clamp(0, 15).to(torch.uint8), of)
        q = (u[..., 0::2] | u[..., 1::2] << 4).reshape(p, g, s * d // 2)
    return torch.cat([q, scale.half().view(p, g, -1).contiguous().view(torch.uint8)], -1).contiguous()


def _unpack(c, pool, of, dtype=torch.float32):
    """Pages of a pool [..., KV head, chunk], of keys ("k") or values, as numbers [..., KV head, key, d]."""
    if c["type"] == "f16":
        return pool.to(dtype)
    d, s = c["d"], c["page"]
    n = s * d if c["type"] == "q8_0" else s * d // 2
    lead = pool.shape[:-1]
    scale = pool[..., n:].contiguous().view(torch.float16).view(*lead, s, d // 32, 1).to(dtype)
    if c["type"] == "q8_0":
        q = pool[..., :n].contiguous().view(torch.int8).to(dtype)
    else:
        b = pool[..., :n].unsqueeze(-1)
        q = torch.cat([b & 15, b >> 4], -1).to(dtype) - 8
    q = q.view(*lead, s, *((4, d // 32, 8) if of == "k" else (16, d // 32, 2))).transpose(-3, -2).flatten(-2)
    return (q * scale).view(*lead, s, d)


def prepare(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(7919 * int(seed) + 13)
    kv, nq = _lengths(c)
    h, g, d, page = c["heads"], c["kv_heads"], c["d"], c["page"]
    n_tok, n_seq = sum(nq), c["n_seq"]
    ours = [_pages(a, page) for a in kv]
    pre = _pages(c["prefix"], page)
    n_pages = sum(ours) + pre + 3
    # pages lie anywhere in the pool; entries behind a sequence's last page say none
    order = torch.randperm(n_pages, generator=gen, device=DEV).int()
    table = torch.full((n_seq, max(ours)), -1, dtype=torch.int32, device=DEV)
    at = torch.tensor([sum(ours[:i]) for i in range(n_seq)], device=DEV)
    col = torch.arange(max(ours), device=DEV)
    has = col[None] < torch.tensor(ours, device=DEV)[:, None]
    table[has] = order[(at[:, None] + col[None])[has]]
    s = {"case": c, "n_tok": n_tok, "max_q": max(nq), "max_kv": max(kv), "scale": d ** -0.5}
    s["n_kv"] = torch.tensor(kv, dtype=torch.int32, device=DEV)
    s["cu_q"] = torch.tensor([sum(nq[:i]) for i in range(n_seq + 1)], dtype=torch.int32, device=DEV)
    s["table"] = table
    s["prefix_table"] = order[sum(ours):sum(ours) + pre].clone()
    # keys: a common part, a part of their page (pages differ in what they are about), a part of their own
    x = _randn(gen, n_pages, g, page, d)
    x += 0.5 * _randn(gen, 1, g, 1, d)
    if c["kind"] == "sparse":
        x += 0.7 * _randn(gen, n_pages, g, 1, d)
    s["k"] = _pack(c, x, "k")
    if c["kind"] in ("append", "sparse"):
        x16 = x.half()
        s["bounds"] = torch.stack([x16.amin(2), x16.amax(2)], 2).contiguous()
    s["v"] = _pack(c, _randn(gen, n_pages, g, page, d), "v")
    if c["kind"] in ("append", "step"):
        s["qkv"] = _randn(gen, n_tok, h + 2 * g, d)
    else:
        s["q"] = 1.3 * _randn(gen, n_tok, h, d)
    if c["pos0"]:  # the rotation's positions where they are not the places in the cache
        kq = torch.tensor([a - b for a, b in zip(kv, nq)], device=DEV)
        s["pos"] = (torch.repeat_interleave(kq - s["cu_q"][:-1], torch.tensor(nq, device=DEV)) + torch.arange(n_tok, device=DEV)
                    + c["pos0"]).int()
    if own:
        from ameva_compute_amd import ops
        s["cache"] = ops.PagedKV(TYPES[c["type"]], s["k"], s["v"], page, g, d, bounds=s.get("bounds"))
        s["batch"] = ops.PagedBatch(s["n_kv"], s["table"], s["max_kv"], n_tok, cu_q=s["cu_q"] if n_tok > n_seq else None,
                                    max_q=s["max_q"])
    return s


# --------------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        from ameva_compute_amd import ops
        kv, b = s["cache"], s["batch"]
        if c["kind"] in ("append", "step"):
            q = ops.paged_rope_append(kv, b, s["qkv"], c["heads"], pos=s.get("pos"), mode=2 if c["neox"] else 0, freq_base=500000.0)
            if c["kind"] == "append":
                return [q, s["k"], s["v"], s["bounds"]]
            return [q, ops.paged_attn(kv, b, q, s["scale"])]
        if c["kind"] == "attn":
            return [ops.paged_attn(kv, b, s["q"], s["scale"])]
        if c["kind"] == "shared":
            return [ops.paged_attn_shared(kv, b, s["q"], s["scale"], s["prefix_table"], c["prefix"])]
        sel = ops.paged_select(kv, b, s["q"], c["sel"], n_first=1, n_last=2)
        return [sel, ops.paged_attn_sparse(kv, b, s["q"], sel, s["scale"])]
    if c["kind"] in ("append", "step"):
        q = _append(s, c)
        if c["kind"] == "append":
            return [q, s["k"], s["v"], s["bounds"]]
        return [q, _attend(s, c, q)]
    if c["kind"] in ("attn", "shared"):
        return [_attend(s, c, s["q"])]
    sel = _select(s, c)
    return [sel, _attend_selected(s, c, sel)]


def _tokens(s):
    """Sequence and place in its cache of each token."""
    cu = s["cu_q"].long()
    seq = torch.repeat_interleave(cu[1:] - cu[:-1], output_size=s["n_tok"])
    return seq, s["n_kv"].long()[seq] - cu[1:][seq] + torch.arange(s["n_tok"], device=DEV)


def _append(s, c):
    h, g, d, page = c["heads"], c["kv_heads"], c["d"], c["page"]
    seq, place = _tokens(s)
    pos = s.get("pos", place).double()
    # angles, their cosines and the rotation in 64 bits: a far position's angle has lost its fraction in 32, and a key that
    # lies next to a rounding border of its stored type goes to the side where it belongs
    ang = pos[:, None] * torch.pow(torch.tensor(500000.0, dtype=torch.float64, device=DEV),
                                   torch.arange(d // 2, dtype=torch.float64, device=DEV) * (-2.0 / d))
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    x = s["qkv"][:, :h + g].double()
    a, b = (x[..., :d // 2], x[..., d // 2:]) if c["neox"] else (x[..., 0::2], x[..., 1::2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    x = (torch.cat([ra, rb], -1) if c["neox"] else torch.stack([ra, rb], -1).flatten(-2)).float()
    q, k, v = x[:, :h].contiguous(), x[:, h:], s["qkv"][:, h + g:]
    at, slot = s["table"][seq, place // page].long(), place % page
    if c["type"] == "f16":
        s["k"][at, :, slot] = k.half()
        s["v"][at, :, slot] = v.half()
    else:
        for of, new in (("k", k), ("v", v)):
            pool, one = s[of], _pack(c, new[:, :, None].contiguous(), of)  # [token][KV head][integers | scales]
            ni = d if c["type"] == "q8_0" else d // 2
            n = pool.shape[-1] // (ni + d // 16) * ni
            col = slot[:, None, None]
            head = torch.arange(g, device=DEV)[None, :, None]
            pool[at[:, None, None], head, col * ni + torch.arange(ni, device=DEV)] = one[..., :ni]
            pool[at[:, None, None], head, n + col * (d // 16) + torch.arange(d // 16, device=DEV)] = one[..., ni:]
    if "bounds" in s:
        k16, low, high = k.half(), s["bounds"][:, :, 0], s["bounds"][:, :, 1]
        begun = at[slot == 0]
        low[begun], high[begun] = math.inf, -math.inf
        where = at[:, None, None].expand_as(k16)
        low.scatter_reduce_(0, where, k16, "amin")
        high.scatter_reduce_(0, where, k16, "amax")
    return q


def _softmax_parts(scores, see, v):
    """Maximum, sum and weighted values of scores [.., rows, keys] where see, v [.., keys, d]."""
    scores = scores.masked_fill(~see, -math.inf)
    m = scores.amax(-1, keepdim=True)
    e = (scores - m.masked_fill(m == -math.inf, 0.0)).exp()
    return m, e.sum(-1, keepdim=True), e @ v


def _attend(s, c, q):
    h, g, d, page = c["heads"], c["kv_heads"], c["d"], c["page"]
    n, cu = c["n_seq"], s["cu_q"].long()
    nq, n_kv, mq = cu[1:] - cu[:-1], s["n_kv"].long(), s["max_q"]
    t = torch.arange(mq, device=DEV)
    tok, has = cu[:-1, None] + t, t < nq[:, None]
    rows = (q[tok.clamp(max=s["n_tok"] - 1)] * s["scale"]).view(n, mq, g, h // g, d).permute(0, 2, 1, 3, 4).reshape(n, g, -1, d)
    k, v = (_unpack(c, s[p][s["table"].clamp(min=0).long()], p).transpose(1, 2).reshape(n, g, -1, d) for p in "kv")
    key = torch.arange(k.shape[2], device=DEV)
    there = key < n_kv[:, None]
    k, v = (x.masked_fill(~there[:, None, :, None], 0.0) for x in (k, v))
    place = (n_kv - nq)[:, None] + t
    see = (key <= place[..., None]) & there[:, None]  # [sequence][token][key]
    see = see.repeat_interleave(h // g, 1)[:, None]
    m, l, o = _softmax_parts(rows @ k.transpose(-1, -2).contiguous(), see, v)
    if c["prefix"]:
        pk, pv = (_unpack(c, s[p][s["prefix_table"].long()], p).transpose(0, 1).reshape(g, -1, d)[:, :c["prefix"]] for p in "kv")
        all_rows = rows.transpose(0, 1).reshape(g, -1, d)
        pm, pl, po = _softmax_parts(all_rows @ pk.transpose(-1, -2).contiguous(), torch.ones((), dtype=torch.bool, device=DEV), pv)
        pm, pl, po = (x.view(g, n, -1, x.shape[-1]).transpose(0, 1) for x in (pm, pl, po))
        top = torch.maximum(m, pm)
        a, b = (m - top).exp(), (pm - top).exp()
        l, o = l * a + pl * b, o * a + po * b
    o = (o / l.clamp(min=EPS)).view(n, g, mq, h // g, d).permute(0, 2, 1, 3, 4).reshape(n, mq, h, d)
    return o[has]


def _select(s, c):
    h, g, d = c["heads"], c["kv_heads"], c["d"]
    seq, place = _tokens(s)
    n_pages = place // c["page"] + 1  # those that hold a key the token may see
    # sum over the group's heads of the largest q . k that the page's bounds allow, in 64 bits: pages next to the border
    q = s["q"].view(-1, g, h // g, d).double()
    up, down = q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)
    b = s["bounds"][s["table"].clamp(min=0).long()].double()[seq]  # [token][page][KV head][2][d]
    score = ((b[..., 1, :] * up[:, None]).sum(-1) + (b[..., 0, :] * down[:, None]).sum(-1)).transpose(1, 2)
    col = torch.arange(score.shape[-1], device=DEV)
    n = n_pages[:, None, None]
    score = score.masked_fill((col < 1) | (col >= n - 2), math.inf).masked_fill(col >= n, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True)[1][..., :c["sel"]]
    order = order.masked_fill(order >= n, score.shape[-1]).sort(-1)[0]
    sel = torch.full((s["n_tok"], g, c["sel"]), -1, dtype=torch.int32, device=DEV)
    sel[..., :order.shape[-1]] = order.masked_fill(order >= n, -1).int()
    return sel


def _attend_selected(s, c, sel):
    h, g, d, page = c["heads"], c["kv_heads"], c["d"], c["page"]
    seq, place = _tokens(s)
    t = s["n_tok"]
    at = s["table"][seq[:, None, None], sel.clamp(min=0).long()].clamp(min=0).long()  # [token][KV head][selected]
    head = torch.arange(g, device=DEV)[None, :, None]
    k, v = (_unpack(c, s[p][at, head], p).view(t, g, -1, d) for p in "kv")
    key = (sel[..., None] * page + torch.arange(page, device=DEV)).view(t, g, -1)
    see = ((key <= place[:, None, None]) & (key >= 0))[:, :, None]
    k, v = (x.masked_fill(~see.transpose(-1, -2), 0.0) for x in (k, v))
    m, l, o = _softmax_parts((s["q"] * s["scale"]).view(t, g, h // g, d) @ k.transpose(-1, -2).contiguous(), see, v)
    return (o / l.clamp(min=EPS)).view(t, h, d)


# --------------------------------------------------------------------------------------------------- in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    h, g, d, page = c["heads"], c["kv_heads"], c["d"], c["page"]
    kv, nq = _lengths(c)
    kval, vval = (_unpack(c, s[p], p, torch.float64) if c["kind"] == "step" else None for p in "kv")
    table = s["table"].long()

    def rows(p, pages, head, n):  # the first n keys or values of a list of pages, one KV head
        if kval is not None:
            return (kval if p == "k" else vval)[pages, head].reshape(-1, d)[:n]
        return _unpack(c, s[p][pages, head], p, torch.float64).reshape(-1, d)[:n]

    out, first = [], 0
    q_all = []
    if c["kind"] in ("append", "step"):
        bounds = s["bounds"].double() if "bounds" in s else None
        for i in range(c["n_seq"]):
            for j0 in range(0, nq[i], 256):
                j1 = min(nq[i], j0 + 256)
                places = torch.arange(kv[i] - nq[i] + j0, kv[i] - nq[i] + j1, device=DEV)
                freq = torch.exp(torch.arange(0, d, 2, dtype=torch.float64, device=DEV) * (-math.log(500000.0) / d))
                turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), (places + c["pos0"]).double()[:, None] * freq)[:, None]
                x = s["qkv"][first + j0:first + j1].double()
                if c["neox"]:
                    z = torch.complex(x[:, :h + g, :d // 2].contiguous(), x[:, :h + g, d // 2:].contiguous()) * turn
                    r = torch.cat([z.real, z.imag], -1)
                else:
                    z = torch.view_as_complex(x[:, :h + g].reshape(j1 - j0, h + g, d // 2, 2).contiguous()) * turn
                    r = torch.view_as_real(z).flatten(-2)
                q_all.append(r[:, :h])
                pg, sl = table[i, places // page], places % page
                new = [r[:, h:].float(), x[:, h + g:].float()]
                if c["kind"] == "append":
                    s["k"][pg, :, sl], s["v"][pg, :, sl] = new[0].half(), new[1].half()
                    for p in sorted(set((places // page).tolist())):
                        mine = new[0][places // page == p].half().double()
                        at, old = table[i, p], p * page < kv[i] - nq[i] + j0
                        low, high = mine.amin(0), mine.amax(0)
                        bounds[at, :, 0] = torch.minimum(bounds[at, :, 0], low) if old else low
                        bounds[at, :, 1] = torch.maximum(bounds[at, :, 1], high) if old else high
                else:
                    kval[pg, :, sl], vval[pg, :, sl] = (_unpack({**c, "page": 1}, _pack(c, y[:, :, None].contiguous(), p), p, torch.float64)[:, :, 0]
                                                        for y, p in zip(new, "kv"))
            first += nq[i]
        q = torch.cat(q_all)
        if c["kind"] == "append":
            return [q, s["k"].double(), s["v"].double(), bounds]
        q_for = q.float().double()  # what the attention is given
    else:
        q = q_for = s["q"].double()
    sels = [] if c["kind"] == "sparse" else None
    first = 0
    pk = [[rows(p, s["prefix_table"].long(), j, c["prefix"]) for j in range(g)] for p in "kv"] if c["prefix"] else None
    for i in range(c["n_seq"]):
        mine = q_for[first:first + nq[i]]
        first += nq[i]
        pages = table[i, :_pages(kv[i], page)]
        place = torch.arange(kv[i] - nq[i], kv[i], device=DEV)
        o = torch.empty(nq[i], h, d, dtype=torch.float64, device=DEV)
        picked = torch.full((nq[i], g, c["sel"]), -1, dtype=torch.int64, device=DEV)
        for j in range(g):
            k, v = rows("k", pages, j, kv[i]), rows("v", pages, j, kv[i])
            see = torch.arange(kv[i], device=DEV)[None] <= place[:, None]
            if sels is not None:
                b = s["bounds"][pages, j].double()
                for t in range(nq[i]):
                    n = int(place[t]) // page + 1
                    score = sum(torch.maximum(mine[t, e] * b[:n, 0], mine[t, e] * b[:n, 1]).sum(-1) for e in range(j * (h // g), (j + 1) * (h // g)))
                    score[0] = math.inf
                    score[max(0, n - 2):] = math.inf
                    got = score.sort(dim=-1, descending=True, stable=True)[1][:c["sel"]].sort()[0]
                    picked[t, j, :got.numel()] = got
                    keep = torch.zeros(pages.numel(), dtype=torch.bool, device=DEV)
                    keep[got] = True
                    see[t] &= keep.repeat_interleave(page)[:kv[i]]
            if pk:
                k, v = torch.cat([pk[0][j], k]), torch.cat([pk[1][j], v])
                see = torch.cat([torch.ones(nq[i], c["prefix"], dtype=torch.bool, device=DEV), see], 1)
            for e in range(j * (h // g), (j + 1) * (h // g)):
                w = (mine[:, e] @ k.T * c["d"] ** -0.5).masked_fill(~see, -math.inf).softmax(-1)
                o[:, e] = w @ v
        out.append(o)
        if sels is not None:
            sels.append(picked)
    out = torch.cat(out)
    return [q, out] if c["kind"] == "step" else [torch.cat(sels).int(), out] if sels is not None else [out]
