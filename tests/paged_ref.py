"""Plain 64-bit forms of the paged KV cache operators, and pools to try them on. A pool here is a PagedKV with the numbers that it
stands for beside it (f64 [page, KV head, key, d]); whatever no key owns holds values that must not matter."""
import math

import torch

F16, Q4_0, Q8_0 = 1, 2, 8
DEV = "cuda"


def places(x, of):
    """Integers [..., blocks, 32] of keys ("k") or values ("v") in a chunk's order [..., d]."""
    return x.unflatten(-1, (4, 8) if of == "k" else (16, 2)).transpose(-3, -2).flatten(-3)


def quantize(x, t, rule=0):
    """f32 [..., d] -> (integers [..., d / 32, 32], scales f32 [..., d / 32]) by ggml's rules, in 32-bit arithmetic."""
    b = x.unflatten(-1, (-1, 32))
    if t == Q8_0:
        big = b.abs().amax(-1)
        d = big / 127
        inv = torch.where(big == 0, big, 127 / big) if rule == 0 else torch.where(d == 0, d, 1 / d)
        q = b * inv[..., None]
        q = torch.where(q < 0, (q - 0.5).ceil(), (q + 0.5).floor()) if rule == 2 else q.round()
        return q.clamp(-127, 127).int(), d
    first = (b.abs() == b.abs().amax(-1, keepdim=True)).int().argmax(-1, keepdim=True)
    d = b.gather(-1, first)[..., 0] / -8
    inv = torch.where(d == 0, d, 1 / d)
    return (b * inv[..., None] + 8.5).int().clamp(0, 15) - 8, d


def pack(x, t, of, rule=0):
    """f32 [pages, KV head, key, d] as (a pool's tensor of type t, the numbers it stands for in f64)."""
    if t == F16:
        return x.half(), x.half().double()
    p, g, s, d = x.shape
    q, scale = quantize(x, t, rule)
    scale = scale.half()
    value = (q.double() * scale.double()[..., None]).flatten(-2)
    q = places(q, of)
    q = (q & 0xFF) if t == Q8_0 else (q[..., 0::2] + 8) | (q[..., 1::2] + 8) << 4
    q = q.to(torch.uint8).reshape(p, g, -1)
    return torch.cat([q, scale.reshape(p, g, -1).contiguous().view(torch.uint8)], -1).contiguous(), value


def unpack(pool, t, of, s, d):
    if t == F16:
        return pool.double()
    p, g, _ = pool.shape
    n = s * d if t == Q8_0 else s * d // 2
    scale = pool[..., n:].contiguous().view(torch.float16).view(p, g, s, d // 32, 1).double()
    q = pool[..., :n].contiguous()
    q = q.view(torch.int8).double() if t == Q8_0 else torch.stack([q & 15, q >> 4], -1).double() - 8
    q = q.reshape(p, g, s, *((4, d // 32, 8) if of == "k" else (16, d // 32, 2))).transpose(-3, -2).flatten(-2)
    return (q * scale).reshape(p, g, s, d)


class World:
    """Sequences of n_kv keys, n_q of them this call's tokens, in scattered pages; `spare` pages belong to nobody, rows behind a
    sequence's last key hold infinities (F16) or the largest scales."""

    def __init__(self, t, g, d, page, n_kv, n_q=None, seed=0, bounds=False, spare=2, k_gain=1.0, v_gain=1.0, extra=0):
        from ameva_compute_amd import ops
        gen = torch.Generator(device=DEV)
        gen.manual_seed(seed)
        self.t, self.g, self.d, self.page = t, g, d, page
        self.n_kv, self.n_q = list(n_kv), [1] * len(n_kv) if n_q is None else list(n_q)
        count = [-(-max(n, 0) // page) for n in n_kv]
        n_pages = sum(count) + spare + extra
        order = torch.randperm(n_pages, generator=gen, device=DEV).int()
        self.rand = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
        x, y = self.rand(n_pages, g, page, d) * k_gain, self.rand(n_pages, g, page, d) * v_gain
        k, self.k = pack(x, t, "k")
        v, self.v = pack(y, t, "v")
        owned = torch.zeros(n_pages, page, dtype=torch.bool, device=DEV)
        self.table = torch.full((len(n_kv), max(count + [1])), -1, dtype=torch.int32, device=DEV)
        at = 0
        for s, n in enumerate(count):
            self.table[s, :n] = order[at:at + n]
            for j in range(n):
                owned[order[at + j].long(), :max(0, min(page, n_kv[s] - j * page))] = True
            at += n
        self.free = order[at:]
        owned[self.free[:extra].long()] = True
        gone = ~owned[:, None, :, None].expand(-1, g, -1, d)
        if t == F16:
            k[gone], v[gone] = math.nan, math.inf
        else:
            ni = page * d // (1 if t == Q8_0 else 2)
            for p in (k, v):
                scale = p[..., ni:].view(torch.float16).view(n_pages, g, page, d // 32)
                scale[~owned[:, None, :, None].expand_as(scale)] = math.nan
        b = None
        if bounds:
            x16 = x.half().masked_fill(gone, math.inf)
            b = torch.stack([x16.amin(2), x.half().masked_fill(gone, -math.inf).amax(2)], 2).contiguous()
        self.cache = ops.PagedKV(t, k, v, page, g, d, bounds=b)
        ends = [0]
        for n in self.n_q:
            ends.append(ends[-1] + n)
        self.first = ends
        self.cu_q = torch.tensor(ends, dtype=torch.int32, device=DEV)
        self.n_kv_dev = torch.tensor(self.n_kv, dtype=torch.int32, device=DEV)

    def batch(self, max_kv=None, pad=0, one=None):
        from ameva_compute_amd import ops
        one = all(n == 1 for n in self.n_q) and not pad if one is None else one
        return ops.PagedBatch(self.n_kv_dev, self.table, max(max(self.n_kv), 0) if max_kv is None else max_kv, self.first[-1] + pad,
                              cu_q=None if one else self.cu_q, max_q=max(self.n_q + [1]))

    def rows(self, what, s, head, n=None):
        n = max(self.n_kv[s], 0) if n is None else n
        return what[self.table[s, :-(-n // self.page)].long(), head].reshape(-1, self.d)[:n]


def attend(w, q, scale, prefix=None, see=None):
    """Attention in f64: q [n_tok, heads, d]; prefix (k, v) f64 [KV head, n, d]; see(s, i, KV head) -> truth per own key, on top of the
    causal rule. Rows that belong to no sequence are NaN."""
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    G = q.shape[1] // w.g
    for s, (n_kv, n_q) in enumerate(zip(w.n_kv, w.n_q)):
        if n_q == 0:
            continue
        mine = q[w.first[s]:w.first[s] + n_q].double()
        place = torch.arange(n_kv - n_q, n_kv, device=q.device)
        for j in range(w.g):
            k, v = w.rows(w.k, s, j), w.rows(w.v, s, j)
            ok = torch.arange(k.shape[0], device=q.device)[None] <= place[:, None]
            if see is not None:
                ok = ok & torch.stack([see(s, i, j) for i in range(n_q)])
            if prefix is not None:
                k, v = torch.cat([prefix[0][j], k]), torch.cat([prefix[1][j], v])
                ok = torch.cat([torch.ones(n_q, prefix[0].shape[1], dtype=torch.bool, device=q.device), ok], 1)
            x = (mine[:, j * G:(j + 1) * G].transpose(0, 1) @ k.T * scale).masked_fill(~ok, -math.inf)
            p = torch.nan_to_num((x - x.amax(-1, keepdim=True).clamp(min=-1e300)).exp()) if k.shape[0] else x
            o = p @ v / p.sum(-1, keepdim=True).clamp(min=1e-300)
            out[w.first[s]:w.first[s] + n_q, j * G:(j + 1) * G] = o.transpose(0, 1)
    return out


def off(y, r):
    """Relative error in the 2-norm."""
    n = r.norm().item()
    return ((y.double() - r).norm().item() / n) if n else y.double().norm().item()
