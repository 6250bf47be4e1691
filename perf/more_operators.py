"""The operators of a mixture of experts' feed-forward part, measured over the ranges a server has: the residual's addition with the
norm and its 8-bit output, the routing of tokens to experts, the experts' gate and up products with SWIGLU and its 8-bit output, and
their down product summed with the routing's weights.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what a program holds before the call, run()
is one pass (own: through ameva_compute_amd.ops, else in elementary torch operations), work() what the pass cannot do
without, exact() its outputs in 64 bits. Weights and activations are made here, in plain torch, in the layouts that
include/ameva_hip.h describes; an expert's matrix is one repacked weight, the experts lie one after the other:

  Q4_0  qs [n][k/32][16] (byte i: elements i and 16 + i, value + 8) | scales f16 [n/2][k/32][2]
  Q8_0  qs int8 [n][k/32][32] | scales f16 [n][k/32]
  Q4_K  qs [n][k/256][128] | heads [n][k/256][16]: d, dmin f16, 8 scales and 8 mins of 6 bits
  Q6_K  ql [n][k/256][128] | qh [..][64] | scales int8 [..][16] | d f16
  activations  Q8_0: int8 [m][k] | {f32 d, i32 sum} [m][k/32]; Q8_K: int8 [m][k] | f32 d [m][k/256] | i32 sums [m][k/16]
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"q4_0": 2, "q8_0": 8, "q4_k": 12, "q6_k": 14, "q8_k": 15}
EPS = 1e-5


def _act_of(wtype):
    return "q8_k" if wtype in ("q4_k", "q6_k") else "q8_0"


# --------------------------------------------------------------------------------------------------- the cases
# tokens; n: row length (norm); experts, used: of the routing; k, rows: an expert matrix is rows x k (gate and up have `rows` each);
# type: of the experts' weights; act: of the 8-bit output; pad: tokens at the end that go to no expert (a padded batch)
def _case(name, kind, **more):
    base = {"name": name, "kind": kind, "tokens": 1, "n": 4096, "experts": 128, "used": 8, "k": 2048, "rows": 1024, "type": "q4_0",
            "act": "q8_0", "pad": 0, "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_best": 1, "renorm": True,
            "scale": 1.0, "residual": False}
    return {**base, **more}


def listed():
    return [
        # one token of a decode step
        _case("norm_decode_1", "norm", n=4096),
        # a prompt chunk before experts in K-quants
        _case("norm_prompt_4096", "norm", tokens=4096, n=4096, act="q8_k"),
        # the router of a decode step
        _case("route_decode_1", "route"),
        # a prompt's router with balanced experts in groups
        _case("route_groups_4096", "route", tokens=4096, experts=256, score="sigmoid", bias=True, groups=8, top_groups=4, group_best=2,
              scale=2.5),
        # one token, many small experts
        _case("gate_up_decode_1", "gate_up", type="q4_k", act="q8_k"),
        # a server's decode batch, part of it padding
        _case("gate_up_batch_48", "gate_up", tokens=48, experts=64, pad=3),
        # a prompt chunk of odd size, rows of an odd number of blocks, the number of experts no power of two
        _case("gate_up_odd_331", "gate_up", tokens=331, experts=60, used=4, k=2080, rows=1408, type="q8_0"),
        # a long prompt
        _case("gate_up_prompt_4096", "gate_up", tokens=4096),
        # one token, few large experts
        _case("down_decode_1", "down", experts=8, used=2, k=14336, rows=4096, type="q6_k", residual=True),
        # a decode batch
        _case("down_batch_40", "down", tokens=40, experts=64, k=1408, rows=2048, type="q8_0", residual=True),
        # a prompt chunk over few large experts
        _case("down_prompt_600", "down", tokens=600, experts=8, used=2, k=6144, rows=4096, type="q4_0"),
        # a long prompt
        _case("down_prompt_4096", "down", tokens=4096, k=1024, rows=2048, type="q4_k", residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "route", "route", "gate_up", "gate_up", "gate_up", "down", "down", "down"])
    tokens = rng.choice([1, _log(rng, 2, 64), _log(rng, 2, 64), _log(rng, 16, 4096)])
    c = {"kind": kind, "tokens": tokens}
    if kind == "norm":
        c.update(act=rng.choice(["q8_0", "q8_k"]), n=256 * rng.randrange(2, 25))
        if c["act"] == "q8_0":
            c["n"] += 32 * rng.randrange(8)
        c["tokens"] = min(tokens, 16 * 2 ** 20 // c["n"])
    elif kind == "route":
        e = rng.choice([8, 16, 60, 64, 128, 160, 256])
        c.update(experts=e, used=min(e, rng.choice([1, 2, 4, 6, 8])), score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                 renorm=rng.random() < 0.7, scale=rng.choice([1.0, 1.0, 2.5]))
        if e % 32 == 0 and rng.random() < 0.5:
            c.update(groups=8, top_groups=rng.choice([3, 4]), group_best=rng.choice([1, 2]))
            c["used"] = min(c["used"], c["top_groups"] * e // 8)
    else:
        wtype = rng.choice(["q4_0", "q8_0", "q4_k", "q6_k"])
        unit = 256 if wtype in ("q4_k", "q6_k") else 32
        e, used = rng.choice([(8, 2), (16, 2), (32, 4), (60, 4), (64, 6), (64, 8), (128, 8)])
        k, rows = max(1, _log(rng, 512, 6144) // unit) * unit, max(1, _log(rng, 512, 4096) // 32) * 32
        if kind == "gate_up":
            c["act"] = rng.choice(["q8_0", "q8_k"])
            rows = max(1, _log(rng, 512, 2048) // 256) * 256 if c["act"] == "q8_k" else max(1, _log(rng, 512, 2048) // 32) * 32
        per = 2 if kind == "gate_up" else 1
        e, used = (e, used) if e * rows * k * per < 2 ** 30 else (8, 2)  # (the plain form holds the experts in 32 bits)
        rows = rows if e * rows * k * per < 2 ** 30 else rows // 512 * 256
        c["tokens"] = max(1, min(tokens, int(1.3e11 / (2 * used * rows * k * per))))
        c.update(type=wtype, experts=e, used=used, k=k, rows=rows, residual=kind == "down" and rng.random() < 0.5,
                 pad=rng.choice([0, 0, c["tokens"] // 10]))
    return {a: b for a, b in {**_case("", kind), **c}.items() if a != "name"}


def _row_bytes(wtype, k):
    return {"q4_0": k // 32 * 18, "q8_0": k // 32 * 34, "q4_k": k // 256 * 144, "q6_k": k // 256 * 210, "act_q8_0": k + k // 4,
            "act_q8_k": k + k // 64 + k // 4}[wtype]


def work(c):
    t, n, e, u, k, rows = c["tokens"], c["n"], c["experts"], c["used"], c["k"], c["rows"]
    if c["kind"] == "norm":
        return {"bytes": t * (16 * n + _row_bytes("act_" + c["act"], n)) + 4 * n, "flops": 8 * t * n}
    if c["kind"] == "route":
        return {"bytes": 4 * t * e + 8 * t * u, "flops": 12 * t * e}
    live = t - c["pad"]
    read = e * (1 - (1 - u / e) ** live)  # experts that some token goes to, when they are chosen evenly
    act = _row_bytes("act_" + _act_of(c["type"]), k)
    if c["kind"] == "gate_up":
        return {"bytes": read * 2 * rows * _row_bytes(c["type"], k) + t * act + t * u * (4 + _row_bytes("act_" + c["act"], rows)),
                "flops": 4 * live * u * rows * k}
    return {"bytes": read * rows * _row_bytes(c["type"], k) + t * u * (8 + act) + 4 * t * rows * (2 if c["residual"] else 1),
            "flops": 2 * live * u * rows * k}


# --------------------------------------------------------------------------------------------------- weights and activations
def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _bytes(gen, *shape):
    return torch.randint(0, 256, shape, generator=gen, device=DEV, dtype=torch.uint8)


def _raw(x):
    return x.contiguous().view(torch.uint8).flatten(1)


def _experts(gen, wtype, e, n, k):
    """Random weights [e][bytes of one matrix] whose values are about k^-1/2 in size."""
    s = k ** -0.5
    if wtype in ("q4_0", "q8_0"):
        b = k // 32
        q = _bytes(gen, e, n * b * (16 if wtype == "q4_0" else 32))
        d = (0.8 + 0.4 * torch.rand(e, n * b, generator=gen, device=DEV)) * s / (4.6 if wtype == "q4_0" else 74)
        return torch.cat([q, _raw(d.half())], 1)
    b = n * (k // 256)
    if wtype == "q4_k":  # scales about 31, integers about 7.5, so a min takes what the integers' mean brings in
        d = (0.8 + 0.4 * torch.rand(e, b, 1, generator=gen, device=DEV)) * s / 190
        head = torch.cat([torch.cat([d, 7.5 * d], 2).half().view(torch.uint8), _bytes(gen, e, b, 12)], 2)
        return torch.cat([_bytes(gen, e, b * 128), head.flatten(1)], 1)
    d = (0.8 + 0.4 * torch.rand(e, b, generator=gen, device=DEV)) * s / 1360
    return torch.cat([_bytes(gen, e, b * 208), _raw(d.half())], 1)


def _numbers(wtype, w, n, k):
    """The weights [matrices][bytes] as f32 [matrices][n][k]."""
    e = w.shape[0]
    if wtype == "q4_0":
        b = k // 32
        q = w[:, :n * b * 16].reshape(e, n, b, 1, 16)
        q = torch.cat([q & 15, q >> 4], 3).flatten(3).float() - 8
        d = w[:, n * b * 16:].contiguous().view(torch.float16).view(e, n // 2, b, 2).transpose(2, 3).reshape(e, n, b, 1)
        return (q * d.float()).view(e, n, k)
    if wtype == "q8_0":
        b = k // 32
        q = w[:, :n * k].contiguous().view(torch.int8).view(e, n, b, 32)
        return (q.float() * w[:, n * k:].contiguous().view(torch.float16).view(e, n, b, 1).float()).view(e, n, k)
    b = n * (k // 256)
    if wtype == "q4_k":
        q = w[:, :b * 128].reshape(e, b, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], 3).flatten(2, 3).float()  # [unit][32]
        head = w[:, b * 128:].reshape(e, b, 16)
        d = head[..., :4].contiguous().view(torch.float16).float()
        lo, mid, hi = head[..., 4:8], head[..., 8:12], head[..., 12:16]
        sc = torch.cat([lo & 63, (hi & 15) | ((lo >> 6) << 4)], 2).float()
        mn = torch.cat([mid & 63, (hi >> 4) | ((mid >> 6) << 4)], 2).float()
        return (q * (d[..., :1] * sc)[..., None] - (d[..., 1:] * mn)[..., None]).view(e, n, k)
    ql, qh = w[:, :b * 128].reshape(e, b, 2, 1, 2, 32), w[:, b * 128:b * 192].reshape(e, b, 2, 1, 32)
    low = torch.cat([ql & 15, ql >> 4], 3).flatten(3, 4)  # [half][quarter][32]
    high = torch.cat([(qh >> s) & 3 for s in (0, 2, 4, 6)], 3)
    q = (low | (high << 4)).float() - 32
    sc = w[:, b * 192:b * 208].contiguous().view(torch.int8).float() * w[:, b * 208:].contiguous().view(torch.float16).float().repeat_interleave(16, 1)
    return (q.reshape(e, b, 16, 16) * sc.view(e, b, 16, 1)).view(e, n, k)


def _quantize(x, atype):
    """Rows of x as integers and block scales: (f32 integers [m][blocks][block], f32 scales [m][blocks]), ggml's rules."""
    b = x.view(x.shape[0], -1, 32 if atype == "q8_0" else 256)
    if atype == "q8_0":
        big = b.abs().amax(-1)
        inv = torch.where(big == 0, big, 127 / big)
        return (b * inv[..., None]).round().clamp(-127, 127), (big / 127).half().to(x.dtype)
    big = b.gather(-1, b.abs().argmax(-1, keepdim=True))[..., 0]
    inv = torch.where(big == 0, big, -127 / big)
    return (b * inv[..., None]).round().clamp(max=127), torch.where(big == 0, big, 1 / inv)


def _store(x, atype):
    """An activation buffer that holds the rows of x."""
    q, d = _quantize(x, atype)
    m = x.shape[0]
    if atype == "q8_0":
        meta = torch.stack([d, q.sum(-1).int().view(torch.float32)], -1)
    else:
        meta = torch.cat([d.flatten(), q.view(m, -1, 16).sum(-1).int().view(torch.float32).flatten()])
    return torch.cat([q.to(torch.int8).view(torch.uint8).flatten(), meta.contiguous().view(torch.uint8).flatten()])


def _values(act, atype, m, k):
    """The numbers an activation buffer of m rows of k stands for, f32 [m][k]."""
    q = act[:m * k].view(torch.int8).view(m, k).float()
    if atype == "q8_0":
        d = act[m * k:].view(torch.float32).view(m, k // 32, 2)[..., :1]
        return (q.view(m, -1, 32) * d).view(m, k)
    return (q.view(m, -1, 256) * act[m * k:m * k + m * k // 64].view(torch.float32).view(m, -1, 1)).view(m, k)


def prepare(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(7919 * int(seed) + 29)
    t, e, u = c["tokens"], c["experts"], c["used"]
    s = {"case": c}
    if c["kind"] == "norm":
        s["x"], s["r"] = _randn(gen, t, c["n"]), 2 * _randn(gen, t, c["n"])
        s["w"] = 1 + 0.2 * _randn(gen, c["n"])
        return s
    # experts differ in how often they are chosen
    logits = 1.5 * _randn(gen, t, e) + 0.7 * _randn(gen, e)
    if c["kind"] == "route":
        s["logits"] = logits
        s["bias"] = 0.1 * _randn(gen, e) if c["bias"] else None
        return s
    chosen = logits.topk(u, dim=1)
    ids = chosen[1].int()
    ids[t - c["pad"]:] = -1
    s["ids"], s["weights"] = ids.contiguous(), chosen[0].softmax(1)
    host = ids.flatten().cpu()
    s["most"] = int(torch.bincount(host[host >= 0], minlength=e).max()) if (host >= 0).any() else 1  # rows of the busiest expert
    k, rows, at = c["k"], c["rows"], _act_of(c["type"])
    if c["kind"] == "gate_up":
        s["gate"], s["up"] = (_experts(gen, c["type"], e, rows, k) for _ in range(2))
        s["act"] = _store(_randn(gen, t, k), at)
    else:
        s["down"] = _experts(gen, c["type"], e, rows, k)
        # SWIGLU's outputs: many small values, a few large ones
        g = 1.2 * _randn(gen, t * u, k)
        s["act"] = _store(g * g.sigmoid() * _randn(gen, t * u, k), at)
        s["add"] = _randn(gen, t, rows) if c["residual"] else None
    if own:
        from ameva_compute_amd import ops
        for name in ("gate", "up", "down"):
            if name in s:
                s[name] = ops.QExperts(TYPES[c["type"]], e, rows, k, s[name])
        if c["kind"] == "down":
            s["plan"] = ops.moe_plan(s["ids"], e)  # the gate and up products before it were made with the same one
    return s


# --------------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        from ameva_compute_amd import ops
        if c["kind"] == "norm":
            at = TYPES[c["act"]]
            total, y, act = ops.add_rms_norm(s["x"], s["r"], EPS, s["w"], act_type=at)
            return [total, y, ops.act_values(act, at, c["tokens"], c["n"])]
        if c["kind"] == "route":
            ids, weights = ops.moe_route(s["logits"], c["used"], score=c["score"], bias=s["bias"], n_group=c["groups"],
                                         top_group=c["top_groups"], group_best=c["group_best"], renorm=c["renorm"], scale=c["scale"])
            return [ids, weights]
        if c["kind"] == "gate_up":
            at = TYPES[c["act"]]
            plan = ops.moe_plan(s["ids"], c["experts"])
            act = ops.moe_gate_up(s["gate"], s["up"], s["act"], plan, act_type=at)
            return [ops.act_values(act, at, c["tokens"] * c["used"], c["rows"])]
        return [ops.moe_down(s["down"], s["act"], s["plan"], s["weights"], add=s["add"])]
    if c["kind"] == "norm":
        total = s["x"] + s["r"]
        # the mean in 64 bits: a scale that is off by its last bit moves integers that lie next to a border
        y = total * (1 / ((total * total).double().mean(1, keepdim=True).float() + EPS).sqrt()) * s["w"]
        return [total, y, _rounded(y, c["act"])]
    if c["kind"] == "route":
        return _route(s, c)
    if c["kind"] == "gate_up":
        g, u = (_products(s, c, s[name], _values(s["act"], _act_of(c["type"]), c["tokens"], c["k"]), c["used"]) for name in ("gate", "up"))
        return [_rounded(g / (1 + (-g).exp()) * u, c["act"])]
    y = _products(s, c, s["down"], _values(s["act"], _act_of(c["type"]), c["tokens"] * c["used"], c["k"]), 1)
    y = (y.view(c["tokens"], c["used"], -1) * s["weights"][..., None]).sum(1)
    return [y if s["add"] is None else y + s["add"]]


def _rounded(x, atype):
    q, d = _quantize(x, atype)
    return (q * d[..., None]).half().view(x.shape)


def _route(s, c):
    # scores in 64 bits: which of two close ones is the larger decides over an expert
    logits, t, e = s["logits"].double(), c["tokens"], c["experts"]
    if c["score"] == "softmax":
        p = (logits - logits.amax(1, keepdim=True)).exp()
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + (-logits).exp())
    choice = p if s["bias"] is None else p + s["bias"].double()
    if c["groups"] > 1:
        by = choice.view(t, c["groups"], -1)
        score = by.sort(dim=-1, descending=True)[0][..., :c["group_best"]].sum(-1)
        best = score.sort(dim=-1, descending=True, stable=True)[1][:, :c["top_groups"]]
        keep = torch.zeros(t, c["groups"], dtype=torch.bool, device=DEV).scatter_(1, best, True)
        choice = by.masked_fill(~keep[..., None], -math.inf).view(t, e)
    ids = choice.sort(dim=-1, descending=True, stable=True)[1][:, :c["used"]]
    w = p.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return [ids.int(), (w * c["scale"]).float()]


def _products(s, c, w, x, per):
    """Rows of the experts' products f32 [tokens * used][rows]: pair p takes row p // per of x; pairs without an expert give 0."""
    ids, e, k, n = s["ids"].flatten().long(), c["experts"], c["k"], c["rows"]
    x = x.repeat_interleave(per, 0) if per > 1 else x
    if ids.numel() <= e:  # a matrix for each pair
        y = (_numbers(c["type"], w[ids.clamp(min=0)], n, k) @ x[..., None])[..., 0]
        return y.masked_fill(ids[:, None] < 0, 0.0)
    # the pairs of each expert side by side, as many columns as the busiest one has
    order = torch.where(ids < 0, e, ids).sort(stable=True)
    count = torch.zeros(e + 1, dtype=torch.long, device=DEV).scatter_add_(0, order[0], torch.ones_like(ids))
    col = torch.arange(ids.numel(), device=DEV) - (count.cumsum(0) - count)[order[0]]
    cols = torch.zeros(e + 1, s["most"], k, device=DEV)
    cols[order[0], torch.where(order[0] == e, 0, col)] = x[order[1]]
    y = _numbers(c["type"], w, n, k) @ cols[:e].transpose(1, 2).contiguous()
    out = torch.zeros(ids.numel(), n, device=DEV)
    out[order[1]] = y[order[0].clamp(max=e - 1), :, torch.where(order[0] == e, 0, col)]
    return out.masked_fill_(ids[:, None] < 0, 0.0)


# --------------------------------------------------------------------------------------------------- in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    w_of = lambda name: s[name].data if own else s[name]  # noqa: E731
    if c["kind"] == "norm":
        total = s["x"].double() + s["r"].double()
        y = torch.nn.functional.normalize(total, dim=1) * math.sqrt(c["n"])
        size = total.square().sum(1, keepdim=True) / c["n"]
        y = y * (size / (size + EPS)).sqrt() * s["w"].double()
        return [total, y, _exact_rounded(y, c["act"])]
    if c["kind"] == "route":
        z = s["logits"].double().cpu()
        p = z.softmax(1) if c["score"] == "softmax" else z.sigmoid()
        pick = p + (0 if s["bias"] is None else s["bias"].double().cpu())
        all_ids, all_w = [], []
        for row in range(c["tokens"]):
            choice, size = pick[row].tolist(), c["experts"] // c["groups"]
            names = range(c["experts"])
            if c["groups"] > 1:
                score = [sum(sorted(choice[g * size:(g + 1) * size], reverse=True)[:c["group_best"]]) for g in range(c["groups"])]
                kept = set(sorted(range(c["groups"]), key=lambda g: (-score[g], g))[:c["top_groups"]])
                names = [i for i in names if i // size in kept]
            ids = sorted(names, key=lambda i: (-choice[i], i))[:c["used"]]
            w = p[row][ids]
            all_ids.append(ids)
            all_w.append(w / (w.sum() if c["renorm"] else 1) * c["scale"])
        return [torch.tensor(all_ids, dtype=torch.int32), torch.stack(all_w)]
    t, u, k, n = c["tokens"], c["used"], c["k"], c["rows"]
    ids = s["ids"].flatten().long()

    def rows_of(name, x, per):
        y = torch.zeros(t * u, n, dtype=torch.float64, device=DEV)
        for e in range(c["experts"]):
            mine = (ids == e).nonzero()[:, 0]
            if mine.numel():
                # a weight is an integer of up to 8 bits times a scale of 11 (and 6), both in 32 bits without loss
                y[mine] = x[mine // per] @ _exact_numbers(c["type"], w_of(name)[e], n, k).T
        return y
    x = _exact_values(s["act"], _act_of(c["type"]), t if c["kind"] == "gate_up" else t * u, k)
    if c["kind"] == "gate_up":
        g = rows_of("gate", x, u)
        return [_exact_rounded(g * torch.sigmoid(g) * rows_of("up", x, u), c["act"])]
    y = (rows_of("down", x, 1).view(t, u, n).transpose(1, 2) @ s["weights"].double()[..., None])[..., 0]
    return [y if s["add"] is None else y + s["add"].double()]


def _exact_values(act, atype, m, k):
    q = act[:m * k].view(torch.int8).double().view(m, k)
    f = act[m * k:].view(torch.float32).double()
    return q * (f[0::2].view(m, -1).repeat_interleave(32, 1) if atype == "q8_0" else f[:m * k // 256].view(m, -1).repeat_interleave(256, 1))


def _exact_rounded(y, atype):
    if atype == "q8_0":
        b = y.reshape(-1, 32)
        d = b.abs().max(1, keepdim=True)[0] / 127
        q = torch.where(d > 0, b / d, 0.0).round()
        return (q * d.half().double()).view(y.shape)
    b = y.reshape(-1, 256)
    top, low = b.max(1, keepdim=True)[0], b.min(1, keepdim=True)[0]
    d = torch.where(top >= -low, top, low) / -127
    return (torch.where(d != 0, b / d, 0.0).round().clamp(max=127) * d).view(y.shape)


def _exact_numbers(wtype, w, n, k):
    """One matrix f64 [n][k], element by element of its block."""
    dev, h = w.device, torch.float16
    j = torch.arange(k, device=dev)
    if wtype in ("q4_0", "q8_0"):
        b, i = j // 32, j % 32
        if wtype == "q8_0":
            return w[:n * k].view(torch.int8).view(n, k).double() * w[n * k:].view(h).view(n, -1)[:, b].double()
        q = w[:n * k // 2].view(n, -1)[:, 16 * b + i % 16].int()
        r = torch.arange(n, device=dev)
        d = w[n * k // 2:].view(h)[((r // 2)[:, None] * (k // 32) + b) * 2 + (r % 2)[:, None]]
        return (((q >> (i // 16 * 4)) & 15) - 8).double() * d.double()
    sb, i = j // 256, j % 256
    m = n * (k // 256)
    if wtype == "q4_k":
        unit = i // 32
        q = (w[:m * 128].view(n, -1)[:, 128 * sb + 32 * (unit // 2) + i % 32].int() >> (4 * (unit % 2))) & 15
        head = w[m * 128:].view(n, -1, 16)
        at = lambda p: head[:, sb, 4 + p].int()  # noqa: E731
        low = unit % 4
        sc = torch.where(unit < 4, at(low) & 63, (at(8 + low) & 15) + (at(low) >> 6) * 16)
        mn = torch.where(unit < 4, at(4 + low) & 63, (at(8 + low) >> 4) + (at(4 + low) >> 6) * 16)
        d = head[..., :4].contiguous().view(h).double()
        return d[:, sb, 0] * (sc * q).double() - d[:, sb, 1] * mn.double()
    half, part, l = i // 128, i % 128 // 32, i % 32
    lo = (w[:m * 128].view(n, -1)[:, 128 * sb + 64 * half + 32 * (part % 2) + l].int() >> (4 * (part // 2))) & 15
    hi = (w[m * 128:m * 192].view(n, -1)[:, 64 * sb + 32 * half + l].int() >> (2 * part)) & 3
    sc = w[m * 192:m * 208].view(torch.int8).view(n, -1)[:, j // 16].double()
    return (lo + 16 * hi - 32).double() * sc * w[m * 208:].view(h).view(n, -1)[:, sb].double()
