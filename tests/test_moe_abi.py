"""Refusals of the mixture-of-experts entry points, on the host before any launch (no GPU call is made), and their sizes."""
import pytest

from ameva_compute_amd._lib import lib

Q4_0, Q8_0, Q4_K, Q6_K, Q8_K = 2, 8, 12, 14, 15
A = 4096  # an address that is aligned and never read


def refused(rc, word):
    assert rc == -1 and word in lib().amv_last_error().decode(), (rc, lib().amv_last_error())


def norm(x=A, add=A, rows=2, n=512, w=A, out=A, o=A, act=A, t=Q8_0, rule=0):
    return lib().amv_add_rms_norm_act(x, add, rows, n, 1e-5, w, out, o, act, t, rule, None)


def route(logits=A, stride=64, tok=3, n=64, used=4, score=0, bias=None, groups=1, top=1, best=1, ids=A, w=A):
    return lib().amv_moe_route(logits, stride, tok, n, used, score, bias, groups, top, best, 1, 1.0, ids, w, None)


def plan(ids=A, tok=3, used=2, n=8, p=A):
    return lib().amv_moe_plan(ids, tok, used, n, p, None)


def gate_up(t=Q4_0, w=A, w2=A, stride=None, n=8, rows=256, k=512, act=A, tok=3, used=2, ids=A, p=A, eout=None, out=A, at=Q8_0, rule=0, ws=A,
            ws_bytes=1 << 40):
    stride = max(16, lib().amv_weight_bytes(t, rows, k)) if stride is None else stride
    return lib().amv_moe_gate_up(t, w, w2, stride, n, rows, k, act, tok, used, ids, p, eout, out, at, rule, ws, ws_bytes, None)


def down(t=Q4_0, w=A, stride=None, n=8, rows=256, k=512, act=A, tok=3, used=2, ids=A, p=A, weights=A, add=None, dst=A, ws=A, ws_bytes=1 << 40):
    stride = max(16, lib().amv_weight_bytes(t, rows, k)) if stride is None else stride
    return lib().amv_moe_down(t, w, stride, n, rows, k, act, tok, used, ids, p, weights, add, dst, ws, ws_bytes, None)


def test_norm():
    for bad in (dict(x=None), dict(add=None), dict(out=None)):
        refused(norm(**bad), "null")
    for bad in (dict(rows=-1), dict(rows=1 << 22), dict(n=0), dict(n=(1 << 24) + 4)):
        refused(norm(**bad), "bad shape")
    refused(norm(n=510, act=None), "n % 4")
    for name in ("x", "add", "w", "out", "o", "act"):
        refused(norm(**{name: A + 8}), "16-byte aligned")
    refused(norm(t=Q4_0), "act_type")
    refused(norm(n=516), "block size")
    refused(norm(n=544, t=Q8_K), "block size")
    refused(norm(rule=3), "bad rule")
    assert norm(rows=0) == 0


def test_act_values():
    f = lib().amv_act_values
    refused(f(Q8_0, None, 1, 32, 0, A, None), "null")
    refused(f(Q4_0, A, 1, 32, 0, A, None), "type")
    refused(f(Q8_0, A, 1, 33, 0, A, None), "bad shape")
    refused(f(Q8_K, A, 1, 32, 0, A, None), "bad shape")
    refused(f(Q8_0, A, -1, 32, 0, A, None), "bad shape")
    refused(f(Q8_0, A, 1 << 29, 32, 0, A, None), "too many")
    refused(f(Q8_0, A, 1, 32, 2, A, None), "output type")
    refused(f(Q8_0, A + 4, 1, 32, 0, A, None), "aligned")
    assert f(Q8_0, A, 0, 32, 0, A, None) == 0


def test_route():
    for bad in (dict(logits=None), dict(ids=None), dict(w=None)):
        refused(route(**bad), "null")
    for bad in (dict(tok=-1), dict(n=0), dict(n=1025)):
        refused(route(**bad), "experts (1 to")
    for bad in (dict(used=0), dict(used=65, n=128), dict(used=9, n=8), dict(used=-1)):
        refused(route(**bad), "experts a token")
    for tok in (1 << 22, 1 << 62):
        refused(route(tok=tok), "pairs")
    refused(route(stride=63), "stride")
    refused(route(score=2), "score")
    for bad in (dict(groups=0), dict(groups=65, n=650, stride=650), dict(groups=3), dict(groups=4, top=0), dict(groups=4, top=5)):
        refused(route(**bad), "groups")
    refused(route(best=3), "group_best")
    assert route(tok=0) == 0


def test_plan():
    for bad in (dict(tok=-1), dict(used=0), dict(used=65), dict(n=0), dict(n=1025)):
        refused(plan(**bad), "tokens with")
        b = {**dict(tok=3, used=2, n=8), **bad}
        assert lib().amv_moe_plan_bytes(b["tok"], b["used"], b["n"]) == -1
    refused(plan(tok=1 << 22), "pairs")
    for bad in (dict(ids=None), dict(p=None), dict(p=A + 4)):
        refused(plan(**bad), "null")
    assert plan(tok=0) == 0
    for tok, used, n in ((1, 8, 128), (7, 3, 5), (600, 8, 64), (4096, 8, 256), (1 << 16, 64, 1024)):
        pairs = tok * used
        worst = (pairs - min(pairs, n + 1)) // 16 + min(pairs, n + 1)  # tiles, if every expert had one row more than whole tiles
        assert lib().amv_moe_plan_bytes(tok, used, n) >= 4 * pairs + 8 * worst


@pytest.mark.parametrize("call", [gate_up, down])
def test_products(call):
    for bad in (dict(tok=-1), dict(used=0), dict(n=0), dict(n=2000)):
        refused(call(**bad), "tokens with")
    refused(call(tok=1 << 22), "pairs")
    for t in (0, 1, 3, 15):
        refused(call(t=t), "not supported")
    for bad in (dict(rows=0), dict(rows=250), dict(k=0), dict(k=500), dict(t=Q4_K, k=544), dict(t=Q6_K, k=128)):
        refused(call(**bad), "experts of")
    for bad in (dict(rows=1 << 16, k=1 << 15, stride=1 << 40), dict(k=1 << 21, stride=1 << 40)):
        refused(call(**bad), "too large")
    for bad in (dict(w=None), dict(w=A + 8), dict(ids=None)):
        refused(call(**bad), "weights")
    for s in (0, 256 * 16 * 18 - 16, 256 * 16 * 18 + 8):
        refused(call(stride=s), "bytes apart")
    for bad in (dict(act=None), dict(act=A + 4), dict(p=A + 4)):
        refused(call(**bad), "activations or plan")
    refused(call(tok=1 << 20, rows=1 << 12), "too many")
    refused(call(tok=1 << 17, p=None), "without a plan")
    refused(call(tok=512, n=1024, rows=1 << 20, k=512, stride=1 << 40), "tiles of")
    assert call(tok=0) == 0


def test_gate_up():
    refused(gate_up(w2=None), "weights")
    refused(gate_up(out=None), "no output")
    for bad in (dict(out=A + 8), dict(eout=A + 4), dict(ws=A + 8)):
        refused(gate_up(**bad), "aligned")
    refused(gate_up(at=Q4_0), "act_type")
    refused(gate_up(at=Q8_K, rows=288), "Q8_K output")
    refused(gate_up(rule=-1), "bad rule")
    need = lib().amv_moe_gate_up_workspace_bytes(3, 2, 256, Q8_K)
    for bad in (dict(ws=None), dict(ws_bytes=need - 1)):
        if need:
            refused(gate_up(at=Q8_K, **bad), "workspace")
    assert lib().amv_moe_gate_up_workspace_bytes(-1, 2, 256, Q8_K) == -1


def test_down():
    for bad in (dict(weights=None), dict(dst=None), dict(dst=A + 4), dict(add=A + 8), dict(ws=A + 4)):
        refused(down(**bad), "null weights")
    need = lib().amv_moe_down_workspace_bytes(300, 2, 256)
    assert need >= 0
    for bad in (dict(ws=None), dict(ws_bytes=need - 1)):
        if need:
            refused(down(tok=300, **bad), "workspace")
    assert lib().amv_moe_down_workspace_bytes(3, 0, 256) == -1


def test_python_side():
    torch = pytest.importorskip("torch")
    from ameva_compute_amd import ops
    x = torch.zeros(2, 64)
    for call in (lambda: ops.QExperts(Q4_0, 1, 32, 32, torch.zeros(1, 576, dtype=torch.uint8)), lambda: ops.add_rms_norm(x, x, 1e-5),
                 lambda: ops.moe_route(x, 2), lambda: ops.moe_plan(torch.zeros(2, 2, dtype=torch.int32), 8),
                 lambda: ops.act_values(torch.zeros(80, dtype=torch.uint8), Q8_0, 2, 32)):
        with pytest.raises(ValueError, match="GPU"):
            call()
