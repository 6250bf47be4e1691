"""The paged operators as a server uses them together: prompts appended and attended in chunks, decode steps captured in a HIP graph
and replayed at growing lengths, sequences behind a common prompt, selected pages; streams, devices, workspaces."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from paged_ref import DEV, F16, Q8_0, off  # noqa: E402

H, G, D, PAGE = 8, 2, 128, 16
SCALE = D ** -0.5
TOL = 2e-5  # test_gpu_paged_attn's, twice: both sides are the kernels'


def rows(n, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(n, H + 2 * G, D, generator=g, device=DEV)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("t", [F16, Q8_0])
def test_chunks_steps_and_graphs(t):
    """Two sequences token by token in a replayed graph against one prompt of all their tokens."""
    from ameva_compute_amd import ops
    lens, chunk = [90, 61], [70, 41]
    x = [rows(n, s) for s, n in enumerate(lens)]
    order = torch.randperm(16, device=DEV).int()
    table = torch.stack([order[:8], order[8:]]).contiguous()
    whole = ops.PagedKV.alloc(t, 16, PAGE, G, D, DEV, bounds=True)
    b = ops.PagedBatch(ints(lens), table, 128, sum(lens), cu_q=ints([0, lens[0], sum(lens)]), max_q=90)
    want = ops.paged_attn(whole, b, ops.paged_rope_append(whole, b, torch.cat(x), H), SCALE)
    want = [want[:lens[0]], want[lens[0]:]]

    kv = ops.PagedKV.alloc(t, 16, PAGE, G, D, DEV, bounds=True)
    n_kv = ints([0, 0])
    for a, e in ((0, 33), (33, None)):  # the prompts in two chunks
        n = [len(r[a:e if e else c]) for r, c in zip(x, chunk)]
        n_kv += ints(n)
        b = ops.PagedBatch(n_kv, table, 128, sum(n), cu_q=ints([0, n[0], sum(n)]), max_q=max(n))
        y = ops.paged_attn(kv, b, ops.paged_rope_append(kv, b, torch.cat([r[a:e if e else c] for r, c in zip(x, chunk)]), H), SCALE)
        for s in range(2):
            assert off(y[s * n[0]:][:n[s]], want[s][a:a + n[s]].double()) < TOL
    # decode steps: one graph, the row and the lengths in device memory
    row, q = torch.zeros(2, H + 2 * G, D, device=DEV), torch.zeros(2, H, D, device=DEV)
    out, dense = torch.zeros_like(q), torch.zeros_like(q)
    step = ops.PagedBatch(n_kv, table, 128)
    ws = torch.empty(max(64, ops.paged_workspace_bytes(kv, step, H), ops.paged_workspace_bytes(kv, step, H, n_sel=8)),
                     dtype=torch.uint8, device=DEV)

    def body():
        n_kv.add_(1)
        ops.paged_rope_append(kv, step, row, H, out=q)
        ops.paged_attn(kv, step, q, SCALE, out=dense, workspace=ws)
        sel = ops.paged_select(kv, step, q, 8)  # all the pages there are
        ops.paged_attn_sparse(kv, step, q, sel, SCALE, out=out, workspace=ws)
    n_kv -= 1
    row.copy_(torch.stack([r[c - 1] for r, c in zip(x, chunk)]))
    body()  # the last prompt tokens once more, before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    for i in range(20):
        row.copy_(torch.stack([r[c + i] for r, c in zip(x, chunk)]))
        graph.replay()
        torch.zeros(1000, device=DEV).sum()
        for s in range(2):
            assert off(dense[s], want[s][chunk[s] + i].double()) < TOL
            assert off(out[s], want[s][chunk[s] + i].double()) < TOL
    assert torch.equal(kv.k[order.long()][:5].view(torch.uint8), whole.k[order.long()][:5].view(torch.uint8))
    used = order[:6].long()  # pages with keys
    assert torch.equal(kv.bounds[used], whole.bounds[used])


def test_prefix_is_the_same_as_a_copy_of_it():
    """Sequences behind one prompt, appended after it with positions that go on, against each holding the prompt itself."""
    from ameva_compute_amd import ops
    n_pre, own = 50, [3, 20, 1]
    pre, x = rows(n_pre, 7), [rows(n, 8 + s) for s, n in enumerate(own)]
    kv = ops.PagedKV.alloc(F16, 40, PAGE, G, D, DEV)
    pre_table = ints([[30, 2, 31, 3]])
    b = ops.PagedBatch(ints([n_pre]), pre_table, 64, n_pre, cu_q=ints([0, n_pre]), max_q=n_pre)
    ops.paged_rope_append(kv, b, pre, H)
    table = ints([[4, -1], [5, 6], [7, -1]])
    cu = ints([0, 3, 23, 24])
    b = ops.PagedBatch(ints(own), table, 32, sum(own), cu_q=cu, max_q=20)
    pos = torch.cat([torch.arange(n_pre, n_pre + n) for n in own]).int().to(DEV)
    q = ops.paged_rope_append(kv, b, torch.cat(x), H, pos=pos)
    y = ops.paged_attn_shared(kv, b, q, SCALE, pre_table[0], n_pre)
    full = ops.PagedBatch(ints([n_pre + n for n in own]), ints([[8, 9, 10, 11, 12], [13, 14, 15, 16, 17], [18, 19, 20, 21, 22]]), 80,
                          3 * n_pre + sum(own), cu_q=ints([0, n_pre + 3, 2 * n_pre + 23, 3 * n_pre + 24]), max_q=n_pre + 20)
    q2 = ops.paged_rope_append(kv, full, torch.cat([torch.cat([pre, r]) for r in x]), H)
    z = ops.paged_attn(kv, full, q2, SCALE)
    at = 0
    for s, n in enumerate(own):
        at += n_pre
        assert torch.equal(q[int(cu[s]):int(cu[s + 1])], q2[at:at + n])
        assert off(y[int(cu[s]):int(cu[s + 1])], z[at:at + n].double()) < TOL
        at += n


def test_streams_and_two_graphs():
    """Calls on a side stream, and two captured graphs in turn, each with the workspace it was captured with."""
    from ameva_compute_amd import ops
    kv = ops.PagedKV.alloc(F16, 800, PAGE, G, D, DEV, bounds=True)
    table = torch.randperm(800, device=DEV).int().view(2, 400)
    n_kv = ints([6000, 333])
    fill = ops.PagedBatch(n_kv, table, 6400, 6333, cu_q=ints([0, 6000, 6333]), max_q=6000)
    ops.paged_rope_append(kv, fill, rows(6333, 1), H)
    b = ops.PagedBatch(n_kv, table, 6400)
    qs = [torch.randn(2, H, D, device=DEV) for _ in range(2)]
    want = [ops.paged_attn(kv, b, q, SCALE) for q in qs]
    wsel = [ops.paged_select(kv, b, q, 6) for q in qs]
    assert ops.paged_workspace_bytes(kv, b, H) > 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.paged_attn(kv, b, qs[0], SCALE)
    side.synchronize()
    assert torch.equal(got, want[0])
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((ops.paged_attn(kv, b, q, SCALE), ops.paged_select(kv, b, q, 6)))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o[0].zero_()
            o[1].zero_()
        for g in graphs:
            g.replay()
        torch.randn(1 << 20, device=DEV).sum()
        torch.cuda.synchronize()
        for (y, sel), r, rs in zip(outs, want, wsel):
            assert torch.equal(y, r) and torch.equal(sel, rs)


def test_same_call_same_bits():
    from ameva_compute_amd import ops
    kv = ops.PagedKV.alloc(Q8_0, 300, PAGE, G, D, DEV)
    table = torch.randperm(300, device=DEV).int().view(1, 300)
    b = ops.PagedBatch(ints([4800]), table, 4800, 4800, cu_q=ints([0, 4800]), max_q=4800)
    q = ops.paged_rope_append(kv, b, rows(4800, 3), H)
    last = ops.PagedBatch(ints([4800]), table, 4800)
    y = ops.paged_attn(kv, last, q[-1:], SCALE)
    for _ in range(5):
        assert torch.equal(ops.paged_attn(kv, last, q[-1:], SCALE), y)


def test_no_tokens():
    from ameva_compute_amd import ops
    kv = ops.PagedKV.alloc(F16, 4, PAGE, G, D, DEV, bounds=True)
    b = ops.PagedBatch(ints([3]), ints([[0]]), 16, 0, cu_q=ints([0, 0]))
    q = torch.empty(0, H, D, device=DEV)
    assert ops.paged_rope_append(kv, b, torch.empty(0, H + 2 * G, D, device=DEV), H).shape == (0, H, D)
    assert ops.paged_attn(kv, b, q, SCALE).shape == (0, H, D)
    sel = ops.paged_select(kv, b, q, 3)
    assert sel.shape == (0, G, 3) and ops.paged_attn_sparse(kv, b, q, sel, SCALE).shape == (0, H, D)
