"""One captured step of the paged KV cache over batches of any split."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from paged_ref import DEV, F16, Q8_0, off  # noqa: E402


@pytest.mark.parametrize("t", [F16, Q8_0])
def test_one_graph_for_batches_of_any_split(t):
    """A captured append, attention, shared attention and selection, replayed with other tokens a sequence, lengths and pages in the same
    tensors (prompts, steps, sequences without tokens, rows behind the last), against a pool and a batch of each split's own."""
    from ameva_compute_amd import ops
    H, G, D, page, n_seq, n_tok, cols = 8, 2, 128, 16, 5, 160, 40
    splits = [([100, 1, 1, 20, 1], [130, 500, 33, 20, 1]), ([1, 1, 1, 1, 1], [640, 1, 17, 16, 300]), ([0, 160, 0, 0, 0], [5, 400, 0, 1, 9]),
              ([3, 0, 4, 2, 0], [3, 70, 64, 2, 0]), ([0, 0, 0, 0, 0], [9, 9, 9, 9, 9])]
    fill = torch.randn(2, 220, G, page, D, device=DEV)

    def pool():
        kv = ops.PagedKV.alloc(t, 220, page, G, D, DEV, bounds=True)
        if t == F16:
            kv.k.copy_(fill[0])
            kv.v.copy_(fill[1])
        else:
            from paged_ref import pack
            kv.k.copy_(pack(fill[0], t, "k")[0])
            kv.v.copy_(pack(fill[1], t, "v")[0])
        kv.bounds.copy_(torch.stack([fill[0].half().amin(2), fill[0].half().amax(2)], 2))
        return kv
    kv, pre = pool(), torch.arange(200, 220, device=DEV).int()
    n_kv, cu_q = torch.zeros(n_seq, dtype=torch.int32, device=DEV), torch.zeros(n_seq + 1, dtype=torch.int32, device=DEV)
    table = torch.zeros(n_seq, cols, dtype=torch.int32, device=DEV)
    x = torch.zeros(n_tok, H + 2 * G, D, device=DEV)
    b = ops.PagedBatch(n_kv, table, cols * page, n_tok, cu_q=cu_q, max_q=n_tok)
    ws = torch.empty(max(64, ops.paged_workspace_bytes(kv, b, H), ops.paged_workspace_bytes(kv, b, H, n_prefix=300)), dtype=torch.uint8,
                     device=DEV)
    outs = [torch.zeros(n_tok, H, D, device=DEV) for _ in range(3)]
    sel = torch.zeros(n_tok, G, 6, dtype=torch.int32, device=DEV)

    def body():
        ops.paged_rope_append(kv, b, x, H, out=outs[0])
        ops.paged_attn(kv, b, outs[0], 0.09, out=outs[1], workspace=ws)
        ops.paged_attn_shared(kv, b, outs[0], 0.09, pre, 300, out=outs[2], workspace=ws)
        ops.paged_select(kv, b, outs[0], 6, sel=sel)

    def load(split, seed):
        n_q, lengths = split
        torch.manual_seed(seed)
        order = torch.randperm(200, device=DEV).int().view(n_seq, cols)
        rows = torch.randn(n_tok, H + 2 * G, D, device=DEV)
        ends = torch.tensor([sum(n_q[:i]) for i in range(n_seq + 1)], dtype=torch.int32, device=DEV)
        return rows, order, ends, torch.tensor(lengths, dtype=torch.int32, device=DEV)
    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    for i, split in enumerate(splits + splits[:2]):
        rows, order, ends, lengths = load(split, i)
        kv2 = pool()
        for a, src in ((kv.k, kv2.k), (kv.v, kv2.v), (kv.bounds, kv2.bounds), (x, rows), (table, order), (cu_q, ends), (n_kv, lengths)):
            a.copy_(src)
        for o in outs:
            o.fill_(7.0)
        sel.fill_(-7)
        graph.replay()
        torch.zeros(1000, device=DEV).sum()
        n = sum(split[0])
        assert all(bool((o[n:] == 7.0).all()) for o in outs) and bool((sel[n:] == -7).all())
        if not n:
            assert torch.equal(kv.k, kv2.k) and torch.equal(kv.v, kv2.v)
            continue
        b2 = ops.PagedBatch(lengths, order, max(split[1]), n, cu_q=ends, max_q=max(split[0]))
        q = ops.paged_rope_append(kv2, b2, rows[:n], H)
        assert torch.equal(q, outs[0][:n]) and torch.equal(kv.k, kv2.k) and torch.equal(kv.v, kv2.v) and torch.equal(kv.bounds, kv2.bounds)
        assert off(outs[1][:n], ops.paged_attn(kv2, b2, q, 0.09).double()) < 2e-5  # (both are the kernels': twice the tolerance)
        assert off(outs[2][:n], ops.paged_attn_shared(kv2, b2, q, 0.09, pre, 300).double()) < 2e-5
        assert torch.equal(sel[:n], ops.paged_select(kv2, b2, q, 6))
