"""The feed-forward part of a mixture of experts on two streams at once: eager layers beside eager ones, and beside a captured one's
replays. Nothing of a call (plans, workspaces, outputs) is another's."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from moe_ref import DEV, Q4_0, Q4_K, Q6_K, Q8_0  # noqa: E402
from test_gpu_moe import gen, layer, setup  # noqa: E402

ROUNDS = 12


@pytest.mark.parametrize("t,t2", [(Q4_0, Q4_K), (Q8_0, Q8_0), (Q4_K, Q6_K)])
@pytest.mark.parametrize("toks", [(1, 70), (6, 300), (70, 70), (1500, 40)])
def test_two_streams_at_once(t, t2, toks):
    from ameva_compute_amd import ops
    s, router, nw = setup(t, t2)
    x = [torch.randn(ROUNDS, tok, 512, generator=gen(i), device=DEV) for i, tok in enumerate(toks)]
    r = [torch.randn(ROUNDS, tok, 512, generator=gen(50 + i), device=DEV) for i, tok in enumerate(toks)]
    alone = [[layer(ops, s, x[i][j], r[i][j], router, nw) for j in range(ROUNDS)] for i in range(2)]
    # the first one's layer captured, its inputs copied in on the replaying stream
    cx, cr = torch.zeros(toks[0], 512, device=DEV), torch.zeros(toks[0], 512, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer(ops, s, cx, cr, router, nw)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    big = torch.randn(8192, 8192, device=DEV)
    torch.cuda.synchronize()
    for replay in (False, True):
        got = [[], []]
        for _ in range(4):  # both streams wait for these products, so that their calls stand in line and then run side by side
            big @ big
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        for j in range(ROUNDS):  # no wait between the streams, nor for the host
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    if replay and i == 0:
                        cx.copy_(x[0][j])
                        cr.copy_(r[0][j])
                        graph.replay()
                        got[0].append([v.clone() for v in captured])
                    else:
                        got[i].append(layer(ops, s, x[i][j], r[i][j], router, nw))
        torch.cuda.synchronize()
        for i in range(2):
            for j in range(ROUNDS):
                assert all(torch.equal(a, b) for a, b in zip(got[i][j], alone[i][j])), (replay, i, j)
