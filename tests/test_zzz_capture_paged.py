"""Steps of requests served from one pool, recorded into graphs: replayed with other inputs, beside eager steps, and by two graphs that share a stream's workspace."""
import pytest
import torch

from dtas_amd import ops
from test_paged_run import HKV, L, D, Served
from test_zzz_capture import new_stream

pytestmark = pytest.mark.gpu


def served(seed, G=3, W=4, prompt=(700, 90, 300)):
    columns = 64
    s = Served(G, W, columns, G * W * columns, seed)
    keys = torch.randn(L, sum(prompt), HKV, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).half()
    s.prompt(list(prompt), keys, -keys)
    return s


def same(a, b):
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.int16) if x.dtype == torch.float16 else x, y.view(torch.int16) if y.dtype == torch.float16 else y)


def recorded(s, stream):
    """A graph of one step, the first that the stream sees."""
    graph, start = torch.cuda.CUDAGraph(), s.state()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        s.step()
    same(start, s.state())  # (recording runs nothing)
    return graph


def test_a_recorded_step_goes_on_like_an_eager_one():
    s, eager = served(1), served(1)
    graph = recorded(s, new_stream())
    for i in range(20):  # over the end of a page
        s.fill(i)
        eager.fill(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        same(s.state(), eager.state())


def test_two_graphs_share_a_workspace():
    # of different sizes, replayed in turn, with eager steps of a third on the same stream between them
    stream = new_stream()
    makers = [lambda: served(2), lambda: served(3, 2, 8, (900, 33)), lambda: served(4, 1, 1, (1000,))]
    mine, others = [m() for m in makers], [m() for m in makers]
    graphs = [recorded(s, stream) for s in mine[:2]]
    for i in range(6):
        for s, e in zip(mine, others):
            s.fill(i)
            e.fill(i)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[i % 2].replay()
            mine[2].step()
            graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        for s, e in zip(mine, others):
            e.step()
            same(s.state(), e.state())


def test_a_recorded_attention_goes_by_the_lengths_of_its_replay():
    # beams apart, beams read together, one long among short ones: the device finds out, each time anew
    B, W, heads, kv_heads, d, page, columns = 8, 4, 64, 32, 64, 16, 140
    g = torch.Generator(device="cuda").manual_seed(7)
    K, V = (torch.randn(B * columns, kv_heads, page, d, device="cuda", generator=g).half() for _ in range(2))
    table = torch.randperm(B * columns, device="cuda", generator=g).int().view(B, columns)
    table.view(B // W, W, columns)[:, :, :90] = table.view(B // W, W, columns)[:, :1, :90].clone()
    Q = torch.randn(B, heads, d, device="cuda", generator=g).half()
    lens, out, eager = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.empty_like(Q), torch.empty_like(Q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=new_stream()):
        ops.attn_paged(Q, K, V, table, lens, out, None, W)
    for now in ([1] * B, [2200 - b for b in range(B)], [0, 5, 2240, 3, 1, 2, 0, 700], [900] * B, [2239, 1600, 1700, 1800, 9, 8, 7, 6], [30] * B, [2240] * B):
        lens.copy_(torch.tensor(now))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ops.attn_paged(Q, K, V, table, lens, eager, None, W)
        same([out], [eager])
        apart = torch.empty_like(Q)
        ops.attn_paged(Q, K, V, table, lens, apart, None, 1)
        # (both within the bound of either: weights 2^-11 each way of values up to 6, and the answer's own rounding)
        assert float((out.float() - apart.float()).abs().max()) <= 2 * (2.0 ** -11 * 6 * 2 + 2.0 ** -11 * 6)
