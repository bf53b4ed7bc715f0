"""Decoding steps with drafted tokens, put together from the framework's operators: one after the other, recorded into a graph, on several
streams."""
import threading

import pytest
import torch

from dtas_amd import ops

pytestmark = pytest.mark.gpu
LAYERS, HEADS, KV, DIM, ROT, HIDDEN, VOCAB, MAX_POS = 2, 8, 2, 64, 16, 512, 1000, 512


def h(*s):
    return torch.empty(*s, device="cuda", dtype=torch.float16)


class Model:
    """Two layers with 4-bit weights, rotated queries and keys, an RMSNorm in front of each, an fp16 head."""

    def __init__(self):
        g = torch.Generator(device="cuda").manual_seed(11)
        width = (HEADS + 2 * KV) * DIM

        def q4(N, K):
            words = torch.randint(-2 ** 31, 2 ** 31, (N, K // 8), device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
            return words, ((0.5 + torch.rand(N, K // 32, device="cuda", generator=g)) / (4.6 * K ** 0.5)).half()

        self.qkv = [q4(width, HIDDEN) for _ in range(LAYERS)]
        self.o = [q4(HIDDEN, HEADS * DIM) for _ in range(LAYERS)]
        self.norm = [torch.ones(HIDDEN, device="cuda").half() for _ in range(LAYERS)]
        self.embed = torch.randn(VOCAB, HIDDEN, device="cuda", generator=g).half()
        self.head = (torch.randn(VOCAB, HIDDEN, device="cuda", generator=g) * 0.1).half()
        angle = torch.arange(MAX_POS, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, ROT, 2, device="cuda") / ROT)
        self.cos, self.sin = (f(torch.cat((angle, angle), 1)).half() for f in (torch.cos, torch.sin))
        self.temperature = torch.full((1,), 1.5, device="cuda")


class Step:
    """The buffers of one pass of B x T nodes, allocated once."""

    def __init__(self, model, B, T, capacity=256, caches=None):
        self.m, self.B, self.T = model, B, T
        rows = B * T
        self.x, self.normed, self.context = h(rows, HIDDEN), h(rows, HIDDEN), h(B, T, HEADS, DIM)
        self.qkv = h(rows, (HEADS + 2 * KV) * DIM)
        self.q, self.k = h(1, rows, HEADS, DIM), h(1, rows, KV, DIM)
        self.cos, self.sin = h(rows, ROT), h(rows, ROT)
        self.K, self.V = h(LAYERS, B, T, KV, DIM), h(LAYERS, B, T, KV, DIM)
        self.logits16, self.logits = h(rows, VOCAB), torch.empty(rows, VOCAB, device="cuda")
        self.P = torch.empty(B, T, VOCAB, device="cuda")
        self.tokens, self.parents, self.positions = (torch.zeros(B, T, device="cuda", dtype=torch.int32) for _ in range(3))
        self.caches = caches or [torch.full((LAYERS, B, KV, capacity, DIM), float("nan"), device="cuda", dtype=torch.float16) for _ in range(2)]
        self.lens = torch.zeros(B, device="cuda", dtype=torch.int32)

    def forward(self):
        m, rows = self.m, self.B * self.T
        ops.take(m.embed, self.tokens, self.x)
        ops.take(m.cos, self.positions, self.cos)
        ops.take(m.sin, self.positions, self.sin)
        for layer in range(LAYERS):
            ops.rms_norm(self.x, m.norm[layer], self.normed)
            ops.gemv_q4(self.normed, *m.qkv[layer], None, self.qkv)
            parts = self.qkv.view(1, rows, HEADS + 2 * KV, DIM)
            q, k, v = (parts[:, :, a:b].contiguous() for a, b in ((0, HEADS), (HEADS, HEADS + KV), (HEADS + KV, HEADS + 2 * KV)))
            ops.rotary(q, self.cos, self.sin, self.q, rows)
            ops.rotary(k, self.cos, self.sin, self.K[layer].view(1, rows, KV, DIM), rows)
            self.V[layer].copy_(v.view(self.B, self.T, KV, DIM))
            ops.attn_tree(self.q.view(self.B, self.T, HEADS, DIM), self.K[layer], self.V[layer], self.caches[0][layer], self.caches[1][layer],
                          self.lens, self.parents, self.context)
            ops.gemv_q4(self.context.view(rows, HIDDEN), *m.o[layer], None, self.x, epilogue=1, res1=self.x.clone(), res2=torch.zeros_like(self.x))
        ops.gemm(self.x, m.head, None, self.logits16)
        ops.cast(self.logits16, self.logits)
        ops.softmax_temperature(self.logits, m.temperature, self.P.view(rows, VOCAB))


def depths(parents):
    out = []
    for i, p in enumerate(parents):
        out.append(0 if not 0 <= p < i else out[p] + 1)
    return out


def prompt(model, B, n, capacity=256):
    """Caches that hold n tokens of each of B sequences, appended in one piece."""
    step = Step(model, B, n, capacity)
    step.tokens.copy_(torch.randint(0, VOCAB, (B, n), generator=torch.Generator().manual_seed(5)))
    step.parents.copy_(torch.arange(-1, n - 1).expand(B, n))
    step.positions.copy_(torch.arange(n).expand(B, n))
    step.forward()
    ops.cache_append(step.K, step.V, None, None, *step.caches, step.lens)
    return step.caches


@pytest.mark.parametrize("parents", [[-1, 0, 1, 2, 3, 4, 5], [-1, 0, 0, 1, 1, 2, 5, 6, 0]])
def test_a_tree_scores_what_single_tokens_would(parents):
    # every node of the tree, once as part of it and once as the end of its own line of single decode steps
    model, B, n, T = Model(), 2, 37, len(parents)
    caches = prompt(model, B, n)
    step = Step(model, B, T, caches=caches)
    step.lens.fill_(n)
    step.tokens.copy_(torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(6)))
    step.parents.copy_(torch.tensor(parents).expand(B, T))
    step.positions.copy_((n + torch.tensor(depths(parents))).expand(B, T))
    step.forward()
    assert bool(torch.isfinite(step.logits).all())
    for node in range(T):
        line, at = [node], node
        while 0 <= parents[at] < at:
            at = parents[at]
            line.insert(0, at)
        one = Step(model, B, 1, caches=[c.clone() for c in caches])
        for j, i in enumerate(line):
            one.tokens.copy_(step.tokens[:, i:i + 1])
            one.parents.fill_(-1)
            one.positions.fill_(n + j)
            one.lens.fill_(n + j)
            one.forward()
            ops.cache_append(one.K, one.V, None, None, *one.caches, one.lens)
        # The same sums in another order, through two layers of fp16 activations.  Each activation is off by half a step (2^-11) and what a layer
        # adds to the stream of size s is of order s as well: some ten roundings of 2^-11 of the logits' size in all
        close = (one.logits - step.logits.view(B, T, VOCAB)[:, node]).abs().max() <= 10 * 2.0 ** -11 * step.logits.abs().max()
        assert bool(close), node


def test_accepted_rows_are_those_of_single_steps():
    """A whole step: a tree scored, verified, its path appended; the cache then holds the rows that decoding the accepted tokens one by one
    would have put there, and nothing else changed."""
    model, B, n = Model(), 3, 20
    parents = [-1, 0, 0, 1, 1, 3, 2]
    T = len(parents)
    caches = prompt(model, B, n)
    step = Step(model, B, T, caches=caches)
    step.lens.fill_(n)
    g = torch.Generator().manual_seed(8)
    step.tokens.copy_(torch.randint(0, VOCAB, (B, T), generator=g))
    step.parents.copy_(torch.tensor(parents).expand(B, T))
    step.positions.copy_((n + torch.tensor(depths(parents))).expand(B, T))
    step.forward()
    # the draft: the target, so that every first child is accepted and the walk follows 0, 1, 3, 5
    path, count, nxt = torch.empty(B, T, device="cuda", dtype=torch.int32), torch.empty(B, device="cuda", dtype=torch.int32), torch.empty(B, device="cuda", dtype=torch.int32)
    accept, sample = torch.rand(B, T, generator=g).cuda(), torch.rand(B, generator=g).cuda()
    ops.verify_tree(step.P, step.P.clone(), step.tokens, step.parents, accept, sample, path, count, nxt)
    assert path.tolist() == [[0, 1, 3, 5, -1, -1, -1]] * B and count.tolist() == [4] * B
    upto = step.P[:, 5].double().cumsum(-1)
    assert nxt.tolist() == [int((upto[b] <= float(sample[b]) * upto[b, -1]).sum()) for b in range(B)]
    before = [c.clone() for c in caches]
    ops.cache_append(step.K, step.V, path, count, *caches, step.lens)
    for new, cache, old in zip((step.K, step.V), caches, before):
        assert torch.equal(cache[:, :, :, n:n + 4], new[:, :, [0, 1, 3, 5]].transpose(2, 3))
        cache[:, :, :, n:n + 4] = old[:, :, :, n:n + 4]
        assert torch.equal(cache.view(torch.int16), old.view(torch.int16))


def _recorded(step, extra):
    """The pass and its verification as one graph; `extra` holds what the verification writes."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step.forward()  # (the workspace and torch's buffers exist before the capture)
        ops.verify_tree(step.P, step.P, step.tokens, step.parents, *extra)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step.forward()
        ops.verify_tree(step.P, step.P, step.tokens, step.parents, *extra)
        ops.cache_append(step.K, step.V, extra[2], extra[3], *step.caches, step.lens)
        step.lens.add_(extra[3])
    return graph


def test_a_recorded_step_replays_the_eager_bits():
    model, B, n, T = Model(), 2, 60, 9
    parents = [-1, 0, 0, 1, 1, 2, 5, 6, 0]

    def fresh():
        step = Step(model, B, T, caches=prompt(model, B, n))
        step.lens.fill_(n)
        step.parents.copy_(torch.tensor(parents).expand(B, T))
        extra = [torch.zeros(B, T, device="cuda"), torch.zeros(B, device="cuda"), torch.zeros(B, T, device="cuda", dtype=torch.int32),
                 torch.zeros(B, device="cuda", dtype=torch.int32), torch.zeros(B, device="cuda", dtype=torch.int32)]
        return step, extra

    def feed(step, extra, seed):
        g = torch.Generator().manual_seed(seed)
        step.tokens.copy_(torch.randint(0, VOCAB, (B, T), generator=g))
        step.positions.copy_(step.lens[:, None] + torch.tensor(depths(parents), device="cuda", dtype=torch.int32))
        extra[0].copy_(torch.rand(B, T, generator=g))
        extra[1].copy_(torch.rand(B, generator=g))

    eager, eager_out = fresh()
    played, played_out = fresh()
    feed(played, played_out, 0)
    graph = _recorded(played, played_out)
    for replay in range(6):
        feed(eager, eager_out, replay)
        feed(played, played_out, replay)
        torch.cuda.synchronize()
        eager.forward()
        ops.verify_tree(eager.P, eager.P, eager.tokens, eager.parents, *eager_out)
        ops.cache_append(eager.K, eager.V, eager_out[2], eager_out[3], *eager.caches, eager.lens)
        eager.lens.add_(eager_out[3])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.P, played.P) and all(torch.equal(a, b) for a, b in zip(eager_out, played_out)), replay
        assert torch.equal(eager.lens, played.lens)
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(eager.caches, played.caches)), replay
    assert int(eager.lens.min()) > n + 6


class _Subclass(torch.Tensor):
    """An object that only the Python body takes."""


def _calls():
    """(name, arguments, keywords, index of each output) of the operators' ordinary forms."""
    g = torch.Generator(device="cuda").manual_seed(3)
    half = lambda *s: torch.randn(*s, device="cuda", generator=g).half()
    f = lambda *s: torch.rand(*s, device="cuda", generator=g)
    z = lambda *s, dtype=torch.float16: torch.zeros(*s, device="cuda", dtype=dtype)
    words = lambda N, K: torch.randint(-2 ** 31, 2 ** 31, (N, K // 8), device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
    i = lambda *v: torch.tensor(v, device="cuda", dtype=torch.int32)
    yield "gemv_q4", [half(256), words(24, 256), half(24, 8).abs(), half(24), z(24)], {}, [4]
    yield "gemv_q4", [half(1, 5, 256), words(24, 256).view(torch.uint32), half(24, 2).abs(), None, z(1, 5, 24)], {"epilogue": 3}, [4]
    yield "gemv_q4", [half(5, 256), words(24, 256), half(24, 4).abs(), half(24), z(5, 24, dtype=torch.float32), 2, half(5, 24), half(5, 24)], {}, [4]
    parents, lens = i(-1, 0, 0, -1, 0, 1).view(2, 3), i(9, 4)
    tree = [half(2, 3, 4, 64), half(2, 3, 2, 64), half(2, 3, 2, 64), half(2, 2, 10, 64), half(2, 2, 10, 64), lens, parents, z(2, 3, 4, 64)]
    yield "attn_tree", tree, {}, [7]
    yield "attn_tree", [*tree[:7], z(2, 3, 4, 64)], {"scale": 0.5}, [7]
    target, draft = torch.softmax(half(2, 3, 40).float(), -1), torch.softmax(half(2, 3, 40).float(), -1)
    outs = [z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32), z(2, dtype=torch.int32)]
    yield "verify_tree", [target, draft, i(1, 7, 9, 2, 5, 39).view(2, 3), parents, f(2, 3), f(2) * 0.5 + 0.4, *outs], {}, [6, 7, 8]
    yield "cache_append", [half(2, 2, 3, 2, 64), half(2, 2, 3, 2, 64), i(0, 2, -1, 0, 1, 2).view(2, 3), i(2, 3), z(2, 2, 2, 10, 64), z(2, 2, 2, 10, 64), i(0, 7)], {}, [4, 5]
    yield "cache_append", [half(2, 3, 2, 64), half(2, 3, 2, 64), None, None, z(2, 2, 10, 64), z(2, 2, 10, 64), i(4, 7)], {}, [4, 5]


def test_the_native_check_and_the_body_are_one_function(monkeypatch):
    for name, args, kw, outs in _calls():
        took = []
        native = getattr(ops._fastcall, "_" + name)
        results = []
        for as_given in (True, False):
            for at in outs:
                args[at].zero_()
            given = args if as_given else [a.as_subclass(_Subclass) if isinstance(a, torch.Tensor) else a for a in args]
            with monkeypatch.context() as m:
                m.setattr(ops._fastcall, "_" + name, lambda *a: took.append(native(*a)) or took[-1])
                getattr(ops, name)(*given, **kw)
            results.append([args[at].clone() for at in outs])
        assert took == [True, False], name
        for one, other in zip(*results):
            assert one.count_nonzero() > 0 and torch.equal(one, other), name


def test_calls_after_an_error_go_on():
    h2 = lambda *s: torch.ones(*s, device="cuda", dtype=torch.float16)
    i = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)
    out = h2(1, 1, 4, 64)
    with pytest.raises(RuntimeError, match="share 3 key heads"):
        ops.attn_tree(h2(1, 1, 4, 64), h2(1, 1, 3, 64), h2(1, 1, 3, 64), h2(1, 3, 5, 64), h2(1, 3, 5, 64), i(1), i(1, 1), out)
    ops.attn_tree(h2(1, 1, 4, 64), h2(1, 1, 2, 64), h2(1, 1, 2, 64), h2(1, 2, 5, 64), h2(1, 2, 5, 64), i(1), i(1, 1), out)
    assert bool((out == 1).all())


def test_two_streams_and_two_threads_at_once():
    model = Model()
    steps = []
    for i in range(2):
        step = Step(model, 2, 5, caches=prompt(model, 2, 50 + i))
        step.lens.fill_(50 + i)
        step.parents.copy_(torch.arange(-1, 4).expand(2, 5))
        step.positions.copy_(50 + i + torch.arange(5).expand(2, 5))
        step.tokens.copy_(torch.randint(0, VOCAB, (2, 5), generator=torch.Generator().manual_seed(i)))
        step.forward()
        steps.append((step, step.P.clone()))
    torch.cuda.synchronize()
    wrong = []

    def work(step, want):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                step.forward()
                if not torch.equal(step.P, want):
                    wrong.append(step)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=s) for s in steps]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_two_recorded_graphs_share_a_workspace():
    # recorded on one stream, the second needing a larger workspace than the first; lengths change between the replays
    g = torch.Generator(device="cuda").manual_seed(9)
    half = lambda *s: torch.randn(*s, device="cuda", generator=g).half()
    words = lambda N, K: torch.randint(-2 ** 31, 2 ** 31, (N, K // 8), device="cuda", generator=g, dtype=torch.int64).to(torch.int32)

    def attention(B, T, heads, kv, d, capacity):
        parents = torch.arange(-1, T - 1, device="cuda", dtype=torch.int32).expand(B, T).contiguous()
        return [half(B, T, heads, d), half(B, T, kv, d), half(B, T, kv, d), half(B, kv, capacity, d), half(B, kv, capacity, d),
                torch.zeros(B, device="cuda", dtype=torch.int32), parents]

    small = [attention(2, 3, 4, 2, 64, 3000), attention(1, 48, 4, 1, 128, 2000)]
    large = [attention(3, 64, 32, 8, 128, 6000), attention(2, 1, 16, 8, 256, 3000)]
    x, Wq, scale = half(20, 10240), words(300, 10240), half(300, 320).abs() * 0.01
    target = torch.softmax(half(3, 5, 9000).float(), -1)
    verify = [target, torch.softmax(half(3, 5, 9000).float(), -1), torch.randint(0, 9000, (3, 5), device="cuda", generator=g, dtype=torch.int64).to(torch.int32),
              torch.tensor([-1, 0, 0, 1, 1], device="cuda", dtype=torch.int32).expand(3, 5).contiguous(), torch.rand(3, 5, device="cuda", generator=g),
              torch.rand(3, device="cuda", generator=g)]

    def outputs(sets):
        return [torch.zeros_like(s[0]) for s in sets] + [torch.zeros(20, 300, device="cuda", dtype=torch.float16)] + \
               [torch.zeros(3, 5, device="cuda", dtype=torch.int32), torch.zeros(3, device="cuda", dtype=torch.int32), torch.zeros(3, device="cuda", dtype=torch.int32)]

    def run(sets, out):
        for s, o in zip(sets, out):
            ops.attn_tree(*s, o)
        ops.gemv_q4(x, Wq, scale, None, out[2])
        ops.verify_tree(*verify, *out[3:])

    stream, graphs = torch.cuda.Stream(), []
    for sets in (small, large):
        played = outputs(sets)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run(sets, played)
        graphs.append((graph, sets, played))
    for replay in range(8):
        graph, sets, played = graphs[replay % 2]
        for s in sets:
            s[5].copy_(torch.tensor([(replay * 977 + b * 1403) % (s[3].shape[2] + 1) for b in range(s[0].shape[0])]))
        for t in played:
            t.zero_()
        eager = outputs(sets)
        run(sets, eager)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        for one, other in zip(played, eager):
            assert torch.equal(one, other), replay


def test_a_recorded_graph_keeps_the_workspace_that_a_larger_one_outgrew():
    # The first recording takes the stream's first workspace.  The second needs a larger one, in sums (two parts of K for each tile of 32 x 64: 69 MB) and in counters (4224 tiles),
    # and the library allocates it while it is recorded: seen in the memory that is left.  The first one's replays go on in what it recorded.
    g = torch.Generator(device="cuda").manual_seed(21)
    half = lambda *s: torch.randn(*s, device="cuda", generator=g).half()

    def product(M, N, K):
        words = torch.randint(-2 ** 31, 2 ** 31, (N, K // 8), device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
        return half(M, K), words, half(N, K // 32).abs() * 0.01

    parents = torch.arange(-1, 15, device="cuda", dtype=torch.int32).view(1, 16)
    tree = [half(1, 16, 8, 64), half(1, 16, 2, 64), half(1, 16, 2, 64), half(1, 2, 3000, 64), half(1, 2, 3000, 64), torch.full((1,), 2900, device="cuda", dtype=torch.int32), parents]
    sets = [product(20, 300, 10240), product(2100, 4096, 5120)]

    def run(product, out):
        ops.gemv_q4(*product, None, out[0])
        ops.attn_tree(*tree, out[1])

    def outputs(product):
        return [torch.zeros(product[0].shape[0], product[1].shape[0], device="cuda", dtype=torch.float16), torch.zeros_like(tree[0])]

    ops.gemv_q4(*sets[0], None, outputs(sets[0])[0])
    stream, graphs, grown = torch.cuda.Stream(), [], []
    for product in sets:
        played, eager = outputs(product), outputs(product)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            left = torch.cuda.mem_get_info()[0]
            run(product, played)
            grown.append(left - torch.cuda.mem_get_info()[0])
        graphs.append((graph, product, played, eager))
    assert grown[0] >= 32 << 20 and grown[1] >= 64 << 20, grown
    for replay in range(8):
        graph, product, played, eager = graphs[(0, 1, 0, 0, 1, 1, 0, 1)[replay]]
        tree[5].fill_(2900 - 413 * replay)
        for t in (*played, *eager):
            t.zero_()
        run(product, eager)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        for one, other in zip(played, eager):
            assert one.count_nonzero() > 0 and torch.equal(one, other), replay
