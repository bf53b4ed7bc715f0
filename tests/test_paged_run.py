"""Requests served from one pool, step by step: prompts in, beams handed their pages, tokens appended, read, chosen and followed, pages given back -- against caches that
are one tensor per beam."""
import threading
import types

import pytest
import torch

from dtas_amd import ops
from test_parity_paged import chosen, expected, ints

pytestmark = pytest.mark.gpu

L, HKV, GROUP, D, PAGE, V = 2, 2, 2, 64, 16, 1200
EOS = 7


class Served:
    """G requests of W beams: the pool, the tables and the stack on the device."""

    def __init__(self, G, W, columns, pages, seed=0):
        g = torch.Generator().manual_seed(seed)
        i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        self.G, self.W, self.columns, self.pages = G, W, columns, pages
        self.table, self.lens = i(G, W, columns), i(G, W)
        self.table.fill_(-1)
        self.free, self.height = torch.randperm(pages, generator=g).int().cuda(), ints([pages]).cuda()
        self.K, self.V = (torch.full((L, pages, HKV, PAGE, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
        self.scores = torch.full((G, W), -float("inf"), device="cuda")
        self.scores[:, 0] = 0
        self.done, self.tokens, self.parents = i(G, W), i(G, W), i(G, W)
        self.slots, self.one = i(G * W, 1), i(G * W).fill_(1)
        self.keys, self.values = (torch.zeros(L, G * W, HKV, D, dtype=torch.float16, device="cuda") for _ in range(2))
        self.Q = torch.zeros(L, G * W, HKV * GROUP, D, dtype=torch.float16, device="cuda")
        self.out = torch.zeros_like(self.Q)
        self.logits = torch.zeros(G, W, V, device="cuda")

    def prompt(self, lengths, keys, values):
        """Prompts of the requests' first beams, packed; then each is all its beams'."""
        count = torch.zeros(self.G, self.W, dtype=torch.int32)
        count[:, 0] = ints(lengths)
        starts, slots = torch.zeros(self.G * self.W + 1, dtype=torch.int32, device="cuda"), torch.zeros(keys.shape[1], dtype=torch.int32, device="cuda")
        flat = self.lens.view(-1)
        ops.page_assign(flat, count.view(-1).cuda(), self.table.view(-1, self.columns), self.free, self.height, PAGE, slots, flat, self.height, starts=starts)
        ops.page_append(keys, values, slots, self.K, self.V)
        self.parents.zero_()
        self.follow()
        return starts

    def follow(self):
        ops.page_reorder(self.parents, self.table, self.lens, self.free, self.height, self.table, self.lens, self.height, self.K, self.V)

    def step(self):
        """A token of every beam (its keys, values, queries and logits are there): in, read, chosen, followed."""
        flat, table = self.lens.view(-1), self.table.view(-1, self.columns)
        ops.page_assign(flat, self.one, table, self.free, self.height, PAGE, self.slots, flat, self.height)
        ops.page_append(self.keys, self.values, self.slots, self.K, self.V)
        for l in range(L):
            ops.attn_paged(self.Q[l], self.K[l], self.V[l], table, flat, self.out[l], None, self.W)
        ops.beam_select(self.logits, self.scores, self.done, self.tokens, self.parents, self.scores, self.done, EOS)
        self.follow()

    def state(self):
        return [t.clone() for t in (self.table, self.lens, self.free, self.height, self.scores, self.done, self.tokens, self.parents, self.out, self.K, self.V)]

    def restore(self, state):
        for t, s in zip((self.table, self.lens, self.free, self.height, self.scores, self.done, self.tokens, self.parents, self.out, self.K, self.V), state):
            t.copy_(s)

    def fill(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (self.keys, self.values, self.Q, self.logits):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        self.logits *= 2


def held(s, b):
    """Sequence b's keys and values, of all layers, and the pages that it names."""
    n = int(s.lens.view(-1)[b])
    names = s.table.view(-1, s.columns)[b, :-(-n // PAGE)].long()
    flat = lambda pool: pool[:, names].permute(0, 2, 1, 3, 4).reshape(L, HKV, -1, D)[:, :, :n].cpu()
    return flat(s.K), flat(s.V), names.tolist()


def check_pool(s):
    """Every page is named by one group, or on the stack, once."""
    stack = s.free[:int(s.height)].tolist()
    named = [{p for w in range(s.W) for p in held(s, i * s.W + w)[2]} for i in range(s.G)]
    assert sorted(stack + [p for n in named for p in n]) == list(range(s.pages))
    for i in range(s.G):  # the page that a row is filling belongs to it alone
        filling = [held(s, i * s.W + w)[2][-1] for w in range(s.W) if int(s.lens[i, w]) % PAGE]
        for w in range(s.W):
            names = held(s, i * s.W + w)[2]
            for p in filling:
                assert p not in names or p == names[-1]
        assert len(filling) == len(set(filling))


@pytest.mark.parametrize("G,W,lengths,steps", [(1, 1, [5], 20), (1, 4, [33], 20), (3, 4, [1, 16, 40], 36), (2, 8, [15, 700], 20), (5, 3, [0, 31, 32, 100, 2], 18)])
def test_requests_from_prompt_to_end(G, W, lengths, steps):
    columns = -(-(max(lengths) + steps) // PAGE)
    s = Served(G, W, columns, G * W * columns + 2)
    g = torch.Generator().manual_seed(G + W)
    keys, values = (torch.randn(L, sum(lengths) + 3, HKV, D, generator=g).half() for _ in range(2))
    starts = s.prompt(lengths, keys.cuda(), values.cuda())
    begin = [sum(lengths[:i]) for i in range(G)]
    assert starts.tolist() == [begin[b // W] + (lengths[b // W] if b % W else 0) for b in range(G * W)] + [sum(lengths)]
    caches = [[t[:, begin[b // W]:begin[b // W] + lengths[b // W]].transpose(1, 2) for t in (keys, values)] for b in range(G * W)]
    check_pool(s)
    for step in range(steps):
        s.fill(step)
        before = [t.cpu() for t in (s.logits, s.scores, s.done)]
        want = chosen(*before, EOS)
        s.step()
        for b in range(G * W):
            caches[b] = [torch.cat((c, t[:, b, :, None].cpu()), 2) for c, t in zip(caches[b], (s.keys, s.values))]
        for l in range(L):
            for b in range(G * W):
                k, v = caches[b]
                n = k.shape[2]
                host = {"Q": s.Q[l, b:b + 1].cpu(), "K": k[l][None], "V": v[l][None], "table": ints([[0]]), "lens": ints([n])}
                out, slack = expected(host)
                assert bool(((s.out[l, b:b + 1].cpu().double() - out).abs() <= slack).all())
        assert torch.equal(s.tokens.cpu(), want[0]) and torch.equal(s.parents.cpu(), want[1]) and torch.equal(s.done.cpu(), want[3])
        caches = [caches[b // W * W + int(want[1].view(-1)[b])] for b in range(G * W)]
        assert s.lens.view(-1).tolist() == [c[0].shape[2] for c in caches]
        for b in range(G * W):
            k, v, _ = held(s, b)
            assert torch.equal(k, caches[b][0]) and torch.equal(v, caches[b][1])
        check_pool(s)
    s.parents.fill_(-1)
    s.follow()
    assert s.lens.eq(0).all() and s.height.tolist() == [s.pages] and sorted(s.free.tolist()) == list(range(s.pages))


@pytest.mark.parametrize("beams", [1, 3])
def test_pages_give_what_one_cache_gives(beams):
    # the same keys in one tensor per sequence, read as a tree of one node (the token's own)
    B, n = 6, 500
    g = torch.Generator().manual_seed(beams)
    K, Vv = (torch.randn(B, HKV, n, D, generator=g).half() for _ in range(2))
    Q = torch.randn(B, 1, HKV * GROUP, D, generator=g).half().cuda()
    pages = n // PAGE + 1
    table = torch.randperm(B * pages, generator=g).int().view(B, pages)
    pools = [torch.zeros(1, B * pages, HKV, PAGE, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    slots = torch.stack([table[b, torch.arange(n) // PAGE] * PAGE + torch.arange(n) % PAGE for b in range(B)]).int().cuda()
    ops.page_append(*(t.transpose(1, 2).reshape(1, B * n, HKV, D).contiguous().cuda() for t in (K, Vv)), slots, *pools)
    lens = ints([n, 1, 17, 400, 256, 499])
    last = lens.long() - 1
    own = [torch.stack([t[b, :, last[b]] for b in range(B)])[:, None].cuda() for t in (K, Vv)]
    one, two = torch.zeros_like(Q), torch.zeros_like(Q)
    ops.attn_paged(Q[:, 0], pools[0][0], pools[1][0], table.cuda(), lens.cuda(), one[:, 0], None, beams)
    ops.attn_tree(Q, *own, K.cuda(), Vv.cuda(), (lens - 1).cuda(), torch.full((B, 1), -1, dtype=torch.int32, device="cuda"), two)
    host = {"Q": Q[:, 0].cpu(), "K": pools[0][0].cpu(), "V": pools[1][0].cpu(), "table": table, "lens": lens}
    assert bool(((one - two)[:, 0].cpu().double().abs() <= 2 * expected(host)[1]).all())


def test_both_ways_into_the_library_are_one_function(monkeypatch):
    # the natively checked call and the Python body: the same bits, and the same refusals
    s = Served(2, 3, 4, 30)
    keys = torch.randn(L, 50, HKV, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).half()
    names = ("_page_assign", "_page_append", "_attn_paged", "_beam_select", "_page_reorder")
    calls = {n: 0 for n in names}

    def counted(n):
        def call(*args):
            taken = getattr(ops_fast, n)(*args)
            calls[n] += bool(taken)
            return taken
        return call

    ops_fast = ops._fastcall
    fill = lambda: s.fill(3)
    start = s.state()
    results = []
    for way in (counted, lambda n: lambda *args: False):
        monkeypatch.setattr(ops, "_fastcall", types.SimpleNamespace(**{n: way(n) for n in names}))
        s.restore(start)
        s.prompt([17, 30], keys, -keys)
        fill()
        for _ in range(3):
            s.step()
        results.append(s.state())
        with pytest.raises(Exception):
            ops.page_assign(s.lens, s.one, s.table, s.free, s.height, PAGE, s.slots, s.lens, s.height)
        with pytest.raises(Exception):
            ops.page_append(s.keys, s.values, s.slots.float(), s.K, s.V)
        with pytest.raises(Exception):
            ops.attn_paged(s.Q[0], s.K[0], s.V[0], s.table.view(6, 4), s.lens.view(-1), s.out[0], None, 4)
        with pytest.raises(Exception):
            ops.beam_select(s.logits, s.scores, s.done, s.tokens, s.parents, s.scores, None, EOS)
        with pytest.raises(Exception):
            ops.page_reorder(s.parents, s.table[..., ::2], s.lens, s.free, s.height, s.table, s.lens, s.height, s.K, s.V)
    assert calls == {"_page_assign": 4, "_page_append": 4, "_attn_paged": 6, "_beam_select": 3, "_page_reorder": 4}
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.int16) if a.dtype == torch.float16 else a, b.view(torch.int16) if b.dtype == torch.float16 else b)


def test_streams_and_threads_side_by_side():
    # each with requests of its own and the workspace of its stream; the same bits as alone
    def run(seed, stream):
        with torch.cuda.stream(stream):
            s = Served(3, 4, 50, 3 * 4 * 50, seed)
            keys = torch.randn(L, 1600, HKV, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).half()
            s.prompt([700, 300, 600], keys, -keys)
            for i in range(12):
                s.fill(seed + i)
                s.step()
            out = s.state()
            stream.synchronize()
            return out

    streams = [torch.cuda.Stream() for _ in range(3)]
    alone = [run(10 * i, torch.cuda.current_stream()) for i in range(3)]
    got = [None] * 3

    def work(i):
        got[i] = run(10 * i, streams[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, got):
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.int16) if x.dtype == torch.float16 else x, y.view(torch.int16) if y.dtype == torch.float16 else y)


def test_a_step_gives_the_same_bits_again():
    # what is handed over between workgroups arrives in any order; it is joined in one
    s = Served(4, 4, 80, 4 * 4 * 80)
    keys = torch.randn(L, 2000, HKV, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    s.prompt([1200, 100, 600, 90], keys, -keys)
    s.fill(4)
    start = s.state()
    s.step()
    first = s.state()
    for _ in range(20):
        s.restore(start)
        s.step()
        for x, y in zip(first, s.state()):
            assert torch.equal(x.view(torch.int16) if x.dtype == torch.float16 else x, y.view(torch.int16) if y.dtype == torch.float16 else y)
