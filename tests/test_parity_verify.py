"""Verification of drafted tokens, and what is kept of them, against the definitions."""
import math

import pytest
import torch

from dtas_amd import ops

pytestmark = pytest.mark.gpu


def walk(target, draft, tokens, parents, accept, sample):
    """One sequence by the recursive definition, in 64 bits: the path and the next token."""
    T, V = target.shape
    at, path = 0, [0]
    while True:
        p, q = target[at].double(), draft[at].double()
        here, step = p.clone(), None
        for i in range(at + 1, T):
            x = int(tokens[i])
            if int(parents[i]) != at or not 0 <= x < V:
                continue
            if float(accept[i]) * float(q[x]) < float(here[x]):
                step = i
                break
            left = torch.relu(here - q)
            here = left / left.sum() if float(left.sum()) > 0 else left
        if step is None:
            break
        path.append(step)
        at = step
    if not float(here.sum()) > 0:
        here = p
    upto = torch.cumsum(here, 0)
    behind = torch.nonzero(upto > float(sample) * upto[-1])
    some = torch.nonzero(here > 0)
    return path, int(behind[0]) if len(behind) else int(some[-1]) if len(some) else -1


def run(target, draft, tokens, parents, accept, sample):
    B, T, _ = target.shape
    wide = [torch.full((n + 128,), 777, device="cuda", dtype=torch.int32) for n in (B * T, B, B)]
    path, count, nxt = (w[64:-64] for w in wide)
    ops.verify_tree(target.cuda(), draft.cuda(), tokens.cuda(), parents.cuda(), accept.cuda(), sample.cuda(), path.view(B, T), count, nxt)
    torch.cuda.synchronize()
    assert all(bool((w[:64] == 777).all()) and bool((w[-64:] == 777).all()) for w in wide)
    return path.view(B, T).cpu(), count.cpu(), nxt.cpu()


def check(target, draft, tokens, parents, accept, sample):
    path, count, nxt = run(target, draft, tokens, parents, accept, sample)
    B, T, _ = target.shape
    for b in range(B):
        want, token = walk(target[b], draft[b], tokens[b], parents[b], accept[b], sample[b])
        assert path[b].tolist() == want + [-1] * (T - len(want)), (b, path[b].tolist(), want)
        assert int(count[b]) == len(want) and int(nxt[b]) == token, (b, int(nxt[b]), token)
    return path, count, nxt


def make(B, T, V, shape="tree", seed=0, near=0.5):
    """Distributions, a tree each, tokens drawn from the drafts, uniform numbers."""
    g = torch.Generator().manual_seed(seed + 31 * T + V)
    logits = torch.randn(B, T, V, generator=g) * 2
    target, draft = torch.softmax(logits, -1), torch.softmax(logits + near * torch.randn(B, T, V, generator=g), -1)
    parents = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        for i in range(1, T):
            parents[b, i] = i - 1 if shape == "chain" else 0 if shape == "star" else int(torch.randint(max(0, i - 6), i, (1,), generator=g))
    tokens = torch.zeros(B, T, dtype=torch.int32)
    for b in range(B):
        tokens[b] = torch.multinomial(draft[b, parents[b].clamp(min=0).long()], 1, generator=g)[:, 0].to(torch.int32)
    return target, draft, tokens, parents, torch.rand(B, T, generator=g), torch.rand(B, generator=g)


@pytest.mark.parametrize("shape", ["chain", "star", "tree"])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (1, 2, 2), (3, 4, 7), (2, 5, 63), (2, 16, 64), (4, 9, 1000), (1, 64, 257), (5, 3, 4097), (2, 31, 8191), (1, 5, 50280), (2, 8, 128256)])
def test_sizes(B, T, V, shape):
    check(*make(B, T, V, shape))


@pytest.mark.parametrize("near", [0.0, 0.05, 2.0])
def test_near_and_far_drafts(near):
    check(*make(8, 16, 500, "tree", near=near))
    check(*make(8, 40, 33, "star", near=near))


def test_many_sequences():
    check(*make(300, 6, 100))


def test_every_child_refused():
    # accept = 1 - 2^-24 against tokens that the draft holds too likely: the walk stays at the root and refuses all
    target, draft, tokens, parents, accept, sample = make(4, 33, 50, "star", near=1.5)
    tokens[:] = (draft[:, 0] / target[:, 0]).argmax(-1, keepdim=True).to(torch.int32)
    accept[:] = 1 - 2.0 ** -24
    _, count, _ = check(target, draft, tokens, parents, accept, sample)
    assert count.tolist() == [1] * 4


def test_certain_acceptance_walks_to_the_end():
    target, _, tokens, parents, accept, sample = make(3, 64, 40, "chain")
    _, count, _ = check(target, target.clone(), tokens, parents, accept, sample)
    assert count.tolist() == [64] * 3


def test_tokens_that_are_no_tokens_and_nodes_without_a_parent():
    target, draft, tokens, parents, accept, sample = make(6, 12, 30)
    tokens[0, 1], tokens[1, 2], tokens[2, 1:], parents[3, 4], parents[4, 3], parents[5, 1] = -1, 30, -5, 4, 11, -1
    parents[:, 0] = torch.tensor([3, -1, 0, 99, -7, 5], dtype=torch.int32)   # (node 0 leads whatever stands there)
    check(target, draft, tokens, parents, accept, sample)


def test_the_ends_of_the_sample():
    target, draft, tokens, parents, accept, sample = make(8, 3, 1000)
    for value in (0.0, 2.0 ** -24, 1 - 2.0 ** -24):
        check(target, draft, tokens, parents, accept, torch.full_like(sample, value))


def test_exact_borders():
    # powers of two: prefix sums and goals are exact, and the token behind a border is the one that exceeds it
    for V in (4, 256, 4096):
        target = torch.full((V, 1, V), 1 / V)
        sample = torch.arange(V).float() / V
        zero = torch.zeros(V, 1)
        _, _, nxt = run(target, target, zero.int(), zero.int() - 1, zero, sample)
        assert nxt.tolist() == list(range(V))


def test_tokens_without_probability_are_never_chosen():
    B, V = 64, 2000
    g = torch.Generator().manual_seed(2)
    target = torch.rand(B, 1, V, generator=g)
    keep = torch.rand(B, 1, V, generator=g) < 0.01
    target = torch.where(keep, target, torch.zeros(()))
    target = target / target.sum(-1, keepdim=True)
    zero = torch.zeros(B, 1)
    for value in (0.0, 0.3, 1 - 2.0 ** -24, 1.0, 5.0, float("nan"), -1.0):
        _, _, nxt = run(target, target, zero.int(), zero.int(), zero, torch.full((B,), value))
        assert bool(keep[torch.arange(B), 0, nxt.long()].all())


def test_rows_of_zeros():
    target, draft, tokens, parents, accept, sample = make(2, 3, 40)
    target[0] = 0
    _, count, nxt = run(target, draft, tokens, parents, accept, sample)
    assert int(nxt[0]) == -1 and int(count[0]) == 1


def test_nothing_left_of_the_target():
    # dyadic rows that are equal: a refusal (of a token the target does not hold) leaves nothing, and the target itself is sampled
    target = torch.zeros(1, 2, 8)
    target[..., 2], target[..., 5] = 0.5, 0.5
    tokens, parents = torch.tensor([[0, 3]], dtype=torch.int32), torch.tensor([[-1, 0]], dtype=torch.int32)
    for r, want in ((0.25, 2), (0.75, 5)):
        _, count, nxt = run(target, target.clone(), tokens, parents, torch.full((1, 2), 0.5), torch.tensor([r]))
        assert int(count) == 1 and int(nxt) == want


def test_what_is_chosen_is_distributed_as_the_target():
    # two draws from the draft below the root, then the rest: the first chosen token follows the target.  Frequencies of n draws are off by
    # sqrt(p (1 - p) / n) at a standard deviation; five of them, for six tokens of one fixed draw
    n, V = 200000, 6
    g = torch.Generator().manual_seed(4)
    p, q = torch.tensor([0.4, 0.05, 0.2, 0.1, 0.24, 0.01]), torch.tensor([0.1, 0.3, 0.2, 0.25, 0.1, 0.05])
    target, draft = p.expand(n, 3, V).contiguous(), q.expand(n, 3, V).contiguous()
    tokens = torch.multinomial(q, 3 * n, replacement=True, generator=g).view(n, 3).to(torch.int32)
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32).expand(n, 3).contiguous()
    path, count, nxt = run(target, draft, tokens, parents, torch.rand(n, 3, generator=g), torch.rand(n, generator=g))
    first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], nxt)
    share = torch.bincount(first.long(), minlength=V).double() / n
    assert bool(((share - p.double()).abs() <= 5 * torch.sqrt(p.double() * (1 - p.double()) / n)).all()), share
    assert 0.3 < float((count > 1).float().mean()) < 0.95


def test_refusals_of_verify():
    f = lambda *s: torch.zeros(*s, device="cuda")
    i = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)
    good = [f(2, 3, 9), f(2, 3, 9), i(2, 3), i(2, 3), f(2, 3), f(2), i(2, 3), i(2), i(2)]
    ops.verify_tree(*good)
    for at, bad, why in ((0, f(2, 9), "expects target"), (1, f(2, 3, 8), "expects target"), (1, f(2, 3, 9).half(), "expects fp32"), (2, i(2, 4), "shape"),
                         (3, i(2, 3).long(), "int32"), (4, f(3, 2), "shape"), (5, f(2, 1), "shape"), (6, i(2), "shape"), (7, i(3), "shape"), (8, f(2), "int32")):
        with pytest.raises(ValueError, match=why):
            ops.verify_tree(*good[:at], bad, *good[at + 1:])


# ---- cache_append ----------------------------------------------------------------------------------------------------
def append_case(lead, B, T, Hkv, d, C, slots, seed=0, offset=0):
    g = torch.Generator().manual_seed(seed)

    def there(*s):
        raw = torch.randn(math.prod(s) + offset, generator=g).half().cuda()
        return raw[offset:].view(*s)

    new = [there(*lead, B, T, Hkv, d) for _ in range(2)]
    caches = [there(*lead, B, Hkv, C, d) for _ in range(2)]
    path = torch.randint(0, T, (B, slots), generator=g).to(torch.int32) if slots else None
    return new, caches, path


def appended(new, cache, path, count, lens):
    """The definition, row by row."""
    cache = cache.cpu().clone()
    new = new.cpu()
    B, T, C = new.shape[-4], new.shape[-3], cache.shape[-2]
    for b in range(B):
        for j in range(T if path is None else min(int(count[b]), path.shape[1])):
            node, row = j if path is None else int(path[b, j]), int(lens[b]) + j
            if 0 <= node < T and 0 <= row < C:
                cache[..., b, :, row, :] = new[..., b, node, :, :]
    return cache


def check_append(new, caches, path, count, lens):
    want = [appended(n, c, path, count, lens) for n, c in zip(new, caches)]
    up = lambda t: None if t is None else t.cuda()
    ops.cache_append(*new, up(path), up(count), *caches, lens.cuda())
    for c, w in zip(caches, want):
        assert torch.equal(c.cpu().view(torch.int16), w.view(torch.int16))


@pytest.mark.parametrize("lead", [(), (3,), (2, 2)])
@pytest.mark.parametrize("B,T,Hkv,d,C", [(1, 1, 1, 8, 4), (2, 5, 3, 80, 40), (3, 25, 2, 128, 64), (1, 64, 8, 72, 100), (2, 7, 2, 20, 33), (4, 3, 1, 256, 9), (2, 300, 2, 64, 700)])
def test_append(lead, B, T, Hkv, d, C):
    lens = torch.tensor([(7 * b) % max(1, C - T + 1) for b in range(B)], dtype=torch.int32)
    new, caches, path = append_case(lead, B, T, Hkv, d, C, T)
    check_append(new, caches, path, torch.tensor([(3 * b) % (T + 1) for b in range(B)], dtype=torch.int32), lens)
    new, caches, _ = append_case(lead, B, T, Hkv, d, C, 0, 1)
    check_append(new, caches, None, None, lens)


def test_append_leaves_out_what_has_no_place():
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    new, caches, path = append_case((2,), 6, 8, 2, 64, 20, 5)
    path[0], path[1, 2], path[2, 0] = i(-1, 8, 99, -2147483648, 2147483647), -1, 3
    check_append(new, caches, path, i(5, 5, 99, -3, 5, 2147483647), i(0, 18, 20, 3, -2, 17))
    check_append(new, caches, path, i(5, 5, 5, 5, 5, 5), i(2147483647, -2147483648, 2147483645, 19, 21, -4))
    new, caches, _ = append_case((), 3, 8, 2, 64, 10, 0)
    check_append(new, caches, None, None, i(5, 0, -7))


@pytest.mark.parametrize("offset", [1, 4])
def test_append_off_every_boundary(offset):
    new, caches, path = append_case((2,), 2, 5, 2, 64, 30, 5, offset=offset)
    check_append(new, caches, path, torch.tensor([4, 2], dtype=torch.int32), torch.tensor([3, 9], dtype=torch.int32))


def test_append_past_32_bits():
    B, Hkv, C, d = 2, 8, 1310720, 128
    caches = [torch.empty(B, Hkv, C, d, device="cuda", dtype=torch.float16) for _ in range(2)]
    new, _, _ = append_case((), B, 3, Hkv, d, 4, 0)
    lens = torch.tensor([C - 3, C - 2], dtype=torch.int32)
    for c in caches:
        c[:, :, -5:] = 0
    ops.cache_append(*new, None, None, *caches, lens.cuda())
    for n, c in zip(new, caches):
        assert torch.equal(c[0, :, -3:].transpose(0, 1), n[0]) and torch.equal(c[1, :, -2:].transpose(0, 1), n[1, :2])
        assert not bool(c[0, :, -5:-3].any()) and not bool(c[1, :, -5:-2].any())


def test_refusals_of_append():
    h = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.float16)
    i = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)
    good = [h(3, 2, 4, 2, 64), h(3, 2, 4, 2, 64), i(2, 4), i(2), h(3, 2, 2, 9, 64), h(3, 2, 2, 9, 64), i(2)]
    ops.cache_append(*good)
    for at, bad, why in ((0, h(3, 2, 4, 2, 32), "shape"), (1, h(2, 2, 4, 2, 64), "shape"), (2, i(3, 4), "shape"), (2, None, "go together"), (3, i(3), "shape"),
                         (4, h(2, 2, 2, 9, 64), "shape"), (5, h(3, 2, 2, 8, 64), "shape"), (6, i(3), "shape"), (6, i(2).long(), "int32"),
                         (4, h(2, 2, 9, 64), "expects K"), (0, h(3, 2, 4, 2, 64).float(), "expects fp16")):
        with pytest.raises(ValueError, match=why):
            ops.cache_append(*good[:at], bad, *good[at + 1:])
