"""Attention of a tree of drafted tokens over a cache against the definition in 64 bits."""
import math

import pytest
import torch

from dtas_amd import ops
from gpu_util import Guarded

pytestmark = pytest.mark.gpu


def forest(T, g, shape):
    """Parents of T nodes: a chain, a star, nodes with parents anywhere before them, or several roots and values to be ignored."""
    if shape == "chain":
        return [i - 1 for i in range(T)]
    if shape == "star":
        return [-1] + [0] * (T - 1)
    draw = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))
    if shape == "any":
        return [-1] + [draw(max(0, i - 6), i) for i in range(1, T)]
    return [draw(-3, T + 3) if i % 3 else -7 - i for i in range(T)]  # (at or behind the node itself: no parent)


def make(B, T, Tq, Hkv, group, d, lens, capacity, shape="any", seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed + 1000 * T + d)
    n = lambda *s: torch.randn(*s, generator=g)
    host = {"Q": (n(B, Tq, Hkv * group, d) * spread).half(), "K": n(B, T, Hkv, d).half(), "V": n(B, T, Hkv, d).half(),
            "Kc": n(B, Hkv, capacity, d).half(), "Vc": n(B, Hkv, capacity, d).half(), "lens": torch.tensor(lens, dtype=torch.int32),
            "parents": torch.tensor([forest(T, g, shape) for _ in range(B)], dtype=torch.int32)}
    return host


def seen_by(parents, node):
    line = [node]
    while 0 <= parents[node] < node:
        node = parents[node]
        line.append(node)
    return line


def expected(host, scale=None):
    """The value, and how far an answer may be from it.

    Scores: d products in fp32, (d + 8) 2^-24 of their magnitudes, times the scale: e.  Probabilities, in units of the largest, are rounded
    to fp16 for the product with the values: 2^-11 of each and 2^-25 at least; e on both sides of the quotient; sums of n keys joined in
    any order: n 2^-24.  On the weighted sum of |v| (and of the quotient, |out|).  Storing: 2^-11, 2^-25 at least."""
    Q, K, V, Kc, Vc = (host[k].double() for k in ("Q", "K", "V", "Kc", "Vc"))
    B, Tq, H, d = Q.shape
    T, Hkv, capacity = K.shape[1], K.shape[2], Kc.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, slack = torch.zeros_like(Q), torch.zeros_like(Q)
    for b in range(B):
        n = min(max(int(host["lens"][b]), 0), capacity)
        for t in range(Tq):
            line = seen_by(host["parents"][b].tolist(), T - Tq + t)
            for hk in range(Hkv):
                k, v = torch.cat((Kc[b, hk, :n], K[b, line, hk])), torch.cat((Vc[b, hk, :n], V[b, line, hk]))
                q = Q[b, t, hk * (H // Hkv):(hk + 1) * (H // Hkv)]
                p = torch.softmax(q @ k.t() * scale, -1)
                e = (d + 8) * 2.0 ** -24 * abs(scale) * (q.abs() @ k.abs().t()).amax(-1, keepdim=True)
                out[b, t, hk * (H // Hkv):(hk + 1) * (H // Hkv)] = o = p @ v
                # (the smallest a probability can be in units of the largest is nothing: 2^-25 for each of the n keys, over a sum of 1 or more)
                weight = (2.0 ** -11 + 2 * e + len(k) * 2.0 ** -23 + 2.0 ** -21) * (p @ v.abs() + o.abs()) + 2.0 ** -25 * len(k) * (p.amax(-1, keepdim=True) * v.abs().amax(0) * 2)
                slack[b, t, hk * (H // Hkv):(hk + 1) * (H // Hkv)] = weight + 2.0 ** -11 * (o.abs() + weight) + 2.0 ** -25
    return out, slack


def launch(host, scale=None, offset=0):
    def there(t):
        raw = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
        raw[offset:] = t.flatten().cuda()
        return raw[offset:].view(t.shape)

    out = Guarded(tuple(host["Q"].shape), torch.float16)
    ops.attn_tree(*(there(host[k]) for k in ("Q", "K", "V", "Kc", "Vc")), host["lens"].cuda(), host["parents"].cuda(), out.t, scale)
    return torch.from_numpy(out.check())


def check(host, scale=None, offset=0):
    got = launch(host, scale, offset).double()
    want, tolerance = expected(host, scale)
    off = (got - want).abs() - tolerance
    assert bool((off <= 0).all()), (off.max().item(), (off > 0).sum().item(), int(torch.isnan(got).sum()))


@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 104, 128, 160, 192, 256])
@pytest.mark.parametrize("group,T,Tq", [(1, 1, 1), (4, 5, 5), (3, 17, 4), (8, 9, 9)])
def test_head_dimensions(d, group, T, Tq):
    check(make(2, T, Tq, 2, group, d, [61, 130], 140))


@pytest.mark.parametrize("d", [1, 5, 20, 65, 100, 255])
def test_head_dimensions_off_eight(d):
    check(make(2, 6, 6, 2, 2, d, [33, 0], 40))


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1000, 2049])
@pytest.mark.parametrize("T,group", [(1, 1), (7, 2), (33, 4)])
def test_lengths(length, T, group):
    check(make(1, T, T, 2, group, 80, [length], length + 3))


@pytest.mark.parametrize("shape", ["chain", "star", "any", "loose"])
@pytest.mark.parametrize("T", [2, 16, 31, 32, 33, 48, 64])
def test_trees(T, shape):
    check(make(2, T, T, 1, 2, 64, [40, 7], 50, shape))
    check(make(2, T, max(1, T // 3), 2, 1, 128, [3, 90], 100, shape))


@pytest.mark.parametrize("T,Tq,group", [(64, 64, 8), (64, 5, 8), (40, 40, 3), (1, 1, 16), (3, 3, 32), (64, 64, 1)])
def test_rows_of_a_key_head(T, Tq, group):
    check(make(1, T, Tq, 2, group, 128, [300], 300))


def test_ragged_batches():
    check(make(9, 6, 6, 2, 2, 80, [0, 1, 500, 37, 999, 64, 256, 3, 128], 1000))
    check(make(40, 1, 1, 3, 2, 64, [7 * b for b in range(40)], 280))


@pytest.mark.parametrize("B,Hkv,group,T", [(100, 1, 2, 1), (70, 2, 5, 8), (130, 1, 1, 3), (300, 1, 1, 1), (66, 1, 70, 1)])
def test_many_sequences(B, Hkv, group, T):
    # more sequences than a wavefront has lanes, their keys dealt out to the workgroups
    check(make(B, T, T, Hkv, group, 64, [(37 * b * b) % 700 for b in range(B)], 700))


@pytest.mark.parametrize("B,Hkv,group,T,lens", [(8, 8, 8, 16, [250, 3, 0, 249, 251, 17, 250, 192]), (6, 2, 7, 12, [0, 1, 63, 64, 65, 400]), (3, 4, 4, 64, [300, 90, 0]),
                                                 (2, 8, 4, 8, [600, 20]), (2, 16, 1, 30, [607, 609]), (1, 16, 1, 5, [575]), (1, 16, 1, 5, [577])])
def test_caches_around_what_is_worth_cutting(B, Hkv, group, T, lens):
    check(make(B, T, T, Hkv, group, 64, lens, 640))


@pytest.mark.parametrize("capacity", [380, 384, 385, 900])
@pytest.mark.parametrize("d", [64, 80, 128, 192, 256])
@pytest.mark.parametrize("Hkv,group,T", [(1, 2, 10), (2, 8, 4), (1, 3, 5), (1, 8, 1), (1, 9, 1)])
def test_capacities_around_the_choice_of_kernel(Hkv, group, T, d, capacity):
    check(make(2, T, T, Hkv, group, d, [capacity, capacity - 70], capacity))
    check(make(1, T, T, Hkv, group, d, [capacity - 1], capacity))


@pytest.mark.parametrize("Hkv,d,capacity,lens", [(32, 64, 4200, [4097]), (32, 64, 4200, [1]), (32, 72, 6600, [6533]), (32, 128, 9100, [9001]), (16, 64, 4200, [4200, 63]),
                                                 (32, 64, 2000, [1999]), (8, 128, 4000, [3907]), (4, 256, 8000, [7001]), (4, 192, 4000, [4000]), (2, 80, 1000, [999, 0])])
def test_blocks_of_all_sizes(Hkv, d, capacity, lens):
    # 256 rows of each key head: in blocks of 64, 128 or 256
    check(make(len(lens), 64, 64, Hkv, 4, d, lens, capacity))


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("Hkv,d,capacity", [(32, 64, 4200), (32, 64, 2000), (32, 128, 9100), (4, 256, 8000), (1, 64, 100)])
def test_a_value_that_is_no_number_in_blocks_of_all_sizes(Hkv, d, capacity, value):
    host = make(1, 64, 64, Hkv, 4, d, [97], capacity)
    host["parents"][:] = -1  # every node sees the cache and itself
    host["V"][0, 7] = 0
    want, tolerance = expected(host)
    host["V"][0, 7, :, 3] = value
    got = launch(host).double()
    others = [t for t in range(64) if t != 7]
    assert bool(((got - want).abs() <= tolerance)[:, others].all())
    assert not bool(torch.isfinite(got[0, 7, :, 3]).any()) and bool(torch.isfinite(got[0, 7, :, :3]).all()) and bool(torch.isfinite(got[0, 7, :, 4:]).all())


@pytest.mark.parametrize("Hkv,d,capacity", [(32, 64, 4200), (16, 128, 3000), (2, 256, 6000), (1, 80, 500)])
def test_blocks_that_are_not_full(Hkv, d, capacity):
    check(make(1, 43, 43, Hkv, 5, d, [capacity - 3], capacity))
    check(make(1, 64, 21, Hkv, 5, d, [capacity - 3], capacity))


def test_one_long_sequence_among_short_ones():
    for group, T in ((2, 1), (8, 7)):
        check(make(6, T, T, 1, group, 64, [3, 9001, 0, 40, 1, 700], 9001))


def test_lengths_are_clipped_to_the_cache():
    host = make(4, 3, 3, 2, 2, 64, [-5, 1 << 30, 70, 71], 70)
    check(host)


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_data_off_every_boundary(offset):
    check(make(2, 5, 5, 2, 2, 64, [50, 9], 60), offset=offset)


def test_a_long_cache_splits_over_workgroups():
    for B, Hkv, group, T, n in ((1, 1, 1, 1, 20001), (1, 2, 4, 16, 9000), (2, 1, 8, 64, 5003), (3, 2, 1, 1, 7777)):
        check(make(B, T, T, Hkv, group, 64, [n - 1001 * b for b in range(B)], n + 5))


@pytest.mark.parametrize("spread", [30.0, 200.0])
def test_sharp_rows(spread):
    # one key takes nearly everything, and the running maximum moves far
    check(make(2, 9, 9, 2, 2, 64, [700, 300], 700, spread=spread))


def test_scales():
    host = make(1, 4, 4, 2, 2, 64, [90], 100)
    for scale in (0.0, -0.3, 1.0, 0.01):
        check(host, scale)


def test_rising_and_falling_scores():
    host = make(1, 2, 2, 1, 1, 64, [1500], 1500)
    ramp = torch.linspace(-20, 20, 1500)
    for order in (ramp, ramp.flip(0)):
        host["Q"].zero_(), host["Kc"].zero_(), host["K"].zero_()
        host["Q"][..., 0], host["Kc"][0, 0, :, 0] = 8.0, order.half()
        check(host)


def test_nothing_behind_the_length_is_used():
    host = make(3, 5, 5, 2, 2, 80, [0, 33, 64], 96)
    want = launch(host)
    for value in (float("nan"), float("inf"), -65504.0):
        for b, n in enumerate((0, 33, 64)):
            host["Kc"][b, :, n:], host["Vc"][b, :, n:] = value, value
        assert torch.equal(launch(host).view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf"), 65504.0])
def test_nodes_that_a_row_does_not_see_do_not_reach_it(d, value):
    # four lines of nodes, i - 4 above i; three of the nodes hold no numbers, and what does not descend from them is as if they held zeros
    host = make(1, 50, 50, 2, 3, d, [70], 70)
    host["parents"][0] = torch.tensor([-1, 0, 0, 0] + list(range(46)))
    bad = (13, 33, 47)
    for node in bad:
        host["K"][0, node], host["V"][0, node] = 0, 0
    want, tolerance = expected(host)
    for node in bad:
        host["V"][0, node] = value
        host["K"][0, node] = value
    got = launch(host).double()
    parents = host["parents"][0].tolist()
    clean = [t for t in range(50) if not set(seen_by(parents, t)) & set(bad)]
    assert len(clean) == 39
    assert bool(((got - want).abs() <= tolerance)[0, clean].all())
    if value != 65504.0:
        dirty = [t for t in range(50) if t not in clean]
        assert not bool(torch.isfinite(got[0, dirty]).all(-1).any())


def test_a_value_that_is_infinite_reaches_the_rows_that_see_it():
    host = make(1, 6, 6, 1, 2, 64, [40], 40, "chain")
    host["V"][0, 3, 0, 5] = float("inf")
    got = launch(host)
    assert bool(torch.isfinite(got[0, :3]).all()) and bool((got[0, 3:, :, 5] == float("inf")).all())
    assert bool(torch.isfinite(got[0, 3:, :, :5]).all()) and bool(torch.isfinite(got[0, 3:, :, 6:]).all())


def test_one_row_equals_the_same_row_of_a_tree():
    # a chain decoded row by row against a growing cache, and in one pass beside it
    host = make(1, 12, 12, 2, 4, 128, [200], 212, "chain")
    together = launch(host).double()
    _, tolerance = expected(host)
    for t in range(12):
        one = dict(host, Q=host["Q"][:, t:t + 1].clone(), K=host["K"][:, t:t + 1].clone(), V=host["V"][:, t:t + 1].clone(),
                   parents=torch.tensor([[-1]], dtype=torch.int32), lens=torch.tensor([200 + t], dtype=torch.int32))
        assert bool(((launch(one).double() - together[:, t:t + 1]).abs() <= 2 * tolerance[:, t:t + 1]).all())
        host["Kc"][:, :, 200 + t], host["Vc"][:, :, 200 + t] = host["K"][:, t], host["V"][:, t]


def test_the_same_call_gives_the_same_bits():
    host = make(2, 16, 16, 2, 4, 128, [5000, 3001], 5000)
    first = launch(host)
    for _ in range(5):
        assert torch.equal(launch(host).view(torch.int16), first.view(torch.int16))


def test_offsets_past_32_bits():
    # two caches of 5 GiB: the second sequence's rows lie past 2^31 elements
    B, Hkv, capacity, d = 2, 8, 1310720, 128
    Kc = torch.empty(B, Hkv, capacity, d, device="cuda", dtype=torch.float16)
    Vc = torch.empty(B, Hkv, capacity, d, device="cuda", dtype=torch.float16)
    host = make(B, 4, 4, Hkv, 1, d, [90, 77], 100)
    assert Kc[:, :, :100].numel() * Kc.element_size() and Kc[1, 7].data_ptr() - Kc.data_ptr() > 2 ** 32
    Kc[:, :, :100], Vc[:, :, :100] = host["Kc"].cuda(), host["Vc"].cuda()
    out = torch.empty_like(host["Q"], device="cuda")
    ops.attn_tree(host["Q"].cuda(), host["K"].cuda(), host["V"].cuda(), Kc, Vc, host["lens"].cuda(), host["parents"].cuda(), out)
    want, tolerance = expected(host)
    assert bool(((out.cpu().double() - want).abs() <= tolerance).all())


def test_what_lies_in_the_cache_and_is_seen_spreads():
    host = make(1, 4, 4, 2, 2, 80, [100], 100, "chain")
    host["Vc"][0, 0, 50, 3], host["Kc"][0, 1, 20, 0] = float("inf"), float("nan")
    got = launch(host)
    assert bool((got[0, :, :2, 3] == float("inf")).all()) and bool(torch.isfinite(got[0, :, :2, :3]).all()) and bool(torch.isfinite(got[0, :, :2, 4:]).all())
    assert bool(torch.isnan(got[0, :, 2:]).all())


def test_refusals():
    h = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.float16)
    i = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)
    good = [h(2, 3, 4, 64), h(2, 3, 2, 64), h(2, 3, 2, 64), h(2, 2, 9, 64), h(2, 2, 9, 64), i(2), i(2, 3), h(2, 3, 4, 64)]
    ops.attn_tree(*good)
    for at, bad, why in ((0, h(2, 3, 4, 32), "shape mismatch"), (0, h(3, 4, 64), "expects Q"), (1, h(1, 3, 2, 64), "shape mismatch"),
                         (2, h(2, 4, 2, 64), "shape mismatch"), (3, h(2, 2, 8, 64), "shape mismatch"), (4, h(2, 1, 9, 64), "shape mismatch"),
                         (5, i(3), "shape mismatch"), (5, i(2).long(), "int32"), (6, i(2, 4), "shape mismatch"), (7, h(2, 3, 4, 64).float(), "expects fp16"),
                         (3, h(2, 9, 2, 64).transpose(1, 2), "compact")):
        with pytest.raises(ValueError, match=why):
            ops.attn_tree(*good[:at], bad, *good[at + 1:])
    with pytest.raises(RuntimeError, match="share 2 key heads"):
        ops.attn_tree(h(2, 3, 3, 64), *good[1:7], h(2, 3, 3, 64))
    with pytest.raises(RuntimeError, match="4 query rows"):
        ops.attn_tree(h(2, 4, 4, 64), *good[1:7], h(2, 4, 4, 64))
    assert ops.attn_tree(h(2, 0, 4, 64), *good[1:7], h(2, 0, 4, 64)) is None
