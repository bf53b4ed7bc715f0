"""Attention over pages: keys and values that are no numbers, weights and scales at the ends of their range, pools behind 32 bits, in every kernel."""
import math

import pytest
import torch

from dtas_amd import ops
from test_parity_paged import expected, ints, launch, make, seen

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
# (sequences, key heads, query heads to each, d, page, beams, elements off an aligned address): eight wavefronts to a sequence, four where there are many, 32 rows, heads
# of more than 128, and many of those; groups too short to be read together; element by element (an odd address, a page of 10); groups read together where they are long, by eight wavefronts and by four
FORMS = [(2, 2, 1, 64, 16, 1, 0), (1, 3, 9, 80, 48, 1, 0), (1, 1, 4, 128, 32, 1, 0), (256, 2, 1, 64, 16, 1, 0), (2, 1, 17, 96, 16, 1, 0), (2, 2, 2, 256, 16, 1, 0), (1, 1, 20, 192, 32, 1, 0),
         (4, 2, 2, 64, 16, 2, 0), (4, 1, 4, 128, 32, 4, 0), (512, 2, 1, 64, 16, 2, 0), (8, 2, 4, 80, 16, 8, 0), (10, 1, 9, 128, 16, 5, 0), (4, 2, 2, 256, 16, 4, 0),
         (128, 4, 1, 256, 16, 1, 0), (2, 2, 2, 64, 16, 1, 1), (4, 1, 3, 40, 10, 2, 0),
         (8, 32, 1, 128, 16, 8, 0), (4, 32, 4, 96, 32, 4, 0), (16, 64, 1, 64, 16, 2, 0)]  # (long: groups read together)
LENGTHS = (1, 16, 31, 32, 33, 47, 97, 2049)


def few(form, length):
    """Many sequences stay short, many heads long."""
    return length == 2049 if form[1] >= 32 else form[0] < 100 or length <= 97


CASES = [(*f, n) for f in FORMS for n in LENGTHS if few(f, n)]


def alone(host, b):
    """Sequence b's inputs."""
    return {**host, "Q": host["Q"][b:b + 1], "table": host["table"][b:b + 1], "lens": host["lens"][b:b + 1]}


def place(host, b, j):
    page = host["K"].shape[2]
    return int(host["table"][b, j // page]), j % page


def made(B, Hkv, group, d, page, beams, length, shared=0):
    return make(B, Hkv, group, d, page, [length] * B, beams=beams, shared=shared)


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("B,Hkv,group,d,page,beams,offset,length", CASES)
def test_the_last_value_is_no_number(B, Hkv, group, d, page, beams, offset, length, value):
    # it reaches the channel it stands in, of the rows of its sequence and key head, wherever the last page ends
    host = made(B, Hkv, group, d, page, beams, length)
    p, row = place(host, B - 1, length - 1)
    host["V"][p, 0, row, 3] = 0
    want, tolerance = expected(alone(host, B - 1))
    host["V"][p, 0, row, 3] = value
    got = launch(host, offset=offset, beams=beams).double()
    assert bool(torch.isfinite(got[:B - 1]).all()) and bool(torch.isfinite(got[:, group:]).all())
    mine = got[B - 1, :group]
    assert bool((torch.isnan(mine[:, 3]) if math.isnan(value) else mine[:, 3] == value).all())
    others = [c for c in range(d) if c != 3]
    assert bool(((got[B - 1] - want[0]).abs() <= tolerance[0])[:group, others].all()) and bool(((got[B - 1] - want[0]).abs() <= tolerance[0])[group:].all())


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("B,Hkv,group,d,page,beams,offset,length", [c for c in CASES if c[-1] in (33, 97, 2049)])
def test_a_query_that_is_no_number_is_its_rows_own(B, Hkv, group, d, page, beams, offset, length, value):
    host = made(B, Hkv, group, d, page, beams, length)
    want, tolerance = expected(host)
    host["Q"][B - 1, group - 1, 2] = value
    got = launch(host, offset=offset, beams=beams).double()
    assert bool(torch.isnan(got[B - 1, group - 1]).all())
    # (the others' bits may change: the rows of a problem move their running maxima together, which rounds their weights at other places; the bound of the error is the same)
    got[B - 1, group - 1] = want[B - 1, group - 1]
    assert bool(((got - want).abs() <= tolerance).all())


@pytest.mark.parametrize("beams", [1, 3])
@pytest.mark.parametrize("offset", [0, 1])
def test_no_columns_no_pages_no_keys(beams, offset):
    host = make(3, 2, 2, 64, 16, [5, 0, 20], beams=beams)
    for change in (dict(table=host["table"][:, :0]), dict(K=host["K"][:0], V=host["V"][:0]), dict(lens=ints([0, 0, -3]))):
        assert bool((launch({**host, **change}, offset=offset, beams=beams) == 0).all())


@pytest.mark.parametrize("at", [0, 5, 40, -1])
@pytest.mark.parametrize("B,Hkv,group,d,page,beams,offset,length", [c for c in CASES if c[-1] in (47, 97, 2049)])
def test_a_key_that_is_no_number_wherever_it_stands(B, Hkv, group, d, page, beams, offset, length, at):
    # also where everything in front of it has the score -inf: the rows that see it have no answer, others theirs
    host = made(B, Hkv, group, d, page, beams, length)
    at %= length
    host["Q"][..., 0] = 1
    for j in range(at):
        p, row = place(host, 0, j)
        host["K"][p, 0, row, 0] = -INF
    p, row = place(host, 0, at)
    host["K"][p, 0, row, 0] = NAN
    got = launch(host, offset=offset, beams=beams)
    assert bool(torch.isnan(got[0, :group]).all()) and bool(torch.isfinite(got[0, group:]).all()) and bool(torch.isfinite(got[1:]).all())


@pytest.mark.parametrize("B,Hkv,group,d,page,beams,offset,length", [c for c in CASES if c[-1] in (1, 33, 97, 2049)])
def test_scores_that_are_all_minus_infinity(B, Hkv, group, d, page, beams, offset, length):
    # nothing to divide by is no number; but for one key, the answer is its value; a row that sees nothing is zeros
    host = made(B, Hkv, group, d, page, beams, length)
    host["Q"][..., 0] = 1
    host["K"][:, 0, :, 0] = torch.where(torch.isnan(host["K"][:, 0, :, 0]), NAN, -INF).half()
    got = launch(host, offset=offset, beams=beams)
    assert bool(torch.isnan(got[:, :group]).all()) and bool(torch.isfinite(got[:, group:]).all())
    p, row = place(host, B - 1, length // 2)
    host["K"][p, 0, row, 0] = 1
    got = launch(host, offset=offset, beams=beams)
    assert bool(torch.isnan(got[:B - 1, :group]).all()) and torch.equal(got[B - 1, :group], host["V"][p, 0, row].expand(group, d))
    host["lens"][0] = 0
    got = launch(host, offset=offset, beams=beams)
    assert bool((got[0] == 0).all())


@pytest.mark.parametrize("gap", [20.0, 26.0, 40.0])
@pytest.mark.parametrize("B,Hkv,group,d,page,beams,offset,length", [c for c in CASES if c[-1] in (33, 97, 2049)])
def test_an_infinite_value_of_a_small_weight(B, Hkv, group, d, page, beams, offset, length, gap):
    # its weight is exp(-gap) of the largest, a number in 32 bits: the channel is infinite, the others are what they were
    host = made(B, Hkv, group, d, page, beams, length)
    host["Q"][:] = 0
    host["Q"][..., 0] = 1
    host["K"][:] = torch.where(torch.isnan(host["K"]), NAN, 0.0).half()
    top = place(host, B - 1, length // 2)
    host["K"][top[0], :, top[1], 0] = gap
    p, row = place(host, B - 1, length - 1)
    host["V"][p, :, row, 3] = 0
    want, tolerance = expected(alone(host, B - 1), 1.0)
    for value in (INF, -INF, NAN):
        host["V"][p, :, row, 3] = value
        got = launch(host, 1.0, offset, beams).double()
        assert bool(torch.isfinite(got[:B - 1]).all())
        mine = got[B - 1]
        assert bool((torch.isnan(mine[:, 3]) if math.isnan(value) else mine[:, 3] == value).all())
        others = [c for c in range(d) if c != 3]
        assert bool(((mine - want[0]).abs() <= tolerance[0])[:, others].all())


@pytest.mark.parametrize("value", [INF, NAN, 65504.0])
@pytest.mark.parametrize("B,Hkv,group,d,beams,lens", [(4, 2, 2, 64, 2, [70, 70, 200, 181]), (4, 32, 2, 128, 4, [1700, 1710, 1721, 1701]), (8, 1, 4, 128, 8, [700 + i for i in range(8)]), (3, 3, 1, 80, 3, [97, 1500, 1501]), (5, 2, 9, 128, 5, [40, 41, 47, 39, 33])])
def test_what_a_beam_does_not_see_does_not_reach_it(B, Hkv, group, d, beams, lens, value):
    # the beams share their first two pages and grow apart behind them; what is wrong with one's own page, or lies behind its length, is not the others'
    host = make(B, Hkv, group, d, 16, lens, beams=beams, shared=2)
    first = launch(host, beams=beams)
    p, row = place(host, B - 1, lens[B - 1] - 1)
    if row < 15:
        host["V"][p, :, row + 1:], host["K"][p, :, row + 1:] = value, value
    host["V"][p, :, row], host["K"][p, :, row] = 0, 0
    want, tolerance = expected(host)
    host["V"][p, 0, row, 5] = value
    got = launch(host, beams=beams).double()
    others = [b for b in range(B) if b != B - 1]
    assert bool(((got - want).abs() <= tolerance)[others].all()) and bool((first[others].double() - want[others]).abs().le(2 * tolerance[others]).all())
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[others] = rest[B - 1, :group, 5] = False
    assert bool(((got - want).abs() <= tolerance)[rest].all())
    if value == value and value < INF:
        host["K"][p, :, row] = 0
        full, slack = expected(host)
        assert bool(((got - full).abs() <= slack).all())
    else:
        assert not bool(torch.isfinite(got[B - 1, :group, 5]).any())
    # a page that some share, with a value that is no number: of those that see it the channel is
    at = place(host, 0, 3)
    host["V"][at[0], 0, at[1], 2] = NAN
    got = launch(host, beams=beams)
    mine = [b for b in range(B) if place(host, b, 3) == at and lens[b] > 3]
    for b in range(B):
        assert bool(torch.isnan(got[b, :group, 2]).all()) == (b in mine) and bool(torch.isfinite(got[b, :group, 6]).all())


@pytest.mark.parametrize("gap", [9.0, 13.875, 15.0, 16.5])
@pytest.mark.parametrize("B,Hkv,group,d,page,beams", [(1, 2, 1, 64, 16, 1), (10, 32, 4, 128, 16, 1), (4, 2, 2, 80, 32, 4), (8, 2, 4, 64, 64, 8), (2, 1, 17, 96, 16, 1), (2, 2, 2, 256, 16, 1), (64, 32, 1, 64, 16, 2), (8, 32, 2, 128, 16, 8)])
def test_a_long_flat_tail_behind_few_large_weights(B, Hkv, group, d, page, beams, gap):
    """Eight keys of no value whose scores lead those of all others by `gap`: what is left are the others' values, weighted by exp(-gap) each.

    The others' weights are one number, off by half a step of fp16 (2^-11) and a rounding of its exponent (gap log2(e) 2^-23, exp2 of which is within 2^-22 besides),
    and the products with values that are powers of two and their sums are exact (11 bits, less than 2^13 of them).  The sum of the weights has n additions in
    fp32 at most, 2^-24 each, and as many again over wavefronts and parts.  Storing: 2^-11 of values above 2^-14."""
    n = 3999
    columns = -(-n // page)
    Q = torch.zeros(B, Hkv * group, d, device="cuda", dtype=torch.float16)
    K, V = (torch.zeros(columns, Hkv, page, d, device="cuda", dtype=torch.float16) for _ in range(2))
    Q[..., 0] = 1
    power = torch.exp2(torch.arange(d, device="cuda") % 3 + 6).half()
    V[:] = power
    for j in range(0, 256, 32):
        K[j // page, :, j % page, 0] = gap
        V[j // page, :, j % page] = 0
    table = torch.arange(columns, device="cuda", dtype=torch.int32).expand(B, columns).contiguous()
    out = torch.empty_like(Q)
    ops.attn_paged(Q, K, V, table, torch.full((B,), n, device="cuda", dtype=torch.int32), out, 1.0, beams)
    tail = (n - 8) * math.exp(-gap)
    want = tail / (tail + 8) * power.double()
    assert float(want.min()) > 2.0 ** -14
    tolerance = 2.0 ** -11 + gap * 1.45 * 2.0 ** -23 + 2.0 ** -22 + 2 * n * 2.0 ** -24 + 2.0 ** -11
    assert float(((out.double() - want).abs() / want).max()) <= tolerance


@pytest.mark.parametrize("B,Hkv,group,d,page,beams,offset,length", [c for c in CASES if c[-1] in (97, 2049)])
def test_scores_far_from_nought(B, Hkv, group, d, page, beams, offset, length):
    """Scores 4096 + i / 8, i < 64, exact in fp32 (q = 64, k = 64 and i / 8): differences of up to 8 stay what they are.

    A weight is off by 2^-11 in fp16 and by its exponent's rounding, 12 2^-23 of it (differences up to 8, times log2 e), exp2's 2^-22, sums as in `expected`; 2^-25 of the largest at least."""
    host = made(B, Hkv, group, d, page, beams, length)
    host["Q"][:] = 0
    host["Q"][..., 0], host["Q"][..., 1] = 64, 1
    host["K"][:] = torch.where(torch.isnan(host["K"]), NAN, 0.0).half()
    host["K"][..., 0] = torch.where(torch.isnan(host["K"][..., 0]), NAN, 64.0).half()
    rows = torch.arange(host["K"].shape[0] * page).view(-1, 1, page)
    host["K"][..., 1] = torch.where(torch.isnan(host["K"][..., 1]), NAN, (rows * 37 % 64 / 8.0).float()).half()
    got = launch(host, 1.0, offset, beams).double()
    for b in {0, B - 1}:
        at, row = (torch.tensor(x) for x in zip(*seen(host, b)))
        p = torch.softmax(host["K"][at, 0, row, 1].double(), 0)
        for hk in range(Hkv):
            v = host["V"][at, hk, row].double()
            o = p @ v
            weight = (2.0 ** -11 + 12 * 2.0 ** -23 + 2.0 ** -22 + length * 2.0 ** -23) * (p @ v.abs() + o.abs()) + 2.0 ** -25 * length * p.max() * v.abs().amax(0) * 2
            off = (got[b, hk * group:(hk + 1) * group] - o).abs() - (weight + 2.0 ** -11 * (o.abs() + weight) + 2.0 ** -25)
            assert bool((off <= 0).all()), off.max()


@pytest.mark.parametrize("spread", [30.0, 200.0])
@pytest.mark.parametrize("beams", [1, 4])
def test_sharp_rows(spread, beams):
    # one key takes nearly everything, and the running maximum moves far
    host = make(4, 2, 2, 64, 16, [700, 300, 700, 3000], beams=beams, spread=spread)
    got, (want, tolerance) = launch(host, beams=beams).double(), expected(host)
    assert bool(((got - want).abs() <= tolerance).all())


def test_nothing_behind_the_lengths_is_used():
    for beams, lens, Hkv in ((1, [0, 33, 64, 2000], 2), (4, [50, 33, 64, 49], 2), (2, [700, 689, 1, 15], 2), (4, [1700, 1689, 1600, 15], 32)):
        host = make(4, Hkv, 3, 80, 32, lens, beams=beams)
        want = launch(host, beams=beams)
        for value in (NAN, INF, -65504.0):
            for b, n in enumerate(lens):
                for j in range(n, host["table"].shape[1] * 32):
                    p, row = place(host, b, j)
                    host["K"][p, :, row], host["V"][p, :, row] = value, value
            assert torch.equal(launch(host, beams=beams).view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("lens", [[(61 * b * b) % 1000 for b in range(100)] + [9001], [3, 9001] + [40] * 70, [5000] + [0] * 66, [1800 + b for b in range(130)]])
def test_many_sequences_some_of_them_cut(lens):
    # more sequences than a wavefront has lanes, their blocks dealt out in equal shares where one is long
    host = make(len(lens), 2, 2, 64, 16, lens)
    got, (want, tolerance) = launch(host).double(), expected(host)
    assert bool(((got - want).abs() <= tolerance).all())
    lens = [n for n in lens for _ in range(2)]
    host = make(len(lens), 1, 2, 64, 16, lens, beams=2, shared=1)
    got, (want, tolerance) = launch(host, beams=2).double(), expected(host)
    assert bool(((got - want).abs() <= tolerance).all())


@pytest.mark.parametrize("beams", [1, 2])
def test_more_sequences_than_are_cut(beams):
    # thousands of them, one of them long; all tables name pages of a small pool
    B, page = 4100, 16
    host = make(2, 2, 2, 64, page, [3000, 3000])
    g = torch.Generator().manual_seed(beams)
    host["Q"] = torch.randn(B, 4, 64, generator=g).half()
    host["table"] = host["table"][:1].expand(B, -1).contiguous()
    host["lens"] = ints([5 + b % 30 for b in range(B - 2)] + [3000, 0])
    got, (want, tolerance) = launch(host, beams=beams).double(), expected(host)
    assert bool(((got - want).abs() <= tolerance).all())


@pytest.mark.parametrize("group,d", [(17, 64), (33, 128), (40, 80), (70, 64), (20, 256)])
def test_many_rows_of_a_key_head_cut(group, d):
    host = make(2, 1, group, d, 32, [3001, 65])
    got, (want, tolerance) = launch(host).double(), expected(host)
    assert bool(((got - want).abs() <= tolerance).all())


@pytest.mark.parametrize("scale", [1e-38, 2e38, -2e38])
@pytest.mark.parametrize("page", [16, 10])
def test_scales_at_the_ends_of_their_range(scale, page):
    # with scores that a large one leaves apart by far: the largest takes all, or with none of it all are the same
    host = make(2, 1, 2, 64, page, [100, 1000])
    host["Q"][:] = 0
    host["Q"][..., 0] = 1
    host["K"][:] = torch.where(torch.isnan(host["K"]), NAN, 0.0).half()
    for b in range(2):
        p, row = place(host, b, 57)
        host["K"][p, 0, row, 0] = math.copysign(0.5, scale)
    got = launch(host, scale).double()
    for b in range(2):
        at, row = (torch.tensor(x) for x in zip(*seen(host, b)))
        v = host["V"][at, 0, row].double()
        if abs(scale) > 1:
            assert torch.equal(got[b], v[57].expand(2, 64))
        else:
            want, tolerance = expected(alone(host, b), 0.0)
            assert bool(((got[b] - want[0]).abs() <= tolerance[0]).all())


def test_pools_behind_32_bits():
    # 9 GB of keys: pages whose first byte lies behind 2^32, and elements behind 2^32, in one layer and over layers; the same bits as from a small pool
    pages, Hkv, page, d = 140000, 8, 32, 128
    lens, W = [130, 133, 160, 97], 2
    small = make(4, Hkv, 2, d, page, lens, beams=W, shared=1)
    used = small["K"].shape[0]
    names = torch.randperm(200, generator=torch.Generator().manual_seed(1))[:used] + pages - 200
    K, V = (torch.empty(pages, Hkv, page, d, dtype=torch.float16, device="cuda") for _ in range(2))
    assert K[pages - 200:].storage_offset() > 2 ** 32
    K[names.cuda()], V[names.cuda()] = small["K"].cuda(), small["V"].cuda()
    Q, table, far, d_lens = small["Q"].cuda(), small["table"].cuda(), names.int()[small["table"].long()].cuda(), ints(lens).cuda()
    for beams in (1, W):
        outs = [torch.empty_like(Q) for _ in range(2)]
        ops.attn_paged(Q, small["K"].cuda(), small["V"].cuda(), table, d_lens, outs[0], None, beams)
        ops.attn_paged(Q, K, V, far, d_lens, outs[1], None, beams)
        assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))
    # rows into such pages, in the last of five layers, and copies of them
    layered = [t.view(5, pages // 5, Hkv, page, d) for t in (K, V)]
    rows = torch.randn(5, 3, Hkv, d, device="cuda").half()
    last = pages // 5 - 1
    ops.page_append(rows, -rows, ints([last * page + 3, 5, last * page + 31]).cuda(), *layered)
    for t, r in zip(layered, (rows, -rows)):
        assert torch.equal(t[:, last, :, 3], r[:, 0]) and torch.equal(t[:, 0, :, 5], r[:, 1]) and torch.equal(t[:, last, :, 31], r[:, 2])
    state = [ints(x).cuda() for x in ([[0, 0]], [[[last], [1]]], [[31, 31]], [last - 1] + [0] * last, [1])]
    outputs = [torch.empty_like(state[1]), torch.empty_like(state[2]), torch.empty_like(state[4])]
    ops.page_reorder(*state, *outputs, *layered)
    # (page 1, which nobody names any more, lies on top of the stack then)
    assert outputs[0].tolist() == [[[last], [1]]] and outputs[1].tolist() == [[31, 31]] and outputs[2].tolist() == [1]
    for t in layered:
        assert torch.equal(t[:, 1, :, :31].view(torch.int16), t[:, last, :, :31].view(torch.int16))
