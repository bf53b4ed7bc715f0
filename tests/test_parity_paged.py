"""Pages, slots, tables of beams and the choice of beams against plain loops; attention over pages against the definition in 64 bits."""
import math

import pytest
import torch

from dtas_amd import ops
from gpu_util import Guarded

pytestmark = pytest.mark.gpu

up = lambda n, page: -(-n // page)
ints = lambda v: torch.tensor(v, dtype=torch.int32)


def guarded(t):
    g = Guarded(tuple(t.shape), t.dtype)
    if t.dtype == torch.int32:
        g.fill = 1234  # (a whole number)
    g.t.copy_(t)
    return g


# ---- pages and slots

def assigned(lens, count, table, free, height, page, rows, packed):
    """What page_assign is to leave: table, slots, new_lens, left, starts."""
    pages, columns = len(free), len(table[0]) if table else 0
    there = min(max(height, 0), pages)
    table, new_lens, starts = [list(r) for r in table], list(lens), [0]
    slots = [-1] * (rows if packed else rows * len(lens))
    asked = wanted = taken = 0
    for b, n in enumerate(lens):
        c = count[b]
        begin = asked if packed else b * rows
        asked += max(c, 0)
        starts.append(min(asked, 2 ** 31 - 1))
        if n < 0 or c < 0 or n + c > min(columns * page, 2 ** 31 - 1) or (asked if packed else c) > rows:
            continue
        have, to = up(n, page), up(n + c, page)
        wanted += to - have
        if to > have and wanted > there:
            continue
        for i in range(have, to):
            table[b][i] = free[there - 1 - taken]
            taken += 1
        for t in range(c):
            p = table[b][(n + t) // page]
            if 0 <= p < pages:
                slots[begin + t] = p * page + (n + t) % page
        new_lens[b] = n + c
    return table, slots, new_lens, there - taken, starts


def check_assign(lens, count, table, free, height, page, rows, packed, in_place=False):
    B, columns = len(lens), len(table[0]) if table else 0
    want = assigned(lens, count, table, free, height, page, rows, packed)
    d_lens, d_count, d_free, d_height = (guarded(ints(v)) for v in (lens, count, free, [height]))
    d_table = guarded(ints(table).view(B, columns))
    d_slots = guarded(torch.full((rows,) if packed else (B, rows), 99, dtype=torch.int32))
    d_starts = guarded(torch.full((B + 1,), 99, dtype=torch.int32)) if packed else None
    d_new, d_left = (d_lens, d_height) if in_place else (guarded(torch.full((B,), 99, dtype=torch.int32)), guarded(ints([99])))
    ops.page_assign(d_lens.t, d_count.t, d_table.t, d_free.t, d_height.t, page, d_slots.t, d_new.t, d_left.t, starts=d_starts.t if packed else None)
    assert d_table.check().tolist() == want[0] and d_new.check().tolist() == want[2] and d_left.check().tolist() == [want[3]]
    assert d_slots.check().reshape(-1).tolist() == want[1]
    assert not packed or d_starts.check().tolist() == want[4]
    assert d_free.check().tolist() == free and d_count.check().tolist() == count


def pool_of(lens, page, columns, extra, g):
    """A table of distinct pages for such lengths, and the stack of the others, `extra` of them."""
    held = [min(up(max(n, 0), page), columns) for n in lens]
    pages = sum(held) + extra
    order = torch.randperm(pages, generator=g).tolist()
    table, at = [], 0
    for n in held:
        table.append(order[at:at + n] + [-7] * (columns - n))
        at += n
    return table, order[at:] + [order[0]] * at, extra


@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 257, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("page,rows,packed", [(16, 1, False), (1, 3, False), (7, 11, False), (16, 40, True), (32, 3000, True), (5, 1, True)])
def test_pages_and_slots(B, page, rows, packed):
    g = torch.Generator().manual_seed(B * 7 + page)
    lens = torch.randint(0, 50, (B,), generator=g).tolist()
    most = max(1, 2 * rows // B) if packed else rows
    count = torch.randint(0, most + 1, (B,), generator=g).tolist()
    columns = up(50 + most, page)
    for extra in (0, 3, B // 2 + 1, B * up(most, page) + B):
        table, free, height = pool_of(lens, page, columns, extra, g)
        check_assign(lens, count, table, free, height, page, rows, packed)
        check_assign(lens, count, table, free, height, page, rows, packed, in_place=True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_many_rows_by_several_workgroups(packed, in_place):
    g = torch.Generator().manual_seed(3)
    B, page = 37, 16
    lens = torch.randint(0, 900, (B,), generator=g).tolist()
    count = torch.randint(0, 1400, (B,), generator=g).tolist()
    rows = sum(count) + 70 if packed else 1399
    columns = up(2300, page)
    for extra in (up(sum(count), 2 * page), B * 90):
        table, free, height = pool_of(lens, page, columns, extra, g)
        check_assign(lens, count, table, free, height, page, rows, packed, in_place)


@pytest.mark.parametrize("packed", [False, True])
def test_sequences_that_cannot_be_served(packed):
    # negative lengths and counts, tables and slot maps without room, lengths at the type's end, pages outside the pool in table and stack
    big = 2 ** 31 - 1
    lens = [5, -1, 3, 31, 32, 0, big, 17, -big - 1, 2, 30, 0]
    count = [4, 2, -3, 2, 1, 40, 1, 9, 1, big, 2, 0]
    free = [3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14]
    table = [[20 + 4 * b, 21 + 4 * b, 22 + 4 * b, 23 + 4 * b] for b in range(len(lens))]
    pages = 80
    free = free + [0] * (pages - len(free))
    for height in (-5, 0, 1, 2, 4, 12, 80, 1000):
        check_assign(lens, count, table, free, height, 8, 30, packed)
    table[0][0] = 80
    table[7][2] = -1
    free[10] = 99
    free[11] = -4
    check_assign(lens, count, table, free, 12, 8, 30, packed)


def test_starts_stop_at_the_types_end():
    big = 2 ** 31 - 1
    lens, count = [0] * 6, [3, big, big, big, 2, 1]
    table, free = [[-1, -1]] * 6, [0, 1, 2, 3]
    check_assign(lens, count, table, free, 4, 4, 10, True)


def test_no_sequences_and_no_columns():
    check_assign([], [], [], [1, 0], 2, 4, 9, True)
    check_assign([0, 0], [1, 0], [[], []], [1, 0], 2, 4, 9, True)
    check_assign([0, 0], [0, 0], [[], []], [1, 0], 2, 4, 0, False)


# ---- rows into their slots

@pytest.mark.parametrize("layers,rows,Hkv,d,page,pages,offset", [((), 1, 1, 8, 16, 3, 0), ((), 64, 8, 128, 16, 90, 0), ((3,), 7, 2, 80, 5, 4, 0), ((2, 2), 33, 1, 20, 16, 9, 0),
                                                                 ((), 300, 32, 80, 32, 17, 0), ((2,), 19, 3, 64, 1, 40, 0), ((2,), 19, 3, 64, 16, 5, 1), ((), 5, 1, 3, 2, 7, 0)])
def test_rows_into_slots(layers, rows, Hkv, d, page, pages, offset):
    g = torch.Generator().manual_seed(rows)
    n = lambda *s: torch.randn(*s, generator=g).half()
    K, V = n(*layers, rows, Hkv, d), n(*layers, rows, Hkv, d)
    pools = [n(*layers, pages, Hkv, page, d) for _ in range(2)]
    places = torch.randperm(pages * page, generator=g).tolist()
    slots = [places[i] if i < len(places) and i % 5 != 3 else (-1, -2 ** 31, pages * page, 2 ** 31 - 1)[i % 4] for i in range(rows)]
    want = [p.clone() for p in pools]
    for i, s in enumerate(slots):
        if 0 <= s < pages * page:
            want[0][..., s // page, :, s % page, :] = K[..., i, :, :]
            want[1][..., s // page, :, s % page, :] = V[..., i, :, :]

    def there(t):
        raw = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
        raw[offset:] = t.flatten().cuda()
        return raw[offset:].view(t.shape)

    got = [guarded(p) for p in pools]
    if offset:
        got = None
        moved = [there(p) for p in pools]
        ops.page_append(there(K), there(V), ints(slots).cuda(), *moved)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(moved, want))
        return
    ops.page_append(there(K), there(V), ints(slots).cuda(), got[0].t, got[1].t)
    for a, b in zip(got, want):
        assert torch.equal(torch.from_numpy(a.check()), b)


# ---- attention

def make(B, Hkv, group, d, page, lens, seed=0, spread=1.0, beams=1, shared=0, columns=None, spare=2):
    """Sequences over distinct pages in no order; the first `shared` columns of each group of `beams` name the same.  Pages that nobody names are NaN."""
    g = torch.Generator().manual_seed(seed + 31 * d + page)
    n = lambda *s: torch.randn(*s, generator=g)
    columns = columns or max(1, max(up(max(x, 0), page) for x in lens))
    wanted = B * columns
    order = torch.randperm(wanted + spare, generator=g)
    table = order[:wanted].view(B, columns).clone()
    if beams > 1:
        table.view(B // beams, beams, columns)[:, :, :shared] = table.view(B // beams, beams, columns)[:, :1, :shared].clone()
    K, V = n(wanted + spare, Hkv, page, d).half(), n(wanted + spare, Hkv, page, d).half()
    K[order[wanted:]] = V[order[wanted:]] = float("nan")
    return {"Q": (n(B, Hkv * group, d) * spread).half(), "K": K, "V": V, "table": table.to(torch.int32), "lens": ints(lens)}


def seen(host, b):
    """The places (page, row) that sequence b sees, in their order."""
    pages, page, columns = host["K"].shape[0], host["K"].shape[2], host["table"].shape[1]
    n = min(max(int(host["lens"][b]), 0), columns * page)
    names = host["table"][b].tolist()
    return [(names[j // page], j % page) for j in range(n) if 0 <= names[j // page] < pages]


def expected(host, scale=None):
    """The value, and how far an answer may be from it.

    Scores: d products in fp32, (d + 8) 2^-24 of their magnitudes, times the scale: e.  Probabilities, in units of the largest, are rounded
    to fp16 for the product with the values: 2^-11 of each and 2^-25 at least; e on both sides of the quotient; sums of n keys joined in
    any order: n 2^-24 twice.  On the weighted sum of |v| (and of the quotient, |out|).  Storing: 2^-11, 2^-25 at least."""
    Q, K, V = (host[k].double() for k in ("Q", "K", "V"))
    B, H, d = Q.shape
    Hkv = K.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out, slack = torch.zeros_like(Q), torch.zeros_like(Q)
    for b in range(B):
        places = seen(host, b)
        if not places:
            continue
        at, row = (torch.tensor(x) for x in zip(*places))
        for hk in range(Hkv):
            k, v = K[at, hk, row], V[at, hk, row]
            mine = slice(hk * (H // Hkv), (hk + 1) * (H // Hkv))
            q = Q[b, mine]
            p = torch.softmax(q @ k.t() * scale, -1)
            e = (d + 8) * 2.0 ** -24 * abs(scale) * (q.abs() @ k.abs().t()).amax(-1, keepdim=True)
            out[b, mine] = o = p @ v
            weight = (2.0 ** -11 + 2 * e + len(k) * 2.0 ** -23 + 2.0 ** -21) * (p @ v.abs() + o.abs()) + 2.0 ** -25 * len(k) * (p.amax(-1, keepdim=True) * v.abs().amax(0) * 2)
            slack[b, mine] = weight + 2.0 ** -11 * (o.abs() + weight) + 2.0 ** -25
    return out, slack


def launch(host, scale=None, offset=0, beams=1):
    def there(t):
        raw = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
        raw[offset:] = t.flatten().cuda()
        return raw[offset:].view(t.shape)

    out = Guarded(tuple(host["Q"].shape), torch.float16)
    ops.attn_paged(there(host["Q"]), there(host["K"]), there(host["V"]), host["table"].cuda(), host["lens"].cuda(), out.t, scale, beams)
    return torch.from_numpy(out.check())


def check(host, scale=None, offset=0, beams=1):
    got = launch(host, scale, offset, beams).double()
    want, tolerance = expected(host, scale)
    off = (got - want).abs() - tolerance
    assert bool((off <= 0).all()), (off.max().item(), (off > 0).sum().item(), int(torch.isnan(got).sum()))


@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 104, 128, 160, 192, 256])
@pytest.mark.parametrize("group,page", [(1, 16), (4, 32), (3, 48), (17, 16), (8, 128)])
def test_head_dimensions(d, group, page):
    check(make(2, 2, group, d, page, [61, 130]))


@pytest.mark.parametrize("d,page,offset", [(1, 16, 0), (5, 3, 0), (20, 16, 0), (65, 8, 0), (255, 16, 0), (64, 1, 0), (64, 7, 0), (128, 24, 0), (80, 40, 0), (64, 16, 1), (128, 32, 3)])
def test_element_by_element(d, page, offset):
    check(make(3, 2, 2, d, page, [33, 0, 70]), offset=offset)
    check(make(4, 1, 3, d, page, [33, 33, 40, 38], beams=2, shared=33 // page), offset=offset, beams=2)


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1000, 2049, 5000])
@pytest.mark.parametrize("page,group,d", [(16, 1, 80), (64, 4, 128), (48, 9, 64)])
def test_lengths(length, page, group, d):
    check(make(1, 2, group, d, page, [length]))


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 256, 512])
def test_ragged_batches(page):
    check(make(9, 2, 2, 80, page, [0, 1, 500, 37, 999, 64, 256, 3, 128]))
    check(make(40, 3, 2, 64, page, [7 * b for b in range(40)]))


def test_lengths_outside_the_table():
    host = make(4, 2, 2, 64, 16, [-1, 1000, -2 ** 31, 2 ** 31 - 1], columns=5)
    assert len(seen(host, 0)) == len(seen(host, 2)) == 0 and len(seen(host, 1)) == len(seen(host, 3)) == 80
    check(host)


@pytest.mark.parametrize("page,d,group,offset", [(16, 64, 1, 0), (16, 128, 4, 0), (32, 80, 4, 0), (128, 128, 9, 0), (24, 64, 2, 0), (16, 256, 20, 0), (16, 64, 2, 1)])
def test_pages_outside_the_pool_are_not_seen(page, d, group, offset):
    host = make(7, 2, group, d, page, [5 * page, 5 * page - 3, 4 * page + 1, page, 3 * page, 8, 0])
    pages = host["K"].shape[0]
    for b, c, bad in ((0, 0, -1), (0, 3, pages), (1, 4, 2 ** 31 - 1), (2, 1, -2 ** 31), (2, 4, pages + 5), (3, 0, -1), (4, 0, -3), (4, 1, -3), (4, 2, pages), (5, 0, pages)):
        host["table"][b, c] = bad
    assert not seen(host, 3) and not seen(host, 4) and not seen(host, 5) and not seen(host, 6)
    check(host, offset=offset)
    got = launch(host, offset=offset)
    assert bool((got[3:] == 0).all())


@pytest.mark.parametrize("beams,B,shared,lens", [(2, 4, 3, [60, 60, 75, 75]), (4, 4, 0, [33, 33, 33, 33]), (4, 8, 7, [130] * 4 + [117, 130, 127, 113]), (5, 10, 2, [40] * 5 + [0, 33, 40, 34, 48]),
                                                 (8, 8, 30, [500 + 3 * i for i in range(8)]), (3, 6, 62, [1000, 1001, 1002, 992, 993, 1024]), (16, 16, 9, [150 + i for i in range(16)]),
                                                 (7, 7, 4, [-1, 70, 64, 64, 65, 80, 79]), (33, 33, 3, [50] * 33)])
@pytest.mark.parametrize("group,d,Hkv", [(1, 80, 3), (4, 128, 2), (8, 64, 1), (3, 256, 1)])
def test_beams_with_shared_pages(beams, B, shared, lens, group, d, Hkv):
    check(make(B, Hkv, group, d, 16, lens, beams=beams, shared=shared), beams=beams)


@pytest.mark.parametrize("page", [32, 48, 64, 128])
def test_beams_that_share_here_and_there(page):
    # some of the beams name the same page, at the end too; one names none; pages outside the pool among them
    host = make(6, 2, 2, 128, page, [6 * page - 5] * 6, beams=6, shared=2)
    t = host["table"]
    t[3, 2:] = t[1, 2:]
    t[4, 3] = t[0, 3]
    t[5, 4] = t[2, 4]
    t[2, 1] = -1
    t[4, 0] = t[5, 0] = host["K"].shape[0]
    host["lens"][4] = 3 * page + 1
    check(host, beams=6)
    check(host, beams=3)
    check(host, beams=1)


@pytest.mark.parametrize("beams,B,Hkv,group,d,page,shared,lens", [
    (8, 8, 32, 1, 128, 16, 120, [2060 + i for i in range(8)]), (4, 8, 16, 4, 128, 32, 0, [2100] * 4 + [1, 0, 2080, 700]), (4, 4, 16, 4, 80, 48, 40, [3000, 2999, 2990, 3001]),
    (5, 10, 32, 3, 64, 16, 60, [1700 + 9 * i for i in range(10)]), (33, 33, 16, 2, 64, 128, 15, [2000 - 3 * i for i in range(33)]), (2, 4, 32, 8, 96, 64, 20, [2500, 1400, 0, 2499]),
    (7, 7, 64, 2, 72, 80, 24, [-1, 2000, 1999, 30, 2 ** 31 - 1, 1936, 1905]), (2, 16, 64, 1, 64, 16, 97, [1700, 1600, 1555, 1556] + [50 * i for i in range(12)])])
def test_long_groups_read_together(beams, B, Hkv, group, d, page, shared, lens):
    # long enough, and enough of them, that pages are read once for all; the last with more problems than four wavefronts each need
    host = make(B, Hkv, group, d, page, lens, beams=beams, shared=shared, columns=up(max(n for n in lens if n < 2 ** 31 - 1), page))
    if page == 32:  # the same page here and there, and pages outside the pool
        t = host["table"]
        t[2, 5:9], t[3, 20:] = t[0, 5:9], t[1, 20:]
        t[1, 30], t[2, 31], t[0, 64] = -1, host["K"].shape[0], -5
    check(host, beams=beams)


def test_short_groups_in_long_tables():
    # the tables have room for much more: the lengths decide
    for lens in ([5, 40, 33, 0, 1, 64, 300, 299], [900] * 8, [2100, 5, 3, 2, 1, 0, 7, 9]):
        check(make(8, 32, 2, 64, 16, lens, beams=4, shared=1, columns=140), beams=4)


@pytest.mark.parametrize("d", [160, 192, 200, 256])
def test_many_sequences_of_large_heads(d):
    lens = [(53 * b) % 200 for b in range(64)]
    check(make(64, 8, 2, d, 16, lens))
    check(make(64, 8, 17, d, 32, lens[:62] + [1500, 700], columns=47))


def test_many_sequences():
    check(make(300, 1, 2, 64, 16, [(37 * b) % 150 for b in range(300)]))
    check(make(96, 8, 1, 64, 16, [(37 * b) % 90 for b in range(96)], beams=4, shared=1), beams=4)


@pytest.mark.parametrize("scale", [0.0, -0.25, 1.0, 1e-30, 3.0])
@pytest.mark.parametrize("page,offset", [(16, 0), (64, 0), (10, 0)])
def test_scales(scale, page, offset):
    check(make(2, 2, 4, 64, page, [70, 200], spread=0.5), scale, offset)


# ---- tables of beams

def reordered(parents, table, lens, free, height, page, pages):
    """What page_reorder is to leave: new_table entries {(g, w, c): page}, new_lens, free, left, copies (from, to, rows)."""
    free, left = list(free), min(max(height, 0), len(free))
    entries, new_lens, wanted = {}, [], []
    for g, (rows, ps) in enumerate(zip(table, parents)):
        columns = len(rows[0])
        n = [min(max(x, 0), columns * page) for x in lens[g]]
        named = [rows[w][:up(n[w], page)] for w in range(len(rows))]
        taken = [(named[p], n[p]) if 0 <= p < len(rows) else ([], 0) for p in ps]
        for c in range(columns):
            kept = {r[c] for r, _ in taken if c < len(r)}
            for r in named:
                if c < len(r) and 0 <= r[c] < pages and r[c] not in kept:
                    kept.add(r[c])
                    if left < len(free):
                        free[left] = r[c]
                    left += 1
        new_lens.append([m for _, m in taken])
        for w, (r, m) in enumerate(taken):
            for c, p in enumerate(r):
                entries[g, w, c] = p
            if m % page and 0 <= r[m // page] < pages and ps[w] in ps[:w]:
                wanted.append((g, w, m))
    copies = []
    left = min(left, len(free))
    for g, w, m in wanted:
        to = -1
        if left > 0:
            left -= 1
            to = free[left]
        if 0 <= to < pages:
            copies.append((entries[g, w, m // page], to, m % page))
            entries[g, w, m // page] = to
        else:
            del entries[g, w, m // page]
            new_lens[g][w] = -1
    return entries, new_lens, free, left, copies


def check_reorder(parents, table, lens, free, height, page, layers=(2,), Hkv=2, d=16, in_place=False, seed=0, offset=0):
    pages = len(free)
    entries, new_lens, new_free, left, copies = reordered(parents, table, lens, free, height, page, pages)
    gen = torch.Generator().manual_seed(seed)
    pools = [torch.randn(*layers, pages, Hkv, page, d, generator=gen).half() for _ in range(2)]
    want = [p.clone() for p in pools]
    for p in want:
        for a, b, rows in copies:
            p[..., b, :, :rows, :] = p[..., a, :, :rows, :].clone()
    G, W, columns = len(table), len(table[0]), len(table[0][0])
    d_parents, d_lens, d_free, d_height = (guarded(ints(v)) for v in (parents, lens, free, [height]))
    d_table = guarded(ints(table).view(G, W, columns))
    before = ints(table).view(G, W, columns) if in_place else torch.full((G, W, columns), -55, dtype=torch.int32)
    d_new = d_table if in_place else guarded(before)
    d_new_lens, d_left = (d_lens, d_height) if in_place else (guarded(torch.full((G, W), 99, dtype=torch.int32)), guarded(ints([99])))
    raw = [torch.empty(p.numel() + offset, dtype=torch.float16, device="cuda") for p in pools]
    d_pools = [r[offset:].view(p.shape) for r, p in zip(raw, pools)]
    for a, b in zip(d_pools, pools):
        a.copy_(b)
    ops.page_reorder(d_parents.t, d_table.t, d_lens.t, d_free.t, d_height.t, d_new.t, d_new_lens.t, d_left.t, *d_pools)
    want_table = before.clone()
    for (g, w, c), p in entries.items():
        want_table[g, w, c] = p
    assert torch.equal(torch.from_numpy(d_new.check()), want_table)
    assert d_new_lens.check().tolist() == new_lens and d_left.check().tolist() == [left]
    assert d_free.check().tolist() == new_free and d_parents.check().tolist() == parents
    for a, b in zip(d_pools, want):
        assert torch.equal(a.cpu(), b)


def beam_tables(G, W, columns, lens, page, shared, extra, g):
    """Tables of groups that share their first `shared` columns, other pages distinct; the stack of `extra` others."""
    table, at = [], 0
    order = torch.randperm(G * (shared + W * columns) + extra, generator=g).tolist()
    for i in range(G):
        front = order[at:at + shared]
        at += shared
        rows = []
        for w in range(W):
            n = up(lens[i][w], page)
            rows.append((front + order[at:at + columns - shared])[:n] + [-9] * (columns - n))
            at += columns - shared
        table.append(rows)
    free = order[at:at + extra]
    return table, free + [0] * (len(order) - extra)


@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 8, 17, 32])
@pytest.mark.parametrize("G,columns,page", [(1, 3, 16), (3, 40, 4), (2, 300, 2), (20, 9, 16), (1, 2100, 1)])
def test_tables_of_beams(W, G, columns, page):
    g = torch.Generator().manual_seed(W * 1000 + columns)
    for kind in range(4):
        shared = (0, columns // 2, columns // 2, columns - 1)[kind]
        same = torch.randint(shared * page + 1, columns * page + 1, (G, 1), generator=g).expand(G, W)
        lens = (same if kind < 3 else torch.randint(shared * page, columns * page + 1, (G, W), generator=g)).tolist()
        parents = torch.randint(-1 if kind % 2 else 0, W, (G, W), generator=g).tolist()
        if kind == 2:
            parents = [[0] * W for _ in range(G)]
        table, free = beam_tables(G, W, columns, lens, page, shared, G * W, g)
        check_reorder(parents, table, lens, free, G * W, page, in_place=kind % 2 == 0, d=(16, 5, 8, 64)[kind], offset=kind == 3)


def test_a_pool_without_room():
    g = torch.Generator().manual_seed(1)
    G, W, columns, page = 3, 4, 5, 8
    lens = [[35] * W, [32] * W, [17] * W]
    table, free = beam_tables(G, W, columns, lens, page, 2, 6, g)
    for height in (-3, 0, 1, 2, 5, 6):
        for parents in ([[0] * W] * G, [[3, 3, 1, 1], [0, 1, 2, 3], [2, 2, 2, 2]], [[0, 1, 2, 3], [1, 1, 1, 1], [0, 0, 3, 3]]):
            check_reorder(parents, table, lens, free, height, page)
            check_reorder(parents, table, lens, free, height, page, in_place=True)
    # more given back than the stack holds is dropped, pages outside the pool on the stack are no pages
    check_reorder([[-1] * W] * G, table, lens, free, len(free) - 3, page)
    check_reorder([[0] * W] * G, table, lens, [-1] * 3 + free[3:], 3, page)
    check_reorder([[0] * W] * G, table, lens, [len(free)] * 3 + free[3:], 3, page)


def test_entries_and_lengths_outside_their_range():
    table = [[[3, -1, 5, 99], [3, 99, 6, 7]], [[-4, 8, 9, 10], [-4, 8, 11, 12]]]
    free = [0, 1, 2] + [0] * 17
    for lens in ([[1000, 28], [-5, 31]], [[30, 13], [26, 26]], [[16, 9], [2, 3]]):
        for parents in ([[0, 0], [1, 1]], [[1, 7], [-9, 0]], [[1, 0], [2, -1]], [[-1, -1], [2 ** 31 - 1, -2 ** 31]]):
            check_reorder(parents, table, lens, free, 3, 8)
            check_reorder(parents, table, lens, free, 3, 8, in_place=True)


@pytest.mark.parametrize("G,W", [(0, 4), (3, 0)])
def test_no_rows_at_all(G, W):
    i = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)
    pool, left = torch.zeros(5, 1, 16, 8, device="cuda", dtype=torch.float16), i(1)
    ops.page_reorder(i(G, W), i(G, W, 2), i(G, W), i(5), i(1) + 4, i(G, W, 2), i(G, W), left, pool, pool.clone())
    assert left.item() == 4


def test_many_requests_let_go():
    g = torch.Generator().manual_seed(4)
    G, page, columns = 1500, 4, 7
    lens = torch.randint(0, columns * page + 1, (G, 1), generator=g).tolist()
    table, free = beam_tables(G, 1, columns, lens, page, 0, 10, g)
    parents = torch.randint(-1, 1, (G, 1), generator=g).tolist()
    check_reorder(parents, table, lens, free, 10, page, layers=(), Hkv=1, d=8)
    check_reorder(parents, table, lens, free, 10, page, layers=(), Hkv=1, d=8, in_place=True)


@pytest.mark.parametrize("G,W,shared,extra,height", [(200, 8, 0, 3, 3), (200, 8, 2, 1500, 1500), (200, 8, 2, 700, 700), (3, 32, 0, 2, 2), (600, 4, 1, 40, 40), (130, 32, 1, 0, 0)])
def test_many_copies(G, W, shared, extra, height):
    # copies take what is given back in the same call, what was there before, some of both, or there are too few; more of them than a workgroup has threads
    g = torch.Generator().manual_seed(G)
    page, columns = 4, 3
    lens = torch.randint(9, 12, (G, 1), generator=g).expand(G, W).tolist()
    table, free = beam_tables(G, W, columns, lens, page, shared, extra, g)
    for parents in (torch.randint(0, 2, (G, W), generator=g).tolist(), torch.randint(0, W, (G, W), generator=g).tolist()):
        check_reorder(parents, table, lens, free, height, page, layers=(), Hkv=1, d=8)
        check_reorder(parents, table, lens, free, height, page, layers=(), Hkv=1, d=8, in_place=True)


# ---- the choice of beams

def chosen(logits, scores, done, eos):
    """The best candidates in 64 bits: tokens, parents, scores, done; and how far apart the scores of the last taken and the first left are."""
    G, W, V = logits.shape
    x = torch.where(torch.isnan(logits), torch.nan, logits.double())
    logs = x - torch.logsumexp(x, -1, keepdim=True)
    total = scores.double()[:, :, None] + logs
    bad = ~torch.isfinite(torch.logsumexp(x, -1)) | ~torch.isfinite(scores)
    total = torch.where(bad[:, :, None] | ~torch.isfinite(total), -math.inf, total)
    ended = done != 0
    only = torch.where((torch.arange(V) == eos) & torch.isfinite(scores)[:, :, None], scores.double()[:, :, None], -math.inf)
    total = torch.where(ended[:, :, None], only, total)
    # (of equal sums of one beam the greater logit goes first: the sum is that of numbers, not of their roundings)
    best, at = torch.sort(total.view(G, W * V), dim=1, descending=True, stable=True)
    return (at[:, :W] % V).int(), (at[:, :W] // V).int(), best[:, :W], ((torch.gather(done, 1, at[:, :W] // V) != 0) | (at[:, :W] % V == eos)).int()


def check_beams(logits, scores, done=None, eos=-1, in_place=False):
    want = chosen(logits, scores, torch.zeros_like(scores).int() if done is None else done, eos)
    G, W, V = logits.shape
    out = [guarded(torch.full((G, W), 7, dtype=dtype)) for dtype in (torch.int32, torch.int32, torch.float32, torch.int32)]
    d_scores, d_done = guarded(scores), None if done is None else guarded(done)
    if in_place:
        out[2] = d_scores
        out[3] = d_done
    ops.beam_select(logits.cuda(), d_scores.t, None if done is None else d_done.t, out[0].t, out[1].t, out[2].t, None if done is None else out[3].t, eos)
    got = [None if o is None else torch.from_numpy(o.check()) for o in out]
    assert torch.equal(got[1], want[1]) and torch.equal(got[0], want[0]), (got[:2], want[:2])
    if done is not None:
        assert torch.equal(got[3], want[3])
    # A term exp(-y), y its distance to the maximum, is off by 1.23 y 2^-24 (its exponent's rounding, and log2 e's) and 2^-22 (exp2); weighted by the terms the mean of y is the
    # entropy less log(sum), at most log(V) < 13; sixteen terms are added in 32 bits, two by two: 4 2^-24; what all have in common is off by 2 2^-24: (16 + 4 + 4 + 2) 2^-24 < 2^-19
    # of the sum, and of its logarithm.  Storing: 2^-24 of the value.
    same = torch.isinf(want[2])
    assert torch.equal(torch.isinf(got[2]), same)
    off = torch.where(same, 0.0, (got[2].double() - want[2]).abs() - 2.0 ** -24 * want[2].abs() - 2.0 ** -19)
    assert bool((off <= 0).all()), off.max()


def some_logits(G, W, V, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(G, W, V, generator=g) * spread, (-20 * torch.rand(G, W, generator=g)).float(), g


@pytest.mark.parametrize("W", [1, 2, 3, 4, 7, 8, 16, 31, 32])
@pytest.mark.parametrize("G,V", [(1, 1), (2, 5), (3, 33), (1, 1000), (2, 4097), (1, 50280), (3, 8193), (1, 151937)])
def test_beams(W, G, V):
    logits, scores, g = some_logits(G, W, V, W + V)
    check_beams(logits, scores)
    done = (torch.rand(G, W, generator=g) < 0.3).int()
    check_beams(logits, scores, done, eos=V // 2)
    check_beams(logits, scores, done * 5, eos=V // 2, in_place=True)
    scores[:, 1:] = -math.inf  # a request's first step
    check_beams(logits, scores, torch.zeros_like(done), eos=0, in_place=True)


@pytest.mark.parametrize("W", [1, 4, 32])
@pytest.mark.parametrize("V", [3, 600, 9001, 20000])
def test_equal_candidates_go_by_beam_and_token(W, V):
    # a beam's logits take few values, both noughts among them; the beams are the same
    g = torch.Generator().manual_seed(V)
    row = torch.randint(-1, 2, (V,), generator=g).float() * 0.5
    row[::3] *= -1.0
    row = torch.where((row == 0) & (torch.arange(V) % 2 == 0), -0.0, row)
    logits = row.expand(2, W, V).contiguous()
    check_beams(logits, torch.full((2, W), -1.0))
    check_beams(torch.zeros(2, W, V), torch.full((2, W), -1.0))
    check_beams(torch.full((1, W, V), -2.5), torch.arange(W).float().flip(0).view(1, W))


@pytest.mark.parametrize("W", [1, 3, 8, 32])
@pytest.mark.parametrize("V", [40, 5000, 50280])
def test_masked_vocabularies(W, V):
    # most tokens have -inf: fewer candidates with a number than beams, none at all, or just as many
    for left in (0, 1, 2, W, W + 1, 5 * W):
        logits, scores, g = some_logits(2, W, V, left + V)
        allowed = torch.randperm(V, generator=g)[:left]
        masked = torch.full_like(logits, -math.inf)
        masked[:, :, allowed] = logits[:, :, allowed]
        check_beams(masked, scores)
        masked[0, 0] = logits[0, 0]
        check_beams(masked, scores, (torch.rand(2, W, generator=g) < 0.5).int(), eos=3)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("W,V", [(1, 50), (4, 3000), (32, 5000), (5, 50280)])
def test_what_is_no_number(W, V, bad):
    logits, scores, g = some_logits(3, W, V, 9)
    logits[0, 0, V - 1] = bad           # a beam without a sum
    logits[1, :, V // 2] = bad          # all beams of a request
    scores[2, W - 1] = bad
    check_beams(logits, scores)
    check_beams(logits, scores, torch.ones(3, W).int(), eos=-1)  # done, and nothing to go on with
    check_beams(logits, scores, torch.ones(3, W).int(), eos=V)
    check_beams(logits, -scores.abs() * math.inf)


def test_logits_far_apart():
    g = torch.Generator().manual_seed(2)
    for spread in (30.0, 1e4, 3e37):
        logits = (torch.rand(2, 4, 6000, generator=g) * 2 - 1) * spread
        scores = torch.tensor([[0.0, -1.0, -2.0, -3.0], [-5.0, -5.5, -5.25, -5.125]])
        out = [torch.zeros(2, 4, device="cuda", dtype=dtype) for dtype in (torch.int32, torch.int32, torch.float32)]
        ops.beam_select(logits.cuda(), scores.cuda(), None, *out, None)
        want = chosen(logits, scores, torch.zeros(2, 4).int(), -1)
        assert torch.equal(out[0].cpu(), want[0]) and torch.equal(out[1].cpu(), want[1])


@pytest.mark.parametrize("base", [1e5, -1e5, 2.0 ** 20 - 40, 2.0 ** 20 + 40, -2.0 ** 20, 3e6])
def test_logits_far_from_nought(base):
    # steps of a quarter up to 64, exact in fp32 beside the base: the differences alone count
    g = torch.Generator().manual_seed(3)
    logits = (torch.randint(0, 256, (3, 4, 20000), generator=g) / 4.0 + base).float()
    check_beams(logits, -torch.rand(3, 4, generator=g))


@pytest.mark.parametrize("W,step", [(8, 1e-3), (2, 1e-3), (32, 1e-3), (8, -1e-3), (8, 0.0)])
def test_rising_and_falling_logits(W, step):
    # every one beats what came before it, or none does, or all are the same; rows of several pieces each
    G, V = 520 // W, 20001
    logits = (torch.arange(V) * step).expand(G, W, V).contiguous()
    check_beams(logits, -torch.arange(G * W).view(G, W) / 64.0)


@pytest.mark.parametrize("W", [3, 8, 16, 32])
@pytest.mark.parametrize("G,V", [(1, 3000), (2, 20000), (2, 92931), (20, 3157)])
@pytest.mark.parametrize("apart", [0.0, 0.3, 2.0, 50.0])
def test_some_beams_lead_the_others(W, G, V, apart):
    # most of the best, or all of them, are one beam's
    logits, scores, g = some_logits(G, W, V, W + G, spread=1.0)
    check_beams(logits, (-apart * torch.randperm(W, generator=g)).expand(G, W).contiguous(), (torch.arange(W) % 5 == 4).int().expand(G, W).contiguous(), eos=2)


def test_many_groups():
    logits, scores, g = some_logits(700, 2, 301, 4)
    check_beams(logits, scores, (torch.rand(700, 2, generator=g) < 0.2).int(), eos=7)
    logits, scores, g = some_logits(70001, 1, 3, 4)  # (more than a grid holds)
    check_beams(logits, scores, (torch.rand(70001, 1, generator=g) < 0.2).int(), eos=1, in_place=True)
