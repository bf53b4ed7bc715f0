"""The operators of requests served together from one pool of pages, beams among them, and the work they are measured by.

Keys and values of all requests lie in pages, taken as the requests grow; a table names each sequence's pages in order.

  assign   pages for the rows that join, and the slot of each of them, from the requests' lengths
  append   the rows' keys and values into their slots
  paged    attention of one new token per sequence over its pages
  beam     the best continuations of each request's beams over the vocabulary
  reorder  tables and lengths follow the beams that were chosen, part-filled pages are copied, pages nobody names are given back

`run` is one pass: the framework's call where `own` is set, else the same in elementary torch operations.  `exact` is the
definition in 64 bits, written apart from both.
"""
import math

import torch

own = False


def listed():
    return [
        # a step of a server with 64 conversations: a token each, one in ten finished
        {"name": "assign_64_tokens", "kind": "assign", "B": 64, "rows": 1, "packed": False, "page": 16, "len": 4096, "short": False},
        # prompts and pieces of prompts of very different lengths, one behind the other, joining an almost full pool
        {"name": "assign_packed_16384", "kind": "assign", "B": 37, "rows": 16384, "packed": True, "page": 32, "len": 8192, "short": True},
        # a layer's new keys and values of 64 conversations
        {"name": "append_64_tokens", "kind": "append", "L": 1, "N": 64, "run": 1, "Hkv": 8, "d": 128, "page": 16, "pages": 2048},
        # a layer's of packed prompts, the end of the batch unused
        {"name": "append_packed_2047", "kind": "append", "L": 1, "N": 2047, "run": 190, "Hkv": 32, "d": 80, "page": 32, "pages": 160},
        # one conversation at its start, 32 heads of 80 without sharing: the shortest call
        {"name": "paged_1_after_127", "kind": "paged", "B": 1, "beams": 1, "Hkv": 32, "g": 1, "d": 80, "page": 16, "len": 127},
        # four beams behind one long document
        {"name": "paged_4_beams_after_32749", "kind": "paged", "B": 4, "beams": 4, "Hkv": 8, "g": 4, "d": 128, "page": 64, "len": 32749},
        # conversations of all lengths served together, one of them empty
        {"name": "paged_61_after_2047", "kind": "paged", "B": 61, "beams": 1, "Hkv": 8, "g": 4, "d": 128, "page": 16, "len": 2047},
        # the largest: few, long, eight query heads to a key head
        {"name": "paged_16_after_65533", "kind": "paged", "B": 16, "beams": 1, "Hkv": 8, "g": 8, "d": 128, "page": 128, "len": 65533},
        # one request of four beams
        {"name": "beam_1x4", "kind": "beam", "G": 1, "W": 4, "V": 50280},
        # 32 requests of eight
        {"name": "beam_32x8", "kind": "beam", "G": 32, "W": 8, "V": 50280},
        # the four beams of one request, early, 32 layers
        {"name": "reorder_1x4", "kind": "reorder", "G": 1, "W": 4, "L": 32, "Hkv": 8, "d": 128, "page": 16, "len": 301},
        # 24 requests of eight beams, half a page to copy for many of them
        {"name": "reorder_24x8", "kind": "reorder", "G": 24, "W": 8, "L": 16, "Hkv": 8, "d": 128, "page": 32, "len": 1037},
    ]


def _log_int(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    limit = max(work(c)["bytes"] for c in listed()), max(work(c)["flops"] for c in listed())
    while True:
        kind = rng.choice(("assign", "append", "paged", "paged", "paged", "beam", "reorder"))
        if kind == "assign":
            packed = rng.random() < 0.5
            B = _log_int(rng, 1, 256)
            case = {"kind": kind, "B": B, "rows": _log_int(rng, B, 32768) if packed else _log_int(rng, 1, 64), "packed": packed,
                    "page": rng.choice((1, 8, 16, 24, 32, 64, 128)), "len": _log_int(rng, 1, 16384), "short": rng.random() < 0.5}
            if B * case["len"] > 1 << 20:
                continue
        elif kind == "append":
            N = _log_int(rng, 1, 4096)
            case = {"kind": kind, "L": _log_int(rng, 1, 32), "N": N, "run": _log_int(rng, 1, max(1, N // 2)), "Hkv": rng.choice((1, 2, 8, 32)),
                    "d": rng.choice((64, 72, 80, 128, 256)), "page": rng.choice((8, 16, 24, 32, 64, 128)), "pages": 0}
            case["pages"] = N // case["page"] + 2 * _up(N, case["run"]) + _log_int(rng, 1, 64)
            if case["L"] * case["pages"] * case["page"] * case["Hkv"] * case["d"] > 1 << 27:
                continue
        elif kind == "paged":
            beams = rng.choice((1, 1, 2, 4, 5, 8))
            case = {"kind": kind, "B": beams * _log_int(rng, 1, max(1, 64 // beams)), "beams": beams, "Hkv": rng.choice((1, 2, 4, 8, 32)),
                    "g": rng.choice((1, 2, 3, 4, 8)), "d": rng.choice((64, 72, 80, 96, 128, 256)), "page": rng.choice((16, 16, 32, 48, 64, 128, 256)),
                    "len": _log_int(rng, 1, 65536)}
        elif kind == "beam":
            case = {"kind": kind, "G": _log_int(rng, 1, 64), "W": rng.choice((1, 2, 3, 4, 5, 8, 16, 32)), "V": _log_int(rng, 1000, 151936)}
            if case["G"] * case["W"] * case["V"] > 32 * 8 * 50280:
                continue
        else:
            case = {"kind": kind, "G": _log_int(rng, 1, 32), "W": rng.choice((1, 2, 3, 4, 5, 8, 16, 32)), "L": _log_int(rng, 1, 32),
                    "Hkv": rng.choice((1, 2, 8, 32)), "d": rng.choice((64, 72, 80, 128, 256)), "page": rng.choice((8, 16, 24, 32, 64, 128)),
                    "len": _log_int(rng, 1, 4096)}
            if case["G"] * case["W"] * case["len"] > 1 << 18 or _pool(case) * case["L"] * case["page"] * case["Hkv"] * case["d"] > 1 << 28:
                continue
        w = work(case)
        if w["bytes"] <= limit[0] and w["flops"] <= limit[1]:
            return case


def _up(n, page):
    return -(-n // page)


def _groups(case):
    """Per request (a group of beams): the length of its beams, and how many of their first pages they share."""
    page, n = case["page"], case["len"]
    count, beams = (case["G"], case["W"]) if case["kind"] == "reorder" else (case["B"] // case["beams"], case["beams"])
    found = []
    for i in range(count):
        length = 0 if i == 5 and case["kind"] == "paged" else max(1, n - 7 * n * i // (8 * count) - i % 3)
        found.append((length, 0 if beams == 1 else 9 * length // 10 // page))
    return found


def _pool(case):
    """How many pages the pool of such a case holds: those that are named, and some more."""
    beams = case["W"] if case["kind"] == "reorder" else case["beams"]
    return sum(s + beams * (_up(n, case["page"]) - s) for n, s in _groups(case)) + beams * len(_groups(case)) + 3


def work(case):
    kind = case["kind"]
    if kind == "assign":
        B, rows = case["B"], case["rows"] * (1 if case["packed"] else case["B"])
        return {"bytes": 4 * rows + 12 * B + 8 * (rows // case["page"] + B) + 8, "flops": 0}
    if kind == "append":
        return {"bytes": 2 * 2 * 2 * case["L"] * case["N"] * case["Hkv"] * case["d"] + 4 * case["N"], "flops": 0}
    if kind == "paged":
        B, beams, Hkv, g, d, page = (case[k] for k in ("B", "beams", "Hkv", "g", "d", "page"))
        keys = sum(s * page + beams * (n - s * page) for n, s in _groups(case))
        return {"bytes": 4 * keys * Hkv * d + 4 * B * Hkv * g * d + 4 * B + 4 * beams * sum(_up(n, page) for n, _ in _groups(case)),
                "flops": 4 * sum(beams * n for n, _ in _groups(case)) * Hkv * g * d}
    if kind == "beam":
        G, W, V = case["G"], case["W"], case["V"]
        return {"bytes": 4 * G * W * V + 24 * G * W, "flops": 2 * G * W * V}
    # the tables, and about half of the rows of a part-filled page for each beam but its parent's first
    G, W, L, Hkv, d, page = (case[k] for k in ("G", "W", "L", "Hkv", "d", "page"))
    copied = sum((W // 3) * (n % page) for n, _ in _groups(case))
    return {"bytes": 8 * W * sum(_up(n, page) for n, _ in _groups(case)) + 12 * G * W + 2 * 2 * 2 * L * copied * Hkv * d, "flops": 0}


def _random_pages(gen, pages, *shape):
    """fp16 values for a pool of pages, made in pieces; the last three pages, which no table names, hold what memory holds."""
    cache = torch.empty(pages, *shape, device="cuda", dtype=torch.float16)
    lean = torch.randn(shape[-3] if len(shape) > 2 else 1, 1, shape[-1], generator=gen, device="cuda")  # a head's channels do not centre on zero
    step = max(1, (1 << 26) // max(1, math.prod(shape)))
    for at in range(0, pages, step):
        piece = cache[at:at + step]
        piece.copy_(torch.randn(piece.shape, generator=gen, device="cuda") + lean)
    cache[-3:] = float("nan")
    return cache


def _group_tables(case, gen, pages, columns):
    """Tables (groups, beams, columns) of distinct pages, the shared ones of a group in front; what is left of the pool."""
    beams = case["W"] if case["kind"] == "reorder" else case["beams"]
    order = torch.randperm(pages - 3, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(_groups(case)), beams, columns), -1, device="cuda", dtype=torch.int32)
    at = 0
    for i, (n, shared) in enumerate(_groups(case)):
        table[i, :, :shared] = order[at:at + shared]
        at += shared
        tail = _up(n, case["page"]) - shared
        table[i, :, shared:shared + tail] = order[at:at + beams * tail].view(beams, tail)
        at += beams * tail
    return table, order[at:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int32)

    def empty(dtype, *shape):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    state = dict(case)
    kind = case["kind"]
    if kind == "assign":
        B, rows, packed, page, n = (case[k] for k in ("B", "rows", "packed", "page", "len"))
        lens = whole(0, n + 1, B)
        if packed:  # pieces of prompts: half of the requests begin, and the batch is filled but for a little
            lens = torch.where(torch.rand(B, generator=gen, device="cuda") < 0.5, 0, lens)
            share = torch.exp(normal(B))
            count = torch.floor(share / share.sum() * rows * 0.98).to(torch.int32)
        else:
            count = whole(1, rows + 1, B) if rows > 1 else torch.ones_like(lens)
            count = torch.where(torch.rand(B, generator=gen, device="cuda") < 0.1, 0, count).to(torch.int32)
        lens = lens.to(torch.int32)
        have = (lens + page - 1) // page
        need = (lens + count + page - 1) // page - have
        columns = _up(n + rows, page)
        held, wanted = int(have.sum()), int(need.sum())
        left = max(1, wanted * 3 // 4) if case["short"] else wanted + B
        pages = held + left
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        column = torch.arange(columns, device="cuda")
        first = (have.cumsum(0) - have)[:, None]
        state["table"] = torch.where(column < have[:, None], order[(first + column).clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
        state["free"] = torch.cat((order[held:], torch.zeros_like(order[:held])))
        state["free_count"] = torch.tensor([left], device="cuda", dtype=torch.int32)
        state["lens"], state["count"] = lens, count
        state["starts"] = empty(torch.int32, B + 1) if packed else None
        state["slots"] = empty(torch.int32, rows) if packed else empty(torch.int32, B, rows)
        state["new_lens"], state["left"] = empty(torch.int32, B), empty(torch.int32, 1)
    elif kind == "append":
        L, N, run, Hkv, d, page, pages = (case[k] for k in ("L", "N", "run", "Hkv", "d", "page", "pages"))
        state["K"], state["V"] = normal(L, N, Hkv, d).half(), normal(L, N, Hkv, d).half()
        state["K_pages"] = normal(L, pages, Hkv, page, d).half()
        state["V_pages"] = normal(L, pages, Hkv, page, d).half()
        # runs of rows, each from some place in its first page on, through pages of its own; the last rows of a batch of runs are not in use
        row = torch.arange(N, device="cuda")
        each = row // run
        offset = whole(0, page, N)[each] + row % run
        needs = torch.zeros(_up(N, run) + 1, device="cuda", dtype=torch.long)
        needs[1:].scatter_reduce_(0, each, (offset // page + 1).long(), "amax", include_self=True)
        order = torch.randperm(pages, generator=gen, device="cuda")
        slots = order[needs.cumsum(0)[each] + offset // page] * page + offset % page
        slots = torch.where(row >= N - N // 50, -1, slots) if run > 1 else slots
        state["slots"] = slots.to(torch.int32)
    elif kind == "paged":
        B, beams, Hkv, g, d, page = (case[k] for k in ("B", "beams", "Hkv", "g", "d", "page"))
        pages, columns = _pool(case), _up(case["len"], page)
        state["Q"] = normal(B, Hkv * g, d).half()
        state["K_pages"] = _random_pages(gen, pages, Hkv, page, d)
        state["V_pages"] = _random_pages(gen, pages, Hkv, page, d)
        table, _ = _group_tables(case, gen, pages, columns)
        state["table"] = table.view(B, columns)
        state["host_lens"] = [n for n, _ in _groups(case) for _ in range(beams)]
        state["lens"] = torch.tensor(state["host_lens"], device="cuda", dtype=torch.int32)
        state["out"] = empty(torch.float16, B, Hkv * g, d)
    elif kind == "beam":
        G, W, V = case["G"], case["W"], case["V"]
        common = normal(G, 1, V) * 1.5  # the beams of a request expect much the same
        state["logits"] = (common + normal(G, W, V) * 1.5).contiguous()
        state["scores"] = (-8.0 - 2.0 * torch.rand(G, W, generator=gen, device="cuda")).sort(1, descending=True)[0].contiguous()
        state["done"] = (torch.rand(G, W, generator=gen, device="cuda") < 0.15).to(torch.int32)
        state["eos"] = 0
        state["tokens"], state["parents"], state["new_done"] = (empty(torch.int32, G, W) for _ in range(3))
        state["new_scores"] = empty(torch.float32, G, W)
    else:
        G, W, L, Hkv, d, page = (case[k] for k in ("G", "W", "L", "Hkv", "d", "page"))
        pages, columns = _pool(case), _up(case["len"], page) + 2
        table, rest = _group_tables(case, gen, pages, columns)
        state["table"] = table
        state["lens"] = torch.tensor([[n] * W for n, _ in _groups(case)], device="cuda", dtype=torch.int32)
        state["parents"] = torch.floor(W * torch.rand(G, W, generator=gen, device="cuda") ** 1.5).to(torch.int32)  # the better beams have more
        if G > 3:
            state["parents"][3] = -1  # a request that has come to its end
        state["free"] = torch.cat((rest, torch.zeros(pages - len(rest), device="cuda", dtype=torch.int32)))
        state["free_count"] = torch.tensor([len(rest)], device="cuda", dtype=torch.int32)
        state["new_table"], state["new_lens"], state["left"] = torch.full_like(table, -1), empty(torch.int32, G, W), empty(torch.int32, 1)
        state["K_pages"] = empty(torch.float16, L, pages, Hkv, page, d)
        state["V_pages"] = empty(torch.float16, L, pages, Hkv, page, d)
        for layer in range(L):
            state["K_pages"][layer] = normal(pages, Hkv, page, d).half()
            state["V_pages"][layer] = normal(pages, Hkv, page, d).half()
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from dtas_amd import ops
    if s["kind"] == "assign":
        ops.page_assign(s["lens"], s["count"], s["table"], s["free"], s["free_count"], s["page"], s["slots"], s["new_lens"], s["left"], starts=s["starts"])
        return _assigned(s)
    if s["kind"] == "append":
        ops.page_append(s["K"], s["V"], s["slots"], s["K_pages"], s["V_pages"])
        return s["K_pages"], s["V_pages"]
    if s["kind"] == "paged":
        ops.attn_paged(s["Q"], s["K_pages"], s["V_pages"], s["table"], s["lens"], s["out"], beams=s["beams"])
        return s["out"]
    if s["kind"] == "beam":
        ops.beam_select(s["logits"], s["scores"], s["done"], s["tokens"], s["parents"], s["new_scores"], s["new_done"], eos=s["eos"])
        return s["tokens"], s["parents"], s["new_scores"], s["new_done"]
    ops.page_reorder(s["parents"], s["table"], s["lens"], s["free"], s["free_count"], s["new_table"], s["new_lens"], s["left"], s["K_pages"], s["V_pages"])
    return s["new_table"], s["new_lens"], s["free"], s["left"], s["K_pages"], s["V_pages"]


def _assigned(s):
    return {k: s[k] for k in ("table", "slots", "new_lens", "left", "starts") if s[k] is not None}


def _plain(s):
    return {"assign": _plain_assign, "append": _plain_append, "paged": _plain_paged, "beam": _plain_beam, "reorder": _plain_reorder}[s["kind"]](s)


def _plain_assign(s):
    page, rows, packed = s["page"], s["rows"], s["packed"]
    B, columns = s["table"].shape
    lens, count = s["lens"].long(), s["count"].long()
    asked = count.clamp(min=0)
    behind = asked.cumsum(0)
    have = (lens + page - 1) // page
    fits = (lens >= 0) & (count >= 0) & (lens + count <= columns * page) & (behind <= rows if packed else count <= rows)
    need = torch.where(fits, (lens + asked + page - 1) // page - have, 0)
    upto, free_count = need.cumsum(0), s["free_count"].long()
    served = fits & ((need == 0) | (upto <= free_count))
    need = torch.where(served, need, 0)
    taken = need.sum()
    column = torch.arange(columns, device=lens.device)
    fresh = (column >= have[:, None]) & (column < (have + need)[:, None])
    at = free_count - 1 - (upto - need)[:, None] - (column - have[:, None])
    s["table"] = torch.where(fresh, s["free"][at.clamp(0, len(s["free"]) - 1)], s["table"])
    if packed:
        row = torch.arange(rows, device=lens.device)
        b = torch.searchsorted(behind, row, right=True).clamp(max=B - 1)
        t = row - (behind - asked)[b]
        real = (row < behind[-1]) & served[b]
    else:
        b = torch.arange(B, device=lens.device)[:, None]
        t = torch.arange(rows, device=lens.device)[None]
        real = (t < count[:, None]) & served[:, None]
    to = lens[b] + t
    slots = s["table"][b, (to // page).clamp(0, columns - 1)].long() * page + to % page
    s["slots"] = torch.where(real, slots, -1).to(torch.int32)
    s["new_lens"] = torch.where(served, lens + count, lens).to(torch.int32)
    s["left"] = (free_count - taken).to(torch.int32)
    if packed:
        s["starts"] = torch.cat((torch.zeros_like(behind[:1]), behind)).to(torch.int32)
    return _assigned(s)


def _plain_append(s):
    page = s["page"]
    keep = torch.nonzero(s["slots"] >= 0)[:, 0]
    slot = s["slots"].long()[keep]
    for new, cache in ((s["K"], s["K_pages"]), (s["V"], s["V_pages"])):
        cache[:, slot // page, :, slot % page] = new[:, keep].transpose(0, 1)
    return s["K_pages"], s["V_pages"]


def _plain_paged(s):
    B, Hkv, g, d, page = (s[k] for k in ("B", "Hkv", "g", "d", "page"))
    out = torch.zeros(B, Hkv * g, d, device=s["Q"].device)
    for b in range(B):
        n = s["host_lens"][b]
        if n == 0:
            continue
        held = s["table"][b, :_up(n, page)].long()
        k = s["K_pages"][held].transpose(0, 1).reshape(Hkv, -1, d)[:, :n].float()
        v = s["V_pages"][held].transpose(0, 1).reshape(Hkv, -1, d)[:, :n].float()
        q = s["Q"][b].float().view(Hkv, g, d) / math.sqrt(d)
        scores = q @ k.transpose(1, 2)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        out[b] = ((p @ v) / p.sum(-1, keepdim=True)).view(Hkv * g, d)
    return out.half()


def _plain_beam(s):
    # 64 bits: a beam is chosen next to a border
    G, W, V = s["G"], s["W"], s["V"]
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    total = s["scores"].double()[:, :, None] + x - torch.log(torch.exp(x).sum(-1, keepdim=True))
    ended = s["done"][:, :, None] != 0
    token = torch.arange(V, device=x.device)
    total = torch.where(ended, torch.where(token == s["eos"], s["scores"].double()[:, :, None], float("-inf")), total)
    best, at = torch.sort(total.view(G, W * V), dim=1, descending=True, stable=True)
    best, at = best[:, :W], at[:, :W]
    parents, tokens = at // V, at % V
    done = (torch.gather(s["done"].long(), 1, parents) != 0) | (tokens == s["eos"])
    return tokens.to(torch.int32), parents.to(torch.int32), best.float(), done.to(torch.int32)


def _plain_reorder(s):
    G, W, page = s["G"], s["W"], s["page"]
    table, lens, parents = s["table"], s["lens"].long(), s["parents"].long()
    columns, pages, device = table.shape[2], s["K_pages"].shape[1], table.device
    some = parents >= 0
    from_row = parents.clamp(min=0)
    new_lens = torch.where(some, torch.gather(lens, 1, from_row), 0)
    column = torch.arange(columns, device=device)
    named = column < ((lens + page - 1) // page)[:, :, None]
    new_named = column < ((new_lens + page - 1) // page)[:, :, None]
    wanted = torch.gather(table, 1, from_row[:, :, None].expand(G, W, columns))
    # pages of the old rows that no new row has in the same place, each once
    kept = torch.zeros_like(named)
    again = torch.zeros_like(named)
    for i in range(W):
        kept |= (table == wanted[:, i:i + 1]) & new_named[:, i:i + 1]
        again[:, i + 1:] |= (table[:, i + 1:] == table[:, i:i + 1]) & named[:, i:i + 1]
    given_back = torch.nonzero((named & ~kept & ~again).transpose(1, 2))
    returned = table[given_back[:, 0], given_back[:, 2], given_back[:, 1]]
    count = s["free_count"].long()
    n_back = len(returned)
    back_at = count + torch.arange(n_back, device=device)
    free = s["free"].clone()
    free[back_at] = returned
    # a part-filled page belongs to its row alone: all but a parent's first take a copy
    earlier = torch.zeros_like(some)
    for i in range(W):
        earlier[:, i + 1:] |= (parents[:, i + 1:] == parents[:, i:i + 1])
    copies = torch.nonzero(some & earlier & (new_lens % page != 0))
    n_copies = len(copies)
    new = free[(count + n_back - 1 - torch.arange(n_copies, device=device))]
    s["new_table"] = torch.where(new_named, wanted, s["new_table"])
    last = new_lens[copies[:, 0], copies[:, 1]] // page
    old = s["new_table"][copies[:, 0], copies[:, 1], last].long()
    s["new_table"][copies[:, 0], copies[:, 1], last] = new
    filled = (new_lens[copies[:, 0], copies[:, 1]] % page)[:, None] > torch.arange(page, device=device)
    new = new.long()
    for cache in (s["K_pages"], s["V_pages"]):
        cache[:, new] = torch.where(filled[None, :, None, :, None], cache[:, old], cache[:, new])
    return s["new_table"], new_lens.to(torch.int32), free, (count + n_back - n_copies).to(torch.int32), s["K_pages"], s["V_pages"]


def exact(case, seed):
    s = prepare(case, seed)
    return {"assign": _exact_assign, "append": _exact_append, "paged": _exact_paged, "beam": _exact_beam, "reorder": _exact_reorder}[case["kind"]](s)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _exact_assign(s):
    page, rows = s["page"], s["rows"]
    lens, count, table, free = (s[k].tolist() for k in ("lens", "count", "table", "free"))
    left, asked, short = int(s["free_count"]), 0, False
    slots = [-1] * (rows if s["packed"] else rows * len(lens))
    starts, new_lens = [0], list(lens)
    wanted = 0
    for b, n in enumerate(lens):
        begin = asked if s["packed"] else b * rows
        asked += max(0, count[b])
        starts.append(asked)
        if n < 0 or count[b] < 0 or n + count[b] > len(table[b]) * page or (asked if s["packed"] else count[b]) > rows:
            continue
        have, to = _up(n, page), _up(n + count[b], page)
        wanted += to - have
        if to > have and wanted > int(s["free_count"]):
            continue
        for c in range(have, to):
            left -= 1
            table[b][c] = free[left]
        for t in range(count[b]):
            slots[begin + t] = table[b][(n + t) // page] * page + (n + t) % page
        new_lens[b] = n + count[b]
    found = {"table": _ints(table), "slots": _ints(slots).view(s["slots"].shape), "new_lens": _ints(new_lens), "left": _ints([left])}
    if s["packed"]:
        found["starts"] = _ints(starts)
    return found


def _exact_append(s):
    caches = []
    for new, cache in ((s["K"], s["K_pages"]), (s["V"], s["V_pages"])):
        cache = cache.double()
        for n, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                cache[:, slot // s["page"], :, slot % s["page"]] = new[:, n].double()
        caches.append(cache)
    return tuple(caches)


def _exact_paged(s):
    B, Hkv, g, d, page = (s[k] for k in ("B", "Hkv", "g", "d", "page"))
    if sum(s["host_lens"]) * Hkv * g * d > 1 << 34:
        return None
    out = torch.zeros(B, Hkv * g, d, device="cuda", dtype=torch.float64)
    for b, n in enumerate(s["host_lens"]):
        if n == 0:
            continue
        place = torch.arange(n, device="cuda")
        pages = s["table"][b].long()[place // page]
        for h in range(Hkv):
            keys = s["K_pages"][pages, h, place % page].double()
            values = s["V_pages"][pages, h, place % page].double().t().contiguous()
            for r in range(h * g, (h + 1) * g):
                out[b, r] = torch.mv(values, torch.softmax(torch.mv(keys, s["Q"][b, r].double()) * d ** -0.5, 0))
    return out


def _exact_beam(s):
    G, W, V = s["G"], s["W"], s["V"]
    tokens, parents, scores, dones = [], [], [], []
    for i in range(G):
        candidates = []
        for w in range(W):
            score = float(s["scores"][i, w])
            if int(s["done"][i, w]):
                candidates.append((-score, w, s["eos"], 1))
                continue
            row = s["logits"][i, w].double()
            logs = torch.log_softmax(row, 0)
            bound = torch.topk(logs, min(W, V))[0][-1]
            for v in torch.nonzero(logs >= bound)[:, 0].tolist():
                candidates.append((-(score + float(logs[v])), w, v, int(v == s["eos"])))
        best = sorted(candidates)[:W]
        if len(best) < W:  # (all others have no chance: the first of them)
            taken = {(w, v) for _, w, v, _ in best}
            rest = ((w, v) for w in range(W) for v in range(V))
            while len(best) < W:
                w, v = next(rest)
                if (w, v) not in taken:
                    best.append((math.inf, w, v, int(bool(s["done"][i, w]) or v == s["eos"])))
        tokens.append([v for _, _, v, _ in best])
        parents.append([w for _, w, _, _ in best])
        scores.append([-c for c, _, _, _ in best])
        dones.append([e for _, _, _, e in best])
    return _ints(tokens), _ints(parents), torch.tensor(scores, device="cuda", dtype=torch.float64), _ints(dones)


def _exact_reorder(s):
    G, W, page = s["G"], s["W"], s["page"]
    table, lens, parents, free, new_table = (s[k].tolist() for k in ("table", "lens", "parents", "free", "new_table"))
    left = int(s["free_count"])
    caches = [s["K_pages"].double(), s["V_pages"].double()]
    new_lens, copies = [], []
    for i in range(G):
        rows = [table[i][w][:_up(lens[i][w], page)] for w in range(W)]
        taken = [rows[p] if p >= 0 else [] for p in parents[i]]
        new_lens.append([lens[i][p] if p >= 0 else 0 for p in parents[i]])
        for c in range(max(map(len, rows))):
            still = {row[c] for row in taken if c < len(row)}
            for row in rows:
                if c < len(row) and row[c] not in still:
                    still.add(row[c])
                    free[left] = row[c]
                    left += 1
        for w in range(W):
            new_table[i][w][:len(taken[w])] = taken[w]
            if parents[i][w] >= 0 and parents[i][w] in parents[i][:w] and new_lens[i][w] % page:
                copies.append((i, w))
    for i, w in copies:
        left -= 1
        column, filled = new_lens[i][w] // page, new_lens[i][w] % page
        old = new_table[i][w][column]
        new_table[i][w][column] = free[left]
        for cache in caches:
            cache[:, free[left], :, :filled] = cache[:, old, :, :filled]
    return _ints(new_table), _ints(new_lens), _ints(free), _ints([left]), caches[0], caches[1]
