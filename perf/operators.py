"""The operators of one decoding step with drafted tokens, and the work they are measured by.

A small model proposes a tree of tokens behind the last chosen one, the large model scores every node in one pass over its
key/value cache, the proposals are checked against its probabilities, and what was accepted joins the cache:

  q4      products of one row, or of the few rows of a tree, with 4-bit weights and group scales
  tree    attention of the tree's nodes over the cache, over their ancestors and over themselves
  verify  which path of the tree the target's probabilities accept, and the token behind it, from given random numbers
  append  the keys and values of the accepted path (or of a prompt) into the caches of all layers

`run` is one pass: the framework's call where `own` is set, else the same in elementary torch operations.  `exact` is the
definition in 64 bits, written apart from both.
"""
import math

import torch

own = False

EPI_BIAS, EPI_ADD2, EPI_ADD2_F32, EPI_GELU = 0, 1, 2, 3


def listed():
    return [
        # the fused query/key/value projection of a 2560-wide model's decode step: a launch more than a stream
        {"name": "q4_row_7680x2560", "kind": "q4", "M": 1, "N": 7680, "K": 2560, "group": 32, "epi": EPI_BIAS},
        # the vocabulary projection of the drafting model: the largest product of a single row
        {"name": "q4_row_50280x4096", "kind": "q4", "M": 1, "N": 50280, "K": 4096, "group": 32, "epi": EPI_BIAS},
        # a tree of 13 nodes through an up projection with its GELU (odd rows, the wide groups of other checkpoints)
        {"name": "q4_13_rows_11008x4096", "kind": "q4", "M": 13, "N": 11008, "K": 4096, "group": 128, "epi": EPI_GELU},
        # the largest tree through the down projection, both residuals added, widened for the next norm
        {"name": "q4_64_rows_2560x10240", "kind": "q4", "M": 64, "N": 2560, "K": 10240, "group": 32, "epi": EPI_ADD2_F32},
        # early in a conversation, nothing drafted: the shortest call
        {"name": "tree_1_after_127", "kind": "tree", "B": 1, "T": 1, "Tq": 1, "Hkv": 32, "g": 1, "d": 80, "len": 127},
        # a tree of 16 late in a long conversation
        {"name": "tree_16_after_3001", "kind": "tree", "B": 1, "T": 16, "Tq": 16, "Hkv": 32, "g": 1, "d": 80, "len": 3001},
        # sequences of different lengths served together, the last 9 nodes of trees of 25, four query heads to a key head
        {"name": "tree_7x9_after_2047", "kind": "tree", "B": 7, "T": 25, "Tq": 9, "Hkv": 8, "g": 4, "d": 128, "len": 2047},
        # the largest tree over a long document
        {"name": "tree_64_after_65533", "kind": "tree", "B": 1, "T": 64, "Tq": 64, "Hkv": 8, "g": 4, "d": 128, "len": 65533},
        # one conversation, four tokens drafted in a row
        {"name": "verify_1x5", "kind": "verify", "B": 1, "T": 5, "V": 50280, "shape": "chain"},
        # sequences served together, wide trees
        {"name": "verify_32x31", "kind": "verify", "B": 32, "T": 31, "V": 50280, "shape": "tree"},
        # what a step keeps of its trees, in all layers
        {"name": "append_path_4x25", "kind": "append", "L": 32, "B": 4, "T": 25, "Hkv": 8, "d": 128, "C": 512, "path": True},
        # a prompt joins an empty cache
        {"name": "append_prompt_2047", "kind": "append", "L": 1, "B": 1, "T": 2047, "Hkv": 32, "d": 80, "C": 4096, "path": False},
    ]


def _log_int(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    limit = max(work(c)["bytes"] for c in listed()), max(work(c)["flops"] for c in listed())
    while True:
        kind = rng.choice(("q4", "tree", "tree", "verify", "append"))
        if kind == "q4":
            group = rng.choice((32, 64, 128))
            case = {"kind": kind, "M": _log_int(rng, 1, 64), "N": _log_int(rng, 64, 50280), "K": group * _log_int(rng, 4, 11008 // group),
                    "group": group, "epi": rng.choice((EPI_BIAS, EPI_ADD2, EPI_ADD2_F32, EPI_GELU))}
        elif kind == "tree":
            T = _log_int(rng, 1, 64)
            case = {"kind": kind, "B": _log_int(rng, 1, 16), "T": T, "Tq": rng.choice((T, T, rng.randint(1, T))),
                    "Hkv": rng.choice((1, 2, 4, 8, 32)), "g": rng.choice((1, 2, 3, 4, 8)), "d": rng.choice((64, 72, 80, 96, 128, 256)),
                    "len": _log_int(rng, 1, 32768)}
        elif kind == "verify":
            case = {"kind": kind, "B": _log_int(rng, 1, 32), "T": _log_int(rng, 1, 64), "V": _log_int(rng, 1000, 128256),
                    "shape": rng.choice(("chain", "tree"))}
            if case["B"] * case["T"] * case["V"] > 32 * 31 * 50280:
                continue
        else:
            path = rng.random() < 0.5
            case = {"kind": kind, "L": _log_int(rng, 1, 32), "B": _log_int(rng, 1, 8), "T": _log_int(rng, 1, 64 if path else 1024),
                    "Hkv": rng.choice((1, 2, 8, 32)), "d": rng.choice((64, 72, 80, 128, 256)), "C": _log_int(rng, 1024, 4096), "path": path}
            if case["L"] * case["B"] * case["C"] * case["Hkv"] * case["d"] > 1 << 28:
                continue
        w = work(case)
        if w["bytes"] <= limit[0] and w["flops"] <= limit[1]:
            return case


def _lens(case):
    """The sequences' lengths before the call: the first the longest, the others down to about half of it."""
    n = case["len"]
    return [max(0, n - b * n // (2 * case["B"]) - b % 3) for b in range(case["B"])]


def work(case):
    if case["kind"] == "q4":
        M, N, K, epi = case["M"], case["N"], case["K"], case["epi"]
        out = M * N * (4 if epi == EPI_ADD2_F32 else 2)
        res = 2 * M * N * 2 if epi in (EPI_ADD2, EPI_ADD2_F32) else 0
        return {"bytes": N * K // 2 + 2 * N * K // case["group"] + 2 * M * K + 2 * N + res + out, "flops": 2 * M * N * K}
    if case["kind"] == "tree":
        B, T, Tq, Hkv, g, d = (case[k] for k in ("B", "T", "Tq", "Hkv", "g", "d"))
        keys = sum(_lens(case))
        return {"bytes": 4 * keys * Hkv * d + 4 * B * T * Hkv * d + 4 * B * Tq * Hkv * g * d + 4 * B * (T + 1),
                "flops": 4 * keys * Hkv * g * Tq * d}
    if case["kind"] == "verify":
        # a row of the target's at each sequence's end, and of the draft's where a proposal was turned down there
        B, T, V = case["B"], case["T"], case["V"]
        return {"bytes": 8 * B * V + 16 * B * T, "flops": 4 * B * V}
    L, B, T, Hkv, d = (case[k] for k in ("L", "B", "T", "Hkv", "d"))
    rows = sum(_kept(case, b) for b in range(B))
    return {"bytes": 2 * 2 * 2 * L * rows * Hkv * d, "flops": 0}


def _kept(case, b):
    """How many rows of sequence b an append keeps: all, or a path of up to six nodes."""
    return min(case["T"], 2 + b % 5) if case["path"] else case["T"]


def _parents(B, T, shape, gen):
    """A node's parent, -1 at the root: a chain, or one of the up to eight nodes before it."""
    node = torch.arange(T, device="cuda").expand(B, T)
    back = torch.ones(B, T, device="cuda") if shape == "chain" else 1 + torch.floor(torch.rand(B, T, generator=gen, device="cuda") * 8)
    parents = torch.maximum(node - back, torch.zeros_like(back))
    return torch.where(node == 0, torch.full_like(back, -1), parents).to(torch.int32).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def whole(hi, *shape):
        return torch.randint(0, hi, shape, generator=gen, device="cuda", dtype=torch.int32)

    state = dict(case)
    if case["kind"] == "q4":
        M, N, K, group = (case[k] for k in ("M", "N", "K", "group"))
        x = normal(M, K) * torch.where(torch.rand(K, generator=gen, device="cuda") < 0.01, 8.0, 1.0)  # a few loud channels
        state["x"] = x.half()
        words = torch.randint(-2 ** 31, 2 ** 31, (N, K // 8), generator=gen, device="cuda", dtype=torch.int64)
        state["Wq"] = words.to(torch.int32)
        state["scale"] = ((0.5 + torch.rand(N, K // group, generator=gen, device="cuda")) / (4 * math.sqrt(K))).half()
        state["bias"] = normal(N).half()
        two = case["epi"] in (EPI_ADD2, EPI_ADD2_F32)
        state["res1"], state["res2"] = (normal(M, N).half(), normal(M, N).half()) if two else (None, None)
        state["y"] = torch.empty(M, N, device="cuda", dtype=torch.float32 if case["epi"] == EPI_ADD2_F32 else torch.float16)
    elif case["kind"] == "tree":
        B, T, Tq, Hkv, g, d = (case[k] for k in ("B", "T", "Tq", "Hkv", "g", "d"))
        C = case["len"] + T
        lean = normal(Hkv, 1, d)  # the channels of a key head do not centre on zero
        state["Q"] = normal(B, Tq, Hkv * g, d).half()
        state["K"] = (normal(B, T, Hkv, d) + lean.transpose(0, 1)).half()
        state["V"] = normal(B, T, Hkv, d).half()
        state["K_cache"] = torch.empty(B, Hkv, C, d, device="cuda", dtype=torch.float16)
        state["V_cache"] = torch.empty(B, Hkv, C, d, device="cuda", dtype=torch.float16)
        for b in range(B):
            state["K_cache"][b] = (normal(Hkv, C, d) + lean).half()
            state["V_cache"][b] = normal(Hkv, C, d).half()
        state["host_lens"] = _lens(case)
        state["lens"] = torch.tensor(state["host_lens"], device="cuda", dtype=torch.int32)
        state["parents"] = _parents(B, T, "tree", gen)
        state["out"] = torch.empty(B, Tq, Hkv * g, d, device="cuda", dtype=torch.float16)
    elif case["kind"] == "verify":
        B, T, V = case["B"], case["T"], case["V"]
        state["parents"] = _parents(B, T, case["shape"], gen)
        logits = normal(B * T, V) * 2.5
        state["target"] = torch.softmax(logits, -1).view(B, T, V)
        state["draft"] = torch.softmax(logits + 0.5 * normal(B * T, V), -1).view(B, T, V)
        tokens = torch.empty(B, T, device="cuda", dtype=torch.int32)
        for b in range(B):  # a node's token is drawn from its parent's draft
            rows = state["draft"][b, state["parents"][b].clamp(min=0).long()]
            tokens[b] = torch.multinomial(rows, 1, generator=gen)[:, 0].to(torch.int32)
        state["tokens"] = tokens
        state["accept"] = torch.rand(B, T, generator=gen, device="cuda")
        state["sample"] = torch.rand(B, generator=gen, device="cuda")
        state["path"] = torch.empty(B, T, device="cuda", dtype=torch.int32)
        state["count"] = torch.empty(B, device="cuda", dtype=torch.int32)
        state["next_token"] = torch.empty(B, device="cuda", dtype=torch.int32)
    else:
        L, B, T, Hkv, d, C = (case[k] for k in ("L", "B", "T", "Hkv", "d", "C"))
        state["K"], state["V"] = normal(L, B, T, Hkv, d).half(), normal(L, B, T, Hkv, d).half()
        state["K_cache"] = torch.empty(L, B, Hkv, C, d, device="cuda", dtype=torch.float16)
        state["V_cache"] = torch.empty(L, B, Hkv, C, d, device="cuda", dtype=torch.float16)
        for layer in range(L):
            state["K_cache"][layer] = normal(B, Hkv, C, d).half()
            state["V_cache"][layer] = normal(B, Hkv, C, d).half()
        room = C - T  # a prompt's cache is empty, a path's at any length that leaves room
        state["lens"] = whole(room + 1, B) if case["path"] else torch.zeros(B, device="cuda", dtype=torch.int32)
        if case["path"]:
            order = torch.rand(B, T, generator=gen, device="cuda")
            count = torch.tensor([_kept(case, b) for b in range(B)], device="cuda", dtype=torch.int32)
            order[:, 0] = -1.0  # the root leads, the others follow in ascending order, -1 behind the last
            kept = torch.argsort(order, dim=1)
            slot = torch.arange(T, device="cuda")
            kept = torch.where(slot < count[:, None], kept, torch.full_like(kept, T)).sort(dim=1)[0]
            state["path"] = torch.where(kept < T, kept, torch.full_like(kept, -1)).to(torch.int32).contiguous()
            state["count"] = count
        else:
            state["path"] = state["count"] = None
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from dtas_amd import ops
    if s["kind"] == "q4":
        ops.gemv_q4(s["x"], s["Wq"], s["scale"], s["bias"], s["y"], epilogue=s["epi"], res1=s["res1"], res2=s["res2"])
        return s["y"]
    if s["kind"] == "tree":
        ops.attn_tree(s["Q"], s["K"], s["V"], s["K_cache"], s["V_cache"], s["lens"], s["parents"], s["out"])
        return s["out"]
    if s["kind"] == "verify":
        ops.verify_tree(s["target"], s["draft"], s["tokens"], s["parents"], s["accept"], s["sample"], s["path"], s["count"], s["next_token"])
        return s["path"], s["count"], s["next_token"]
    ops.cache_append(s["K"], s["V"], s["path"], s["count"], s["K_cache"], s["V_cache"], s["lens"])
    return s["K_cache"], s["V_cache"]


def _plain(s):
    return {"q4": _plain_q4, "tree": _plain_tree, "verify": _plain_verify, "append": _plain_append}[s["kind"]](s)


def _plain_q4(s):
    N, K = s["N"], s["K"]
    shifts = torch.arange(0, 32, 4, device=s["Wq"].device, dtype=torch.int32)
    W = ((s["Wq"][:, :, None] >> shifts) & 15).view(N, K // s["group"], s["group"]).float() - 7.0
    W = (W * s["scale"].float()[:, :, None]).view(N, K)
    y = s["x"].float() @ W.t() + s["bias"].float()
    if s["epi"] == EPI_GELU:
        y = 0.5 * y * torch.erfc(-y * math.sqrt(0.5))
    elif s["epi"] != EPI_BIAS:
        y = y + s["res1"].float() + s["res2"].float()
    return y if s["epi"] == EPI_ADD2_F32 else y.half()


def _visible(parents, rows):
    """[B, rows, T]: which nodes the last `rows` nodes see, their ancestors and themselves."""
    B, T = parents.shape
    node = torch.arange(T, device=parents.device)
    at = node.expand(B, T).clone()
    seen = torch.zeros(B, T, T, device=parents.device, dtype=torch.bool)
    for _ in range(T):
        seen = seen | (at[:, :, None] == node)
        up = torch.gather(parents.long(), 1, at.clamp(min=0))
        at = torch.where((at >= 0) & (up >= 0) & (up < at), up, torch.full_like(at, -1))
    return seen[:, T - rows:]


def _plain_tree(s):
    B, Tq, Hkv, g, d = (s[k] for k in ("B", "Tq", "Hkv", "g", "d"))
    seen = _visible(s["parents"], Tq)
    out = []
    for b in range(B):
        n = s["host_lens"][b]
        q = s["Q"][b].float().view(Tq, Hkv, g, d).permute(1, 2, 0, 3).reshape(Hkv, g * Tq, d) / math.sqrt(d)
        k = torch.cat((s["K_cache"][b, :, :n], s["K"][b].transpose(0, 1)), 1).float()
        v = torch.cat((s["V_cache"][b, :, :n], s["V"][b].transpose(0, 1)), 1).float()
        scores = q @ k.transpose(1, 2)
        hidden = torch.cat((torch.zeros(Tq, n, device=q.device, dtype=torch.bool), ~seen[b]), 1).repeat(g, 1)
        scores = scores.masked_fill(hidden, float("-inf"))
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = (p @ v) / p.sum(-1, keepdim=True)
        out.append(o.view(Hkv, g, Tq, d).permute(2, 0, 1, 3).reshape(Tq, Hkv * g, d))
    return torch.stack(out).half()


def _plain_verify(s):
    # every sequence walks one node at a time; 64 bits, since a token is chosen next to a border
    target, draft, tokens, parents = s["target"], s["draft"], s["tokens"].long(), s["parents"].long()
    B, T, V = target.shape
    each = torch.arange(B, device=target.device)
    at = torch.zeros(B, device=target.device, dtype=torch.long)
    c = torch.zeros(B, device=target.device, dtype=torch.float64)
    left = torch.ones_like(c)  # the sum of max(p - c q, 0)
    path = torch.full((B, T), -1, device=target.device, dtype=torch.int32)
    path[:, 0] = 0
    count = torch.ones_like(at)
    for i in range(1, T):
        x = tokens[:, i]
        offered = (parents[:, i] == at) & (x >= 0) & (x < V)
        xs = x.clamp(0, V - 1)
        p, q = target[each, at, xs].double(), draft[each, at, xs].double()
        taken = offered & (s["accept"][:, i].double() * q * left < (p - c * q).clamp(min=0))
        refused = offered & ~taken
        c = torch.where(refused, c + left, c)
        rest = (target[each, at].double() - c[:, None] * draft[each, at].double()).clamp(min=0).sum(-1)
        left = torch.where(refused, rest, left)
        at = torch.where(taken, torch.full_like(at, i), at)
        c = torch.where(taken, torch.zeros_like(c), c)
        left = torch.where(taken, torch.ones_like(left), left)
        path.scatter_(1, torch.where(taken, count, torch.zeros_like(count))[:, None], torch.where(taken, at, torch.zeros_like(at))[:, None].to(torch.int32))
        count = count + taken
    p = target[each, at].double()
    w = (p - c[:, None] * draft[each, at].double()).clamp(min=0)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p)
    upto = w.cumsum(-1)
    before = (upto <= s["sample"].double()[:, None] * upto[:, -1:]).sum(-1)
    last = torch.where(w > 0, torch.arange(V, device=w.device), torch.zeros(1, device=w.device, dtype=torch.long)).amax(-1)
    return path, count.to(torch.int32), torch.minimum(before, last).to(torch.int32)


def _plain_append(s):
    L, B, T, C = s["L"], s["B"], s["T"], s["C"]
    slot = torch.arange(T, device=s["K"].device)
    to = (s["lens"].long()[:, None] + slot) % C
    keep = slot.expand(B, T) < (s["count"][:, None] if s["path"] is not None else T)
    source = s["path"].long().clamp(min=0) if s["path"] is not None else slot.expand(B, T)
    each = torch.arange(B, device=s["K"].device)[:, None]
    for new, cache in ((s["K"], s["K_cache"]), (s["V"], s["V_cache"])):
        old = cache[:, each, :, to]  # (B, T, L, Hkv, d): the rows that are not kept stay as they were
        rows = new[:, each, source].permute(1, 2, 0, 3, 4)
        cache[:, each, :, to] = torch.where(keep[:, :, None, None, None], rows, old)
    return s["K_cache"], s["V_cache"]


def exact(case, seed):
    s = prepare(case, seed)
    return {"q4": _exact_q4, "tree": _exact_tree, "verify": _exact_verify, "append": _exact_append}[case["kind"]](s)


def _exact_q4(s):
    total = torch.zeros(s["M"], s["N"], device="cuda", dtype=torch.float64)
    x, scale = s["x"].double(), s["scale"].double().repeat_interleave(s["group"] // 8, dim=1)
    for j in range(8):  # the j-th of every eight weights
        w = (torch.bitwise_right_shift(s["Wq"].long(), 4 * j) % 16 - 7).double()
        total += x[:, j::8] @ (w * scale).t()
    total += s["bias"].double()
    if s["epi"] == EPI_GELU:
        total = total * torch.special.ndtr(total)
    elif s["epi"] != EPI_BIAS:
        total = (total + s["res1"].double()) + s["res2"].double()
    return total


def _exact_tree(s):
    B, T, Tq, Hkv, g, d = (s[k] for k in ("B", "T", "Tq", "Hkv", "g", "d"))
    if 2 * Hkv * g * Tq * sum(s["host_lens"]) * d > 1 << 37:
        return None
    parents = s["parents"].tolist()
    out = torch.empty(B, Tq, Hkv * g, d, device="cuda", dtype=torch.float64)
    for b in range(B):
        n = s["host_lens"][b]
        for h in range(Hkv):
            keys = torch.cat((s["K_cache"][b, h, :n], s["K"][b, :, h])).double()
            values = torch.cat((s["V_cache"][b, h, :n], s["V"][b, :, h])).double()
            scores = torch.matmul(s["Q"][b, :, h * g:(h + 1) * g].double(), keys.t().contiguous()) * d ** -0.5
            for t in range(Tq):
                line, node = {T - Tq + t}, T - Tq + t
                while 0 <= parents[b][node] < node:
                    node = parents[b][node]
                    line.add(node)
                others = [n + i for i in range(T) if i not in line]
                scores[t, :, others] = -math.inf
            out[b, :, h * g:(h + 1) * g] = torch.matmul(torch.softmax(scores, -1), values)
    return out


def _exact_verify(s):
    target, draft = s["target"], s["draft"]
    tokens, parents, accept, sample = (s[k].tolist() for k in ("tokens", "parents", "accept", "sample"))
    B, T, V = target.shape
    paths, counts, nexts = [], [], []
    for b in range(B):
        at, path = 0, [0]
        while True:
            p, q = target[b, at].double().cpu(), draft[b, at].double().cpu()
            here = p.clone()
            for i in range(at + 1, T):
                x = tokens[b][i]
                if parents[b][i] != at or not 0 <= x < V:
                    continue
                if accept[b][i] * float(q[x]) < float(here[x]):
                    path.append(i)
                    break
                rest = torch.relu(here - q)  # what is left of the target once a draw of q was turned down
                mass = float(rest.sum())
                here = rest / mass if mass > 0 else rest
            if path[-1] == at:
                break
            at = path[-1]
        if float(here.sum()) == 0:
            here = p
        upto = torch.cumsum(here, 0)
        behind = torch.nonzero(upto > sample[b] * float(upto[-1]))
        nexts.append(int(behind[0]) if len(behind) else int(torch.nonzero(here)[-1]))
        counts.append(len(path))
        paths.append(path + [-1] * (T - len(path)))
    return (torch.tensor(paths, device="cuda", dtype=torch.int32), torch.tensor(counts, device="cuda", dtype=torch.int32),
            torch.tensor(nexts, device="cuda", dtype=torch.int32))


def _exact_append(s):
    caches = []
    for new, cache in ((s["K"], s["K_cache"]), (s["V"], s["V_cache"])):
        cache = cache.clone()
        for b in range(s["B"]):
            rows = s["path"][b, :int(s["count"][b])].tolist() if s["path"] is not None else list(range(s["T"]))
            start = int(s["lens"][b])
            cache[:, b, :, start:start + len(rows)] = new[:, b, rows].transpose(1, 2)
        caches.append(cache.double())
    return tuple(caches)
