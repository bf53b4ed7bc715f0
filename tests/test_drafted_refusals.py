"""What the operators of a step with drafted tokens refuse, and what they do nothing for: decided before any launch."""
import pytest
import torch

from dtas_amd import _lib, ops

A, B, C, D, E, F, G, H, I = (0x10000000 * (i + 1) for i in range(9))  # never dereferenced: every call ends before a launch


def call(name, *args):
    return getattr(_lib.lib(), name)(*args), _lib.last_error()


def q4(x=A, Wq=B, scale=C, bias=D, res1=None, res2=None, y=E, M=3, N=64, K=256, group=32, epilogue=0):
    return call("dtas_gemv_q4_f16", x, Wq, scale, bias, res1, res2, y, M, N, K, group, epilogue, None)


def tree(Q=A, K=B, V=C, Kc=D, Vc=E, lens=F, parents=G, out=H, batch=2, nodes=9, rows=9, heads=8, kv_heads=2, d=64, capacity=100, scale=0.125):
    return call("dtas_attn_tree_f16", Q, K, V, Kc, Vc, lens, parents, out, batch, nodes, rows, heads, kv_heads, d, capacity, scale, None)


def verify(target=A, draft=B, tokens=C, parents=D, accept=E, sample=F, path=G, count=H, next_token=I, batch=2, nodes=9, V=100):
    return call("dtas_verify_tree_f32", target, draft, tokens, parents, accept, sample, path, count, next_token, batch, nodes, V, None)


def append(K=A, V=B, path=C, count=D, Kc=E, Vc=F, lens=G, layers=2, batch=2, nodes=9, slots=9, kv_heads=2, d=64, capacity=100):
    return call("dtas_cache_append_f16", K, V, path, count, Kc, Vc, lens, layers, batch, nodes, slots, kv_heads, d, capacity, None)


@pytest.mark.parametrize("bad,why", [
    (dict(M=-1), "negative extent"), (dict(N=-1), "negative extent"), (dict(K=-32), "negative extent"), (dict(group=16), "groups are of"),
    (dict(group=0), "groups are of"), (dict(K=288, group=64), "multiple of the scale group"), (dict(epilogue=4), "unknown epilogue"),
    (dict(epilogue=-1), "unknown epilogue"), (dict(N=1 << 40, K=1 << 30), "overflow"), (dict(M=1 << 40, N=1 << 30), "overflow"),
    (dict(x=None), "NULL"), (dict(Wq=None), "NULL"), (dict(scale=None), "NULL"), (dict(y=None), "NULL"),
    (dict(res1=F, res2=G), "residuals"), (dict(epilogue=1, res1=F), "residuals"), (dict(epilogue=2), "residuals"),
    (dict(y=A + 8), "overlaps"), (dict(y=B + 8), "overlaps"), (dict(y=C), "overlaps"), (dict(y=D + 126), "overlaps"),
    (dict(epilogue=1, res1=E, res2=G), "overlaps"), (dict(epilogue=2, res1=G, res2=E + 700), "overlaps")])
def test_gemv_q4_refuses(bad, why):
    rc, message = q4(**bad)
    assert rc == -1 and "gemv_q4" in message and why in message


@pytest.mark.parametrize("bad,why", [
    (dict(batch=-1), "negative extent"), (dict(capacity=-1), "negative extent"), (dict(nodes=65, rows=65), "up to 64 nodes"),
    (dict(rows=10), "10 query rows of a tree of 9"), (dict(heads=7), "share 2 key heads"), (dict(kv_heads=0), "share 0 key heads"),
    (dict(d=257), "up to 256"), (dict(capacity=1 << 31), "overflow"), (dict(heads=65536), "overflow"),
    (dict(batch=1 << 31, capacity=1 << 30, kv_heads=8), "overflow"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(scale=-3e38), "finite"),
    *((dict([(name, None)]), "NULL") for name in ("Q", "K", "V", "Kc", "Vc", "lens", "parents", "out")),
    *((dict(out=at), "overlaps") for at in (A, B, C, D + 64, E, F, G))])
def test_attn_tree_refuses(bad, why):
    rc, message = tree(**bad)
    assert rc == -1 and "attn_tree" in message and why in message


@pytest.mark.parametrize("bad,why", [
    (dict(batch=-1), "negative extent"), (dict(nodes=65), "up to 64 nodes"), (dict(nodes=0), "no node"), (dict(V=0), "no node, or no token"),
    (dict(V=1 << 31), "overflow"), *((dict([(name, None)]), "NULL") for name in
                                     ("target", "draft", "tokens", "parents", "accept", "sample", "path", "count", "next_token")),
    *((dict(path=at), "output overlaps") for at in (A, B, C, D, E, F)), (dict(count=F + 4), "output overlaps"), (dict(next_token=C + 8), "output overlaps"),
    (dict(count=G + 4), "outputs overlap"), (dict(next_token=H), "outputs overlap")])
def test_verify_tree_refuses(bad, why):
    rc, message = verify(**bad)
    assert rc == -1 and "verify_tree" in message and why in message


@pytest.mark.parametrize("bad,why", [
    (dict(layers=-1), "negative extent"), (dict(slots=-1), "negative extent"), (dict(path=None), "go together"), (dict(count=None), "go together"),
    (dict(path=None, count=None, slots=8), "every row has its slot"), (dict(batch=1 << 31), "overflow"), (dict(layers=1 << 40, d=1 << 20), "overflow"),
    *((dict([(name, None)]), "NULL") for name in ("K", "V", "Kc", "Vc", "lens")), (dict(Kc=A + 64), "overlaps an input"),
    (dict(Vc=B), "overlaps an input"), (dict(Kc=C), "overlaps an input"), (dict(Vc=D), "overlaps an input"), (dict(Kc=G), "overlaps an input"),
    (dict(Vc=E + 64), "caches overlap")])
def test_cache_append_refuses(bad, why):
    rc, message = append(**bad)
    assert rc == -1 and "cache_append" in message and why in message


def test_empty_extents_do_nothing():
    assert q4(M=0) == q4(N=0) == (0, "")
    assert tree(batch=0) == tree(rows=0) == tree(nodes=0, rows=0) == tree(heads=0) == tree(d=0) == (0, "")
    assert verify(batch=0) == (0, "")
    for name in ("layers", "batch", "slots", "kv_heads", "d", "capacity"):
        assert append(**{name: 0}) == (0, "")
    assert append(path=None, count=None, nodes=0, slots=0) == (0, "")


def test_cpu_tensors_are_refused():
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)
    f = lambda *s: torch.zeros(*s)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for call_it in (lambda: ops.gemv_q4(h(2, 64), i(8, 8), h(8, 2), None, h(2, 8)),
                    lambda: ops.attn_tree(h(1, 2, 4, 64), h(1, 2, 4, 64), h(1, 2, 4, 64), h(1, 4, 9, 64), h(1, 4, 9, 64), i(1), i(1, 2), h(1, 2, 4, 64)),
                    lambda: ops.verify_tree(f(1, 2, 9), f(1, 2, 9), i(1, 2), i(1, 2), f(1, 2), f(1), i(1, 2), i(1), i(1)),
                    lambda: ops.cache_append(h(1, 2, 4, 64), h(1, 2, 4, 64), None, None, h(1, 4, 9, 64), h(1, 4, 9, 64), i(1))):
        with pytest.raises(ValueError, match="no CPU path"):
            call_it()


def test_the_limit_is_the_headers():
    import os
    import re
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dtas_abi.h")).read()
    assert int(re.search(r"#define DTAS_MAX_TREE_NODES (\d+)", header).group(1)) == _lib.MAX_TREE_NODES


@pytest.mark.parametrize("extents", [dict(batch=(1 << 31) - 1, nodes=64, V=(1 << 31) - 1), dict(batch=1 << 25, nodes=64, V=1 << 30), dict(batch=(1 << 31) - 1, nodes=1, V=(1 << 31) - 1)])
def test_verify_tree_refuses_rows_beyond_64_bits(extents):
    # each extent is within its own range, the distributions' bytes are not
    rc, message = verify(**extents)
    assert rc == -1 and "verify_tree: the extents overflow" in message


def test_empty_paths_and_batches_do_nothing():
    # (an empty tensor has no address)
    assert append(path=None, slots=0) == append(path=None, count=None, slots=0) == (0, "")
    assert append(batch=0, path=None, count=None, slots=4) == append(layers=0, K=None, V=None, Kc=None, Vc=None) == (0, "")
    assert append(path=None)[0] == append(count=None)[0] == append(path=None, count=None, slots=8)[0] == -1
