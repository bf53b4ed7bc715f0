"""What the operators of requests in pages refuse, and what they do nothing for: decided before any launch."""
import os
import re

import pytest
import torch

from dtas_amd import _lib, ops

A, B, C, D, E, F, G, H, I, J = (0x10000000 * (i + 1) for i in range(10))  # never dereferenced: every call ends before a launch


def call(name, *args):
    return getattr(_lib.lib(), name)(*args), _lib.last_error()


def assign(lens=A, count=B, table=C, free=D, free_count=E, starts=None, slots=F, new_lens=G, left=H, batch=3, rows=5, columns=7, page=16, pages=40):
    return call("dtas_page_assign_i32", lens, count, table, free, free_count, starts, slots, new_lens, left, batch, rows, columns, page, pages, None)


def append(K=A, V=B, slots=C, Kp=D, Vp=E, layers=2, rows=9, kv_heads=2, d=64, page=16, pages=10):
    return call("dtas_page_append_f16", K, V, slots, Kp, Vp, layers, rows, kv_heads, d, page, pages, None)


def paged(Q=A, Kp=B, Vp=C, table=D, lens=E, out=F, batch=6, heads=8, kv_heads=2, d=64, page=16, pages=10, columns=4, beams=1, scale=0.125):
    return call("dtas_attn_paged_f16", Q, Kp, Vp, table, lens, out, batch, heads, kv_heads, d, page, pages, columns, beams, scale, None)


def beam(logits=A, scores=B, done=C, tokens=D, parents=E, new_scores=F, new_done=G, groups=2, beams=4, V=100, eos=0):
    return call("dtas_beam_select_f32", logits, scores, done, tokens, parents, new_scores, new_done, groups, beams, V, eos, None)


def reorder(parents=A, table=B, lens=C, free=D, free_count=E, new_table=F, new_lens=G, left=H, Kp=I, Vp=J, layers=2, groups=2, beams=4, columns=5, kv_heads=2, d=64,
            page=16, pages=40):
    return call("dtas_page_reorder_f16", parents, table, lens, free, free_count, new_table, new_lens, left, Kp, Vp, layers, groups, beams, columns, kv_heads, d, page,
                pages, None)


@pytest.mark.parametrize("bad,why", [
    (dict(batch=-1), "negative extent"), (dict(rows=-1), "negative extent"), (dict(columns=-1), "negative extent"), (dict(pages=-1), "negative extent"),
    (dict(page=0), "at least one position"), (dict(page=-16), "at least one position"), (dict(batch=1 << 31), "overflow"), (dict(rows=1 << 31), "overflow"),
    (dict(batch=1 << 16, rows=1 << 15), "overflow"), (dict(page=1 << 16, pages=1 << 15), "overflow"), (dict(columns=1 << 31), "overflow"),
    *((dict([(name, None)]), "NULL") for name in ("lens", "count", "table", "free", "free_count", "slots", "new_lens", "left")),
    (dict(table=A), "output overlaps"), (dict(slots=B + 8), "output overlaps"), (dict(new_lens=A + 4), "output overlaps"), (dict(new_lens=B), "output overlaps"),
    (dict(left=E + 2), "output overlaps"), (dict(left=D), "output overlaps"), (dict(starts=E), "output overlaps"), (dict(slots=C + 80), "outputs overlap"),
    (dict(starts=F, rows=2), "outputs overlap"), (dict(left=G + 8), "outputs overlap"), (dict(new_lens=F), "outputs overlap")])
def test_page_assign_refuses(bad, why):
    rc, message = assign(**bad)
    assert rc == -1 and "page_assign" in message and why in message


@pytest.mark.parametrize("bad,why", [
    (dict(layers=-1), "negative extent"), (dict(rows=-1), "negative extent"), (dict(page=-1), "negative extent"), (dict(rows=1 << 31), "overflow"),
    (dict(page=1 << 16, pages=1 << 15), "overflow"), (dict(layers=1 << 40, d=1 << 20), "overflow"), (dict(kv_heads=1 << 20, d=1 << 12), "overflow"),
    *((dict([(name, None)]), "NULL") for name in ("K", "V", "slots", "Kp", "Vp")),
    (dict(Kp=A + 64), "output overlaps"), (dict(Vp=B), "output overlaps"), (dict(Kp=C), "output overlaps"), (dict(Vp=D + 128), "outputs overlap")])
def test_page_append_refuses(bad, why):
    rc, message = append(**bad)
    assert rc == -1 and "page_append" in message and why in message


@pytest.mark.parametrize("bad,why", [
    (dict(batch=-1), "negative extent"), (dict(columns=-1), "negative extent"), (dict(page=0), "at least one position"), (dict(beams=0), "groups of 0"),
    (dict(beams=-1), "groups of -1"), (dict(beams=4), "groups of 4"), (dict(heads=7), "share 2 key heads"), (dict(kv_heads=0), "share 0 key heads"), (dict(d=257), "up to 256"),
    (dict(heads=65536), "overflow"), (dict(batch=3 << 30), "overflow"), (dict(page=1 << 16, pages=1 << 15), "overflow"), (dict(columns=1 << 31), "overflow"),
    (dict(page=1 << 31, pages=0), "overflow"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(scale=-3e38), "finite"),
    *((dict([(name, None)]), "NULL") for name in ("Q", "Kp", "Vp", "table", "lens", "out")),
    *((dict(out=at), "overlaps") for at in (A, B + 64, C, D + 4, E))])
def test_attn_paged_refuses(bad, why):
    rc, message = paged(**bad)
    assert rc == -1 and "attn_paged" in message and why in message


@pytest.mark.parametrize("bad,why", [
    (dict(groups=-1), "negative extent"), (dict(beams=33), "up to 32 beams"), (dict(V=0), "no token"), (dict(V=(1 << 30) + 1), "overflow"), (dict(groups=1 << 31), "overflow"),
    (dict(done=None), "go together"), (dict(new_done=None), "go together"),
    *((dict([(name, None)]), "NULL") for name in ("logits", "scores", "tokens", "parents", "new_scores")),
    (dict(tokens=A), "output overlaps"), (dict(new_scores=B + 4), "output overlaps"), (dict(new_done=C + 4), "output overlaps"), (dict(new_scores=C), "output overlaps"),
    (dict(new_done=B), "output overlaps"), (dict(parents=D + 4), "outputs overlap"), (dict(new_scores=E), "outputs overlap"), (dict(new_done=F), "outputs overlap")])
def test_beam_select_refuses(bad, why):
    rc, message = beam(**bad)
    assert rc == -1 and "beam_select" in message and why in message


@pytest.mark.parametrize("bad,why", [
    (dict(layers=-1), "negative extent"), (dict(columns=-1), "negative extent"), (dict(page=0), "at least one position"), (dict(beams=33), "up to 32 beams"),
    (dict(groups=1 << 30), "overflow"), (dict(page=1 << 16, pages=1 << 15), "overflow"), (dict(layers=1 << 40, d=1 << 14), "overflow"), (dict(columns=1 << 31), "overflow"),
    (dict(columns=1 << 28), "too large"),
    *((dict([(name, None)]), "NULL") for name in ("parents", "table", "lens", "free", "free_count", "new_table", "new_lens", "left", "Kp", "Vp")),
    (dict(new_table=B + 4), "output overlaps"), (dict(new_lens=A), "output overlaps"), (dict(new_lens=C + 4), "output overlaps"), (dict(left=E + 2), "output overlaps"),
    (dict(free=B), "output overlaps"), (dict(Kp=C), "output overlaps"), (dict(new_table=D), "outputs overlap"), (dict(left=G), "outputs overlap"),
    (dict(Vp=I + 64), "outputs overlap"), (dict(new_lens=F + 4), "outputs overlap")])
def test_page_reorder_refuses(bad, why):
    rc, message = reorder(**bad)
    assert rc == -1 and "page_reorder" in message and why in message


@pytest.mark.parametrize("nothing", [lambda: append(rows=0, K=None), lambda: append(pages=0, Kp=None), lambda: append(layers=0), lambda: append(d=0), lambda: paged(batch=0, Q=None),
                                     lambda: paged(heads=0), lambda: paged(d=0), lambda: beam(groups=0, logits=None), lambda: beam(beams=0),
                                     lambda: reorder(groups=0, left=E), lambda: reorder(beams=0, left=E)])
def test_nothing_to_do(nothing):
    assert nothing()[0] == 0


def test_tables_of_too_many_positions():
    # 2^26 blocks of 32 keys to a table: sixteen of them, or of the sequences of groups, are as many as a launch counts
    for many in (dict(batch=17), dict(batch=32, beams=32), dict(batch=34, beams=2)):
        rc, message = paged(columns=1 << 27, table=1 << 44, **many)
        assert rc == -1 and "too many positions" in message, message


def test_no_kernel_keeps_registers_in_memory():
    # what the built library says of its kernels: bytes of scratch memory per lane
    with open(os.path.join(os.path.dirname(_lib.__file__), "libdtas_gfx950.so"), "rb") as f:
        found = re.findall(rb"(_ZN4dtas\w*(?:attn_paged|beam_select|page_)\w+)\xbb\.private_segment_fixed_size(.)", f.read(), re.S)
    assert len(found) >= 20 and all(size == b"\0" for _, size in found), found


def test_tensors_on_the_host_are_refused():
    i, h, f = (lambda *s: torch.zeros(*s, dtype=torch.int32)), (lambda *s: torch.zeros(*s, dtype=torch.float16)), (lambda *s: torch.zeros(*s))
    for bad in (lambda: ops.page_assign(i(2), i(2), i(2, 3), i(9), i(1), 16, i(2, 1), i(2), i(1)), lambda: ops.page_append(h(2, 1, 8), h(2, 1, 8), i(2), h(3, 1, 16, 8), h(3, 1, 16, 8)),
                lambda: ops.attn_paged(h(2, 1, 8), h(3, 1, 16, 8), h(3, 1, 16, 8), i(2, 3), i(2), h(2, 1, 8)),
                lambda: ops.beam_select(f(1, 2, 9), f(1, 2), None, i(1, 2), i(1, 2), f(1, 2), None),
                lambda: ops.page_reorder(i(1, 2), i(1, 2, 3), i(1, 2), i(3), i(1), i(1, 2, 3), i(1, 2), i(1), h(3, 1, 16, 8), h(3, 1, 16, 8))):
        with pytest.raises(ValueError, match="no CPU path"):
            bad()


@pytest.mark.gpu
def test_tensors_that_do_not_fit_are_refused():
    z = lambda dtype: lambda *s: torch.zeros(*s, dtype=dtype, device="cuda")
    i, h, f = z(torch.int32), z(torch.float16), z(torch.float32)
    pool = lambda: h(3, 1, 16, 8)
    for match, bad in (
            ("int32", lambda: ops.page_assign(i(2).long(), i(2), i(2, 3), i(9), i(1), 16, i(2, 1), i(2), i(1))),
            ("shape", lambda: ops.page_assign(i(2), i(3), i(2, 3), i(9), i(1), 16, i(2, 1), i(2), i(1))),
            ("shape", lambda: ops.page_assign(i(2), i(2), i(2, 3), i(9), i(2), 16, i(2, 1), i(2), i(1))),
            ("shape", lambda: ops.page_assign(i(2), i(2), i(2, 3), i(9), i(1), 16, i(6), i(2), i(1), starts=i(2))),
            ("expects", lambda: ops.page_assign(i(2), i(2), i(2, 3), i(9), i(1), 16, i(6), i(2), i(1))),
            ("expects", lambda: ops.page_assign(i(2), i(2), i(2, 3), i(9), i(1), 16, i(2, 3), i(2), i(1), starts=i(3))),
            ("compact", lambda: ops.page_assign(i(2), i(2), i(3, 2).t(), i(9), i(1), 16, i(2, 3), i(2), i(1))),
            ("fp16", lambda: ops.page_append(f(2, 1, 8), h(2, 1, 8), i(2), pool(), pool())), ("int32", lambda: ops.page_append(h(2, 1, 8), h(2, 1, 8), i(2).long(), pool(), pool())),
            ("shape", lambda: ops.page_append(h(2, 1, 8), h(2, 1, 8), i(3), pool(), pool())), ("shape", lambda: ops.page_append(h(2, 2, 8), h(2, 2, 8), i(2), pool(), pool())),
            ("expects", lambda: ops.page_append(h(2, 2, 1, 8), h(2, 2, 1, 8), i(2), pool(), pool())),
            ("fp16", lambda: ops.attn_paged(h(2, 1, 8), pool(), pool(), i(2, 3), i(2), f(2, 1, 8))), ("int32", lambda: ops.attn_paged(h(2, 1, 8), pool(), pool(), f(2, 3), i(2), h(2, 1, 8))),
            ("expects", lambda: ops.attn_paged(h(2, 8), pool(), pool(), i(2, 3), i(2), h(2, 8))), ("shape", lambda: ops.attn_paged(h(2, 1, 8), pool(), pool(), i(3, 3), i(2), h(2, 1, 8))),
            ("shape", lambda: ops.attn_paged(h(2, 1, 8), pool(), h(3, 1, 8, 8), i(2, 3), i(2), h(2, 1, 8))),
            ("fp32", lambda: ops.beam_select(h(1, 2, 9), f(1, 2), None, i(1, 2), i(1, 2), f(1, 2), None)), ("shape", lambda: ops.beam_select(f(1, 2, 9), f(2), None, i(1, 2), i(1, 2), f(1, 2), None)),
            ("expects", lambda: ops.beam_select(f(2, 9), f(1, 2), None, i(1, 2), i(1, 2), f(1, 2), None)), ("int32", lambda: ops.beam_select(f(1, 2, 9), f(1, 2), f(1, 2), i(1, 2), i(1, 2), f(1, 2), i(1, 2))),
            ("shape", lambda: ops.page_reorder(i(1, 2), i(1, 2, 3), i(1, 2), i(4), i(1), i(1, 2, 3), i(1, 2), i(1), pool(), pool())),
            ("fp16", lambda: ops.page_reorder(i(1, 2), i(1, 2, 3), i(1, 2), i(3), i(1), i(1, 2, 3), i(1, 2), i(1), f(3, 1, 16, 8), pool())),
            ("expects", lambda: ops.page_reorder(i(1, 2), i(2, 3), i(1, 2), i(3), i(1), i(2, 3), i(1, 2), i(1), pool(), pool()))):
        with pytest.raises(ValueError, match=match):
            bad()
    with pytest.raises(_lib.DtasError, match="groups of 3"):
        ops.attn_paged(h(2, 1, 8), pool(), pool(), i(2, 3), i(2), h(2, 1, 8), beams=3)
