"""Attention of a tree: keys and values that are no numbers, weights and scales at the ends of their range, in every kernel."""
import math

import pytest
import torch

from dtas_amd import ops
from test_parity_tree import expected, launch, make

pytestmark = pytest.mark.gpu

# (nodes, key heads, query heads to each, d, capacity, elements off an aligned address): a wavefront's rows share the keys (16 rows, 32 rows, heads of 256), the
# rows share the keys by 64, 128 and 256 (heads of 256 among them), element by element (an odd address, an odd head)
FORMS = [(1, 2, 1, 64, 2300, 0), (4, 2, 2, 80, 2300, 0), (16, 3, 1, 128, 300, 0), (16, 1, 2, 64, 300, 0), (8, 2, 4, 128, 300, 0), (4, 1, 2, 256, 2300, 0), (9, 1, 3, 256, 300, 0),
         (13, 2, 4, 96, 2300, 0), (64, 32, 4, 64, 2000, 0), (64, 32, 4, 64, 4200, 0), (64, 32, 4, 128, 9100, 0), (64, 4, 4, 256, 8000, 0), (40, 1, 1, 192, 2300, 0),
         (4, 2, 2, 64, 300, 1), (3, 2, 2, 20, 300, 0)]


def first_head(host, group):
    """The inputs of the first key head and its rows alone."""
    cut = {"Q": lambda t: t[:, :, :group], "K": lambda t: t[:, :, :1], "V": lambda t: t[:, :, :1], "Kc": lambda t: t[:, :1], "Vc": lambda t: t[:, :1]}
    return {name: cut.get(name, lambda t: t)(t) for name, t in host.items()}


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("T,Hkv,group,d,capacity,offset,length",
                         [(*form, length) for form in FORMS for length in ((1, 31, 32, 33, 63, 64, 65, 97, 259) if form[1] < 32 else (31, 64, 97))])
def test_the_last_value_of_the_cache_is_no_number(T, Hkv, group, d, capacity, offset, length, value):
    # it reaches the channel it stands in, of the rows of its key head, wherever the cache's last block ends
    host = make(1, T, T, Hkv, group, d, [length], capacity)
    host["Vc"][0, 0, length - 1, 3] = 0
    want, tolerance = expected(first_head(host, group))
    host["Vc"][0, 0, length - 1, 3] = value
    got = launch(host, offset=offset).double()
    assert bool(torch.isfinite(got[:, :, group:]).all())
    mine = got[:, :, :group]
    assert bool((torch.isnan(mine[..., 3]) if math.isnan(value) else mine[..., 3] == value).all())
    others = [c for c in range(d) if c != 3]
    assert bool(((mine - want).abs() <= tolerance)[..., others].all())


@pytest.mark.parametrize("gap", [9.0, 13.875, 15.0, 16.5])
@pytest.mark.parametrize("T,Hkv,group,d", [(1, 32, 4, 64), (4, 32, 4, 128), (2, 32, 4, 256), (7, 32, 8, 64), (32, 32, 4, 64), (64, 32, 4, 64), (64, 32, 4, 128), (20, 32, 4, 256), (8, 32, 4, 80)])
def test_a_long_flat_tail_behind_few_large_weights(T, Hkv, group, d, gap):
    """Eight keys of no value whose scores lead those of all others by `gap`: what is left are the others' values, weighted by exp(-gap) each.

    The others' weights are one number, off by half a step of fp16 (2^-11) and a rounding of its exponent (gap log2(e) 2^-23, exp2 of which is within 2^-22 besides),
    and the products with values that are powers of two and their sums are exact (11 bits, less than 2^13 of them).  The sum of the weights has n additions in
    fp32 at most, 2^-24 each, and as many again over wavefronts and parts.  Storing: 2^-11 of values above 2^-14."""
    B, n = 10, 3999  # (more sequences than parts: each in one piece)
    Q = torch.zeros(B, T, Hkv * group, d, device="cuda", dtype=torch.float16)
    K, V = (torch.zeros(B, T, Hkv, d, device="cuda", dtype=torch.float16) for _ in range(2))
    Kc, Vc = (torch.zeros(B, Hkv, n, d, device="cuda", dtype=torch.float16) for _ in range(2))
    Q[..., 0] = 1
    Kc[:, :, 0:256:32, 0] = gap
    power = torch.exp2(torch.arange(d, device="cuda") % 3 + 6).half()
    Vc[:], V[:] = power, power
    Vc[:, :, 0:256:32] = 0
    parents = torch.arange(-1, T - 1, device="cuda", dtype=torch.int32).expand(B, T).contiguous()
    lens = torch.full((B,), n, device="cuda", dtype=torch.int32)
    out = torch.empty_like(Q)
    ops.attn_tree(Q, K, V, Kc, Vc, lens, parents, out, 1.0)
    tail = (n - 8 + 1 + torch.arange(T, device="cuda").double()) * math.exp(-gap)  # (a node sees the nodes before it and itself)
    want = (tail / (tail + 8))[None, :, None, None] * power.double()
    assert float(want.min()) > 2.0 ** -14
    tolerance = 2.0 ** -11 + gap * 1.45 * 2.0 ** -23 + 2.0 ** -22 + 2 * (n + T) * 2.0 ** -24 + 2.0 ** -11
    assert float(((out.double() - want).abs() / want).max()) <= tolerance


@pytest.mark.parametrize("at", [0, 5, 255, 258, "node"])
@pytest.mark.parametrize("T,Hkv,group,d,capacity,offset", FORMS)
def test_a_key_that_is_no_number_wherever_it_stands(T, Hkv, group, d, capacity, offset, at):
    # also where everything in front of it has the score -inf, or nothing is in front of it: the rows that see it have no answer
    length = 0 if at == "node" else 259
    host = make(1, T, T, Hkv, group, d, [length], capacity, "chain")
    host["Q"][..., 0] = 1
    if at == "node":
        host["K"][0, 0, 0, 0] = float("nan")
    else:
        host["Kc"][0, 0, :at, 0] = float("-inf")
        host["Kc"][0, 0, at, 0] = float("nan")
    got = launch(host, offset=offset)
    assert bool(torch.isnan(got[:, :, :group]).all())
    assert bool(torch.isfinite(got[:, :, group:]).all())


@pytest.mark.parametrize("T,Hkv,group,d,capacity,offset", FORMS)
def test_scores_of_minus_infinity_have_no_weight(T, Hkv, group, d, capacity, offset):
    host = make(1, T, T, Hkv, group, d, [259], capacity, "chain")
    host["Q"][..., 0] = 1
    host["Kc"][0, 0, :, 0] = float("-inf")  # (the cache of the first key head: its rows see the nodes alone)
    one = first_head(host, group)
    want, tolerance = expected(dict(one, lens=torch.zeros(1, dtype=torch.int32)))
    got = launch(host, offset=offset).double()
    assert bool(((got[:, :, :group] - want).abs() <= tolerance).all())
    assert bool(torch.isfinite(got[:, :, group:]).all())


@pytest.mark.parametrize("scale", [2e26, 2.5e26, 1e38, -1e38, 2e38])
@pytest.mark.parametrize("T,Hkv,group,d,capacity,offset", FORMS)
def test_scales_up_to_the_largest(T, Hkv, group, d, capacity, offset, scale):
    # products that are whole numbers: the keys with the row's largest (smallest, by a negative scale) share it, whatever the largest is
    host = make(1, T, T, Hkv, group, d, [259], capacity, "chain")
    g = torch.Generator().manual_seed(d)
    for name in ("Q", "K", "Kc"):
        host[name] = torch.randint(-3, 4, host[name].shape, generator=g).half()
    host["Q"][..., 0], host["Kc"][..., 0], host["K"][..., 0] = 64, 64, 64  # (no product is near nought)
    one = first_head(host, group)
    want, _ = expected(one, scale)
    got = launch(host, scale, offset).double()
    # n equal weights of one key each: fp32 sums of up to 259 + 64 values (2^-24 each), a quotient and half a step
    tolerance = 2.0 ** -10 * one["V"].double().abs().amax().clamp(min=float(one["Vc"].abs().max()))
    assert bool(((got[:, :, :group] - want).abs() <= tolerance).all()), (got[0, 0, 0, :4], want[0, 0, 0, :4])


@pytest.mark.parametrize("gap", [10.0, 20.0, 30.0, 60.0])
@pytest.mark.parametrize("at", [0, 40, 255, 258])
@pytest.mark.parametrize("T,Hkv,group,d,capacity,offset", FORMS)
def test_an_infinite_value_of_little_weight(T, Hkv, group, d, capacity, offset, at, gap):
    # exp(-60) is a number in fp32 still: the channel is infinite, every other one as it would be
    length = 259
    host = make(1, T, T, Hkv, group, d, [length], capacity)
    for name in ("Q", "K", "Kc"):
        host[name][:] = 0
    host["Q"][..., 0], host["Kc"][0, :, at, 0] = 1, -gap
    host["Vc"][0, 0, at, 3] = 0
    one = first_head(host, group)
    want, tolerance = expected(one, 1.0)
    host["Vc"][0, 0, at, 3] = float("inf")
    got = launch(host, 1.0, offset).double()
    mine, others = got[:, :, :group], [c for c in range(d) if c != 3]
    assert bool((mine[..., 3] == float("inf")).all())
    assert bool(((mine - want).abs() <= tolerance)[..., others].all())
    assert bool(torch.isfinite(got[:, :, group:]).all())
