"""Attention over pages: its weights have the bits of fp32, in every kernel alike."""
import pytest
import torch

from test_paged_extremes import FORMS, few
from test_parity_paged import launch, make, seen

pytestmark = pytest.mark.gpu

LIVE = 64


@pytest.mark.parametrize("B,Hkv,group,d,page,beams,offset,length", [(*f, n) for f in FORMS for n in (31, 97, 2049) if few(f, n)])
@pytest.mark.parametrize("below", [0.875, 1.25, 2.75, 3.25])
def test_weights_that_cancel(B, Hkv, group, d, page, beams, offset, length, below):
    """Of the first 64 keys one in sixteen leads the others by `below`; its values are theirs the other way round, times the sum of their weights in fp16, so that 2^-12 of the sums is
    left.  All keys behind are 60000 below: weights of nought.  exp(-below) lies between two numbers of 11 bits, up to 2^-11.3 of itself from the nearer one, and all such
    weights on one side.

    Scores are exact (one product each).  A weight: its exponent, below log2(e) < 5 from 11, is rounded to 2^-21 at most and has 2^-22 of log2(e)'s rounding, 2^-21 of the weight
    both; exp2 2^-22; two halves of 11 bits each 2^-22: 2^-20 together.  Sums of n keys in any order, joined over wavefronts and parts (16 roundings), n 2^-24 + 2^-20 each, on
    the weighted sum of |v| and, of the quotient, on |out|; 2^-36 of the largest weight for each key where fp16 has no more bits.  Storing: 2^-11, 2^-25 at least."""
    host = make(B, Hkv, group, d, page, [length] * B, beams=beams)
    n = min(length, LIVE)
    host["Q"][:] = 0
    host["Q"][..., 0] = 1
    host["K"][:] = 0
    host["K"][..., 0] = -60000
    weight = torch.exp(torch.tensor(-below, dtype=torch.float64))
    lead = torch.arange(n) % 16 == 0
    rest = (weight * int((~lead).sum()) / int(lead.sum())).half()
    power = torch.exp2(torch.arange(d) % 5 - 2.0).half()
    for b in range(B):
        for j, (p, row) in enumerate(seen(host, b)[:n]):
            host["K"][p, :, row, 0] = 0 if lead[j] else -below
            host["V"][p, :, row] = -rest * power if lead[j] else power
    got = launch(host, 1.0, offset, beams).double()
    p = torch.where(lead, 1.0, weight)
    p = p / p.sum()
    out = (p * torch.where(lead, -rest.double(), 1.0)).sum() * power.double()
    size = (p * torch.where(lead, rest.double(), 1.0)).sum() * power.double()
    assert float((out.abs() / size).max()) < 2.0 ** -11
    off = 2.0 ** -20 * size + (n * 2.0 ** -24 + 2.0 ** -20) * (size + out.abs()) + 2.0 ** -36 * n * rest.double().clamp(min=1.0) * power.double()
    assert bool(((got - out).abs() <= off + 2.0 ** -11 * (out.abs() + off) + 2.0 ** -25).all()), float(((got - out).abs() / size).max())
