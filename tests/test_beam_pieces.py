"""The choice of beams over rows that a workgroup goes through in several pieces of 8192 logits: what is no number counts wherever it stands."""
import math

import pytest
import torch

from test_parity_paged import check_beams, some_logits

pytestmark = pytest.mark.gpu

PIECE = 8192


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("G,W,V", [(64, 8, 8300), (16, 32, 20001), (32, 8, 33000)])  # (the last: two parts of 16500)
def test_what_is_no_number_in_any_piece(G, W, V, bad):
    logits, scores, g = some_logits(G, W, V, W + V)
    parts = 512 // (G * W)
    per = V // parts
    starts = [(p * per, i) for p in range(parts) for i in range(0, per, PIECE)]
    for n in range(G - 1):  # (the last request has numbers alone)
        start, i = starts[n % len(starts)]
        n_here = min(PIECE, per - i)
        at = start + i + int(torch.randint(0, n_here, (1,), generator=g))
        how = n // len(starts) % 3
        if how != 0:  # among -inf: the piece alone, or the whole part up to its end
            logits[n, :, (start if how == 2 else start + i):start + i + n_here] = -math.inf
        some = slice(0, W if n % 5 == 4 else 1)
        scores[n, 0] = 0.0  # (the beam without a sum would lead the others)
        logits[n, some, at] = bad
    check_beams(logits, scores)
    check_beams(logits, scores, (torch.rand(G, W, generator=g) < 0.3).int(), eos=V // 3)
