"""Products with 4-bit weights: scales that are no numbers."""
import pytest
import torch

from dtas_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("K,group", [(32, 32), (160, 32), (224, 32), (64, 64), (192, 64), (2624, 32), (384, 128)])
@pytest.mark.parametrize("M,N", [(1, 40), (4, 5000), (7, 40), (16, 8500), (33, 70), (64, 8500)])
def test_a_last_scale_that_is_no_number(M, N, K, group, value):
    # the last scale of a row is its last group's alone: x and the weights positive, that column is what the scale is and every other one as ever
    g = torch.Generator().manual_seed(M + K)
    x = torch.randint(1, 4, (M, K), generator=g).half()
    nibbles = torch.randint(8, 16, (N, K), generator=g)
    words = (nibbles.view(N, K // 8, 8) << (4 * torch.arange(8))).sum(-1)
    words = (words - (words >> 31 << 32)).to(torch.int32)
    scale = torch.full((N, K // group), 1 / 64).half()
    columns = [0, N // 2, N - 1]
    scale[columns, -1] = value
    y = torch.empty(M, N, device="cuda", dtype=torch.float16)
    ops.gemv_q4(x.cuda(), words.cuda(), scale.cuda(), None, y)
    y = y.cpu()
    mine = y[:, columns]
    assert bool((torch.isnan(mine) if value != value else mine == value).all())
    others = torch.ones(N, dtype=torch.bool)
    others[columns] = False
    assert torch.equal(y[:, others], ((x.double() @ (nibbles - 7).double().T) / 64)[:, others].half())  # (whole numbers of 1 / 64: exact before the rounding)
