"""Attention over pages of many groups: whether they are read together does not go by which of them stand in front."""
import pytest
import torch

from dtas_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,beams", [(1024, 2), (1500, 4)])
def test_the_batchs_order_does_not_matter(B, beams):
    # short groups and long ones, half of the batch each and none of them cut into pieces: the same bits whether the short or the long ones stand in front
    heads, d, page, columns = 1, 64, 16, 110
    g = torch.Generator(device="cuda").manual_seed(B)
    pages = 4000
    K, V = (torch.randn(pages, heads, page, d, device="cuda", generator=g).half() for _ in range(2))
    table = torch.randint(0, pages, (B // beams, beams, columns), device="cuda", generator=g).int()
    table[:, :, :70] = table[:, :1, :70].clone()
    table = table.view(B, columns)
    lens = torch.full((B,), 9, device="cuda", dtype=torch.int32)
    half = B // beams // 2 * beams
    lens[half:] = 1700 + torch.arange(B - half, device="cuda").int() % 40
    Q = torch.randn(B, heads, d, device="cuda", generator=g).half() * 2
    outs = []
    for order in (torch.arange(B, device="cuda"), torch.arange(B, device="cuda").roll(half)):
        out = torch.empty_like(Q)
        ops.attn_paged(Q[order].contiguous(), K, V, table[order].contiguous(), lens[order].contiguous(), out, None, beams)
        outs.append(torch.empty_like(out).index_copy_(0, order, out))
    assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))
