"""Rows into their slots: more of them, and more layers, than a grid holds."""
import pytest
import torch

from dtas_amd import ops

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_grid_has_workgroups():
    # a workgroup per row of 129 elements (off 16 bytes), 2^24 and some of them: 4.3 GB
    rows, d, page = (1 << 24) + 5, 129, 4
    K = torch.zeros(rows, 1, d, device="cuda", dtype=torch.float16)
    slots = torch.full((rows,), -1, device="cuda", dtype=torch.int32)
    pool = [torch.full((2, 1, page, d), 9.0, device="cuda", dtype=torch.float16) for _ in range(2)]
    want = pool[0].clone()
    for slot, n in ((3, 0), (0, (1 << 23) - 1), (7, 1 << 23), (5, (1 << 24) - 1), (1, 1 << 24), (6, rows - 1)):
        K[n] = slot + torch.arange(d, device="cuda") / 256
        slots[n] = slot
        want[slot // page, 0, slot % page] = K[n, 0]
    ops.page_append(K, K, slots, *pool)
    assert torch.equal(pool[0], want) and torch.equal(pool[1], want)


def test_more_layers_and_rows_than_a_grid_has_workgroups():
    # five layers of 2^22 such rows: two to a launch
    layers, rows, d, page, pages = 5, 1 << 22, 129, 2, 3
    K = torch.zeros(layers, rows, 1, d, device="cuda", dtype=torch.float16)
    slots = torch.full((rows,), -1, device="cuda", dtype=torch.int32)
    pool = [torch.full((layers, pages, 1, page, d), 9.0, device="cuda", dtype=torch.float16) for _ in range(2)]
    want = pool[0].clone()
    for slot, n in ((4, 0), (1, rows // 2), (2, rows - 1)):
        slots[n] = slot
        for l in range(layers):
            K[l, n] = 10 * l + slot + torch.arange(d, device="cuda") / 128
            want[l, slot // page, 0, slot % page] = K[l, n, 0]
    ops.page_append(K, K, slots, *pool)
    assert torch.equal(pool[0], want) and torch.equal(pool[1], want)


@pytest.mark.parametrize("d", [8, 5])
def test_a_great_many_layers(d):
    layers, rows, heads, page, pages = 65535 * 2 + 7, 3, 2, 2, 2
    g = torch.Generator(device="cuda").manual_seed(d)
    K, V = (torch.randn(layers, rows, heads, d, device="cuda", generator=g).half() for _ in range(2))
    pools = [torch.randn(layers, pages, heads, page, d, device="cuda", generator=g).half() for _ in range(2)]
    want = [p.clone() for p in pools]
    for n, slot in ((0, 2), (2, 1)):
        for new, cache in ((K, want[0]), (V, want[1])):
            cache[:, slot // page, :, slot % page] = new[:, n]
    ops.page_append(K, V, torch.tensor([2, -1, 1], device="cuda", dtype=torch.int32), *pools)
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])
