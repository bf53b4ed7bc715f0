"""Tables of beams where there are hardly any, or a great many."""
import pytest
import torch

from dtas_amd import ops
from test_zzz_capture import new_stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("G,W", [(0, 4), (0, 1), (3, 0)])
def test_without_rows_the_height_is_handed_on_without_a_workspace(G, W):
    # tables of so many columns that a workgroup would have sixteen wavefronts, each with its list; on a stream that has done something, but has no workspace yet
    i = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)
    pool, left = torch.zeros(5, 1, 16, 8, device="cuda", dtype=torch.float16), i(3)
    call = lambda height: ops.page_reorder(i(G, W), i(G, W, 2100), i(G, W), i(5), i(1) + height, i(G, W, 2100), i(G, W), left[1:2], pool, pool.clone())
    call(0)
    stream = new_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(2):
            left.zero_()
            (pool.clone(), i(5) + 1)
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved()
        for height, want in ((4, 4), (0, 0), (-3, 0), (99, 5)):
            call(height)
            assert left.tolist() == [0, want, 0]
        assert torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved() == before


def test_more_groups_than_a_launch_has_room_for_at_512_threads():
    # 2^23 and some groups of two beams, a page of two positions each: kept as they are or swapped, both handed one page or a copy of it, let go
    G, W, page, d = (1 << 23) + 9, 2, 2, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    pages = G * W + 7
    table = torch.randperm(pages, device="cuda", generator=g)[:G * W].int().view(G, W, 1)
    left_over = torch.ones(pages, dtype=torch.bool, device="cuda")
    left_over[table.flatten().long()] = False
    free = torch.full((pages,), -5, device="cuda", dtype=torch.int32)
    free[:7] = left_over.nonzero()[:, 0].int()
    lens = torch.randint(1, 3, (G, 1), device="cuda", generator=g).int().expand(G, W).contiguous()
    kind = torch.randint(0, 4, (G,), device="cuda", generator=g)
    parents = torch.tensor([[0, 1], [1, 0], [0, 0], [-1, -1]], device="cuda", dtype=torch.int32)[kind]
    K = torch.arange(pages, device="cuda")[:, None, None, None].remainder(1021).half().expand(pages, 1, page, d).contiguous()
    K[:, :, 1] += 0.25
    V = -K
    height = torch.tensor([7], device="cuda", dtype=torch.int32)

    want_table, want_lens, want_free, want_K = table[:, :, 0].clone(), torch.where(kind[:, None] == 3, 0, lens), free.clone(), K.clone()
    want_table[kind == 1] = table[kind == 1][:, [1, 0], 0]
    want_table[kind == 2] = table[kind == 2][:, [0, 0], 0]
    goes = torch.stack((kind == 3, kind >= 2), 1)
    back = table[:, :, 0][goes]
    want_free[7:7 + len(back)] = back
    top = 7 + len(back)
    copied = ((kind == 2) & (lens[:, 0] == 1)).nonzero()[:, 0]
    fresh = want_free[top - 1 - torch.arange(len(copied), device="cuda")]
    want_table[copied, 1] = fresh
    want_K[fresh.long(), :, 0] = K[table[copied, 0, 0].long(), :, 0]
    want_V = V.clone()
    want_V[fresh.long(), :, 0] = V[table[copied, 0, 0].long(), :, 0]
    assert len(copied) > 1 << 19

    new_table, new_lens, left = torch.full_like(table, -9), torch.full_like(lens, -9), torch.zeros_like(height)
    ops.page_reorder(parents, table, lens, free, height, new_table, new_lens, left, K, V)
    torch.cuda.synchronize()
    assert left.item() == top - len(copied) and torch.equal(new_lens, want_lens)
    some = kind < 3
    assert torch.equal(new_table[some][:, :, 0], want_table[some]) and torch.equal(free, want_free)
    assert torch.equal(K, want_K) and torch.equal(V, want_V)
