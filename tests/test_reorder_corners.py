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
