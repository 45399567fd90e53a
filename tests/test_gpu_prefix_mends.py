"""Shared-prefix attention where it once read, rounded or reported what it should not have."""
import pytest
import torch

from test_gpu_prefix_attention import DEV, Case

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("rows", [5, 40])                  # schedules of one warp's registers and of the whole block
@pytest.mark.parametrize("q8", [False, True])
def test_a_prefix_longer_than_a_table_row_ends_with_the_row(rows, q8):
    """Lengths that a captured call finds on the card: every key of these rows is in their table, and nothing behind it is read."""
    c = Case([(192, [1 + i * 191 // (rows - 1) for i in range(rows)])], 32, 4, 128, q8, seed=21, max_pages=3)
    c.table = c.table.contiguous()
    plan = c.plan()
    first = c.run(plan)
    c.check(first)
    out = torch.zeros_like(first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            c.run(plan, out)
    with pytest.raises(ValueError):
        plan.set_prefix([640])
    plan.max_pages = None                                  # past the host's check, as another holder of the lengths could
    for longer in (640, 1 << 28):
        plan.set_prefix([longer])
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    assert int(c.fault) == -1
