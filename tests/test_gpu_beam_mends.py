"""Reordering where a page that should be there is not."""
import pytest
import torch

from test_gpu_beam import DEV, _follow, _states

gpu = pytest.mark.gpu


def _reorder(k, v, table, slots, parent, held):
    from bloomery_b200.ops.beam import beam_reorder
    on = [t.to(DEV) for t in (k, v, table, slots, parent, held)]
    new = torch.full_like(on[2], -7)
    fault = torch.full((1,), -1, dtype=torch.int32, device=DEV)
    beam_reorder(on[0], on[1], on[2], new, *on[3:], fault)
    return new.cpu(), on[0].cpu(), on[1].cpu(), int(fault)


@gpu
@pytest.mark.parametrize("missing", [-1, "past"])
@pytest.mark.parametrize("parents,gone,lost", [
    ([1, 0, 2, 3], 1, [0]),                # the page of a first child's parent
    ([1, 1, 2, 3], 1, [0, 1]),             # of a first child's and a further child's, which is the parent itself
    ([0, 0, 2, 3], 0, [1]),                # the parent goes on in its own place, whatever that is; a further child has nothing to copy
    ([0, 0, 2, 3], 1, [1]),                # the page that a further child takes over
    ([3, 1, 1, 3], 0, [2]),                # the same, further on
])
def test_a_child_without_a_page_keeps_its_row_and_raises_the_fault(parents, gone, lost, missing):
    """``gone``: the beam of the first search whose page being filled is missing; ``lost``: children that cannot move."""
    k, v, table, slots = _states(2, 4, 100, seed=11)
    parent = torch.tensor([parents, [1, 1, 3, 0]], dtype=torch.int32)
    held = torch.tensor([100, 100], dtype=torch.int32)
    table[slots[gone], 1] = -1 if missing == -1 else k.shape[1]
    new, k_new, v_new, fault = _reorder(k, v, table, slots, parent, held)
    assert fault == 6                                      # layer 0, no such page
    # the others' state is what it is without these children's copies
    sane = table.clone()
    sane[slots[gone], 1] = 0                               # page 0 stands for the missing one; nobody's copy of it is kept
    kept = (k.clone(), v.clone())
    want = _follow(*kept, sane, slots, parent, held)
    for i in range(8):
        s = int(slots[i])
        if i < 4 and i in lost:
            assert new[s].tolist() == table[s].tolist(), i
            continue
        row = want[s].clone()
        if i == gone and parents[i] == i:
            row[1] = table[s, 1]
        assert new[s].tolist() == row.tolist(), i
    spare = {int(want[slots[i], 1]) for i in lost} | {0}   # pages that only a lost child would have written
    for got, ref in ((k_new, kept[0]), (v_new, kept[1])):
        for page in range(got.shape[1]):
            if page not in spare:
                assert torch.equal(got[:, page], ref[:, page]), page
    for page in spare - {0}:
        assert torch.equal(k_new[:, page], k[:, page]) and torch.equal(v_new[:, page], v[:, page])


@gpu
def test_places_without_a_beam_need_no_page():
    k, v, table, slots = _states(1, 4, 100, seed=12)
    table[slots[2:], 1] = -1                               # nobody follows these two but themselves
    parent = torch.tensor([[1, 0, 2, 3]], dtype=torch.int32)
    held = torch.tensor([100], dtype=torch.int32)
    new, k_new, v_new, fault = _reorder(k, v, table, slots, parent, held)
    assert fault == -1 and torch.equal(k_new, k) and torch.equal(v_new, v)
    for i, p in enumerate([1, 0, 2, 3]):
        assert new[slots[i], :2].tolist() == table[slots[p], :2].tolist()
