"""Slots outside a SlotHistory (the -1 of a padded batch, numbers beyond its last slot) are left alone: nobody
else's tokens change, and their own history is empty.  On CPU tensors."""

import numpy as np
import torch

from leat_b200.history import SlotHistory


def _filled(slots=5, capacity=4, vocab=50):
    h = SlotHistory(slots, capacity, vocab, special_ids=[9])
    for step in range(6):
        h.append(torch.arange(slots), torch.arange(slots) + 10 * (step % 4) + 10)
    return h


def test_append_leaves_other_slots_alone():
    h = _filled()
    ids, count = h.ids.clone(), h.count.clone()
    h.append(torch.tensor([-1, 2, 5, -7, 1 << 40, 9]), torch.tensor([41, 42, 43, 44, 45, 46]))
    h.append(torch.tensor([-1, 5]), torch.tensor([47, 48]))
    want = ids.clone()
    want[2, int(count[2]) % 4] = 42
    count[2] += 1
    assert torch.equal(h.ids, want) and torch.equal(h.count, count)


def test_append_to_the_first_and_last_slot_beside_outside_ones():
    """What stands in for a slot outside is no slot that the call also appends to."""
    h = SlotHistory(3, 2, 50)
    for _ in range(5):
        h.append(torch.tensor([-1, 0, 3, 2, 1, -1]), torch.tensor([1, 2, 3, 4, 5, 6]))
    assert h.ids.tolist() == [[2, 2], [5, 5], [4, 4]] and h.count.tolist() == [5, 5, 5]


def test_reset_and_rows():
    h = _filled()
    ids, count = h.ids.clone(), h.count.clone()
    h.reset(torch.tensor([-1, 1, 5]))
    ids[1], count[1] = -1, 0
    assert torch.equal(h.ids, ids) and torch.equal(h.count, count)
    shown, length = h.rows(torch.tensor([3, -1, 5, 1 << 35]))
    assert torch.equal(shown[0], ids[3]) and length.tolist() == [4, 0, 0, 0]
    assert bool((shown[1:] == -1).all())
    assert not bool(h.dense(torch.tensor([-1, 5])).any())
    run = h.rows_of_run(torch.tensor([-1, 3]), torch.tensor([[20, 21], [22, 9]]))
    np.testing.assert_array_equal(run[:2].numpy(), [[-1] * 4 + [20, -1], [-1] * 4 + [20, 21]])
    np.testing.assert_array_equal(run[2:, :4].numpy(), ids[3].expand(2, 4).numpy())


def test_shapes_are_the_slots():
    h = SlotHistory(3, 2, 50)
    assert h.ids.shape == (3, 2) and h.count.shape == (3,) and h.ids.is_contiguous() and h.count.is_contiguous()


def test_reorder_on_the_cpu_as_on_the_gpu():
    """A slot outside is no destination, and a beam whose parent's slot is outside keeps its own tokens."""
    h = _filled(slots=6)
    ids, count = h.ids.clone(), h.count.clone()
    slots = torch.tensor([[0, -1, 3], [6, 5, 1], [-1, -1, 1 << 30]])
    h.reorder(slots, torch.tensor([[2, 0, 1], [1, 2, 0], [1, 0, 0]]))
    #       0 takes 3's; -1 nothing; 3's parent has no slot; 6 nothing; 5 takes 1's; 1's parent has no slot
    want = {0: 3, 5: 1}
    for slot in range(6):
        of = want.get(slot, slot)
        assert torch.equal(h.ids[slot], ids[of]) and h.count[slot] == count[of]
    assert h.rows(torch.tensor([-1, 6]))[1].tolist() == [0, 0]


def test_copies_and_assigned_tensors_work_on():
    import copy
    import pickle

    for other in (lambda h: h, copy.copy, copy.deepcopy, lambda h: pickle.loads(pickle.dumps(h))):
        h = other(SlotHistory(3, 2, 50))
        h.append(torch.tensor([1]), torch.tensor([4]))
        assert h.ids.tolist() == [[-1, -1], [4, -1], [-1, -1]] and h.count.tolist() == [0, 1, 0]
        h.ids, h.count = torch.tensor([[7, 8], [9, -1], [-1, -1]], dtype=torch.int32), torch.tensor([2, 1, 0], dtype=torch.int32)
        h.append(torch.tensor([1, -1]), torch.tensor([5, 6]))
        assert h.ids.tolist() == [[7, 8], [9, 5], [-1, -1]] and h.rows(torch.tensor([1, -1]))[1].tolist() == [2, 0]
