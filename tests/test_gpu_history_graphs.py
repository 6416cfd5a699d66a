"""SlotHistory's calls inside a captured graph, all of them."""

import pytest

pytestmark = pytest.mark.gpu


def test_every_call_captured(device):
    import torch

    from leat_b200.history import SlotHistory

    h, plain = (SlotHistory(6, 4, 100, special_ids=[9], device=device) for _ in range(2))
    slots = torch.tensor([[4, 1, -1], [0, 5, 6]], device=device)
    tokens = torch.tensor([[11, 9, 12], [13, 14, 15]], device=device)
    parents = torch.tensor([[1, 0, 0], [1, 1, 2]], dtype=torch.int32, device=device)
    again = torch.tensor([1, 3], device=device)
    run = torch.tensor([[20, 21], [22, 9]], device=device)

    def step(history):
        history.append(slots, tokens)
        history.reorder(slots, parents)
        history.reset(again)
        return *history.rows(slots), history.rows_of_run(torch.stack([slots[0, 0], slots[1, 1]]), run)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(h)
    for _ in range(6):
        graph.replay()
        torch.cuda.synchronize()
        want = step(plain)
        for a, b in zip((h.ids, h.count, *got), (plain.ids, plain.count, *want)):
            assert torch.equal(a, b)
    assert bool((h.ids >= 0).any())
