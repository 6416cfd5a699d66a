"""A search of a padded batch: groups without cache slots of their own have -1 or a number beyond the last."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("outside", [-1, 12, 1 << 30])
def test_padding_groups_touch_nothing(device, outside):
    import torch

    from leat_b200.beam import BeamSearch
    from leat_b200.history import SlotHistory

    groups, beams, steps, vocab = 3, 4, 6, 500
    g = torch.Generator().manual_seed(1)
    used = torch.tensor([[2, 0, 7, 5], [0, 0, 0, 0], [9, 11, 1, 10]], dtype=torch.int32, device=device)  # slot 11 is the last
    slots = used.clone()
    slots[1] = outside
    cache = torch.randn((12, 2, steps, 3), generator=g).to(device)
    history = SlotHistory(12, steps, vocab, special_ids=[3], device=device)
    history.append(torch.arange(12), torch.arange(12) + 100)
    alone = BeamSearch(2, beams, steps, device=device)
    alone_cache, alone_history = cache.clone(), SlotHistory(12, steps, vocab, special_ids=[3], device=device)
    alone_history.append(torch.arange(12), torch.arange(12) + 100)
    search = BeamSearch(groups, beams, steps, device=device)
    for step in range(steps):
        logits = torch.randn((groups * beams, vocab), generator=g).to(device) * 3
        tokens = search.step(logits, cache, slots=slots, dim=2, length=step + 1, history=history)
        rest = alone.step(torch.cat([logits[:beams], logits[2 * beams:]]), alone_cache, slots=used[[0, 2]].contiguous(), dim=2,
                          length=step + 1, history=alone_history)  # fmt: skip
        assert torch.equal(tokens.reshape(groups, beams)[[0, 2]], rest.reshape(2, beams))
    torch.cuda.synchronize()
    assert torch.equal(cache, alone_cache)
    assert torch.equal(history.ids, alone_history.ids) and torch.equal(history.count, alone_history.count)
    shown, length = history.rows(slots)
    assert bool((shown[4:8] == -1).all()) and length[4:8].tolist() == [0] * 4
    np.testing.assert_array_equal(shown[:4].cpu().numpy(), history.ids[used[0].long()].cpu().numpy())
