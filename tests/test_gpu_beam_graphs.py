"""A whole search as one captured graph, from reset() to sequences(): every replay is a new search."""

import pytest

pytestmark = pytest.mark.gpu


def test_a_search_captured_whole(device):
    import torch

    from leat_b200.beam import BeamSearch
    from leat_b200.history import SlotHistory

    groups, beams, steps, vocab = 2, 4, 5, 700
    slots = torch.tensor([[3, 0, 6, 1], [2, 7, 5, 4]], dtype=torch.int32, device=device)
    table = torch.empty((steps, groups * beams, vocab), device=device)
    cache = torch.empty((8, steps, 6), device=device)
    history = SlotHistory(8, steps, vocab, special_ids=[5], device=device)

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        table.copy_(torch.randn(table.shape, generator=g) * 2)
        cache.copy_(torch.randn(cache.shape, generator=g))

    def run(search):
        search.reset()
        history.reset(slots)
        for step in range(steps):
            # the step's logits depend on the cache, and so on the beams that were followed
            logits = table[step] + cache[slots.long().reshape(-1)].sum((1, 2)).unsqueeze(1) * table[0]
            tokens = search.step(logits, cache, slots=slots, dim=1, length=step + 1, history=history)
            cache[slots.long().reshape(-1), step] = tokens.float() / vocab
        got = search.sequences()
        return got.tokens, got.lengths, search.scores, search.finished, search.lengths

    make = lambda: BeamSearch(groups, beams, steps, end_id=7, length_penalty=0.6, device=device)  # noqa: E731
    fill(0)
    captured = make()
    run(captured)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = run(captured)
    for seed in (1, 2, 3):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*outputs, cache, history.ids, history.count)]
        fill(seed)
        want = [*run(make()), cache, history.ids, history.count]
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    assert captured.steps == steps
