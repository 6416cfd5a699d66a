"""Beam search as it is used: a small model with a cache, stepped to the end on the GPU, against a search in
64 bits on the CPU that keeps every beam's whole sequence."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

VOCAB, SIZE, END = 211, 12, 7


class _Model:
    """Logits from the whole sequence through a cache (rows, heads, positions, size): position t holds the
    embedding of the token run there, and the logits come from their decayed sum."""

    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        self.embed = rng.standard_normal((VOCAB, 2, SIZE))
        self.head = rng.standard_normal((2 * SIZE, VOCAB)) * 0.9
        self.head[:, END] += 0.05

    def logits(self, cache, upto):
        weight = 0.8 ** np.arange(upto - 1, -1, -1)
        return ((cache[:, :, :upto] * weight[:, None]).sum(2).reshape(len(cache), -1) @ self.head).astype(np.float32)


def _search_on_cpu(model, prompts, beams, steps, alpha):
    """Per group: [(score, tokens)] of the last beams, best first; whole sequences, no cache."""
    answers = []
    for prompt in prompts:
        live = [(0.0, [], False)]
        for _ in range(steps):
            found = []
            for k, (score, tokens, done) in enumerate(live):
                if done:
                    found.append((score / ((5 + len(tokens)) / 6) ** alpha, k, 0.0, END, score, tokens, True))
                    continue
                run = list(prompt) + tokens
                cache = np.stack([model.embed[t] for t in run], 1)[None]  # (1, 2, positions, size)
                x = model.logits(cache, len(run))[0].astype(np.float64)
                share = x - (x.max() + np.log(np.exp(x - x.max()).sum()))
                for t in range(VOCAB):
                    s = score + share[t]
                    found.append((s / ((6 + len(tokens)) / 6) ** alpha, k, x[t], t, s, tokens + [t], t == END))
            found.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
            live = [(c[4], c[5], c[6]) for c in found[:beams]]
        answers.append(live)
    return answers


@pytest.mark.parametrize("alpha", [0.0, 0.7])
@pytest.mark.parametrize("with_slots", [False, True])
def test_search_with_a_cache(device, alpha, with_slots):
    import torch

    from leat_b200.beam import BeamSearch
    from leat_b200.history import SlotHistory

    groups, beams, steps, prompt = 3, 4, 12, 5
    model = _Model(1)
    rng = np.random.default_rng(2)
    prompts = rng.integers(8, VOCAB, (groups, prompt))
    rows = groups * beams + (3 if with_slots else 0)
    places = rng.permutation(rows)[: groups * beams] if with_slots else np.arange(groups * beams)
    slots = torch.tensor(places.reshape(groups, beams), dtype=torch.int32, device=device)
    # float64 caches follow bit for bit, so the logits are the CPU's but for nothing
    cache = torch.zeros((rows, 2, prompt + steps, SIZE), dtype=torch.float64, device=device)
    for g in range(groups):
        run = torch.tensor(np.stack([model.embed[t] for t in prompts[g]], 1), device=device)
        for k in range(beams):
            cache[places[g * beams + k], :, :prompt] = run
    history = SlotHistory(rows, steps, VOCAB, device=device)
    search = BeamSearch(groups, beams, steps, end_id=END, length_penalty=alpha, device=device)
    used = torch.tensor(places, device=device)
    for step in range(steps):
        logits = torch.tensor(model.logits(cache[used].cpu().numpy(), prompt + step), device=device)
        tokens = search.step(logits, cache, slots=slots if with_slots else None, dim=2, start=prompt, length=prompt + step)
        if with_slots:
            history.reorder(slots, search.parents)
            history.append(slots, search._tokens[step])
        cache[used, :, prompt + step] = torch.tensor(model.embed[tokens.cpu().numpy().reshape(-1)], device=device)
    got = search.sequences()
    want = _search_on_cpu(model, prompts, beams, steps, alpha)
    for g in range(groups):
        for k, (score, tokens, done) in enumerate(want[g]):
            length = int(got.lengths[g, k])
            assert got.tokens[g, k, :length].tolist() == tokens
            assert bool((got.tokens[g, k, length:] == END).all())
            assert length == len(tokens) == int(search.lengths[g, k]) and bool(search.finished[g, k]) == done
            # a float32 log-sum and a float32 score per step
            assert abs(float(search.scores[g, k]) - score) <= steps * (60 + abs(score)) * 2.0**-24
            if with_slots and not done:
                assert history.ids[places[g * beams + k]].tolist() == tokens
    with pytest.raises(ValueError):
        search.step(logits)
    search.reset()
    assert search.steps == 0 and search.scores[:, 0].tolist() == [0.0] * groups


def test_step_keeps_history_itself_and_dead_beams_run_token_zero(device):
    import torch

    from leat_b200.beam import BeamSearch
    from leat_b200.history import SlotHistory

    search = BeamSearch(2, 3, 4, device=device)
    slots = torch.tensor([[4, 1, 0], [2, 5, 3]], dtype=torch.int32, device=device)
    history = SlotHistory(6, 4, 50, device=device)
    logits = torch.full((6, 50), float("-inf"), device=device)
    logits[:, 10], logits[:, 20] = 1.0, 0.5  # two continuations for three beams
    tokens = search.step(logits, slots=slots, history=history)
    assert tokens.tolist() == [[10], [20], [0], [10], [20], [0]]
    assert torch.isneginf(search.scores[:, 2]).all()
    tokens = search.step(logits, slots=slots, history=history)
    assert search.parents.tolist()[0] == [0, 0, 1]  # 10 10, 10 20, 20 10: equal ranks by beam
    assert history.ids[4].tolist()[:2] == [10, 10] and history.ids[1].tolist()[:2] == [10, 20] and history.ids[0].tolist()[:2] == [20, 10]
    with pytest.raises(ValueError):
        search.step(logits, history=history)


def test_a_finished_beam_adds_nothing_to_its_history(device):
    import torch

    from leat_b200.beam import BeamSearch
    from leat_b200.history import SlotHistory

    search = BeamSearch(1, 2, 4, end_id=3, device=device)
    slots = torch.tensor([[0, 1]], dtype=torch.int32, device=device)
    history = SlotHistory(2, 6, 20, device=device)
    logits = torch.zeros((2, 20), device=device)
    logits[:, 3], logits[:, 5] = 4.0, 3.9
    for _ in range(3):
        search.step(logits, slots=slots, history=history)
    got = search.sequences()
    for k in range(2):
        length = int(got.lengths[0, k])
        assert int(history.count[k]) == length and history.ids[k, :length].tolist() == got.tokens[0, k, :length].tolist()
    assert int(got.lengths[0].min()) == 1 and bool(search.finished[0].any())


@pytest.mark.parametrize("bad", [dict(groups=0), dict(beams=0), dict(beams=65), dict(max_steps=0)])
def test_search_refusals(device, bad):
    from leat_b200.beam import BeamSearch

    with pytest.raises(ValueError):
        BeamSearch(**{"groups": 1, "beams": 2, "max_steps": 3, **bad}, device=device)
