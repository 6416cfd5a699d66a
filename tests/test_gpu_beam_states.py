"""reorder_states and beam_sequences on the GPU: every layout and width of copy, ranges of positions,
slots, cycles among the parents, what must stay as it was; and the read-back of long searches."""

import numpy as np
import pytest

from tests import beam_reference as plain

pytestmark = pytest.mark.gpu


def _expected(t, parents, rows, dim, start, length):
    """What the state holds afterwards, by plain indexing."""
    import torch

    out = t.clone()
    groups, beams = parents.shape
    for g in range(groups):
        lo = start[g] if isinstance(start, list) else start
        hi = length[g] if isinstance(length, list) else length
        for k in range(beams):
            p = int(parents[g, k])
            if not 0 <= p < beams:
                continue
            to, of = int(rows[g, k]), int(rows[g, p])
            if not (0 <= to < t.shape[0] and 0 <= of < t.shape[0]):
                continue
            if dim is None:
                out[to] = t[of]
            else:
                places = torch.arange(max(lo, 0), max(lo, 0, min(hi, t.shape[dim])), device=t.device)
                out[to] = out[to].index_copy(dim - 1, places, t[of].index_select(dim - 1, places))
    return out


def _random(shape, dtype, seed, device):
    import torch

    g = torch.Generator().manual_seed(seed)
    if dtype == torch.bool:
        return (torch.rand(shape, generator=g) < 0.5).to(device)
    if dtype.is_floating_point:
        return torch.randn(shape, generator=g).to(dtype).to(device)
    return torch.randint(0, 100, shape, generator=g).to(dtype).to(device)


def _plain_rows(groups, beams):
    return np.arange(groups * beams).reshape(groups, beams)


@pytest.mark.parametrize("beams", [1, 2, 3, 5, 8, 12, 16, 17, 23, 24, 32, 33, 64])
def test_parents_of_every_kind(device, beams):
    import torch

    from leat_b200.beam import reorder_states

    rng = np.random.default_rng(beams)
    groups = 5
    parents = rng.integers(0, beams, (groups, beams))
    parents[0] = np.arange(beams)  # nothing moves
    parents[1] = rng.permutation(beams)  # cycles
    parents[2] = np.roll(np.arange(beams), 1)  # one cycle
    parents[3] = beams - 1  # all of one
    p = torch.tensor(parents, dtype=torch.int32, device=device)
    states = [_random((groups * beams, 3, 40, 16), torch.bfloat16, 1, device), _random((groups * beams, 7), torch.int32, 2, device)]
    want = [_expected(t, parents, _plain_rows(groups, beams), None, 0, None) for t in states]
    reorder_states(states, p)
    for a, b in zip(states, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["uint8", "bool", "int16", "bfloat16", "float32", "int64", "float64"])
@pytest.mark.parametrize("shape,dim", [
    ((12, 5, 33, 8), 2), ((12, 33, 5, 8), 1), ((12, 2, 3, 33, 4), 3), ((12, 33), 1), ((12, 33, 1), 1), ((12, 1, 33, 7), 2),
    ((12, 4, 16), None), ((12, 1027), None), ((12, 3, 11), None), ((12,), None), ((12, 1), None),
])  # fmt: skip
def test_types_and_layouts(device, dtype, shape, dim):
    import torch

    from leat_b200.beam import reorder_states

    dtype = getattr(torch, dtype)
    parents = np.random.default_rng(3).integers(0, 4, (3, 4))
    t = _random(shape, dtype, 5, device)
    ranges = [(0, None)] if dim is None else [(0, None), (3, 20), (0, 1), (32, 33), (7, 7), (9, 2), (0, 1000), (40, 50)]
    for start, length in ranges:
        now = t.clone()
        want = _expected(t, parents, _plain_rows(3, 4), dim, start, 1 << 30 if length is None else length)
        reorder_states(now, torch.tensor(parents, dtype=torch.int32, device=device), dim=dim, start=start, length=length)
        assert torch.equal(now, want), (start, length)


def test_views_offsets_and_strided_rows(device):
    """Rows of a larger tensor, an odd first byte, a layer of a stacked cache, heads outside the rows."""
    import torch

    from leat_b200.beam import reorder_states

    parents = np.array([[1, 0, 0], [2, 2, 1]])
    p = torch.tensor(parents, dtype=torch.int32, device=device)
    whole = _random((6 * 130 + 1,), torch.uint8, 1, device)
    views = [
        whole[1:].as_strided((6, 101), (130, 1)),
        _random((4, 6, 2, 20, 8), torch.float16, 2, device)[2],
        _random((2, 6, 20, 8), torch.float16, 3, device).transpose(0, 1),
        _random((6, 20, 24), torch.float32, 4, device)[:, :, :24][:, 2:18],
    ]
    for t, dim in zip(views, [None, 2, 2, 1]):
        want = _expected(t.clone(), parents, _plain_rows(2, 3), dim, 0, 1 << 30)
        base = whole.clone()
        reorder_states([t], p, dim=dim)
        assert torch.equal(t, want)
        if t is views[0]:  # the bytes between the rows are as they were
            gaps = torch.ones(whole.numel(), dtype=torch.bool, device=device)
            gaps[1:].as_strided((6, 101), (130, 1)).fill_(False)
            assert torch.equal(whole[gaps], base[gaps])


def test_slots_ranges_per_group_and_bad_indices(device):
    import torch

    from leat_b200.beam import reorder_states

    rng = np.random.default_rng(9)
    groups, beams, rows = 4, 6, 40
    parents = rng.integers(0, beams, (groups, beams))
    parents[0, 0], parents[0, 1], parents[1, 2] = -1, beams, 1 << 30
    slots = rng.permutation(rows)[: groups * beams].reshape(groups, beams)
    slots[2, 0], slots[2, 1], slots[3, 3] = -3, rows, 1 << 30
    start, length = [0, 5, 100, 17], [64, 5, 3, 200]
    t = _random((rows, 2, 64, 24), torch.bfloat16, 1, device)
    want = _expected(t, parents, slots, 2, start, length)
    as32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
    reorder_states([t], as32(parents), slots=as32(slots), dim=2, start=as32(start), length=as32(length))
    assert torch.equal(t, want)


def test_many_states_of_different_widths(device):
    import torch

    from leat_b200.beam import reorder_states

    parents = np.random.default_rng(1).integers(0, 3, (7, 3))
    dtypes = [torch.bfloat16, torch.float32, torch.uint8, torch.int64]
    states = [_random((21, 1 + i % 5, 1 + i), dtypes[i % 4], i, device) for i in range(150)]
    want = [_expected(t, parents, _plain_rows(7, 3), None, 0, None) for t in states]
    reorder_states(states, torch.tensor(parents, dtype=torch.int32, device=device))
    for a, b in zip(states, want):
        assert torch.equal(a, b)


def test_a_cache_beyond_four_gigabytes(device):
    """Byte offsets past 32 bits, rows and runs of places alike."""
    import torch

    from leat_b200.beam import reorder_states

    t = torch.zeros((4, 3, 1 << 20, 192), dtype=torch.bfloat16, device=device)  # 4.8 GB
    last = (1 << 20) - 5
    t[:, :, last:] = _random((4, 3, 5, 192), torch.bfloat16, 1, device)
    want = t[:, :, last:][torch.tensor([3, 0, 1, 1], device=device)].clone()
    reorder_states(t, torch.tensor([[3, 0, 1, 1]], dtype=torch.int32, device=device), dim=2, start=last)
    assert torch.equal(t[:, :, last:], want)


def test_empty_states_and_groups(device):
    import torch

    from leat_b200.beam import reorder_states

    p = torch.tensor([[1, 0]], dtype=torch.int32, device=device)
    reorder_states([], p)
    reorder_states([torch.empty((2, 0), device=device), torch.empty((2, 3, 0, 4), device=device)[:, :, :, 0]], p)
    reorder_states(torch.empty((2, 0, 4), device=device), p, dim=1)
    reorder_states(torch.ones((3, 4), device=device), torch.empty((0, 2), dtype=torch.int32, device=device))


def test_captured_on_another_stream(device):
    import torch

    from leat_b200.beam import reorder_states

    parents = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=device)
    t = _random((3, 100, 50), torch.float32, 2, device)
    before = t.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        reorder_states(t, parents)
    with torch.cuda.stream(stream):
        for _ in range(2):
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(t, before[torch.tensor([1, 2, 0], device=device)])


def test_reorder_refusals(device):
    import torch

    from leat_b200.beam import reorder_states

    p = torch.tensor([[1, 0]], dtype=torch.int32, device=device)
    t = torch.zeros((2, 3, 8, 4), device=device)
    two = torch.zeros(2, dtype=torch.int32, device=device)
    bad = [
        dict(parents=p.long()), dict(parents=p[0]), dict(parents=p.cpu()), dict(states=t.cpu()), dict(states=[t, None]),
        dict(states=t[:1]), dict(slots=p.long()), dict(slots=p[:, :1]), dict(start=1), dict(length=4), dict(dim=0), dict(dim=4),
        dict(dim=2, start=-1), dict(dim=2, length=-1), dict(dim=2, length=two), dict(dim=2, start=1.0), dict(dim=2, start=True),
        dict(states=t.transpose(2, 3), dim=2), dict(states=t[:, :, ::2], dim=2), dict(states=t[:1].expand(2, 3, 8, 4), dim=2),
        dict(states=t[:, :1].expand(2, 3, 8, 4), dim=2), dict(states=torch.zeros((), device=device)),
        dict(states=[t, t]), dict(states=[t, t[:, :2]]), dict(states=t.clone().requires_grad_()), dict(states=t.transpose(1, 3)),
        dict(parents=torch.zeros((1, 65), dtype=torch.int32, device=device), states=torch.zeros((65, 4), device=device)),
    ]  # fmt: skip
    for more in bad:
        with pytest.raises(ValueError):
            reorder_states(**{"states": t, "parents": p, **more})


@pytest.mark.parametrize("steps,groups,beams", [
    (1, 1, 1), (1, 3, 4), (2, 2, 2), (5, 300, 3), (48, 1, 4), (63, 2, 5), (64, 2, 7), (65, 2, 8), (257, 3, 16), (1000, 2, 24),
    (513, 1, 64), (700, 1, 33), (7000, 1, 64), (2000, 20, 2), (511, 1, 1),
])  # fmt: skip
def test_sequences(device, steps, groups, beams):
    import torch

    from leat_b200.beam import beam_sequences

    rng = np.random.default_rng(steps)
    tokens = rng.integers(1, 1000, (steps, groups, beams)).astype(np.int32)
    tokens[rng.random(tokens.shape) < 1.0 / steps] = 0
    parents = rng.integers(0, beams, (steps, groups, beams)).astype(np.int32)
    a, b = torch.tensor(tokens, device=device), torch.tensor(parents, device=device)
    for end in (None, 0):
        got = beam_sequences(a, b, end)
        want, lengths = plain.sequences(tokens, parents, end)
        np.testing.assert_array_equal(got.tokens.cpu().numpy(), want)
        np.testing.assert_array_equal(got.lengths.cpu().numpy(), lengths)


def test_sequences_that_keep_many_paths(device):
    """Parents as permutations: the paths never join, so every run's map matters in full."""
    import torch

    from leat_b200.beam import beam_sequences

    rng = np.random.default_rng(5)
    tokens = rng.integers(0, 50000, (900, 3, 12)).astype(np.int32)
    parents = np.stack([np.stack([rng.permutation(12) for _ in range(3)]) for _ in range(900)]).astype(np.int32)
    got = beam_sequences(torch.tensor(tokens, device=device), torch.tensor(parents, device=device))
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), plain.sequences(tokens, parents)[0])


def test_sequences_behind_a_bad_parent(device):
    import torch

    from leat_b200.beam import beam_sequences

    rng = np.random.default_rng(6)
    tokens = rng.integers(0, 9, (300, 2, 4)).astype(np.int32)
    parents = rng.integers(0, 4, (300, 2, 4)).astype(np.int32)
    parents[0] = 77  # never followed
    parents[150, 0], parents[40, 1, 2], parents[299, 1, 0] = -1, 4, 1 << 30
    for end in (None, 8):
        got = beam_sequences(torch.tensor(tokens, device=device), torch.tensor(parents, device=device), end)
        want, lengths = plain.sequences(tokens, parents, end)
        np.testing.assert_array_equal(got.tokens.cpu().numpy(), want)
        np.testing.assert_array_equal(got.lengths.cpu().numpy(), lengths)


def test_no_steps_and_refusals(device):
    import torch

    from leat_b200.beam import beam_sequences

    none = torch.empty((0, 2, 3), dtype=torch.int32, device=device)
    got = beam_sequences(none, none, 1)
    assert got.tokens.shape == (2, 3, 0) and got.lengths.tolist() == [[0] * 3] * 2
    t = torch.zeros((4, 2, 3), dtype=torch.int32, device=device)
    for a, b, end in [(t.long(), t, None), (t, t.long(), None), (t, t[:3], None), (t[0], t[0], None), (t.cpu(), t.cpu(), None),
                      (t, t, -1), (t, t, True), (torch.zeros((2, 1, 65), dtype=torch.int32, device=device),) * 2 + (None,)]:  # fmt: skip
        with pytest.raises(ValueError):
            beam_sequences(a, b, end)
