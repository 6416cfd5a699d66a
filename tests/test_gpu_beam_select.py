"""beam_select on the GPU against all continuations in 64 bits: sizes from one token up, types, strides,
masks that leave a row empty, ties, finished and dead beams, streams and graphs."""

import numpy as np
import pytest

from tests import beam_reference as plain

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


def _inputs(groups, beams, vocab, kind, seed, device, pad=0, scale=3.0):
    import torch

    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((groups * beams, vocab + pad), generator=g) * scale).to(getattr(torch, kind))
    scores = (-2.0 * torch.rand((groups, beams), generator=g)).cumsum(1)
    return logits.to(device)[:, :vocab], scores.to(device)


def _numpy(x):
    return x.double().cpu().numpy()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("groups,beams,vocab,width,pad", [
    (1, 1, 1, 1, 0), (1, 4, 3, 4, 0), (2, 3, 17, 64, 0), (3, 5, 1000, 10, 0), (3, 4, 8192, 8, 0), (2, 3, 8193, 6, 0),
    (2, 2, 16384, 4, 8), (4, 8, 16411, 16, 1), (1, 64, 300, 64, 4), (2, 2, 50000, 64, 0), (5, 7, 40001, 7, 3), (150, 2, 2000, 2, 0),
])  # fmt: skip
def test_sizes_types_and_strides(device, kind, groups, beams, vocab, width, pad):
    from leat_b200.beam import beam_select

    logits, scores = _inputs(groups, beams, vocab, kind, vocab + width, device, pad)
    got = beam_select(logits, scores, width)
    plain.check_selected(got, _numpy(logits), scores.cpu().numpy(), width)


def test_a_transposed_and_an_offset_matrix(device):
    import torch

    from leat_b200.beam import beam_select

    logits, scores = _inputs(2, 3, 9000, "float32", 5, device)
    want = beam_select(logits, scores, 6)
    moved = torch.empty(6 * 9001 + 1, device=device)[1:].as_strided((6, 9000), (9001, 1)).copy_(logits)  # four bytes off
    for other in (logits.t().contiguous().t(), moved):
        got = beam_select(other, scores, 6)
        assert torch.equal(got.tokens, want.tokens) and torch.equal(got.parents, want.parents)
        torch.testing.assert_close(got.scores, want.scores, rtol=2.0**-23, atol=2 * plain.LOG_SUM_ERROR)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("vocab", [4000, 8191, 20000])
def test_masks(device, kind, vocab):
    """Rows with nothing, with one token, with a few among the type's lowest value, and with NaN and
    infinities in places."""
    import torch

    from leat_b200.beam import beam_select

    logits, scores = _inputs(4, 4, vocab, kind, 3, device)
    lowest = torch.finfo(logits.dtype).min
    logits[0] = float("-inf")
    logits[1] = float("-inf")
    logits[1, vocab - 1] = -5.0
    logits[2, 5:] = lowest
    logits[3] = lowest
    logits[4:8] = float("-inf")  # a group without any
    logits[8, ::3] = float("nan")
    logits[9, 7::2] = float("-inf")
    logits[10, :] = float("nan")
    logits[11, 100] = float("inf")
    logits[12] = float("-inf")
    logits[12, 3], logits[12, 9] = float("inf"), float("inf")
    got = beam_select(logits, scores, 8)
    plain.check_selected(got, _numpy(logits), scores.cpu().numpy(), 8)
    assert bool((got.tokens[1] == -1).all())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("vocab,width", [(300, 5), (9000, 64), (9001, 64), (40000, 8)])
def test_equal_logits_go_by_beam_and_token(device, kind, vocab, width):
    """Constant rows, and rows of a few whole numbers: equal beams tie, and their equal logits with
    them, in the kernel's 64 bits as in the formula's."""
    import torch

    from leat_b200.beam import beam_select

    logits = torch.zeros((6, vocab), device=device).to(getattr(torch, kind))
    logits[3:] = torch.randint(0, 3, (vocab,), generator=torch.Generator().manual_seed(1)).to(device).to(logits.dtype)
    scores = torch.zeros((2, 3), device=device)
    got = beam_select(logits, scores, width)
    for g in range(2):
        order = np.lexsort((np.arange(vocab), -_numpy(logits[3 * g])))
        best = order[_numpy(logits[3 * g])[order] == _numpy(logits[3 * g]).max()]
        n = min(width, len(best))
        assert got.tokens[g, :n].tolist() == best[:n].tolist()
        assert got.parents[g, :n].tolist() == [0] * n
    plain.check_selected(got, _numpy(logits), scores.cpu().numpy(), width, exact_order=True)


@pytest.mark.parametrize("kind", TYPES)
def test_many_large_logits_in_few_threads(device, kind):
    """More logits above a tile's floor than its list holds: 120 of them side by side."""
    from leat_b200.beam import beam_select

    logits, scores = _inputs(2, 2, 30000, kind, 11, device)
    logits[0, 8000:8120] += 30.0
    logits[1, 0:200] += 20.0
    logits[2, 29000:] += 10.0
    got = beam_select(logits, scores, 64)
    plain.check_selected(got, _numpy(logits), scores.cpu().numpy(), 64)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("beams,vocab,allowed,width", [(8, 70000, 5, 8), (8, 70000, 5, 60), (1, 50000, 3, 8), (4, 40000, 1, 16), (24, 20000, 30, 48), (2, 33000, 9, 64)])
def test_fewer_allowed_tokens_than_parts(device, kind, beams, vocab, allowed, width):
    """All but a few tokens, side by side, at the type's lowest value: the best lie in one corner of the rows,
    and where they are too few the lowest token ids among equals follow."""
    import torch

    from leat_b200.beam import beam_select

    logits, scores = _inputs(2, beams, vocab, kind, 41, device)
    kept = logits[:, 100:100 + allowed].clone()
    logits[:] = torch.finfo(logits.dtype).min
    logits[:, 100:100 + allowed] = kept
    got = beam_select(logits, scores, width)
    n = min(width, beams * allowed)
    plain.check_selected(got, _numpy(logits), scores.cpu().numpy(), width)
    assert bool(((got.tokens[:, :n] >= 100) & (got.tokens[:, :n] < 100 + allowed)).all())
    if beams == 1:
        assert got.tokens[:, n:].tolist() == [list(range(width - n))] * 2


@pytest.mark.parametrize("vocab,width", [(60000, 8), (60000, 64), (300, 64)])
def test_many_beams_of_one_ramp(device, vocab, width):
    """Sorted rows that differ by their scores alone: every level's best lie side by side."""
    import torch

    from leat_b200.beam import beam_select

    row = torch.linspace(30, 0, vocab, device=device)
    scores = -torch.arange(12, device=device, dtype=torch.float32).reshape(2, 6) * 0.37
    for logits in (row.expand(12, vocab).contiguous(), row.flip(0).expand(12, vocab).contiguous()):
        got = beam_select(logits, scores, width)
        plain.check_selected(got, _numpy(logits), scores.cpu().numpy(), width)


def test_ascending_and_descending_logits(device):
    import torch

    from leat_b200.beam import beam_select

    ramp = torch.linspace(-20, 20, 33000, device=device)
    logits = torch.stack([ramp, ramp.flip(0)])
    got = beam_select(logits, torch.tensor([[0.0, -1e-3]], device=device), 64)
    plain.check_selected(got, _numpy(logits), np.array([[0.0, -1e-3]], np.float32), 64)


@pytest.mark.parametrize("scale", [1e30, 3e38])
def test_logits_near_the_largest_float(device, scale):
    import torch

    from leat_b200.beam import beam_select

    logits = torch.rand((4, 9000), generator=torch.Generator().manual_seed(2)).to(device) * 2 - 1
    logits *= scale
    logits[1] = torch.finfo(torch.float32).max
    got = beam_select(logits, torch.zeros((4, 1), device=device), 2)
    for row in range(4):  # one token has it all, or equal ones share it
        best = int(logits[row].argmax())
        assert int(got.tokens[row, 0]) == best
    assert got.scores[0, 0] == 0.0
    assert abs(float(got.scores[1, 0]) + np.log(9000)) <= plain.LOG_SUM_ERROR + 10 * 2.0**-24


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("low,high", [(-62.0, 25.0), (-62.0, 22.5), (-62.0, 21.0), (-62.0, 20.0), (-40.0, 60.0), (-900.0, 10.0), (-1500.0, -1400.0), (30.0, -40.0)])
def test_rows_that_begin_far_from_their_maximum(device, kind, low, high):
    """The sums start from a row's first logits: the others may lie up to the exponentials' whole range above."""
    import torch

    from leat_b200.beam import beam_select

    logits, scores = _inputs(2, 2, 9000, "float32", 23, device, scale=0.5)
    logits += high
    logits[:, :512] = low
    logits = logits.to(getattr(torch, kind))
    got = beam_select(logits, scores, 5)
    plain.check_selected(got, _numpy(logits), scores.cpu().numpy(), 5)


@pytest.mark.parametrize("alpha", [0.0, 0.6, 1.0, -0.5])
@pytest.mark.parametrize("vocab", [40, 9001])
def test_finished_dead_beams_and_lengths(device, alpha, vocab):
    import torch

    from leat_b200.beam import beam_select

    logits, scores = _inputs(6, 5, vocab, "float32", 21, device)
    g = torch.Generator().manual_seed(4)
    finished = (torch.rand((6, 5), generator=g) < 0.4).to(device)
    lengths = torch.randint(0, 50, (6, 5), generator=g, dtype=torch.int32).to(device)
    scores[1, 2:] = float("-inf")
    scores[2] = float("-inf")
    finished[2, 0] = True  # dead and finished: dead
    scores[3, 1] = float("nan")
    finished[4] = True
    logits[:, 3] += 2.0  # the end token is likely
    logits[4 * 5:5 * 5] = float("nan")  # not read
    got = beam_select(logits, scores, 7, finished=finished, end_id=3, lengths=lengths, length_penalty=alpha)
    plain.check_selected(got, _numpy(logits), scores.cpu().numpy(), 7, finished.cpu().numpy(), 3, lengths.cpu().numpy(), alpha)
    assert bool((got.tokens[2] == -1).all())


def test_first_step_and_no_flags(device):
    import torch

    from leat_b200.beam import beam_select

    logits, scores = _inputs(3, 4, 5000, "bfloat16", 8, device)
    scores[:, 1:] = float("-inf")
    got = beam_select(logits, scores)
    assert got.finished is None and got.lengths is None
    assert bool((got.parents == 0).all())
    plain.check_selected(got, _numpy(logits), scores.cpu().numpy(), 4)
    ended = beam_select(logits, scores, end_id=2)  # ends wanted, none finished yet
    assert torch.equal(ended.tokens, got.tokens) and torch.equal(ended.finished, got.tokens == 2)


def test_rows_beyond_two_to_the_thirty_first_logit(device):
    import torch

    from leat_b200.beam import beam_select

    stride = (1 << 31) // 3 + 8 * 1237
    held = torch.empty(3 * stride + 20000, dtype=torch.bfloat16, device=device)
    logits = held.as_strided((4, 20000), (stride, 1))
    small, scores = _inputs(1, 4, 20000, "bfloat16", 13, device)
    logits.copy_(small)
    got, want = beam_select(logits, scores), beam_select(small.contiguous(), scores)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.scores, want.scores)


def test_same_answer_every_time_into_given_tensors(device):
    import torch

    from leat_b200.beam import Selected, beam_select

    logits, scores = _inputs(8, 8, 30000, "float16", 17, device)
    lengths = torch.ones((8, 8), dtype=torch.int32, device=device)
    first = beam_select(logits, scores, 16, end_id=1, lengths=lengths, length_penalty=0.7)
    out = Selected(*(torch.full_like(t, 1) for t in (first.tokens, first.parents, first.scores, first.finished, first.lengths)))
    for _ in range(5):
        got = beam_select(logits, scores, 16, end_id=1, lengths=lengths, length_penalty=0.7, out=out)
        assert got is out
        for name in ("tokens", "parents", "scores", "finished", "lengths"):
            assert torch.equal(getattr(got, name), getattr(first, name)), name


def test_two_captured_graphs_and_an_eager_call_share_nothing(device):
    import torch

    from leat_b200.beam import beam_select

    inputs = [_inputs(4, 4, 30000, "float32", s, device) for s in (31, 32)]
    want = [beam_select(*x, 8) for x in inputs]
    graphs, got, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(beam_select(*x, 8))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        again = beam_select(*inputs[0], 8)
    torch.cuda.synchronize()
    assert torch.equal(again.tokens, want[0].tokens)
    for a, b in zip(got, want):
        assert torch.equal(a.tokens, b.tokens) and torch.equal(a.parents, b.parents) and torch.equal(a.scores, b.scores)


def test_no_groups(device):
    import torch

    from leat_b200.beam import beam_select

    got = beam_select(torch.empty((0, 100), device=device), torch.empty((0, 4), device=device), 6)
    assert got.tokens.shape == (0, 6) and got.scores.dtype == torch.float32


def test_refusals(device):
    import torch

    from leat_b200.beam import Selected, beam_select

    logits, scores = _inputs(2, 3, 100, "float32", 1, device)
    lengths = torch.zeros((2, 3), dtype=torch.int32, device=device)
    done = torch.zeros((2, 3), dtype=torch.bool, device=device)
    ints = lambda: torch.zeros((2, 3), dtype=torch.int32, device=device)  # noqa: E731
    bad = [
        dict(logits=logits.double()), dict(logits=logits[0]), dict(logits=logits.cpu()), dict(logits=logits[:5]),
        dict(logits=logits[:, :0]), dict(scores=scores.double()), dict(scores=scores.cpu()), dict(scores=scores.reshape(-1)),
        dict(width=0), dict(width=65), dict(width=2.0), dict(width=True), dict(end_id=100), dict(end_id=-1), dict(finished=done),
        dict(finished=done.int(), end_id=1), dict(finished=done[:1], end_id=1), dict(lengths=lengths.long()),
        dict(length_penalty=0.5), dict(length_penalty=float("nan"), lengths=lengths), dict(length_penalty=17.0, lengths=lengths),
        dict(out=Selected(ints(), ints(), scores.clone()), width=4), dict(out=Selected(ints(), ints(), scores)),
        dict(out=Selected(ints(), ints(), scores.clone()), end_id=1), dict(out=Selected(ints(), ints().long(), scores.clone())),
    ]  # fmt: skip
    for more in bad:
        with pytest.raises(ValueError):
            beam_select(**{"logits": logits, "scores": scores, **more})
    with pytest.raises(ValueError):
        beam_select(torch.zeros((130, 10), device=device), torch.zeros((2, 65), device=device))
