"""+inf logits, which count as the largest float, where as many of them as are wanted lie in different
parts of the rows; and ranks beyond float32's range."""

import numpy as np
import pytest

from tests import beam_reference as plain

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]
VOCABS = [300, 9001, 200000]  # levels that begin at the chunks, of one tile and of several, and at the tiles
INF = float("inf")


def _logits(rows, vocab, kind, seed, device):
    import torch

    return (torch.randn((rows, vocab), generator=torch.Generator().manual_seed(seed)) * 3).to(getattr(torch, kind)).to(device)


def _check_top(got, logits, top):
    """Ids in order, and values to within the log-sum's error and one rounding."""
    share, x = plain.log_softmax(logits), plain.clean(logits)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    np.testing.assert_array_equal(got.top_ids.cpu().numpy(), order)
    want = np.take_along_axis(share, order, 1)
    error = np.abs(got.top_logprobs.cpu().numpy().astype(np.float64) - want)
    assert (error <= plain.LOG_SUM_ERROR + np.abs(want) * 2.0**-24).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_one_infinity_and_one_wanted(device, kind, vocab):
    import torch

    from leat_b200.beam import beam_select
    from leat_b200.logprobs import token_logprobs

    logits = _logits(4, vocab, kind, 1, device)
    for row, token in enumerate([0, vocab // 2, vocab - 1, 130]):
        logits[row, token] = INF
    _check_top(token_logprobs(logits, top=1), logits.double().cpu().numpy(), 1)
    scores = torch.tensor([[-1.0], [0.0], [2.5], [-70.0]], device=device)
    plain.check_selected(beam_select(logits, scores, 1), logits.double().cpu().numpy(), scores.cpu().numpy(), 1, exact_order=True)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("groups,beams,apart", [(2, 4, 0), (2, 4, 61), (1, 12, 0), (1, 12, 19)])
def test_one_infinity_per_beam(device, kind, vocab, groups, beams, apart):
    """A token forced by +inf: the same one in every row, or one each, and every beam goes on with it."""
    import torch

    from leat_b200.beam import beam_select

    logits = _logits(groups * beams, vocab, kind, 2, device)
    for row in range(groups * beams):
        logits[row, (7 + apart * row) % vocab] = INF
    scores = -torch.arange(groups * beams, dtype=torch.float32, device=device).reshape(groups, beams) * 0.3
    got = beam_select(logits, scores)
    plain.check_selected(got, logits.double().cpu().numpy(), scores.cpu().numpy(), beams, exact_order=True)
    assert torch.equal(got.scores, scores)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("top,have", [(5, 5), (5, 7), (20, 40), (64, 200)])
def test_more_infinities_than_wanted(device, kind, vocab, top, have):
    from leat_b200.logprobs import token_logprobs

    logits = _logits(3, vocab, kind, 3, device)
    rng = np.random.default_rng(vocab)
    for row in range(3):
        logits[row, rng.permutation(vocab)[:have].tolist()] = INF
    _check_top(token_logprobs(logits, top=top), logits.double().cpu().numpy(), top)


@pytest.mark.parametrize("vocab", VOCABS)
def test_an_infinity_ties_with_the_largest_float(device, vocab):
    import torch

    from leat_b200.beam import beam_select
    from leat_b200.logprobs import token_logprobs

    logits = _logits(2, vocab, "float32", 4, device)
    logits[:, 5], logits[:, 200], logits[:, 290] = torch.finfo(torch.float32).max, INF, torch.finfo(torch.float32).max
    for top in (1, 2, 3):
        _check_top(token_logprobs(logits, top=top), logits.double().cpu().numpy(), top)
    scores = torch.tensor([[0.0, -0.5]], device=device)
    plain.check_selected(beam_select(logits, scores, 3), logits.double().cpu().numpy(), scores.cpu().numpy(), 3, exact_order=True)


@pytest.mark.parametrize("vocab", [300, 9001])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_ranks_beyond_float32(device, vocab, sign):
    """Scores whose penalised ranks only 64 bits hold.  (Next to them logits count for nothing: a beam's
    continuations tie, and the larger logit goes first.)"""
    import torch

    from leat_b200.beam import beam_select

    logits = _logits(2, vocab, "float32", 5, device)
    scores = sign * torch.tensor([[2e38, 3e38]], device=device)
    lengths = torch.tensor([[50, 50]], dtype=torch.int32, device=device)
    for width in (1, 3):
        got = beam_select(logits, scores, width, lengths=lengths, length_penalty=-4.0)
        plain.check_selected(got, logits.double().cpu().numpy(), scores.cpu().numpy(), width, lengths=lengths.cpu().numpy(), alpha=-4.0,
                             exact_order=True)  # fmt: skip
