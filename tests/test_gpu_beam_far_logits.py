"""Logits further below their row's largest than float32 holds, next to one another through their beams' length
penalties."""

import numpy as np
import pytest

from tests import beam_reference as plain

pytestmark = pytest.mark.gpu


def _check(logits, scores, lengths, alpha, width, device):
    """The 64-bit order, ranks as good as equal (2^-40) apart: what is ranked lies so far down that the sums'
    errors are nothing next to it, but for the likeliest tokens, one a beam, which come first."""
    import torch

    from leat_b200.beam import beam_select

    beams = scores.shape[1]
    got = beam_select(logits, scores, width, lengths=lengths, length_penalty=alpha)
    found = plain.continuations(logits.double().cpu().numpy(), scores.cpu().numpy(), lengths=lengths.cpu().numpy(), alpha=alpha)[0]
    names = list(zip(got.parents[0].tolist(), got.tokens[0].tolist()))
    assert sorted(names[:beams]) == sorted((c[1], c[3]) for c in found[:beams])
    exact = {(c[1], c[3]): c[0] for c in found}
    assert len(set(names)) == width
    for j in range(beams, width):
        assert abs(exact[names[j]] - found[j][0]) <= 2.0**-40 * abs(found[j][0]), (j, names[j], exact[names[j]], found[j])
    values = got.scores[0, beams:].cpu().numpy()
    with np.errstate(over="ignore"):  # (a score beyond float32's range is -inf)
        want = np.array([c[4] for c in found[beams:width]], np.float64).astype(np.float32)
    assert torch.isfinite(got.scores[0, :beams]).all() and np.array_equal(np.isfinite(values), np.isfinite(want))


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [85, 9001])
@pytest.mark.parametrize("alpha", [1.0, 2.0, -1.0])
def test_the_lowest_value_below_an_infinity(device, kind, vocab, alpha):
    """A token forced by +inf while the others are masked by the type's lowest value: twice the range apart."""
    import torch

    logits = torch.randn((5, vocab), generator=torch.Generator().manual_seed(1)).to(getattr(torch, kind)).to(device)
    lowest = torch.finfo(logits.dtype).min
    logits[:, 20:] = lowest
    for k in range(5):
        logits[k, 3 * k + 1] = float("inf")
    logits[1, 2:12], logits[3, 30] = lowest / 2, lowest / 4
    scores = torch.tensor([[-1.0, -2.0, -0.5, -30.0, 0.0]], device=device)
    lengths = torch.tensor([[1, 90, 12000, 450000000, 7]], dtype=torch.int32, device=device)
    for width in (8, 40, 64):
        _check(logits, scores, lengths, alpha, width, device)


@pytest.mark.parametrize("alpha", [0.0, 0.5])
def test_differences_around_the_largest_float(device, alpha):
    import torch

    top = float(np.finfo(np.float32).max)
    logits = torch.linspace(-1.0, 0.6, 200, device=device).repeat(4, 1) * top
    logits[:, 7] = torch.tensor([1.0, 0.7, 0.1, 1.0], device=device) * top
    scores = torch.tensor([[0.0, -1.0, -2.0, -3.0]], device=device)
    lengths = torch.tensor([[3, 5, 1000, 100]], dtype=torch.int32, device=device)
    logits[2] = logits[2] * 0.1
    _check(logits, scores, lengths, alpha, 64, device)
