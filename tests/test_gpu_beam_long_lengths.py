"""Length penalties of long sequences: the float32 ranks that leave continuations out are furthest from the exact
ones where the lengths are long, the exponent is large and what is ranked lies far below its beam's score."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("alpha", [4.0, 2.5, 1.0, -1.0, -4.0])
@pytest.mark.parametrize("vocab", [64, 9000, 150000])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_close_ranks_of_beams_of_very_different_lengths(device, alpha, vocab, seed):
    """Every beam's likeliest token has all the probability and a rank of zero; the others, a few tokens of each
    beam, have ranks that differ by steps of 2^-18 of themselves and by their logits' rounding.  Their order is
    that of the 64-bit ranks (logit / penalty: the sums are 1 to the last bit); both sides' penalties are good to
    2^-50, which 2^-40 leaves room for."""
    import torch

    from leat_b200.beam import beam_select

    rng = np.random.default_rng(seed)
    beams, width = 12, 40
    lengths = np.unique(np.concatenate([[0, 1, 2**31 - 2], (2.0 ** rng.uniform(1, 31, 30)).astype(np.int64)]))
    lengths = rng.permutation(lengths)[:beams].astype(np.int32)
    divide = ((5.0 + lengths.astype(np.float64) + 1) / 6.0) ** alpha
    logits = np.full((beams, vocab), -np.inf, np.float32)
    unit = max(1.0, 200.0 / divide.min())  # far enough below the likeliest token to count for nothing in the sum
    found = []
    for k in range(beams):
        tokens = rng.permutation(vocab - 1)[:20] + 1
        logits[k, tokens] = -unit * divide[k] * (1 + 2.0**-18 * rng.permutation(64)[:20])
        logits[k, 0] = 0.0
        found += [(logits[k, t].astype(np.float64) / divide[k], k, int(t)) for t in [0, *tokens]]
    found.sort(key=lambda c: (-c[0], c[1]))
    ranks = np.array([c[0] for c in found[beams:]])
    assert (np.abs(logits[np.isfinite(logits)]) < 3e38).all()
    got = beam_select(torch.tensor(logits, device=device), torch.zeros((1, beams), device=device), width,
                      lengths=torch.tensor(lengths.reshape(1, -1), device=device), length_penalty=alpha)  # fmt: skip
    names = list(zip(got.parents[0].tolist(), got.tokens[0].tolist()))
    assert names[:beams] == [(k, 0) for k in range(beams)]
    exact = {(c[1], c[2]): c[0] for c in found}
    for j in range(beams, width):
        assert names[j] in exact, (j, names[j])
        # the j-th best rank itself, whichever of two as good as equal ones stands there
        assert abs(exact[names[j]] - ranks[j - beams]) <= 2.0**-40 * abs(ranks[j - beams]), (j, names[j], found[j])
    assert len(set(names)) == width
