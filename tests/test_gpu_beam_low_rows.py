"""Rows of logits around -1000, where the float32 sums stop taking a chunk's word for the row's range: every
chunk counts, whichever side of it the chunk lies on and whichever comes first."""

import numpy as np
import pytest

from tests import beam_reference as plain

pytestmark = pytest.mark.gpu


def _check(logits, scores, device):
    import torch

    from leat_b200.beam import beam_select
    from leat_b200.logprobs import token_logprobs

    exact = logits.double().cpu().numpy()
    share = plain.log_softmax(exact)
    ids = torch.arange(logits.shape[0], dtype=torch.int32, device=device).reshape(-1, 1)
    got = token_logprobs(logits, ids, 3)
    want = np.take_along_axis(share, ids.cpu().numpy().astype(np.int64), 1)
    assert (np.abs(got.logprobs.cpu().numpy() - want) <= plain.LOG_SUM_ERROR + np.abs(want) * 2.0**-24).all()
    plain.check_selected(beam_select(logits, scores, 4), exact, scores.cpu().numpy(), 4)


@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [300, 9000, 9001, 40000])
@pytest.mark.parametrize("centre", [-1012.0, -1008.0, -1003.0, -996.0, -900.0, -899.0])
def test_rows_across_the_border(device, kind, vocab, centre):
    import torch

    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn((4, vocab), generator=g) * 3 + centre).to(getattr(torch, kind)).to(device)
    _check(logits, torch.tensor([[0.0, -0.5], [-0.25, -0.5]], device=device), device)


@pytest.mark.parametrize("low,high", [(-1000.0, -999.5), (-1001.0, -999.0), (-1000.5, -950.0), (-1050.0, -999.0), (-1000.0, -901.0), (-1000.0, -899.0)])
@pytest.mark.parametrize("where", [0, 128, 512, 3000, 4095])
def test_one_chunk_above_the_border(device, low, high, where):
    """A few logits above the rest, in the first chunk, a later one, the last of the tile."""
    import torch

    logits = torch.full((2, 8192), low, device=device)
    logits += torch.rand((2, 8192), generator=torch.Generator().manual_seed(where)).to(device) * 0.25 - 0.25
    logits[:, where], logits[1, 8000] = high, high
    _check(logits, torch.tensor([[0.0, -1.0]], device=device), device)
