"""Nothing here has a backward pass: logits and scores that a gradient is wanted of are refused, not cut off from
it without a word.  (The check comes before any look at the device.)"""

import pytest
import torch

from leat_b200 import beam_select, token_logprobs


def test_gradients_are_refused():
    logits, scores = torch.zeros((6, 10), requires_grad=True), torch.zeros((2, 3))
    with pytest.raises(ValueError, match="gradient"):
        token_logprobs(logits, torch.zeros(6, dtype=torch.int32))
    with pytest.raises(ValueError, match="gradient"):
        beam_select(logits, scores)


@pytest.mark.gpu
def test_gradients_that_are_off(device):
    from leat_b200.beam import BeamSearch

    logits = torch.randn((6, 500), device=device).requires_grad_()
    scores = torch.zeros((2, 3), device=device)
    ids = torch.zeros(6, dtype=torch.int32, device=device)
    for call in (lambda: token_logprobs(logits, ids), lambda: beam_select(logits, scores), lambda: BeamSearch(2, 3, 2, device=device).step(logits),
                 lambda: beam_select(logits.detach(), scores.clone().requires_grad_())):  # fmt: skip
        with pytest.raises(ValueError, match="gradient"):
            call()
    want = token_logprobs(logits.detach(), ids).logprobs
    with torch.no_grad():
        assert torch.equal(token_logprobs(logits, ids).logprobs, want)
        beam_select(logits, scores.clone().requires_grad_())
    with torch.inference_mode():
        assert torch.equal(token_logprobs(logits, ids).logprobs, want)
        assert torch.equal(beam_select(logits, scores).tokens, beam_select(logits.detach(), scores).tokens)
