"""What beam_select refuses to write into: memory that the step reads, or that it writes twice."""

import numpy as np
import pytest

from tests import beam_reference as plain

pytestmark = pytest.mark.gpu


def test_outputs_that_overlap(device):
    import torch

    from leat_b200.beam import Selected, beam_select

    logits = torch.randn((6, 300), generator=torch.Generator().manual_seed(1)).to(device)
    floats, ints, bools = torch.zeros(64, device=device), torch.zeros(128, dtype=torch.int32, device=device), torch.zeros(64, dtype=torch.bool, device=device)
    view = lambda t, at, width=3: t[at:at + 2 * width].view(2, width)  # noqa: E731

    def call(scores=0, lengths=0, finished=0, tokens=16, parents=32, out_scores=16, out_lengths=48, out_finished=16):
        out = Selected(view(ints, tokens), view(ints, parents), view(floats, out_scores), view(bools, out_finished), view(ints, out_lengths))
        return beam_select(logits, view(floats, scores), finished=view(bools, finished), end_id=1, lengths=view(ints, lengths),
                           length_penalty=0.5, out=out)  # fmt: skip

    want = beam_select(logits, view(floats, 0), finished=view(bools, 0), end_id=1, lengths=view(ints, 0), length_penalty=0.5)
    for fine in (dict(), dict(scores=6, out_scores=0), dict(out_scores=6), dict(tokens=6, parents=12, out_lengths=18), dict(finished=16, out_finished=22)):
        floats.zero_(), ints.zero_(), bools.zero_()
        got = call(**fine)
        for name in ("tokens", "parents", "scores", "finished", "lengths"):
            assert torch.equal(getattr(got, name), getattr(want, name)), (fine, name)
    bad = [dict(out_scores=0), dict(out_scores=5), dict(scores=6, out_scores=1), dict(tokens=5), dict(lengths=40, out_lengths=44), dict(lengths=40, parents=35),
           dict(finished=16, out_finished=11), dict(finished=20, out_finished=16), dict(tokens=32), dict(tokens=30), dict(out_lengths=37)]  # fmt: skip
    for more in bad:
        with pytest.raises(ValueError, match="out must not"):
            call(**more)


def test_outputs_inside_the_logits(device):
    import torch

    from leat_b200.beam import Selected, beam_select

    held = torch.zeros(2 * 500 + 4, device=device)
    logits = held.as_strided((2, 500), (502, 1))
    ints = lambda: torch.zeros((1, 2), dtype=torch.int32, device=device)  # noqa: E731
    scores = torch.zeros((1, 2), device=device)
    for at in (0, 499, 502, 1000):
        with pytest.raises(ValueError, match="out must not"):
            beam_select(logits, scores, out=Selected(ints(), ints(), held[at:at + 2].view(1, 2)))
    behind = held[1002:1004].view(1, 2)
    got = beam_select(logits, scores, out=Selected(ints(), ints(), behind))
    plain.check_selected(got, np.zeros((2, 500)), np.zeros((1, 2)), 2, exact_order=True)


def test_an_earlier_result_as_what_the_next_step_reads(device):
    """More continuations than beams, the first of them taken as the next step's beams: what is read is a copy
    where it is not contiguous, and is refused as output where it is the same memory."""
    import torch

    from leat_b200.beam import Selected, beam_select

    logits = torch.randn((6, 300), generator=torch.Generator().manual_seed(2)).to(device)
    first = beam_select(logits, torch.zeros((2, 3), device=device), 6)
    scores = first.scores[:, :3]
    want = beam_select(logits, scores, 6)
    keep = [t.clone() for t in (want.tokens, want.parents, want.scores)]
    got = beam_select(logits, scores, 6, out=first)
    assert got is first
    for a, b in zip((got.tokens, got.parents, got.scores), keep):
        assert torch.equal(a, b)
    one = Selected(torch.zeros((1, 6), dtype=torch.int32, device=device), torch.zeros((1, 6), dtype=torch.int32, device=device), torch.zeros((1, 6), device=device))
    for at in (0, 2):
        with pytest.raises(ValueError, match="out must not"):
            beam_select(logits[:3], one.scores[:, at:at + 3], 6, out=one)
