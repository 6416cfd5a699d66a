"""The calls by torch's public entry points alone: what they come to where torch has not the inner ones."""

import pytest

pytestmark = pytest.mark.gpu


def test_without_the_inner_entries(device, monkeypatch):
    import torch

    from leat_b200 import beam, logprobs

    g = torch.Generator().manual_seed(1)
    logits = torch.randn((6, 9001), generator=g).to(device)
    scores = -torch.rand((2, 3), generator=g).to(device)
    lengths = torch.full((2, 3), 4, dtype=torch.int32, device=device)
    ids = torch.arange(6, dtype=torch.int32, device=device)
    state = torch.randn((6, 40), generator=g).to(device)

    def run():
        r = beam.beam_select(logits, scores, 5, end_id=2, lengths=lengths, length_penalty=0.5)
        moved = state.clone()
        beam.reorder_states(moved, r.parents[:, :3])
        s = beam.beam_sequences(r.tokens.unsqueeze(0), torch.zeros_like(r.parents).unsqueeze(0))
        p = logprobs.token_logprobs(logits, ids, 4)
        return r.tokens, r.parents, r.scores, r.finished, r.lengths, moved, s.tokens, s.lengths, p.logprobs, p.top_logprobs, p.top_ids

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = run()
        for module in (beam, logprobs):
            monkeypatch.setattr(module, "empty_strided", logprobs.plain_empty_strided)
            monkeypatch.setattr(module, "raw_stream", logprobs.plain_raw_stream)
        got = run()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and a.device == b.device and a.stride() == b.stride() and torch.equal(a, b)
