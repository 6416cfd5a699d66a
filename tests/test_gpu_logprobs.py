"""token_logprobs on the GPU against log-probabilities in 64 bits."""

import numpy as np
import pytest

from tests import beam_reference as plain

pytestmark = pytest.mark.gpu


def _check(got, logits, ids, top):
    share, x = plain.log_softmax(logits), plain.clean(logits)
    rows, vocab = share.shape

    def close(a, b):
        a = a.astype(np.float64)
        assert np.array_equal(np.isneginf(a), np.isneginf(b))
        fine = ~np.isneginf(b)
        assert (np.abs(a[fine] - b[fine]) <= plain.LOG_SUM_ERROR + np.abs(b[fine]) * 2.0**-24).all()

    if ids is not None:
        ids = ids.reshape(rows, -1)
        inside = (ids >= 0) & (ids < vocab)
        close(got.logprobs.cpu().numpy(), np.where(inside, np.take_along_axis(share, np.where(inside, ids, 0), 1), -np.inf))
    if top:
        n = min(top, vocab)
        order = np.argsort(-x, axis=1, kind="stable")[:, :n]
        values = np.take_along_axis(share, order, 1)
        order = np.where(np.isneginf(values), -1, order)
        np.testing.assert_array_equal(got.top_ids.cpu().numpy(), np.pad(order, ((0, 0), (0, top - n)), constant_values=-1))
        close(got.top_logprobs.cpu().numpy(), np.pad(values, ((0, 0), (0, top - n)), constant_values=-np.inf))


@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab,given,top,pad", [
    (1, 1, 1, 1, 0), (3, 7, 2, 20, 0), (5, 1000, 1, 0, 0), (4, 8192, 1, 5, 8), (2, 8193, 3, 64, 0), (9, 33333, 1, 20, 1),
    (300, 2000, 1, 5, 0), (2, 150000, 0, 40, 0), (6, 16384, 4, 1, 4),
])  # fmt: skip
def test_sizes_types_and_strides(device, kind, rows, vocab, given, top, pad):
    import torch

    from leat_b200.logprobs import token_logprobs

    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn((rows, vocab + pad), generator=g) * 3).to(getattr(torch, kind)).to(device)[:, :vocab]
    ids = torch.randint(-1, vocab + 1, (rows, given), generator=g, dtype=torch.int32) if given else None
    got = token_logprobs(logits, None if ids is None else ids.to(device), top)
    _check(got, logits.double().cpu().numpy(), None if ids is None else ids.numpy(), top)
    if given == 1:  # the shapes a sampler's ids come in, and 64-bit ids
        for other in (ids[:, 0], ids.long(), ids[:, 0].long()):
            again = token_logprobs(logits, other.to(device))
            assert again.logprobs.shape == (rows, 1) and torch.equal(again.logprobs, got.logprobs)


@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [500, 9001, 40000])
def test_masks_ties_and_infinities(device, kind, vocab):
    import torch

    from leat_b200.logprobs import token_logprobs

    logits = (torch.randn((9, vocab), generator=torch.Generator().manual_seed(1)) * 2).to(getattr(torch, kind)).to(device)
    logits[0] = float("-inf")
    logits[1] = torch.finfo(logits.dtype).min
    logits[2, 10:] = float("-inf")
    logits[3] = 1.5
    logits[4, ::2] = float("nan")
    logits[5, 7] = float("inf")
    logits[6, 10:] = torch.finfo(logits.dtype).min
    logits[7] = torch.randint(0, 2, (vocab,), generator=torch.Generator().manual_seed(2)).to(logits.dtype).to(device)
    logits[8] = float("nan")
    ids = torch.arange(9, dtype=torch.int32).reshape(9, 1).expand(9, 3) + torch.tensor([0, 2, 100], dtype=torch.int32)
    got = token_logprobs(logits, ids.to(device), 64)
    _check(got, logits.double().cpu().numpy(), ids.numpy(), 64)


def test_more_rows_than_a_grid_is_high(device):
    import torch

    from leat_b200.logprobs import token_logprobs

    rows = 70001
    logits = torch.randn((rows, 40), generator=torch.Generator().manual_seed(5)).to(device)
    ids = torch.randint(0, 40, (rows, 1), generator=torch.Generator().manual_seed(6), dtype=torch.int32)
    _check(token_logprobs(logits, ids.to(device), 3), logits.double().cpu().numpy(), ids.numpy(), 3)


def test_more_given_ids_than_a_warp(device):
    import torch

    from leat_b200.logprobs import token_logprobs

    logits = torch.randn((5, 700), generator=torch.Generator().manual_seed(7)).to(device)
    ids = torch.randint(-2, 702, (5, 75), generator=torch.Generator().manual_seed(8), dtype=torch.int32)
    for top in (0, 2, 30):
        _check(token_logprobs(logits, ids.to(device), top), logits.double().cpu().numpy(), ids.numpy(), top)


def test_ids_beyond_32_bits_are_outside(device):
    import torch

    from leat_b200.logprobs import token_logprobs

    logits = torch.zeros((2, 10), device=device)
    got = token_logprobs(logits, torch.tensor([1 << 32, -(1 << 32)], device=device))
    assert bool(torch.isneginf(got.logprobs).all())


def test_after_sampling_and_captured(device):
    """The ids sample() has just drawn, in one graph with it."""
    import torch

    from leat_b200.logprobs import token_logprobs
    from leat_b200.sampler import Sampler

    logits = torch.randn((6, 32000), generator=torch.Generator().manual_seed(3)).to(device) * 3
    options = torch.tensor([[0.8, 40, 0.95, 0.0, 0.0]], device=device)
    seed = torch.arange(6, device=device).to(torch.uint32)
    sampler = Sampler(6, 32000, 64, device)
    sampler.sample(logits, options, seed, 5)
    token_logprobs(logits, top=5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids = sampler.sample(logits, options, seed, 5)
        got = token_logprobs(logits, ids, top=5)
    graph.replay()
    torch.cuda.synchronize()
    _check(got, logits.double().cpu().numpy(), ids.cpu().numpy(), 5)


def test_nothing_asked_and_refusals(device):
    import torch

    from leat_b200.logprobs import token_logprobs

    logits = torch.zeros((3, 50), device=device)
    ids = torch.zeros((3, 1), dtype=torch.int32, device=device)
    assert token_logprobs(logits).logprobs is None
    assert token_logprobs(logits, ids[:, :0]).logprobs.shape == (3, 0)
    assert token_logprobs(logits[:0], ids[:0], 4).top_ids.shape == (0, 4)
    bad = [dict(logits=logits.cpu()), dict(logits=logits.double()), dict(logits=logits[0]), dict(logits=logits[:, :0]), dict(ids=ids.float()),
           dict(ids=ids.cpu()), dict(ids=ids[:2]), dict(ids=ids.reshape(3, 1, 1)), dict(top=-1), dict(top=65), dict(top=True), dict(top=1.0)]  # fmt: skip
    for more in bad:
        with pytest.raises(ValueError):
            token_logprobs(**{"logits": logits, "ids": ids, **more})
