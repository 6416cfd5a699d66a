"""Calls from several host threads at once, each on a stream of its own: they share nothing."""

import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _at_once(jobs, rounds):
    """Runs every job, a call of the C library (which runs without the interpreter's lock) that returns its
    code, in a thread of its own, and returns how often each failed."""
    failed = [0] * len(jobs)
    ready = threading.Barrier(len(jobs))

    def work(i, call):
        ready.wait()
        for _ in range(rounds):
            if call() != 0:
                failed[i] += 1

    threads = [threading.Thread(target=work, args=(i, call)) for i, call in enumerate(jobs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return failed


def test_reorders_of_different_sizes(device):
    """64 beams want more shared memory than 24: neither's call may set what the other's launch may ask for."""
    import torch

    from leat_b200 import _lib

    held, jobs = [], []
    for beams in (64, 24, 48, 28, 64, 32):
        state = torch.arange(beams * 16, dtype=torch.int32, device=device).reshape(beams, 16)
        parents = torch.arange(beams, dtype=torch.int32, device=device).flip(0).contiguous()
        stream = torch.cuda.Stream()
        args = (_lib.State * 1)(_lib.State(data=state.data_ptr(), row_stride=64, outer_stride=0, place_bytes=64, outer=1, places=1, rows=beams))
        held.append((state, state.clone(), parents, stream, args))

        def call(args=args, parents=parents.data_ptr(), beams=beams, stream=stream.cuda_stream):
            return _lib.lib.leat_reorder_states(args, 1, parents, None, 1, beams, None, 0, None, 1, stream)

        jobs.append(call)
    torch.cuda.synchronize()
    assert _at_once(jobs, 2001) == [0] * len(jobs)
    torch.cuda.synchronize()
    for state, before, *_ in held:
        assert torch.equal(state, before.flip(0))


def test_sequences_of_different_lengths(device):
    import torch

    from leat_b200 import _lib

    held, jobs = [], []
    rng = np.random.default_rng(1)
    for steps, beams in ((1200, 64), (700, 48), (5000, 64), (800, 64), (1000, 56), (5000, 61)):
        tokens = torch.tensor(rng.integers(0, 1000, (steps, 1, beams)), dtype=torch.int32, device=device)
        parents = torch.arange(beams, dtype=torch.int32, device=device).expand(steps, 1, beams).contiguous()
        out = torch.zeros((1, beams, steps), dtype=torch.int32, device=device)
        lengths = torch.zeros((1, beams), dtype=torch.int32, device=device)
        stream = torch.cuda.Stream()
        held.append((tokens, parents, out, lengths, stream))

        def call(at=(tokens.data_ptr(), parents.data_ptr(), steps, 1, beams, -1, out.data_ptr(), lengths.data_ptr()), stream=stream.cuda_stream):
            return _lib.lib.leat_beam_sequences(*at, stream)

        jobs.append(call)
    torch.cuda.synchronize()
    assert _at_once(jobs, 1000) == [0] * len(jobs)
    torch.cuda.synchronize()
    for tokens, _, out, lengths, _ in held:
        assert torch.equal(out[0], tokens[:, 0].t()) and bool((lengths == tokens.shape[0]).all())
