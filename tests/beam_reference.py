"""Plain statements of beam search and of log-probabilities in 64 bits, on the CPU, for the tests."""

from __future__ import annotations

import numpy as np

# What float32 arithmetic may move a row's log-sum by, in half steps of float32 (2^-24, relative to a
# sum whose logarithm is taken, so absolute): a thread adds up to 32 exponentials one after the other
# (32); ex2 is good to two steps (4); its argument, -z log2 e for a logit z below the largest, is
# rounded once, and z averages at most ln V < 13 under the row's own probabilities (13 * 1.45 = 19);
# the constant log2 e is off by 2^-26 relative (z again: 5).  Everything after that is in 64 bits.
LOG_SUM_ERROR = 60 * 2.0**-24


def clean(logits):
    """Logits as 64-bit numbers: a NaN counts as -inf, +inf as the largest float32."""
    x = np.asarray(logits, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    return np.minimum(x, float(np.finfo(np.float32).max))


def log_softmax(logits):
    x = clean(logits)
    top = x.max(1, keepdims=True)
    safe = np.where(np.isneginf(top), 0.0, top)
    with np.errstate(divide="ignore", invalid="ignore"):
        out = (x - safe) - np.log(np.exp(x - safe).sum(1, keepdims=True))
    return np.where(np.isneginf(x), -np.inf, out)


def continuations(logits, scores, finished=None, end_id=None, lengths=None, alpha=0.0):
    """Every continuation of every group, best first: lists of (rank, beam, token, score, finished, length)."""
    groups, beams = scores.shape
    share = log_softmax(logits)
    x = clean(logits)
    out = []
    for g in range(groups):
        found = []
        for k in range(beams):
            s = float(scores[g, k])
            if not np.isfinite(s):
                continue
            done = finished is not None and bool(finished[g, k])
            length = (0 if lengths is None else int(lengths[g, k])) + (0 if done else 1)
            divide = ((5.0 + length) / 6.0) ** alpha if alpha else 1.0
            if done:
                found.append((s / divide, k, 0.0, end_id, s, True, length))
                continue
            row = g * beams + k
            for t in np.nonzero(~np.isneginf(share[row]))[0]:
                score = s + share[row, t]
                found.append((score / divide, k, x[row, t], int(t), score, end_id is not None and int(t) == end_id, length))
        found.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
        out.append(found)
    return out


def check_selected(got, logits, scores, width, finished=None, end_id=None, lengths=None, alpha=0.0, exact_order=False):
    """A beam_select result against the continuations in 64 bits.  Ids have to be equal wherever the
    neighbouring ranks are further apart than both sides' errors; with exact_order everywhere."""
    groups, beams = scores.shape
    tokens, parents = got.tokens.cpu().numpy(), got.parents.cpu().numpy()
    values = got.scores.cpu().numpy().astype(np.float64)
    ended = None if got.finished is None else got.finished.cpu().numpy()
    length = None if got.lengths is None else got.lengths.cpu().numpy()
    assert tokens.shape == parents.shape == values.shape == (groups, width)
    for g, found in enumerate(continuations(logits, scores, finished, end_id, lengths, alpha)):
        by_name = {(c[1], c[3]): c for c in found}
        n = min(width, len(found))
        names = list(zip(parents[g, :n].tolist(), tokens[g, :n].tolist()))
        assert len(set(names)) == n, f"group {g}: a continuation twice"
        for j in range(n):
            want = found[j]
            assert names[j] in by_name, f"group {g}, place {j}: {names[j]} is no continuation"
            mine = by_name[names[j]]
            # its own score, rounded once; and its rank is the j-th best's, but for the errors
            assert abs(values[g, j] - mine[4]) <= LOG_SUM_ERROR + abs(mine[4]) * 2.0**-24, (g, j, values[g, j], mine)
            assert abs(mine[0] - want[0]) <= 2 * LOG_SUM_ERROR, (g, j, mine, want)
            near = [i for i in (j - 1, j + 1) if 0 <= i < len(found) and abs(found[i][0] - want[0]) <= 2 * LOG_SUM_ERROR]
            if exact_order or not near:
                assert names[j] == (want[1], want[3]), (g, j, names[j], want)
            if ended is not None:
                assert bool(ended[g, j]) == mine[5]
            if length is not None:
                assert int(length[g, j]) == mine[6]
        for j in range(n, width):
            assert tokens[g, j] == -1 and parents[g, j] == j % beams and values[g, j] == -np.inf
            assert ended is None or not ended[g, j]
            assert length is None or length[g, j] == 0


def sequences(tokens, parents, end_id=None):
    """tokens and parents (T, G, K) -> (G, K, T) and (G, K), walked back from the last step."""
    steps, groups, beams = tokens.shape
    out = np.full((groups, beams, steps), -1, np.int64)
    lengths = np.full((groups, beams), steps, np.int64)
    for g in range(groups):
        for k in range(beams):
            b = k
            for t in range(steps - 1, -1, -1):
                out[g, k, t] = tokens[t, g, b]
                b = parents[t, g, b]
                if not 0 <= b < beams:
                    break
            ends = np.nonzero(out[g, k] == end_id)[0] if end_id is not None else []
            if len(ends):
                lengths[g, k] = ends[0] + 1
                out[g, k, ends[0]:] = end_id
    return out, lengths
