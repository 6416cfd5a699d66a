"""Beam search on the device: the selection over beams and vocabulary, the caches and other states that
follow their beams, and the sequences read back at the end.  leat decodes one sequence per request; this
serves requests that ask for the best of several.

`BeamSearch` runs a batch of searches step by step; `beam_select`, `reorder_states` and
`beam_sequences` are its parts.  Nothing here waits for the device or copies to the host, and a call's
scratch is its own, so every part can be captured into a CUDA graph, and a search as a whole; a single
step of a `BeamSearch` cannot be captured and replayed for the others (the class says why)."""

from __future__ import annotations

from dataclasses import dataclass
from math import prod
from struct import pack

import torch

from leat_b200 import _lib
from leat_b200.logprobs import FORMATS, empty_strided, raw_stream, rows_of_logits, scratch

MAX_BEAMS = 64
MAX_WIDTH = 64
SELECT_ARGS = "PiiiiqIiPPPf4xPPPPPPN"  # struct leat_beam_args
STATE_REST = "qqqiiiI"  # struct leat_state behind its address, with the padding at its end


@dataclass
class Selected:
    """The continuations of a step, (G, width) each, best first."""

    tokens: torch.Tensor  # int32; -1 where a group has no further continuation
    parents: torch.Tensor  # int32: the beam of the group that each continues
    scores: torch.Tensor  # float32: summed log-probabilities; -inf where there is none
    finished: torch.Tensor | None = None  # bool: the sequence has ended (with end_id)
    lengths: torch.Tensor | None = None  # int32: tokens so far, the end token included (with lengths)


@dataclass
class Sequences:
    tokens: torch.Tensor  # (G, K, T) int32
    lengths: torch.Tensor  # (G, K) int32: tokens up to the first end token, which is included


def _whole(x, dtype, shape, device, name: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor) or x.dtype != dtype or x.shape != shape or x.device != device:
        raise ValueError(f"{name} must be a {tuple(shape)} {str(dtype).removeprefix('torch.')} tensor on {device}")
    return x if x.is_contiguous() else x.contiguous()


def beam_select(logits, scores: torch.Tensor, width: int | None = None, *, finished: torch.Tensor | None = None,
                end_id: int | None = None, lengths: torch.Tensor | None = None, length_penalty: float = 0.0,
                out: Selected | None = None) -> Selected:  # fmt: skip
    """The `width` (1..64, default K) best continuations of each of G groups of K beams (up to 64).

    logits (G * K, V) float32, bfloat16 or float16, row g * K + k for beam k of group g; scores (G, K)
    float32, what each beam's tokens add up to.  A beam continues with any token whose logit is above
    -inf, to its score plus the token's log-probability; a beam of score -inf (or NaN) is dead and
    continues with nothing (the first step of a search has one live beam per group, the others dead).
    With `end_id`, a beam marked in `finished` (G, K) bool goes on as itself: one continuation, end_id,
    its score unchanged; its logits are not read.  With `lengths` (G, K) int32, continuations are ranked
    by score / ((5 + length) / 6) ** length_penalty (Wu et al. 2016) over their own lengths.  Equal
    ranks: the lower beam, then the larger logit, then the lower token.  Ranks are held in 64 bits.

    Masks are the caller's: set a forbidden token's logit to -inf (or the type's lowest value, which
    makes it the last resort).  A row with nothing left has no continuations; a group with too few of
    them has tokens of -1 and scores of -inf in the last places, with their own place as parent.
    There is no backward pass: logits and scores that a gradient is wanted of are refused (detach them, or
    call under torch.no_grad()).
    `out`: a Selected of an earlier call (or of your own contiguous tensors) to write into; it shares no
    memory with what the call reads."""
    logits = rows_of_logits(logits)
    dev = logits.device
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return beam_select(logits, scores, width, finished=finished, end_id=end_id, lengths=lengths, length_penalty=length_penalty, out=out)
    rows, vocab = logits.shape
    if not isinstance(scores, torch.Tensor) or scores.dim() != 2:
        raise ValueError("scores must be a (G, K) float32 tensor")
    if scores.requires_grad and torch.is_grad_enabled():
        raise ValueError("no gradient flows through this call: detach the scores, or call under torch.no_grad()")
    shape = scores.shape
    groups, beams = shape
    scores = _whole(scores, torch.float32, shape, dev, "scores")
    if not 1 <= beams <= MAX_BEAMS or groups * beams != rows:
        raise ValueError(f"logits must have a row per beam of scores (G, K), K from 1 to {MAX_BEAMS}")
    if width is None:
        width = beams
    elif type(width) is not int or not 1 <= width <= MAX_WIDTH:
        raise ValueError(f"width must be an integer from 1 to {MAX_WIDTH}")
    done_at = lengths_at = ended_at = new_lengths_at = 0
    if end_id is not None:
        if type(end_id) is not int or not 0 <= end_id < vocab:
            raise ValueError("end_id must be a token of the vocabulary")
        if finished is not None:
            finished = _whole(finished, torch.bool, shape, dev, "finished")
            done_at = finished.data_ptr()
    elif finished is not None:
        raise ValueError("finished beams continue with end_id: give one")
    if lengths is not None:
        lengths = _whole(lengths, torch.int32, shape, dev, "lengths")
        lengths_at = lengths.data_ptr()
        if not -4.0 <= length_penalty <= 4.0:
            raise ValueError("length_penalty must be a number from -4 to 4")
    elif length_penalty != 0.0:
        raise ValueError("length_penalty needs the beams' lengths")
    if out is None:
        size, stride = (groups, width), (width, 1)
        out = Selected(empty_strided(size, stride, torch.int32), empty_strided(size, stride, torch.int32), empty_strided(size, stride, torch.float32),
                       None if end_id is None else empty_strided(size, stride, torch.bool),
                       None if lengths is None else empty_strided(size, stride, torch.int32))  # fmt: skip
    else:
        wanted = [(out.tokens, torch.int32), (out.parents, torch.int32), (out.scores, torch.float32)]
        wanted += [(out.finished, torch.bool)] if end_id is not None else []
        wanted += [(out.lengths, torch.int32)] if lengths is not None else []
        # groups write while others still read: the logits (their padding included), the beams', one another's
        at, scores_at = logits.data_ptr(), scores.data_ptr()
        taken = [(at, at + ((rows - 1) * logits.stride(0) + vocab) * logits.element_size()), (scores_at, scores_at + 4 * rows),
                 (lengths_at, lengths_at + 4 * rows), (done_at, done_at + rows)]  # fmt: skip
        for t, dtype in wanted:
            if t is None or t.dtype != dtype or t.shape != (groups, width) or t.device != dev or not t.is_contiguous():
                raise ValueError(f"out must hold contiguous ({groups}, {width}) tensors on {dev}, of the types of a Selected")
            begin = t.data_ptr()
            end = begin + groups * width * (1 if dtype == torch.bool else 4)
            for low, high in taken:
                if begin < high and low < end:
                    raise ValueError("out must not be, or overlap, what the step reads or another of its outputs")
            taken.append((begin, end))
    if groups == 0:
        return out
    if end_id is not None:
        ended_at = out.finished.data_ptr()
    if lengths is not None:
        new_lengths_at = out.lengths.data_ptr()
    held, at, size = scratch(rows, vocab, width)
    a = pack(SELECT_ARGS, logits.data_ptr(), groups, beams, vocab, width, logits.stride(0), FORMATS[logits.dtype], -1 if end_id is None else end_id,
             scores.data_ptr(), done_at, lengths_at, length_penalty, out.tokens.data_ptr(), out.parents.data_ptr(), out.scores.data_ptr(),
             ended_at, new_lengths_at, at, size)  # fmt: skip
    code = _lib.lib.leat_beam_select(a, raw_stream(dev.index))
    if code != _lib.OK:
        _lib.check(code, "leat_beam_select")
    return out


def _state(t: torch.Tensor, dim: int | None) -> tuple:
    """A tensor as leat_state has it behind its address: the bytes from row to row, from run to run of its
    places and of a place, and how many runs, places and rows there are."""
    shape, stride, size = t.shape, t.stride(), t.element_size()
    if dim is None:
        if t.dim() == 1:
            return (stride[0] * size, 0, size, 1, 1, shape[0])
        dim = 1
        places_are_all = True
    else:
        places_are_all = False
    # a place is everything behind `dim`, a run its places: both must lie back to back
    inner = 1
    for i in range(t.dim() - 1, dim, -1):
        if shape[i] != 1 and stride[i] != inner:
            raise ValueError("the dimensions behind the places' must be contiguous")
        inner *= shape[i]
    places = shape[dim]
    if places > 1 and stride[dim] != inner:
        raise ValueError("places must lie back to back")
    # the dimensions between the rows' and the places' make one run after another of one stride
    outer, outer_stride = 1, 0
    for i in range(dim - 1, 0, -1):
        if shape[i] == 1:
            continue
        if outer == 1:
            outer_stride = stride[i]
        elif stride[i] != outer_stride * outer:
            raise ValueError("the dimensions between rows and places must have one common stride")
        outer *= shape[i]
    if places_are_all:
        inner, places = inner * places, 1
    return (stride[0] * size, outer_stride * size, inner * size, outer, places, shape[0])


def _overlaps(row_stride: int, outer_stride: int, place_bytes: int, outer: int, places: int, rows: int) -> bool:
    run = place_bytes * places
    if rows < 2:
        return outer > 1 and outer_stride < run
    if outer < 2:
        return row_stride < run
    rows_outside = outer_stride >= run and row_stride >= outer_stride * (outer - 1) + run
    rows_inside = row_stride >= run and outer_stride >= row_stride * (rows - 1) + run
    return not (rows_outside or rows_inside)


def _range_end(x, default: int, groups: int, device, name: str):
    """A bound of the places: (pointer or None, value for all groups, what to keep until the launch)."""
    if x is None:
        return None, default, None
    if type(x) is int and x >= 0:
        return None, min(x, 0x7FFFFFFF), None
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name} must be a number of places, or a ({groups},) int32 tensor of them")
    x = _whole(x, torch.int32, (groups,), device, name)
    return x.data_ptr(), 0, x


def reorder_states(states, parents: torch.Tensor, *, slots: torch.Tensor | None = None, dim: int | None = None,
                   start=0, length=None) -> None:  # fmt: skip
    """Makes per-beam states follow their beams, in place: in every tensor of `states`, the row of beam k
    of group g takes what the row of beam parents[g, k] held.  Rows that keep their place are not touched.

    states: a tensor or a list of them, of any type, rows first, no two of the same memory; row g * K + k
    belongs to beam k of group g, or row slots[g, k] where `slots` (G, K) int32 is given (cache slots; all
    different: the rows of a slot that two beams share are either's).  parents (G, K)
    int32, K up to 64, as beam_select returns them.

    `dim`: the dimension that counts positions, the same in every tensor (a cache (rows, heads,
    positions, size) has 2, a cache (rows, positions, heads, size) has 1); then only positions `start`
    to `length` follow, each an int or a (G,) int32 tensor on the device: positions before `start` (a
    prompt that the beams share) and from `length` on stay as they are.  The places of a row, and what
    lies behind `dim`, must be back to back.  Without `dim` whole rows follow.

    Parents outside 0..K-1 and slots outside the tensor leave their row as it is."""
    states = [states] if isinstance(states, torch.Tensor) else list(states)
    if not isinstance(parents, torch.Tensor) or parents.dim() != 2 or not parents.is_cuda:
        raise ValueError("parents must be a (G, K) int32 CUDA tensor")
    dev = parents.device
    index = dev.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(dev):
            return reorder_states(states, parents, slots=slots, dim=dim, start=start, length=length)
    groups, beams = parents.shape
    if parents.dtype != torch.int32:
        raise ValueError("parents must be a (G, K) int32 CUDA tensor")
    if not parents.is_contiguous():
        parents = parents.contiguous()
    if not 1 <= beams <= MAX_BEAMS or groups > 65535:
        raise ValueError(f"parents must be (G, K) with K from 1 to {MAX_BEAMS} and G up to 65535")
    slots_at = None
    if slots is not None:
        slots = _whole(slots, torch.int32, parents.shape, dev, "slots")
        slots_at = slots.data_ptr()
    start_at, start_all, end_at, end_all = None, 0, None, 0x7FFFFFFF
    if dim is not None:
        start_at, start_all, start = _range_end(start, 0, groups, dev, "start")
        end_at, end_all, length = _range_end(length, 0x7FFFFFFF, groups, dev, "length")
    elif length is not None or (start is not None and (isinstance(start, torch.Tensor) or start != 0)):
        raise ValueError("start and length count positions: say which dimension they are with dim")
    # a search's caches are mostly alike: what one comes to holds for the next of its shape and strides
    described: list[bytes] = []
    shape = dtype = stride = None
    plain = False  # the last was contiguous: the next is alike if it is, too
    for t in states:
        if not isinstance(t, torch.Tensor) or t.get_device() != index or t.requires_grad:
            raise ValueError(f"states must be tensors on {dev}, rows first, that need no gradient")
        if t.shape != shape or t.dtype != dtype or not (t.is_contiguous() if plain else t.stride() == stride):
            if t.layout is not torch.strided or t.dim() == 0:
                raise ValueError("states must be strided tensors with their rows as first dimension")
            if slots is None and t.shape[0] < groups * beams:
                raise ValueError("states must have a row per beam, or slots must say which rows are the beams'")
            if dim is not None and not 0 < dim < t.dim():
                raise ValueError("dim must be a dimension of every state, behind the rows'")
            if t.numel() == 0:
                continue
            shape, dtype, plain = t.shape, t.dtype, t.is_contiguous()
            if plain:
                place, run = prod(shape[dim + 1:]) if dim is not None else prod(shape[1:]), shape[dim] if dim is not None else 1
                outer, size = prod(shape[1:dim]) if dim is not None else 1, t.element_size()
                rest = pack(STATE_REST, outer * run * place * size, run * place * size, place * size, outer, run, shape[0], 0)
            else:
                stride = t.stride()
                like = _state(t, dim)
                if _overlaps(*like):
                    raise ValueError("the rows of a state must not overlap")
                rest = pack(STATE_REST, *like, 0)
        described.append(pack("P", t.data_ptr()) + rest)
    count = len(described)
    if count == 0 or groups == 0:
        return
    if count > 1 and len({d[:8] for d in described}) != count:
        raise ValueError("a state may only be given once: it would be reordered twice, at the same time")
    code = _lib.lib.leat_reorder_states(b"".join(described), count, parents.data_ptr(), slots_at, groups, beams,
                                        start_at, start_all, end_at, end_all, raw_stream(index))  # fmt: skip
    if code != _lib.OK:
        _lib.check(code, "leat_reorder_states")


def beam_sequences(tokens: torch.Tensor, parents: torch.Tensor, end_id: int | None = None) -> Sequences:
    """The sequences of the last step's beams: tokens and parents (T, G, K) int32, a step's beam_select
    results (width K) one behind the other -> tokens (G, K, T) and lengths (G, K).  With `end_id` a
    sequence's length ends with its first end token, and only end tokens stand behind it."""
    if not isinstance(tokens, torch.Tensor) or tokens.dim() != 3 or not tokens.is_cuda:
        raise ValueError("tokens must be a (T, G, K) int32 CUDA tensor")
    dev = tokens.device
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return beam_sequences(tokens, parents, end_id)
    steps, groups, beams = shape = tokens.shape
    tokens = _whole(tokens, torch.int32, shape, dev, "tokens")
    parents = _whole(parents, torch.int32, shape, dev, "parents")
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"there must be 1 to {MAX_BEAMS} beams")
    if end_id is not None and (isinstance(end_id, bool) or not isinstance(end_id, int) or not 0 <= end_id <= 0x7FFFFFFF):
        raise ValueError("end_id must be a token")
    shape = (groups, beams, steps)
    out = Sequences(empty_strided(shape, (beams * steps, steps, 1), torch.int32), empty_strided((groups, beams), (beams, 1), torch.int32))
    if groups:
        code = _lib.lib.leat_beam_sequences(tokens.data_ptr(), parents.data_ptr(), steps, groups, beams, -1 if end_id is None else end_id,
                                            out.tokens.data_ptr(), out.lengths.data_ptr(), raw_stream(dev.index))  # fmt: skip
        if code != _lib.OK:
            _lib.check(code, "leat_beam_sequences")
    return out


class BeamSearch:
    """G searches of K beams, step by step, up to `max_steps` tokens each, on one device and stream.

        search = BeamSearch(groups, beams, max_steps, end_id=end, length_penalty=0.6, device=device)
        for position in range(prompt, prompt + max_steps):
            logits = model(tokens, caches, position)              # (G * K, V)
            tokens = search.step(logits, caches, dim=2, start=prompt, length=position + 1)
        best = search.sequences()                                 # tokens (G, K, T), best beam first

    A step selects the beams' continuations, makes `states` follow their beams (reorder_states), and
    returns the tokens the beams run next.

    Steps are counted on the host: the count says which of two sets of beams a step reads and writes, and where
    its tokens go.  A captured step does that step again whenever it is replayed, so a graph takes a whole
    search, from reset() to sequences(), or one step of a known number."""

    def __init__(self, groups: int, beams: int, max_steps: int, *, end_id: int | None = None, length_penalty: float = 0.0, device=None):
        if groups <= 0 or not 1 <= beams <= MAX_BEAMS or max_steps <= 0:
            raise ValueError(f"groups and max_steps must be positive, beams from 1 to {MAX_BEAMS}")
        self.groups, self.beams, self.max_steps = groups, beams, max_steps
        self.end_id, self.length_penalty = end_id, length_penalty
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self._tokens = torch.empty((max_steps, groups, beams), dtype=torch.int32, device=self.device)
        self._parents = torch.empty((max_steps, groups, beams), dtype=torch.int32, device=self.device)
        # what a step reads and what it writes, in turn
        make = lambda: (torch.empty((groups, beams), dtype=torch.float32, device=self.device),  # noqa: E731
                        torch.zeros((groups, beams), dtype=torch.bool, device=self.device),
                        torch.zeros((groups, beams), dtype=torch.int32, device=self.device))  # fmt: skip
        self._beams = [make(), make()]
        self.steps = 0
        self.reset()

    def reset(self) -> None:
        """New searches: one live beam per group."""
        scores, finished, lengths = self._beams[0]
        scores.fill_(float("-inf"))
        scores[:, 0] = 0.0
        finished.zero_()
        lengths.zero_()
        self.steps = 0

    @property
    def scores(self) -> torch.Tensor:
        """(G, K) float32 summed log-probabilities of the beams, best rank first."""
        return self._beams[self.steps & 1][0]

    @property
    def finished(self) -> torch.Tensor:
        """(G, K) bool"""
        return self._beams[self.steps & 1][1]

    @property
    def lengths(self) -> torch.Tensor:
        """(G, K) int32"""
        return self._beams[self.steps & 1][2]

    @property
    def parents(self) -> torch.Tensor:
        """(G, K) int32: the beams that the last step's beams continue."""
        if self.steps == 0:
            raise ValueError("no step has been taken")
        return self._parents[self.steps - 1]

    def step(self, logits, states=(), *, slots: torch.Tensor | None = None, dim: int | None = None, start=0, length=None,
             history=None) -> torch.Tensor:  # fmt: skip
        """One token for every beam: logits (G * K, V) of the beams' last tokens -> tokens (G * K, 1) int32
        to run next (0 for beams that are dead: a group with fewer continuations than beams).  `states`
        follow their beams as reorder_states says, and `history` (a SlotHistory whose slots `slots` are
        the beams') does too and takes the tokens."""
        if self.steps >= self.max_steps:
            raise ValueError(f"the search was made for {self.max_steps} steps")
        if history is not None and slots is None:
            raise ValueError("history needs the beams' slots")
        (scores, finished, lengths), (new_scores, new_finished, new_lengths) = self._beams[self.steps & 1], self._beams[1 - (self.steps & 1)]
        out = Selected(self._tokens[self.steps], self._parents[self.steps], new_scores, new_finished, new_lengths)
        ends = self.end_id is not None
        beam_select(logits, scores, finished=finished if ends else None, end_id=self.end_id, lengths=lengths,
                    length_penalty=self.length_penalty, out=out)  # fmt: skip
        states = [states] if isinstance(states, torch.Tensor) else list(states)
        if states:
            reorder_states(states, out.parents, slots=slots, dim=dim, start=start, length=length)
        if history is not None:
            history.reorder(slots, out.parents)
            tokens = out.tokens
            if ends:  # what a finished beam goes on with is no token of its sequence
                tokens = tokens.masked_fill(finished.gather(1, out.parents.long()), -1)
            history.append(slots, tokens)
        self.steps += 1
        return out.tokens.clamp(min=0).reshape(-1, 1)

    def sequences(self) -> Sequences:
        """The tokens of the steps so far, of every beam."""
        return beam_sequences(self._tokens[: self.steps], self._parents[: self.steps], self.end_id)
