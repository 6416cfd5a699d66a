"""What beam search and log-probabilities refuse on the host, without a GPU: the C entry points' argument
checks return before anything is launched, and the Python face takes no CPU tensors; the slot history
follows its beams on CPU tensors."""

import ctypes as C
import subprocess

import numpy as np
import pytest
import torch

from leat_b200 import _lib
from tests import beam_reference as plain
from tests.test_abi import HEADER

BYTES = (C.c_byte * 4096)()
AT = (C.addressof(BYTES) + 255) // 256 * 256  # some address: refused calls do not look at it


def _select(**more):
    a = dict(logits=AT, groups=2, beams=3, vocab=100, width=4, row_stride=100, flags=0, end_id=-1, scores=AT, finished=None, lengths=None,
             length_penalty=0.0, out_tokens=AT, out_parents=AT, out_scores=AT, out_finished=None, out_lengths=None, workspace=AT,
             workspace_bytes=0)  # fmt: skip
    a.update(more)
    return _lib.lib.leat_beam_select(C.byref(_lib.BeamArgs(**a)), None)


def test_select_arguments():
    assert _lib.lib.leat_beam_select(None, None) == _lib.E_ARGUMENT
    for more in (dict(logits=None), dict(scores=None), dict(out_tokens=None), dict(out_parents=None), dict(out_scores=None), dict(groups=-1),
                 dict(beams=0), dict(vocab=0), dict(width=0), dict(row_stride=99), dict(flags=12), dict(flags=1), dict(end_id=100),
                 dict(finished=AT), dict(out_finished=AT), dict(out_lengths=AT), dict(length_penalty=0.5), dict(length_penalty=float("nan")),
                 dict(length_penalty=17.0, lengths=AT), dict(logits=AT + 2), dict(logits=AT + 1, flags=4)):  # fmt: skip
        assert _select(**more) == _lib.E_ARGUMENT, more
    assert _select(beams=65) == _lib.E_CAPACITY and _select(width=65) == _lib.E_CAPACITY
    assert _select(groups=1 << 30, beams=64) == _lib.E_CAPACITY
    need = _lib.lib.leat_beam_workspace_bytes(6, 100, 4)
    assert need > 0
    assert _select() == _select(workspace_bytes=need - 1) == _lib.E_WORKSPACE
    assert _select(workspace=None, workspace_bytes=need) == _select(workspace=AT + 16, workspace_bytes=need) == _lib.E_WORKSPACE
    assert _select(groups=0) == _lib.OK  # nothing to do


def test_workspace_sizes():
    size = _lib.lib.leat_beam_workspace_bytes
    assert size(0, 10, 4) == size(4, 0, 4) == size(4, 10, -1) == size(4, 10, 65) == 0
    assert 0 < size(4, 8192, 0) < size(4, 8192, 4) < size(4, 8193, 4) < size(5, 8193, 4)
    assert size(1 << 20, 1 << 18, 64) > 1 << 32  # (sizes do not wrap)


def test_logprob_arguments():
    def call(**more):
        a = dict(logits=AT, rows=2, vocab=100, row_stride=100, flags=0, given=1, top=3, ids=AT, out_logprobs=AT, out_top_logprobs=AT,
                 out_top_ids=AT, workspace=AT, workspace_bytes=0)  # fmt: skip
        a.update(more)
        return _lib.lib.leat_token_logprobs(C.byref(_lib.LogprobArgs(**a)), None)

    assert _lib.lib.leat_token_logprobs(None, None) == _lib.E_ARGUMENT
    for more in (dict(logits=None), dict(rows=-1), dict(vocab=0), dict(row_stride=50), dict(flags=12), dict(given=-1), dict(top=-1),
                 dict(ids=None), dict(out_logprobs=None), dict(out_top_logprobs=None), dict(out_top_ids=None)):  # fmt: skip
        assert call(**more) == _lib.E_ARGUMENT, more
    assert call(top=65) == _lib.E_CAPACITY
    assert call() == _lib.E_WORKSPACE
    assert call(rows=0) == _lib.OK


def test_reorder_arguments():
    def call(parents=AT, slots=None, groups=2, beams=3, count=1, states=None, **more):
        s = dict(data=AT, row_stride=64, outer_stride=0, place_bytes=64, outer=1, places=1, rows=6)
        s.update(more)
        array = (_lib.State * 1)(_lib.State(**s))
        return _lib.lib.leat_reorder_states(array if states is None else states, count, parents, slots, groups, beams, None, 0, None, 1 << 30, None)

    for more in (dict(parents=None), dict(groups=-1), dict(beams=0), dict(count=-1), dict(data=None), dict(rows=5), dict(place_bytes=0),
                 dict(outer=2, outer_stride=32), dict(row_stride=-64), dict(places=-1), dict(outer=-1)):  # fmt: skip
        assert call(**more) == _lib.E_ARGUMENT, more
    assert call(beams=65) == call(groups=65536, beams=1, rows=65536) == _lib.E_CAPACITY
    assert call(groups=0) == call(count=0) == _lib.OK


def test_sequence_arguments():
    def call(tokens=AT, parents=AT, steps=4, groups=2, beams=3, out=AT, lengths=AT):
        return _lib.lib.leat_beam_sequences(tokens, parents, steps, groups, beams, -1, out, lengths, None)

    for more in (dict(tokens=None), dict(parents=None), dict(out=None), dict(lengths=None), dict(steps=-1), dict(groups=-1), dict(beams=0)):
        assert call(**more) == _lib.E_ARGUMENT, more
    assert call(beams=65) == _lib.E_CAPACITY
    assert call(groups=0) == _lib.OK


@pytest.mark.parametrize("struct,name", [(_lib.BeamArgs, "leat_beam_args"), (_lib.State, "leat_state"), (_lib.LogprobArgs, "leat_logprob_args")])
def test_struct_layouts_match_the_header(tmp_path, struct, name):
    fields = [f for f, _ in struct._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {", f'  printf("%zu\\n", sizeof({name}));']
    lines += [f'  printf("%zu\\n", offsetof({name}, {f}));' for f in fields]
    (tmp_path / "layout.c").write_text("\n".join([*lines, "  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [C.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


def test_packed_arguments_are_the_structs():
    """The Python face packs a call's arguments itself; every field lies where the struct has it."""
    import struct

    from leat_b200 import beam, logprobs

    for fmt, kind in ((beam.SELECT_ARGS, _lib.BeamArgs), (logprobs.ARGS, _lib.LogprobArgs), ("P" + beam.STATE_REST, _lib.State)):
        assert struct.calcsize(fmt) == C.sizeof(kind)
        values = [float(i + 1) if f[1] is C.c_float else i + 1 for i, f in enumerate(kind._fields_)]
        extra = [0] if kind is _lib.State else []  # the padding at its end
        got = kind.from_buffer_copy(struct.pack(fmt, *values, *extra))
        assert [getattr(got, f) for f, _ in kind._fields_] == values


def test_cpu_tensors_are_refused():
    from leat_b200 import beam_select, beam_sequences, reorder_states, token_logprobs

    ints = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises(ValueError):
        beam_select(torch.zeros((6, 10)), torch.zeros((2, 3)))
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros((6, 10)), ints.reshape(6, 1))
    with pytest.raises(ValueError):
        reorder_states(torch.zeros((6, 10)), ints)
    with pytest.raises(ValueError):
        beam_sequences(ints.reshape(1, 2, 3), ints.reshape(1, 2, 3))


def test_history_follows_its_beams_on_the_cpu():
    from leat_b200.history import SlotHistory

    rng = np.random.default_rng(1)
    h = SlotHistory(10, 6, 100)
    h.ids[:] = torch.tensor(rng.integers(0, 100, (10, 6)), dtype=torch.int32)
    h.count[:] = torch.arange(10, dtype=torch.int32)
    ids, count = h.ids.clone(), h.count.clone()
    slots = torch.tensor([[7, 2, 9], [0, 4, 5]])
    h.reorder(slots, torch.tensor([[2, 0, 0], [1, 1, -1]]))
    want = {7: 9, 2: 7, 9: 7, 0: 4, 4: 4, 5: 5}
    for slot in range(10):
        of = want.get(slot, slot)
        assert torch.equal(h.ids[slot], ids[of]) and h.count[slot] == count[of]
    with pytest.raises(ValueError):
        h.reorder(slots[0], slots[0])


def test_plain_statements_agree_with_each_other():
    """The 64-bit statements the GPU tests compare with: a search's scores are the sums of log-probabilities
    along the sequences that are read back."""
    rng = np.random.default_rng(3)
    table = rng.standard_normal((20, 20)) * 2  # logits by last token
    groups, beams, steps = 2, 3, 6
    scores = np.full((groups, beams), -np.inf)
    scores[:, 0] = 0.0
    last = np.zeros((groups, beams), int)
    tokens, parents = [], []
    for _ in range(steps):
        found = plain.continuations(table[last.reshape(-1)], scores)
        tokens.append(np.array([[c[3] for c in f[:beams]] for f in found]))
        parents.append(np.array([[c[1] for c in f[:beams]] for f in found]))
        scores = np.array([[c[4] for c in f[:beams]] for f in found])
        last = tokens[-1]
    read, lengths = plain.sequences(np.stack(tokens), np.stack(parents))
    share = plain.log_softmax(table)
    for g in range(groups):
        for k in range(beams):
            run = [0, *read[g, k]]
            assert abs(sum(share[a, b] for a, b in zip(run, run[1:])) - scores[g, k]) < 1e-12
    assert (lengths == steps).all()
