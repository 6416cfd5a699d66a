"""Beam search over the logits this package samples from, and the log-probabilities a server reports:
the cases that stand for their use, and each operator in its plain form (elementary torch operations).

* select: one step of beam search, from logits (groups * beams, vocab) and the beams' scores to the
  `width` best (parent, token) continuations of each group.
* reorder: the rows of caches and other per-beam states follow the chosen parents, in place.
* sequences: the tokens of every final beam, read back through the parents of all steps.
* logprobs: log-probabilities of given tokens, and of each row's `top` likeliest ones.
"""

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # the first step of one request: only the first beam is live; latency counts
        dict(name="select_one", op="select", groups=1, beams=4, vocab=128256, width=4, type="float32",
             pad=0, first=True, ends=False, masked=False, penalty=0.0),
        # a server's step: 16 requests of 5 beams, twice as many continuations as beams, so that the
        # caller can set finished ones aside itself
        dict(name="select_server", op="select", groups=16, beams=5, vocab=151936, width=10, type="bfloat16",
             pad=0, first=False, ends=False, masked=False, penalty=0.0),
        # an lm_head of an odd width, some rows held to a grammar's few tokens, one row with none
        dict(name="select_odd", op="select", groups=7, beams=3, vocab=32003, width=6, type="float16",
             pad=0, first=False, ends=True, masked=True, penalty=1.0),
        # a large batch and vocabulary, finished beams kept, scores compared per length
        dict(name="select_batch", op="select", groups=32, beams=8, vocab=262144, width=8, type="float32",
             pad=64, first=False, ends=True, masked=False, penalty=0.6),
        # the caches of one request's beams behind a shared prompt of 256 positions
        dict(name="reorder_one", op="reorder", groups=1, beams=4, states=24, heads=8, places=1024, inner=64,
             type="bfloat16", start=256, length=320, ragged=False, slots=False),
        # generated tokens kept in rings per cache slot, and other states without positions: odd widths
        dict(name="reorder_slots", op="reorder", groups=12, beams=6, states=6, heads=3, places=0, inner=1027,
             type="float32", start=0, length=0, ragged=False, slots=True),
        # a batch's caches, prompts and lengths of their own
        dict(name="reorder_batch", op="reorder", groups=8, beams=8, states=8, heads=8, places=2048, inner=128,
             type="bfloat16", start=512, length=1500, ragged=True, slots=False),
        # a short answer of one request
        dict(name="sequences_one", op="sequences", groups=1, beams=4, steps=48, vocab=128256),
        # long answers of a batch
        dict(name="sequences_long", op="sequences", groups=64, beams=8, steps=4096, vocab=262144),
        # one decode step's tokens with their five likeliest alternatives
        dict(name="logprobs_step", op="logprobs", rows=16, vocab=151936, given=1, top=5, type="float32", pad=0),
        # the verification rows of a speculative step
        dict(name="logprobs_verify", op="logprobs", rows=72, vocab=151936, given=1, top=20, type="bfloat16", pad=0),
        # a chunk of a prompt scored
        dict(name="logprobs_prompt", op="logprobs", rows=512, vocab=201088, given=1, top=0, type="bfloat16", pad=0),
    ]  # fmt: skip


def _spread(rng, low, high):
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "sequences", "logprobs"])
    kind = rng.choice(["float32", "bfloat16", "float16"])
    if op == "select":
        vocab = _spread(rng, 1000, 262144)
        beams = _spread(rng, 2, 24)
        groups = _spread(rng, 1, max(1, min(64, 32 * 8 * 262144 // (2 * beams * vocab))))
        return dict(op=op, groups=groups, beams=beams, vocab=vocab, width=min(64, beams * rng.choice([1, 1, 2])), type=kind,
                    pad=rng.choice([0, 0, 1, 64]), first=rng.random() < 0.2, ends=rng.random() < 0.5,
                    masked=rng.random() < 0.3, penalty=rng.choice([0.0, 0.6, 1.0]))  # fmt: skip
    if op == "logprobs":
        vocab = _spread(rng, 1000, 262144)
        return dict(op=op, rows=_spread(rng, 1, min(1024, 32 * 8 * 262144 // (2 * vocab))), vocab=vocab, given=rng.choice([1, 1, 3]),
                    top=rng.choice([0, 1, 5, 20]), type=kind, pad=rng.choice([0, 0, 1, 64]))  # fmt: skip
    if op == "sequences":
        return dict(op=op, groups=_spread(rng, 1, 64), beams=_spread(rng, 2, 24), steps=_spread(rng, 1, 1024), vocab=128256)
    beams, groups = _spread(rng, 2, 16), _spread(rng, 1, 16)
    if rng.random() < 0.3:  # states without positions
        return dict(op=op, groups=groups, beams=beams, states=rng.randint(1, 12), heads=rng.randint(1, 4), places=0, inner=_spread(rng, 1, 20000),
                    type=rng.choice(["float32", "bfloat16"]), start=0, length=0, ragged=False, slots=rng.random() < 0.5)  # fmt: skip
    places = _spread(rng, 16, 2048)
    length = rng.randint(1, places)
    return dict(op=op, groups=groups, beams=beams, states=rng.randint(1, 8), heads=rng.choice([1, 2, 5, 8]), places=places,
                inner=rng.choice([40, 64, 80, 128]), type="bfloat16", start=rng.randint(0, length), length=length,
                ragged=rng.random() < 0.5, slots=rng.random() < 0.3)  # fmt: skip


def _logits(g, rows, vocab, pad, kind):
    wide = torch.randn((rows, vocab + pad), generator=g, device="cuda").mul_(3.0).to(TYPES[kind])
    return wide[:, :vocab]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    rand = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
    if c["op"] == "logprobs":
        logits = _logits(g, c["rows"], c["vocab"], c["pad"], c["type"])
        ids = torch.randint(0, c["vocab"], (c["rows"], c["given"]), generator=g, device="cuda", dtype=torch.int32)
        ids[:, 0] = logits.argmax(1)  # what a greedy step has just picked
        return dict(c, logits=logits, ids=ids)
    groups, beams = c["groups"], c["beams"]
    if c["op"] == "select":
        logits = _logits(g, groups * beams, c["vocab"], c["pad"], c["type"])
        if c["masked"]:  # every third row may only go on with about 1 % of the tokens; one with none
            held = rand(groups * beams, c["vocab"]) > 0.01
            held[1::3] = False
            held[2::3] = False
            logits.masked_fill_(held, torch.finfo(logits.dtype).min)
            logits[-1] = float("-inf")
        scores = (-4.0 * rand(groups, beams)).cumsum(1)
        if c["first"]:
            scores[:, 1:] = float("-inf")
        s = dict(c, logits=logits, scores=scores, finished=None, lengths=None)
        if c["ends"]:
            s["finished"] = rand(groups, beams) < 0.25
            s["lengths"] = 1 + (rand(groups, beams) * 60).to(torch.int32)
        return s
    if c["op"] == "sequences":
        steps = c["steps"]
        tokens = (rand(steps, groups, beams) * (c["vocab"] - 1)).to(torch.int32) + 1
        ended = rand(steps, groups, beams) < 1.0 / steps
        return dict(c, tokens=tokens.masked_fill_(ended, 0), parents=(rand(steps, groups, beams) * beams).to(torch.int32))
    # about two thirds of the beams live on; their children lie anywhere
    live = _live(beams)
    kept = rand(groups, beams).argsort(1)[:, :live]
    child = torch.cat([torch.arange(live, device="cuda").expand(groups, live), (rand(groups, beams - live) * live).long()], 1)
    parents = kept.gather(1, child).gather(1, rand(groups, beams).argsort(1)).to(torch.int32)
    rows = groups * beams + (5 if c["slots"] else 0)
    shape = (rows, c["heads"], c["places"], c["inner"]) if c["places"] else (rows, c["heads"], c["inner"])
    states = [torch.randn(shape, generator=g, device="cuda").to(TYPES[c["type"]]) for _ in range(c["states"])]
    s = dict(c, parents=parents, states=states, rows=None, first_place=None, end_place=None)
    if c["slots"]:
        s["rows"] = rand(rows).argsort()[: groups * beams].reshape(groups, beams).to(torch.int32)
    if c["places"]:
        s["first_place"], s["end_place"] = c["start"], c["length"]
        if c["ragged"]:
            span = c["length"] - c["start"]
            s["first_place"] = (c["start"] - (rand(groups) * c["start"] * 0.5)).to(torch.int32)
            s["end_place"] = s["first_place"] + span
    return s


def _live(beams):
    return max(1, (2 * beams + 2) // 3)


def _order(x):
    # float32 -> whole numbers in the floats' order
    bits = (x + 0.0).view(torch.int32)
    return torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()


def _best(x, n):
    """Values and indices of each row's n largest, the lower index first among equals."""
    low = 0xFFFFFFFF - torch.arange(x.shape[1], device=x.device)
    at = 0xFFFFFFFF - ((_order(x) * 4294967296 + low).topk(min(n, x.shape[1]), 1).values & 0xFFFFFFFF)
    return x.gather(1, at), at


def _log_sum(x):
    # in 64 bits: differences of the sums decide which beam goes on
    x = x.double()
    top = x.amax(1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    return top + (x - top).exp().sum(1, keepdim=True).log()


def _plain_select(s):
    groups, beams, width = s["groups"], s["beams"], s["width"]
    x = s["logits"].float()
    value, token = _best(x, width)
    score = s["scores"].double().reshape(-1, 1) + (value.double() - _log_sum(x))
    score = torch.where((value > float("-inf")) & (s["scores"].reshape(-1, 1) > float("-inf")), score, float("-inf"))
    n = value.shape[1]
    finished = torch.zeros_like(token, dtype=torch.bool)
    length = torch.zeros_like(token)
    if s["finished"] is not None:
        done = s["finished"].reshape(-1, 1)
        only = torch.where(torch.arange(n, device=x.device) == 0, s["scores"].double().reshape(-1, 1), float("-inf"))
        score, token = torch.where(done, only, score), torch.where(done, 0, token)
        finished = done | (token == 0)
        length = s["lengths"].reshape(-1, 1) + torch.where(done, 0, 1)
        length = length.expand_as(token)
    rank = score if s["penalty"] == 0.0 or s["finished"] is None else score / ((5.0 + length.double()) / 6.0) ** s["penalty"]
    rank, at = rank.reshape(groups, beams * n).sort(dim=1, descending=True, stable=True)
    if beams * n < width:
        raise ValueError("fewer continuations than asked for")
    at = at[:, :width]
    pick = lambda v: v.reshape(groups, beams * n).gather(1, at)  # noqa: E731
    score, token, finished, length = pick(score), pick(token), pick(finished), pick(length)
    none = score == float("-inf")
    place = torch.arange(width, device=x.device) % beams
    out = dict(tokens=torch.where(none, -1, token).to(torch.int32), parents=torch.where(none, place, at // n).to(torch.int32), scores=score.float())
    if s["finished"] is not None:
        out.update(finished=finished & ~none, lengths=torch.where(none, 0, length).to(torch.int32))
    return out


def _plain_reorder(s):
    groups, beams = s["groups"], s["beams"]
    at = torch.arange(groups * beams, device="cuda").reshape(groups, beams) if s["rows"] is None else s["rows"].long()
    to, of = at.reshape(-1), at.gather(1, s["parents"].long()).reshape(-1)
    moves = None
    if s["places"]:
        place = torch.arange(s["places"], device="cuda")
        per_row = lambda v: v.long().repeat_interleave(beams).reshape(-1, 1) if isinstance(v, torch.Tensor) else v  # noqa: E731
        moves = ((place >= per_row(s["first_place"])) & (place < per_row(s["end_place"]))).reshape(-1, 1, s["places"], 1)
    for t in s["states"]:
        t[to] = t[of] if moves is None else torch.where(moves, t[of], t[to])
    return list(s["states"])


def _plain_sequences(s):
    steps, groups, beams = s["tokens"].shape
    # path[t][k]: the beam that final beam k passed through at step t; joined in twice as long runs
    path = torch.cat([s["parents"][1:].long(), torch.arange(beams, device="cuda").expand(1, groups, beams)])
    run = 1
    while run < steps:
        path = torch.cat([path[:-run].gather(2, path[run:]), path[-run:]])
        run *= 2
    token = s["tokens"].gather(2, path)
    ended = (token == 0).cumsum(0) > 0
    length = steps - ended.sum(0) + ended[-1]
    return dict(sequences=token.masked_fill(ended, 0).permute(1, 2, 0).contiguous(), lengths=length.to(torch.int32))


def _plain_logprobs(s):
    x = s["logits"].float()
    total = _log_sum(x)
    out = dict(logprobs=(x.gather(1, s["ids"].long()).double() - total).float())
    if s["top"]:
        value, at = _best(x, s["top"])
        out.update(top_logprobs=(value.double() - total).float(), top_ids=at.to(torch.int32))
    return out


def run(s):
    if not own:
        return {"select": _plain_select, "reorder": _plain_reorder, "sequences": _plain_sequences, "logprobs": _plain_logprobs}[s["op"]](s)
    from leat_b200 import beam, logprobs

    if s["op"] == "select":
        r = beam.beam_select(s["logits"], s["scores"], s["width"], finished=s["finished"], lengths=s["lengths"],
                             end_id=0 if s["ends"] else None, length_penalty=s["penalty"] if s["ends"] else 0.0)  # fmt: skip
        out = dict(tokens=r.tokens, parents=r.parents, scores=r.scores)
        if s["ends"]:
            out.update(finished=r.finished, lengths=r.lengths)
        return out
    if s["op"] == "reorder":
        beam.reorder_states(s["states"], s["parents"], slots=s["rows"], dim=2 if s["places"] else None,
                            start=s["first_place"], length=s["end_place"])  # fmt: skip
        return list(s["states"])
    if s["op"] == "sequences":
        r = beam.beam_sequences(s["tokens"], s["parents"], end_id=0)
        return dict(sequences=r.tokens, lengths=r.lengths)
    r = logprobs.token_logprobs(s["logits"], s["ids"], top=s["top"])
    out = dict(logprobs=r.logprobs)
    if s["top"]:
        out.update(top_logprobs=r.top_logprobs, top_ids=r.top_ids)
    return out


def work(case):
    c = case
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        # a difference, an exponential and a sum per logit, and its comparison with the row's best
        return dict(bytes=n * BYTES[c["type"]] + c["rows"] * (8 * c["given"] + 8 * c["top"]), flops=(4 if c["top"] else 3) * n)
    rows = c["groups"] * c["beams"]
    if c["op"] == "select":
        # logits of finished and dead beams need not be read
        live = rows * (0.75 if c["ends"] else 1.0) / (c["beams"] if c["first"] else 1)
        n = live * c["vocab"]
        return dict(bytes=n * BYTES[c["type"]] + rows * (9 if c["ends"] else 4) + c["groups"] * c["width"] * (17 if c["ends"] else 12), flops=4 * n)
    if c["op"] == "sequences":
        return dict(bytes=c["steps"] * rows * 12 + rows * 4, flops=c["steps"] * rows)
    # a beam keeps its place one time in `beams`; the others' rows are written, and those of the live ones read
    span = c["heads"] * c["inner"] * ((c["length"] - c["start"]) if c["places"] else 1) * BYTES[c["type"]]
    moved = c["beams"] - 1
    return dict(bytes=c["groups"] * c["states"] * span * (moved + min(moved, _live(c["beams"]))) + 4 * rows, flops=0)


def exact(case, seed):
    if case["op"] not in ("select", "logprobs"):
        return None  # they move whole values
    s = prepare(case, seed)
    share = torch.log_softmax(s["logits"].double(), 1)
    if case["op"] == "logprobs":
        out = dict(logprobs=share.gather(1, s["ids"].long()))
        if case["top"]:
            out.update(top_logprobs=share.topk(case["top"], 1).values, top_ids=None)
        return out
    groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
    # every continuation of every beam; a row without any token has none
    share = torch.where(torch.isnan(share), float("-inf"), share).reshape(groups, beams, vocab)
    total = share.add_(s["scores"].double().unsqueeze(2))
    divide = torch.ones((groups, beams, 1), dtype=torch.float64, device="cuda")
    if case["ends"]:
        total[s["finished"]] = float("-inf")
        total[..., 0] = torch.where(s["finished"], s["scores"].double(), total[..., 0])
        length = s["lengths"].double() + (~s["finished"]).double()
        divide = ((5.0 + length) / 6.0).pow(case["penalty"]).unsqueeze(2)
    at = (total / divide).reshape(groups, beams * vocab).topk(case["width"], 1).indices
    out = dict(tokens=None, parents=None, scores=total.reshape(groups, beams * vocab).gather(1, at))
    if case["ends"]:
        out.update(finished=None, lengths=None)
    return out
