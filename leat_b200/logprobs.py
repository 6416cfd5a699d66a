"""Log-probabilities of tokens under rows of logits, as a server reports them beside what it sampled and
as a score of a prompt: of given ids, and of each row's likeliest tokens.  One pass over the logits,
no handle, no host synchronisation; scratch is allocated per call on the current stream."""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache
from struct import pack

import torch

from leat_b200 import _lib
from leat_b200.sampler import device_tensor

FORMATS = {torch.float32: 0, torch.bfloat16: _lib.FLAG_LOGITS_BF16, torch.float16: _lib.FLAG_LOGITS_F16}
MAX_TOP = 64
ARGS = "PiiqIii4xPPPPPN"  # struct leat_logprob_args


@dataclass
class TokenLogprobs:
    logprobs: torch.Tensor | None  # (B, M) float32: of the given ids
    top_logprobs: torch.Tensor | None = None  # (B, top) float32, likeliest first, -inf-padded
    top_ids: torch.Tensor | None = None  # (B, top) int32, the lower id first among equals, -1-padded


def rows_of_logits(logits) -> torch.Tensor:
    """`logits` as the kernels take it: (B, V) on the device, adjacent logits adjacent in memory."""
    if not isinstance(logits, torch.Tensor):
        logits = device_tensor(logits)
    elif logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("no gradient flows through this call: detach the logits, or call under torch.no_grad()")
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or logits.dtype not in FORMATS or not logits.is_cuda:
        raise ValueError("logits must be a (B, V) float32, bfloat16 or float16 CUDA tensor")
    rows, vocab = logits.shape
    if vocab == 0:
        raise ValueError("logits must have at least one token per row")
    if not logits.is_contiguous():
        stride = logits.stride()
        if (stride[1] != 1 and vocab > 1) or (stride[0] < vocab and rows > 1):
            logits = logits.contiguous()
    return logits


@lru_cache(maxsize=256)
def _scratch_bytes(rows: int, vocab: int, width: int) -> int:
    size = _lib.lib.leat_beam_workspace_bytes(rows, vocab, width)
    if size == 0:
        raise ValueError(f"({rows}, {vocab}) logits are beyond the kernels' sizes")
    return size + 256


# A call's time on the host is most of what a small one takes, so two of torch's inner entry points are
# used where they are there: the current stream's handle without a Stream object around it (0.1 us for
# 3.2), and memory of the current device without the keyword arguments' parsing (0.8 us for 1.8).
def plain_raw_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or plain_raw_stream


def plain_empty_strided(size, stride, dtype):
    return torch.empty_strided(size, stride, dtype=dtype, device="cuda")


empty_strided = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None) or plain_empty_strided


def scratch(rows: int, vocab: int, width: int) -> tuple[torch.Tensor, int, int]:
    """A call's workspace on the current device: the tensor that holds it, its 256-byte aligned address and
    its size.  It is the call's own (the caching allocator keeps it for the current stream), so calls on
    several streams or in several graphs share nothing."""
    size = _scratch_bytes(rows, vocab, width)
    held = empty_strided((size,), (1,), torch.uint8)
    return held, (held.data_ptr() + 255) & ~255, size - 256


def token_logprobs(logits, ids=None, top: int = 0) -> TokenLogprobs:
    """Log-probabilities under softmax(logits): of `ids` (B,) or (B, M) (int32 or int64, on the device),
    and of each row's `top` likeliest tokens (0..64), with their ids.  logits (B, V) float32, bfloat16
    or float16.  Results are float32, (B, M) and (B, top).

    There is no backward pass: logits that a gradient is wanted of are refused (detach them, or call under
    torch.no_grad()).

    A NaN logit counts as -inf, +inf as the largest float.  Ids outside the vocabulary (a -1 of padding) and
    tokens of logit -inf have log-probability -inf, as does everything in a row without a logit above -inf."""
    logits = rows_of_logits(logits)
    dev = logits.device
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return token_logprobs(logits, ids, top)
    rows, vocab = logits.shape
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be an integer from 0 to {MAX_TOP}")
    given = 0
    if ids is not None:
        ids = device_tensor(ids)
        if not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int32, torch.int64) or ids.device != dev:
            raise ValueError("ids must be an int32 or int64 tensor on the logits' device")
        if ids.dim() not in (1, 2) or ids.shape[0] != rows:
            raise ValueError("ids must be (B,) or (B, M), a row per row of logits")
        given = ids.shape[1] if ids.dim() == 2 else 1
        if ids.dtype == torch.int64:  # (what does not fit 32 bits is outside every vocabulary)
            ids = ids.clamp(-1, vocab).to(torch.int32)
        if not ids.is_contiguous():
            ids = ids.contiguous()
    out = TokenLogprobs(None if ids is None else empty_strided((rows, given), (given, 1), torch.float32))
    if top:
        out.top_logprobs = empty_strided((rows, top), (top, 1), torch.float32)
        out.top_ids = empty_strided((rows, top), (top, 1), torch.int32)
    if rows == 0 or given + top == 0:
        return out
    held, at, size = scratch(rows, vocab, top)
    a = pack(ARGS, logits.data_ptr(), rows, vocab, logits.stride(0), FORMATS[logits.dtype], given, top, ids.data_ptr() if given else 0,
             out.logprobs.data_ptr() if given else 0, out.top_logprobs.data_ptr() if top else 0, out.top_ids.data_ptr() if top else 0,
             at, size)  # fmt: skip
    code = _lib.lib.leat_token_logprobs(a, raw_stream(dev.index))
    if code != _lib.OK:
        _lib.check(code, "leat_token_logprobs")
    return out
