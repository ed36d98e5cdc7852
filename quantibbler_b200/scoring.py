"""Log probabilities of given tokens, with the entropy of their distributions and the most probable entries."""

from __future__ import annotations

from typing import NamedTuple

from . import _lib
from ._lib import KernelError, check
from .cache import check_tensor, ordered, workspace
from .gpu import GpuContext

MAX_TOP = 32


class LogProbs(NamedTuple):
    """Per row of logits, on the device: ``lse`` (ln of the sum of exponentials), ``logprob`` of the target (None
    without targets), ``entropy`` in nats, and the ``top`` most probable entries, ``top_ids`` (int32, ties: the
    lowest id first) and ``top_logprob``."""
    lse: object
    logprob: object
    entropy: object
    top_logprob: object
    top_ids: object


def log_probs(ctx: GpuContext, logits, targets=None, top: int = 0) -> LogProbs:
    """``logits`` float32 ``[rows, vocab]``, rows possibly apart; ``targets`` int32 ``[rows]`` or None, a negative
    one marks a row without a token (its logprob is 0).  A row that holds a NaN or +infinity, or nothing above
    -infinity, gives NaN (its ids: -1); entries of -infinity are impossible ones.  Runs on the context's stream,
    ordered with torch's current one."""
    import torch
    shape, dev = logits.shape, logits.device
    if len(shape) != 2:
        raise KernelError(f"logits must be [rows, vocab], got {tuple(shape)}")
    if dev.type != "cuda" or dev.index != ctx.device_index:
        raise KernelError(f"logits are on {dev}, the context on cuda:{ctx.device_index}")
    if logits.dtype is not torch.float32:
        check_tensor("logits", logits, torch.float32, dev)
    n, vocab = shape
    if logits.stride(1) != 1 and vocab > 1:
        raise KernelError(f"a row of logits must be contiguous, got strides {logits.stride()}")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise KernelError(f"top must lie in 0 .. {min(MAX_TOP, vocab)}, got {top}")
    if targets is not None:
        check_tensor("targets", targets, torch.int32, dev, (n,))
        if not targets.is_contiguous():
            raise KernelError("targets must be contiguous")
    new = logits.new_empty    # (cheaper than views of one tensor)
    lse, entropy, logprob, top_logprob = new(n), new(n), None if targets is None else new(n), new((n, top))
    top_ids = torch.empty((n, top), dtype=torch.int32, device=dev) if targets is None else targets.new_empty((n, top))
    lib = _lib.lib()
    if n:
        scratch = workspace(ctx, lib.qk_log_probs_scratch(n, vocab, top), dev)
        with ordered(ctx, dev):
            check(lib.qk_log_probs(ctx.handle, logits.data_ptr(), n, vocab, logits.stride(0) if n > 1 else vocab,
                                   None if targets is None else targets.data_ptr(), top,
                                   None if scratch is None else scratch.data_ptr(), lse.data_ptr(),
                                   None if logprob is None else logprob.data_ptr(), entropy.data_ptr(),
                                   top_logprob.data_ptr() if top else None, top_ids.data_ptr() if top else None))
    return LogProbs(lse, logprob, entropy, top_logprob, top_ids)
