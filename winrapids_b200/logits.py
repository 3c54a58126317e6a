"""Rows of logits: a teacher's top logits, a student's distillation loss, sampled tokens.

Functions over the library calls of the same names (tbgb_top_logits, tbgb_distill_*,
tbgb_sample_tokens) for logits of any leading shape [..., vocab] on the device:

* ``top_logits(logits, k)`` -> ``TopLogits``: what to keep of a teacher's logits;
* ``distill_loss(logits, record)``: the loss of every position, differentiable by the logits;
* ``sample_tokens(logits, u)``: one token per position from given uniform numbers.

They enqueue on torch's current stream and do not wait; ``synchronize(device)`` waits and raises
what the device reported (a token id outside the vocabulary, an id named twice in a record).

They may be called from any host thread (a backward pass runs on one of autograd's): the context that they
share per device takes one call at a time.
"""
from __future__ import annotations

import threading
from dataclasses import dataclass

from . import Context, InvalidArgument, _torch

_LOCK = threading.Lock()
_CTX: dict[int, Context] = {}


def _call(device: int, method: str, *args, **kwargs):
    """Context.<method> on the device's context, alone."""
    with _LOCK:
        if device not in _CTX:
            _CTX[device] = Context(device)
        return getattr(_CTX[device], method)(*args, **kwargs)


def _device(logits) -> int:
    if not isinstance(logits, _torch().Tensor) or not logits.is_cuda:
        raise InvalidArgument(7, "logits must be a tensor on a CUDA device")
    return logits.get_device()


def synchronize(device: int = 0):
    """Wait for torch's current stream on `device` and raise what the kernels reported."""
    stream = _torch().cuda.current_stream(device)
    stream.synchronize()  # (not while other threads' calls wait for the context)
    _call(device, "sync", stream)


def _rows(t):
    """[..., n] as [rows, n] without a copy."""
    if t.dim() == 2:
        return t
    try:
        return t.view(-1, t.shape[-1])
    except RuntimeError:
        raise InvalidArgument(7, "the leading dimensions must be viewable as one (make the tensor contiguous)") from None


def _mask(mask, logits):
    """A token mask as the library takes it: [words] for every position, or [rows, words]."""
    if mask is None or mask.dim() <= 2:
        return mask
    if mask.shape[:-1] != logits.shape[:-1]:
        raise InvalidArgument(7, f"mask has leading shape {tuple(mask.shape[:-1])}, logits {tuple(logits.shape[:-1])}")
    return _rows(mask)


@dataclass
class TopLogits:
    """A teacher's record: per position the k largest logits (values) with their token ids, the
    temperature it is meant for, and the log-sum-exp of all logits at that temperature (None: the
    teacher is closed among its entries)."""

    values: object
    ids: object
    lse: object
    temperature: float

    def closed(self) -> "TopLogits":
        """The same entries as a distribution of their own."""
        return TopLogits(self.values, self.ids, None, self.temperature)


def top_logits(logits, k: int, temperature: float = 1.0, mask=None) -> TopLogits:
    """The record of a teacher's logits [..., vocab].  mask: words of the vocabulary [words] for every position, or
    [..., words]."""
    lead = logits.shape[:-1]
    out = _call(_device(logits), "top_logits", _rows(logits), k, temperature=temperature, mask=_mask(mask, logits), sync=False)
    return TopLogits(out["values"].view(*lead, k), out["ids"].view(*lead, k), out["lse"].view(lead), float(temperature))


def _distill_function():
    torch = _torch()

    class DistillLoss(torch.autograd.Function):
        @staticmethod
        def forward(logits, values, ids, lse, temperature):
            out = _call(_device(logits), "distill_loss", logits, ids, values, teacher_lse=lse, temperature=temperature,
                        sync=False, full_stats=True)
            return out["loss"], out["stats"]

        @staticmethod
        def setup_context(ctx, inputs, output):
            logits, values, ids, lse, ctx.temperature = inputs
            ctx.mark_non_differentiable(output[1])
            ctx.save_for_backward(logits, values, ids, lse, output[1])

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad_loss, _):
            logits, values, ids, lse, stats = ctx.saved_tensors
            grad = _call(_device(logits), "distill_grad", logits, ids, values, stats, grad_loss.float().contiguous(),
                         teacher_lse=lse, temperature=ctx.temperature, sync=False)
            return grad, None, None, None, None

    return DistillLoss


_function = None


def distill_loss(logits, record: TopLogits):
    """KL divergence of the student softmax(logits / T) from the recorded teacher at every position
    (f32, the leading shape of `logits`), differentiable by the logits (once)."""
    global _function
    if _function is None:
        _function = _distill_function()
    lead = logits.shape[:-1]
    lse = None if record.lse is None else record.lse.reshape(-1)
    loss, _ = _function.apply(_rows(logits), _rows(record.values), _rows(record.ids), lse, record.temperature)
    return loss.view(lead)


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """(tokens int32, log-probabilities f32) of the leading shape, from uniform numbers u of that shape.
    The settings are numbers or tensors of that shape, mask is [words] or [..., words]; see Context.sample_tokens."""
    torch = _torch()
    lead = logits.shape[:-1]

    def flat(v, dtype):
        if not isinstance(v, torch.Tensor):
            return v
        if dtype == torch.int32 and v.dtype == torch.int64:  # (a wider number would be cut to its low bits)
            v = v.clamp(0, 0x7FFFFFFF)
        return v.reshape(-1).to(dtype)

    out = _call(
        _device(logits), "sample_tokens", _rows(logits), flat(u, torch.float32), temperature=flat(temperature, torch.float32),
        top_k=flat(top_k, torch.int32), top_p=flat(top_p, torch.float32), min_p=flat(min_p, torch.float32),
        mask=_mask(mask, logits), sync=False)
    return out["tokens"].view(lead), out["logprobs"].view(lead)
