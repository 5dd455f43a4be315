"""How likely given tokens are under a model's logits: scores of texts, the loss of a training step, what a sampler reports."""
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["TokenLogprobs", "next_token_targets", "token_logprobs"]

_n = _lib.native

TokenLogprobs = namedtuple("TokenLogprobs", ["logprobs", "entropy", "top_logprobs", "top_ids"])


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, return_entropy, ignore_index):
        lp, ent, lse, top, ids = _n().logprobs_fwd(logits, targets, top_k, return_entropy, ignore_index)
        ctx.save_for_backward(logits, targets, lse, ent)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        if top is not None:
            ctx.mark_non_differentiable(top, ids)
        return lp, ent, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g, h, *unused):
        if g is None and h is None:
            return (None,) * 5
        logits, targets, lse, ent = ctx.saved_tensors
        return _n().logprobs_bwd(logits, targets, lse, ent, ctx.ignore_index, g, h), None, None, None, None


def token_logprobs(logits, targets, top_k=0, return_entropy=False, ignore_index=-100):
    """A :class:`TokenLogprobs` of float32 results for logits (rows, vocab) or (batch, seqlen, vocab) -- CUDA, float32, float16 or
    bfloat16, contiguous in the last dim, rows at any stride (``model_logits[:, :-1]`` and ``[..., :vocab]`` are not copied) -- and
    int64 targets of the leading shape:

    ``logprobs``       log p(target); 0 where the target is ``ignore_index``.  A target outside the vocabulary gives NaN and
                       makes :func:`quamba_b200.check_device_status` raise.
    ``entropy``        of the row's distribution, with ``return_entropy``, else None
    ``top_logprobs``, ``top_ids`` (..., top_k)  the most likely columns, largest first, equal logits in the order of their
                       columns; None with ``top_k`` 0, at most 32

    Columns of -inf have probability 0.  A row of nothing but -inf gives log probabilities of -inf, entropy 0 and no gradient; a row with a NaN
    or +inf gives NaN.  ``logprobs`` and ``entropy`` are differentiable (once) in the logits, the alternatives are not."""
    if torch.is_grad_enabled() and logits.requires_grad:
        lp, ent, top, ids = _TokenLogprobs.apply(logits, targets, top_k, return_entropy, ignore_index)
    else:
        lp, ent, _, top, ids = _n().logprobs_fwd(logits, targets, top_k, return_entropy, ignore_index)
    return TokenLogprobs(lp, ent, top, ids)


def next_token_targets(input_ids, lengths=None, ignore_index=-100):
    """The targets (batch, seqlen - 1), int64, of a batch of token ids: each position's next token, ``ignore_index`` where that is at or past
    ``lengths[b]``."""
    targets = input_ids[:, 1:].to(torch.int64)
    if lengths is None:
        return targets
    lengths = torch.as_tensor(lengths, device=input_ids.device)
    return targets.masked_fill(torch.arange(1, input_ids.shape[1], device=input_ids.device)[None] >= lengths[:, None], ignore_index)
