"""The Mamba1 recurrence in floating point: what a float model runs before it is quantised (calibration, fine-tuning), next to
the int8 scan of :mod:`quamba_b200.ops`.

    delta = softplus(dt + dt_bias)                              (dt_softplus, else dt + dt_bias)
    h_t   = exp(delta_t A) h_{t-1} + delta_t x_t B_t            float32, one row of dstate values per channel
    y_t   = (C_t . h_t + D x_t) silu(z_t)

The float counterpart of the interface the reference quantises (``selective_scan_fn`` / ``selective_state_update``, called in
quamba/qMambaLayer.py), channel-last: tokens are rows, as ``in_proj``, the conv and ``x_proj`` write them, and nothing is
transposed.  There is no CPU path.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["selective_scan", "selective_scan_update"]

_n = _lib.native


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, lengths):
        y, last, kept = _n().float_scan_fwd(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, lengths, True, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, initial_state, lengths, kept)
        ctx.dt_softplus = dt_softplus
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, dt, A, B, C, D, z, dt_bias, initial_state, lengths, kept = ctx.saved_tensors
        if dy is None and dlast is None:
            return (None,) * 11
        if dy is None:
            dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
        dx, ddt, dA, dB, dC, dD, dz, dbias, dinit = _n().float_scan_bwd(x, dt, A, B, C, D, z, dt_bias, ctx.dt_softplus, initial_state, lengths, kept,
                                                                        dy, dlast)
        return dx, ddt, dA, dB, dC, dD, dz, dbias, None, dinit, None


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None, lengths=None,
                   return_final_state=False):
    """y (batch, seqlen, dim), or (y, final state float32 (batch, dim, dstate)) with ``return_final_state``.

    x, dt, z (batch, seqlen, dim) and B, C (batch, seqlen, dstate) or (batch, seqlen, groups, dstate) are CUDA tensors of one
    type (float32, float16, bfloat16), contiguous in their last dim; other strides are free, so halves and column blocks of a
    projection's rows are passed as they are.  A (dim, dstate), D and dt_bias (dim,), initial_state (batch, dim, dstate) are float32;
    dstate is 1 to 64, and channel d reads group ``d // (dim // groups)`` of B and C.

    ``lengths`` (int32 (batch,), on the device) gives the tokens of each sequence of a padded batch: from there on y is 0, the state
    stays, gradients are 0 and nothing in the inputs matters; values outside 0..seqlen count as the nearer end.

    Differentiable once, in every floating-point argument, the initial and the final state included.  States, sums over
    channels and parameters' gradients are float32, summed in a fixed order.  For the backward pass the state is kept every
    8 tokens (half of dstate, rounded up to 16, 32 or 64, bytes per token and channel).  To capture forward and backward into a CUDA graph let no
    eager graph of the same leaves be alive, as for every torch operator."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, dt, A, B, C, D, z, dt_bias, initial_state)):
        y, last = _SelectiveScan.apply(x, dt, A, B, C, D, z, dt_bias, bool(dt_softplus), initial_state, lengths)
    else:
        y, last, _ = _n().float_scan_fwd(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, lengths, return_final_state, False)
    return (y, last) if return_final_state else y


def selective_scan_update(state, x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, state_out=None):
    """One token per sequence: x, dt, z (batch, dim), B, C (batch, dstate) or (batch, groups, dstate), state float32
    (batch, dim, dstate), contiguous in its last dim.  Returns y (batch, dim); the state is advanced in place, or written to
    ``state_out`` when that is given (``state`` itself or memory that it shares nothing with).  Types and
    parameters as in :func:`selective_scan`; not differentiable."""
    return _n().float_scan_update(state, x, dt, A, B, C, D, z, dt_bias, dt_softplus, state_out)
