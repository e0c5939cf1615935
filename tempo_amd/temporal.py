"""Differentiable operators of a temporal head on channel-last features.

The reference carries features over time with a GRU (``tempo/models/fiery_temporal.py:109``,
used at ``tempo/models/model_utils.py:10-16``), one step after the other.  Here the gates depend
on the input alone, so that the recurrence is linear and runs over a whole sequence in one pass.

Everything runs in HIP kernels on the current stream; there is no CPU path.  The backward
passes use no atomics: gradients do not change from run to run.  There are no forward-mode
derivatives; asking for one raises.
"""
import torch
from torch.autograd.function import once_differentiable

from . import ops


def _records(*tensors):
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad
                                           for t in tensors)


class _GatedRecurrence(torch.autograd.Function):

    @staticmethod
    def forward(ctx, gate, value, state, lengths):
        h, last, ckpt = ops.recurrence_forward(gate, value, state, lengths, want_ckpt=True)
        # beyond one span the stored states replace the initial one
        ctx.save_for_backward(gate, value, state if ckpt is None else None, ckpt, lengths)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_last):
        if grad_h is None and grad_last is None:
            return None, None, None, None
        gate, value, state, ckpt, lengths = ctx.saved_tensors
        need = ctx.needs_input_grad
        if grad_h is not None and grad_h.stride(2) != 1:
            grad_h = grad_h.contiguous()
        if grad_last is not None:
            grad_last = grad_last.contiguous()
        dgate, dvalue, dstate = ops._recurrence_backward(grad_h, grad_last, gate, value, state,
                                                         ckpt, lengths, need[2])
        return (dgate if need[0] else None, dvalue if need[1] else None,
                dstate if need[2] else None, None)


def gated_recurrence(gate, value=None, state=None, lengths=None, out=None, state_out=None):
    """Gated linear recurrence over time, ``h_t = (1 - z_t) h_{t-1} + z_t v_t`` with
    ``z = sigmoid(gate)``: a GRU's update with gates from the input alone.

    ``gate``, ``value``: ``[B,T,D]`` in fp32, fp16 or bf16, channels adjacent, any strides over
    B and T (a transposed ``[T,B,D]`` tensor is read where it lies).  Without ``value``,
    ``gate`` is ``[B,T,2D]`` with gate and value side by side, as one product leaves them.
    ``state``: fp32 ``[B,D]``, the state before the first step (default: zeros).
    ``lengths``: int32 ``[B]`` on the device; rows ``t >= lengths[b]`` are padding: not read,
    0 in the result and in the gradients (values outside ``[0,T]`` count as the nearer end).

    Returns ``(h [B,T,D], last [B,D])``: every state in the inputs' type and the fp32 state
    after the last step, to go on from (a serving loop passes T = 1 and the carried state).
    Differentiable once, with respect to ``gate``, ``value`` and ``state``.  States and sums are
    fp32.  An infinity among the inputs leaves its channel's later states infinite or NaN, as does
    a value whose difference from the state in front of it is beyond fp32's range.

    ``out`` / ``state_out`` (not under autograd): where to write the two results, apart from the
    inputs in memory and no row over another; only ``state_out`` may be ``state`` itself.

    To capture a training step into a graph, drop eager results of the same leaves first: torch
    itself ends the process when a captured backward meets their gradient accumulators."""
    if _records(gate, value, state, out, state_out):
        if out is not None or state_out is not None:
            raise NotImplementedError('gated_recurrence: out / state_out are for calls without '
                                      'gradients (torch.no_grad() or detached tensors)')
        return _GatedRecurrence.apply(gate, value, state, lengths)
    h, last, _ = ops.recurrence_forward(gate, value, state, lengths, out, state_out)
    return h, last


class _FusedLinear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, pre = ops.linear_forward(x, weight, bias, residual, activation, want_pre=True)
        ctx.save_for_backward(x, weight, pre)
        ctx.activation = ops.ACTIVATIONS[activation]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = ops._linear_backward(grad_y, x, weight, pre, ctx.activation, need)
        return dx, dw, db, grad_y if need[3] else None, None


def fused_linear(x, weight, bias=None, residual=None, activation='none', out=None):
    """``act(x W^T + bias) + residual`` in one pass over memory: a 1x1 convolution of
    channel-last maps with its epilogue.

    ``x``: ``[..., K]`` in fp32, fp16 or bf16, channels adjacent and rows at one distance from
    each other (a ``torch.channels_last`` map is ``map.permute(0, 2, 3, 1)``); ``weight``
    ``[N,K]`` or a convolution's ``[N,K,1,1]``; ``bias`` ``[N]``; ``residual`` ``[..., N]``, all
    of x's type.  ``activation``: none, relu, silu, gelu (with the normal distribution itself),
    sigmoid or tanh.  Returns ``[..., N]``.

    Sums are fp32, the result is rounded once; fp32 inputs are multiplied in fp32.
    Differentiable once, with respect to every tensor; for the backward pass the value in front
    of the activation is kept in x's type, as a layer's output would be.  relu's slope is that of
    the sum as computed: 0 or 1 where the sum lies within its rounding of 0.  ``out`` (not under
    autograd): where to write the result; it may be the residual (the same memory in the same
    order), but share none with the other inputs.

    To capture a training step into a graph, drop eager results of the same leaves first: torch
    itself ends the process when a captured backward meets their gradient accumulators."""
    if isinstance(weight, torch.Tensor) and weight.dim() == 4 and weight.shape[2:] == (1, 1):
        weight = weight.flatten(1)
    if _records(x, weight, bias, residual, out):
        if out is not None:
            raise NotImplementedError('fused_linear: out is for calls without gradients '
                                      '(torch.no_grad() or detached tensors)')
        return _FusedLinear.apply(x, weight, bias, residual, activation)
    return ops.linear_forward(x, weight, bias, residual, activation, out)[0]
