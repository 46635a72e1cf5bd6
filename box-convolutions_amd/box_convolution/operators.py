"""What a network puts around a box convolution: the pointwise product (1 x 1 convolution, linear layer) with bias,
residual and activation in its epilogue, and group norm with a residual and an activation. Both work on channels-last
data in float32, float16 or bfloat16, with gradients; sums and statistics are float32.

(The reference builds such a block from torch's own layers: BottleneckBoxConv,
examples/Cityscapes/models/ENet.py:282-304.)
"""
import math

import torch

from . import _native


def _channels_last(t):
    """The ``[B, ..., C]`` view of a ``[B, C, ...]`` tensor; a copy where its memory is laid out otherwise."""
    t = t.movedim(1, -1)
    return t if t.is_contiguous() else t.contiguous()


class _OnceFunction(torch.autograd.Function):
    """``apply(grad, *of)``: ``grad``, with a node that refuses to be differentiated."""

    @staticmethod
    def forward(ctx, grad, *of):
        return grad.detach()

    @staticmethod
    def backward(ctx, grad_output):
        raise RuntimeError("box_convolution: group_norm_act and linear_act can be differentiated once, not twice")


def _once(grads, x, grad_output):
    """The gradients of a backward pass. They come from kernels that leave no graph: where one is asked for, they must
    not count as constants."""
    if not torch.is_grad_enabled():
        return grads
    needs_grad = torch.empty(0, device=x.device, requires_grad=True)
    return tuple(g if g is None else _OnceFunction.apply(g, x, grad_output, needs_grad) for g in grads)


def _refuse_tangents(*tensors):
    """Neither the kernels nor the autograd functions know forward-mode derivatives: a tangent is refused, since dropping
    it would make it zero."""
    for t in tensors:
        if t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("box_convolution: group_norm_act and linear_act have no forward-mode derivative")


def _contiguous(*tensors):
    """What was saved, as the kernels take it: hooks on saved tensors may hand the values back in any memory order."""
    return [None if t is None else t.contiguous() for t in tensors]


class GroupNormActFunction(torch.autograd.Function):
    """``apply(input, weight, bias, residual, num_groups, activation, eps)``, tensors ``[B, ..., C]``, contiguous."""

    @staticmethod
    def forward(ctx, input, weight, bias, residual, num_groups, activation, eps):
        output, mean, rstd = _native.group_norm_forward(input, num_groups, weight, bias, residual, activation, eps, True)
        # (the residual moves the point at which the activation's derivative is taken, and nothing else)
        ctx.save_for_backward(input, weight, bias, residual if activation is not None else None, mean, rstd)
        ctx.num_groups, ctx.activation = num_groups, activation
        return output

    @staticmethod
    def backward(ctx, grad_output):
        _refuse_tangents(grad_output)
        input, weight, bias, residual, mean, rstd = _contiguous(*ctx.saved_tensors)
        grads = _native.group_norm_backward(
            input, ctx.num_groups, weight, bias, residual, ctx.activation, mean, rstd, grad_output.contiguous(),
            ctx.needs_input_grad[:4])
        return (*_once(grads, input, grad_output), None, None, None)


def group_norm_act(input, num_groups, weight=None, bias=None, residual=None, activation=None, eps=1e-5):
    """``act(group_norm(input) * weight + bias + residual)`` with gradients.

    input:      ``[B, C, ...]``; channels-last memory (``torch.channels_last`` for images) is used as it
                is, anything else is copied once (planes, as ``BoxConv2d`` returns them: the copy takes two to three times
                the norm's own time). The result has channels-last memory, and so has the gradient.
    weight, bias: ``[C]``, both float32 or both of the input's type; ``None`` is 1 and 0.
    residual:   same shape and type as ``input``, added before the activation.
    activation: ``None``, ``"relu"``, ``"silu"`` or ``"gelu"``.
    """
    act = _native._activation(activation)
    _native._require_device(input, "group norm input")
    glue = _native.glue()
    if glue is not None:
        # checks, allocations and the autograd node in C++ (csrc/operators_glue.hpp): what follows, with less host time
        with _native._on_device(input.device):
            return glue.group_norm_act(input, num_groups, weight, bias, residual, act, eps, _native._stream(input.device) or 0)
    _native._operator_dtype(input, "group norm input")
    _refuse_tangents(input, weight, bias, residual)
    if input.dim() < 2:
        raise RuntimeError("box_convolution: group norm input must have >=2 dimensions")
    if num_groups < 1 or input.size(1) < 1 or input.size(1) % num_groups != 0:
        raise RuntimeError("box_convolution: %d channels cannot be split into %d groups" % (input.size(1), num_groups))
    _native._norm_parameters(input, input.size(1), weight, bias)
    x, r = _channels_last(input), None
    if residual is not None:
        r = _channels_last(_native._same_as(residual, input, "residual"))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (input, weight, bias, residual)):
        y = GroupNormActFunction.apply(x, weight, bias, r, num_groups, activation, eps)
    else:
        y = _native.group_norm_forward(x, num_groups, weight, bias, r, activation, eps, False)[0]
    return y.movedim(-1, 1)


def _rows(t, rows, width):
    """``[rows, width]`` view of a ``[..., width]`` tensor with contiguous rows any distance apart; a copy where its memory
    is laid out otherwise."""
    t = t.reshape(rows, width) if t.dim() != 2 else t
    return t if t.stride(1) == 1 or width == 1 else t.contiguous()


class LinearActFunction(torch.autograd.Function):
    """``apply(input, weight, bias, residual, activation)``, input ``[rows, K]`` and residual ``[rows, N]`` with contiguous
    rows."""

    @staticmethod
    def forward(ctx, input, weight, bias, residual, activation):
        output, kept = _native.linear_forward(input, weight, bias, residual, activation, any(ctx.needs_input_grad))
        ctx.save_for_backward(input, weight, kept)
        ctx.activation = activation
        return output

    @staticmethod
    def backward(ctx, grad_output):
        _refuse_tangents(grad_output)
        input, weight, kept = ctx.saved_tensors
        input, (weight, kept) = _rows(input, *input.shape), _contiguous(weight, kept)
        grads = _native.linear_backward(input, weight, kept, ctx.activation, grad_output.contiguous(), ctx.needs_input_grad[:4])
        return (*_once(grads, input, grad_output), None)


def linear_act(input, weight, bias=None, residual=None, activation=None):
    """``act(input @ weight.T + bias + residual)`` with gradients.

    input:      ``[..., K]``; rows may lie apart (a slice of wider rows is not copied).
    weight:     ``[N, K]``; bias ``[N]``; residual ``[..., N]``, added before the activation: all of the input's type.
    activation: ``None``, ``"relu"``, ``"silu"`` or ``"gelu"``.

    Sums are float32. For float16 and bfloat16 the gradient in front of the activation is rounded to the input's type before it is
    multiplied by weight and input, as it would be between two layers.
    """
    act = _native._activation(activation)
    _native._require_device(input, "linear input")
    glue = _native.glue()
    if glue is not None:                               # as in group_norm_act
        with _native._on_device(input.device):
            return glue.linear_act(input, weight, bias, residual, act, _native._stream(input.device) or 0)
    _native._operator_dtype(input, "linear input")
    _refuse_tangents(input, weight, bias, residual)
    if input.dim() < 1 or weight.dim() != 2 or weight.size(1) != input.size(-1):
        raise RuntimeError("box_convolution: linear needs an input [..., K] and a weight [N, K], got %s and %s"
                           % (tuple(input.shape), tuple(weight.shape)))
    N, K = weight.shape
    for name, t, shape in (("weight", weight, (N, K)), ("bias", bias, (N,)),
                           ("residual", residual, tuple(input.shape[:-1]) + (N,))):
        if t is not None and (t.device != input.device or t.dtype != input.dtype or tuple(t.shape) != shape):
            raise RuntimeError("box_convolution: %s must have the shape %s, type %s and device %s, got %s, %s, %s"
                               % (name, shape, input.dtype, input.device, tuple(t.shape), t.dtype, t.device))
    out_shape = (*input.shape[:-1], N)
    rows = math.prod(out_shape[:-1])
    x, r = _rows(input, rows, K), None if residual is None else _rows(residual, rows, N)
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (input, weight, bias, residual)):
        y = LinearActFunction.apply(x, weight, bias, r, activation)
    else:
        y = _native.linear_forward(x, weight, bias, r, activation, False)[0]
    return y.view(out_shape)


class GroupNormAct(torch.nn.GroupNorm):
    """``torch.nn.GroupNorm`` (same arguments and parameters, so state dicts interchange) followed by a residual add
    and an activation in the same kernels: ``module(x, residual=None)``. See ``group_norm_act``."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation=None, device=None, dtype=None):
        super().__init__(num_groups, num_channels, eps, affine, device=device, dtype=dtype)
        _native._activation(activation)
        self.activation = activation

    def forward(self, input, residual=None):
        return group_norm_act(input, self.num_groups, self.weight, self.bias, residual, self.activation, self.eps)

    def extra_repr(self):
        return super().extra_repr() + ", activation=%r" % (self.activation,)


class PointwiseConv2d(torch.nn.Conv2d):
    """A 1 x 1 ``torch.nn.Conv2d`` (same parameters, so state dicts interchange) with a residual add and an activation in
    the same kernel: ``module(x, residual=None)``. The output has channels-last memory; so should the input (see
    ``linear_act``; other layouts are copied). Parameters have the input's type, under ``torch.autocast`` too: nothing is cast."""

    def __init__(self, in_channels, out_channels, bias=True, activation=None, device=None, dtype=None):
        super().__init__(in_channels, out_channels, 1, bias=bias, device=device, dtype=dtype)
        _native._activation(activation)
        self.activation = activation

    def forward(self, input, residual=None):
        if input.dim() != 4:
            raise RuntimeError("PointwiseConv2d: input must have 4 dimensions")
        y = linear_act(input.permute(0, 2, 3, 1), self.weight.flatten(1), self.bias,
                       None if residual is None else residual.permute(0, 2, 3, 1), self.activation)
        return y.permute(0, 3, 1, 2)

    def extra_repr(self):
        return super().extra_repr() + ", activation=%r" % (self.activation,)
