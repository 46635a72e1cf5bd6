"""What a network puts around a box convolution: the pointwise product (1 x 1 convolution, linear layer) with bias,
residual and activation in its epilogue, group norm with a residual and an activation, and what lies between two residual
blocks (a norm after the one, gate, residual add, a norm before the other). All work on channels-last data in float32, float16
or bfloat16, with gradients; sums and statistics are float32. For inference the product also comes in 8-bit floating point,
in blocks of 128 with a power of two each.

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
        raise RuntimeError("box_convolution: group_norm_act, linear_act and residual_norm can be differentiated once, not twice")


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
            raise RuntimeError("box_convolution: group_norm_act, linear_act and residual_norm have no forward-mode derivative")


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


class ResidualNormFunction(torch.autograd.Function):
    """``apply(input, residual, gate, after_weight, after_bias, before_weight, before_bias, gate_kind, scale, norms, eps, want_stream)``,
    tensors ``[B, ..., C]`` and parameters contiguous. Returns the stream (unless it is the input itself) and, with a norm
    before, the normed rows."""

    @staticmethod
    def forward(ctx, input, residual, gate, after_weight, after_bias, before_weight, before_bias, gate_kind, scale, norms, eps, want_stream):
        params = (after_weight, after_bias, before_weight, before_bias)
        *outputs, statistics = _native.residual_norm_forward(input, residual, gate, gate_kind, scale, norms, params, eps, want_stream, None, True)
        ctx.save_for_backward(input, residual, gate, *params, statistics)
        ctx.rest = gate_kind, scale, norms
        ctx.eps, ctx.want_stream = eps, want_stream
        ctx.set_materialize_grads(False)
        outputs = tuple(t for t in outputs if t is not None)
        return outputs if len(outputs) > 1 else outputs[0]

    @staticmethod
    def backward(ctx, *grad_outputs):
        given = [None if g is None else g.contiguous() for g in grad_outputs]
        _refuse_tangents(*grad_outputs)
        grad_stream = given.pop(0) if ctx.want_stream else None
        grad_normed = given.pop(0) if given else None
        input, residual, gate, *params, statistics = _contiguous(*ctx.saved_tensors)
        gate_kind, scale, norms = ctx.rest
        needs = [n and t is not None for n, t in zip(ctx.needs_input_grad, (input, residual, gate, *params))]
        grads = _native.residual_norm_backward(input, residual, gate, gate_kind, scale, norms, params, ctx.eps, statistics, grad_stream,
                                               grad_normed, needs)
        like = next((g for g in grad_outputs if g is not None), input)
        return (*_once(grads, input, like), None, None, None, None, None)


def _gate_kind(gate, input):
    if gate is None:
        return _native.GATE_NONE
    B, C = input.size(0), input.size(1)
    for kind, shape in ((_native.GATE_FULL, tuple(input.shape)), (_native.GATE_CHANNEL, (C,)), (_native.GATE_ITEM, (B, C))):
        if kind == _native.GATE_FULL and input.dim() == 2 and gate.dtype != input.dtype:
            continue                                   # (an input [B, C] has one value per item and channel itself)
        if tuple(gate.shape) == shape:
            if gate.device != input.device or gate.dtype not in ((input.dtype,) if kind == _native.GATE_FULL else (input.dtype, torch.float32)):
                raise RuntimeError("box_convolution: gate must be on %s, of the input's type or, where it is [C] or [B, C], float32" % input.device)
            return kind
    raise RuntimeError("box_convolution: gate must have the shape [C], [B, C] or that of the input, got %s for an input of %s"
                       % (tuple(gate.shape), tuple(input.shape)))


def _norm_pairs(input, after, before):
    """The four parameters, contiguous, of norms given as None or (weight, bias)."""
    out, kind = [], None
    for pair in (after, before):
        for p in pair or (None, None):
            if p is not None:
                if p.device != input.device or p.dim() != 1 or p.size(0) != input.size(1):
                    raise RuntimeError("box_convolution: the parameters of a norm must hold %d values on %s" % (input.size(1), input.device))
                if p.dtype not in (torch.float32, input.dtype) or kind not in (None, p.dtype):
                    raise RuntimeError("box_convolution: the norms' parameters must all be float32 or all of the input's type")
                kind = p.dtype
                p = p.contiguous()
            out.append(p)
    return out


def residual_norm(input, residual=None, gate=None, scale=1.0, after=None, before=None, kind="rms", eps=1e-6, quantize=False):
    """What lies between two blocks of a residual network, with gradients: ``input`` is what a block gives, ``residual`` the stream it
    is added to:

        ``stream = residual + scale * gate * norm(input; after)``,  ``normed = norm(stream; before)``.

    Returns ``(stream, normed)``, or the stream alone where there is no norm before the next block.

    input:    ``[B, C, ...]``; channels-last memory is used as it is, anything else is copied once. The results have channels-last memory.
    residual: same shape and type, or ``None`` for 0.
    gate:     ``None`` for 1, ``[C]`` (a layer scale), ``[B, C]`` (a gate per batch item) or of the input's shape; of the input's type, or
              float32 where it is ``[C]`` or ``[B, C]``.
    after, before: the norms behind this block and before the next one: ``None`` where there is none, or ``(weight, bias)``,
              each ``[C]`` or ``None`` for 1 and 0, all float32 or all of the input's type.
    kind:     ``"rms"``: ``v / sqrt(mean(v * v) + eps)`` over a row's channels; ``"layer"``: the same of ``v - mean(v)``.
    quantize: the normed rows as ``Float8Blocks``, for ``linear_act_float8`` (inference only: nothing here may require a gradient).

    Where nothing is done to the input (no residual, gate or norm behind the block, scale 1), the stream is the input itself.
    Statistics and sums are float32: a row with a value beyond 1.8e19, whose square float32 does not hold, has an infinite deviation, and is normalised to 0.
    ``normed`` is formed from the stream before it is rounded to the input's type.
    """
    _native._require_device(input, "residual norm input")
    if kind not in ("rms", "layer"):
        raise RuntimeError("box_convolution: kind must be 'rms' or 'layer', got %r" % (kind,))
    for name, pair in (("after", after), ("before", before)):
        if pair is not None and (not isinstance(pair, (tuple, list)) or len(pair) != 2):
            raise RuntimeError("box_convolution: %s must be None or a pair (weight, bias), either of which may be None" % name)
    glue = _native.glue()
    if glue is not None:                               # as in group_norm_act
        with _native._on_device(input.device):
            out = glue.residual_norm(input, residual, gate, scale, after is not None, *(after or (None, None)), before is not None,
                                     *(before or (None, None)), kind == "layer", eps, quantize, _native._stream(input.device) or 0)
        if before is None:
            return out[0]
        return out[0], Float8Blocks._of(out[1], out[2], input.size(1)) if quantize else out[1]
    _native._operator_dtype(input, "residual norm input")
    if input.dim() < 2 or input.size(1) < 1:
        raise RuntimeError("box_convolution: residual norm input must have >=2 dimensions and a channel")
    gate_kind = _gate_kind(gate, input)
    params = _norm_pairs(input, after, before)
    if residual is not None:
        _native._same_as(residual, input, "residual")
    tensors = (input, residual, gate, *params)
    _refuse_tangents(*tensors)
    norms = (_native.NORM_AFTER * (after is not None) | _native.NORM_BEFORE * (before is not None) | _native.NORM_CENTRE * (kind == "layer"))
    scale, eps = float(scale), float(eps)
    same = residual is None and gate is None and after is None and scale == 1.0
    recorded = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
    if quantize and (before is None or recorded):
        raise RuntimeError("box_convolution: quantize needs a norm before the next block, and is for inference only")
    if same and before is None:
        return input
    x = _channels_last(input)
    r = None if residual is None else _channels_last(residual)
    g = None if gate is None else _channels_last(gate) if gate_kind == _native.GATE_FULL else gate.contiguous()
    if recorded:
        outputs = ResidualNormFunction.apply(x, r, g, *params, gate_kind, scale, norms, eps, not same)
        outputs = list(outputs) if isinstance(outputs, tuple) else [outputs]
        stream, normed = None if same else outputs.pop(0), outputs.pop(0) if outputs else None
    else:
        blocks = None
        if quantize:
            codes, exponents = _native.block_sizes(x.size(-1))
            blocks = (torch.empty((*x.shape[:-1], codes), dtype=torch.float8_e4m3fn, device=x.device),
                      torch.empty((*x.shape[:-1], exponents), dtype=torch.uint8, device=x.device))
        stream, normed, _ = _native.residual_norm_forward(x, r, g, gate_kind, scale, norms, params, eps, not same, blocks)
        if quantize:
            normed = Float8Blocks._of(*blocks, x.size(-1))
    stream = input if same else stream.movedim(-1, 1)
    if before is None:
        return stream
    return stream, normed if quantize else normed.movedim(-1, 1)


class Float8Blocks:
    """Rows ``[..., columns]`` in 8-bit floating point (e4m3), a power of two for each block of 128 columns: value =
    ``codes * 2**(exponents - 127)``. ``codes``: ``[..., columns rounded up to 128]`` float8_e4m3fn, zeros beyond the columns;
    ``exponents``: ``[..., blocks rounded up to 4]`` uint8, from 1 to 254, 127 beyond the blocks. Both contiguous, on one device. What belongs together stays
    together: none of the three can be assigned (their values can be written in place)."""

    __slots__ = ("_codes", "_exponents", "_columns")           # read-only: kernels address codes and exponents by what was checked

    def __init__(self, codes, exponents, columns):
        self._codes, self._exponents, self._columns = codes, exponents, columns
        self._check()

    @classmethod
    def _of(cls, codes, exponents, columns):
        """Of tensors that an operator made: nothing to check."""
        self = object.__new__(cls)
        self._codes, self._exponents, self._columns = codes, exponents, columns
        return self

    def _check(self):
        """Raises unless the tensors are what the columns need. (Again in every call: tensors can be resized, and point to other memory later.)"""
        codes, exponents, columns = self._codes, self._exponents, self._columns
        width, words = _native.block_sizes(columns)
        if (codes.dtype != torch.float8_e4m3fn or exponents.dtype != torch.uint8 or codes.device != exponents.device or columns < 1
                or codes.dim() < 1 or codes.size(-1) != width or tuple(exponents.shape) != (*codes.shape[:-1], words)):
            raise RuntimeError("box_convolution: Float8Blocks needs float8_e4m3fn codes [..., %d] and uint8 exponents [..., %d] on one device for %d "
                               "columns, got %s %s and %s %s" % (width, words, columns, codes.dtype, tuple(codes.shape), exponents.dtype, tuple(exponents.shape)))
        if not codes.is_contiguous() or not exponents.is_contiguous() or codes.data_ptr() % 16 or exponents.data_ptr() % 4:
            raise RuntimeError("box_convolution: the codes and exponents of Float8Blocks must be contiguous, at addresses of whole 16 and 4 bytes")

    codes = property(lambda self: self._codes)
    exponents = property(lambda self: self._exponents)
    columns = property(lambda self: self._columns)

    @property
    def shape(self):
        return torch.Size((*self.codes.shape[:-1], self.columns))

    @property
    def device(self):
        return self.codes.device

    def to(self, device):
        return Float8Blocks(self.codes.to(device), self.exponents.to(device), self.columns)

    def dequantize(self, dtype=torch.float32):
        """The values, ``[..., columns]`` (elementary torch operations: to look at, not for a fast path). Of float32 and narrower types those above the type's
        largest are infinite: a value next to float32's own largest may be rounded up to 2**128."""
        wide = torch.float64 if dtype == torch.float64 else torch.float32
        blocks = self.codes.to(wide).unflatten(-1, (-1, _native.BLOCK))
        # 2**(exponent - 127), put together from its bits
        power = (self.exponents[..., :blocks.size(-2)].int() << 23).view(torch.float32).to(wide)
        return (blocks * power[..., None]).flatten(-2)[..., :self.columns].to(dtype)


def quantize_blocks(input):
    """``[..., K]`` values in float32, float16 or bfloat16 as ``Float8Blocks``: per block of 128 the least power of two (from 2**-126 on) that
    keeps its largest finite magnitude at or below 448 times it; values rounded to nearest, ties to even, once. NaN and infinities
    become NaN and leave the rest of their block alone. Not differentiable: an input that requires a gradient is refused while
    gradients are recorded."""
    _native._require_device(input, "quantize input")
    glue = _native.glue()
    if glue is not None:                               # as in group_norm_act
        with _native._on_device(input.device):
            return Float8Blocks._of(*glue.quantize_blocks(input, _native._stream(input.device) or 0), input.size(-1))
    _native._operator_dtype(input, "quantize input")
    if input.dim() < 1 or input.size(-1) < 1:
        raise RuntimeError("box_convolution: quantize_blocks needs an input [..., K] with at least one column")
    _refuse_gradients("quantize_blocks", input)
    codes, exponents = _native.quantize_blocks(_rows(input, math.prod(input.shape[:-1]), input.size(-1)))
    return Float8Blocks._of(codes.view(*input.shape[:-1], codes.size(-1)), exponents.view(*input.shape[:-1], exponents.size(-1)), input.size(-1))


def _refuse_gradients(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("box_convolution: %s is for inference only: it has no gradient (call it under torch.no_grad())" % what)
    _refuse_tangents(*tensors)


def linear_act_float8(input, weight, bias=None, residual=None, activation=None, dtype=None):
    """``act(input @ weight.T + bias + residual)`` of 8-bit rows, for inference: see ``linear_act`` for training.

    input:    ``Float8Blocks`` ``[..., K]``, or values ``[..., K]``, which are quantized on the way as by ``quantize_blocks``.
    weight:   ``Float8Blocks`` ``[N, K]`` (``quantize_blocks(weight)``, once).
    bias:     ``[N]``; residual ``[..., N]``, added before the activation: both of the result's type.
    activation: ``None``, ``"relu"``, ``"silu"`` or ``"gelu"``.
    dtype:    the result's type: that of the values; for ``Float8Blocks`` float32, float16 or bfloat16 (default).

    float32 results: products of codes and powers of two are exact, sums are float32. float16 and bfloat16 results come from the matrix instructions of
    the 8-bit format, which cut each product, towards zero, to a multiple of 2**-13 of the largest among 8 neighbouring columns (columns 0 to 7, 8 to 15, ...)
    before they add them up in float32: where large products cancel, small ones beside them are lost. A float32 result of ``Float8Blocks`` has none of that,
    at half the speed or less.
    """
    act = _native._activation(activation)
    coded = isinstance(input, Float8Blocks)
    rows_of = input.codes if coded else input
    _native._require_device(rows_of, "linear float8 input")
    if not isinstance(weight, Float8Blocks):
        raise RuntimeError("box_convolution: weight must be Float8Blocks (quantize_blocks(weight)), got %s" % type(weight).__name__)
    glue = _native.glue()
    if glue is not None:                               # as in group_norm_act
        with _native._on_device(rows_of.device):
            return glue.linear_act_float8(rows_of, input.exponents if coded else None, input.columns if coded else input.shape[-1] if input.dim() else 0,
                                          weight.codes, weight.exponents, weight.columns, bias, residual, act, dtype, _native._stream(rows_of.device) or 0)
    if not coded:
        _native._operator_dtype(input, "linear float8 input")
    for blocks in (input, weight) if coded else (weight,):
        blocks._check()
    dtype = dtype or (torch.bfloat16 if coded else input.dtype)
    if dtype not in _native._FUSED_OUTPUT or (not coded and dtype != input.dtype):
        raise RuntimeError("box_convolution: the result's type must be that of the values, or float32, float16 or bfloat16 for Float8Blocks, got %s" % dtype)
    if len(input.shape) < 1 or len(weight.shape) != 2 or weight.columns != input.shape[-1] or weight.device != rows_of.device:
        raise RuntimeError("box_convolution: linear float8 needs an input [..., K] and a weight [N, K] on one device, got %s and %s"
                           % (tuple(input.shape), tuple(weight.shape)))
    N, K = weight.shape
    out_shape = (*input.shape[:-1], N)
    for name, t, shape in (("bias", bias, (N,)), ("residual", residual, out_shape)):
        if t is not None and (t.device != rows_of.device or t.dtype != dtype or tuple(t.shape) != shape):
            raise RuntimeError("box_convolution: %s must have the shape %s, type %s and device %s, got %s, %s, %s"
                               % (name, shape, dtype, rows_of.device, tuple(t.shape), t.dtype, t.device))
    _refuse_gradients("linear_act_float8", None if coded else input, bias, residual)
    rows = math.prod(out_shape[:-1])
    x = input.codes.view(rows, weight.codes.size(-1)) if coded else _rows(input, rows, K)
    exponents = input.exponents.view(rows, weight.exponents.size(-1)) if coded else None
    y = _native.linear_float8_forward(x, exponents, weight.codes, weight.exponents, K,
                                      None if bias is None else bias.contiguous(), None if residual is None else _rows(residual, rows, N), activation, dtype)
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


class ResidualNorm(torch.nn.Module):
    """``residual_norm`` with its parameters: ``module(x, residual=None, gate=None)`` for ``[B, channels, ...]``.

    after, before: whether there is a norm behind the block and one before the next; ``kind`` "rms" (weights) or "layer" (weights and
    biases). layer_scale: the initial value of a learned gate per channel, ``None`` for none; it excludes a gate in the call.
    Parameters may be float32 beside inputs in half precision."""

    def __init__(self, channels, after=True, before=True, kind="rms", scale=1.0, layer_scale=None, eps=1e-6, device=None, dtype=None):
        super().__init__()
        if kind not in ("rms", "layer"):
            raise RuntimeError("box_convolution: kind must be 'rms' or 'layer', got %r" % (kind,))
        self.channels, self.kind, self.scale, self.eps = channels, kind, scale, eps

        def parameter(value):
            return torch.nn.Parameter(torch.full((channels,), float(value), device=device, dtype=dtype))
        for name, there in (("after", after), ("before", before)):
            setattr(self, name, there)
            self.register_parameter(name + "_weight", parameter(1) if there else None)
            self.register_parameter(name + "_bias", parameter(0) if there and kind == "layer" else None)
        self.register_parameter("layer_scale", None if layer_scale is None else parameter(layer_scale))

    def forward(self, input, residual=None, gate=None, quantize=False):
        if gate is not None and self.layer_scale is not None:
            raise RuntimeError("ResidualNorm: a gate and a layer scale exclude each other")
        return residual_norm(input, residual, self.layer_scale if gate is None else gate, self.scale,
                             (self.after_weight, self.after_bias) if self.after else None,
                             (self.before_weight, self.before_bias) if self.before else None, self.kind, self.eps, quantize)

    def extra_repr(self):
        return "%d, after=%r, before=%r, kind=%r, scale=%r, eps=%r" % (self.channels, self.after, self.before, self.kind, self.scale, self.eps)


class PointwiseConv2dFloat8(torch.nn.Module):
    """The inference form of a ``PointwiseConv2d`` (or 1 x 1 ``torch.nn.Conv2d``) in 8 bits: ``PointwiseConv2dFloat8(conv)`` quantizes its
    weight once; ``module(x, residual=None)`` takes ``[B, C, h, w]`` values of the bias's type, or the ``Float8Blocks`` ``[B, h, w, C]``
    of a quantizing ``ResidualNorm``, and returns ``[B, out_channels, h, w]`` in channels-last memory, of the values' type, or the bias's
    (without a bias, the convolution's) for blocks. Codes (as bytes), exponents and bias are buffers."""

    def __init__(self, conv, activation=None):
        super().__init__()
        if (not isinstance(conv, torch.nn.Conv2d) or conv.kernel_size != (1, 1) or conv.stride != (1, 1) or conv.padding not in ((0, 0), "valid")
                or conv.groups != 1):
            raise RuntimeError("PointwiseConv2dFloat8: needs a 1 x 1 convolution without stride, padding and groups")
        _native._activation(activation)
        self.activation = activation or getattr(conv, "activation", None)
        self.in_channels, self.out_channels, self.dtype = conv.in_channels, conv.out_channels, conv.weight.dtype
        with torch.no_grad():
            weight = quantize_blocks(conv.weight.flatten(1))
        self.register_buffer("codes", weight.codes.view(torch.uint8))        # (as bytes: module.to(dtype) converts floating-point buffers)
        self.register_buffer("exponents", weight.exponents)
        self.register_buffer("bias", None if conv.bias is None else conv.bias.detach().clone())

    def forward(self, input, residual=None):
        coded = isinstance(input, Float8Blocks)
        if len(input.shape) != 4:
            raise RuntimeError("PointwiseConv2dFloat8: input must have 4 dimensions")
        weight = Float8Blocks(self.codes.view(torch.float8_e4m3fn), self.exponents, self.in_channels)
        dtype = None if not coded else self.dtype if self.bias is None else self.bias.dtype
        y = linear_act_float8(input if coded else input.permute(0, 2, 3, 1), weight, self.bias, None if residual is None else residual.permute(0, 2, 3, 1),
                              self.activation, dtype)
        return y.permute(0, 3, 1, 2)

    def extra_repr(self):
        return "%d, %d, bias=%r, activation=%r" % (self.in_channels, self.out_channels, self.bias is not None, self.activation)
