"""The dense layers around the routed experts: a gated feed-forward block with its gradients, and linear layers with 8-bit and
4-bit weights, over the library's calls (_native.ffn_forward / ffn_backward / linear_i8 / linear_i4 / linear_i4_dx).

They hold plain torch tensors and run on torch's current stream of their device; every call takes its workspace from
torch's allocator, so calls on several streams and captured graphs share nothing but the weights.
"""
import torch
from torch.autograd import forward_ad

import _native


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, act_limit):
        out, g, u = _native.ffn_forward(x, wg, wu, wd, act_limit=act_limit, save=True)
        ctx.save_for_backward(x, g, u, wg, wu, wd)
        ctx.act_limit = act_limit
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, g, u, wg, wu, wd = ctx.saved_tensors
        _no_capture(x, "gated_ffn", "backward", _FFN_HOW)
        # dy may be a broadcast (of a sum) or a view with other strides
        return _native.ffn_backward(dy.contiguous(), x, g, u, wg, wu, wd, act_limit=ctx.act_limit,
                                    need=ctx.needs_input_grad[:4]) + (None,)


_FFN_HOW = "_native.ffn_forward(save=True) and ffn_backward"


def _no_capture(x, who, what, how):
    # autograd accumulates into .grad on the streams of nodes made before the capture, which ends the process when they
    # wait for a captured event
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{who}: no {what} with gradients in a stream capture: capture {how}, with gradients in tensors of "
                           "your own")


def _no_tangents(who, *inputs):
    # a dual tensor need not have requires_grad, and the library's calls do not see its tangent
    if any(forward_ad.unpack_dual(t).tangent is not None for t in inputs):
        raise RuntimeError(f"{who}: no forward-mode differentiation: an input has a tangent, which would be dropped")


def gated_ffn(x, wg, wu, wd, act_limit=0.0):
    """_native.ffn_forward's block, differentiable: x fp16 or bf16 [..., H], wg and wu [I, H], wd [H, I] of its type. Keeps
    8 bytes a token and I channel (g and u in fp32) for the backward where a gradient is wanted. Once differentiable, in reverse
    mode: refuses inputs with tangents, and stream capture with gradients (RuntimeError)."""
    _no_tangents("gated_ffn", x, wg, wu, wd)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, wg, wu, wd)):
        _no_capture(x, "gated_ffn", "forward", _FFN_HOW)
        return _GatedFFN.apply(x, wg, wu, wd, float(act_limit))
    return _native.ffn_forward(x, wg, wu, wd, act_limit=act_limit)


class Linear8:
    """A linear layer with 8-bit weights and one scale per output channel, its tokens quantised per token as they come
    (_native.linear_i8): an output head of V x H takes half the bytes of fp16."""

    def __init__(self, weight):
        """weight fp16 or bf16 [N, K] on the device; K up to 131071 (32-bit sums)."""
        if weight.dim() != 2 or not 0 < weight.shape[1] <= 131071:
            raise ValueError(f"Linear8: weight must be [N, K] with K in 1..131071, not {list(weight.shape)}")
        self.weight, self.scale = _native.quant_i8(weight.detach())

    def __call__(self, x, out=None, dtype=None):
        """x fp16 or bf16 [..., K] -> [..., N] in `dtype` (x's by default), or into `out`. Has no gradient: an x or out that
        requires one, or an x with a tangent, is refused (RuntimeError); call it under torch.no_grad() or on x.detach()."""
        if torch.is_grad_enabled() and (x.requires_grad or (out is not None and out.requires_grad)):
            raise RuntimeError("Linear8: rounding to 8 bits has no gradient, and this call would drop the one that is asked "
                               "for: call it under torch.no_grad() or on x.detach()")
        _no_tangents("Linear8", x)
        return _native.linear_i8(x, self.weight, self.scale, out=out, dtype=dtype)


class _Linear4(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, layer):
        ctx.layer = layer
        return _native.linear_i4(x, layer.q, layer.scale, zero=layer.zero, group=layer.group)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _no_capture(dy, "Linear4", "backward", _I4_HOW)
        layer = ctx.layer
        return _native.linear_i4_dx(dy.contiguous(), layer.q, layer.scale, layer.K, zero=layer.zero, group=layer.group), None


_I4_HOW = "_native.linear_i4 and linear_i4_dx"


class Linear4:
    """A linear layer with 4-bit weights, a scale (and, with zeros, a zero point) for each `group` inputs of an output channel: half
    the bytes of 8 bits, and tokens that stay as they are (_native.linear_i4). Frozen: the gradient goes on to its input, for
    adapters and layers before it."""

    def __init__(self, weight, group=128, zeros=False):
        """weight fp16 or bf16 [N, K] on the device; group 32, 64 or 128."""
        if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
            raise ValueError(f"Linear4: weight must be [N, K], not {list(weight.shape)}")
        self.q, self.scale, self.zero = _native.quant_i4(weight.detach(), group=group, zeros=zeros)
        self.K, self.group = weight.shape[1], int(group)

    @classmethod
    def from_values(cls, values, scale, zero=None, group=128):
        """From a checkpoint's own rounding: values uint8 [N, K] of 0..15, scale fp16 or bf16 [ceil(K / group), N], zero uint8 like
        scale (None: 8)."""
        layer = cls.__new__(cls)
        if values.dim() != 2 or group not in (32, 64, 128):
            raise ValueError(f"Linear4: values must be [N, K] and group 32, 64 or 128, not {list(values.shape)} and {group}")
        layer.K, layer.group, layer.zero = values.shape[1], int(group), zero
        want = ((layer.K + layer.group - 1) // layer.group, values.shape[0])
        for name, t in (("scale", scale), ("zero", zero)):
            if t is not None and tuple(t.shape) != want:
                raise ValueError(f"Linear4: {name} must be {list(want)} for values {list(values.shape)}, group {group}, not "
                                 f"{list(t.shape)}")
        layer.q, layer.scale = _native.pack_i4(values), scale.detach()
        return layer

    def __call__(self, x, out=None, dtype=None):
        """x fp16 or bf16 [..., K] -> [..., N] in `dtype` (x's by default), or into `out`. Differentiable in x once, in reverse mode,
        where the output is a new one of x's type; other calls that ask for a gradient, tangents and stream capture with
        gradients are refused (RuntimeError)."""
        _no_tangents("Linear4", x)
        if torch.is_grad_enabled() and (x.requires_grad or (out is not None and out.requires_grad)):
            if out is not None or dtype not in (None, x.dtype):
                raise RuntimeError("Linear4: an out, or a dtype that is not x's, has no gradient, and this call would drop the one "
                                   "that is asked for: call it under torch.no_grad() or on x.detach()")
            _no_capture(x, "Linear4", "forward", _I4_HOW)
            return _Linear4.apply(x, self)
        return _native.linear_i4(x, self.q, self.scale, zero=self.zero, group=self.group, out=out, dtype=dtype)
