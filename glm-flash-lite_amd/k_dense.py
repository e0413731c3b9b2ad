"""The dense layers around the routed experts: a gated feed-forward block with its gradients, and a linear layer with 8-bit
weights, over the library's calls (_native.ffn_forward / ffn_backward / linear_i8).

Both hold plain torch tensors and run on torch's current stream of their device; every call takes its workspace from
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
        _no_capture(x, "backward")
        # dy may be a broadcast (of a sum) or a view with other strides
        return _native.ffn_backward(dy.contiguous(), x, g, u, wg, wu, wd, act_limit=ctx.act_limit,
                                    need=ctx.needs_input_grad[:4]) + (None,)


def _no_capture(x, what):
    # autograd accumulates into .grad on the streams of nodes made before the capture, which ends the process when they
    # wait for a captured event
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"gated_ffn: no {what} with gradients in a stream capture: capture _native.ffn_forward(save=True) "
                           "and ffn_backward, with gradients in tensors of your own")


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
        _no_capture(x, "forward")
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
