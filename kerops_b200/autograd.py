"""Autograd wiring of the depthwise 3x3x3 convolution: forward, input gradient and weight gradient.

The reference ships the forward and the weight-gradient operators but no input gradient and no
autograd.Function (a TODO at kerops/kernels/dw_conv.py:145 plans a fused backward).  The input gradient of a
stride-1, pad-1 cross-correlation is the same cross-correlation of the upstream gradient with the taps flipped
on all three axes, so it runs on the forward kernel unchanged.
"""
import torch

from .ops.conv import DWConv, DWConvWGRAD
from .ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD
from .ops.linear.grouped_linear import grouped_linear_grads


def DWConvDGRAD(grad, weight, *, ACCTYPE='float32'):
    """Input gradient: dx[n,c,h,w,d] = sum_{a,b,t} grad[n,c,h-a+1,w-b+1,d-t+1] * weight[a,b,t,c].

    grad    (N, C, H, W, D) fp16 CUDA tensor, channels_last_3d
    weight  [3, 3, 3, C] fp16 (kerops layout)
    """
    flipped = torch.flip(weight, dims=(0, 1, 2)).contiguous()
    return DWConv(grad, flipped, ACCTYPE=ACCTYPE)


class DepthwiseConv3dFunction(torch.autograd.Function):
    """y = DWConv(x, weight) with gradients for both arguments."""

    @staticmethod
    def forward(ctx, x, weight):
        ctx.save_for_backward(x, weight)
        return DWConv(x, weight)

    @staticmethod
    def backward(ctx, grad_out):
        x, weight = ctx.saved_tensors
        if not grad_out.is_contiguous(memory_format=torch.channels_last_3d):
            grad_out = grad_out.contiguous(memory_format=torch.channels_last_3d)
        grad_x = DWConvDGRAD(grad_out, weight) if ctx.needs_input_grad[0] else None
        grad_w = DWConvWGRAD(x, grad_out) if ctx.needs_input_grad[1] else None
        return grad_x, grad_w


def depthwise_conv3d(x, weight):
    """Differentiable depthwise 3x3x3 convolution (stride 1, zero padding 1, no bias)."""
    return DepthwiseConv3dFunction.apply(x, weight)


class DepthwiseConv3d(torch.nn.Module):
    """Module form; the parameter is kept in the kerops layout [3, 3, 3, C], fp16."""

    def __init__(self, channels, device=None):
        super().__init__()
        bound = 1.0 / 27 ** 0.5  # kaiming_uniform_(a=sqrt(5)) on a (C, 1, 3, 3, 3) weight
        w = (torch.rand(3, 3, 3, channels, device=device) * 2 - 1) * bound
        self.weight = torch.nn.Parameter(w.to(torch.float16))

    def forward(self, x):
        return depthwise_conv3d(x, self.weight)


def _rows_contiguous(t):
    """An expanded or transposed gradient (of a sum, say) has no rows of contiguous channels."""
    if t.ndim == 5:
        return t.contiguous(memory_format=torch.channels_last_3d)
    return t if t.is_contiguous() else t.contiguous()


# The product is linear in each of its arguments, so the gradients of the three operators are the three operators again:
#   y  = F(x, w):   dx = D(dy, w)   dw = W(x, dy)
#   dx = D(g, w):   dg = F(v, w)    dw = W(v, g)        v, V: the gradients of dx, dw
#   dw = W(x, g):   dx = D(g, V)    dg = F(x, V)
# A backward pass that is itself to be differentiated goes through the functions below, any other calls the operators.
class GroupedLinearFunction(torch.autograd.Function):
    """y = GroupedLinear(x, weight, ends) with gradients for x and weight, differentiable any number of times."""

    @staticmethod
    def forward(ctx, x, weight, ends):
        ctx.save_for_backward(x, weight, ends)
        return GroupedLinear(x, weight, ends)

    @staticmethod
    def backward(ctx, grad_out):
        x, weight, ends = ctx.saved_tensors
        grad_out = _rows_contiguous(grad_out)
        need_x, need_w, _ = ctx.needs_input_grad
        if torch.is_grad_enabled():
            return (GroupedLinearDGRADFunction.apply(grad_out, weight, ends) if need_x else None,
                    GroupedLinearWGRADFunction.apply(x, grad_out, weight, ends) if need_w else None, None)
        dx, dw = grouped_linear_grads(x, weight, grad_out, ends, need_x, need_w)
        return dx, dw, None


class GroupedLinearDGRADFunction(torch.autograd.Function):
    """dx = GroupedLinearDGRAD(grad, weight, ends) with gradients for grad and weight."""

    @staticmethod
    def forward(ctx, grad, weight, ends):
        ctx.save_for_backward(grad, weight, ends)
        return GroupedLinearDGRAD(grad, weight, ends)

    @staticmethod
    def backward(ctx, v):
        grad, weight, ends = ctx.saved_tensors
        v = _rows_contiguous(v)
        need_g, need_w, _ = ctx.needs_input_grad
        return (GroupedLinearFunction.apply(v, weight, ends) if need_g else None,
                GroupedLinearWGRADFunction.apply(v, grad, weight, ends) if need_w else None, None)


class GroupedLinearWGRADFunction(torch.autograd.Function):
    """dw = GroupedLinearWGRAD(x, grad, ends) in the form of `like`, with gradients for x and grad."""

    @staticmethod
    def forward(ctx, x, grad, like, ends):
        ctx.save_for_backward(x, grad, ends)
        return GroupedLinearWGRAD(x, grad, ends).view(like.shape)

    @staticmethod
    def backward(ctx, v):
        x, grad, ends = ctx.saved_tensors
        v = v.contiguous()
        return (GroupedLinearDGRADFunction.apply(grad, v, ends) if ctx.needs_input_grad[0] else None,
                GroupedLinearFunction.apply(x, v, ends) if ctx.needs_input_grad[1] else None, None, None)


def grouped_linear(x, weight, ends=None):
    """Differentiable product of row groups with a weight matrix each; see ops.linear.GroupedLinear."""
    return GroupedLinearFunction.apply(x, weight, ends)


class ExpertLinear(torch.nn.Module):
    """Module form of grouped_linear: `experts` bias-free channel-mixing products, weight [experts, out, in]."""

    def __init__(self, experts, in_channels, out_channels, device=None, dtype=torch.float16):
        super().__init__()
        bound = 1.0 / in_channels ** 0.5  # kaiming_uniform_(a=sqrt(5)) on each (out, in) matrix
        w = (torch.rand(experts, out_channels, in_channels, device=device) * 2 - 1) * bound
        self.weight = torch.nn.Parameter(w.to(dtype))

    def forward(self, x, ends=None):
        return grouped_linear(x, self.weight, ends)
