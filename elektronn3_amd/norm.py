"""Group norm with an activation as ONE module, optionally with its input kept in 8 bits for the backward.

:class:`GroupNormAct` stands for the pair ``get_normalization('group<G>', C)`` + ``get_activation(...)`` of a network's block
(elektronn3/models/unet.py:77-105,183-199) in networks that are built from single layers; ``UNet(normalization='group<G>')`` runs its norms
inside the whole-network executor and does not need it.
"""
import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import ops


def _to_ndhwc(x):
    """(N, C, *spatial) with 1 to 3 spatial axes -> an (N, D, H, W, C) view that the ops take; copies only if the memory is not channels last."""
    v = x.movedim(1, -1)
    while v.dim() < 5:
        v = v.unsqueeze(1)
    try:
        ops._ldc(v)
    except ValueError:
        v = v.contiguous()
    return v


def _from_ndhwc(v, like):
    return v.view(v.shape[0], *like.shape[2:], v.shape[-1]).movedim(-1, 1)


class _GroupNormActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, activation, checkpoint):
        xv = _to_ndhwc(x)
        w, b = (None if p is None else p.float() for p in (weight, bias))
        res = ops.group_norm_act(xv, num_groups, w, b, eps, activation, checkpoint)
        y, mean, rstd = res[:3]
        kept = (res[3].q, res[3].scale) if checkpoint else (xv,)
        ctx.save_for_backward(mean, rstd, weight, bias, *kept)
        ctx.activation, ctx.shape, ctx.dtype = activation, xv.shape, x.dtype
        return _from_ndhwc(y, x)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        mean, rstd, weight, bias, *kept = ctx.saved_tensors
        x = ops.Checkpoint8(*kept, ctx.shape, ctx.dtype) if len(kept) == 2 else kept[0]
        w, b = (None if p is None else p.float() for p in (weight, bias))
        dx, dw, db = ops.group_norm_act_bwd(x, mean, rstd, _to_ndhwc(dy), w, b, ctx.activation)
        return (_from_ndhwc(dx, dy), None if weight is None else dw.to(weight.dtype), None if bias is None else db.to(bias.dtype),
                None, None, None, None)


class GroupNormAct(nn.GroupNorm):
    """``activation(GroupNorm(num_groups, num_channels)(x))`` for (N, C), spatial axes 1 to 3, float32 / bfloat16 / float16 on a ROCm device; parameters and
    ``state_dict`` keys are ``nn.GroupNorm``'s.  A channels-last input (``torch.channels_last`` / ``channels_last_3d``) is read as it lies, any other layout
    is copied first; the result is channels last.

    ``checkpoint=True`` keeps the input for the backward as an 8-bit checkpoint (:class:`elektronn3_amd.ops.Checkpoint8`, 1.06 bytes per element)
    instead of the tensor: the outputs are the same, the gradients are those of the rounded input (an element is off by at most 1/254 of the largest of its
    block of 64; with ReLU or LeakyReLU by up to 1/127 next to the activation's border, whose side it keeps).  A parameter that is missing (``affine=False``) is 1 or 0.

    ``activation``: ``'relu'``, ``'leaky'``, ``'lin'``, ``'silu'`` or a module of those types (as in ``UNet(activation=...)``)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation='relu', checkpoint=False, device=None, dtype=None):
        super().__init__(num_groups, num_channels, eps=eps, affine=affine, device=device, dtype=dtype)
        ops._act_slope(activation)               # (raises for an activation that the kernels do not cover)
        self.activation, self.checkpoint = activation, bool(checkpoint)

    def forward(self, x):
        if not isinstance(x, torch.Tensor) or not 3 <= x.dim() <= 5:
            raise ValueError('expected an (N, C, ...) tensor with 1 to 3 spatial axes')
        if x.shape[1] != self.num_channels:
            raise ValueError(f'expected {self.num_channels} channels, got {x.shape[1]}')
        if not x.is_cuda:
            raise RuntimeError('elektronn3_amd.GroupNormAct runs only on a ROCm GPU (hand-written HIP kernels); there is no CPU fallback')
        keep = self.checkpoint and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, self.weight, self.bias))
        return _GroupNormActFunction.apply(x, self.weight, self.bias, self.num_groups, self.eps, self.activation, keep)

    def extra_repr(self):
        return super().extra_repr() + f', activation={self.activation!r}, checkpoint={self.checkpoint}'
