"""Token embedding as a torch module, on the library's lookup and gradient
kernels.  ``KFAC`` gives it a Kronecker-factored block (a plain
``torch.nn.Embedding`` has none and is left to the momentum rule)."""

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from chainerkfac_b200 import ops


class _EmbedIDFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, weight, ids, scale, ignore_label):
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.dtype = weight.shape[0], weight.dtype
        ctx.scale, ctx.ignore_label = scale, ignore_label
        return ops.embedding(weight, ids, scale, ignore_label)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        ids, = ctx.saved_tensors
        order = ops.TokenOrder(ids, ctx.vocab, ctx.ignore_label)
        return ops.embedding_grad(gy.contiguous().to(ctx.dtype), order,
                                  ctx.scale), None, None, None


class EmbedID(nn.Module):
    """Rows of ``weight`` (in_size, out_size) by token, times ``scale``; the
    row of ``ignore_label`` is zeros and gets no gradient.  Weights are drawn
    from the standard normal distribution."""

    def __init__(self, in_size, out_size, ignore_label=None, scale=1.0,
                 device=None, dtype=None):
        super(EmbedID, self).__init__()
        self.weight = nn.Parameter(torch.empty(
            (in_size, out_size), device=device, dtype=dtype))
        self.ignore_label = ignore_label
        self.scale = float(scale)
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.normal_(self.weight)

    def extra_repr(self):
        return '{}, {}, ignore_label={}, scale={}'.format(
            self.weight.shape[0], self.weight.shape[1], self.ignore_label,
            self.scale)

    def forward(self, ids):
        return _EmbedIDFunction.apply(self.weight, ids.contiguous(),
                                      self.scale, self.ignore_label)
