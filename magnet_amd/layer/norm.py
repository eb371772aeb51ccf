"""Group norm of complex features, with the complex ReLU behind it (csrc/norm.hip).

    y = complex_group_norm(x, num_groups, weight, bias, graph_ptr, eps, relu)      # x row-planar [N, 2, F]
    ComplexGroupNorm(num_groups, num_channels).forward(real, imag) -> (real, imag)

Over the nodes of each graph of the batch and the channels of each group, with m = mean z (complex) and v = mean |z - m|^2:
y = weight (z - m) / sqrt(v + eps) + bias on both parts, as the convolutions add their real bias to both
(reference src/layer/sparse_magnet.py:72), then the gate of complex_relu_layer (src/layer/sparse_magnet.py:79-81).  The reference
has no normalisation; it is what lets networks of more than a few convolutions train.  GPU only.
"""
import torch
import torch.nn as nn

from .._lib import ops, MagnetHipError
from .sparse_magnet import _as_packed, _views


def complex_group_norm(x, num_groups, weight=None, bias=None, graph_ptr=None, eps=1e-5, relu=False, checkpoint_bits=32,
                       next_terms=0):
    """x: row-planar float32 [N, 2, F], any row and part strides; num_groups divides F.
    weight, bias: float32 [F] or None (1, 0).
    graph_ptr: integer [B + 1] on the GPU, the rows graph_ptr[b] .. graph_ptr[b + 1] being graph b's; it starts at 0 and does not
        decrease.  Graphs may be empty; rows behind the last one (a padded batch) are returned as zeros and get no gradient.
        None: one graph of all rows.
    relu: the complex ReLU on the result (both parts are kept where the real part is >= 0).
    checkpoint_bits: 32 keeps x itself for the backward pass; 8 keeps a Checkpoint8 of it, and the gate in a byte: the
        gradients are those of the formula with the restored values in the place of x's and the forward's statistics.
    next_terms: above 1, the result is order 0 of a new side-by-side block of that many orders, for the conv that follows."""
    if not eps >= 0.0:
        raise MagnetHipError('eps must not be negative, got %r' % (eps,))
    if graph_ptr is not None and graph_ptr.dtype != torch.int32:
        if graph_ptr.dtype != torch.int64:
            raise MagnetHipError('graph_ptr must be an integer tensor, got %s' % graph_ptr.dtype)
        graph_ptr = graph_ptr.to(torch.int32)
    return ops.group_norm(x, weight, bias, num_groups, graph_ptr, eps, relu, checkpoint_bits, next_terms)


class ComplexGroupNorm(nn.Module):
    """Group norm between a ChebConv and its activation.  `activation` True joins the complex ReLU to it.  `checkpoint_bits`
    8 keeps the input in 8 bits for the backward pass.  forward takes (real, imag) or the pair as one argument, as
    complex_relu_layer does, and the batch's `graph_ptr`."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation=False, checkpoint_bits=32):
        super(ComplexGroupNorm, self).__init__()
        if num_groups < 1 or num_channels % num_groups:
            raise MagnetHipError('%d channels do not divide into %d groups' % (num_channels, num_groups))
        self.num_groups, self.num_channels, self.eps = num_groups, num_channels, eps
        self.activation, self.checkpoint_bits = activation, checkpoint_bits
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels))
            self.bias = nn.Parameter(torch.zeros(num_channels))
        else:
            self.register_parameter('weight', None)
            self.register_parameter('bias', None)

    def forward_packed(self, xp, relu=False, graph_ptr=None, next_terms=0):
        """Row-planar in, row-planar out; `relu` joins the complex ReLU that follows, `next_terms` as in ChebConv."""
        return complex_group_norm(xp, self.num_groups, self.weight, self.bias, graph_ptr, self.eps, relu or self.activation,
                                  self.checkpoint_bits, next_terms)

    def forward(self, real, imag=None, graph_ptr=None):
        if imag is None:
            real, imag = real
        return _views(self.forward_packed(_as_packed(real, imag), graph_ptr=graph_ptr))
