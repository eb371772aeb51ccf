"""Activation checkpoints in 8 bits.

A convolution keeps the K + 1 propagated matrices of its input only for the weight gradient dW = A^T G; kept in 8 bits they
take 1.03 bytes a value instead of 4, and the gradient is taken from the bytes as they are (csrc/ckpt.hip).  The reference
keeps every activation in 32 bits (src/layer/sparse_magnet.py:60-72).

    ck = Checkpoint8.store(x)      # x row-planar [N, 2, m] (or a block [N, 2, K + 1, F]), float32, on the GPU
    ck.restore()                   # [N, 2, m] float32
    ck.gram(g)                     # sum over nodes and parts of ck[:, :, i] g[:, :, j] -> [m, n]

32 neighbouring columns of a row share a power-of-two scale; a value is restored to within half a step, at most 1 / 127.5 of
the largest magnitude of its 32 (scales below 2^-110 do not occur: smaller values round to multiples of 2^-110).  A block with a
value that is not finite is restored as NaN.  The products of `gram` are float32 products of the restored values.
"""
import torch

from ._lib import ops, MagnetHipError

BLOCK = 32                     # columns that share a scale
MOST_RESULTS = 1 << 24         # of a `gram`


def contiguous_columns(t):
    """[N, 2, m] with its columns contiguous (any row and part strides); t itself where it is so already."""
    if t.dim() != 3 or t.size(2) <= 1 or t.stride(2) == 1:
        return t
    return t.contiguous() if t.numel() else t.new_empty(t.shape)      # an empty tensor counts as contiguous at any strides


class Checkpoint8:
    """codes uint8 [2N, m up to a multiple of 32], scales uint8 [blocks of 32 columns, 2N up to a multiple of 8], `shape` of
    what was stored ([N, 2, m] or [N, 2, K + 1, F])."""

    def __init__(self, codes, scales, shape):
        shape = tuple(int(v) for v in shape)
        if len(shape) < 3 or shape[1] != 2 or min(shape[2:]) < 1:
            raise MagnetHipError('a checkpoint holds [N, 2, m] or [N, 2, K + 1, F], got %s' % (shape,))
        self.codes, self.scales, self.shape = codes, scales, shape
        self.columns = 1
        for v in shape[2:]:
            self.columns *= v

    @staticmethod
    def memory(n, m, device):
        """Uninitialised (codes, scales) of a checkpoint of [n, 2, m]."""
        codes = torch.empty((2 * n, -(-m // BLOCK) * BLOCK), dtype=torch.uint8, device=device)
        return codes, torch.empty((codes.size(1) // BLOCK, -(-2 * n // 8) * 8), dtype=torch.uint8, device=device)

    @staticmethod
    def store(x):
        """Checkpoint of x.  Any row and part strides, the columns contiguous; a block [N, 2, K + 1, F] must be contiguous
        in its last two dimensions."""
        if x.dim() < 3 or x.size(1) != 2:
            raise MagnetHipError('a checkpoint holds [N, 2, m] or [N, 2, K + 1, F], got %s' % (tuple(x.shape),))
        shape = tuple(x.shape)
        x = x.detach()
        if x.dim() > 3:
            x = x.flatten(2)
        x = contiguous_columns(x)
        n, _, m = x.shape
        codes, scales = Checkpoint8.memory(n, m, x.device)
        ops.ckpt_store(x, codes, scales)
        return Checkpoint8(codes, scales, shape)

    def restore(self, out=None):
        """The float32 values, in the stored shape; `out`: where to write them ([N, 2, m], contiguous columns)."""
        n, m = self.shape[0], self.columns
        if out is not None:
            if tuple(out.shape) != (n, 2, m):
                raise MagnetHipError('out has shape %s, expected %s' % (tuple(out.shape), (n, 2, m)))
            ops.ckpt_restore(self.codes, self.scales, out)
            return out
        out = torch.empty((n, 2, m), dtype=torch.float32, device=self.codes.device)
        ops.ckpt_restore(self.codes, self.scales, out)
        return out.view(self.shape)

    def gram(self, g):
        """A^T G over nodes and parts, A the restored values [2N, m], g row-planar [N, 2, n] float32 -> [m, n].  At most MOST_RESULTS
        values of the result, and from one row of g to the next."""
        if g.dim() > 3:
            g = g.flatten(2)
        return ops.ckpt_gram(self.codes, self.scales, self.columns, contiguous_columns(g))

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()
