"""What a network answers with: log probabilities of given classes, entropy, top alternatives, and the loss (csrc/scores.hip).

    r = class_logprobs(scores, labels, top=k)      # r.logprob, r.entropy, r.top_logprob, r.top_index
    loss, accuracy = class_nll(scores, labels)

`scores` are class scores as the heads make them, float32, bfloat16 or float16: [M, C] (ChebNet_Edge), or [B, C, N] with the
classes in the middle (ChebNet: [1, C, N]); any strides.  `labels` int64 [M] / [B, N]; a row labelled `ignore_index` counts for
nothing.  Each reads the scores once; the reference takes log_softmax, the loss and the arg max in passes of their own
(src/layer/sparse_magnet.py:128, src/sparse_Magnet.py:155-160).  Computed in float32.  GPU only.

A label outside [0, C) that is not `ignore_index` gives NaN (nothing is read out of range).  A score of -inf is a class of
probability 0; a row of -inf alone, or with +inf or NaN, gives NaN, as log_softmax does.
"""
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

from .._lib import ops, MagnetHipError

IGNORE = -100                  # torch's default ignore_index
MOST_TOP = 16

ClassLogprobs = namedtuple('ClassLogprobs', 'logprob entropy top_logprob top_index')


def _rows_shape(scores):
    if scores.dim() not in (2, 3):
        raise MagnetHipError('scores must be [M, C] or [B, C, N], got %s' % (tuple(scores.shape),))
    return (scores.size(0),) if scores.dim() == 2 else (scores.size(0), scores.size(2))


def _check_labels(labels, scores):
    rows = _rows_shape(scores)
    if labels is not None and tuple(labels.shape) != rows:
        raise MagnetHipError('labels have shape %s, expected %s' % (tuple(labels.shape), rows))
    return None if labels is None else labels.contiguous()


def _like(scores):
    """Memory for a gradient: the scores' own layout where that is dense, so that it is written as the scores are read."""
    return torch.empty_like(scores)


def _row_gradient(g):
    """One value per row: as it is when contiguous or one value expanded (the gradient of a sum or a mean)."""
    if g is None or g.is_contiguous() or all(n <= 1 or s == 0 for n, s in zip(g.shape, g.stride())):
        return g
    return g.contiguous()


class _LogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, labels, ignore, top, keep):
        rows = _rows_shape(scores)
        f32 = dict(dtype=torch.float32, device=scores.device)
        logprob = None if labels is None else torch.empty(rows, **f32)
        entropy = torch.empty(rows, **f32)
        shape = (rows[0], top) + rows[1:]
        top_lp = torch.empty(shape, **f32)
        top_index = torch.empty(shape, dtype=torch.int64, device=scores.device)
        stat = torch.empty(rows + (2,), **f32) if keep else None
        ops.class_logprobs(scores, labels, ignore, logprob, entropy, stat, top_lp, top_index)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_index)
        ctx.ignore = ignore
        ctx.save_for_backward(scores, labels, stat, entropy, top_index)
        return logprob, entropy, top_lp, top_index

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprob, g_entropy, g_top, _):
        scores, labels, stat, entropy, top_index = ctx.saved_tensors
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None, None, None
        d = _like(scores)
        ops.class_logprobs_bwd(scores, labels, ctx.ignore, stat, entropy, _row_gradient(g_logprob), _row_gradient(g_entropy),
                               None if g_top is None else g_top.contiguous(), None if g_top is None else top_index, d)
        return d, None, None, None, None


class _NllFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, labels, ignore, keep):
        f32 = dict(dtype=torch.float32, device=scores.device)
        loss, accuracy, inv_count = (torch.empty((), **f32) for _ in range(3))
        stat = torch.empty(_rows_shape(scores) + (2,), **f32) if keep else None
        ops.class_nll(scores, labels, ignore, stat, loss, accuracy, inv_count)
        ctx.mark_non_differentiable(accuracy)
        ctx.set_materialize_grads(False)
        ctx.ignore = ignore
        ctx.save_for_backward(scores, labels, stat, inv_count)
        return loss, accuracy

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss, _):
        scores, labels, stat, inv_count = ctx.saved_tensors
        if g_loss is None:
            return None, None, None, None
        d = _like(scores)
        ops.class_nll_bwd(scores, labels, ctx.ignore, stat, inv_count, g_loss, d)
        return d, None, None, None


def class_logprobs(scores, labels=None, top=0, ignore_index=IGNORE):
    """ClassLogprobs of every row: `logprob` of its label (0 where it is ignored; None without labels), `entropy` of its
    distribution, the `top` (at most 16) best classes with their log probabilities, best first, ties to the lower class:
    [M, top] or [B, top, N].  Differentiable in the scores, but for `top_index`."""
    labels = _check_labels(labels, scores)
    if not 0 <= top <= min(MOST_TOP, scores.size(1)):
        raise MagnetHipError('top must be between 0 and %d, got %d' % (min(MOST_TOP, scores.size(1)), top))
    keep = torch.is_grad_enabled() and scores.requires_grad
    return ClassLogprobs(*_LogprobsFn.apply(scores, labels, ignore_index, int(top), keep))


def class_nll(scores, labels, ignore_index=IGNORE):
    """(mean of -log p[label] over the rows that are not ignored, share of them whose best class is the label), 0-d float32.
    NaN when every row is ignored."""
    if labels is None:
        raise MagnetHipError('class_nll needs labels')
    keep = torch.is_grad_enabled() and scores.requires_grad
    return _NllFn.apply(scores, _check_labels(labels, scores), ignore_index, keep)
