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

from .._lib import ops

IGNORE = -100                  # torch's default ignore_index
MOST_TOP = 16                  # alternatives of a row

ClassLogprobs = namedtuple('ClassLogprobs', 'logprob entropy top_logprob top_index')


def class_logprobs(scores, labels=None, top=0, ignore_index=IGNORE):
    """ClassLogprobs of every row: `logprob` of its label (0 where it is ignored; None without labels), `entropy` of its
    distribution, the `top` (at most 16) best classes with their log probabilities, best first, ties to the lower class:
    [M, top] or [B, top, N].  Differentiable in the scores, but for `top_index`."""
    return ClassLogprobs(*ops.class_logprobs(scores, labels, ignore_index, top))


def class_nll(scores, labels, ignore_index=IGNORE):
    """(mean of -log p[label] over the rows that are not ignored, share of them whose best class is the label), 0-d float32.
    NaN when every row is ignored."""
    return ops.class_nll(scores, labels, ignore_index)
