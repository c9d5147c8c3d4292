"""Dropout from a counter-based generator, with a mask that is never
stored."""

from chainermn_amd import ops
from chainermn_amd.ops._dropout import (check_key, dropout_plain,
                                        dropout_threshold)


def dropout(x, key, ratio=0.5):
    """Zeroes elements of ``x`` with probability ``ratio`` and divides the
    others by ``1 - ratio``.

    ``key`` is a tensor of two int64, a seed and a call number, on x's
    device; ``ops.dropout_next_key`` draws one from a running state.  Element
    i (in the order of a contiguous x) depends on the key and i alone, and
    the backward pass computes it again.  The CPU and the GPU drop the same
    elements.
    """
    check_key(x, key)
    threshold, scale = dropout_threshold(ratio)
    if x.is_cuda:
        return ops.require().dropout(x, key, threshold, scale)
    return dropout_plain(x, key, threshold, scale)
