"""Embedding lookup with scaling, and its gradient by sorted tokens."""

from chainermn_amd import ops
from chainermn_amd.ops._embedding import check_embedding, embed_plain


def embed_id(x, W, ignore_label=None, scale=1.0):
    """``scale * W[x]``: ``x`` int32 or int64 of any shape, ``W``
    ``[vocabulary, units]`` with contiguous rows; returns
    ``x.shape + (units,)`` in W's type.

    An id equal to ``ignore_label`` (any number, -1 or 0 for instance) gives
    a row of zeros and no gradient.  Padding should be such an id: one that
    is looked up is summed like a word, more slowly the more of it there is.
    Any other id outside of the vocabulary is an error: an IndexError on the
    CPU; on the GPU, where finding out would stop the stream, its row is NaN
    and has no gradient.

    The gradient of W is dense.  It is summed in fp32 in the order of the
    tokens, without atomics: two runs agree bit by bit.
    """
    check_embedding(x, W)
    if W.is_cuda:
        return ops.require().embed_id(
            x, W, float(scale), ignore_label is not None,
            0 if ignore_label is None else int(ignore_label))
    return embed_plain(x, W, ignore_label, float(scale))
