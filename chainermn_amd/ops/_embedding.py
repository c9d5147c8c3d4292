"""Embedding lookup with scaling: argument checks and the CPU form.

Kernels: _hip/csrc/embed.hip.  The reference's model used Chainer's EmbedID
(examples/seq2seq/seq2seq.py), whose ``ignore_label`` this follows.
"""

import torch
import torch.nn.functional as F


def wide(x):
    """What the plain forms compute in: fp32, or fp64 for fp64."""
    return x if x.dtype == torch.float64 else x.float()


def check_embedding(ids, W):
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError('embed_id: ids must be int32 or int64, not {}'
                        .format(ids.dtype))
    if W.dim() != 2 or W.shape[0] == 0 or W.shape[1] == 0:
        raise ValueError('embed_id: W must be a non-empty matrix, not {}'
                         .format(tuple(W.shape)))
    if ids.device != W.device:
        raise ValueError('embed_id: ids are on {}, W on {}'
                         .format(ids.device, W.device))


def embed_plain(ids, W, ignore_label, scale):
    at, skip = ids.long(), None
    if ignore_label is not None:
        skip = at == ignore_label
        at = at.masked_fill(skip, 0)
    y = F.embedding(at, W)
    if scale != 1.0:
        y = (wide(y) * scale).to(W.dtype)
    return y if skip is None else y.masked_fill(skip[..., None], 0)
