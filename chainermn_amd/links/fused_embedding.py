"""FusedEmbedding — an embedding on the gfx950 kernels (embed.hip).

A drop-in for ``nn.Embedding(n_vocab, n_units)``: the same parameter, start
and state dict.  Chainer's EmbedID, which the reference's model used
(examples/seq2seq/seq2seq.py), had ``ignore_label``; ``scale`` multiplies the
rows (the square root of n_units, for instance)."""

import torch.nn as nn

from chainermn_amd import functions


class FusedEmbedding(nn.Embedding):

    def __init__(self, n_vocab, n_units, ignore_label=None, scale=1.0,
                 **kwargs):
        for name in kwargs:
            if name not in ('device', 'dtype'):
                raise TypeError('FusedEmbedding has no {}'.format(name))
        super().__init__(n_vocab, n_units, **kwargs)
        self.ignore_label = ignore_label
        self.scale = float(scale)

    def forward(self, x):
        return functions.embed_id(x, self.weight,
                                  ignore_label=self.ignore_label,
                                  scale=self.scale)

    def extra_repr(self):
        return '{}, {}, ignore_label={}, scale={}'.format(
            self.num_embeddings, self.embedding_dim, self.ignore_label,
            self.scale)
