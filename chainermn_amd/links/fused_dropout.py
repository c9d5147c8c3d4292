"""FusedDropout — dropout whose mask is computed from a counter and never
stored (dropout.hip).

The state is a buffer of two integers, a seed and the number of calls so far:
it moves with the model, is saved with it, and a restored model goes on with
the same numbers.  It is counted up on the GPU, so a replayed graph draws new
ones.  Ranks given their communicator draw from streams of their own, also
after ``bcast_data`` has made their states equal.

A call that is computed again in a backward pass has to drop what it dropped
first: checkpoint it by ``functions.forget``.  Under ``torch.utils.checkpoint``,
which does not know the state, it raises an error."""

import torch
import torch.nn as nn

from chainermn_amd import functions, ops
from chainermn_amd.functions.forget import dropout_key
from chainermn_amd.ops._dropout import dropout_threshold


class FusedDropout(nn.Module):

    def __init__(self, ratio=0.5, seed=None, comm=None):
        super().__init__()
        dropout_threshold(ratio)  # refuses what is not in [0, 1)
        self.ratio = float(ratio)
        self.stream = comm.rank if comm is not None else 0
        if seed is None:
            seed = int(torch.randint(2 ** 62, ()))
        self.register_buffer('rng_state', torch.tensor(
            [seed, 0], dtype=torch.int64))

    def forward(self, x):
        if not self.training or self.ratio == 0.0:
            return x
        key = dropout_key(lambda: ops.dropout_next_key(self.rng_state,
                                                       self.stream))
        return functions.dropout(x, key, ratio=self.ratio)

    def extra_repr(self):
        return 'ratio={}'.format(self.ratio)
