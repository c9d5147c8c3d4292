"""LinearAttentionRNN — layers of linear attention with the calls of an
N-step RNN.

A layer keeps, for each head, a matrix that decays and takes in each token's
k^T v; so it is called like ``nn.LSTM`` (output and state, the state of one
call going into the next), its state can cross ranks in
``create_multi_node_n_step_rnn``, and a generated token costs the same however
long the text before it is.  Unlike an LSTM a sequence is computed in chunks,
on the matrix cores."""

import math

import torch
import torch.nn as nn

from chainermn_amd import functions, ops
from chainermn_amd.links.fused_dropout import FusedDropout
from chainermn_amd.links.fused_rms_norm import FusedRMSNorm


class _Layer(nn.Module):

    def __init__(self, size, n_heads, dropout, comm):
        super().__init__()
        self.norm = FusedRMSNorm(size)
        self.qkv = nn.Linear(size, 3 * size, bias=False)
        self.head_norm = FusedRMSNorm(size // n_heads)
        self.out = nn.Linear(size, size, bias=False)
        self.dropout = FusedDropout(dropout, comm=comm)


class LinearAttentionRNN(nn.Module):
    """``forward(x, state=None, lengths=None) -> (output, state)``.

    ``x`` is ``[batch, length, input_size]``; the state ``[num_layers, batch,
    n_heads, d, d]`` in fp32 with ``d = hidden_size / n_heads`` (at most 128;
    by default there are the fewest equal heads from ``hidden_size // 64`` on).
    ``lengths`` are those of a padded batch.  The heads' memories, after which
    a token's weight has fallen to 1/e, are spread from ``memory[0]`` to
    ``memory[1]`` tokens and are not learned.  Under autocast the sum of the
    layers keeps the type of ``x``.
    """

    def __init__(self, input_size, hidden_size, num_layers=1, n_heads=None,
                 dropout=0.0, memory=(4, 4096), batch_first=True, comm=None):
        super().__init__()
        if n_heads is None:
            n_heads = max(1, hidden_size // 64)
            while hidden_size % n_heads:
                n_heads += 1
            if n_heads > 1 and hidden_size // n_heads < 16:
                raise ValueError('LinearAttentionRNN: {} units have no equal '
                                 'heads of 16 to 128; n_heads has to be '
                                 'given'.format(hidden_size))
        if hidden_size % n_heads or hidden_size // n_heads > 128:
            raise ValueError('LinearAttentionRNN: {} units in {} heads: equal '
                             'heads of at most 128 units'.format(hidden_size,
                                                                 n_heads))
        if num_layers < 1:
            raise ValueError('LinearAttentionRNN: {} layers'.format(
                num_layers))
        if not batch_first:
            raise ValueError('LinearAttentionRNN is batch_first')
        if not 1 <= memory[0] <= memory[1]:
            raise ValueError('LinearAttentionRNN: memory {}'.format(memory))
        self.n_heads, self.head = n_heads, hidden_size // n_heads
        self.batch_first = True
        self.project = nn.Identity() if input_size == hidden_size else \
            nn.Linear(input_size, hidden_size, bias=False)
        self.layers = nn.ModuleList(
            _Layer(hidden_size, n_heads, dropout, comm)
            for _ in range(num_layers))
        self.norm = FusedRMSNorm(hidden_size)
        spread = torch.linspace(math.log(memory[0]), math.log(memory[1]),
                                n_heads, dtype=torch.float64)
        self.register_buffer('log_decay', -torch.exp(-spread).float(),
                             persistent=False)

    def _apply(self, fn, recurse=True):
        # a model cast to 16 bits keeps its decays in fp32
        decay = self.log_decay
        super()._apply(fn, recurse)
        self.log_decay = decay.to(self.log_decay.device)
        return self

    def forward(self, x, state=None, lengths=None):
        b, t, _ = x.shape
        if state is not None and state.shape[0] != len(self.layers):
            raise ValueError('LinearAttentionRNN: a state of {} layers, not '
                             '{}'.format(state.shape[0], len(self.layers)))
        h, branch, last = self.project(x).to(x.dtype), None, []
        for i, layer in enumerate(self.layers):
            if branch is None:
                y = layer.norm(h)
            else:
                y, h = layer.norm(branch.to(h.dtype), residual=h)
            q, k, v = layer.qkv(y).view(
                b, t, 3, self.n_heads, self.head).unbind(2)
            o, s = functions.linear_attention(
                q, k, v, self.log_decay,
                initial_state=None if state is None else state[i],
                lengths=lengths)
            last.append(s)
            o = layer.head_norm(o).flatten(2)
            branch = layer.dropout(layer.out(o))
        y, _ = self.norm(branch.to(h.dtype), residual=h)
        return y, torch.stack(last)

    @torch.no_grad()
    def step(self, x, state):
        """One token for each sequence: ``x [batch, input_size]``, and the
        state of ``forward``, which is updated in place."""
        b = x.shape[0]
        h, branch = self.project(x).to(x.dtype), None
        for i, layer in enumerate(self.layers):
            if branch is None:
                y = layer.norm(h)
            else:
                y, h = layer.norm(branch.to(h.dtype), residual=h)
            q, k, v = layer.qkv(y).view(
                b, 3, self.n_heads, self.head).unbind(1)
            o = ops.linear_attention_step(q, k, v, state[i], self.log_decay)
            branch = layer.out(layer.head_norm(o).flatten(1))
        return self.norm(branch.to(h.dtype), residual=h)[0]
