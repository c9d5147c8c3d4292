"""Seq2seq LSTM encoder-decoder.

Reference analog: examples/seq2seq/seq2seq.py — an LSTM encoder-decoder
whose model-parallel variant splits encoder and decoder across ranks via
``create_multi_node_n_step_rnn`` / ``MultiNodeChainList``.

``Seq2Seq`` here is the single-process model; ``make_model_parallel``
returns (encoder_part, decoder_part) wrappers for a 2-rank split where the
final hidden state crosses the xGMI link via differentiable send/recv.

``fused_ops`` takes the embedding's own kernels, ``dropout`` (after the
embedding and before the output) the counter-based one, and
``rnn='attention'`` layers of linear attention in the LSTM's place; their
state is one tensor instead of the pair (h, c).
"""

import torch
import torch.nn as nn

from chainermn_amd import functions


def _embedding(n_vocab, n_units, fused_ops):
    if fused_ops:
        from chainermn_amd.links.fused_embedding import FusedEmbedding
        return FusedEmbedding(n_vocab, n_units)
    return nn.Embedding(n_vocab, n_units)


def _rnn(n_units, n_layers, rnn, dropout, comm):
    if rnn == 'lstm':
        return nn.LSTM(n_units, n_units, n_layers, batch_first=True)
    if rnn == 'attention':
        from chainermn_amd.links.linear_attention import LinearAttentionRNN
        return LinearAttentionRNN(n_units, n_units, n_layers,
                                  dropout=dropout, comm=comm)
    raise ValueError("rnn must be 'lstm' or 'attention', not {!r}".format(
        rnn))


def _dropout(ratio, comm):
    if not ratio:
        return nn.Identity()
    from chainermn_amd.links.fused_dropout import FusedDropout
    return FusedDropout(ratio, comm=comm)


class Encoder(nn.Module):

    def __init__(self, n_vocab, n_units, n_layers=2, rnn='lstm', dropout=0.0,
                 fused_ops=False, comm=None):
        super().__init__()
        self.embed = _embedding(n_vocab, n_units, fused_ops)
        self.rnn = _rnn(n_units, n_layers, rnn, dropout, comm)
        self.dropout = _dropout(dropout, comm)

    def forward(self, xs, lengths=None):
        h = self.dropout(self.embed(xs))
        if lengths is None:
            _, state = self.rnn(h)
        elif isinstance(self.rnn, nn.LSTM):
            raise ValueError("lengths of a padded batch need "
                             "rnn='attention'")
        else:
            _, state = self.rnn(h, lengths=lengths)
        return state  # (h_n, c_n), or the attention's state


class Decoder(nn.Module):

    def __init__(self, n_vocab, n_units, n_layers=2, rnn='lstm', dropout=0.0,
                 fused_ops=False, comm=None):
        super().__init__()
        self.embed = _embedding(n_vocab, n_units, fused_ops)
        self.rnn = _rnn(n_units, n_layers, rnn, dropout, comm)
        self.out = nn.Linear(n_units, n_vocab)
        self.dropout = _dropout(dropout, comm)

    def forward(self, ys_in, state):
        h, _ = self.rnn(self.dropout(self.embed(ys_in)), state)
        return self.out(self.dropout(h))

    def step(self, y, state):
        """Logits of one more token ``y [batch]``, and the state behind it
        (the attention's is updated in place)."""
        h = self.embed(y)
        if isinstance(self.rnn, nn.LSTM):
            h, state = self.rnn(h[:, None], state)
            return self.out(h[:, 0]), state
        return self.out(self.rnn.step(h, state)), state


class Seq2Seq(nn.Module):
    """Teacher-forced training model; forward returns mean CE loss."""

    def __init__(self, n_src_vocab, n_tgt_vocab, n_units, n_layers=2,
                 rnn='lstm', dropout=0.0, fused_ops=False, comm=None):
        super().__init__()
        self.encoder = Encoder(n_src_vocab, n_units, n_layers, rnn, dropout,
                               fused_ops, comm)
        self.decoder = Decoder(n_tgt_vocab, n_units, n_layers, rnn, dropout,
                               fused_ops, comm)
        self.loss_fn = nn.CrossEntropyLoss()

    def forward(self, xs, ys_in, ys_out, lengths=None):
        state = self.encoder(xs, lengths)
        logits = self.decoder(ys_in, state)
        return self.loss_fn(logits.reshape(-1, logits.shape[-1]),
                            ys_out.reshape(-1))

    @torch.no_grad()
    def translate(self, xs, max_length, bos=0, lengths=None):
        """Greedy generation (the reference's ``translate``): the
        ``[batch, max_length]`` tokens that follow ``bos``."""
        modes = [(m, m.training) for m in self.modules()]
        self.eval()
        try:
            state = self.encoder(xs, lengths)
            y = torch.full((xs.shape[0],), bos, dtype=torch.long,
                           device=xs.device)
            out = []
            for _ in range(max_length):
                logits, state = self.decoder.step(y, state)
                y = logits.argmax(-1)
                out.append(y)
        finally:
            for m, training in modes:  # parts of it may be frozen
                m.training = training
        return torch.stack(out, 1) if out else xs.new_empty(
            (xs.shape[0], 0), dtype=torch.long)


class EncoderPart(nn.Module):
    """Rank holding the encoder: encode, send its state to decoder rank."""

    def __init__(self, encoder, comm, decoder_rank):
        super().__init__()
        self.encoder = encoder
        self.comm = comm
        self.decoder_rank = decoder_rank

    def forward(self, xs, lengths=None):
        state = self.encoder(xs, lengths)
        state = state.contiguous() if isinstance(state, torch.Tensor) \
            else tuple(x.contiguous() for x in state)
        delegate = functions.send(state, self.comm, self.decoder_rank)
        return delegate  # call .backward() on this


class DecoderPart(nn.Module):
    """Rank holding the decoder: recv the state, decode, return loss."""

    def __init__(self, decoder, comm, encoder_rank):
        super().__init__()
        self.decoder = decoder
        self.comm = comm
        self.encoder_rank = encoder_rank
        self.loss_fn = nn.CrossEntropyLoss()

    def forward(self, ys_in, ys_out):
        state = functions.recv(self.comm, self.encoder_rank,
                               force_tuple=True)
        logits = self.decoder(ys_in, tuple(state) if len(state) > 1
                              else state[0])
        return self.loss_fn(logits.reshape(-1, logits.shape[-1]),
                            ys_out.reshape(-1))


def make_model_parallel(model, comm, encoder_rank=0, decoder_rank=1):
    """Split a Seq2Seq across two ranks; returns this rank's part."""
    if comm.rank == encoder_rank:
        return EncoderPart(model.encoder, comm, decoder_rank)
    elif comm.rank == decoder_rank:
        return DecoderPart(model.decoder, comm, encoder_rank)
    raise ValueError('rank {} not part of this 2-way split'.format(comm.rank))
