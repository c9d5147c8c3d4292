"""Linear attention with a decay for each head."""

from chainermn_amd import ops
from chainermn_amd.ops._linear_attention import (attention_plain,
                                                 check_attention,
                                                 check_state)


def linear_attention(q, k, v, log_decay, initial_state=None, lengths=None,
                     scale=None):
    """``S_t = exp(log_decay) S_(t-1) + k_t^T v_t``, ``o_t = scale q_t S_t``.

    ``q``, ``k`` ``[batch, length, heads, dk]`` and ``v`` ``[batch, length,
    heads, dv]`` (dk and dv from 1 to 128, any strides), ``log_decay``
    ``[heads]`` fp32, at most zero, not differentiable; ``initial_state``
    ``[batch, heads, dk, dv]`` fp32, zero by default; ``scale`` is
    ``dk ** -0.5`` by default.  ``lengths`` (int32 or int64, ``[batch]``)
    are the sequences' lengths in a padded batch, taken as 0 to ``length``
    where they lie outside of it: what lies behind them is
    not read, the output there is zero, and the state stops at the last
    token.

    Returns ``(o, state)``: ``o`` like v, and the fp32 state behind the
    sequences.  States and sums are fp32 whatever the type of q; products
    of fp32 are good to 2^-21, and of values below 2^-110 less so.  A value
    that is not finite spreads to the outputs of its own chunk of 32 tokens,
    those before it included.
    """
    check_attention(q, k, v, log_decay, 4)
    if initial_state is not None:
        check_state(initial_state, q, v)
    if lengths is not None and (lengths.dim() != 1
                                or lengths.shape[0] != q.shape[0]):
        raise ValueError('linear_attention: lengths {} for {} sequences'
                         .format(tuple(lengths.shape), q.shape[0]))
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if q.is_cuda:
        if initial_state is not None:
            initial_state = initial_state.contiguous()
        if lengths is not None:
            lengths = lengths.contiguous()
        return tuple(ops.require().linear_attention(
            q, k, v, log_decay.contiguous(), initial_state, lengths,
            float(scale)))
    return attention_plain(q, k, v, log_decay, initial_state, lengths,
                           float(scale))
