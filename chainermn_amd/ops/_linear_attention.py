"""Linear attention with a decay for each head: checks, the CPU form and the
single-token form.

Kernels: _hip/csrc/linear_attention.hip.
"""

import torch

from chainermn_amd.ops._embedding import wide

MAX_HEAD = 128


def check_attention(q, k, v, log_decay, dims):
    if q.dim() != dims or k.shape != q.shape or v.shape[:-1] != q.shape[:-1]:
        raise ValueError(
            'linear_attention: q {}, k {}, v {}: {} axes, alike but for '
            "v's last".format(tuple(q.shape), tuple(k.shape),
                              tuple(v.shape), dims))
    if not (1 <= q.shape[-1] <= MAX_HEAD and 1 <= v.shape[-1] <= MAX_HEAD):
        raise ValueError('linear_attention: heads of 1 to {} elements, not '
                         '{} and {}'.format(MAX_HEAD, q.shape[-1],
                                            v.shape[-1]))
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError('linear_attention: q, k and v are {}, {} and {}'
                        .format(q.dtype, k.dtype, v.dtype))
    if log_decay.shape != q.shape[-2:-1]:
        raise ValueError('linear_attention: log_decay {} for {} heads'.format(
            tuple(log_decay.shape), q.shape[-2]))
    if log_decay.dtype != torch.float32:
        raise TypeError('linear_attention: log_decay must be float32')
    if log_decay.requires_grad:
        raise ValueError('linear_attention: the decay is not differentiable')


def check_state(state, q, v):
    want = (q.shape[0], q.shape[-2], q.shape[-1], v.shape[-1])
    if tuple(state.shape) != want:
        raise ValueError('linear_attention: the state is {}, not {}'.format(
            tuple(state.shape), want))
    if state.dtype != torch.float32:
        raise TypeError('linear_attention: a state is float32, not {}'
                        .format(state.dtype))


def attention_plain(q, k, v, log_decay, first, lengths, scale):
    """The whole matrix of scores, in fp32: the CPU's form."""
    t = q.shape[1]
    pos = torch.arange(t, device=q.device)
    if lengths is None:
        n = torch.full((q.shape[0],), t, device=q.device)
    else:
        if lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError('linear_attention: lengths must be int32 or '
                            'int64, not {}'.format(lengths.dtype))
        n = lengths.long().clamp(0, t)
    live = (pos < n[:, None])[:, :, None, None]
    zero = torch.zeros((), device=q.device)
    qf, kf, vf = (torch.where(live, wide(x), zero.to(wide(x).dtype))
                  .transpose(1, 2) for x in (q, k, v))
    ld = log_decay.clamp(min=-200.0)[:, None].to(qf.dtype)  # 0 * log(0) is 0
    gap = pos[:, None] - pos
    w = torch.where(gap >= 0, torch.exp(
        gap.clamp(min=0) * ld[:, :, None]), zero)
    o = (qf @ kf.transpose(-1, -2) * w) @ vf
    left = (n[:, None, None] - 1 - pos).clamp(min=0)
    last = kf.transpose(-1, -2) @ (vf * torch.exp(left * ld)[..., None])
    if first is not None:
        first = first.to(qf.dtype)
        o = o + (qf @ first) * torch.exp((pos + 1) * ld)[..., None]
        last = last + first * torch.exp(
            n[:, None, None, None] * ld[..., None])
    return (o * scale).transpose(1, 2).to(q.dtype), last.float()


def linear_attention_step(q, k, v, state, log_decay, scale=None):
    """Linear attention of one new token for each sequence.

    ``q``, ``k`` ``[batch, heads, dk]``, ``v`` ``[batch, heads, dv]``,
    ``state`` ``[batch, heads, dk, dv]`` (fp32, contiguous), which is updated
    IN PLACE: ``state = exp(log_decay) * state + k^T v``.  Returns
    ``scale * q state`` ``[batch, heads, dv]``; ``scale`` is ``dk ** -0.5`` by
    default.  Not differentiable: training uses
    ``functions.linear_attention``.
    """
    check_attention(q, k, v, log_decay, 3)
    check_state(state, q, v)
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad or v.requires_grad
            or state.requires_grad):
        raise ValueError('linear_attention_step is not differentiable: use '
                         'functions.linear_attention, or no_grad()')
    if q.is_cuda:
        from chainermn_amd import ops
        return ops.require().linear_attention_step(
            q, k, v, state, log_decay.contiguous(), float(scale))
    if not state.is_contiguous():
        raise ValueError('linear_attention: a state is contiguous')
    # in fp64: rounded, a decay near one would lose what a long memory forgets
    state.copy_(state.double() * torch.exp(log_decay.double())[:, None, None]
                + k.double()[..., None] * v.double()[..., None, :])
    return ((q.float()[..., None] * state).sum(-2) * scale).to(q.dtype)
