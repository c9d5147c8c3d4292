"""Root-mean-square norm with the residual's addition: checks, the CPU form
and the 8-bit output.

Kernels: _hip/csrc/rms_norm.hip.
"""

import torch

from chainermn_amd.ops._embedding import wide

E4M3_MAX = 448.0
MAX_DIM = 16384


def check_rms_norm(x, weight, residual):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_DIM:
        raise ValueError('rms_norm: rows of 1 to {} elements, not {}'
                         .format(MAX_DIM, tuple(x.shape)))
    if weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError('rms_norm: x is {}, the weight {}'.format(
            tuple(x.shape), tuple(weight.shape)))
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError('rms_norm: x is {}, the weight {}'.format(
            x.dtype, weight.dtype))
    if residual is not None and (residual.shape != x.shape
                                 or residual.dtype != x.dtype):
        raise ValueError('rms_norm: x is {} {}, the residual {} {}'.format(
            x.dtype, tuple(x.shape), residual.dtype, tuple(residual.shape)))
    if weight.device != x.device or (residual is not None
                                     and residual.device != x.device):
        raise ValueError('rms_norm: x, weight and residual are on different '
                         'devices')


def rms_plain(x, weight, residual, eps):
    """(y, h), not yet rounded."""
    h = wide(x)
    if residual is not None:
        h = h + wide(residual)
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
    return y * wide(weight), h


def rms_norm_fp8(x, weight, residual=None, eps=1e-6, group=None):
    """RMS norm with an output in 8 bits, for a product in e4m3.

    Returns ``(q, scales)``, or ``(q, scales, x + residual)``: ``q`` is
    float8_e4m3fn, ``q.float() * scale`` stands for the norm's output.  A
    scale is the largest magnitude / 448 over a row (``scales`` is
    ``[..., 1]``) or over ``group`` columns of it (``[..., dim / group]``;
    16, 32, 64, 128 or 256 that divide the row), and 1 where all are zero.
    Not differentiable.
    """
    check_rms_norm(x, weight, residual)
    dim = x.shape[-1]
    if group is not None and (group not in (16, 32, 64, 128, 256)
                              or dim % group):
        raise ValueError('rms_norm_fp8: groups of 16, 32, 64, 128 or 256 '
                         'columns that divide the row of {}, not {}'
                         .format(dim, group))
    if torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad
            or (residual is not None and residual.requires_grad)):
        raise ValueError('rms_norm_fp8 is not differentiable: use no_grad()')
    shape = x.shape
    groups = dim // group if group else 1
    if x.is_cuda:
        from chainermn_amd import ops
        m = _rows(x.detach())
        r = None if residual is None else _rows(residual.detach())
        q, scales, h = ops.require().rms_norm_fp8(
            m, weight.detach().contiguous(), r, float(eps), group or 0)
        if x.dim() != 2:
            q, scales = q.view(shape), scales.view(shape[:-1] + (groups,))
            h = h.view(shape) if residual is not None else h
        return (q, scales) if residual is None else (q, scales, h)
    with torch.no_grad():
        y, h = rms_plain(x, weight, residual, eps)
        y = y.reshape(shape[:-1] + (groups, dim // groups))
        scales = y.abs().amax(-1, keepdim=True) / E4M3_MAX
        scales = torch.where(scales > 0, scales, torch.ones_like(scales))
        q = (y / scales).clamp(-E4M3_MAX, E4M3_MAX)
        q = q.to(torch.float8_e4m3fn).view(shape)
        scales = scales.squeeze(-1)
        return (q, scales) if residual is None else (q, scales,
                                                     h.to(x.dtype))


def _rows(x):
    """A matrix of x's rows, each of them contiguous."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 else x.contiguous()
