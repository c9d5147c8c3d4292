"""Root-mean-square norm with the residual's addition."""

from chainermn_amd import ops
from chainermn_amd.ops._rms_norm import check_rms_norm, rms_plain


def rms_norm(x, weight, residual=None, eps=1e-6):
    """``h * rsqrt(mean(h^2) + eps) * weight`` over the last axis (1 to 16384
    elements), where ``h = x + residual``.

    Returns the output, or ``(output, h)`` where there is a residual: ``h``
    is the residual of the next layer.  ``weight`` is of x's type or fp32.
    Sums are fp32 and each output and gradient is rounded once.
    """
    check_rms_norm(x, weight, residual)
    if x.is_cuda:
        out = ops.require().rms_norm(x, weight, residual, float(eps))
        return out[0] if residual is None else tuple(out)
    y, h = rms_plain(x, weight, residual, eps)
    y = y.to(x.dtype)
    return y if residual is None else (y, h.to(x.dtype))
