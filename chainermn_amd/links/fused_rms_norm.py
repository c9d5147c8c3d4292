"""FusedRMSNorm — root-mean-square norm, with the residual's addition in the
same kernel (rms_norm.hip)."""

import torch
import torch.nn as nn

from chainermn_amd import functions


class FusedRMSNorm(nn.Module):

    def __init__(self, size, eps=1e-6, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(size, device=device,
                                              dtype=dtype))

    def forward(self, x, residual=None):
        """The norm of ``x``, or ``(norm, x + residual)``."""
        return functions.rms_norm(x, self.weight, residual=residual,
                                  eps=self.eps)

    def extra_repr(self):
        return '{}, eps={}'.format(self.weight.numel(), self.eps)
