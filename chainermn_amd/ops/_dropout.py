"""Dropout from a counter-based generator: the stream, and the CPU form.

Kernels: _hip/csrc/dropout.hip.
"""

import torch

from chainermn_amd.ops._embedding import wide

_M = 0xffffffff


def dropout_threshold(ratio):
    """A word below this drops its element; and the factor of the others."""
    ratio = float(ratio)
    if not 0.0 <= ratio < 1.0:
        raise ValueError('dropout: ratio must be in [0, 1), not {}'
                         .format(ratio))
    return min(int(round(ratio * 2.0 ** 32)), _M), 1.0 / (1.0 - ratio)


def check_key(x, key):
    if key.dtype != torch.int64 or key.numel() != 2:
        raise TypeError('dropout: the key is a tensor of two int64 '
                        '(seed, call)')
    if key.device != x.device:
        raise ValueError('dropout: x is on {}, the key on {}'
                         .format(x.device, key.device))


def _mul(a, c):
    """High and low words of a 32 x 32 bit product, in 63 bits."""
    low, high = a * (c & 0xffff), a * (c >> 16)
    return (high + (low >> 16)) >> 16, (low + (high << 16)) & _M


def philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32-10 of a counter and a key: words below 2^32, as whole
    numbers or int64 tensors."""
    for _ in range(10):
        h0, l0 = _mul(0xD2511F53, c0)
        h1, l1 = _mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _M, (k1 + 0xBB67AE85) & _M
    return c0, c1, c2, c3


def philox_words(key, n, block=0):
    """Words 4 * block .. 4 * block + n - 1 (int64 below 2^32) of the
    Philox4x32-10 stream whose key is ``key[0]`` and whose upper counter half
    is ``key[1]``."""
    block = torch.arange(block, block + (n + 3) // 4, device=key.device)
    c2 = (key[1] & _M).expand_as(block)
    c3 = ((key[1] >> 32) & _M).expand_as(block)
    words = philox(block & _M, block >> 32, c2, c3, key[0] & _M,
                   (key[0] >> 32) & _M)
    return torch.stack(words, 1).reshape(-1)[:n]


def dropout_plain(x, key, threshold, scale):
    keep = (philox_words(key, x.numel()) >= threshold).view(x.shape)
    y = (wide(x) * scale).to(x.dtype)
    return torch.where(keep, y, torch.zeros((), dtype=x.dtype))


def dropout_next_key(state, stream=0):
    """The key (seed, call) of one dropout call, from the int64 pair
    ``state``, whose call number goes up by one.  Each ``stream`` (a rank,
    for instance) of a state has numbers of its own.  On the GPU the state is
    read and counted there, so a replayed graph draws new numbers."""
    if state.dtype != torch.int64 or state.numel() != 2:
        raise TypeError('dropout: the state is a tensor of two int64 '
                        '(seed, call)')
    # streams are an odd constant apart, modulo 2^64
    shift = int(stream) * 0x9E3779B97F4A7C15 & 0xffffffffffffffff
    shift -= (shift >> 63) << 64
    if state.is_cuda:
        from chainermn_amd import ops
        return ops.require().dropout_next_key(state, shift)
    key = state.clone()
    key[0] += shift
    state[1] += 1
    return key
