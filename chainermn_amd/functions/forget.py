"""Activation checkpointing that knows the links' dropout."""

import threading

import torch
from torch.utils.checkpoint import checkpoint

_local = threading.local()  # a recomputation runs in a thread of its own


def _runs():
    if not hasattr(_local, 'runs'):
        _local.runs = []
    return _local.runs


class _Run(object):
    """A call of a forgotten function: the first one, which writes down its
    dropouts' keys, or a later one, which takes them in the same order."""

    def __init__(self, keys, again):
        self.keys, self.again, self.taken = keys, again, 0

    def take(self):
        if self.taken == len(self.keys):
            raise RuntimeError('forget: the recomputation calls dropout more '
                               'often than the forward pass did ({} times)'
                               .format(len(self.keys)))
        self.taken += 1
        return self.keys[self.taken - 1]


def dropout_key(draw):
    """The key of a dropout: ``draw()``, or in a recomputation the key of the
    forward pass."""
    key = None
    for run in _runs():  # the innermost one's, if several recompute
        if run.again:
            key = run.take()
    if key is None:
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError(
                'FusedDropout is called within a backward pass, where it '
                'would drop other elements than in the forward pass: '
                'checkpoint its caller by functions.forget, not by '
                'torch.utils.checkpoint')
        key = draw()
    for run in _runs():
        if not run.again:
            run.keys.append(key)
    return key


def forget(func, *xs, use_reentrant=False, preserve_rng_state=True):
    """``func(*xs)`` that keeps ``xs`` only and computes the rest once more in
    the backward pass (Chainer's ``forget``).

    It is ``torch.utils.checkpoint.checkpoint`` but for ``links.FusedDropout``
    within ``func``: a recomputation takes the keys of the forward pass, and
    the call numbers go up once.  Under ``checkpoint`` itself the link raises
    an error in the backward pass.  Calls can be nested.
    """
    keys, done = [], [False]

    def run(*args):
        here = _Run(keys, done[0])
        _runs().append(here)
        try:
            out = func(*args)
            done[0] = True
            return out
        finally:
            _runs().pop()
            if not done[0]:
                del keys[:]

    return checkpoint(run, *xs, use_reentrant=use_reentrant,
                      preserve_rng_state=preserve_rng_state)
