"""Corners of the sequence-model links and models, on the CPU."""

import pytest
import torch
import torch.nn as nn
from torch.utils.checkpoint import checkpoint

import chainermn_amd
from chainermn_amd import functions, links, ops
from chainermn_amd.models.seq2seq import Seq2Seq, make_model_parallel
from chainermn_amd.ops._dropout import philox, philox_words
from chainermn_amd.testing import run_distributed


# ---- the stream of dropout ---------------------------------------------------

@pytest.mark.parametrize('counter,key,words', [
    ((0,) * 4, (0,) * 2, '6627e8d5 e169c58d bc57ac4c 9b00dbd8'),
    ((2 ** 32 - 1,) * 4, (2 ** 32 - 1,) * 2,
     '408f276d 41c83b0e a20bc7c6 6d5451fd'),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344),
     (0xa4093822, 0x299f31d0), 'd16cfe09 94fdcceb 5001e420 24126ea1')])
def test_philox_published_vectors(counter, key, words):
    # the numbers themselves, and by tensors
    want = [int(w, 16) for w in words.split()]
    assert list(philox(*counter, *key)) == want
    assert [int(w) for w in philox(*(torch.tensor(x)
                                     for x in counter + key))] == want
    # the stream puts a block's number in front of the call's, each with its
    # lower half first, and the seed into the key
    def signed(low, high):
        x = high << 32 | low
        return x - 2 ** 64 if x >= 2 ** 63 else x
    if counter[1] < 2 ** 31:  # a block's number is not negative
        block = signed(*counter[:2])
        assert philox_words(torch.tensor([signed(*key), signed(
            *counter[2:])]), 4, block).tolist() == want


def test_philox_words_of_all_halves():
    seed, call, block = -0x123456789abcdef, 0x7edcba987654321f, 0x35a4e00000007
    m = 2 ** 32 - 1
    want = [list(philox(b & m, b >> 32, call & m, call >> 32, seed & m,
                        (seed >> 32) & m)) for b in (block, block + 1)]
    assert philox_words(torch.tensor([seed, call]), 8, block).tolist() == \
        want[0] + want[1]
    assert philox_words(torch.tensor([seed, call]), 5, block).tolist() == \
        (want[0] + want[1])[:5]


# ---- dropout that is computed again ------------------------------------------

def grads_of(make, run, x):
    """The output, gradients and dropouts' states of a new module."""
    torch.manual_seed(5)
    module = make()
    x = x.clone().requires_grad_()
    y = run(module, x)
    y.square().sum().backward()
    return [y.detach(), x.grad] + [p.grad for p in module.parameters()] + [
        b for name, b in module.named_buffers() if 'rng_state' in name]


def same(got, want):
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert (a is None and b is None) or torch.equal(a, b)


def layers():
    return nn.ModuleList([nn.Linear(12, 12), links.FusedDropout(0.4),
                          nn.Linear(12, 12)])


def segment(module, x):
    a, d, b = module
    h = d(a(x)) * x  # the link twice, and its outputs are factors
    return x + d(b(h)) * h


@pytest.mark.parametrize('reentrant', [False, True])
def test_dropout_in_forgotten_segments(reentrant):
    x = torch.randn(7, 12)

    def plain(module, x):
        return segment(module, segment(module, x))

    def forgotten(module, x):
        for _ in range(2):
            x = functions.forget(lambda t: segment(module, t), x,
                                 use_reentrant=reentrant)
        return x

    want = grads_of(layers, plain, x)
    assert want[-1][1] == 4  # calls
    same(grads_of(layers, forgotten, x), want)


@pytest.mark.parametrize('outer', [False, True])
@pytest.mark.parametrize('inner', [False, True])
def test_dropout_in_nested_forgotten_segments(outer, inner):
    x = torch.randn(7, 12)

    def twice(module, x):
        for _ in range(2):
            x = functions.forget(lambda t: segment(module, t), x,
                                 use_reentrant=inner)
        return segment(module, x)

    want = grads_of(layers, lambda m, x: segment(m, segment(m, segment(
        m, x))), x)
    same(grads_of(layers, lambda m, x: functions.forget(
        lambda t: twice(m, t), x, use_reentrant=outer), x), want)


def test_a_forgotten_segment_can_be_differentiated_twice_over():
    torch.manual_seed(5)
    module, x = layers(), torch.randn(7, 12, requires_grad=True)
    y = functions.forget(lambda t: segment(module, t), x)
    first, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    # a call in between has numbers of its own and takes none away
    module[1](torch.ones(100))
    again, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(first, again) and module[1].rng_state[1] == 3


@pytest.mark.parametrize('reentrant', [False, True])
def test_attention_rnn_with_dropout_forgotten(reentrant):
    x = torch.randn(3, 9, 16)

    def make():
        return links.LinearAttentionRNN(16, 16, num_layers=2, n_heads=2,
                                        dropout=0.3)

    want = grads_of(make, lambda m, x: m(x)[0], x)
    same(grads_of(make, lambda m, x: functions.forget(
        lambda t: m(t)[0], x, use_reentrant=reentrant), x), want)


@pytest.mark.parametrize('reentrant', [False, True])
def test_dropout_under_a_checkpoint_that_does_not_know_it(reentrant):
    module, x = layers(), torch.randn(7, 12, requires_grad=True)

    def run(x):
        return checkpoint(lambda t: segment(module, t), x,
                          use_reentrant=reentrant).sum()

    loss = run(x)
    with pytest.raises(RuntimeError, match='functions.forget'):
        loss.backward()
    # without a forgotten call around it, being within one does not help
    loss = functions.forget(run, x, use_reentrant=False)
    with pytest.raises(RuntimeError, match='functions.forget'):
        loss.backward()
    module.eval()  # nothing is dropped, and nothing is refused
    run(x).backward()
    assert torch.isfinite(x.grad).all()


def test_a_recomputation_that_drops_more_often():
    d, x = links.FusedDropout(0.4), torch.randn(8, requires_grad=True)
    calls = []

    def growing(x):
        calls.append(0)
        for _ in calls:
            x = d(x)
        return x.square()

    y = functions.forget(growing, x, use_reentrant=True)
    with pytest.raises(RuntimeError, match='more often'):
        y.sum().backward()
    # and neither call leaves a recomputation open behind it
    first, second = d(torch.ones(100)), d(torch.ones(100))
    assert not torch.equal(first, second)


def test_a_forgotten_segment_that_fails():
    d, x = links.FusedDropout(0.4), torch.randn(8, requires_grad=True)

    def broken(x):
        d(x)
        raise KeyError('broken')

    with pytest.raises(KeyError):
        functions.forget(broken, x)
    y = functions.forget(lambda t: d(t) * t, x)
    g, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g != 0, y != 0) and d.rng_state[1] == 2


# ---- single tokens -----------------------------------------------------------

def test_single_tokens_keep_a_long_memory():
    # a rounded decay would be off by 2^-25 in each step, the same way for all
    ld = torch.tensor([-1 / 3e4, -1 / 4096])
    state = torch.rand(1, 2, 64, 64) + 0.5
    zero = torch.zeros(1, 2, 64)
    want = state.double() * torch.exp(2000 * ld.double())[:, None, None]
    for _ in range(2000):
        ops.linear_attention_step(zero, zero, zero, state, ld)
    mean = ((state.double() - want) / want).mean((0, 2, 3))
    # 2000 roundings that cancel over 4096 elements: a spread of 45 E / 64
    assert float(mean.abs().max()) <= 8 * 2.0 ** -24


# ---- Seq2Seq -----------------------------------------------------------------

def test_translate_leaves_each_module_in_its_mode():
    model = Seq2Seq(20, 20, 16, 1, rnn='attention', dropout=0.1)
    model.encoder.eval()  # frozen
    before = {name: m.training for name, m in model.named_modules()}
    assert model.training and not model.encoder.dropout.training
    model.translate(torch.tensor([[1, 2]]), 3)
    assert {name: m.training for name, m in model.named_modules()} == before
    with pytest.raises(IndexError):
        model.translate(torch.tensor([[1, 99]]), 3)
    assert {name: m.training for name, m in model.named_modules()} == before


@pytest.mark.parametrize('units,heads', [
    (200, 4), (250, 5), (500, 10), (1000, 20),  # no multiples of 64
    (8, 1), (100, 1), (192, 3), (512, 8), (1024, 16)])
def test_attention_rnn_chooses_heads_that_fit(units, heads):
    rnn = links.LinearAttentionRNN(units, units)
    assert (rnn.n_heads, rnn.head) == (heads, units // heads)
    y, state = rnn(torch.randn(2, 3, units))
    assert y.shape == (2, 3, units)
    assert state.shape == (1, 2, heads, units // heads, units // heads)


def test_seq2seq_of_any_units():
    model = Seq2Seq(9, 9, 200, 1, rnn='attention')
    ids = torch.tensor([[1, 2, 3]])
    model(ids, ids, ids).backward()
    # units without heads of a useful size are still refused
    for units in (509, 262):
        with pytest.raises(ValueError, match='n_heads'):
            links.LinearAttentionRNN(8, units)


def _padded_worker(rank, size):
    comm = chainermn_amd.create_communicator('naive')
    model, xs, ys, lengths = padded_batch()
    part = make_model_parallel(model, comm, 0, 1)
    if rank == 0:
        part(xs, lengths).backward()
        return {'g': model.encoder.embed.weight.grad}
    loss = part(ys, ys)
    loss.backward()
    return {'loss': loss.detach(), 'g': model.decoder.embed.weight.grad}


def padded_batch():
    torch.manual_seed(1)
    model = Seq2Seq(11, 13, 16, n_layers=2, rnn='attention')
    return (model, torch.randint(0, 11, (3, 5)), torch.randint(0, 13, (3, 4)),
            torch.tensor([5, 0, 2]))


def test_a_padded_batch_split_over_ranks():
    results = run_distributed(_padded_worker, 2)
    model, xs, ys, lengths = padded_batch()
    loss = model(xs, ys, ys, lengths)
    loss.backward()
    assert torch.allclose(torch.from_numpy(results[1]['loss']),
                          loss.detach(), atol=1e-5)
    for rank, part in enumerate((model.encoder, model.decoder)):
        assert torch.allclose(torch.from_numpy(results[rank]['g']),
                              part.embed.weight.grad, atol=1e-5)
