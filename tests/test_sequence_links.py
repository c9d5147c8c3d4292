"""The sequence-model links and the models that are made of them, on the
CPU; and one training step of them together on a GPU."""

import pytest
import torch
import torch.nn as nn

import chainermn_amd
from chainermn_amd import links
from chainermn_amd.models.seq2seq import Seq2Seq, make_model_parallel
from chainermn_amd.testing import run_distributed


def test_fused_embedding_is_a_drop_in():
    torch.manual_seed(0)
    a = nn.Embedding(9, 4)
    b = links.FusedEmbedding(9, 4)
    b.load_state_dict(a.state_dict())
    ids = torch.randint(0, 9, (3, 5))
    assert torch.equal(a(ids), b(ids))
    for m in (a, b):
        m(ids).square().sum().backward()
    assert torch.allclose(a.weight.grad, b.weight.grad)
    with pytest.raises(TypeError, match='max_norm'):
        links.FusedEmbedding(9, 4, max_norm=1.0)


def test_fused_dropout_state():
    torch.manual_seed(0)
    d = links.FusedDropout(0.5)
    x = torch.ones(1000)
    first, second = d(x), d(x)
    assert not torch.equal(first, second)
    assert d.rng_state[1] == 2
    again = links.FusedDropout(0.5)
    again.load_state_dict(d.state_dict())
    assert torch.equal(again(x), d(x))
    d.eval()
    assert d(x) is x and d.rng_state[1] == 3
    d.double()  # the state stays whole
    assert d.rng_state.dtype == torch.int64

    class Rank1(object):
        rank = 1

    other = links.FusedDropout(0.5, comm=Rank1())
    other.load_state_dict(again.state_dict())
    assert not torch.equal(other(x), again(x))
    with pytest.raises(ValueError, match='ratio'):
        links.FusedDropout(1.0)


def _rnn(**kwargs):
    torch.manual_seed(3)
    return links.LinearAttentionRNN(6, 16, num_layers=2, n_heads=2,
                                    **kwargs)


def test_attention_rnn_in_pieces():
    rnn = _rnn()
    x = torch.randn(3, 10, 6)
    y, state = rnn(x)
    assert y.shape == (3, 10, 16) and state.shape == (2, 3, 2, 8, 8)
    y1, s1 = rnn(x[:, :4])
    y2, s2 = rnn(x[:, 4:], s1)
    assert torch.allclose(torch.cat((y1, y2), 1), y, atol=1e-5)
    assert torch.allclose(s2, state, atol=1e-5)
    s = s1.detach().clone()
    steps = [rnn.step(x[:, i], s) for i in range(4, 10)]
    assert torch.allclose(torch.stack(steps, 1), y[:, 4:], atol=1e-5)
    assert torch.allclose(s, state, atol=1e-5)


def test_attention_rnn_of_a_padded_batch():
    rnn = _rnn()
    x = torch.randn(3, 10, 6)
    lengths = torch.tensor([10, 0, 7])
    _, state = rnn(x, lengths=lengths)
    for i, n in enumerate(lengths.tolist()):
        _, alone = rnn(x[i:i + 1, :n])
        assert torch.allclose(state[:, i], alone[:, 0], atol=1e-5)


def test_attention_rnn_keeps_its_decays_in_fp32():
    rnn = _rnn().bfloat16()
    assert rnn.log_decay.dtype == torch.float32
    assert rnn.layers[0].qkv.weight.dtype == torch.bfloat16
    y, state = rnn(torch.randn(2, 5, 6, dtype=torch.bfloat16))
    assert y.dtype == torch.bfloat16 and state.dtype == torch.float32
    # its state dict holds what is learned
    assert 'log_decay' not in rnn.state_dict()


def test_refusals():
    with pytest.raises(ValueError, match='heads'):
        links.LinearAttentionRNN(8, 9, n_heads=2)
    with pytest.raises(ValueError, match='128'):
        links.LinearAttentionRNN(8, 512, n_heads=2)
    with pytest.raises(ValueError, match='layers'):
        links.LinearAttentionRNN(8, 8, num_layers=0)
    with pytest.raises(ValueError, match='memory'):
        links.LinearAttentionRNN(8, 8, memory=(9, 3))
    with pytest.raises(ValueError, match='batch_first'):
        links.LinearAttentionRNN(8, 8, batch_first=False)
    with pytest.raises(ValueError, match='layers'):
        _rnn()(torch.randn(1, 2, 6), torch.zeros(1, 1, 2, 8, 8))
    with pytest.raises(ValueError, match='rnn'):
        Seq2Seq(5, 5, 8, rnn='gru')
    with pytest.raises(ValueError, match='lengths'):
        Seq2Seq(5, 5, 8).encoder(torch.zeros(1, 2).long(),
                                 torch.tensor([1]))


def test_seq2seq_without_options_is_what_it_was():
    torch.manual_seed(1)
    names = set(Seq2Seq(11, 13, 16).state_dict())
    assert names == {'encoder.embed.weight', 'decoder.embed.weight',
                     'decoder.out.weight', 'decoder.out.bias'} | {
        '{}.rnn.{}_{}_l{}'.format(part, kind, side, layer)
        for part in ('encoder', 'decoder') for kind in ('weight', 'bias')
        for side in ('ih', 'hh') for layer in (0, 1)}


@pytest.mark.parametrize('rnn', ['lstm', 'attention'])
def test_seq2seq_trains_and_translates(rnn):
    torch.manual_seed(1)
    model = Seq2Seq(11, 13, 16, n_layers=2, rnn=rnn, dropout=0.2,
                    fused_ops=True)
    xs, ys = torch.randint(0, 11, (4, 6)), torch.randint(0, 13, (4, 5))
    model(xs, ys, ys).backward()
    for name, p in model.named_parameters():
        unused = rnn == 'attention' and name.startswith('encoder.rnn') and (
            name == 'encoder.rnn.norm.weight'
            or name.startswith('encoder.rnn.layers.1.out')
            or name.startswith('encoder.rnn.layers.1.head_norm'))
        assert (p.grad is None) == unused, name
        assert p.grad is None or torch.isfinite(p.grad).all()
    out = model.translate(xs, 7)
    assert out.shape == (4, 7) and model.training
    # greedy generation is what teacher forcing on it says
    model.eval()
    ys_in = torch.cat((torch.zeros(4, 1).long(), out[:, :-1]), 1)
    logits = model.decoder(ys_in, model.encoder(xs))
    assert torch.equal(logits.argmax(-1), out)


def test_attention_rnn_under_autocast():
    rnn = _rnn()
    x = torch.randn(2, 5, 6, requires_grad=True)
    with torch.autocast('cpu', dtype=torch.bfloat16):
        y, state = rnn(x)
        one = rnn.step(x[:, 0], torch.zeros_like(state))
    # 16-bit products between an fp32 sum of layers and fp32 states
    assert y.dtype == one.dtype == state.dtype == torch.float32
    y.sum().backward()
    assert torch.isfinite(x.grad).all() and x.grad.any()


def test_translate_leaves_the_mode_as_it_was():
    model = Seq2Seq(20, 20, 16, 1, rnn='attention')
    with pytest.raises(IndexError):
        model.translate(torch.tensor([[1, 99]]), 3)
    assert model.training


def _mp_worker(rank, size):
    comm = chainermn_amd.create_communicator('naive')
    torch.manual_seed(1)
    model = Seq2Seq(11, 13, 16, n_layers=2, rnn='attention', fused_ops=True)
    part = make_model_parallel(model, comm, 0, 1)
    torch.manual_seed(2)
    xs, ys = torch.randint(0, 11, (2, 5)), torch.randint(0, 13, (2, 4))
    if rank == 0:
        part(xs).backward()
        return {'g': model.encoder.embed.weight.grad}
    loss = part(ys, ys)
    loss.backward()
    return {'loss': loss.detach(), 'g': model.decoder.embed.weight.grad}


def test_seq2seq_attention_model_parallel():
    results = run_distributed(_mp_worker, 2)
    torch.manual_seed(1)
    model = Seq2Seq(11, 13, 16, n_layers=2, rnn='attention', fused_ops=True)
    torch.manual_seed(2)
    xs, ys = torch.randint(0, 11, (2, 5)), torch.randint(0, 13, (2, 4))
    loss = model(xs, ys, ys)
    loss.backward()
    assert torch.allclose(torch.from_numpy(results[1]['loss']),
                          loss.detach(), atol=1e-5)
    for rank, part in enumerate((model.encoder, model.decoder)):
        assert torch.allclose(torch.from_numpy(results[rank]['g']),
                              part.embed.weight.grad, atol=1e-5)


def _nstep_worker(rank, size):
    comm = chainermn_amd.create_communicator('naive')
    rnn = _rnn()
    torch.manual_seed(9)
    x = torch.randn(2, 9, 6)
    if rank == 0:
        wrapped = links.create_multi_node_n_step_rnn(rnn, comm, rank_out=1)
        y, _, delegate = wrapped(x[:, :5])
        torch.autograd.backward([y.sum(), delegate],
                                [None, torch.zeros_like(delegate)]
                                if delegate.dim() else [None, None])
    else:
        wrapped = links.create_multi_node_n_step_rnn(rnn, comm, rank_in=0)
        y, _, _ = wrapped(x[:, 5:])
        y.sum().backward()
    return {'y': y.detach(),
            'g': torch.cat([p.grad.reshape(-1) for p in rnn.parameters()])}


def test_a_sequence_split_over_ranks():
    results = run_distributed(_nstep_worker, 2)
    rnn = _rnn()
    torch.manual_seed(9)
    x = torch.randn(2, 9, 6)
    y, _ = rnn(x)
    y.sum().backward()
    got = torch.cat([torch.from_numpy(r['y']) for r in results], 1)
    assert torch.allclose(got, y.detach(), atol=1e-5)
    g = sum(torch.from_numpy(r['g']) for r in results)
    want = torch.cat([p.grad.reshape(-1) for p in rnn.parameters()])
    assert torch.allclose(g, want, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason='needs ROCm GPU')
@pytest.mark.parametrize('rnn', ['lstm', 'attention'])
def test_seq2seq_on_a_gpu_is_what_it_is_on_the_cpu(rnn):
    """Embedding, dropout, norms and attention of a whole training step: the
    CPU computes the same step, dropped elements included, in plain forms."""
    def step(device):
        torch.manual_seed(1)
        model = Seq2Seq(50, 60, 128, n_layers=2, rnn=rnn, dropout=0.2,
                        fused_ops=True).to(device)
        g = torch.Generator().manual_seed(2)
        xs = torch.randint(0, 50, (5, 37), generator=g).to(device)
        ys = torch.randint(0, 60, (5, 21), generator=g).to(device)
        loss = model(xs, ys, ys)
        loss.backward()
        return model, [loss.detach().cpu()] + [
            p.grad.cpu() for p in model.parameters() if p.grad is not None]

    _, want = step('cpu')
    model, got = step('cuda')
    assert len(want) == len(got)
    for a, b in zip(got, want):
        # fp32 on both sides: sums of at most 128 * 185 terms
        assert (a - b).norm() <= 1e-4 * b.norm() + 1e-7
    xs = torch.randint(0, 50, (3, 9), device='cuda')
    out = model.translate(xs, 6)
    model.eval()
    ys_in = torch.cat((torch.zeros_like(out[:, :1]), out[:, :-1]), 1)
    with torch.no_grad():
        logits = model.decoder(ys_in, model.encoder(xs))
    top = logits.topk(2, -1)
    clear = (top.values[..., 0] - top.values[..., 1]) > 1e-4
    assert torch.equal(out[clear], top.indices[..., 0][clear])


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason='needs ROCm GPU')
def test_attention_rnn_under_autocast_on_a_gpu():
    torch.manual_seed(1)
    rnn = links.LinearAttentionRNN(64, 128, num_layers=2).cuda()
    x = torch.randn(3, 40, 64, device='cuda', requires_grad=True)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        y, state = rnn(x)
        one = rnn.step(x[:, 0], torch.zeros_like(state))
    assert y.dtype == one.dtype == state.dtype == torch.float32
    y.sum().backward()
    assert torch.isfinite(x.grad).all() and x.grad.any()
