"""Sequence-model operators on the CPU: their plain forms, gradients against
differences, and what they refuse."""

import pytest
import torch

from chainermn_amd import functions, ops
from chainermn_amd.ops._dropout import philox_words


def key_of(seed, call):
    return torch.tensor([seed, call])


def test_philox_known_answers():
    # the published test vectors of Philox4x32-10: all-zero and all-one
    # counters and keys; the block number is the counter's lower half
    words = philox_words(key_of(0, 0), 4)
    assert [hex(int(w)) for w in words] == [
        '0x6627e8d5', '0xe169c58d', '0xbc57ac4c', '0x9b00dbd8']


def test_dropout():
    x = torch.randn(50, 31, requires_grad=True)
    key = key_of(-5, 3)
    y = functions.dropout(x, key, ratio=0.25)
    kept = y != 0
    assert torch.equal(y[kept], (x.detach().float() * (1 / 0.75))[kept])
    assert 0.70 < kept.float().mean() < 0.80
    g, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g != 0, kept)
    assert not torch.equal(kept, functions.dropout(x, key_of(-5, 4), 0.25)
                           != 0)
    assert torch.equal(functions.dropout(x, key, ratio=0.0), x)


def test_dropout_next_key():
    state = key_of(9, 0)
    keys = [ops.dropout_next_key(state).tolist() for _ in range(3)]
    assert keys == [[9, 0], [9, 1], [9, 2]] and state.tolist() == [9, 3]


def test_embed_id():
    W = torch.randn(7, 5, requires_grad=True)
    ids = torch.tensor([[1, 6, -1], [1, 0, 1]])
    y = functions.embed_id(ids, W, ignore_label=-1, scale=2.0)
    assert y.shape == (2, 3, 5) and not y[0, 2].any()
    assert torch.equal(y[1, 1], 2 * W[0])
    g, = torch.autograd.grad(y.sum(), W)
    assert g[:, 0].tolist() == [2, 6, 0, 0, 0, 0, 2]
    with pytest.raises(IndexError):
        functions.embed_id(torch.tensor([7]), W)
    with pytest.raises(IndexError):
        functions.embed_id(torch.tensor([-2]), W, ignore_label=-1)


def test_gradients_against_differences():
    torch.manual_seed(0)
    ld = torch.tensor([-0.3, 0.0])
    lengths = torch.tensor([5, 3])

    def norm(x, r, w):
        y, h = functions.rms_norm(x, w, residual=r)
        return (y * y.detach().cos()).sum() + (h * 0.3).sum()

    def attn(q, k, v, s):
        o, last = functions.linear_attention(q, k, v, ld, initial_state=s,
                                             lengths=lengths)
        return (o * torch.arange(o.numel()).view(o.shape).cos()).sum() \
            + (last * torch.arange(last.numel()).view(last.shape).sin()).sum()

    # fp32 inside: a step of 2^-6 leaves about 2^-24 / 2^-6 of the values,
    # and the functions are linear or smooth in each argument
    for f, shapes in ((norm, [(3, 4), (3, 4), (4,)]),
                      (attn, [(2, 5, 2, 3), (2, 5, 2, 3), (2, 5, 2, 4),
                              (2, 2, 3, 4)])):
        xs = [torch.randn(s).requires_grad_() for s in shapes]
        if f is norm:  # y.detach() is a constant of the formula
            y0 = functions.rms_norm(xs[0], xs[2], residual=xs[1])[0].detach()

            def f(x, r, w):
                y, h = functions.rms_norm(x, w, residual=r)
                return (y * y0.cos()).sum() + (h * 0.3).sum()
        grads = torch.autograd.grad(f(*xs), xs)
        for i, g in enumerate(grads):
            d = torch.randn(xs[i].shape)
            with torch.no_grad():
                up = [x + (2 ** -6 * d if j == i else 0)
                      for j, x in enumerate(xs)]
                down = [x - (2 ** -6 * d if j == i else 0)
                        for j, x in enumerate(xs)]
                slope = (f(*up) - f(*down)) / 2 ** -5
            assert abs(float(slope) - float((g * d).sum())) < 2e-2 * (
                1 + abs(float(slope)))


def test_linear_attention_is_its_recurrence():
    torch.manual_seed(1)
    q, k = torch.randn(2, 9, 3, 4), torch.randn(2, 9, 3, 4)
    v, s0 = torch.randn(2, 9, 3, 5), torch.randn(2, 3, 4, 5)
    ld = torch.tensor([-0.5, 0.0, float('-inf')])
    o, s = functions.linear_attention(q, k, v, ld, initial_state=s0,
                                      lengths=torch.tensor([9, 4]))
    state = s0.clone()
    for i in range(9):
        if i == 4:
            assert torch.allclose(s[1], state[1], atol=1e-5)
        step = ops.linear_attention_step(q[:, i], k[:, i], v[:, i], state, ld)
        assert torch.allclose(o[0, i], step[0], atol=1e-5)
        assert not o[1, 4:].any()
    assert torch.allclose(s[0], state[0], atol=1e-5)


def test_rms_norm_fp8():
    x, w = torch.randn(6, 64), torch.ones(64)
    x[2] = 0
    q, scales, h = ops.rms_norm_fp8(x, w, residual=x, group=32)
    assert q.dtype == torch.float8_e4m3fn and scales.shape == (6, 2)
    assert torch.equal(h, 2 * x) and (scales[2] == 1).all()
    y = functions.rms_norm(2 * x, w)
    back = q.float().view(6, 2, 32) * scales[..., None]
    # half a step of e4m3 is 2^-4 of the value
    assert ((back.view(6, 64) - y).abs() <= 2 ** -4 * y.abs() * 1.01
            + scales.max() * 2 ** -9).all()


def test_refusals():
    x, ld = torch.randn(2, 3, 2, 8), torch.zeros(2)
    with pytest.raises(ValueError, match='alike'):
        functions.linear_attention(x, x[:, :2], x, ld)
    with pytest.raises(ValueError, match='alike'):
        functions.linear_attention(x[0], x[0], x[0], ld)
    with pytest.raises(ValueError, match='heads'):
        functions.linear_attention(x, x, x, torch.zeros(3))
    with pytest.raises(ValueError, match='1 to 128'):
        y = torch.randn(1, 2, 2, 129)
        functions.linear_attention(y, y, y, ld)
    with pytest.raises(TypeError, match='q, k and v'):
        functions.linear_attention(x, x.bfloat16(), x, ld)
    with pytest.raises(TypeError, match='float32'):
        functions.linear_attention(x, x, x, ld.double())
    with pytest.raises(ValueError, match='not differentiable'):
        functions.linear_attention(x, x, x, ld.clone().requires_grad_())
    with pytest.raises(ValueError, match='state is'):
        functions.linear_attention(x, x, x, ld, initial_state=torch.zeros(
            2, 2, 8, 7))
    with pytest.raises(TypeError, match='state is float32'):
        functions.linear_attention(x, x, x, ld, initial_state=torch.zeros(
            2, 2, 8, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match='lengths'):
        functions.linear_attention(x, x, x, ld, lengths=torch.ones(3))
    q = x[:, 0].clone().requires_grad_()
    with pytest.raises(ValueError, match='not differentiable'):
        ops.linear_attention_step(q, q, q, torch.zeros(2, 2, 8, 8), ld)

    w = torch.ones(8)
    with pytest.raises(ValueError, match='weight'):
        functions.rms_norm(x, torch.ones(7))
    with pytest.raises(TypeError, match='weight'):
        functions.rms_norm(x, w.half())
    with pytest.raises(ValueError, match='residual'):
        functions.rms_norm(x, w, residual=x[:1])
    with pytest.raises(ValueError, match='16384'):
        functions.rms_norm(torch.zeros(1, 16385), torch.ones(16385))
    with pytest.raises(ValueError, match='groups'):
        ops.rms_norm_fp8(torch.zeros(1, 40), torch.ones(40), group=16)
    with pytest.raises(ValueError, match='groups'):
        ops.rms_norm_fp8(torch.zeros(1, 48), torch.ones(48), group=24)

    W = torch.randn(4, 3)
    with pytest.raises(TypeError, match='int32 or int64'):
        functions.embed_id(torch.zeros(2), W)
    with pytest.raises(ValueError, match='non-empty'):
        functions.embed_id(torch.zeros(2).long(), W[:0])
    with pytest.raises(TypeError, match='key'):
        functions.dropout(W, torch.zeros(2))
    for ratio in (1.0, -0.1, float('nan')):
        with pytest.raises(ValueError, match='ratio'):
            functions.dropout(W, key_of(0, 0), ratio=ratio)


def test_float64_stays_float64():
    torch.manual_seed(0)
    x = torch.randn(3, 4, 2, 8, dtype=torch.float64, requires_grad=True)
    w = torch.randn(8, dtype=torch.float64, requires_grad=True)
    ld = torch.tensor([-0.3, -0.1])
    # fp32 anywhere would be off by more than 1e-9 of differences of 1e-6
    assert torch.autograd.gradcheck(
        lambda x, w: functions.rms_norm(x, w, residual=x)[0], (x, w))
    assert torch.autograd.gradcheck(
        lambda x: functions.dropout(x, key_of(1, 2), ratio=0.3), (x,))
    assert torch.autograd.gradcheck(
        lambda x: functions.linear_attention(x, x, x, ld)[0], (x,))
    ids = torch.tensor([0, 2, -1, 2])
    assert torch.autograd.gradcheck(
        lambda W: functions.embed_id(ids, W, ignore_label=-1, scale=3.0),
        (torch.randn(3, 4, dtype=torch.float64, requires_grad=True),))


def test_lengths_of_another_type_are_refused():
    x, ld = torch.randn(2, 3, 2, 8), torch.zeros(2)
    with pytest.raises(TypeError, match='lengths'):
        functions.linear_attention(x, x, x, ld, lengths=torch.ones(2))
