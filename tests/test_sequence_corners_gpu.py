"""Corners of the sequence-model operators on a GPU, against values that are
known in 64 bits.

``E`` is half a step of fp32; the bounds beside the tests count roundings.
"""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from chainermn_amd import functions, links, ops
    from chainermn_amd.ops._dropout import philox_words
    DEV = torch.device('cuda:0')
else:
    pytest.skip('needs ROCm GPU', allow_module_level=True)

TYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24


def rand(*shape, t=torch.float32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.rand(shape, generator=g, device=DEV).to(t) + 0.5


def close(got, want, relative, least):
    """|got - want| <= (u + relative) |want| + least, u half a step of got."""
    assert got.shape == want.shape
    t = got.dtype
    most = (torch.finfo(t).eps / 2 + relative) * want.abs() + least \
        + torch.finfo(t).tiny * torch.finfo(t).eps / 2
    off = (got.double() - want).abs()
    assert bool((off <= most).all()), 'off by {:.3g} of the bound'.format(
        float((off / most).max()))


# ---- linear attention --------------------------------------------------------

@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('length,rate', [
    (1, -0.7), (31, -0.5), (40, -0.3), (64, -0.5), (64, -0.7), (70, -1.0),
    (70, -0.02), (600, -0.13), (600, -0.001)])
def test_a_state_that_nothing_is_added_to_decays(t, length, rate):
    """Long after a state came in, with tokens that add nothing to it, it is
    still lam^n of what it was; so are its outputs, and backwards its
    gradient."""
    h, dk, dv = 2, 48, 40
    ld = torch.full((h,), rate, device=DEV)
    q, v = rand(1, length, h, dk, t=t), rand(1, length, h, dv, t=t, seed=1)
    k = torch.zeros(1, length, h, dk, device=DEV, dtype=t)
    s0, gs = rand(1, h, dk, dv, seed=2), rand(1, h, dk, dv, seed=3)
    k.requires_grad_()
    s0.requires_grad_()
    o, s = functions.linear_attention(q, k, v, ld, initial_state=s0,
                                      scale=1.0)
    gk, g0 = torch.autograd.grad(s, (k, s0), gs)
    rate = float(ld[0])
    lam = torch.exp(rate * torch.arange(
        length + 1, device=DEV, dtype=torch.float64))
    # The state, for each chunk of 32 tokens: the rounding of rate * n, which
    # is |rate| n E of the exponential, the exponential's 2 E and the
    # product's E; one more of these where segments are joined.
    chunks = length // 32 + 2
    state = (4 * chunks + 2 * abs(rate) * length) * E
    # Numbers below 2^-126 may be taken as zero.
    least = 2.0 ** -126
    close(s.detach(), s0.detach().double() * lam[length], state, least)
    close(g0, gs.double() * lam[length], state, least)
    # A token's own decay is exp2 of a product of three rounded factors; then
    # a sum of positive products, of which the cut terms leave out 2^-21, or
    # 2^-14 on the way to 16 bits, for each of two products.
    def sums(n):
        cut = 2.0 ** -21 if t == torch.float32 else 2.0 ** -14
        return state + (n + 8 + 4 * abs(rate) * length) * E + 2 * cut
    want = torch.einsum('bthi,bhij->bthj', q.double(), s0.detach().double())
    close(o.detach(), want * lam[1:, None, None], sums(dk), dk * least)
    want = torch.einsum('bthj,bhij->bthi', v.double(), gs.double())
    close(gk, want * lam[:-1].flip(0)[:, None, None], sums(dv), dv * least)


def test_products_of_terms_at_their_worst():
    """Numbers whose three terms of eight bits are as large as they can be.

    Of a number 2^e (1 + ..) the second term is below 2^-7 2^e and the third
    below 2^-15 2^e.  The products that are left out, of second with third and
    third with third terms, are below 2^-21 of the product, and the one sum of
    its size is off by at most 2^-23.  An output is two such products after
    each other and a factor, the state one."""
    worst = 1 + 2.0 ** -7 - 2.0 ** -23
    g = torch.Generator().manual_seed(0)
    sign = torch.randint(0, 2, (3, 64, 1, 1, 1), generator=g) * 2.0 - 1
    power = 2.0 ** torch.randint(-9, 9, (3, 64, 1, 1, 1), generator=g)
    q, k, v = (worst * sign * power).to(DEV)
    o, s = functions.linear_attention(q, k, v, torch.zeros(1, device=DEV),
                                      scale=1.0)
    q, k, v = q.double(), k.double(), v.double()
    for got, want, bound in (
            (o, q * k * v, 2 * (2.0 ** -21 + 2.0 ** -23) + 2 * E),
            (s, k * v, 2.0 ** -21 + 2.0 ** -23 + E)):
        off = (got.double() - want).abs() / want.abs()
        assert float(off.max()) <= bound


@pytest.mark.parametrize('dv', [64, 61])
def test_single_tokens_forget_as_the_chunks_do(dv):
    """4096 tokens that add nothing: each element takes 4096 roundings of up
    to E, which cancel over the elements (a mean of 16 * 64 * dv of them, each
    of a spread of 64 E at most, is off by less than E).  What is forgotten in
    a step is off by 2 E of itself, 2 * 4096 / memory E in all.  A rounded decay
    would be off by up to E / 2 in each step, the same way for all."""
    memories = torch.tensor([8.0, 200.0, 4096.0, 7000.0, 30000.0], device=DEV)
    ld = -1 / memories
    h = len(ld)
    state, zero = rand(16, h, 64, dv), torch.zeros(16, h, 64, device=DEV)
    none = torch.zeros(16, h, dv, device=DEV)
    want = state.double() * torch.exp(4096 * ld.double())[:, None, None]
    tokens = torch.zeros(16, 4096, h, 64, device=DEV)
    _, chunked = functions.linear_attention(
        tokens, tokens, tokens[..., :dv], ld, initial_state=state)
    for _ in range(4096):
        ops.linear_attention_step(zero, zero, none, state, ld)
    for got in (state, chunked):
        mean = ((got.double() - want) / want)[:, 1:].mean((0, 2, 3))
        assert bool((mean.abs() <= (16 + 8192 / memories[1:]) * E).all()), mean
    # exp(-512); in steps of 2^-149 the rounding of m exp(-1/8) ends at an m of
    # four, since four times 1 - exp(-1/8) is below a half
    assert float(state[:, 0].max()) <= 4 * 2.0 ** -149


def test_a_single_token_of_extreme_decays():
    ld = torch.tensor([float('-inf'), 0.0, -1000.0, -0.7, -0.69], device=DEV)
    state, q = rand(2, 5, 8, 6, seed=1), rand(2, 5, 8)
    k, v = rand(2, 5, 8, seed=2), rand(2, 5, 6, seed=3)
    new = torch.einsum('bhi,bhj->bhij', k.double(), v.double())
    want = state.double() * torch.exp(ld.double())[:, None, None] + new
    o = ops.linear_attention_step(q, k, v, state, ld, scale=1.0)
    close(state, want, 3 * E, 0.0)  # all positive
    close(o, torch.einsum('bhi,bhij->bhj', q.double(), want), 14 * E, 0.0)


@pytest.mark.parametrize('b,h', [(0, 2), (3, 0)])
def test_gradients_of_no_sequences(b, h):
    q = torch.empty(b, 5, h, 8, device=DEV, requires_grad=True)
    v = torch.empty(b, 5, h, 4, device=DEV, requires_grad=True)
    s0 = torch.empty(b, h, 8, 4, device=DEV, requires_grad=True)
    o, s = functions.linear_attention(q, q, v, torch.zeros(h, device=DEV),
                                      initial_state=s0)
    for x, g in zip((q, v, s0), torch.autograd.grad(
            (o, s), (q, v, s0), (torch.ones_like(o), torch.ones_like(s)))):
        assert g.shape == x.shape and g.dtype == x.dtype


# ---- the stream of dropout ---------------------------------------------------

@pytest.mark.parametrize('seed,call', [
    (5, 0), (-0x123456789abcdef, 0x7edcba987654321f)])
def test_dropout_takes_all_halves_of_its_key(seed, call):
    key = torch.tensor([seed, call])
    kept = philox_words(key, 4003) >= 2 ** 31
    y = functions.dropout(torch.ones(4003, device=DEV), key.to(DEV), 0.5)
    assert torch.equal(y.cpu() != 0, kept)


def test_dropout_past_2_32_blocks():
    """2^34 elements and more: the block's number takes two words."""
    n = 2 ** 34 + 4099
    key = torch.tensor([0x1234567890abcdef, 3])
    x = torch.ones(n, device=DEV, dtype=torch.bfloat16)
    y = functions.dropout(x, key.to(DEV), ratio=0.5)
    for block, size in ((0, 4096), (2 ** 32 - 1024, 8192 + 3)):
        kept = philox_words(key, size, block) >= 2 ** 31
        assert torch.equal((y[4 * block:4 * block + size] != 0).cpu(), kept)
    del x, y
    torch.cuda.empty_cache()


# ---- what is changed between the passes --------------------------------------

def test_inputs_changed_between_the_passes_are_seen():
    """As for torch's own operators: an error, and no wrong gradient."""
    ids = torch.arange(6, device=DEV)
    key = torch.tensor([1, 2], device=DEV)
    ld = torch.full((2,), -0.1, device=DEV)
    w = rand(16)

    def attend(x):
        q = x.view(2, 3, 2, 8)
        return functions.linear_attention(q, q, q, ld)[0]

    for run, changed in [
            (lambda x: functions.rms_norm(x, w), None),
            (lambda x: functions.rms_norm(x.view(2, 3, 16), w, x.view(
                2, 3, 16))[0], None),
            (attend, None),
            (lambda x: functions.embed_id(ids, x), ids),
            (lambda x: functions.dropout(x, key), key)]:
        x = rand(6, 16).requires_grad_() * 1
        y = run(x)
        (x if changed is None else changed).add_(1)
        with pytest.raises(RuntimeError, match='inplace'):
            y.sum().backward()


# ---- dropout that is computed again ------------------------------------------

def dropout_layers():
    torch.manual_seed(5)
    return torch.nn.ModuleList([
        torch.nn.Linear(64, 64, bias=False), links.FusedDropout(0.4),
        links.LinearAttentionRNN(64, 64, num_layers=2, n_heads=2,
                                 dropout=0.3)]).to(DEV)


def dropout_segment(module, x):
    a, d, rnn = module
    h = d(a(x)) * x
    return x + d(rnn(h)[0]) * h


def dropout_grads(module, y):
    # of y.square().sum(); a captured sum over many blocks clears memory in a
    # way that replays do not repeat
    return torch.autograd.grad(y, list(module.parameters()), 2 * y.detach())


@pytest.mark.parametrize('reentrant', [False, True])
def test_dropout_in_a_forgotten_segment(reentrant):
    x = rand(3, 50, 64)
    want_module, module = dropout_layers(), dropout_layers()
    want = dropout_segment(want_module, x)
    want_grads = dropout_grads(want_module, want)
    for p in module.parameters():
        p.grad = None
    x.requires_grad_()
    got = functions.forget(lambda t: dropout_segment(module, t), x,
                           use_reentrant=reentrant)
    got.backward(2 * got.detach())
    assert torch.equal(got, want)
    for p, w in zip(module.parameters(), want_grads):
        assert torch.equal(p.grad, w)
    assert module[1].rng_state.tolist() == want_module[1].rng_state.tolist()


@pytest.mark.parametrize('reentrant', [False, True])
def test_dropout_under_a_checkpoint_that_does_not_know_it(reentrant):
    module, x = dropout_layers(), rand(3, 50, 64).requires_grad_()
    y = checkpoint(lambda t: dropout_segment(module, t), x,
                   use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match='functions.forget'):
        y.sum().backward()


def test_a_forgotten_segment_in_a_graph():
    """Each replay draws new numbers, and its recomputation the same ones."""
    module, x = dropout_layers(), rand(3, 50, 64)

    def work():
        y = functions.forget(lambda t: dropout_segment(module, t), x,
                             preserve_rng_state=False)
        return [y.detach()] + list(dropout_grads(module, y))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    states = [b for n, b in module.named_buffers() if 'rng_state' in n]
    start = [b.clone() for b in states]
    replays = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        replays.append([g.clone() for g in got])
    for b, s in zip(states, start):
        b.copy_(s)
    for one in replays:
        y = dropout_segment(module, x)
        want = [y.detach()] + list(dropout_grads(module, y))
        for a, b in zip(one, want):
            assert torch.equal(a, b)
        del y, want
    assert not torch.equal(replays[0][0], replays[1][0])
