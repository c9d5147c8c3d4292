"""Corners of the sequence-model operators on a GPU, against values that are
known in 64 bits.

``E`` is half a step of fp32; the bounds beside the tests count roundings.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from chainermn_amd import functions
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
