"""Sequence-model kernels against their definitions in 64 bits.

Bounds are forward error bounds, not fits: a result rounded to type t is off
by u(t) = eps / 2 of its value, and a sum of n products in fp32 by at most
(n + a few) * 2^-24 of the sum of the products' magnitudes, which the tests
compute beside the result.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from chainermn_amd import functions, ops
    DEV = torch.device('cuda:0')
else:
    pytest.skip('needs ROCm GPU', allow_module_level=True)

TYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24


def u(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half a step below the normal numbers of a type."""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def near(got, want, bound):
    """|got - want| <= u |want| + bound, element by element."""
    assert got.shape == want.shape
    t = got.dtype
    off = (got.double() - want).abs()
    most = u(t) * want.abs() + bound + tiny(t)
    assert torch.isfinite(got.double()).all()
    bad = off > most
    assert not bad.any(), 'off by {:.3g} of the bound at {}'.format(
        float((off / most).max()), int(bad.sum()))


def rand(*shape, t=torch.float32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(t)


# ---- embedding -------------------------------------------------------------

def embed_case(ids, W, gy, scale, ignore):
    W = W.detach().requires_grad_()
    y = functions.embed_id(ids, W, ignore_label=ignore, scale=scale)
    dW, = torch.autograd.grad(y, W, gy)
    n = ids.reshape(-1).long()
    live = torch.ones_like(n, dtype=torch.bool) if ignore is None \
        else n != ignore
    at = torch.where(live, n, 0)
    Wd, g = W.detach().double(), gy.reshape(len(n), -1).double()
    want = torch.where(live[:, None], Wd[at] * scale, 0.0)
    near(y.detach().reshape(want.shape), want, E * want.abs())
    g = torch.where(live[:, None], g, 0.0)
    total = torch.zeros_like(Wd).index_add_(0, at, g) * scale
    size = torch.zeros_like(Wd).index_add_(0, at, g.abs()) * abs(scale)
    count = torch.bincount(at, minlength=len(Wd))[:, None]
    near(dW, total, (count + 2) * E * size)
    return y, dW


@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('vocab,dim,tokens', [
    (1, 1, 1), (1, 7, 33), (2, 8, 31), (64, 512, 1280), (5, 64, 4097),
    (1000, 33, 32), (3000, 100, 2049), (300000, 8, 1500), (257, 1030, 777),
    (1100000, 3, 5000), (700, 5, 70000), (5000, 40, 1), (2000, 513, 33)])
def test_embed(t, vocab, dim, tokens):
    g = torch.Generator(device=DEV).manual_seed(tokens)
    ids = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
    embed_case(ids, rand(vocab, dim, t=t), rand(tokens, dim, t=t, seed=1),
               1.0, None)
    ids[::3] = -1
    embed_case(ids, rand(vocab, dim, t=t), rand(tokens, dim, t=t, seed=1),
               2.5, -1)


@pytest.mark.parametrize('vocab', [40, 3000])
@pytest.mark.parametrize('tokens', [1, 32, 33, 64, 5000])
def test_embed_all_the_same_id(vocab, tokens):
    ids = torch.full((tokens,), 17, device=DEV, dtype=torch.int32)
    embed_case(ids, rand(vocab, 96), rand(tokens, 96, seed=1), -0.5, None)
    # and all ignored: the gradient is zero
    _, dW = embed_case(ids, rand(vocab, 96), rand(tokens, 96, seed=1), 1.0,
                       17)
    assert not dW.any()


def test_embed_runs_that_end_on_chunk_borders():
    ids = torch.arange(256, device=DEV).repeat_interleave(
        torch.tensor([1, 31, 32, 33, 64, 95, 96, 2] * 32, device=DEV))
    order = torch.randperm(len(ids), device=DEV)
    embed_case(ids[order], rand(256, 40), rand(len(ids), 40, seed=1), 1.0,
               None)


def test_embed_shapes_strides_and_empty():
    big = rand(50, 200, t=torch.bfloat16)
    ids = torch.randint(0, 50, (6, 5, 4), device=DEV).transpose(0, 2)
    for W in (big[:, :96], big[:, 3:50], big[::2][:, 8:24]):
        i = ids % len(W)
        gy = rand(*i.shape, W.shape[1], t=torch.bfloat16, seed=1)
        embed_case(i, W, gy, 1.0, None)
        embed_case(i, W, gy.transpose(0, 1).contiguous().transpose(0, 1),
                   1.0, 0)
    W = rand(9, 12).requires_grad_()
    y = functions.embed_id(ids[:0], W)
    assert y.shape == (0, 5, 6, 12)
    dW, = torch.autograd.grad(y, W, torch.zeros_like(y))
    assert dW.shape == W.shape and not dW.any()
    # an expanded gradient (stride zero)
    y = functions.embed_id(torch.tensor([1, 1, 3], device=DEV), W)
    dW, = torch.autograd.grad(y.sum(), W)
    assert torch.equal(dW[:, 0].cpu(), torch.tensor([0., 2, 0, 1] + [0] * 5))


def test_embed_bad_ids_are_seen_and_touch_nothing():
    W = rand(10, 24).requires_grad_()
    ids = torch.tensor([3, 10, -7, 2 ** 40, 4], device=DEV)
    y = functions.embed_id(ids, W, ignore_label=-1)
    bad = torch.isnan(y.detach()).all(1)
    assert bad.tolist() == [False, True, True, True, False]
    dW, = torch.autograd.grad(y, W, torch.ones_like(y))
    want = torch.zeros(10, 24, device=DEV)
    want[3] = want[4] = 1
    assert torch.equal(dW, want)


def test_embed_twice_is_the_same_bit_by_bit():
    ids = (torch.rand(20000, device=DEV) ** 4 * 500).long()
    W, gy = rand(500, 256).requires_grad_(), rand(20000, 256, seed=1)
    g = [torch.autograd.grad(functions.embed_id(ids, W), W, gy)[0]
         for _ in range(2)]
    assert torch.equal(*g)


# ---- dropout ---------------------------------------------------------------

def key_of(seed, call):
    return torch.tensor([seed, call], device=DEV)


@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('n', [1, 3, 8, 9, 2047, 2049, 100003])
def test_dropout(t, n):
    key = key_of(-2 ** 62 + 12345, 2 ** 40 + 7)
    x = rand(n + 1, t=t)[1:].requires_grad_()  # not aligned to 16 bytes
    gy = rand(n, t=t, seed=1)
    for ratio in (0.0, 0.3, 0.999):
        y = functions.dropout(x, key, ratio=ratio)
        dx, = torch.autograd.grad(y, x, gy)
        # the CPU's stream says which are kept
        kept = functions.dropout(torch.ones(n), key.cpu(), ratio=ratio) > 0
        kept = kept.to(DEV)
        assert torch.equal(y != 0, kept & (x != 0))
        for got, of in ((y.detach(), x.detach()), (dx, gy)):
            want = torch.where(kept, of.double() / (1 - ratio), 0.0)
            near(got, want, 2 * E * want.abs())


def test_dropout_past_32_bits_of_blocks():
    # blocks are counted in 64 bits: the tail of a stream of more than 2^32
    # elements is another than its beginning's
    n = 2 ** 32 + 64
    x = torch.ones(n, device=DEV, dtype=torch.bfloat16)
    key = key_of(5, 0)
    y = functions.dropout(x, key, ratio=0.5)
    head, tail = y[:64].float().cpu(), y[-64:].float().cpu()
    kept = functions.dropout(torch.ones(64), key.cpu(), ratio=0.5)
    assert torch.equal(head, kept)
    assert not torch.equal(head, tail)
    assert 0.49 < (y[-2 ** 20:] != 0).float().mean() < 0.51


def test_dropout_of_values_that_are_not_finite():
    x = torch.full((4096,), float('nan'), device=DEV)
    x[::2] = float('inf')
    y = functions.dropout(x, key_of(1, 2), ratio=0.5)
    kept = functions.dropout(torch.ones(4096), key_of(1, 2).cpu()).to(DEV) > 0
    assert (y[~kept] == 0).all() and not torch.isfinite(y[kept]).any()


def test_dropout_strides_and_empty():
    x = rand(60, 50).t().requires_grad_()
    y = functions.dropout(x, key_of(3, 4), ratio=0.4)
    kept = functions.dropout(torch.ones(50, 60), key_of(3, 4).cpu(),
                             ratio=0.4).to(DEV) > 0
    assert torch.equal(y != 0, kept)
    dx, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(dx != 0, kept)
    assert functions.dropout(x[:0], key_of(3, 4)).shape == (0, 60)


def test_dropout_replays_draw_new_numbers():
    state = key_of(42, 0)
    x = torch.ones(10000, device=DEV, requires_grad=True)

    def once():
        y = functions.dropout(x, ops.dropout_next_key(state), ratio=0.5)
        return y, torch.autograd.grad(y, x, torch.ones_like(y))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = once()
    first = int(state[1])
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = functions.dropout(x.detach(), key_of(42, first + i), ratio=0.5)
        assert torch.equal(y, want) and torch.equal(dx, want)
    assert int(state[1]) == first + 4


# ---- RMS norm --------------------------------------------------------------

def norm_reference(x, res, w, gy, gh, eps):
    """(y, h, dh, dw) in 64 bits, and a bound of each."""
    h = x.double() + (0 if res is None else res.double())
    d = h.shape[-1]
    w, gy = w.double(), gy.double()
    r = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh, g = h * r, gy * w
    m = (g * xh).mean(-1, keepdim=True)
    ma = (g * xh).abs().mean(-1, keepdim=True)
    dh = r * (g - xh * m) + (0 if gh is None else gh.double())
    size = r * (g.abs() + xh.abs() * ma) + (0 if gh is None
                                            else gh.double().abs())
    few = (d + 16) * E
    off = few * size
    dw = (gy * xh).sum(0)
    dw_off = (gy * xh).abs().sum(0) * ((len(h) + d + 16) * E)
    y = xh * w
    return (y, h, dh, dw), (few * y.abs(), 2 * E * h.abs(), off, dw_off)


@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('rows,dim', [
    (1, 1), (3, 3), (5, 64), (257, 100), (64, 1024), (1030, 512),
    (700, 1500), (33, 2050), (9, 4097), (5, 8192), (3, 16383), (2, 16384)])
@pytest.mark.parametrize('residual', [False, True])
def test_rms_norm(t, rows, dim, residual):
    x = rand(rows, dim, t=t).requires_grad_()
    w = (1 + 0.3 * rand(dim, seed=1)).to(t).requires_grad_()
    res = (3 * rand(rows, dim, t=t, seed=2)).requires_grad_() \
        if residual else None
    gy = rand(rows, dim, t=t, seed=3)
    gh = rand(rows, dim, t=t, seed=4) if residual else None
    with torch.no_grad():
        want, off = norm_reference(x, res, w, gy, gh, 1e-6)
    if residual:
        y, h = functions.rms_norm(x, w, residual=res)
        dx, dr, dw = torch.autograd.grad((y, h), (x, res, w), (gy, gh))
        near(h.detach(), want[1], off[1])
        assert torch.equal(dx, dr)
    else:
        y = functions.rms_norm(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), gy)
    near(y.detach(), want[0], off[0])
    near(dx, want[2], off[2])
    near(dw, want[3], off[3])


def test_rms_norm_mixed_weight_strides_and_shapes():
    t = torch.bfloat16
    # fp32 beside bf16, every second element of a vector
    w = (1 + 0.3 * rand(192, seed=1))[::2].detach().requires_grad_()
    big = rand(4, 7, 200, t=t)
    for x in (big[..., :96], big[..., 3:99], big.transpose(0, 1)[..., :96],
              rand(4, 96, 7, t=t).transpose(1, 2),
              rand(4, 1, 96, t=t).expand(4, 7, 96)):
        x = x.detach().requires_grad_()
        gy = rand(*x.shape, t=t, seed=2)
        y = functions.rms_norm(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), gy)
        with torch.no_grad():
            want, off = norm_reference(x.reshape(-1, 96), None, w,
                                       gy.reshape(-1, 96), None, 1e-6)
        assert dw.dtype == torch.float32
        near(y.detach().reshape(-1, 96), want[0], off[0])
        near(dx.reshape(-1, 96), want[2], off[2])
        near(dw, want[3], off[3])


def test_rms_norm_parts_of_the_graph():
    x, r = rand(6, 40).requires_grad_(), rand(6, 40, seed=1).requires_grad_()
    w = torch.ones(40, device=DEV, requires_grad=True)
    y, h = functions.rms_norm(x, w, residual=r)
    # only the sum is used
    dx, dr = torch.autograd.grad(h.sum(), (x, r), retain_graph=True)
    assert (dx == 1).all() and (dr == 1).all()
    # only the output
    dx, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    want, off = norm_reference(x.detach(), r.detach(), w.detach(),
                               torch.ones_like(y), None, 1e-6)
    near(dx, want[2], off[2])
    # no rows
    y = functions.rms_norm(x[:0], w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert not dx.any() and not dw.any()
    # rows of zeros: eps keeps them finite
    y = functions.rms_norm(torch.zeros(3, 40, device=DEV), w)
    assert not y.any()


@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('rows,dim,group', [
    (1, 16, 16), (64, 1024, 128), (64, 1024, None), (300, 96, 32),
    (5, 1001, None), (4, 1003, None), (3, 4096, 256), (7, 16384, None), (7, 8192, 64),
    (0, 64, 64)])
@pytest.mark.parametrize('residual', [False, True])
def test_rms_norm_fp8(t, rows, dim, group, residual):
    x, w = rand(rows, dim, t=t), (1 + 0.3 * rand(dim, seed=1)).to(t)
    if rows > 1:
        x[1] = 0
    res = rand(rows, dim, t=t, seed=2) if residual else None
    if residual and rows > 1:
        res[1] = 0
    out = ops.rms_norm_fp8(x, w, residual=res, group=group)
    q, scales = out[:2]
    h = x.double() + (0 if res is None else res.double())
    if residual:
        near(out[2], h, 2 * E * h.abs())
    y = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double()
    yg = y.view(rows, dim // (group or dim), group or dim)
    s = yg.abs().amax(-1) / 448
    s = torch.where(s > 0, s, 1.0)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    near(scales, s, (dim + 20) * E * s)
    back = (q.float().view(yg.shape).double() * scales[..., None].double())
    # half a step of e4m3: 2^-4 of the value, or 2^-10 of a step of one
    # below the normal numbers
    off = (back - yg).abs()
    assert (off <= yg.abs() * (2 ** -4 + (dim + 30) * E)
            + s[..., None] * 2.0 ** -10 * 1.001).all()


# ---- linear attention --------------------------------------------------------

def attention_reference(q, k, v, ld, s0, lengths, scale):
    """The recurrence in 64 bits, token by token, with autograd."""
    b, t, h = q.shape[:3]
    lam = ld.double().exp()[:, None, None]
    s = torch.zeros(b, h, q.shape[3], v.shape[3], device=q.device,
                    dtype=torch.float64) if s0 is None else s0
    out = []
    for i in range(t):
        live = torch.ones(b, device=q.device, dtype=torch.bool) \
            if lengths is None else i < lengths
        live = live[:, None, None, None]
        new = lam * s + k[:, i, :, :, None] * v[:, i, :, None]
        s = torch.where(live, new, s)
        o = (q[:, i, :, :, None] * s).sum(-2) * scale
        out.append(torch.where(live[..., 0], o, 0.0))
    return torch.stack(out, 1) if out else v, s


def attention_case(t, b, length, h, dk, dv, ragged, state, make=None):
    q, k = rand(b, length, h, dk, t=t), rand(b, length, h, dk, t=t, seed=1)
    v, go = rand(b, length, h, dv, t=t, seed=2), rand(b, length, h, dv, t=t,
                                                      seed=3)
    if make is not None:
        q, k, v, go = make(q), make(k), make(v), make(go)
    ld = torch.log1p(-2.0 ** -torch.linspace(1, 9, h, device=DEV))
    s0 = rand(b, h, dk, dv, seed=4) if state else None
    gs = rand(b, h, dk, dv, seed=5)
    lengths = None
    if ragged:
        lengths = torch.randint(0, length + 1, (b,), device=DEV)
        lengths[0] = 0
        lengths[-1] = length
    scale = dk ** -0.5
    ins = [x.detach().requires_grad_() for x in (q, k, v)]
    if state:
        ins.append(s0.requires_grad_())
    o, s = functions.linear_attention(
        *ins[:3], ld, initial_state=s0, lengths=lengths)
    got = [o, s] + list(torch.autograd.grad((o, s), ins, (go, gs)))

    def reference(fold):
        a = [fold(x.detach().double()).requires_grad_() for x in ins]
        o, s = attention_reference(*a[:3], ld, a[3] if state else None,
                                   lengths, scale)
        return [x.detach() for x in (o, s)] + list(torch.autograd.grad(
            (o, s), a, (fold(go.double()), fold(gs.double()))))

    want, size = reference(lambda x: x), reference(torch.abs)
    # A sum over the tokens and the head, its weights (a power of the decay,
    # a few steps off), and what the products of cut terms leave out: 2^-22
    # of each product for three terms of both sides, and 2^-14 where scores
    # and states are cut to 16 bits on their way to a 16-bit result.
    few = (length + dk + dv + 64) * E
    for i, (a, w, z) in enumerate(zip(got, want, size)):
        cutting = 0 if a.dtype == torch.float32 else 2.0 ** -14
        near(a.detach(), w, (few + cutting) * z)
    return got


@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('b,length,h,dk,dv', [
    (1, 1, 1, 1, 1), (2, 3, 2, 5, 7), (3, 31, 2, 16, 16), (2, 64, 3, 64, 64),
    (2, 65, 2, 64, 32), (1, 130, 2, 128, 128), (2, 200, 1, 100, 33),
    (3, 97, 2, 40, 128), (1, 300, 1, 24, 72)])
@pytest.mark.parametrize('ragged', [False, True])
def test_linear_attention(t, b, length, h, dk, dv, ragged):
    attention_case(t, b, length, h, dk, dv, ragged, state=ragged)


@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('ragged,state', [(False, True), (True, False),
                                          (True, True)])
def test_linear_attention_by_segments(t, ragged, state):
    # long and few: the length is split and joined
    attention_case(t, 3, 1111, 2, 64, 64, ragged, state)
    attention_case(t, 1, 1536, 1, 128, 96, ragged, state)


@pytest.mark.parametrize('t', TYPES)
def test_linear_attention_strides(t):
    attention_case(t, 2, 70, 3, 64, 64, False, True,
                   make=lambda x: x.transpose(1, 2).contiguous().transpose(
                       1, 2))
    # a slice of a wider row, not aligned to 16 bytes
    attention_case(t, 2, 70, 3, 30, 64, True, True, make=lambda x: torch.cat(
        (x[..., :1], x, x[..., :2]), -1)[..., 1:-2])
    # the last axis is not contiguous
    attention_case(t, 2, 20, 2, 16, 16, False, False,
                   make=lambda x: x.transpose(1, 3).contiguous().transpose(
                       1, 3))


def test_linear_attention_heads_of_one_projection():
    t = torch.bfloat16
    qkv = rand(2, 90, 3, 4, 64, t=t).requires_grad_()
    ld = torch.full((4,), -0.1, device=DEV)
    o, _ = functions.linear_attention(*qkv.unbind(2), ld)
    go = rand(*o.shape, t=t, seed=1)
    g, = torch.autograd.grad(o, qkv, go)
    parts = [x.detach().contiguous().requires_grad_() for x in qkv.unbind(2)]
    o2, _ = functions.linear_attention(*parts, ld)
    assert torch.equal(o, o2)
    assert torch.equal(g, torch.stack(torch.autograd.grad(o2, parts, go), 2))


def test_linear_attention_shared_and_broadcast_inputs():
    b, n, h, d = 2, 75, 4, 32
    q, k, v = (rand(b, n, x, d, seed=x) for x in (h, 1, 2))
    s0 = rand(1, h, d, d, seed=9)
    go = rand(b, n, h, d, seed=5)
    ld = torch.linspace(-1, -0.01, h, device=DEV)

    def run(expand):
        ins = [x.clone().requires_grad_() for x in (q, k, v, s0)]
        o, s = functions.linear_attention(*expand(*ins[:3]), ld,
                                          initial_state=ins[3].expand(
                                              b, -1, -1, -1))
        return [o.detach(), s.detach()] + list(torch.autograd.grad(
            (o, s), ins, (go, torch.ones_like(s))))

    # one head of k and two of v for four of q, as views and as copies
    views = run(lambda q, k, v: (q, k.expand(-1, -1, h, -1),
                                 v.unsqueeze(3).expand(-1, -1, -1, 2, -1)
                                 .flatten(2, 3)))
    copies = run(lambda q, k, v: (q, k.repeat(1, 1, h, 1),
                                  v.repeat_interleave(2, 2)))
    for x, y in zip(views, copies):
        # the same kernels on the same values; only torch's sums over the
        # shared heads may differ in their order, by 4 terms
        assert (x - y).abs().max() <= 8 * E * y.abs().max()
    # a gradient that is one value everywhere
    ins = [x.requires_grad_() for x in (q, k.repeat(1, 1, h, 1),
                                        v.repeat_interleave(2, 2))]
    o, _ = functions.linear_attention(*ins, ld)
    a = torch.autograd.grad(o.sum(), ins, retain_graph=True)
    for x, y in zip(a, torch.autograd.grad(o, ins, torch.ones_like(o))):
        assert torch.equal(x, y)


@pytest.mark.parametrize('length', [40, 600])
def test_linear_attention_some_of_the_gradients(length):
    ins = [rand(1, length, 2, 64, seed=i).requires_grad_() for i in range(3)]
    s0 = rand(1, 2, 64, 64, seed=4).requires_grad_()
    ld = torch.tensor([-0.3, -0.002], device=DEV)
    o, s = functions.linear_attention(*ins, ld, initial_state=s0)
    go = rand(*o.shape, seed=7)
    every = torch.autograd.grad(o, ins + [s0], go, retain_graph=True)
    for i, x in enumerate(ins + [s0]):
        g, = torch.autograd.grad(o, x, go, retain_graph=True)
        assert torch.equal(g, every[i])
    # a state that is not trained
    o, s = functions.linear_attention(*ins, ld, initial_state=s0.detach())
    for a, b in zip(torch.autograd.grad(o, ins, go), every):
        assert torch.equal(a, b)


def test_linear_attention_behind_the_end_nothing_is_read():
    for bad in (float('nan'), float('inf'), torch.finfo(torch.float32).min):
        q, k, v = (rand(2, 100, 2, 32, seed=i) for i in range(3))
        lengths = torch.tensor([37, 0], device=DEV, dtype=torch.int32)
        ld = torch.tensor([-0.2, 0.0], device=DEV)
        want, ws = functions.linear_attention(
            q[:, :37], k[:, :37], v[:, :37], ld, lengths=lengths)
        for x in (q, k, v):
            x[0, 37:] = bad
            x[1] = bad
        leaves = [x.requires_grad_() for x in (q, k, v)]
        o, s = functions.linear_attention(*leaves, ld, lengths=lengths)
        assert torch.equal(o[:, :37], want) and torch.equal(s, ws)
        assert not o[0, 37:].any() and not o[1].any() and not s[1].any()
        go = torch.full_like(o, bad)
        go[0, :37] = 1
        for g in torch.autograd.grad(o, leaves, go):
            assert torch.isfinite(g).all()
            assert not g[0, 37:].any() and not g[1].any()


def test_linear_attention_extreme_decays():
    q, k, v = (rand(2, 150, 3, 16, seed=i) for i in range(3))
    ld = torch.tensor([float('-inf'), 0.0, -1000.0], device=DEV)
    o, s = functions.linear_attention(q, k, v, ld, scale=1.0)
    # a decay of zero: every token sees itself alone
    alone = (q * k).double().sum(-1, keepdim=True) * v
    size = (q * k).double().abs().sum(-1, keepdim=True) * v.abs()
    for h in (0, 2):
        near(o[:, :, h], alone[:, :, h], 100 * E * size[:, :, h])
    last = k[:, -1, 1].double()
    assert torch.isfinite(s).all() and last.shape == (2, 16)
    near(s[:, 1], k[:, :, 1].double().transpose(1, 2) @ v[:, :, 1].double(),
         214 * E * (k[:, :, 1].double().abs().transpose(1, 2)
                    @ v[:, :, 1].double().abs()))


def test_linear_attention_no_tokens_and_no_sequences():
    ld = torch.full((2,), -0.5, device=DEV)
    s0 = rand(3, 2, 8, 4).requires_grad_()
    q, v = (torch.empty(3, 0, 2, d, device=DEV, requires_grad=True)
            for d in (8, 4))
    o, s = functions.linear_attention(q, q, v, ld, initial_state=s0)
    assert o.shape == (3, 0, 2, 4) and torch.equal(s, s0)
    g, = torch.autograd.grad(s, s0, torch.ones_like(s))
    assert (g == 1).all()
    o, s = functions.linear_attention(q[:0], q[:0], v[:0], ld)
    assert o.shape == (0, 0, 2, 4) and s.shape == (0, 2, 8, 4)


def test_linear_attention_only_the_state_is_used():
    q, k, v = (rand(2, 50, 2, 32, seed=i).requires_grad_() for i in range(3))
    ld = torch.full((2,), -0.1, device=DEV)
    _, s = functions.linear_attention(q, k, v, ld)
    gq, gk, gv = torch.autograd.grad(s.sum(), (q, k, v))
    w = torch.exp(ld * torch.arange(49, -1, -1, device=DEV)[:, None])
    assert not gq.any()
    near(gk, (w.double()[..., None] * v.sum(-1, keepdim=True).double())
         .expand_as(gk).detach(), 100 * E * v.detach().double().abs().sum(
             -1, keepdim=True).expand_as(gk))


@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('b,h,dk,dv', [
    (1, 1, 1, 1), (3, 2, 64, 64), (2, 3, 128, 128), (5, 1, 33, 7),
    (2, 2, 100, 68), (64, 16, 64, 64)])
def test_linear_attention_step(t, b, h, dk, dv):
    q, k, v = rand(b, h, dk, t=t), rand(b, h, dk, t=t, seed=1), rand(
        b, h, dv, t=t, seed=2)
    ld = torch.log1p(-2.0 ** -torch.linspace(1, 9, h, device=DEV))
    s = rand(b, h, dk, dv, seed=3)
    s0 = s.double()
    lam = ld.double().exp()[:, None, None]
    kv = k.double()[..., None] * v.double()[..., None, :]
    want, size = lam * s0 + kv, lam * s0.abs() + kv.abs()
    o = ops.linear_attention_step(q, k, v, s, ld)
    near(s, want, 8 * E * size)
    c = dk ** -0.5
    qd = q.double()[..., None]
    near(o, (qd * want).sum(-2) * c, (dk + 16) * E * (
        qd.abs() * size).sum(-2) * c)


def test_steps_follow_the_chunked_form():
    t, b, n, h, d = torch.float32, 2, 20, 3, 64
    q, k, v = (rand(b, n, h, d, t=t, seed=i) for i in range(3))
    ld = torch.tensor([-0.5, -0.05, -0.001], device=DEV)
    o, s = functions.linear_attention(q, k, v, ld)
    state = torch.zeros(b, h, d, d, device=DEV)
    steps = torch.stack([ops.linear_attention_step(
        q[:, i], k[:, i], v[:, i], state, ld) for i in range(n)], 1)
    size, ssize = attention_reference(
        q.double().abs(), k.double().abs(), v.double().abs(), ld, None, None,
        d ** -0.5)
    near(steps, o.double(), 400 * E * size)
    near(state, s.double(), 400 * E * ssize)


# ---- streams, graphs, devices, refusals -------------------------------------

def training_pass():
    """All four operators and their gradients, as one step uses them."""
    ids = (torch.arange(2 * 70, device=DEV).view(2, 70) * 7) % 50
    W = rand(50, 64).requires_grad_()
    w = (1 + 0.1 * rand(64, seed=1)).requires_grad_()
    ld = torch.tensor([-0.5, -0.01], device=DEV)
    lengths = torch.tensor([70, 41], device=DEV)
    key = key_of(7, 9)

    def once():
        x = functions.dropout(functions.embed_id(ids, W, scale=8.0), key, 0.1)
        y, h = functions.rms_norm(x, w, residual=x)
        heads = y.view(2, 70, 2, 32)
        o, s = functions.linear_attention(heads, heads, heads, ld,
                                          lengths=lengths)
        z = functions.rms_norm(o.reshape(2, 70, 64) + h, w)
        return [z, s] + list(torch.autograd.grad(
            (z, s), (W, w), (torch.ones_like(z), torch.ones_like(s))))

    return once


def test_operators_on_another_stream():
    once = training_pass()
    want = [x.detach() for x in once()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(10000000)
        got = once()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.detach(), b)


def test_operators_in_a_graph():
    once = training_pass()
    want = [x.detach() for x in once()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [x.detach() for x in once()]
    for _ in range(4):
        for x in got:
            x.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        eager = once()  # the program's own work between replays
        assert torch.equal(eager[0].detach(), want[0])


def test_second_derivatives_are_refused():
    x = rand(2, 3, 2, 8).requires_grad_()
    ld, w = torch.zeros(2, device=DEV), torch.ones(8, device=DEV)
    ids = torch.tensor([0, 1], device=DEV)
    for y in (functions.linear_attention(x, x, x, ld)[0],
              functions.rms_norm(x, w), functions.dropout(x, key_of(1, 2)),
              functions.embed_id(ids, x.view(12, 8))):
        with pytest.raises(RuntimeError, match='not differentiable'):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_what_is_updated_in_place_says_so():
    state = torch.zeros(2, 2, 8, 8, device=DEV)
    x = rand(2, 2, 8)
    before = state._version
    ops.linear_attention_step(x, x, x, state, torch.zeros(2, device=DEV))
    assert state._version > before
    key = key_of(1, 2)
    before = key._version
    ops.dropout_next_key(key, stream=3)
    assert key._version > before
    assert torch.equal(ops.dropout_next_key(key, stream=3).cpu(),
                       ops.dropout_next_key(torch.tensor([1, 3]), stream=3))


def test_rms_norm_fp8_of_what_is_not_finite():
    x = rand(3, 64)
    x[1, 5] = float('nan')
    q, scales = ops.rms_norm_fp8(x, torch.ones(64, device=DEV))
    assert torch.isnan(q[1].float()).all()
    assert torch.isfinite(q[::2].float()).all()
    w = torch.ones(64, device=DEV)
    w[7] = float('nan')
    q, scales = ops.rms_norm_fp8(rand(2, 64), w, group=32)
    bad = torch.isnan(q.float())
    assert bad[:, 7].all() and bad.sum() == 2 and torch.isfinite(scales).all()


def test_refusals_on_the_gpu():
    ld = torch.zeros(2, device=DEV)
    x = rand(2, 3, 2, 8)
    with pytest.raises(ValueError, match='not differentiable'):
        ops.rms_norm_fp8(rand(2, 8).requires_grad_(), torch.ones(
            8, device=DEV))
    double = x.double()
    with pytest.raises(RuntimeError, match='float32'):
        functions.linear_attention(double, double, double, ld)
    with pytest.raises(RuntimeError, match='GPU'):
        functions.linear_attention(x, x, x, ld.cpu())
    with pytest.raises(RuntimeError, match='lengths'):
        functions.linear_attention(x, x, x, ld, lengths=torch.ones(
            2, device=DEV))
    with pytest.raises(RuntimeError, match='contiguous'):
        ops.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], rand(
            2, 2, 8, 8).transpose(2, 3), ld)
    with pytest.raises(RuntimeError, match='float32'):
        functions.rms_norm(rand(4, 8).double(), torch.ones(
            8, device=DEV, dtype=torch.float64))
    with pytest.raises(RuntimeError, match='float32'):
        functions.embed_id(torch.zeros(3, device=DEV, dtype=torch.long),
                           rand(4, 8).double())
    with pytest.raises(RuntimeError, match='float32'):
        functions.dropout(rand(4).double(), key_of(1, 2))


# ---- what else a program does with them ------------------------------------

def test_outputs_changed_in_place():
    W, w = rand(20, 64).requires_grad_(), rand(64, seed=1).requires_grad_()
    x = rand(2, 3, 64, seed=2).requires_grad_()
    ids = torch.arange(6, device=DEV).view(2, 3)
    ld = torch.tensor([-0.1], device=DEV)

    def outputs():
        q = x.view(2, 3, 1, 64)
        return [functions.embed_id(ids, W), functions.rms_norm(x, w),
                functions.dropout(x, key_of(1, 2)),
                *functions.rms_norm(x, w, residual=x),
                *functions.linear_attention(q, q, q, ld)]

    for i in range(len(outputs())):
        y = outputs()[i]
        y *= 3
        z = outputs()[i] * 3
        assert torch.equal(y.detach(), z.detach())
        for a, b in zip(*(torch.autograd.grad(o.sum(), (W, w, x),
                                              allow_unused=True)
                          for o in (y, z))):
            assert (a is None) == (b is None)
            assert a is None or torch.equal(a, b)


@pytest.mark.parametrize('reentrant', [False, True])
def test_operators_under_checkpoint(reentrant):
    from torch.utils.checkpoint import checkpoint
    w = rand(64, seed=1).requires_grad_()
    x = rand(2, 40, 64, seed=2).requires_grad_()
    ld, key = torch.tensor([-0.1, -0.2], device=DEV), key_of(1, 2)

    def layer(x):
        y, h = functions.rms_norm(x, w, residual=x)
        q = y.view(2, 40, 2, 32)
        o, _ = functions.linear_attention(q, q, q, ld)
        return functions.dropout(o.flatten(2) + h, key)

    want = torch.autograd.grad(layer(x).sum(), (x, w))
    for p in (x, w):
        p.grad = None
    checkpoint(layer, x, use_reentrant=reentrant).sum().backward()
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])


def test_operators_in_inference_mode():
    with torch.inference_mode():
        W, w = rand(20, 64), rand(64, seed=1)
        state = torch.zeros(6, 1, 64, 64, device=DEV)
        ids = torch.arange(6, device=DEV)
        x = functions.dropout(functions.embed_id(ids, W), key_of(1, 2))
        y, h = functions.rms_norm(x, w, residual=x)
        q = y.view(6, 1, 64)
        ld = torch.tensor([-0.1], device=DEV)
        o = ops.linear_attention_step(q, q, q, state, ld)
        p, s = functions.linear_attention(q[:, None], q[:, None], q[:, None],
                                          ld)
        assert torch.allclose(o, p[:, 0], rtol=1e-5, atol=1e-5)
        assert torch.allclose(s, state, rtol=1e-5, atol=1e-5)
        ops.dropout_next_key(key_of(1, 2))


def test_two_graphs_at_once():
    """Neither shares its workspaces with the other one."""
    ld = torch.tensor([-0.01], device=DEV)
    inputs = [(torch.randint(0, 3000, (20000,), device=DEV),
               rand(20000, 64, seed=i), rand(1, 4096, 1, 64, seed=i))
              for i in range(2)]

    W0 = rand(3000, 64)

    def work(ids, gy, q):
        W, q = W0.detach().requires_grad_(), q.detach().requires_grad_()
        dW, = torch.autograd.grad(functions.embed_id(ids, W), W, gy)
        o, _ = functions.linear_attention(q, q, q, ld)
        dq, = torch.autograd.grad(o, q, torch.ones_like(o))
        return [dW, o.detach(), dq]

    want = [work(*x) for x in inputs]
    graphs, got = [], []
    for x in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(work(*x))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for outs in got:
            for o in outs:
                o.fill_(-1)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for p, q in zip(a, b):
                assert torch.equal(p, q)


def test_a_capture_beside_an_eager_graph_is_refused():
    W = rand(50, 64).requires_grad_()
    ids = torch.arange(9, device=DEV)
    gy = rand(9, 64)
    eager = functions.embed_id(ids, W)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='eager graph'):
        with torch.cuda.graph(graph):
            torch.autograd.grad(functions.embed_id(ids, W), W, gy)
    # a forward pass alone can be captured, and all of it without the other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = functions.embed_id(ids, W).detach()
    graph.replay()
    assert torch.equal(y, eager.detach())
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dW, = torch.autograd.grad(functions.embed_id(ids, W), W, gy)
    graph.replay()
    assert torch.equal(dW[:9], gy) and not dW[9:].any()


def test_dropout_from_any_address():
    for t in TYPES:
        x = rand(5001, t=t)
        for first in (1, 2, 3, 8):
            y = x[first:]
            assert torch.equal(functions.dropout(y, key_of(3, 4)),
                               functions.dropout(y.clone(), key_of(3, 4)))


def test_linear_attention_of_views_of_lengths_and_decays():
    x = rand(2, 40, 2, 16)
    lengths = torch.tensor([40, 9, 7, 9], device=DEV)[::2]
    ld = torch.tensor([-0.1, 0.0, -0.3], device=DEV)[::2]
    a = functions.linear_attention(x, x, x, ld, lengths=lengths)
    b = functions.linear_attention(x, x, x, ld.clone(),
                                   lengths=lengths.clone())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # lengths outside of the batch's
    a = functions.linear_attention(x, x, x, ld, lengths=torch.tensor(
        [99, -5], device=DEV, dtype=torch.int32))
    b = functions.linear_attention(x, x, x, ld, lengths=torch.tensor(
        [40, 0], device=DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_too_many_for_a_launch_is_refused():
    ld = torch.zeros(1, device=DEV)
    x = torch.zeros(2 ** 21, 1, 1, 1, device=DEV)
    with pytest.raises(RuntimeError, match='2.21'):
        functions.linear_attention(x, x, x, ld)
    x = torch.zeros(2 ** 24, 1, 1, device=DEV)
    with pytest.raises(RuntimeError, match='threads'):
        ops.linear_attention_step(x, x, x, x[..., None].contiguous(), ld)
    # rows of 256 elements have 64 lanes each
    ids = torch.zeros(2 ** 26, device=DEV, dtype=torch.int32)
    with pytest.raises(RuntimeError, match='threads'):
        functions.embed_id(ids, torch.zeros(1, 256, device=DEV))


# ---- more than 2^31 elements -----------------------------------------------

def test_embed_past_32_bits():
    t, dim = torch.bfloat16, 520
    vocab = 2 ** 22
    W = torch.zeros(vocab, dim, device=DEV, dtype=t)
    W[-8:] = rand(8, dim, t=t)
    W.requires_grad_()
    ids = torch.tensor([vocab - 1, 5, vocab - 8, vocab - 1], device=DEV)
    gy = rand(4, dim, t=t, seed=1)
    y = functions.embed_id(ids, W)
    assert torch.equal(y.detach(), W.detach()[ids])
    dW, = torch.autograd.grad(y, W, gy)
    near(dW[-1], gy[0].double() + gy[3].double(),
         4 * E * (gy[0].abs() + gy[3].abs()).double())
    assert torch.equal(dW[-8], gy[2]) and torch.equal(dW[5], gy[1])
    dW[-1] = dW[-8] = dW[5] = 0
    assert not dW.view(torch.int64).any()
    del W, dW, y
    ids = torch.arange(vocab, device=DEV) % 50
    ids[-1] = 50
    W = rand(1100, dim, t=t).requires_grad_()
    y = functions.embed_id(ids, W)
    assert torch.equal(y.detach()[-60:], W.detach()[ids[-60:]])
    gy = torch.zeros_like(y.detach())
    gy[-60:] = rand(60, dim, t=t, seed=1)
    dW, = torch.autograd.grad(y, W, gy)
    assert torch.equal(dW[50], gy[-1])
    want = torch.zeros(1100, dim, device=DEV, dtype=torch.float64)
    want.index_add_(0, ids[-60:], gy[-60:].double())
    # at most two of the terms of a sum are not zero
    near(dW, want, 4 * E * torch.zeros_like(want).index_add_(
        0, ids[-60:], gy[-60:].double().abs()))


def test_rms_norm_past_32_bits():
    t, rows, dim = torch.bfloat16, 2 ** 21 + 3, 1030
    x = torch.empty(rows, dim, device=DEV, dtype=t)
    x.copy_(rand(dim, t=t))
    w = rand(dim, seed=1)
    few = x[:7].clone().requires_grad_()
    x.requires_grad_()
    y = functions.rms_norm(x, w)
    want = functions.rms_norm(few, w)
    assert torch.equal(y.detach()[-7:], want.detach())
    dx, = torch.autograd.grad(y, x, y.detach())
    dw, = torch.autograd.grad(want, few, want.detach())
    assert torch.equal(dx[-7:], dw)
    del dx, y
    with torch.no_grad():
        q, scales = ops.rms_norm_fp8(x, w)
        a, b = ops.rms_norm_fp8(few, w)
    assert torch.equal(q[-7:].view(torch.int8), a.view(torch.int8))
    assert torch.equal(scales[-7:], b)


@pytest.mark.parametrize('strides', [
    (2 ** 31 + 64, 128, 64, 1), (2 ** 31 + 65, 128, 64, 1),
    (128, 2 ** 27 + 8, 64, 1)])
def test_linear_attention_strides_past_32_bits(strides):
    shape = (2, 17, 2, 64)
    space = torch.empty(1 + sum(
        (n - 1) * s for n, s in zip(shape, strides)), device=DEV,
        dtype=torch.bfloat16)
    q = space.as_strided(shape, strides)
    q.copy_(rand(*shape, t=torch.bfloat16))
    ld = torch.tensor([-0.1, -0.2], device=DEV)
    c = q.contiguous().requires_grad_()
    q.requires_grad_()
    go = rand(*shape, t=torch.bfloat16, seed=1)
    for a, b in zip(*((lambda o, s, x: [o.detach(), s.detach()] + list(
            torch.autograd.grad(o, x, go)))(
                *functions.linear_attention(x, x, x, ld), x)
            for x in (q, c))):
        assert torch.equal(a.contiguous(), b)


def test_linear_attention_output_past_32_bits():
    b, length, d, few = 4100, 4100, 128, 300  # few enough, and one segment
    x = torch.zeros(b, length, 1, d, device=DEV, dtype=torch.bfloat16)
    x[-few:] = rand(few, length, 1, d, t=torch.bfloat16)
    ld = torch.tensor([-0.02], device=DEV)
    c = x[-few:].clone().requires_grad_()
    x.requires_grad_()
    o, s = functions.linear_attention(x, x, x, ld)
    p, r = functions.linear_attention(c, c, c, ld)
    assert torch.equal(o.detach()[-few:], p.detach())
    assert torch.equal(s.detach()[-few:], r.detach())
    g, = torch.autograd.grad(o, x, o.detach())
    h, = torch.autograd.grad(p, c, p.detach())
    assert torch.equal(g[-few:], h)


def test_step_of_states_past_32_bits():
    b, d, few = 2 ** 17 + 3, 128, 5
    q = rand(b, 1, d)
    state = torch.zeros(b, 1, d, d, device=DEV)
    state[-few:] = rand(few, 1, d, d, seed=1)
    last = state[-few:].clone()
    ld = torch.tensor([-0.02], device=DEV)
    o = ops.linear_attention_step(q, q, q, state, ld)
    p = ops.linear_attention_step(q[-few:], q[-few:], q[-few:], last, ld)
    assert torch.equal(o[-few:], p) and torch.equal(state[-few:], last)


# ---- several rows of a norm in a wave ---------------------------------------

@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('rows,dim', [
    (1, 2), (70000, 16), (300, 17), (1000, 32), (4099, 48), (515, 128),
    (129, 255), (100, 256), (65537, 1)])
@pytest.mark.parametrize('residual', [False, True])
def test_rms_norm_of_short_rows(t, rows, dim, residual):
    test_rms_norm(t, rows, dim, residual)


@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('rows,dim,group', [
    (300, 16, 16), (300, 256, 256), (1000, 512, 256), (77, 64, None),
    (77, 48, 16), (513, 33, None), (129, 128, 128), (70000, 5, None)])
def test_rms_norm_fp8_of_short_rows(t, rows, dim, group):
    test_rms_norm_fp8(t, rows, dim, group, rows % 2 == 1)


# ---- rows of attention that are no whole vectors -----------------------------

@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('b,length,h,dk,dv', [
    (2, 70, 3, 102, 96), (2, 33, 2, 2, 126), (1, 65, 5, 31, 117),
    (3, 40, 1, 82, 20), (2, 37, 4, 7, 5), (1, 64, 1, 127, 1),
    (2, 290, 1, 58, 63)])
@pytest.mark.parametrize('ragged', [False, True])
def test_linear_attention_of_odd_heads(t, b, length, h, dk, dv, ragged):
    attention_case(t, b, length, h, dk, dv, ragged, state=not ragged)


@pytest.mark.parametrize('t', TYPES)
def test_linear_attention_of_odd_strides(t):
    for first, behind in ((1, 0), (1, 1), (2, 1), (0, 3), (3, 1)):
        for d in (64, 33, 30):
            attention_case(
                t, 2, 70, 2, d, d, True, False,
                make=lambda x: torch.nn.functional.pad(
                    x, (first, behind))[..., first:first + x.shape[-1]])


@pytest.mark.parametrize('t', TYPES)
@pytest.mark.parametrize('d', [1, 7, 31, 63, 66, 127])
def test_linear_attention_of_odd_heads_reads_nothing_behind_the_end(t, d):
    """The first word behind a row can hold the next row's first element."""
    ld = torch.tensor([-0.2], device=DEV)
    q, k, v = (rand(3, 70, 1, d, t=t, seed=i) for i in range(3))
    lengths = torch.tensor([37, 0, 64], device=DEV)
    clean, dirty = [], []
    for x in (q, k, v):
        x, y = x.clone(), x.clone()
        for b in range(3):
            x[b, lengths[b]:] = 0
            y[b, lengths[b]:] = float('nan')
        clean.append(x.requires_grad_())
        dirty.append(y.requires_grad_())
    go = rand(3, 70, 1, d, t=t, seed=5)
    for a, b in zip(*(
            (lambda o, s, xs: [o.detach(), s.detach()] + list(
                torch.autograd.grad((o, s), xs, (go, torch.ones_like(s)))))(
                *functions.linear_attention(*xs, ld, lengths=lengths), xs)
            for xs in (clean, dirty))):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_linear_attention_of_tokens_on_top_of_each_other():
    x = rand(2, 200, 2, 16, seed=1)
    for strides in ((32, 0, 16, 1), (6400, 16, 8, 1), (0, 32, 16, 1)):
        y = x.as_strided((2, 90, 2, 16), strides)
        ld = torch.tensor([-0.2, -0.1], device=DEV)
        a = functions.linear_attention(y, y, y, ld)
        b = functions.linear_attention(*[y.contiguous()] * 3, ld)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_too_many_heads_are_refused():
    x = torch.zeros(1, 1, 2 ** 17, 1, device=DEV)
    with pytest.raises(RuntimeError, match='2.17'):
        functions.linear_attention(x, x, x, torch.zeros(2 ** 17, device=DEV))
