"""The sequence-model operators, case by case: what is timed and what it is held to.

Four operators of the training and serving path of a recurrent language model:

* ``embed``  embedding lookup with scaling, and its gradient by sorted tokens
* ``drop``   dropout from a counter-based generator (no mask is stored)
* ``norm``   root-mean-square norm with the residual's addition, trained, or
             with an output in 8 bits (e4m3) with scales
* ``attn``   linear attention with a decay for each head: chunked over a
             prompt or a training batch, recurrent for single tokens

``run`` computes a case with the framework's operators where ``own`` is true,
and with elementary torch operations in 32 bits where it is false.
"""

import math

import torch

own = False

DEV = 'cuda'
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16,
         'fp16': torch.float16}
E4M3_MAX = 448.0


def listed():
    return [
        # The seq2seq example's training batch: 64 sentences of 20 tokens,
        # a vocabulary of 64, so every row of the gradient is a long sum.
        dict(name='embed_example', op='embed', dtype='fp32', vocab=64,
             dim=512, tokens=1280, ignored=0.0, scale=1.0),
        # The seq2seq benchmark: 512 sentences of 64 tokens, 32000 x 1024.
        dict(name='embed_bench', op='embed', dtype='fp32', vocab=32000,
             dim=1024, tokens=32768, ignored=0.0, scale=1.0),
        # A padded batch in bf16 with odd sizes, scaled by sqrt(dim).
        dict(name='embed_padded', op='embed', dtype='bf16', vocab=50021,
             dim=760, tokens=30011, ignored=0.25, scale=27.5),
        # Dropout after the example's embedding: little work, launch-bound.
        dict(name='drop_example', op='drop', dtype='fp32', numel=655360,
             ratio=0.2),
        # Dropout over the widest activation of a long bf16 batch.
        dict(name='drop_large', op='drop', dtype='bf16', numel=134217728,
             ratio=0.1),
        # One norm with the residual of the benchmark's batch, trained.
        dict(name='norm_bench', op='norm', dtype='bf16', rows=32768,
             dim=1024, residual=True, group=-1),
        # A trained norm without residual, fp32, odd sizes.
        dict(name='norm_odd', op='norm', dtype='fp32', rows=5003, dim=1500,
             residual=False, group=-1),
        # Single tokens of 64 sequences on their way to an 8-bit product.
        dict(name='norm_serve_fp8', op='norm', dtype='bf16', rows=64,
             dim=1024, residual=True, group=128),
        # One generated token for each of 64 sentences, 16 heads of 64.
        dict(name='attn_token', op='step', dtype='bf16', batch=64, heads=16,
             dk=64, dv=64),
        # The benchmark's batch, fp32, 16 heads of 64, sentences of their own
        # lengths, forward and backward.
        dict(name='attn_bench', op='attn', dtype='fp32', batch=512, length=64,
             heads=16, dk=64, dv=64, train=True, ragged=True, state=False),
        # Few long sequences, trained: the length has to be split.
        dict(name='attn_long', op='attn', dtype='bf16', batch=2,
             length=16384, heads=8, dk=128, dv=128, train=True, ragged=False,
             state=True),
        # The prompt of one sequence, read before generation, odd length.
        dict(name='attn_prompt', op='attn', dtype='bf16', batch=1,
             length=5001, heads=16, dk=128, dv=128, train=False,
             ragged=False, state=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['embed', 'drop', 'norm', 'norm', 'step', 'attn',
                     'attn'])
    dtype = rng.choice(['fp32', 'bf16', 'bf16', 'fp16'])
    if op == 'embed':
        return dict(op=op, dtype=dtype, vocab=_log(rng, 50, 60000),
                    dim=_log(rng, 16, 1024), tokens=_log(rng, 64, 32768),
                    ignored=rng.choice([0.0, round(rng.uniform(0, 0.6), 2)]),
                    scale=rng.choice([1.0, round(rng.uniform(0.5, 30), 2)]))
    if op == 'drop':
        return dict(op=op, dtype=dtype, numel=_log(rng, 1000, 60000000),
                    ratio=round(rng.uniform(0.02, 0.7), 3))
    if op == 'norm':
        rows = _log(rng, 1, 32768)
        dim = _log(rng, 16, min(8192, 33554432 // rows))
        group = rng.choice([-1, -1, 0, 64])
        if group == 64:
            dim = max(64, dim // 64 * 64)
        return dict(op=op, dtype=dtype, rows=rows, dim=dim,
                    residual=rng.random() < 0.6, group=group)
    if op == 'step':
        return dict(op=op, dtype=dtype, batch=_log(rng, 1, 256),
                    heads=rng.randint(1, 16), dk=_log(rng, 8, 128),
                    dv=_log(rng, 8, 128))
    heads = rng.randint(1, 16)
    dk, dv = _log(rng, 16, 128), _log(rng, 16, 128)
    length = _log(rng, 1, 16384)
    most = 33554432 // (length * heads * 128)
    return dict(op='attn', dtype=dtype,
                batch=_log(rng, 1, max(1, min(512, most))), length=length,
                heads=heads, dk=dk, dv=dv, train=rng.random() < 0.6,
                ragged=rng.random() < 0.4, state=rng.random() < 0.5)


def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    op = case['op']
    if op == 'embed':
        n, d, v = case['tokens'], case['dim'], case['vocab']
        rows = min(n, v)  # rows of the table that the lookup can touch
        return dict(bytes=size * (rows * d + n * d + n * d + v * d) + 16 * n,
                    flops=2.0 * n * d)
    if op == 'drop':
        n = case['numel']
        return dict(bytes=4.0 * size * n, flops=2.0 * n)
    if op == 'norm':
        n, d = case['rows'] * case['dim'], case['dim']
        ins = 2 if case['residual'] else 1
        if case['group'] >= 0:
            groups = case['rows'] * (d // case['group'] if case['group']
                                     else 1)
            return dict(bytes=size * n * (2 * ins - 1) + n + 4 * groups
                        + size * d, flops=6.0 * n)
        # forward: the inputs, y and the sum; backward: y's gradient, the
        # sum (and its gradient), one input gradient
        return dict(bytes=size * n * (2 * ins + 2 + ins) + 3 * size * d,
                    flops=14.0 * n)
    if op == 'step':
        s = case['batch'] * case['heads']
        dk, dv = case['dk'], case['dv']
        return dict(bytes=8.0 * s * dk * dv + size * s * (2 * dk + 2 * dv),
                    flops=6.0 * s * dk * dv)
    s = case['batch'] * case['heads']
    n, dk, dv = s * case['length'], case['dk'], case['dv']
    b = size * n * (2 * dk + 2 * dv) + 4.0 * s * dk * dv * (
        2 if case['state'] else 1)
    f = 6.0 * n * dk * dv
    if case['train']:
        b += size * n * (4 * dk + 3 * dv) + 4.0 * s * dk * dv * (
            3 if case['state'] else 0)
        f += 14.0 * n * dk * dv
    return dict(bytes=b, flops=f)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    t = TYPES[case['dtype']]
    op = case['op']

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV).to(t)

    st = dict(case=case)
    if op == 'embed':
        n, d, v = case['tokens'], case['dim'], case['vocab']
        # words come by their rank: log-uniform, as in running text
        u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
        ids = ((v + 1.0) ** u - 1.0).long().clamp_(0, v - 1)
        st['ignore'] = None
        if case['ignored']:
            pad = torch.rand(n, generator=g, device=DEV) < case['ignored']
            ids = torch.where(pad, torch.full_like(ids, -1), ids)
            st['ignore'] = -1
        st.update(ids=ids, W=randn(v, d).requires_grad_(),
                  gy=randn(n, d))
    elif op == 'drop':
        n = case['numel']
        st.update(x=randn(n).requires_grad_(), gy=randn(n),
                  key=torch.randint(-2 ** 62, 2 ** 62, (2,), generator=g,
                                    device=DEV))
    elif op == 'norm':
        n, d = case['rows'], case['dim']
        st.update(x=randn(n, d), weight=(1 + 0.2 * randn(d)).to(t),
                  residual=randn(n, d) * 2 if case['residual'] else None)
        if case['group'] < 0:
            st.update(gy=randn(n, d),
                      gh=randn(n, d) if case['residual'] else None)
            for k in ('x', 'weight', 'residual'):
                if st[k] is not None:
                    st[k].requires_grad_()
    else:
        b, h, dk, dv = case['batch'], case['heads'], case['dk'], case['dv']
        # heads from a short memory (4 tokens) to a long one (4096)
        rate = torch.linspace(2, 12, h, device=DEV, dtype=torch.float64)
        st.update(log_decay=torch.log1p(-2.0 ** -rate).float(),
                  scale=dk ** -0.5)
        shape = (b, h) if op == 'step' else (b, case['length'], h)
        st.update(q=randn(*shape, dk), k=randn(*shape, dk),
                  v=randn(*shape, dv))
        state = torch.randn(b, h, dk, dv, generator=g, device=DEV)
        if op == 'step':
            st['state'] = state
        else:
            st['state'] = state if case['state'] else None
            st['lengths'] = torch.randint(
                0, case['length'] + 1, (b,), generator=g,
                device=DEV) if case['ragged'] else None
            if case['train']:
                st['go'] = randn(*shape, dv)
                st['gs'] = torch.randn(b, h, dk, dv, generator=g,
                                       device=DEV) if case['state'] else None
                for k in ('q', 'k', 'v', 'state'):
                    if st[k] is not None:
                        st[k].requires_grad_()
    return st


def run(state):
    return _RUN[own][state['case']['op']](state)


# ---- the framework's operators -------------------------------------------

def _own_embed(st):
    from chainermn_amd import functions
    y = functions.embed_id(st['ids'], st['W'], scale=st['case']['scale'],
                           ignore_label=st['ignore'])
    return y.detach(), torch.autograd.grad(y, st['W'], st['gy'])[0]


def _own_drop(st):
    from chainermn_amd import functions
    y = functions.dropout(st['x'], st['key'], ratio=st['case']['ratio'])
    return y.detach(), torch.autograd.grad(y, st['x'], st['gy'])[0]


def _own_norm(st):
    from chainermn_amd import functions, ops
    case, x, w, res = st['case'], st['x'], st['weight'], st['residual']
    if case['group'] >= 0:
        return ops.rms_norm_fp8(x, w, residual=res, eps=1e-6,
                                group=case['group'] or None)
    if res is None:
        y = functions.rms_norm(x, w, eps=1e-6)
        return (y.detach(),) + torch.autograd.grad(y, (x, w), st['gy'])
    y, h = functions.rms_norm(x, w, residual=res, eps=1e-6)
    return (y.detach(), h.detach()) + torch.autograd.grad(
        (y, h), (x, res, w), (st['gy'], st['gh']))


def _own_step(st):
    from chainermn_amd import ops
    o = ops.linear_attention_step(st['q'], st['k'], st['v'], st['state'],
                                  st['log_decay'], scale=st['scale'])
    return o, st['state']


def _own_attn(st):
    from chainermn_amd import functions
    o, s = functions.linear_attention(
        st['q'], st['k'], st['v'], st['log_decay'],
        initial_state=st['state'], lengths=st['lengths'], scale=st['scale'])
    if not st['case']['train']:
        return o, s
    if st['state'] is None:
        return (o.detach(),) + torch.autograd.grad(
            o, (st['q'], st['k'], st['v']), st['go'])
    return (o.detach(), s.detach()) + torch.autograd.grad(
        (o, s), (st['q'], st['k'], st['v'], st['state']),
        (st['go'], st['gs']))


# ---- the plain forms -------------------------------------------------------

def _plain_embed(st):
    ids, gy, c = st['ids'], st['gy'], st['case']
    W = st['W'].detach()
    live = ids >= 0
    at = ids.clamp(min=0)
    y = W[at].float() * c['scale']
    y = torch.where(live[:, None], y, 0.0).to(W.dtype)
    g = torch.where(live[:, None], gy.float() * c['scale'], 0.0)
    dW = torch.zeros(W.shape, device=W.device).index_add_(0, at, g)
    return y, dW.to(W.dtype)


def _philox_words(key, n):
    """Philox4x32-10 (Salmon et al., 2011): words 0..n-1 of the stream whose
    key is key[0] and whose upper counter half is key[1]."""
    m = 0xffffffff
    blk = torch.arange((n + 3) // 4, device=key.device)
    c0, c1 = blk & m, blk >> 32
    c2 = (key[1] & m).expand_as(blk)
    c3 = ((key[1] >> 32) & m).expand_as(blk)
    k0, k1 = key[0] & m, (key[0] >> 32) & m

    def mul(a, c):  # 32 x 32 -> high and low words, in 63 bits
        low, high = a * (c & 0xffff), a * (c >> 16)
        return (high + (low >> 16)) >> 16, (low + (high << 16)) & m

    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


def _plain_drop(st):
    r = st['case']['ratio']
    x = st['x'].detach()
    keep = _philox_words(st['key'], x.numel()) >= int(round(r * 2.0 ** 32))
    s = 1.0 / (1.0 - r)
    return (torch.where(keep, x.float() * s, 0.0).to(x.dtype),
            torch.where(keep, st['gy'].float() * s, 0.0).to(x.dtype))


def _plain_norm(st):
    case, t = st['case'], st['x'].dtype
    x, w = st['x'].detach().float(), st['weight'].detach().float()
    res = st['residual']
    h = x if res is None else x + res.detach().float()
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6)
    xhat = h * rstd
    y = xhat * w
    if case['group'] >= 0:
        n, d = h.shape
        yg = y.view(n, -1, case['group'] or d)
        amax = yg.abs().amax(-1, keepdim=True)
        scale = torch.where(amax > 0, amax / E4M3_MAX, 1.0)
        q = (yg / scale).clamp(-E4M3_MAX, E4M3_MAX)
        out = (q.to(torch.float8_e4m3fn).view(n, d), scale.squeeze(-1))
        return out if res is None else out + (h.to(t),)
    gy = st['gy'].float()
    g = gy * w
    dh = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    dw = (gy * xhat).sum(0).to(t)
    if res is None:
        return y.to(t), dh.to(t), dw
    dh = (dh + st['gh'].float()).to(t)
    return y.to(t), h.to(t), dh, dh, dw


def _plain_step(st):
    s, q = st['state'], st['q'].float()
    lam = torch.exp(st['log_decay'])[None, :, None, None]
    s.mul_(lam).add_(st['k'].float()[..., None] * st['v'].float()[..., None, :])
    o = (q[..., None] * s).sum(-2) * st['scale']
    return o.to(st['q'].dtype), s


def _plain_chunked(q, k, v, ld, s0, lengths, scale, C=64):
    """Linear attention over [B, H, T, D] in fp32 by chunks of C tokens: the
    scores inside a chunk, and the state that comes into it."""
    b, h, t, dk = q.shape
    dv = v.shape[-1]
    ld = ld.double()
    pos = torch.arange(t, device=q.device)
    n = torch.full((b,), t, device=q.device) if lengths is None else lengths
    live = (pos[None] < n[:, None])[:, None, :, None]
    q, k, v = (torch.where(live, x, 0.0) for x in (q, k, v))
    left = (n[:, None] - 1 - pos[None]).clamp(min=0)[:, None]  # [b, 1, t]
    w = torch.exp(left * ld[:, None]).float()[..., None]
    fin = k.transpose(-1, -2) @ (v * w)
    if s0 is not None:
        fin = fin + s0 * torch.exp(n[:, None] * ld).float()[..., None, None]
    nc = (t + C - 1) // C
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, nc * C - t))
               .view(b, h, nc, C, -1) for x in (q, k, v))
    i = torch.arange(C, device=q.device)
    c = torch.arange(nc, device=q.device)
    gap = i[:, None] - i[None]
    inside = torch.where(gap >= 0, torch.exp(
        gap.clamp(min=0) * ld[:, None, None]), 0.0).float()[:, None]
    o = ((q @ k.transpose(-1, -2)) * inside) @ v
    if nc > 1 or s0 is not None:
        u = k.transpose(-1, -2) @ (
            v * torch.exp((C - 1 - i) * ld[:, None]).float()[:, None, :, None])
        far = c[:, None] - 1 - c[None]
        join = torch.where(far >= 0, torch.exp(
            C * far.clamp(min=0) * ld[:, None, None]), 0.0).float()
        s = (join @ u.reshape(b, h, nc, dk * dv)).view(b, h, nc, dk, dv)
        if s0 is not None:
            s = s + s0[:, :, None] * torch.exp(
                C * c * ld[:, None]).float()[..., None, None]
        o = o + (q @ s) * torch.exp(
            (i + 1) * ld[:, None]).float()[:, None, :, None]
    o = o.reshape(b, h, nc * C, dv)[:, :, :t] * scale
    return torch.where(live, o, 0.0), fin


def _plain_attn(st):
    case, t = st['case'], st['q'].dtype
    train = case['train']
    q, k, v = (st[x].detach().float().transpose(1, 2).requires_grad_(train)
               for x in 'qkv')
    s0 = st['state']
    if s0 is not None:
        s0 = s0.detach().requires_grad_(train)
    o, s = _plain_chunked(q, k, v, st['log_decay'], s0, st['lengths'],
                          st['scale'])
    out = o.detach().transpose(1, 2).to(t).contiguous()
    if not train:
        return out, s
    go = st['go'].float().transpose(1, 2)
    if s0 is None:
        g = torch.autograd.grad(o, (q, k, v), go)
        return (out,) + tuple(x.transpose(1, 2).to(t).contiguous() for x in g)
    g = torch.autograd.grad((o, s), (q, k, v, s0), (go, st['gs']))
    return (out, s.detach()) + tuple(
        x.transpose(1, 2).to(t).contiguous() for x in g[:3]) + (g[3],)


_RUN = {
    True: dict(embed=_own_embed, drop=_own_drop, norm=_own_norm,
               step=_own_step, attn=_own_attn),
    False: dict(embed=_plain_embed, drop=_plain_drop, norm=_plain_norm,
                step=_plain_step, attn=_plain_attn),
}


# ---- the definitions, in 64 bits -------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    st = {k: v.detach() if isinstance(v, torch.Tensor) else v
          for k, v in st.items()}
    with torch.no_grad():
        return _EXACT[case['op']](st)


def _exact_embed(st):
    c, W = st['case'], st['W'].double()
    table = torch.cat((W, W.new_zeros(1, W.shape[1])))  # row of the ignored
    ids = torch.where(st['ids'] < 0, c['vocab'], st['ids'])
    grad = torch.zeros_like(table)
    grad.index_put_((ids,), st['gy'].double(), accumulate=True)
    return table[ids] * c['scale'], grad[:-1] * c['scale']


def _exact_drop(st):
    c, n = st['case'], st['case']['numel']
    seed, call = (int(x) % 2 ** 64 for x in st['key'].tolist())
    full = 2 ** 32

    def words(lo, hi):  # the counters' words as float64, whole and exact
        return [x.double() for x in (lo, hi)]

    def product(a, x):
        # a * x for whole x < 2^32 held in float64: x is cut at 2^11 so that
        # every part stays below 2^53
        top, low = torch.floor(x / 2048), torch.remainder(x, 2048)
        p, q = a * top, a * low          # < 2^53, < 2^43
        p_hi, p_lo = torch.floor(p / 2 ** 21), torch.remainder(p, 2 ** 21)
        rest = p_lo * 2048 + q           # < 2^32 + 2^43
        return (p_hi + torch.floor(rest / full), torch.remainder(rest, full))

    def xor(x, y, z):
        y = y.long() if isinstance(y, torch.Tensor) else y
        return (x.long() ^ y ^ z).double()

    blk = torch.arange((n + 3) // 4, device=DEV)
    a, b = words(blk % full, blk // full)
    c2 = torch.full_like(a, float(call % full))
    d = torch.full_like(a, float(call // full))
    k0, k1 = seed % full, seed // full
    for r in range(10):
        kr0 = (k0 + r * 2654435769) % full
        kr1 = (k1 + r * 3144134277) % full
        ph, pl = product(3528531795.0, a)
        qh, ql = product(3449720151.0, c2)
        a, b, c2, d = xor(qh, b, kr0), ql, xor(ph, d, kr1), pl
    u = torch.stack((a, b, c2, d), 1).view(-1)[:n] / full
    kept = (u >= round(c['ratio'] * full) / full).double() / (1 - c['ratio'])
    return st['x'].double() * kept, st['gy'].double() * kept


def _exact_norm(st):
    case = st['case']
    h, w = st['x'].double(), st['weight'].double()
    if st['residual'] is not None:
        h = h + st['residual'].double()
    d = h.shape[1]
    r = 1.0 / torch.sqrt(h.square().sum(1, keepdim=True) / d + 1e-6)
    if case['group'] >= 0:
        y = (h * r * w).reshape(h.shape[0], -1, case['group'] or d)
        s = y.abs().max(-1).values / E4M3_MAX
        s[s == 0] = 1.0
        out = ((y / s[..., None]).reshape(h.shape), s)
        return out if st['residual'] is None else out + (h,)
    gy = st['gy'].double()
    dot = (gy * w * h).sum(1, keepdim=True)
    dh = gy * w * r - h * dot * r ** 3 / d
    dw = torch.mv((gy * h).t(), r[:, 0])
    if st['residual'] is None:
        return h * r * w, dh, dw
    dh = dh + st['gh'].double()
    return h * r * w, h, dh, dh, dw


def _exact_step(st):
    q, k, v = (st[x].double() for x in 'qkv')
    lam = st['log_decay'].double().exp()
    s = torch.einsum('bhij,h->bhij', st['state'].double(), lam)
    s = s + torch.einsum('bhi,bhj->bhij', k, v)
    return torch.einsum('bhi,bhij->bhj', q, s) * st['scale'], s


def _exact_attn(st):
    """The recurrence itself, token by token."""
    case = st['case']
    b, t, h = case['batch'], case['length'], case['heads']
    dk, dv, scale = case['dk'], case['dv'], st['scale']
    if b * h * dk * dv * t > 5e9:
        return None
    q, k, v = (st[x].double().permute(1, 0, 2, 3).reshape(t, b * h, -1)
               for x in 'qkv')
    lam = st['log_decay'].double().exp().repeat(b)[:, None, None]
    n = torch.full((b,), t, device=DEV) if st['lengths'] is None \
        else st['lengths']
    live = (torch.arange(t, device=DEV)[:, None] < n).repeat_interleave(
        h, 1)[..., None].double()                        # [t, b * h, 1]
    s = torch.zeros(b * h, dk, dv, device=DEV, dtype=torch.float64)
    if st['state'] is not None:
        s = s + st['state'].double().view(b * h, dk, dv)
    train = case['train']
    o, dq = torch.zeros_like(v), torch.zeros_like(q)
    if train:
        go = st['go'].double().permute(1, 0, 2, 3).reshape(t, b * h, dv)
        go = go * live
    k, v, q = k * live, v * live, q * live
    keep = 1 + (lam[None] - 1) * live[..., None]         # 1 behind the end
    for i in range(t):
        s = torch.baddbmm(s * keep[i], k[i][:, :, None], v[i][:, None])
        o[i] = torch.bmm(q[i][:, None], s)[:, 0]
        if train:
            dq[i] = torch.bmm(s, go[i][:, :, None])[..., 0]

    def back(x):
        return x.view(t, b, h, -1).permute(1, 0, 2, 3)

    fin = s.view(b, h, dk, dv)
    if not train:
        return back(o * scale * live), fin
    a = torch.zeros_like(s)
    if st['state'] is not None:
        a = a + st['gs'].double().view(b * h, dk, dv)
    dk_, dv_ = torch.zeros_like(q), torch.zeros_like(v)
    for i in range(t - 1, -1, -1):
        a = torch.baddbmm(a, q[i][:, :, None], go[i][:, None] * scale)
        dk_[i] = torch.bmm(a, v[i][:, :, None])[..., 0]
        dv_[i] = torch.bmm(k[i][:, None], a)[:, 0]
        a = a * keep[i]
    g = [back(dq * scale * live), back(dk_ * live), back(dv_ * live)]
    if st['state'] is None:
        return [back(o * scale * live)] + g
    return [back(o * scale * live), fin] + g + [a.view(b, h, dk, dv)]


_EXACT = dict(embed=_exact_embed, drop=_exact_drop, norm=_exact_norm,
              step=_exact_step, attn=_exact_attn)
