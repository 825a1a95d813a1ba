"""Work of the gated linear recurrence and of the norms around a residual block, case by case.

`run` makes one pass of a case: with `own` false in elementary torch operations in 32 bits, with `own` true through
`magvit2_pytorch_amd.functional`.  `exact` computes the same outputs from the definitions in 64 bits.

Gated recurrence, per sample, pixel and channel along the tokens t (state 0 is `state`, or zero):
    h_t = sigmoid(a_t) h_{t-1} + kv_t        y_t = q_t h_t
tokens from `lengths[b]` on do not exist (their outputs and gradients are zero), and where `resets[b, t]` is set the sequence
starts anew with an empty state (documents packed into one row).

Block norm, per row of C channels, with N(v; gamma) = v / max(|v|, 1e-12) * sqrt(C) * gamma:
    out = x + scale * act(gate) * N(branch; post_gamma)        normed = N(out; pre_gamma)
"""
import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


# ------------------------------------------------------------------------------------------------------------------- cases
def _loop(name, mode, dtype, B, T, P, C, state=False, lengths=False, resets=False):
    return dict(name=name, op='gate_loop', mode=mode, dtype=dtype, B=B, T=T, P=P, C=C, state=state, lengths=lengths, resets=resets)


def _norm(name, mode, dtype, rows, C, post=True, gate='silu', scale=True, pre=True):
    return dict(name=name, op='block_norm', mode=mode, dtype=dtype, rows=rows, C=C, post=post, gate=gate, scale=scale, pre=pre)


def listed():
    return [
        # one stream, one new token: the call is all latency
        _loop('loop step 1x512', 'step', 'bf16', 1, 1, 1, 512, state=True),
        # one new token of each of many streams
        _loop('loop step 192x2048', 'step', 'bf16', 192, 1, 1, 2048, state=True),
        # four 17-frame clips, 32 x 32 positions, the time layer of the tokenizer: very many short sequences
        _loop('loop clip 4x17x1024x256', 'infer', 'bf16', 4, 17, 1024, 256),
        # prompts of different lengths in one padded batch, a continued state, sizes that fit no tile
        _loop('loop prefill 6x4095x1000', 'infer', 'bf16', 6, 4095, 1, 1000, state=True, lengths=True),
        # one very long sequence at a narrow width: all the parallelism is along the tokens
        _loop('loop long 1x131072x512', 'infer', 'bf16', 1, 131072, 1, 512, state=True),
        # a training step over documents packed into rows
        _loop('loop train 8x2048x2048', 'train', 'bf16', 8, 2048, 1, 2048, resets=True),
        # a training step in 32 bits at odd sizes, padded
        _loop('loop train odd 3x1023x777', 'train', 'fp32', 3, 1023, 1, 777, state=True, lengths=True),
        # around one block of a decoding batch: latency
        _norm('norm decode 32x2048', 'infer', 'bf16', 32, 2048),
        # the same over a prompt batch
        _norm('norm prefill 16384x2048', 'infer', 'bf16', 16384, 2048),
        # and in training
        _norm('norm train 16384x2048', 'train', 'bf16', 16384, 2048),
        # every position of four clips at a tokenizer width: residual add with the next layer's norm
        _norm('norm train clip 69632x256', 'train', 'bf16', 69632, 256, post=False, gate='none', scale=False),
        # odd rows and width in 32 bits
        _norm('norm train odd 4097x501', 'train', 'fp32', 4097, 501, gate='sigmoid'),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    dtype = rng.choice(['bf16', 'bf16', 'fp32'])
    room = 32_000_000 // (2 if dtype == 'fp32' else 1)    # elements: the work of the largest listed cases
    if rng.random() < 0.6:
        kind = rng.choice(['step', 'clip', 'tokens', 'tokens', 'tokens'])
        C = _log_int(rng, 16, 4096)
        if rng.random() < 0.6:
            C = max(16, C // 8 * 8)                       # whole 16-byte chunks, the usual case; the rest stays ragged
        if kind == 'step':
            return _loop('', 'step', dtype, _log_int(rng, 1, 512), 1, 1, C, state=True)
        mode = rng.choice(['infer', 'train'])
        if kind == 'clip':
            C = min(C, 512)
            B, T = rng.randint(1, 4), rng.randint(1, 33)
            P = min(_log_int(rng, 16, 1024), room // (B * T * C))
            return _loop('', mode, dtype, B, T, P, C)
        T = _log_int(rng, 2, 100000)
        C = min(C, max(16, room // T))
        B = rng.randint(1, max(1, min(16, room // (T * C))))
        return _loop('', mode, dtype, B, T, 1, C, state=rng.random() < 0.5, lengths=rng.random() < 0.5, resets=rng.random() < 0.3)
    C = _log_int(rng, 16, 8192)
    if rng.random() < 0.6:
        C = max(16, C // 8 * 8)
    rows = _log_int(rng, 1, min(100000, room // C))
    branch = rng.random() < 0.85
    return _norm('', rng.choice(['infer', 'train']), dtype, rows, C, post=branch and rng.random() < 0.7,
                 gate=rng.choice(['none', 'silu', 'sigmoid']) if branch else 'absent', scale=branch and rng.random() < 0.6,
                 pre=(not branch) or rng.random() < 0.8)


# ------------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case['dtype']]
    train = case['mode'] == 'train'

    def normal(*shape, mean=0., std=1., dtype=dt, grad=False):
        t = torch.empty(shape, device=dev, dtype=torch.float32).normal_(mean, std, generator=gen).to(dtype)
        return t.requires_grad_(grad)

    st = dict(case)
    if case['op'] == 'gate_loop':
        B, T, P, C = case['B'], case['T'], case['P'], case['C']
        lead = (B,) if case['mode'] == 'step' else (B, T)
        lead += (P,) if P > 1 else ()
        qkva = normal(*lead, 3 * C)
        qkva[..., 2 * C:].mul_(1.5).add_(2.)              # decays from about 0.3 to 0.999: memories of a few tokens and of hundreds
        st['qkva'] = qkva.requires_grad_(train)
        hs = (B, P, C) if P > 1 else (B, C)
        st['h'] = normal(*hs, dtype=torch.float32, grad=train) if case['state'] else None
        if case['mode'] == 'step':
            st['h_new'] = torch.empty_like(st['h'])       # a decoder's second state buffer: the two change places from token to token
        st['len'] = None
        if case['lengths']:
            n = torch.randint(0, T + 1, (B,), device=dev, generator=gen)
            n[0] = T                                      # a padded batch is as long as its longest sequence
            st['len'] = n.to(torch.int32)
        st['res'] = None
        if case['resets']:                                # documents of some 300 tokens
            st['res'] = torch.rand(B, T, device=dev, generator=gen) < 1 / 300
        if train:
            st['dy'] = normal(*lead, C)
            st['dh'] = normal(*hs, dtype=torch.float32)
        return st
    R, C = case['rows'], case['C']
    st['x'] = normal(R, C, std=2., grad=train)
    branch = case['gate'] != 'absent'
    st['b'] = normal(R, C, grad=train) if branch else None
    st['g'] = normal(R, C, grad=train) if branch and case['gate'] != 'none' else None
    st['post_w'] = normal(C, mean=1., std=0.1, dtype=torch.float32, grad=train) if case['post'] else None
    st['scale_w'] = normal(C, mean=0.3, std=0.1, dtype=torch.float32, grad=train) if case['scale'] else None
    st['pre_w'] = normal(C, mean=1., std=0.1, dtype=torch.float32, grad=train) if case['pre'] else None
    if train:
        st['dout'] = normal(R, C) if branch else None
        st['dn'] = normal(R, C) if case['pre'] else None
    return st


def work(case):
    es = 2 if case['dtype'] == 'bf16' else 4
    train = case['mode'] == 'train'
    if case['op'] == 'gate_loop':
        n = case['B'] * case['T'] * case['P'] * case['C']
        s = case['B'] * case['P'] * case['C'] * 4
        extra = (case['B'] * 4 if case['lengths'] else 0) + (case['B'] * case['T'] if case['resets'] else 0)
        by = n * 4 * es + s * (1 + case['state']) + extra
        fl = 8 * n
        if train:                                         # q, kv, a and dy again, three gradients, the state's gradients
            by += n * 7 * es + s * (1 + case['state']) + extra
            fl += 16 * n
        return dict(bytes=by, flops=fl)
    n, w = case['rows'] * case['C'], case['C'] * 4
    branch = case['gate'] != 'absent'
    gated = branch and case['gate'] != 'none'
    ins, nw = 1 + branch + gated, case['post'] + case['scale'] + case['pre']
    by = n * es * (ins + branch + case['pre']) + nw * w
    fl = 12 * n
    if train:                                             # the inputs again, the outputs' gradients, the inputs' gradients
        by += n * es * (ins + branch + case['pre'] + ins) + 2 * nw * w
        fl += 30 * n
    return dict(bytes=by, flops=fl)


# ------------------------------------------------------------------------------------------------------------------- plain form
def _scan(g, v):
    """h_t = g_t h_{t-1} + v_t along axis 1, the spans that are joined doubling from pass to pass"""
    d = 1
    while d < v.shape[1]:
        v = torch.cat([v[:, :d], v[:, d:] + g[:, d:] * v[:, :-d]], 1)
        g = torch.cat([g[:, :d], g[:, d:] * g[:, :-d]], 1)
        d *= 2
    return v


def _plain_loop(st):
    x = st['qkva'].detach()
    dt, C = x.dtype, st['C']
    step = st['mode'] == 'step'
    if step:
        x = x.unsqueeze(1)
    B, T = x.shape[:2]
    x = x.float()
    q, kv, a = x[..., :C], x[..., C:2 * C], x[..., 2 * C:]
    h0 = st['h'].detach() if st['h'] is not None else torch.zeros(B, *x.shape[2:-1], C, device=x.device)
    wide = (B, T) + (1,) * (x.dim() - 2)
    keep = 1 / (1 + torch.exp(-a))
    if st['res'] is not None:
        keep = torch.where(st['res'].view(wide), 0., keep)
    live = None
    if st['len'] is not None:
        live = (torch.arange(T, device=x.device) < st['len'].unsqueeze(1)).view(wide)
        keep, kv, q = torch.where(live, keep, 1.), torch.where(live, kv, 0.), torch.where(live, q, 0.)
    first = kv[:, :1] + keep[:, :1] * h0.unsqueeze(1)
    h = _scan(keep, torch.cat([first, kv[:, 1:]], 1))
    y = (q * h).to(dt)
    if step:
        return y.squeeze(1), h[:, -1]
    if st['mode'] == 'infer':
        return y, h[:, -1]
    dy = st['dy'].float()
    if live is not None:
        dy = torch.where(live, dy, 0.)
    before = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    # gradient of h_t: what y_t passes on, and what h_{t+1} passes back through its decay; the last state's own comes in at the end
    v = q * dy
    v = torch.cat([v[:, :-1], v[:, -1:] + st['dh'].unsqueeze(1)], 1)
    gn = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)
    dh = _scan(gn.flip(1), v.flip(1)).flip(1)
    slope = torch.exp(-a.abs()) / (1 + torch.exp(-a.abs())) ** 2
    dq, dkv, da = h * dy, dh, dh * before * slope
    if st['res'] is not None:
        da = torch.where(st['res'].view(wide), 0., da)
    if live is not None:
        dkv, da = torch.where(live, dkv, 0.), torch.where(live, da, 0.)
    out = [y, h[:, -1], torch.cat([dq, dkv, da], -1).to(dt)]
    if st['h'] is not None:
        out.append(keep[:, 0] * dh[:, 0])
    return tuple(out)


def _plain_norm(st):
    dt, root = st['x'].dtype, math.sqrt(st['C'])
    f = lambda k: None if st[k] is None else st[k].detach().float()
    x, b, g, w1, s, w2 = f('x'), f('b'), f('g'), f('post_w'), f('scale_w'), f('pre_w')
    out = x
    if b is not None:
        inv1 = 1 / b.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-12)
        unit = b * inv1 if w1 is not None else b
        u = unit * (root * w1) if w1 is not None else b
        sig = 1 / (1 + torch.exp(-g)) if g is not None else None
        act = 1. if g is None else (g * sig if st['gate'] == 'silu' else sig)
        sc = 1. if s is None else s
        out = x + sc * act * u
    inv2 = 1 / out.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-12)
    n = out * inv2 * (root * w2) if w2 is not None else None
    res = [t.to(dt) for t in (out if b is not None else None, n) if t is not None]
    if st['mode'] == 'infer':
        return tuple(res)
    dx = f('dout') if b is not None else torch.zeros_like(x)
    if w2 is not None:
        dn = f('dn')
        hat, v = out * inv2, dn * (root * w2)
        dx = dx + inv2 * (v - hat * (hat * v).sum(-1, keepdim=True))
        dw2 = (dn * hat * root).sum(0)
    res.append(dx.to(dt))
    if b is not None:
        dbranch = dx * sc * act
        if w1 is not None:
            v = dbranch * (root * w1)
            res.append((inv1 * (v - unit * (unit * v).sum(-1, keepdim=True))).to(dt))
        else:
            res.append(dbranch.to(dt))
        if g is not None:
            slope = sig * (1 + g * (1 - sig)) if st['gate'] == 'silu' else sig * (1 - sig)
            res.append((dx * sc * u * slope).to(dt))
        if w1 is not None:
            res.append((dbranch * unit * root).sum(0))
        if s is not None:
            res.append((dx * act * u).sum(0))
    if w2 is not None:
        res.append(dw2)
    return tuple(res)


# ------------------------------------------------------------------------------------------------------------------- the framework's calls
def _own_loop(st):
    from magvit2_pytorch_amd import functional as F
    if st['mode'] == 'step':
        return F.gate_loop_step(st['qkva'], st['h'], state_out=st['h_new']), st['h_new']
    y, h = F.gate_loop(st['qkva'], state=st['h'], lengths=st['len'], resets=st['res'], return_state=True)
    if st['mode'] == 'infer':
        return y, h
    leaves = [st['qkva']] + ([st['h']] if st['h'] is not None else [])
    return (y.detach(), h.detach()) + torch.autograd.grad((y, h), leaves, (st['dy'], st['dh']))


def _own_norm(st):
    from magvit2_pytorch_amd import functional as F
    out, n = F.block_norm(st['x'], st['b'], gate=st['g'], gate_act=st['gate'] if st['g'] is not None else 'none', post_gamma=st['post_w'],
                          scale=st['scale_w'], pre_gamma=st['pre_w'])
    res = [t for t in (out if st['b'] is not None else None, n) if t is not None]
    if st['mode'] == 'infer':
        return tuple(res)
    grads = [t for t in (st['dout'], st['dn']) if t is not None]
    leaves = [st[k] for k in ('x', 'b', 'g', 'post_w', 'scale_w', 'pre_w') if st[k] is not None]
    return tuple(t.detach() for t in res) + torch.autograd.grad(res, leaves, grads)


def run(state):
    loop = state['op'] == 'gate_loop'
    if own:
        return _own_loop(state) if loop else _own_norm(state)
    return _plain_loop(state) if loop else _plain_norm(state)


# ------------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_loop(st):
    """token by token, forward and then back"""
    z = st['qkva'].detach().double()
    if st['mode'] == 'step':
        z = z.unsqueeze(1)
    B, T, C = z.shape[0], z.shape[1], st['C']
    q, kv, logit = z.split(C, dim=-1)
    decay = torch.sigmoid(logit)
    per_token = (B, T) + (1,) * (z.dim() - 2)
    if st['res'] is not None:
        decay = decay.masked_fill(st['res'].view(per_token), 0.)
    dead = None
    if st['len'] is not None:                             # the state passes by a token that does not exist
        dead = (torch.arange(T, device=z.device)[None, :] >= st['len'].long()[:, None]).view(per_token)
        q, kv, decay = q.masked_fill(dead, 0.), kv.masked_fill(dead, 0.), decay.masked_fill(dead, 1.)
    start = torch.zeros_like(kv[:, 0]) if st['h'] is None else st['h'].detach().double()
    hist = torch.empty(kv.shape, dtype=torch.float64, device=z.device)
    h = start
    for new, keep, add in zip(hist.unbind(1), decay.unbind(1), kv.unbind(1)):
        h = torch.addcmul(add, keep, h, out=new)
    y = q * hist
    if st['mode'] == 'step':
        return y[:, 0], h
    if st['mode'] == 'infer':
        return y, h
    dy = st['dy'].double()
    if dead is not None:
        dy = dy.masked_fill(dead, 0.)
    arriving = torch.empty_like(hist)                     # at h_t: from y_t, and from h_{t+1}
    back = st['dh'].double()
    for d, keep, own_part in zip(reversed(arriving.unbind(1)), reversed(decay.unbind(1)), reversed((q * dy).unbind(1))):
        torch.add(own_part, back, out=d)
        back = d * keep
    before = torch.cat([start.unsqueeze(1), hist[:, :-1]], 1)
    dlogit = arriving * before * decay * torch.sigmoid(-logit)
    dkv = arriving
    if dead is not None:
        dkv, dlogit = dkv.masked_fill(dead, 0.), dlogit.masked_fill(dead, 0.)
    return (y, h, torch.cat([hist * dy, dkv, dlogit], -1)) + ((back,) if st['h'] is not None else ())


def _exact_norm(st):
    """the forward formulas, differentiated by autograd"""
    names = ('x', 'b', 'g', 'post_w', 'scale_w', 'pre_w')
    train = st['mode'] == 'train'
    v = {k: None if st[k] is None else st[k].detach().double().requires_grad_(train) for k in names}

    def rms(t, w):
        return torch.nn.functional.normalize(t, dim=-1, eps=1e-12) * (st['C'] ** 0.5) * w

    total = v['x']
    if v['b'] is not None:
        u = v['b'] if v['post_w'] is None else rms(v['b'], v['post_w'])
        if v['g'] is not None:
            u = u * (torch.nn.functional.silu(v['g']) if st['gate'] == 'silu' else torch.sigmoid(v['g']))
        if v['scale_w'] is not None:
            u = u * v['scale_w']
        total = total + u
    res = [total] if v['b'] is not None else []
    if v['pre_w'] is not None:
        res.append(rms(total, v['pre_w']))
    if not train:
        return tuple(res)
    ups = [st[k].double() for k in ('dout', 'dn') if st[k] is not None]
    return tuple(t.detach() for t in res) + torch.autograd.grad(res, [t for t in v.values() if t is not None], ups)


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_loop(st) if case['op'] == 'gate_loop' else _exact_norm(st)
