"""The sequence operators (gated recurrence, block norms) on the GPU against the 64-bit references of tests/_sequence_ref.py, within the
running error bounds derived there."""
import contextlib
import math

import pytest
import torch
import torch.utils.checkpoint

from magvit2_pytorch_amd import functional as F
from magvit2_pytorch_amd.ops_hip import BlockNormDesc, GateLoopDesc, HipOps
from oracle.ndhwc_ops import CpuOps
from tests._sequence_ref import assert_within, block_norm_ref, gate_loop_ref

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float32]
NAN, INF = float('nan'), float('inf')


def rnd(*shape, seed=0, dtype=torch.float32, mean=0., std=1.):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype)


def loop_inputs(B, T, P, C, dtype, seed=0):
    qkva = rnd(B, T, P, 3 * C, seed=seed, dtype=dtype)
    qkva[..., 2 * C:] = qkva[..., 2 * C:] * 1.5 + 2
    return qkva


def check_loop(qkva, C, state=None, lengths=None, resets=None, train=True, fused=True):
    """qkva (B, T, P, 3C) on the GPU, any strides; every output of forward and backward against the reference"""
    dtype = qkva.dtype
    B, T, P = qkva.shape[:3]
    leaves = [qkva.detach().requires_grad_(train)] if fused else [t.detach().requires_grad_(train) for t in qkva.split(C, -1)]
    st = None if state is None else state.cuda().requires_grad_(train)
    cu = lambda t: None if t is None else t.cuda()
    y, h = F.gate_loop(leaves[0] if fused else tuple(leaves), state=st, lengths=cu(lengths), resets=cu(resets), return_state=True)
    parts = [t.cpu() for t in qkva.detach().split(C, -1)]
    dy, dh = rnd(B, T, P, C, seed=90, dtype=dtype), rnd(B, P, C, seed=91)
    ref = gate_loop_ref(*parts, state, lengths, resets, dy, dh, fast_exp=dtype == torch.bfloat16)
    assert_within(y, ref['y'], dtype, 'y')
    assert_within(h, ref['h'], torch.float32, 'h')
    if not train:
        return
    grads = torch.autograd.grad((y, h), leaves + ([st] if st is not None else []), (dy.cuda(), dh.cuda()))
    got = grads[0].split(C, -1) if fused else grads[:3]
    for name, g in zip(('dq', 'dkv', 'da'), got):
        assert_within(g, ref[name], dtype, name)
    if st is not None:
        assert_within(grads[-1], ref['dstate'], torch.float32, 'dstate')


# lengths around the spans that the kernels keep, join and split along (8, 16, 32, 64, 256, 512 and their neighbours)
LENGTHS = [1, 2, 7, 8, 9, 15, 17, 31, 33, 63, 64, 65, 255, 256, 257, 300, 511, 513, 1025]


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T', LENGTHS)
def test_gate_loop_lengths(T, dtype):
    B, P, C = 2, 1, 72
    check_loop(loop_inputs(B, T, P, C, dtype, T).cuda(), C, state=rnd(B, P, C, seed=1))


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('C', [1, 3, 4, 8, 12, 63, 64, 65, 130, 512, 1000])
def test_gate_loop_widths(C, dtype):
    B, T, P = 2, 70, 1
    check_loop(loop_inputs(B, T, P, C, dtype, C).cuda(), C, state=rnd(B, P, C, seed=1))


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('B,T,P,C', [(2, 5, 16, 64), (1, 17, 9, 24), (3, 33, 5, 7), (2, 600, 3, 40), (1, 2, 1000, 8)])
def test_gate_loop_pixels(B, T, P, C, dtype):
    check_loop(loop_inputs(B, T, P, C, dtype, T).cuda(), C, state=rnd(B, P, C, seed=1))
    check_loop(loop_inputs(B, T, P, C, dtype, T).cuda(), C, fused=False)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T', [9, 300, 1100])
@pytest.mark.parametrize('C', [64, 33])
def test_padded_batch(T, C, dtype):
    """lengths of zero, one, T, past T and below zero; what lies behind a sequence is never read (NaN), is zero in every result, and
    a reset there changes nothing"""
    lengths = torch.tensor([0, 1, T, T + 5, -3, T // 2, T - 1, 8])
    B = len(lengths)
    qkva = loop_inputs(B, T, 1, C, dtype, T)
    clean = qkva.clone()
    resets = rnd(B, T, seed=5) > 1.5
    for b, n in enumerate(lengths.clamp(0, T).tolist()):
        qkva[b, n:] = NAN
        clean[b, n:] = 0
        resets[b, n:] = True
    state = rnd(B, 1, C, seed=1)
    parts = clean.split(C, -1)
    leaf, st = qkva.cuda().requires_grad_(), state.cuda().requires_grad_()
    dy, dh = rnd(B, T, 1, C, seed=90, dtype=dtype), rnd(B, 1, C, seed=91)
    dyn = dy.clone()
    for b, n in enumerate(lengths.clamp(0, T).tolist()):
        dyn[b, n:] = NAN                                  # nor are the gradients that arrive there
    ref = gate_loop_ref(*parts, state, lengths, resets, dy, dh, fast_exp=dtype == torch.bfloat16)
    for ln in (lengths, lengths.int()):
        y, h = F.gate_loop(leaf, state=st, lengths=ln.cuda(), resets=resets.cuda(), return_state=True)
        g, gs = torch.autograd.grad((y, h), (leaf, st), (dyn.cuda(), dh.cuda()))
        assert_within(y, ref['y'], dtype, 'y')
        assert_within(h, ref['h'], torch.float32, 'h')
        for name, t in zip(('dq', 'dkv', 'da'), g.split(C, -1)):
            assert_within(t, ref[name], dtype, name)
        assert_within(gs, ref['dstate'], torch.float32, 'dstate')
        for b, n in enumerate(lengths.clamp(0, T).tolist()):
            assert not y[b, n:].any() and not g[b, n:].any()


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T', [20, 700, 1500])
def test_document_starts(T, dtype):
    """every kind of start: the first token, the last, neighbours, none in a long run"""
    B, C = 4, 40
    resets = torch.zeros(B, T, dtype=torch.bool)
    resets[0, 0] = resets[1, T - 1] = True
    resets[2, T // 2: T // 2 + 3] = True
    resets[3] = True
    check_loop(loop_inputs(B, T, 1, C, dtype, T).cuda(), C, state=rnd(B, 1, C, seed=1), resets=resets)
    check_loop(loop_inputs(B, T, 1, C, dtype, T).cuda(), C, state=rnd(B, 1, C, seed=1), resets=resets.to(torch.uint8) * 7, train=False)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T', [24, 900])
@pytest.mark.parametrize('poison', [NAN, INF, -INF])
def test_nothing_crosses_a_document_start(T, dtype, poison):
    """a document that holds infinities or NaN leaves its neighbours, forward and backward, as they are without it"""
    B, C, cut, end = 1, 16, T // 3, 2 * T // 3
    resets = torch.zeros(B, T, dtype=torch.bool)
    resets[:, cut] = resets[:, end] = True
    good = loop_inputs(B, T, 1, C, dtype, T)
    bad = good.clone()
    bad[:, cut:end] = poison
    dy, dh = rnd(B, T, 1, C, seed=90, dtype=dtype).cuda(), rnd(B, 1, C, seed=91).cuda()
    res = []
    for z in (good, bad):
        leaf = z.cuda().requires_grad_()
        y, h = F.gate_loop(leaf, resets=resets.cuda(), return_state=True)
        res.append((y, h, torch.autograd.grad((y, h), leaf, (dy, dh))[0]))
    (y0, h0, g0), (y1, h1, g1) = res
    assert torch.equal(h0, h1)
    for s in (slice(0, cut), slice(end, T)):
        assert torch.equal(y0[:, s], y1[:, s]) and torch.equal(g0[:, s], g1[:, s])


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T', [12, 800])
def test_extreme_decays(T, dtype):
    """decays of exactly one and exactly zero (the type's largest and lowest values, infinities), and close to both"""
    B, C = 2, 32
    top = torch.finfo(dtype).max
    qkva = loop_inputs(B, T, 1, C, dtype, T)
    qkva[..., C:2 * C] *= 0.05                            # sums of T terms stay moderate
    vals = torch.tensor([top, -top, INF, -INF, 30., -30., 12., -12.])
    qkva[..., 2 * C:] = vals.to(dtype).repeat(C // 8)
    check_loop(qkva.cuda(), C, state=rnd(B, 1, C, seed=1))


@pytest.mark.parametrize('dtype', DT)
def test_strides(dtype):
    """batch and token axes exchanged, parts of wider rows, rows that start off a 16-byte boundary, repeated rows, transposed channels"""
    B, T, P, C = 3, 70, 2, 16
    base = loop_inputs(B, T, P, C, dtype)
    for z in (loop_inputs(T, B, P, C, dtype, 1).cuda().transpose(0, 1),
              loop_inputs(B, P, T, C, dtype, 2).cuda().transpose(1, 2),
              torch.nn.functional.pad(base, (16, 24)).cuda()[..., 16:16 + 3 * C],
              torch.nn.functional.pad(base, (1, 2)).cuda()[..., 1:1 + 3 * C],
              base.cuda()[:1].expand(B, T, P, 3 * C),
              base.cuda()[:, ::2],
              base.cuda().transpose(2, 3).contiguous().transpose(2, 3)):
        check_loop(z, C, state=rnd(B, P, C, seed=1))
        check_loop(z, C, fused=False)
    # three tensors whose strides differ
    q, kv, a = (t.cuda() for t in base.split(C, -1))
    y = F.gate_loop((q.contiguous(), kv, a.transpose(0, 1).contiguous().transpose(0, 1)))
    assert torch.equal(y, F.gate_loop(base.cuda()))


@pytest.mark.parametrize('dtype', DT)
def test_rows_past_32_bit_offsets(dtype):
    """two sequences more than 2^31 elements apart, and a token stride that leaves 32 bits"""
    B, T, C = 2, 40, 32
    far = (1 << 31) + 64
    store = torch.zeros(far + T * 3 * C, dtype=dtype, device='cuda')
    z = store.as_strided((B, T, 1, 3 * C), (far, 3 * C, 3 * C, 1))
    z.copy_(loop_inputs(B, T, 1, C, dtype))
    check_loop(z, C, state=rnd(B, 1, C, seed=1))
    wide = 1 << 26                                        # 40 tokens: 2.7e9 elements
    store = torch.zeros(T * wide + 3 * C, dtype=dtype, device='cuda')
    z = store.as_strided((1, T, 1, 3 * C), (0, wide, 0, 1))
    z.copy_(loop_inputs(1, T, 1, C, dtype))
    check_loop(z, C)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T,C', [(20011, 8), (9000, 70), (33000, 3)])
def test_long_sequences(T, C, dtype):
    check_loop(loop_inputs(1, T, 1, C, dtype, T).cuda(), C, state=rnd(1, 1, C, seed=1))


@pytest.mark.parametrize('dtype', DT)
def test_steps_follow_the_whole_sequence(dtype):
    """prefill, then token by token in place: states and outputs of the one call over all tokens"""
    B, T, C, pre = 3, 40, 72, 29
    z = loop_inputs(B, T, 1, C, dtype).squeeze(2).cuda()
    parts = [t.cpu().unsqueeze(2) for t in z.split(C, -1)]
    ref = gate_loop_ref(*parts, fast_exp=dtype == torch.bfloat16)
    y, state = F.gate_loop(z[:, :pre], return_state=True)
    ys = [y]
    for t in range(pre, T):
        if t % 2:
            ys.append(F.gate_loop_step(z[:, t], state)[:, None])
        else:
            new = torch.full_like(state, NAN)
            ys.append(F.gate_loop_step(tuple(z[:, t].split(C, -1)), state, state_out=new)[:, None])
            state = new
    assert_within(torch.cat(ys, 1), ref['y'], dtype, 'y')
    assert_within(state, ref['h'], torch.float32, 'h')
    pix = loop_inputs(2, 1, 6, 24, dtype).cuda()
    s0 = rnd(2, 6, 24, seed=3).cuda()
    y, h = F.gate_loop(pix, state=s0, return_state=True)
    s = s0.clone()
    assert torch.equal(F.gate_loop_step(pix[:, 0], s), y[:, 0]) and torch.equal(s, h)


@pytest.mark.parametrize('dtype', DT)
def test_last_state_written_over_the_first(dtype):
    """the C ABI lets h_last be h0 itself, for any length"""
    for B, T, C in ((2, 1, 64), (2, 600, 40), (1, 5000, 64), (1, 5000, 9)):
        z = loop_inputs(B, T, 1, C, dtype).cuda()
        y, h = F.gate_loop(z, state=(s0 := rnd(B, C, seed=2).cuda())[:, None], return_state=True)
        ops = HipOps(z.device)
        d = GateLoopDesc(dtype=0 if dtype == torch.bfloat16 else 1, B=B, T=T, P=1, C=C, in_b=z.stride(0), in_t=z.stride(1), in_p=z.stride(2),
                         grad_b=0, grad_t=0, grad_p=0)
        ws = torch.empty(max(1, ops.gateloop_sizes(d)[1]), dtype=torch.uint8, device='cuda')
        s, y2 = s0.clone(), torch.empty_like(y)
        ops.gateloop_forward(d, *z.split(C, -1), s, None, None, y2, s, None, ws)(ops.current_stream())
        assert torch.equal(s, h[:, 0]) and torch.equal(y2, y)


def test_results_do_not_change_from_call_to_call():
    z = loop_inputs(2, 5000, 1, 136, torch.bfloat16).cuda().requires_grad_()
    w = [torch.ones(136, device='cuda', requires_grad=True) for _ in range(3)]
    first = None
    for _ in range(4):
        y, h = F.gate_loop(z, return_state=True)
        g = torch.autograd.grad((y, h), z, (torch.ones_like(y), torch.ones_like(h)))[0]
        out, n = F.block_norm(y, y * 2, gate=y, post_gamma=w[0], scale=w[1], pre_gamma=w[2])
        gw = torch.autograd.grad((out, n), w, (y, y))
        now = [y, h, g, out, n, *gw]
        if first is None:
            first = now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


# ----------------------------------------------------------------------------------------------------------------- block norm
def check_norm(R, C, dtype, act='silu', branch=True, gate=True, post=True, scale=True, pre=True, make=None, train=True, up=('dout', 'dn'), seed=0):
    make = make or (lambda t: t.cuda())
    row = lambda i, std=1.: rnd(R, C, seed=seed + i, dtype=dtype, std=std)
    vec = lambda i: rnd(C, seed=seed + 10 + i, mean=1., std=0.3)
    t = dict(x=row(0, 2.))
    if branch:
        t['branch'] = row(1)
        if gate:
            t['gate'] = row(2, 3.)
        if post:
            t['post'] = vec(0)
        if scale:
            t['scale'] = vec(1)
    if pre:
        t['pre'] = vec(2)
    return run_norm(t, act, make, train, up)


def run_norm(t, act, make, train=True, up=('dout', 'dn')):
    dtype = t['x'].dtype
    d = {k: (make(v) if v.dim() == 2 else v.cuda()).detach().requires_grad_(train) for k, v in t.items()}
    out, n = F.block_norm(d['x'], d.get('branch'), gate=d.get('gate'), gate_act=act, post_gamma=d.get('post'), scale=d.get('scale'), pre_gamma=d.get('pre'))
    ups = {}
    if 'branch' in t and 'dout' in up:
        ups['dout'] = rnd(*t['x'].shape, seed=80, dtype=dtype)
    if 'pre' in t and 'dn' in up:
        ups['dn'] = rnd(*t['x'].shape, seed=81, dtype=dtype)
    ref = block_norm_ref(t['x'], t.get('branch'), t.get('gate'), act, t.get('post'), t.get('scale'), t.get('pre'), grads=train, **ups)
    for name, v in (('out', out), ('normed', n)):
        if name in ref:
            assert_within(v, ref[name], dtype, name)
    if not train:
        return
    outs = [v for k, v in (('dout', out), ('dn', n)) if k in ups]
    names = [k for k in t if not (k == 'pre' and 'dn' not in ups)]
    grads = torch.autograd.grad(outs, [d[k] for k in names], [v.cuda() for v in ups.values()])
    for k, g in zip(names, grads):
        assert_within(g, ref['d' + k], dtype if t[k].dim() == 2 else torch.float32, 'd' + k)


# widths around the thread and chunk counts of a row (64, 256, 512, 1024 threads; chunks of 1, 4 and 8), up to the widest
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('C', [1, 2, 7, 8, 16, 63, 64, 72, 127, 255, 256, 257, 500, 512, 520, 1001, 1023, 1032, 2048, 2056, 4096, 4100, 5001, 8192, 8200, 16383, 16384])
def test_block_norm_widths(C, dtype):
    check_norm(5, C, dtype)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('R', [1, 2, 3, 31, 33, 257, 5000])
@pytest.mark.parametrize('C', [24, 130])
def test_block_norm_rows(R, C, dtype):
    check_norm(R, C, dtype)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('act', ['silu', 'sigmoid', 'none'])
@pytest.mark.parametrize('C', [64, 33])
def test_block_norm_parts(act, C, dtype):
    for mask in range(16):
        gate, post, scale, pre = (bool(mask >> i & 1) for i in range(4))
        check_norm(9, C, dtype, act, True, gate, post, scale, pre)
    check_norm(9, C, dtype, branch=False)
    check_norm(9, C, dtype, up=('dout',))
    check_norm(9, C, dtype, up=('dn',))
    check_norm(9, C, dtype, train=False)


@pytest.mark.parametrize('dtype', DT)
def test_block_norm_strides(dtype):
    """thirds of a fused projection, rows off a 16-byte boundary, transposed rows, repeated rows, leading axes"""
    C, R = 40, 12

    def part(t, lo, width):
        w = torch.zeros(R, width, dtype=dtype, device='cuda')
        v = w[:, lo:lo + C]
        v.copy_(t)
        return v
    for make in (lambda t: part(t, 16, 160), lambda t: part(t, 3, 47), lambda t: t.t().contiguous().t().cuda(),
                 lambda t: part(t, 0, 80)):
        check_norm(R, C, dtype, make=make)
    x = rnd(2, 6, C, dtype=dtype).cuda()
    g = torch.ones(C, device='cuda')
    o1, n1 = F.block_norm(x, x.transpose(0, 1).contiguous().transpose(0, 1), pre_gamma=g)
    o2, n2 = F.block_norm(x.reshape(12, C), x.reshape(12, C), pre_gamma=g)
    assert o1.shape == x.shape and torch.equal(o1.reshape(12, C), o2) and torch.equal(n1.reshape(12, C), n2)
    row = x[0, :1].expand(R, C)
    o3, _ = F.block_norm(row, row, pre_gamma=g)
    assert torch.equal(o3, o2[:1].expand(R, C))
    o4, n4 = F.block_norm(x[0, 0], x[0, 0], pre_gamma=g)
    assert o4.shape == (C,) and torch.equal(n4, n2[0])


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('C', [48, 37])
def test_block_norm_rows_of_zeros_and_extremes(C, dtype):
    """rows of zeros (the floor of the norm: N is linear there), of tiny numbers, and gates at the ends of the type"""
    R = 6
    t = dict(x=rnd(R, C, dtype=dtype), branch=rnd(R, C, seed=1, dtype=dtype), gate=rnd(R, C, seed=2, dtype=dtype), post=rnd(C, seed=3, mean=1.),
             scale=rnd(C, seed=4), pre=rnd(C, seed=5, mean=1.))
    t['branch'][0] = 0
    t['x'][1] = 0
    t['branch'][1] = 0                                    # both norms at their floor
    t['x'][2] *= 1e-6
    t['branch'][2] *= 1e-6
    top = torch.finfo(dtype).max
    t['gate'][3] = torch.tensor([top, -top, 90., -90.]).repeat(C // 4 + 1)[:C].to(dtype)
    zeroed = dict(t, x=t['x'].clone(), branch=t['branch'].clone(), gate=t['gate'].clone())
    for act in ('silu', 'sigmoid'):
        if act == 'silu':                                 # silu of the largest number overflows the row by design
            zeroed['gate'][3] = torch.tensor([60., -top, 90., -90.]).repeat(C // 4 + 1)[:C].to(dtype)
        run_norm(zeroed if act == 'silu' else t, act, lambda v: v.cuda())


@pytest.mark.parametrize('dtype', DT)
def test_a_row_of_nan_stays_in_its_row(dtype):
    R, C = 70, 24
    x, b = rnd(R, C, dtype=dtype).cuda(), rnd(R, C, seed=1, dtype=dtype).cuda()
    g = torch.ones(C, device='cuda')
    o1, n1 = F.block_norm(x, b, post_gamma=g, pre_gamma=g)
    b2 = b.clone()
    b2[33, 5] = NAN                                       # one element: the row's norm is NaN, and so is all of the row
    o2, n2 = F.block_norm(x, b2, post_gamma=g, pre_gamma=g)
    rest = torch.arange(R, device='cuda') != 33
    assert o2[33].isnan().all() and n2[33].isnan().all() and torch.equal(o1[rest], o2[rest]) and torch.equal(n1[rest], n2[rest])


def test_block_norm_rows_past_32_bit_offsets():
    C, R = 64, 40
    step = 1 << 20
    far = torch.zeros((1 << 31) + 64 + R * C, dtype=torch.bfloat16, device='cuda')
    x = far[-R * C:].view(R, C)
    x.copy_(rnd(R, C, dtype=torch.bfloat16))
    wide = torch.zeros(2100 * step, dtype=torch.bfloat16, device='cuda').view(2100, step)[:, 8:8 + C]      # the last row begins past 2^31 elements
    val = rnd(2100, C, seed=1, dtype=torch.bfloat16)
    wide.copy_(val)
    g = torch.ones(C, device='cuda')
    o, n = F.block_norm(wide, wide, pre_gamma=g)
    ref = block_norm_ref(val, val, pre=torch.ones(C))
    assert_within(o, ref['out'], torch.bfloat16, 'out')
    assert_within(n, ref['normed'], torch.bfloat16, 'normed')
    assert_within(F.block_norm(x, pre_gamma=g)[1], block_norm_ref(rnd(R, C, dtype=torch.bfloat16), pre=torch.ones(C))['normed'], torch.bfloat16, 'normed')


# ----------------------------------------------------------------------------------------------------------------- as used together
def two_blocks(x, weights, lengths=None, states=None, gate=F.gate_loop, norm=F.block_norm):
    """norm, projection, recurrence, norm / gate / scale / residual add and the next norm: two blocks; x (B, T, C)"""
    C = x.shape[-1]
    _, n = norm(x, pre_gamma=weights['n0'])
    new = []
    for i in range(2):
        z = n @ weights[f'p{i}'].t()
        y, s = gate(z[..., :3 * C], state=None if states is None else states[i], lengths=lengths, return_state=True)
        new.append(s)
        x, n = norm(x, y, gate=z[..., 3 * C:], post_gamma=weights[f'w{i}'], scale=weights[f's{i}'], pre_gamma=weights[f'n{i + 1}'])
    return n, new


def block_weights(C, dtype=torch.float32):
    w = {f'p{i}': (rnd(4 * C, C, seed=i) / C ** 0.5).to(dtype) for i in range(2)}
    w.update({f'{k}{i}': rnd(C, seed=20 + 3 * i + j, mean=1., std=0.2) for j, k in enumerate('nws') for i in range(3)})
    return {k: v for k, v in w.items() if k not in ('w2', 's2')}


def plain_gate(z, state=None, lengths=None, return_state=True):
    C = z.shape[-1] // 3
    q, kv, a = z.split(C, -1)
    h = torch.zeros_like(q[:, 0]) if state is None else state
    ys = []
    for t in range(z.shape[1]):
        on = (torch.full((z.shape[0],), z.shape[1]) if lengths is None else lengths)[:, None] > t
        h = torch.where(on, torch.sigmoid(a[:, t]) * h + kv[:, t], h)
        ys.append(torch.where(on, q[:, t] * h, torch.zeros_like(h)))
    return torch.stack(ys, 1), h


def plain_norm(x, branch=None, gate=None, post_gamma=None, scale=None, pre_gamma=None):
    N = lambda v, w: torch.nn.functional.normalize(v, dim=-1) * v.shape[-1] ** 0.5 * w
    if branch is not None:
        x = x + scale * torch.nn.functional.silu(gate) * N(branch, post_gamma)
    return x, N(x, pre_gamma)


def test_two_blocks_train_and_decode():
    """the operators in a chain, in 32 bits: outputs, states and every gradient against the same chain in 64 bits; then prefill and
    single tokens against the whole sequence.  Tolerance: the chain multiplies errors of 1e-7 by its condition, of order 100 here (two norms,
    two recurrences and two projections of unit gain, gradients up to ten times larger): 2e-5 of each result's largest value."""
    B, T, C = 2, 37, 48
    w = block_weights(C)
    x = rnd(B, T, C, seed=50)
    lengths = torch.tensor([T, 20])
    w64 = {k: v.double().requires_grad_() for k, v in w.items()}
    x64 = x.double().requires_grad_()
    n64, s64 = two_blocks(x64, w64, lengths, gate=plain_gate, norm=plain_norm)
    up = rnd(B, T, C, seed=51)
    live = (torch.arange(T)[None] < lengths[:, None])[..., None]
    want = torch.autograd.grad((n64 * live * up.double()).sum() + s64[0].sum() + s64[1].sum(), [x64, *w64.values()])
    wg = {k: v.cuda().requires_grad_() for k, v in w.items()}
    xg = x.cuda().requires_grad_()
    n, s = two_blocks(xg, wg, lengths.cuda())
    got = torch.autograd.grad((n * live.cuda() * up.cuda()).sum() + s[0].sum() + s[1].sum(), [xg, *wg.values()])
    for what, a, b in [('n', n * live.cuda(), n64 * live), ('s0', s[0], s64[0]), ('s1', s[1], s64[1])] + list(zip(['x', *w], got, want)):
        assert (a.detach().double().cpu() - b.detach()).abs().max() <= 2e-5 * b.detach().abs().max(), what
    with torch.no_grad():
        full, last = two_blocks(xg[:1], wg)
        pre, st = two_blocks(xg[:1, :30], wg)
        assert (pre - full[:, :30]).abs().max() <= 2e-5 * full.abs().max()
        for t in range(30, T):
            tok = xg[:1, t]
            _, nn = F.block_norm(tok, pre_gamma=wg['n0'])
            for i in range(2):
                z = nn @ wg[f'p{i}'].t()
                y = F.gate_loop_step(z[:, :3 * C], st[i])
                tok, nn = F.block_norm(tok, y, gate=z[:, 3 * C:], post_gamma=wg[f'w{i}'], scale=wg[f's{i}'], pre_gamma=wg[f'n{i + 1}'])
            assert (nn - full[:, t]).abs().max() <= 2e-5 * full.abs().max()
        for a, b in zip(st, last):
            assert (a - b).abs().max() <= 2e-5 * b.abs().max()


@pytest.mark.parametrize('T,C', [(40, 64), (3000, 40)])
def test_captured_and_replayed(T, C):
    """forward and backward of both operators in one graph, replayed on new inputs with eager work of the same operators in between"""
    B, dtype = 2, torch.bfloat16
    w = [torch.ones(C, device='cuda', requires_grad=True) for _ in range(3)]
    data = [loop_inputs(B, T, 1, C, dtype, s).squeeze(2).cuda() for s in range(4)]
    lengths = torch.tensor([T, T // 2], dtype=torch.int32, device='cuda')

    def work(z):
        y, h = F.gate_loop(z, lengths=lengths, return_state=True)
        out, n = F.block_norm(z[..., :C], y, gate=z[..., C:2 * C], post_gamma=w[0], scale=w[1], pre_gamma=w[2])
        g = torch.autograd.grad((out, n, h), [z, *w], (torch.ones_like(out), torch.ones_like(n), torch.ones_like(h)))
        return [t.detach() for t in (y, h, out, n)] + list(g)
    eager = [[t.clone() for t in work(z.clone().requires_grad_())] for z in data]
    static = data[0].clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work(static)
    for rep in (0, 1, 2, 3, 1):
        with torch.no_grad():
            static.copy_(data[rep])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager[rep]):
            assert torch.equal(a, b)
        again = work(data[rep].clone().requires_grad_())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, eager[rep]))


def test_two_graphs_and_two_streams_at_once():
    """two captured calls replayed on two streams, with eager calls on a third: each has its own workspaces"""
    C, T = 64, 20000
    data = [loop_inputs(1, T, 1, C, torch.bfloat16, s).squeeze(2).cuda() for s in range(3)]
    want = [F.gate_loop(z, return_state=True) for z in data]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(3)]
    for z in data[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(F.gate_loop(z, return_state=True))
        graphs.append(g)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = F.gate_loop(data[2], return_state=True)
        torch.cuda.synchronize()
        for got, ref in zip(outs + [third], want):
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T,P,C', [(2048, 1, 1024 + 512), (17, 2048, 256)])
def test_gate_loop_calls_larger_than_the_caches(T, P, C, dtype):
    """calls that move 256 MB and more go past the caches: the same numbers as sample by sample, which do not"""
    B = 12
    z = torch.randn(B, T, P, 3 * C, device='cuda', generator=torch.Generator('cuda').manual_seed(1)).to(dtype)
    dy, dh = torch.randn(B, T, P, C, device='cuda').to(dtype), torch.randn(B, P, C, device='cuda')
    one = T * P * C * z.element_size()
    assert 4 * B * one >= 256 << 20 > 7 * one
    resets = torch.rand(B, T, device='cuda') < 0.01

    def both(i, r):
        leaf = z[i].clone().requires_grad_()
        y, h = F.gate_loop(leaf, resets=None if r is None else r[i], return_state=True)
        return y.detach(), h.detach(), torch.autograd.grad((y, h), leaf, (dy[i], dh[i]))[0]
    for r in (None, resets):
        whole = both(slice(0, B), r)
        for b in range(B):
            assert all(torch.equal(w[b:b + 1], t) for w, t in zip(whole, both(slice(b, b + 1), r)))


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('R,C', [(60000, 768), (20000, 2048), (12000, 4096)])
def test_block_norm_calls_larger_than_the_caches(R, C, dtype):
    """rows of a large call are those of small ones; the column sums agree within the bound of their longer sums"""
    gen = torch.Generator('cuda').manual_seed(2)
    row = lambda: torch.randn(R, C, device='cuda', generator=gen).to(dtype)
    x, b, g, dout, dn = (row() for _ in range(5))
    assert x.numel() * x.element_size() * 4 >= 256 << 20
    w = [torch.rand(C, device='cuda', generator=gen) + 0.5 for _ in range(3)]

    def both(i):
        leaves = [t[i].clone().requires_grad_() for t in (x, b, g)] + [t.clone().requires_grad_() for t in w]
        out, n = F.block_norm(leaves[0], leaves[1], gate=leaves[2], post_gamma=leaves[3], scale=leaves[4], pre_gamma=leaves[5])
        return [out.detach(), n.detach(), *torch.autograd.grad((out, n), leaves, (dout[i], dn[i]))]
    whole = both(slice(0, R))
    step = R // 8
    parts = [both(slice(i, i + step)) for i in range(0, R, step)]
    for k in range(5):
        assert torch.equal(whole[k], torch.cat([p[k] for p in parts]))
    for k in range(5, 8):
        # each of the two sums is off by at most (additions on a value's way: R / 1000 + 800) 2^-24 of the sum of absolute values, which for terms
        # of one size and random sign is about sqrt(R) times the sum's own size
        got, want = whole[k].double(), sum(p[k].double() for p in parts)
        size = want.square().mean().sqrt() * R ** 0.5
        assert (got - want).abs().max() <= 2 * (R / 1000 + 800) * 2.0 ** -24 * size * 4


def test_outputs_past_32_bit_offsets():
    """more than 2^31 outputs of one call: the second half of a sequence and its gradients are those of a call that begins there"""
    half, C, dtype = 1 << 21, 520, torch.bfloat16
    gen = torch.Generator('cuda').manual_seed(3)
    z = torch.empty(1, 2 * half, 3 * C, device='cuda', dtype=dtype)
    for i in range(0, 2 * half, 1 << 18):
        z[:, i:i + (1 << 18)].copy_(torch.randn(1, 1 << 18, 3 * C, device='cuda', generator=gen))
    dy = torch.randn(1, half, C, device='cuda', generator=gen).to(dtype).repeat(1, 2, 1)
    assert dy.numel() > 1 << 31

    def both(z, dy, s):
        leaf = z.requires_grad_()
        y, h = F.gate_loop(leaf, state=s, return_state=True)
        return y.detach(), h.detach(), torch.autograd.grad((y, h), leaf, (dy, torch.ones_like(h)))[0]
    _, mid = F.gate_loop(z[:, :half], return_state=True)
    y, h, g = both(z, dy, None)
    y2, h2, g2 = both(z.detach()[:, half:], dy[:, half:], mid)
    # the spans of the two calls are joined in other groups: some units of 2^-24 apart, at most one step of the type after the store
    near = lambda a, b: bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-4).all())
    assert near(h, h2)
    for i in range(0, half, 1 << 18):
        s = slice(i, i + (1 << 18))
        assert near(y[:, half:][:, s], y2[:, s]) and near(g[:, half:][:, s], g2[:, s])
    del y, y2, g, g2, z
    R, C = (1 << 21) + 5, 1032
    x = torch.empty(R, C, device='cuda', dtype=dtype)
    for i in range(0, R, 1 << 18):
        x[i:i + (1 << 18)].copy_(torch.randn(min(1 << 18, R - i), C, device='cuda', generator=gen))
    w = torch.ones(C, device='cuda')
    out, n = F.block_norm(x, x, gate=x, post_gamma=w, pre_gamma=w)
    o2, n2 = F.block_norm(x[-100:], x[-100:], gate=x[-100:], post_gamma=w, pre_gamma=w)
    assert torch.equal(out[-100:], o2) and torch.equal(n[-100:], n2)


@pytest.mark.parametrize('dtype', DT)
def test_steps_match_the_emulation(dtype):
    """the launchers' steps (arguments frozen, launched on a stream that is passed in) against the kernel emulation: the gradients of a kept forward
    pass and the norms.  Tolerance: one rounding of the store (2^-8, 2^-24) and 2e-5 of the largest value for sums in another order."""
    B, T, P, C, dt = 2, 40, 3, 24, 0 if dtype == torch.bfloat16 else 1
    z, dy = loop_inputs(B, T, P, C, dtype), rnd(B, T, P, C, seed=5, dtype=dtype)
    h0, dh = rnd(B, P, C, seed=6), rnd(B, P, C, seed=7)
    st = (T * P * 3 * C, P * 3 * C, 3 * C)
    d = GateLoopDesc(dtype=dt, B=B, T=T, P=P, C=C, in_b=st[0], in_t=st[1], in_p=st[2], grad_b=st[0], grad_t=st[1], grad_p=st[2])
    x, b, g, dout, dn = (rnd(9, C, seed=10 + i, dtype=dtype) for i in range(5))
    w = [rnd(C, seed=20 + i, mean=1.) for i in range(3)]
    e = BlockNormDesc(dtype=dt, C=C, rows=9, x_stride=C, branch_stride=C, gate_stride=C, gate_act=2, reserved=0)
    res = []
    for ops in (HipOps('cuda:0'), CpuOps()):
        m = ops.to_device
        n, wf, wb = ops.gateloop_sizes(d)
        ws = ops.zeros((max(wf, wb, 1),), torch.uint8)
        zz, y, h, states = m(z), ops.empty((B, T, P, C), dtype), ops.empty((B, P, C), torch.float32), ops.empty((B, max(n, 1), P, C), torch.float32)
        dz, d0 = ops.empty((B, T, P, 3 * C), dtype), ops.empty((B, P, C), torch.float32)
        rows, one, vec = (lambda: ops.empty((9, C), dtype)), (lambda: ops.empty((2, 9), torch.float32)), (lambda: ops.empty((C,), torch.float32))
        out, nn, rstd, gr, gv = rows(), rows(), one(), [rows() for _ in range(3)], [vec() for _ in range(3)]
        nws = ops.zeros((ops.block_norm_workspace_bytes(e),), torch.uint8)
        par = [m(t) for t in w]
        steps = [ops.gateloop_forward(d, *zz.split(C, -1), m(h0), None, None, y, h, states, ws),
                 ops.gateloop_backward(d, *zz.split(C, -1), m(h0), None, None, states, m(dy), m(dh), *dz.split(C, -1), d0, ws),
                 ops.block_norm_forward(e, m(x), m(b), m(g), *par, out, nn, rstd),
                 ops.block_norm_backward(e, m(x), m(b), m(g), *par, rstd, m(dout), m(dn), *gr, *gv, nws)]
        for step in steps:
            step(ops.current_stream())
        ops.synchronize()
        res.append([t.double().cpu() for t in (y, h, dz, d0, out, nn, *gr, *gv)])
    for i, (a, r) in enumerate(zip(*res)):
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
        assert ((a - r).abs() <= 2 * half * r.abs() + 2e-5 * r.abs().max()).all(), i


def test_empty_calls():
    s = rnd(2, 8, seed=1).cuda().requires_grad_()
    z = torch.zeros(2, 0, 24, device='cuda', requires_grad=True)
    y, h = F.gate_loop(z, state=s, return_state=True)
    g = torch.autograd.grad((y, h), (z, s), (y, torch.full_like(h, 3.)))
    assert y.shape == (2, 0, 8) and torch.equal(h, s) and g[0].shape == z.shape and (g[1] == 3).all()
    assert F.gate_loop(torch.zeros(0, 5, 24, device='cuda')).shape == (0, 5, 8)
    x, w = torch.zeros(0, 8, device='cuda', requires_grad=True), torch.ones(8, device='cuda', requires_grad=True)
    out, n = F.block_norm(x, x, pre_gamma=w)
    gw = torch.autograd.grad((out, n), (x, w), (out, n))[1]
    assert n.shape == (0, 8) and not gw.any()


def test_two_host_threads():
    """calls of two threads at the same time, each on a stream of its own"""
    import threading
    data = [loop_inputs(1, 6000, 1, 64, torch.bfloat16, s).squeeze(2).cuda() for s in range(2)]
    w = torch.ones(64, device='cuda')

    def work(z):
        leaf = z.clone().requires_grad_()
        y, h = F.gate_loop(leaf, return_state=True)
        _, n = F.block_norm(leaf[..., :64], y, gate=leaf[..., 64:128], pre_gamma=w)
        return [t.detach() for t in (y, h, n)] + [torch.autograd.grad((y, n), leaf, (y.detach(), n.detach()))[0]]
    want = [work(z) for z in data]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = work(data[i])
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_second_derivatives_are_refused():
    z = loop_inputs(1, 4, 1, 8, torch.float32).cuda().requires_grad_()
    g = torch.autograd.grad(F.gate_loop(z).square().sum(), z, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), z)


def test_inputs_changed_before_the_backward_pass_are_refused():
    z = loop_inputs(1, 4, 1, 8, torch.float32).cuda()
    s = torch.zeros(1, 1, 8, device='cuda', requires_grad=True)
    y = F.gate_loop(z, state=s)
    z.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_step_kernels_leave_neighbours_alone():
    """guard values around every output"""
    for dtype in DT:
        for C in (8, 13):
            B = 3
            z = loop_inputs(B, 1, 1, C, dtype).view(B, 3 * C).cuda()
            pool = torch.full((B * C + 64,), 7., device='cuda')
            state = pool[32:32 + B * C].view(B, C)
            state.zero_()
            F.gate_loop_step(z, state)
            assert (pool[:32] == 7).all() and (pool[32 + B * C:] == 7).all()
            assert torch.equal(state, z[:, C:2 * C].float())


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('B,T,P,C', [(2, 150, 5000, 5), (1, 264, 8192, 8), (1, 264, 8191, 3), (3, 20, 256, 1), (3, 21, 256, 1)])
def test_many_narrow_rows(dtype, B, T, P, C):
    """rows shorter than a tile, on both sides of the counts that change the form, with states, lengths and document starts"""
    z = loop_inputs(B, T, P, C, dtype).cuda()
    n = torch.tensor([T, 0, T // 2][:B], dtype=torch.int32)
    resets = torch.zeros(B, T, dtype=torch.bool)
    resets[:, 7::13] = True
    check_loop(z, C, state=rnd(B, P, C, seed=1), lengths=n, resets=resets)
    check_loop(z, C)


@pytest.mark.parametrize('C', [5, 72, 2048])
@pytest.mark.parametrize('dtype', DT)
def test_rows_beyond_the_norms_range(dtype, C):
    """rows whose sum of squares leaves fp32 have a norm of zero, as documented, and finite gradients; rows below the floor stay linear: 1e-30 / 1e-12
    sqrt(C).  Their neighbours do not see them: bitwise what they are without them."""
    x = rnd(7, C, dtype=dtype).cuda()
    g = rnd(C, seed=1, mean=1.).cuda().requires_grad_()
    n0 = F.block_norm(x, pre_gamma=g)[1]
    x2 = x.clone()
    x2[1], x2[4] = 1e25, 1e-30
    leaf = x2.requires_grad_()
    out, n = F.block_norm(torch.zeros_like(x), leaf, post_gamma=g, pre_gamma=None)[0], F.block_norm(leaf, pre_gamma=g)[1]
    rest = [0, 2, 3, 5, 6]
    assert torch.equal(n[rest], n0[rest]) and torch.equal(out[rest], n0[rest])
    tiny = x2[4].double() * 1e12 * C ** 0.5 * g.double()
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    for v in (out, n):
        assert v[1].eq(0).all()
        assert ((v[4].double() - tiny).abs() <= (half + 8 * 2.0 ** -24) * tiny.abs()).all()
    dx, dg = torch.autograd.grad((out, n), (leaf, g), (rnd(7, C, seed=2, dtype=dtype).cuda(),) * 2)
    assert dx.isfinite().all() and dg.isfinite().all() and dx[1].eq(0).all()


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T', [1024, 1025, 2049, 8192, 8193, 16385, 66100])
def test_groups_and_sets_of_spans(T, dtype):
    """spans are joined in groups of 8 and sets of 64 (of 256 tokens forward and 128 or 256 backward): lengths around them and far beyond, with decays
    that carry a state over thousands of tokens, a first state, a length and a document start"""
    C = 8
    z = loop_inputs(1, T, 1, C, dtype, T)
    z[..., 2 * C::2] += 7
    resets = torch.zeros(1, T, dtype=torch.bool)
    resets[0, T * 3 // 5] = True
    check_loop(z.cuda(), C, state=100 * rnd(1, 1, C, seed=1), lengths=torch.tensor([T - 40]), resets=resets)
    check_loop(z.cuda(), C, state=100 * rnd(1, 1, C, seed=1))


def test_sets_of_groups_in_many_tiles():
    """long sequences of several tiles against the same tokens in shorter calls, the state handed on"""
    B, T, C, cut = 3, 140000, 136, (0, 20000, 64000, 140000)
    z = loop_inputs(B, T, 1, C, torch.float32).cuda()
    z[..., 2 * C:] += 5
    y, h = F.gate_loop(z, return_state=True)
    s, parts = None, []
    for a, b in zip(cut, cut[1:]):
        p, s = F.gate_loop(z[:, a:b], state=s, return_state=True)
        parts.append(p)
    ref = torch.cat(parts, 1)
    # decays of about 1 - e^-7: a state is off by some 20 units of 2^-24 for each of the ~1100 tokens that it holds, in either call
    tol = 2 * 1100 * 20 * 2.0 ** -24
    assert ((y - ref).abs() <= tol * ref.abs().amax(1, keepdim=True)).all() and ((h - s).abs() <= tol * s.abs().amax()).all()


def test_saved_tensors_that_come_back_changed_are_refused():
    """hooks on saved tensors that hand back another type, size or device end in an error before anything is launched"""
    C = 16
    z, x = loop_inputs(1, 9, 1, C, torch.float32).cuda().requires_grad_(), rnd(9, C).cuda().requires_grad_()
    s, g = rnd(1, 1, C, seed=1).cuda().requires_grad_(), torch.ones(C, device='cuda', requires_grad=True)
    loop = lambda: F.gate_loop(z, state=s, lengths=torch.tensor([9], device='cuda', dtype=torch.int32), resets=torch.zeros(1, 9, dtype=torch.bool, device='cuda'))
    norm = lambda: F.block_norm(x, x, gate=x, post_gamma=g, scale=g, pre_gamma=g)[1]
    for call, count in ((loop, 5), (norm, 7)):                # state, lengths, resets, kept states (none for 9 tokens), qkva; x .. pre_gamma, norms
        for change in (torch.Tensor.double, torch.Tensor.cpu, lambda t: t.reshape(-1)[:-1]):
            for which in range(count - (call is loop)):
                n = iter(range(count))
                with torch.autograd.graph.saved_tensors_hooks(lambda t: (next(n), t), lambda p: change(p[1]) if p[0] == which else p[1]):
                    y = call()
                with pytest.raises((RuntimeError, ValueError)):
                    y.sum().backward()
        call().sum().backward()


@pytest.mark.parametrize('fused', [True, False])
def test_saved_tensors_laid_out_anew(fused):
    """hooks on saved tensors give back copies of another layout than the views that were saved"""
    B, T, C = 2, 300, 40
    wide, up = rnd(T, B, 3 * C + 3).cuda().requires_grad_(), rnd(B, T, C, seed=1).cuda()
    rows, w = rnd(70, 3 * C, seed=2).cuda().requires_grad_(), torch.ones(C, device='cuda', requires_grad=True)
    grads = []
    for pack in (None, lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()) if pack else contextlib.nullcontext():
            z = wide.transpose(0, 1)[..., 2:2 + 3 * C]
            y = F.gate_loop(z if fused else z.split(C, -1))
            q, kv, a = rows.split(C, -1)
            out, n = F.block_norm(q, kv, gate=a, post_gamma=w, pre_gamma=w)
        grads.append(torch.autograd.grad((y, out, n), (wide, rows, w), (up, torch.ones_like(out), rnd(70, C, seed=3).cuda())))
    for other in grads[1:]:
        for a, b in zip(grads[0], other):                 # rows at other alignments may be summed by another kernel
            assert ((a - b).abs() <= 64 * 2.0 ** -24 * b.abs().amax()).all()


def test_graphs_of_gradients():
    """gradients of some inputs only, of one output only, twice from a kept graph, added up in .grad, through a checkpoint; a released graph and
    forward-mode derivatives are refused"""
    C = 24
    z, s = loop_inputs(2, 50, 1, C, torch.float32).cuda().requires_grad_(), rnd(2, 1, C, seed=1).cuda().requires_grad_()
    x, b, w = (rnd(*n, seed=i).cuda().requires_grad_() for i, n in enumerate(((30, C), (30, C), (C,))))
    loop, norm = lambda: F.gate_loop(z, state=s, return_state=True), lambda: F.block_norm(x, b, gate=b, post_gamma=w, scale=w, pre_gamma=w)
    for call, leaves in ((loop, (z, s)), (norm, (x, b, w))):
        outs = call()
        ups = [rnd(*o.shape, seed=7 + i).cuda() for i, o in enumerate(outs)]
        full = torch.autograd.grad(outs, leaves, ups, retain_graph=True)
        again = torch.autograd.grad(outs, leaves, ups, retain_graph=True)
        assert all(torch.equal(a, c) for a, c in zip(full, again))
        for i, leaf in enumerate(leaves):
            assert torch.equal(torch.autograd.grad(outs, leaf, ups, retain_graph=True)[0], full[i])
        one = [torch.autograd.grad(o, leaves, u, retain_graph=True) for o, u in zip(outs, ups)]
        zero = [torch.autograd.grad(outs, leaves, [u if i == j else torch.zeros_like(u) for j, u in enumerate(ups)], retain_graph=True) for i in range(2)]
        for a, c in zip(one, zero):
            assert all(torch.allclose(p, q, rtol=1e-5, atol=1e-5 * q.abs().max().item()) for p, q in zip(a, c))
        torch.autograd.backward(outs, ups, retain_graph=True)
        torch.autograd.backward(outs, ups)
        assert all(torch.equal(leaf.grad, 2 * f) for leaf, f in zip(leaves, full))
        with pytest.raises(RuntimeError):
            torch.autograd.backward(outs, ups)
        under = torch.utils.checkpoint.checkpoint(call, use_reentrant=False)
        assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(under, leaves, ups), full))
        with torch.autograd.set_detect_anomaly(True):
            assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(call(), leaves, ups), full))
        with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
            dual = torch.autograd.forward_ad.make_dual(leaves[0].detach(), torch.ones_like(leaves[0])).requires_grad_()
            F.gate_loop(dual) if call is loop else F.block_norm(dual, pre_gamma=w)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('C', [1028, 1284, 1537, 2055, 2560, 3080, 5119, 5120, 6144, 7000, 7168, 10240, 12288, 14000])
def test_block_norm_whole_waves(C, dtype):
    """widths that fill 3 to 16 waves of a workgroup, in one row and in more rows than the chip takes at once"""
    check_norm(3, C, dtype)
    R = 1700
    gen = torch.Generator('cuda').manual_seed(C)
    x, b, g = (torch.randn(R, C, device='cuda', generator=gen).to(dtype) for _ in range(3))
    w = [torch.rand(C, device='cuda', generator=gen) + 0.5 for _ in range(3)]
    part = lambda i: F.block_norm(x[i], b[i], gate=g[i], post_gamma=w[0], scale=w[1], pre_gamma=w[2])
    for whole, *parts in zip(part(slice(0, R)), *(part(slice(i, i + 100)) for i in range(0, R, 100))):
        assert torch.equal(whole, torch.cat(parts))


def test_tangents_are_refused():
    """forward mode through every entry point, by any input, whether or not it requires grad, and by the gradients that arrive: refused, nothing written"""
    from torch.autograd import forward_ad
    C = 16
    z, s, x, w = rnd(2, 40, 3 * C).cuda(), rnd(2, C, seed=1).cuda(), rnd(7, C, seed=2).cuda(), torch.ones(C, device='cuda')
    leaf, rows = z.clone().requires_grad_(), x.clone().requires_grad_()
    y, (out, _) = F.gate_loop(leaf), F.block_norm(rows, x, pre_gamma=w)
    s0, new = s.clone(), torch.full_like(s, 7.)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: F.gate_loop(dual(z)), lambda: F.gate_loop(z, state=dual(s)), lambda: F.gate_loop((z[..., :C], z[..., C:2 * C], dual(z[..., 2 * C:]))),
                     lambda: F.gate_loop_step(dual(z[:, 0]), s), lambda: F.gate_loop_step(z[:, 0], dual(s)), lambda: F.gate_loop_step(z[:, 0], s, state_out=dual(new)),
                     lambda: F.block_norm(dual(x), pre_gamma=w), lambda: F.block_norm(x, dual(x)), lambda: F.block_norm(x, x, gate=dual(x)),
                     lambda: F.block_norm(x, pre_gamma=dual(w)), lambda: F.block_norm(x, x, scale=dual(w)), lambda: F.block_norm(x, x, post_gamma=dual(w)),
                     lambda: torch.autograd.grad(y, leaf, dual(torch.ones_like(y)), retain_graph=True),
                     lambda: torch.autograd.grad(out, rows, dual(torch.ones_like(out)), retain_graph=True)):
            for mode in (contextlib.nullcontext, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError):
                    call()
    assert torch.equal(s, s0) and (new == 7).all()
    torch.autograd.grad((y, out), (leaf, rows), (torch.ones_like(y), torch.ones_like(out)))


@pytest.mark.parametrize('shape', [(0, 3, 2), (0, 3), (2, 3, 0), (2, 0), (0, 0)])
def test_an_empty_batch_keeps_its_graph(shape):
    """no sequences or no tokens, in a training step: gradients reach every input, and what lies behind them"""
    C, w = 8, rnd(5, 24, seed=1).cuda().requires_grad_()
    z, s = torch.zeros(*shape, 5, device='cuda') @ w, torch.zeros(*shape[:1], *shape[2:], C, device='cuda', requires_grad=True)
    for rows in (z, z.bfloat16(), tuple(z.split(C, -1))):
        y, h = F.gate_loop(rows, state=s, return_state=True)
        g = torch.autograd.grad((y.float().sum(), h.sum()), (s, w), retain_graph=True)
        assert y.shape == (*shape, C) and h.shape == s.shape and h.dtype == torch.float32 and g[0].shape == s.shape and not g[1].any()
        out, n = F.block_norm(y, y, pre_gamma=torch.ones(C, device='cuda'))
        assert not torch.autograd.grad(n.float().sum(), w, retain_graph=True)[0].any() and out.shape == y.shape


def kind(t):
    """0 finite, 1 and 2 infinities, 3 NaN"""
    return torch.where(t.isnan(), 3, torch.where(t.isinf(), torch.where(t > 0, 1, 2), 0)).cpu()


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T', [8, 40, 300, 9000])
@pytest.mark.parametrize('C', [3, 40])
def test_infinite_states_decay_as_token_by_token(T, C, dtype):
    """an infinite state stays infinite while the decays are above zero, however small their product gets, in every form that the sizes choose; a
    decay of zero makes it NaN, a document start ends it.  So do infinite gradients on their way back.  Channels without one are as they were."""
    B = 5
    z = loop_inputs(B, T, 1, C, dtype, T)
    z[..., 2 * C:] -= 5                                   # decays of about 0.05: products of hundreds are far below the smallest number
    clean, s, dh = z.clone(), rnd(B, 1, C, seed=1), rnd(B, 1, C, seed=2)
    s0, dh0 = s.clone(), dh.clone()
    dy = rnd(B, T, 1, C, seed=3, dtype=dtype)
    resets = torch.zeros(B, T, dtype=torch.bool)
    s[0, :, 0], s[1, :, -1] = INF, -INF
    z[2, T // 2, 0, C] = INF                              # kv of channel 0
    dh[3, :, 0], dh[4, :, 0], s[4, :, 0] = INF, -INF, INF
    z[4, T // 2, 0, 2 * C] = -INF                         # a decay of zero
    resets[1, T - 2] = True
    hit = torch.zeros(B, C, dtype=torch.bool)
    for b, c in ((0, 0), (1, C - 1), (2, 0), (3, 0), (4, 0)):
        hit[b, c] = True
    res = []
    for zz, ss, dd in ((z, s, dh), (clean, s0, dh0)):
        leaf, st = zz.cuda().requires_grad_(), ss.cuda().requires_grad_()
        y, h = F.gate_loop(leaf, state=st, resets=resets.cuda(), return_state=True)
        g, gs = torch.autograd.grad((y, h), (leaf, st), (dy.cuda(), dd.cuda()))
        res.append(dict(y=y, h=h[:, None], dstate=gs[:, None], **dict(zip(('dq', 'dkv', 'da'), g.split(C, -1)))))
    ref = gate_loop_ref(*z.split(C, -1), s, None, resets, dy, dh)
    for name, got in res[0].items():
        want = ref[name][0].reshape(got.shape)
        assert torch.equal(kind(got), kind(want)), name
        rest = ~hit.cuda()[:, None, None].expand(got.shape)
        assert torch.equal(got[rest], res[1][name][rest]), name


def test_lazily_negated_tensors():
    """imaginary parts of conjugates carry their sign as a mark on the tensor; with one channel, or taken as they are, nothing else makes a copy of them"""
    neg = lambda t: torch.complex(torch.zeros_like(t), -t.detach()).conj().imag
    B, T, C = 2, 30, 4
    parts, s, up = [rnd(B, T, C, seed=i).cuda() for i in range(3)], rnd(B, C, seed=3).cuda(), rnd(B, T, C, seed=4).cuda()
    x, b, g = (rnd(9, C, seed=5 + i).cuda() for i in range(3))
    w, fused = rnd(C, seed=9, mean=1.).cuda(), torch.cat(parts, -1)
    for cut, lazy in ((slice(0, C), torch._neg_view), (slice(0, 1), neg)):
        plain = lambda t: t[..., cut].detach().clone()
        marked = lambda t: lazy(-plain(t)) if lazy is torch._neg_view else lazy(plain(t))
        assert marked(x).is_neg() and torch.equal(marked(x), plain(x))
        res = []
        for f in (plain, marked):
            q, kv, a, st, xx, bb, gg, ww = (f(t).requires_grad_() for t in (*parts, s, x, b, g, w))
            y, h = F.gate_loop((q, kv, a), state=st, return_state=True)
            out, n = F.block_norm(xx, bb, gate=gg, post_gamma=ww, scale=ww, pre_gamma=ww)
            grads = torch.autograd.grad((y, h, out, n), (q, kv, a, st, xx, bb, gg, ww), (f(up), f(s), f(x), f(b)))
            step = plain(s)
            res.append([y, h, out, n, *grads, F.gate_loop_step(tuple(f(t[:, 0]) for t in parts), step), step, F.gate_loop(fused if f is plain else torch._neg_view(-fused))])
        assert all(torch.equal(p, m) for p, m in zip(*res))
    one = torch.zeros(1, 1, device='cuda')
    for state, new in ((neg(one), None), (one, neg(one)), (torch._neg_view(one), None)):
        with pytest.raises(ValueError):
            F.gate_loop_step(torch.zeros(1, 3, device='cuda'), state, state_out=new)
    z = parts[0][..., :3].clone().requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, torch._neg_view):
        y = F.gate_loop(z)
    with pytest.raises(RuntimeError):
        y.sum().backward()


BF, FP = DT


@pytest.mark.parametrize('R,C,dtype', [(4097, 501, FP), (4097, 1001, BF), (4099, 1001, FP), (4097, 2048, BF), (4097, 768, FP), (2049, 1024, FP), (131073, 3, BF), (131073, 3, FP),
                                       (65537, 5, BF), (262145, 5, FP), (262145, 9, BF)])
def test_block_norm_of_many_rows(R, C, dtype):
    """rows taken two at a time (from 2048 turns of a workgroup's rows on), the last turn with one row or none in the second place: whole chunks, ragged
    ones and single elements, every part and the plain add and norm"""
    check_norm(R, C, dtype)
    check_norm(R, C, dtype, branch=False)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('R,C', [(131073, 4), (262145, 9), (4097, 784), (4097, 961), (5000, 2025), (60001, 256), (60001, 729), (3000, 2304), (1023, 5041), (257, 16384), (5, 784), (300, 961)])
def test_column_sums_are_exact_where_every_term_is(R, C, dtype):
    """parameter gradients to the last row: widths that are squares, rows of 4^j numbers +-1 and gradients of small whole numbers make every term and every
    partial sum of them exact in 32 bits, in any order, so the sums have to be equal"""
    gen = torch.Generator('cuda').manual_seed(R + C)
    few = 4 ** int(math.log(C, 4))
    v = torch.zeros(R, C, device='cuda')
    at = torch.rand(R, C, device='cuda', generator=gen).topk(few, -1).indices
    v.scatter_(1, at, torch.randint(0, 2, (R, few), device='cuda', generator=gen) * 2. - 1)
    up = torch.randint(-2, 3, (R, C), device='cuda', generator=gen).float()
    norm, root = few ** 0.5, round(C ** 0.5)
    assert (v.square().sum(-1) == few).all() and root * root == C
    sums = (v.double() * up.double()).sum(0)
    x, d = v.to(dtype), up.to(dtype)
    w = torch.ones(C, device='cuda', requires_grad=True)
    zero = torch.zeros_like(x)
    for call, want in ((lambda: F.block_norm(x, pre_gamma=w)[1], sums * root / norm), (lambda: F.block_norm(zero, x, post_gamma=w)[0], sums * root / norm),
                       (lambda: F.block_norm(zero, x, scale=w)[0], sums)):
        assert torch.equal(torch.autograd.grad(call(), w, d)[0].double(), want)


def test_a_step_over_a_saved_state_is_noticed():
    q, s = rnd(2, 3, 12).cuda().requires_grad_(), torch.ones(2, 4, device='cuda')
    y = F.gate_loop(q, state=s)
    F.gate_loop_step(rnd(2, 12, seed=1).cuda(), s)
    with pytest.raises(RuntimeError):
        y.sum().backward()
    y, other = F.gate_loop(q, state=s), torch.ones(2, 4, device='cuda')
    y2 = F.gate_loop(q, state=other)
    F.gate_loop_step(rnd(2, 12, seed=1).cuda(), s, state_out=other)      # the state is read, its other buffer written
    y.sum().backward()
    with pytest.raises(RuntimeError):
        y2.sum().backward()


def test_bf16_parameters_get_bf16_gradients():
    x, w = rnd(4, 8).cuda().requires_grad_(), [torch.full((8,), 1.5, device='cuda', dtype=t, requires_grad=True) for t in (torch.bfloat16, torch.float32)]
    g = [torch.autograd.grad(F.block_norm(x, x, post_gamma=p, scale=p, pre_gamma=p), p, (x.detach(), x.detach()))[0] for p in w]
    assert g[0].dtype == torch.bfloat16
    # three sums, each rounded to bf16, and two sums of those: 5 half steps of the largest partial result; the sums' own size bounds it for like signs
    parts = [torch.autograd.grad(F.block_norm(x, x, **{'post_gamma': w[1].detach(), 'scale': w[1].detach(), 'pre_gamma': w[1].detach(), k: w[1]}), w[1], (x.detach(), x.detach()))[0]
             for k in ('post_gamma', 'scale', 'pre_gamma')]
    assert ((g[0].float() - g[1]).abs() <= 5 * 2.0 ** -8 * sum(p.abs() for p in parts)).all()


@pytest.mark.parametrize('dtype', DT)
def test_a_captured_decoder_step(dtype):
    """a token's step and norm in a graph: each replay takes the state on, in place and between two buffers; lengths of 64 bits and a copied layout in another.
    The two forms' states differ by 14 units of 2^-24 a token and form at most, y by a step of the type then, the norm by what its gate (up to 3) makes of that and a step"""
    B, T, C = 3, 12, 40
    z = loop_inputs(B, T, 1, C, dtype).squeeze(2).cuda()
    w = rnd(C, seed=9, mean=1.).cuda()
    y0, h0 = F.gate_loop(z, return_state=True)
    tok, state, other = torch.zeros_like(z[:, 0]), torch.zeros(B, C, device='cuda'), torch.zeros(B, C, device='cuda')
    lengths = torch.full((B,), T, device='cuda')

    def step(s, new=None):
        y = F.gate_loop_step(tok, s, state_out=new)
        return y, F.block_norm(tok[:, :C], y, gate=tok[:, C:2 * C], pre_gamma=w)[1]

    def prompt():
        return F.gate_loop(z.transpose(1, 2).contiguous().transpose(1, 2), lengths=lengths, return_state=True)
    step(state.clone())
    prompt()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for call in (lambda: step(state), lambda: step(state, other), lambda: step(other, state), prompt):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for order in ([0] * T, [1, 2] * (T // 2)):
        state.zero_()
        for t, i in enumerate(order):
            tok.copy_(z[:, t])
            graphs[i].replay()
            want, norm = y0[:, t], F.block_norm(z[:, t, :C], y0[:, t], gate=z[:, t, C:2 * C], pre_gamma=w)[1]
            near = lambda a, b: bool(((a.float() - b.float()).abs() <= 4 * torch.finfo(dtype).eps * b.float().abs().amax()).all())
            assert near(outs[i][0], want) and near(outs[i][1], norm)
        assert ((state - h0).abs() <= 2 * 14 * T * 2.0 ** -24 * h0.abs().amax()).all()
    for n in (T, 5, 0, T + 3):
        lengths.fill_(n)
        graphs[3].replay()
        y, h = F.gate_loop(z, lengths=lengths, return_state=True)
        assert torch.equal(outs[3][0], y) and torch.equal(outs[3][1], h)
