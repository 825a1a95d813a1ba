"""The sequence operators without a GPU: their autograd plumbing, layouts, padding and refusals over the kernel emulation, the references of
tests/_sequence_ref.py against autograd and against differences, and the C ABI's refusals."""
import contextlib
import ctypes

import pytest
import torch

from magvit2_pytorch_amd import functional as F
from magvit2_pytorch_amd import ops_hip
from magvit2_pytorch_amd.ops_hip import Mv2Error
from oracle.ndhwc_ops import CpuOps
from tests._sequence_ref import assert_within, block_norm_ref, gate_loop_ref

EINVAL, ETOOLARGE, EWORKSPACE = -1, -2, -3


@pytest.fixture
def emulated(monkeypatch):
    monkeypatch.setattr(F, '_backends', {torch.device('cpu'): CpuOps()})
    monkeypatch.setattr(F, '_plans', {})


def rnd(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def plain_loop(q, kv, a, state, lengths, resets):
    """sequential, differentiable, 64 bits"""
    h, ys = state, []
    for t in range(q.shape[1]):
        col = lambda m: m.view(-1, *([1] * (h.dim() - 1)))
        new = torch.sigmoid(a[:, t]) * h
        if resets is not None:
            new = torch.where(col(resets[:, t]), torch.zeros_like(new), new)
        new = new + kv[:, t]
        on = col(lengths > t)
        h = torch.where(on, new, h)
        ys.append(torch.where(on, q[:, t] * h, torch.zeros_like(h)))
    return torch.stack(ys, 1), h


def test_references_match_autograd():
    B, T, P, C = 3, 7, 2, 5
    q, kv, a = (rnd(B, T, P, C, seed=i).double().requires_grad_() for i in range(3))
    s = rnd(B, P, C, seed=3).double().requires_grad_()
    lengths, resets = torch.tensor([7, 0, 4]), rnd(B, T, seed=4) > 0.8
    y, h = plain_loop(q, kv, a, s, lengths, resets)
    dy, dh = rnd(B, T, P, C, seed=5).double(), rnd(B, P, C, seed=6).double()
    want = torch.autograd.grad((y, h), (q, kv, a, s), (dy, dh))
    ref = gate_loop_ref(q, kv, a, s, lengths, resets, dy, dh)
    for name, w in zip(('y', 'h', 'dq', 'dkv', 'da', 'dstate'), (y, h) + want):
        assert torch.allclose(ref[name][0], w.detach(), rtol=1e-12, atol=1e-13), name
    R, C = 6, 9
    x, b, g = (rnd(R, C, seed=10 + i).double().requires_grad_() for i in range(3))
    w1, sc, w2 = (rnd(C, seed=20 + i).double().requires_grad_() for i in range(3))
    norm = lambda v, w: torch.nn.functional.normalize(v, dim=-1) * C ** 0.5 * w
    for act, fn in (('none', lambda t: t), ('silu', torch.nn.functional.silu), ('sigmoid', torch.sigmoid)):
        out = x + sc * fn(g) * norm(b, w1)
        n = norm(out, w2)
        dout, dn = rnd(R, C, seed=30).double(), rnd(R, C, seed=31).double()
        want = torch.autograd.grad((out, n), (x, b, g, w1, sc, w2), (dout, dn))
        ref = block_norm_ref(x, b, g, act, w1, sc, w2, dout, dn, grads=True)
        for name, w in zip(('out', 'normed', 'dx', 'dbranch', 'dgate', 'dpost', 'dscale', 'dpre'), (out, n) + want):
            assert torch.allclose(ref[name][0], w.detach(), rtol=1e-11, atol=1e-12), (act, name)


def test_reference_gradients_match_differences():
    """one random direction, central differences: the error of a step e is e^2 times a third derivative of order one"""
    B, T, P, C, e = 2, 6, 1, 3, 1e-5
    ts = [rnd(B, T, P, C, seed=i).double() for i in range(3)] + [rnd(B, P, C, seed=3).double()]
    ds = [rnd(*t.shape, seed=9 + i).double() for i, t in enumerate(ts)]
    lengths, resets = torch.tensor([6, 3]), torch.zeros(B, T, dtype=torch.bool)
    resets[0, 2] = True
    dy, dh = rnd(B, T, P, C, seed=5).double(), rnd(B, P, C, seed=6).double()

    def loss(sign):
        r = gate_loop_ref(*[t + sign * e * d for t, d in zip(ts, ds)], lengths, resets)
        return (r['y'][0] * dy).sum() + (r['h'][0] * dh).sum()
    ref = gate_loop_ref(*ts, lengths, resets, dy, dh)
    along = sum((ref[k][0] * d).sum() for k, d in zip(('dq', 'dkv', 'da', 'dstate'), ds))
    assert abs((loss(1) - loss(-1)) / (2 * e) - along) < 1e-7 * (1 + abs(along))
    R, C = 5, 4
    ts = [rnd(R, C, seed=40 + i).double() for i in range(3)] + [rnd(C, seed=50 + i).double() for i in range(3)]
    ds = [rnd(*t.shape, seed=60 + i).double() for i, t in enumerate(ts)]
    dout, dn = rnd(R, C, seed=70).double(), rnd(R, C, seed=71).double()

    def nloss(sign):
        x, b, g, w1, s, w2 = [t + sign * e * d for t, d in zip(ts, ds)]
        r = block_norm_ref(x, b, g, 'silu', w1, s, w2)
        return (r['out'][0] * dout).sum() + (r['normed'][0] * dn).sum()
    x, b, g, w1, s, w2 = ts
    ref = block_norm_ref(x, b, g, 'silu', w1, s, w2, dout, dn, grads=True)
    along = sum((ref[k][0] * d).sum() for k, d in zip(('dx', 'dbranch', 'dgate', 'dpost', 'dscale', 'dpre'), ds))
    assert abs((nloss(1) - nloss(-1)) / (2 * e) - along) < 1e-7 * (1 + abs(along))


@pytest.mark.parametrize('fused', [True, False])
@pytest.mark.parametrize('P', [None, 3])
def test_gate_loop_plumbing(emulated, fused, P):
    B, T, C = 3, 6, 5
    mid = () if P is None else (P,)
    parts = [rnd(B, T, *mid, C, seed=i) for i in range(3)]
    state = rnd(B, *mid, C, seed=3).requires_grad_()
    lengths, resets = torch.tensor([6, 0, 4]), rnd(B, T, seed=4) > 0.8
    leaves = [torch.cat(parts, -1).requires_grad_()] if fused else [p.requires_grad_() for p in parts]
    y, h = F.gate_loop(leaves[0] if fused else tuple(leaves), state=state, lengths=lengths, resets=resets, return_state=True)
    dy, dh = rnd(*y.shape, seed=5), rnd(*h.shape, seed=6)
    grads = torch.autograd.grad((y, h), leaves + [state], (dy, dh))
    four = lambda t: t.reshape(B, T, -1, C)
    ref = gate_loop_ref(*map(four, parts), state.reshape(B, -1, C), lengths, resets, four(dy), dh.reshape(B, -1, C))
    got = grads[0].split(C, -1) if fused else grads[:3]
    for name, t in zip(('y', 'h', 'dq', 'dkv', 'da', 'dstate'), (y, h, *got, grads[-1])):
        assert_within(t, ref[name], torch.float32, name)
    assert torch.equal(y[1], torch.zeros_like(y[1])) and torch.equal(h[1], state[1])
    with torch.no_grad():
        assert torch.equal(F.gate_loop(leaves[0] if fused else tuple(leaves), state=state, lengths=lengths, resets=resets), y)
    # only one of the two results used, and no state at all
    y = F.gate_loop(leaves[0] if fused else tuple(leaves))
    torch.autograd.grad(y.sum(), leaves)
    _, h = F.gate_loop(leaves[0] if fused else tuple(leaves), return_state=True)
    g = torch.autograd.grad(h.sum(), leaves)
    assert all(torch.isfinite(t).all() for t in g)


def test_step_continues_a_prefix(emulated):
    qkva = rnd(2, 5, 3 * 4)
    y, h = F.gate_loop(qkva, return_state=True)
    state = torch.zeros(2, 4)
    for t in range(4):
        assert torch.allclose(F.gate_loop_step(qkva[:, t], state), y[:, t], rtol=1e-6, atol=1e-6)
    other = torch.empty_like(state)
    F.gate_loop_step(tuple(qkva[:, 4].split(4, -1)), state, state_out=other)
    assert torch.allclose(other, h, rtol=1e-6, atol=1e-6) and not torch.equal(other, state)


def test_empty_calls(emulated):
    y, h = F.gate_loop(torch.zeros(2, 0, 12), return_state=True)
    assert y.shape == (2, 0, 4) and torch.equal(h, torch.zeros(2, 4))
    s = rnd(2, 4)
    assert torch.equal(F.gate_loop(torch.zeros(2, 0, 12), state=s, return_state=True)[1], s)
    y, h = F.gate_loop(torch.zeros(0, 3, 12), return_state=True)
    assert y.shape == (0, 3, 4) and h.shape == (0, 4)
    out, n = F.block_norm(torch.zeros(0, 8), torch.zeros(0, 8), pre_gamma=torch.ones(8))
    assert out.shape == n.shape == (0, 8)


@pytest.mark.parametrize('parts', [dict(), dict(gate=1), dict(post=1), dict(scale=1), dict(pre=1), dict(gate=1, post=1, scale=1, pre=1), dict(branch=0, pre=1)])
def test_block_norm_plumbing(emulated, parts):
    R, C = 6, 5
    shape = (2, 3, C)
    has = lambda k: bool(parts.get(k, k == 'branch'))
    t = {k: rnd(*(shape if k in ('x', 'branch', 'gate') else (C,)), seed=i).requires_grad_()
         for i, k in enumerate(('x', 'branch', 'gate', 'post', 'scale', 'pre')) if k == 'x' or has(k)}
    out, n = F.block_norm(t['x'], t.get('branch'), gate=t.get('gate'), post_gamma=t.get('post'), scale=t.get('scale'), pre_gamma=t.get('pre'))
    rows = {k: v.reshape(R, C) if v.dim() == 3 else v for k, v in t.items()}
    outs = [v for v in (out if has('branch') else None, n) if v is not None]
    ups = [rnd(*shape, seed=9 + i) for i in range(len(outs))]
    up = dict(zip([k for k, v in (('dout', has('branch')), ('dn', n is not None)) if v], [u.reshape(R, C) for u in ups]))
    ref = block_norm_ref(rows['x'], rows.get('branch'), rows.get('gate'), 'silu', rows.get('post'), rows.get('scale'), rows.get('pre'), grads=True, **up)
    if not has('branch'):
        assert out is t['x']
    for v, name in zip(outs, [k for k in ('out', 'normed') if k in ref]):
        assert_within(v, ref[name], torch.float32, name)
    grads = torch.autograd.grad(outs, list(t.values()), ups)
    for k, g in zip(t, grads):
        assert_within(g, ref['d' + k], torch.float32, 'd' + k)
    with torch.no_grad():
        o2, n2 = F.block_norm(t['x'], t.get('branch'), gate=t.get('gate'), post_gamma=t.get('post'), scale=t.get('scale'), pre_gamma=t.get('pre'))
    assert torch.equal(o2, out) and (n is None or torch.equal(n2, n))


def test_bf16_parameters_get_bf16_gradients(emulated):
    x, w = rnd(4, 8).requires_grad_(), torch.ones(8, dtype=torch.bfloat16, requires_grad=True)
    F.block_norm(x, pre_gamma=w)[1].sum().backward()
    assert w.grad.dtype == torch.bfloat16


@pytest.mark.parametrize('fused', [True, False])
def test_saved_tensors_laid_out_anew(emulated, fused):
    """hooks on saved tensors give back copies of another layout than the views that were saved"""
    B, T, C = 2, 5, 4
    wide, up = rnd(T, B, 3 * C + 3).requires_grad_(), rnd(B, T, C, seed=1)
    rows, w = rnd(6, 3 * C, seed=2).requires_grad_(), torch.ones(C, requires_grad=True)
    grads = []
    for hooks in (False, True):
        ctx = torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t) if hooks else contextlib.nullcontext()
        with ctx:
            z = wide.transpose(0, 1)[..., 2:2 + 3 * C]
            y = F.gate_loop(z if fused else z.split(C, -1))
            q, kv, a = rows.split(C, -1)
            out, n = F.block_norm(q, kv, gate=a, post_gamma=w, pre_gamma=w)
        grads.append(torch.autograd.grad((y, out, n), (wide, rows, w), (up, torch.ones_like(out), rnd(6, C, seed=3))))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_a_step_over_a_saved_state_is_noticed(emulated):
    q, s = rnd(2, 3, 12).requires_grad_(), torch.ones(2, 4)
    y = F.gate_loop(q, state=s)
    F.gate_loop_step(rnd(2, 12, seed=1), s)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_refusals(emulated):
    q = rnd(2, 4, 12)
    bad = ValueError
    for call in (lambda: F.gate_loop(rnd(2, 4, 13)), lambda: F.gate_loop(rnd(4, 12)), lambda: F.gate_loop((q, q)), lambda: F.gate_loop((q, q, q[:, :3])),
                 lambda: F.gate_loop('qkva'), lambda: F.gate_loop(q, state=rnd(2, 5)), lambda: F.gate_loop(q, state=rnd(2, 4).double()),
                 lambda: F.gate_loop(q, lengths=torch.ones(3, dtype=torch.int32)), lambda: F.gate_loop(q, lengths=torch.ones(2)),
                 lambda: F.gate_loop(q, resets=torch.zeros(2, 3, dtype=torch.bool)), lambda: F.gate_loop(q, resets=torch.zeros(2, 4)),
                 lambda: F.gate_loop_step(q, rnd(2, 4)[:, :3]), lambda: F.gate_loop_step(q[:, 0], rnd(4, 2).t()),
                 lambda: F.gate_loop_step(q[:, 0].clone().requires_grad_(), rnd(2, 4)),
                 lambda: F.gate_loop_step(q[:, 0], rnd(2, 4), state_out=rnd(2, 4).double())):
        with pytest.raises(bad):
            call()
    pool = rnd(12)
    with pytest.raises(bad):
        F.gate_loop_step(q[:, 0], pool[:8].view(2, 4), state_out=pool[4:].view(2, 4))
    x, g = rnd(3, 8), torch.ones(8)
    for call in (lambda: F.block_norm(x), lambda: F.block_norm(x, gate=x, pre_gamma=g), lambda: F.block_norm(x, scale=g, pre_gamma=g),
                 lambda: F.block_norm(x, x[:2]), lambda: F.block_norm(x, x.double()), lambda: F.block_norm(x, x, gate=x, gate_act='gelu'),
                 lambda: F.block_norm(x, x, pre_gamma=torch.ones(7)), lambda: F.block_norm(x, x, scale=torch.ones(8, dtype=torch.int32))):
        with pytest.raises(bad):
            call()
    for call in (lambda: F.gate_loop(q.half()), lambda: F.block_norm(x.double(), pre_gamma=g), lambda: F.block_norm(rnd(1, 16385), pre_gamma=torch.ones(16385))):
        with pytest.raises(NotImplementedError):
            call()


def test_no_cpu_path(monkeypatch):
    monkeypatch.setattr(F, '_plans', {})
    with pytest.raises(Mv2Error):
        F.gate_loop(rnd(1, 2, 6))
    with pytest.raises(Mv2Error):
        F.block_norm(rnd(2, 4), pre_gamma=torch.ones(4))


def test_abi_refuses_before_any_launch():
    lib = ops_hip.load_library()
    buf = ctypes.create_string_buffer(4096)
    ptr = ctypes.cast(buf, ctypes.c_void_p)
    L = lambda **kw: ops_hip.GateLoopDesc(**{**dict(dtype=0, B=2, T=4, P=1, C=8, in_b=96, in_t=24, in_p=24, grad_b=96, grad_t=24, grad_p=24), **kw})

    def fwd(d, q=ptr, y=ptr):
        return lib.mv2_gateloop_forward(ctypes.byref(d), q, ptr, ptr, None, None, None, y, None, None, None, 0, None)

    def bwd(d, q=ptr, st=ptr, ws=0):
        return lib.mv2_gateloop_backward(ctypes.byref(d), q, ptr, ptr, None, None, None, st, ptr, None, ptr, ptr, ptr, None, None, ws, None)
    for kw in (dict(dtype=2), dict(B=0), dict(T=-1), dict(P=0), dict(C=0), dict(in_t=-1), dict(grad_b=-5)):
        assert fwd(L(**kw)) == EINVAL and bwd(L(**kw)) == EINVAL, kw
        assert lib.mv2_gateloop_states(ctypes.byref(L(**kw))) == EINVAL
    for kw in (dict(C=1 << 25), dict(T=(1 << 30) + 1), dict(B=1 << 30, P=1 << 30), dict(in_t=1 << 61)):
        assert fwd(L(**kw)) == ETOOLARGE, kw
    assert fwd(L(), q=None) == EINVAL and fwd(L(), y=None) == EINVAL and bwd(L(), q=None) == EINVAL
    assert lib.mv2_gateloop_forward(None, ptr, ptr, ptr, None, None, None, ptr, None, None, None, 0, None) == EINVAL
    long = L(T=100000)
    assert lib.mv2_gateloop_states(ctypes.byref(long)) > 0 and bwd(long, st=None, ws=1 << 40) == EINVAL          # a backward pass needs the kept states
    need = lib.mv2_gateloop_workspace_bytes(ctypes.byref(long), 0)
    assert need > 0 and fwd(long) == EWORKSPACE and bwd(long) == EWORKSPACE                                       # spans meet in a workspace
    N = lambda **kw: ops_hip.BlockNormDesc(**{**dict(dtype=0, C=8, rows=4, x_stride=8, branch_stride=8, gate_stride=8, gate_act=2, reserved=0), **kw})

    def nf(d, x=ptr, b=ptr, g=ptr, post=ptr, sc=ptr, pre=ptr, out=ptr, n=ptr):
        return lib.mv2_block_norm_forward(ctypes.byref(d), x, b, g, post, sc, pre, out, n, None, None)

    def nb(d, x=ptr, b=ptr, g=ptr, post=ptr, sc=ptr, pre=ptr, rstd=ptr, dn=ptr, dg=ptr, cols=ptr, ws=None, nws=0):
        return lib.mv2_block_norm_backward(ctypes.byref(d), x, b, g, post, sc, pre, rstd, ptr, dn, ptr, ptr, dg, cols, cols, cols, ws, nws, None)
    for kw in (dict(dtype=3), dict(C=0), dict(rows=-1), dict(gate_act=1), dict(reserved=1), dict(x_stride=-8)):
        assert nf(N(**kw)) == EINVAL and nb(N(**kw)) == EINVAL, kw
    for kw in (dict(C=16385), dict(rows=1 << 41), dict(gate_stride=1 << 21)):
        assert nf(N(**kw)) == ETOOLARGE, kw
    assert nf(N(), x=None) == EINVAL and nf(N(), out=None) == EINVAL and nf(N(), n=None) == EINVAL
    assert nf(N(), b=None) == EINVAL and nf(N(), b=None, g=None, post=None, sc=None, pre=None) == EINVAL
    assert nb(N(), rstd=None) == EINVAL and nb(N(), g=None) == EINVAL and nb(N(), pre=None) == EINVAL
    assert nb(N()) == EWORKSPACE and nb(N(), ws=ptr, nws=16) == EWORKSPACE
    assert lib.mv2_block_norm_workspace_bytes(ctypes.byref(N())) > 0 and lib.mv2_block_norm_workspace_bytes(ctypes.byref(N(C=0))) == 0


def test_native_keys_tell_apart_what_the_plain_ones_do():
    native, plain = ops_hip.load_calls().key, F._key
    t = rnd(3, 4)
    calls = [('loop', a, b, None) for b in (None, t, t.double(), t.t(), t[:, :2], t[None], t[0], t.expand(2, 3, 4), t.new_empty(0, 4))
             for a in (t, (t, t), (t, t, t), (t, t, None), 'silu', None)] + [('loopt', t), ('loop', 't'), ('loop',), ('', 'loop')]
    for a in calls:
        for b in calls:
            assert (native(*a) == native(*b)) == (plain(*a) == plain(*b)), (a, b)
    assert native('norm', rnd(3, 4, seed=9)) == native('norm', t) and native('loop', [t, t]) == native('loop', (t, t))
    for bad in (3, t.to_sparse(), object(), [[t]]):
        assert native('loop', bad) is None


def native_plans(B=2, C=4):
    """plans of a token's step / a call of one token and of norms, as functional.py makes them, and the functions that take them"""
    calls = ops_hip.load_calls()
    d = ops_hip.GateLoopDesc(dtype=1, B=B, T=1, P=1, C=C, in_b=3 * C, in_t=0, in_p=0, grad_b=3 * C, grad_t=3 * C, grad_p=3 * C)
    e = ops_hip.BlockNormDesc(dtype=1, C=C, rows=B, x_stride=C, branch_stride=C, gate_stride=C, gate_act=2, reserved=0)
    loop = calls.loop_plan(bytes(d), True, 0, (B, 3 * C), (B, C), (B, C), (), (3 * C, 1), 0, 0)
    norm = calls.norm_plan(bytes(e), 0, (B, C), True, True, True, (C, 1), (C, 1), (C, 1), 0)
    return calls.loop_forward, loop, calls.norm_forward, norm


def test_tangents_are_refused_before_anything_is_launched():
    """an input with a tangent but without requires_grad: neither operator has a forward-mode derivative, and none may be left out in silence"""
    loop_forward, loop, norm_forward, norm = native_plans()
    z, s, x, w = rnd(2, 12), rnd(2, 4, seed=1), rnd(2, 4, seed=2), torch.ones(4)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        for args in ((dual(z), s, None), (z, dual(s), None), (z, s, dual(rnd(2, 4)))):
            for want in (0, 1, 2):
                with pytest.raises(NotImplementedError):
                    loop_forward(loop, args[:1], args[1], None, None, args[2], want)
        args = (x, x, x, w, w, w)
        for i in range(6):
            for train in (False, True):
                with pytest.raises(NotImplementedError):
                    norm_forward(norm, *args[:i], dual(args[i]), *args[i + 1:], train)


@pytest.mark.parametrize('shape', [(0, 3, 2), (0, 3), (2, 3, 0), (0, 0)])
@pytest.mark.parametrize('fused', [True, False])
def test_an_empty_batch_keeps_its_graph(emulated, shape, fused):
    """no sequences (B = 0 or no pixels): gradients of nothing reach every input, and what lies behind them zeros, as with torch's operators"""
    C, w = 4, rnd(5, 12, seed=1).requires_grad_()
    z = torch.zeros(*shape, 5) @ w
    parts = z.split(C, -1)
    s = torch.zeros(*shape[:1], *shape[2:], C, requires_grad=True)
    y, h = F.gate_loop(z if fused else tuple(parts), state=s, return_state=True)
    assert y.shape == (*shape, C) and h.shape == s.shape and y.dtype == z.dtype and h.dtype == torch.float32
    for outs in ((y, h), (y,), (h,)):
        got = torch.autograd.grad([o.sum() for o in outs], [s, w, *((z,) if fused else parts)], retain_graph=True)
        assert not any(g.any() for g in got) and got[0].shape == s.shape
    half = F.gate_loop(z.detach().bfloat16().requires_grad_(), state=s, return_state=True)
    assert half[0].dtype == torch.bfloat16 and half[0].requires_grad and half[1].dtype == torch.float32 and half[1].requires_grad
    with torch.no_grad():
        assert not F.gate_loop(z, state=s).requires_grad
    assert not F.gate_loop(z.detach()).requires_grad


def test_keys_tell_lazily_negated_tensors_apart():
    native, t = ops_hip.load_calls().key, rnd(3, 4)
    for key in (native, F._key):
        assert key('norm', torch._neg_view(t)) != key('norm', t) and key('loop', (t, torch._neg_view(t), t)) != key('loop', (t, t, t))


def test_a_forward_pass_whose_backward_pass_is_too_long_is_refused():
    """one sequence of 150 million tokens: served forward (as far as the launch), but its backward pass would have more workgroups than a launch can"""
    lib, ptr = ops_hip.load_library(), ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)
    T, C = 150_000_000, 8
    d = ops_hip.GateLoopDesc(dtype=0, B=1, T=T, P=1, C=C, in_b=0, in_t=3 * C, in_p=0, grad_b=0, grad_t=3 * C, grad_p=0)
    fwd = lambda states: lib.mv2_gateloop_forward(ctypes.byref(d), ptr, ptr, ptr, None, None, None, ptr, None, states, None, 0, None)
    assert lib.mv2_gateloop_backward(ctypes.byref(d), *[ptr] * 3, None, None, None, ptr, ptr, None, *[ptr] * 3, None, None, 0, None) == ETOOLARGE
    assert fwd(ptr) == ETOOLARGE and fwd(None) == EWORKSPACE


def test_calls_of_another_torch_are_built_anew_and_never_used(monkeypatch, tmp_path):
    """_calls.so holds torch's C++ interface as it was when it was built: after torch is replaced it is stale, whatever its age, and is not loaded"""
    from magvit2_pytorch_amd import build
    stamp = tmp_path / 'calls.for'
    stamp.write_text(build._interfaces())
    with monkeypatch.context() as m:
        m.setattr(build, '_stale', lambda *a: False)
        m.setattr(build, 'CALLS_FOR', str(stamp))
        assert not build._calls_stale()
        m.setattr(torch, '__version__', '9.9.9')
        assert build._calls_stale()
        m.setattr(ops_hip, '_calls', None)
        with pytest.raises(Mv2Error, match='9.9.9'):
            ops_hip.load_calls()
    broken = tmp_path / '_calls.so'
    broken.write_bytes(b'not a library')
    with monkeypatch.context() as m:
        m.setattr(ops_hip, '_calls', None)
        m.setattr(ops_hip, 'CALLS_PATH', str(broken))
        with pytest.raises(Mv2Error, match='does not load'):
            ops_hip.load_calls()
    assert ops_hip.load_calls().built_for == build._interfaces()


def test_the_library_is_built_without_the_calls(monkeypatch, tmp_path):
    """no g++ here: only functional.py needs it, so the build goes on, says so, and leaves no older calls behind"""
    from magvit2_pytorch_amd import build
    old = [tmp_path / n for n in ('_calls.so', 'calls.for')]
    for f in old:
        f.write_text('older')
    monkeypatch.setattr(build, 'CALLS', str(old[0]))
    monkeypatch.setattr(build, 'CALLS_FOR', str(old[1]))
    monkeypatch.setattr(build, '_stale', lambda target, deps: target == str(old[0]))
    monkeypatch.setattr(build, 'CXX', str(tmp_path / 'no-such-compiler'))
    with pytest.warns(UserWarning, match='functional'):
        assert build.build(verbose=False) == build.LIB
    assert not any(f.exists() for f in old)


def test_sizes_beyond_the_descriptors_are_refused(emulated):
    """sizes that leave 32 bits (a view that repeats a row has them without the memory) are refused, not taken modulo 2^32"""
    z = torch.zeros(1, 1, 1, 6)
    for shape in ((1, (1 << 32) + 5, 1, 6), ((1 << 32) + 1, 1, 1, 6), (1, 1, (1 << 32) + 2, 6), (1, 1 << 31, 1, 6), (1, (1 << 30) + 1, 1, 6)):
        with pytest.raises(NotImplementedError):
            F._plan_loop('gate_loop', z.expand(shape), True, None, None, None)
    with pytest.raises(NotImplementedError):
        F._plan_loop('gate_loop', (z[..., :1].expand(1, 1, 1, (1 << 32) + 8),) * 3, True, None, None, None)
    assert F._plan_loop('gate_loop', z.expand(1, 1 << 30, 1, 6), True, None, None, None).desc.T == 1 << 30


def test_sparse_arguments_are_refused(emulated):
    z, s, x, w = rnd(2, 4, 12), rnd(2, 4), rnd(3, 8), torch.ones(8)
    for call in (lambda: F.gate_loop(z.to_sparse()), lambda: F.gate_loop(z, state=s.to_sparse()), lambda: F.gate_loop(z, lengths=torch.ones(2, dtype=torch.int32).to_sparse()),
                 lambda: F.gate_loop((z, z, z.to_sparse())), lambda: F.gate_loop_step(z[:, 0], s.to_sparse()), lambda: F.block_norm(x.to_sparse(), pre_gamma=w),
                 lambda: F.block_norm(x, x.to_sparse_csr()), lambda: F.block_norm(x, pre_gamma=w.to_sparse())):
        with pytest.raises(ValueError):
            call()
