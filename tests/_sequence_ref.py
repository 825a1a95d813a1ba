"""64-bit references of the sequence operators (magvit2_pytorch_amd/functional.py), token by token and row by row, each result with a bound
on how far a 32-bit evaluation may be off: running error analysis.  Every elementary operation of the kernels is off by at most
UNIT = 2^-24 of its result; the bounds count how many of them lie on the way to a value (`c` below), carried along by the same recurrence
or sum as the value itself, over the sums of ABSOLUTE values (so cancellation is allowed for).  A value stored in a narrower type adds half
a step of that type."""
import math

import torch

UNIT = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def stored(bound, value, dtype):
    """bound of a value that is rounded to dtype on its store (tiny: the smallest numbers of the type, below which steps stop shrinking)"""
    return bound * (1 + half_step(dtype)) + half_step(dtype) * value.abs() + torch.finfo(dtype).tiny


def gate_loop_ref(q, kv, a, state=None, lengths=None, resets=None, dy=None, dh=None, fast_exp=False):
    """q, kv, a (B, T, P, C), state / dh (B, P, C).  Returns {name: (value, bound)} for y, h and, with dy, dq, dkv, da, dstate.
    Operations per token on a path: the decay (exp, add, reciprocal / division: <= 6 units; the bf16 kernels' exp is exp2 of a rounded
    product: |a| units more), its product with the state, the sum, and one product and one sum more where spans of tokens are joined."""
    q, kv, a = (t.detach().double().cpu() for t in (q, kv, a))
    B, T, P, C = q.shape
    unit = UNIT * (10 + (2 * a.abs().clamp_max(90) if fast_exp else torch.zeros_like(a)))      # per decay; (B, T, P, C)
    n = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    live = torch.arange(T)[None] < n[:, None]
    cut = torch.zeros(B, T, dtype=torch.bool) if resets is None else resets.cpu().bool()
    g = torch.sigmoid(a)
    zero = torch.zeros(B, P, C, dtype=torch.float64)
    start = zero if state is None else state.detach().double().cpu()
    col = lambda m, t: m[:, t, None, None]
    h, ha, he = start, start.abs(), zero                       # state, sum of absolute values, error bound
    hs, has, hes = [], [], []
    for t in range(T):
        keep = col(cut, t).logical_not()
        mul = lambda s: torch.where(keep, g[:, t] * s, zero)
        nh, na = mul(h) + kv[:, t], mul(ha) + kv[:, t].abs()
        ne = mul(he) + mul(ha) * unit[:, t] + 4 * UNIT * na
        on = col(live, t)
        h, ha, he = torch.where(on, nh, h), torch.where(on, na, ha), torch.where(on, ne, he)
        hs.append(h); has.append(ha); hes.append(he)
    stack = lambda v: torch.stack(v, 1) if v else torch.zeros(B, 0, P, C, dtype=torch.float64)
    H, HE = stack(hs), stack(hes)
    alive = live[:, :, None, None]
    mask = lambda v: torch.where(alive, v, torch.zeros_like(v))
    out = dict(y=(mask(q * H), mask(q.abs() * HE + 2 * UNIT * (q * H).abs())), h=(h, he))
    if dy is None:
        return out
    dy = dy.detach().double().cpu()
    back = zero if dh is None else dh.detach().double().cpu()
    ba, be = back.abs(), zero
    res = {k: [None] * T for k in ('dq', 'dqe', 'dkv', 'dkve', 'da', 'dae')}
    slope = torch.sigmoid(a) * torch.sigmoid(-a)
    for t in range(T - 1, -1, -1):
        on, keep = col(live, t), col(cut, t).logical_not()
        prev, pe = (hs[t - 1], hes[t - 1]) if t else (start, zero)
        x = q[:, t] * dy[:, t]
        D, Da = back + x, ba + x.abs()
        De = be + 4 * UNIT * Da
        res['dq'][t] = hs[t] * dy[:, t]
        res['dqe'][t] = hes[t] * dy[:, t].abs() + 2 * UNIT * res['dq'][t].abs()
        res['dkv'][t], res['dkve'][t] = D, De
        da = torch.where(keep, D * prev * slope[:, t], zero)
        res['da'][t] = da
        res['dae'][t] = torch.where(keep, (De * prev.abs() + Da * pe + De * pe) * slope[:, t], zero) + (2 * unit[:, t] + 6 * UNIT) * da.abs()
        thru = lambda s: torch.where(keep, g[:, t] * s, zero)
        nb, nba, nbe = thru(D), thru(Da), thru(De) + thru(Da) * unit[:, t]
        back, ba, be = torch.where(on, nb, back), torch.where(on, nba, ba), torch.where(on, nbe, be)
    for k in ('dq', 'dkv', 'da'):
        out[k] = (mask(stack(res[k])), mask(stack(res[k + 'e'])))
    out['dstate'] = (back, be + 2 * UNIT * ba)
    return out


def block_norm_ref(x, branch=None, gate=None, act='none', post=None, scale=None, pre=None, dout=None, dn=None, grads=False):
    """rows (R, C).  Returns {name: (value, bound)} for out, normed and, with grads, dx, dbranch, dgate, dpost, dscale, dpre.
    A sum over C is formed by up to C / 64 additions per lane and 10 more between lanes: N = C / 64 + 10 units; a reciprocal norm is off by
    half of that and 4; the gate's exp and division by 6."""
    f = lambda t: None if t is None else t.detach().double().cpu()
    x, b, g, w1, s, w2, dout, dn = (f(t) for t in (x, branch, gate, post, scale, pre, dout, dn))
    R, C = x.shape
    root = math.sqrt(C)
    N = C / 64 + 10
    inv = lambda v: 1 / v.norm(dim=-1, keepdim=True).clamp_min(1e-12)
    res = {}
    out, oa = x, x.abs()
    if b is not None:
        r1 = inv(b)
        bh = b * r1 if w1 is not None else b
        rw = root * w1 if w1 is not None else 1.
        u = bh * rw
        sig = torch.sigmoid(g) if g is not None else None
        v = torch.ones_like(x) if g is None else {'none': g, 'silu': g * torch.sigmoid(g), 'sigmoid': sig}[act]
        sc = 1. if s is None else s
        out = x + sc * v * u
        oa = x.abs() + (sc * v * u).abs()
    oe = UNIT * (N / 2 + 16) * oa                             # absolute error of out before its store
    if b is not None:
        res['out'] = (out, oe)
    if w2 is not None:
        r2 = inv(out)
        o = out * r2
        # the norm's own error: |d|out|| <= |d out|
        re = oe.norm(dim=-1, keepdim=True) * r2 + UNIT * (N / 2 + 4)
        ohe = oe * r2 + o.abs() * re                          # of o
        n = o * (root * w2)
        res['normed'] = (n, (ohe + 4 * UNIT * o.abs()) * (root * w2).abs())
    if not grads:
        return res
    zero = torch.zeros_like(x)
    D = zero if dout is None else dout
    De = 2 * UNIT * D.abs()
    if w2 is not None and dn is not None:
        t = dn * (root * w2)
        free = r2 < 0.999e12                                  # below the floor of the norm, N is linear
        dot = torch.where(free, (o * t).sum(-1, keepdim=True), 0.)
        dota = torch.where(free, (o * t).abs().sum(-1, keepdim=True), 0.)
        dote = torch.where(free, (ohe * t.abs()).sum(-1, keepdim=True), 0.) + UNIT * (N + 6) * dota
        D = D + r2 * (t - o * dot)
        # o times dot is off by each of the two factors' errors
        De = De + r2 * (o.abs() * dote + ohe * dot.abs() + ohe * dote) + (re + 10 * UNIT) * r2 * (t.abs() + o.abs() * dota) + 2 * UNIT * D.abs()
        K = R / 8 + 600                                       # additions on the way of a column sum, at most
        res['dpre'] = ((dn * o * root).sum(0), (dn.abs() * (ohe + (K + 8) * UNIT * o.abs()) * root).sum(0))
    elif w2 is not None:
        res['dpre'] = (torch.zeros(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64))
    res['dx'] = (D, De)
    if b is None:
        return res
    K = R / 8 + 600
    k1 = (N / 2 + 12) * UNIT if w1 is not None else 4 * UNIT  # of b times r1
    if g is not None:
        slope = {'none': torch.ones_like(x), 'silu': sig * (1 + g * (1 - sig)), 'sigmoid': sig * torch.sigmoid(-g)}[act]
        sla = {'none': torch.ones_like(x), 'silu': sig * (1 + g.abs() * torch.sigmoid(-g)), 'sigmoid': slope}[act]      # silu's slope is a difference
        res['dgate'] = (D * sc * u * slope, De * (sc * u * slope).abs() + (k1 + 24 * UNIT) * (D * sc * u).abs() * sla)
    db, dbe = D * sc * v, (De + 14 * UNIT * D.abs()) * (sc * v).abs()
    if s is not None:
        res['dscale'] = ((D * v * u).sum(0), ((De + (k1 + (K + 20) * UNIT) * D.abs()) * (v * u).abs()).sum(0))
    if w1 is None:
        res['dbranch'] = (db, dbe)
        return res
    res['dpost'] = ((db * bh * root).sum(0), ((dbe + (k1 + (K + 8) * UNIT) * db.abs()) * bh.abs() * root).sum(0))
    t, te = db * rw, (dbe + 4 * UNIT * db.abs()) * rw.abs()
    free = r1 < 0.999e12
    dot = torch.where(free, (bh * t).sum(-1, keepdim=True), 0.)
    dota = torch.where(free, (bh * t).abs().sum(-1, keepdim=True), 0.)
    dote = torch.where(free, (bh.abs() * te).sum(-1, keepdim=True), 0.) + (k1 + UNIT * (N + 6)) * dota
    val = r1 * (t - bh * dot)
    res['dbranch'] = (val, r1 * (te + bh.abs() * dote + (2 * k1 + 10 * UNIT) * (t.abs() + bh.abs() * dot.abs())) + 2 * UNIT * val.abs())
    return res


def assert_within(got, ref, dtype, what):
    """got against (value, bound); prints the worst ratio of error to bound on failure"""
    value, bound = ref
    got = got.detach().double().cpu().reshape(value.shape)
    lim = stored(bound, value, dtype)
    err = (got - value).abs()
    bad = ~(err <= lim)                                       # NaN is bad
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} off; first at {i}: got {got[i].item()!r}, expected {value[i].item()!r} +- {lim[i].item():.3e}')
