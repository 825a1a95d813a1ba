"""
Differentiable sequence operators over the C ABI (include/mv2.h): the gated linear recurrence of the ``gateloop_time`` layer in its
general form, and the norms around a residual block with the block's gate and scale.

    y, state = gate_loop(qkva, state=state, lengths=lengths, resets=resets, return_state=True)     # any length, trainable
    y = gate_loop_step(qkva, state)                                                               # one token, state updated in place
    x, n = block_norm(x, y, gate=gate, post_gamma=g1, scale=s, pre_gamma=g2)                      # close one block, open the next

The reference reaches the recurrence through a third-party layer (magvit2_pytorch.py:1216-1222, its RMSNorm :258-276, its Residual :167-174)
and differentiates it with autograd; ``VideoTokenizer``'s own ``gateloop_time`` layers keep their fused scan (``mv2_gateloop_scan``).

Tensors live on one HIP device; bf16 or fp32 rows, fp32 states and parameters.  Calls enqueue on the current stream of that device, allocate
their outputs and workspaces from torch's allocator and can be captured into a HIP graph.  As with every torch operator, a tensor that was
made on another stream must be ordered and recorded (``record_stream``) by the caller.  There is no CPU path: CPU tensors raise ``Mv2Error``.
Gradients are first order and backward mode: inputs or gradients with tangents (forward mode) are refused.  To capture a backward pass, capture the forward pass that belongs to it in the same graph (torch ties the
gradient nodes of a leaf to the stream of its first use: a leaf that an eager graph still holds must not be captured).
"""
from __future__ import annotations

import torch

from .ops_hip import BlockNormDesc, GateLoopDesc, HipOps, Mv2Error, load_calls

__all__ = ['gate_loop', 'gate_loop_step', 'block_norm']

_DTYPES = {torch.bfloat16: 0, torch.float32: 1}
_ACTS = {'none': 0, 'silu': 2, 'sigmoid': 5}
_backends = {}                       # device -> launcher (tests put the kernel emulation here for the CPU)
_plans = {}                          # shapes, strides, types, devices and marks of a call's arguments -> what follows from them
_MAX_PLANS = 1024


def _ops(device):
    ops = _backends.get(device)
    if ops is None:
        if device.type != 'cuda':
            raise Mv2Error(f'tensors on {device}: these operators run on a HIP device and have no CPU fallback')
        ops = _backends[device] = HipOps(device)
        global _key
        _key = load_calls().key
    return ops


def _need(cond, what):
    if not cond:
        raise ValueError(what)


def _strided(name, *args):
    _need(all(t.layout is torch.strided for t in args if isinstance(t, torch.Tensor)), f'{name}: sparse tensors are not taken')


def _row_dtype(t, name):
    if t.dtype not in _DTYPES:
        raise NotImplementedError(f'{name}: rows of {t.dtype}; bf16 and fp32 are built')
    return _DTYPES[t.dtype]


def _key(*args):
    """what a plan depends on: shapes, strides, types, devices and lazy negations; None where arguments are not tensors (the plan says what is wrong).  On a HIP
    device the native form of this takes its place (csrc/calls.cpp)"""
    like = lambda t: t if t is None or isinstance(t, str) else (t.shape, t.stride(), t.dtype, t.device, t.is_neg())
    try:
        return tuple(tuple(map(like, a)) if isinstance(a, (tuple, list)) else like(a) for a in args)
    except (AttributeError, TypeError, RuntimeError):     # (sparse tensors have no strides)
        return None


def _plan(key, make, *args):
    """the plan of a call: arguments that look alike (never: that are the same) are checked once"""
    plan = _plans.get(key) if key is not None else None
    if plan is None:
        plan = make(*args)
        if key is not None:
            if len(_plans) >= _MAX_PLANS:
                _plans.clear()
            _plans[key] = plan
    return plan


def _dense(t):
    return t if t.is_contiguous() else t.contiguous()


def _copied(t):
    """dense, and with the sign that a lazily negated tensor (the imaginary part of a conjugate) only carries as a mark"""
    return t if t is None else t.resolve_neg().contiguous()


# ----------------------------------------------------------------------------------------------------------------- gated recurrence
class _LoopPlan:
    """what follows from the arguments' shapes, strides and types"""
    __slots__ = ('ops', 'desc', 'fused', 'copy', 'empty', 'T', 'C', 'stride', 'part_shape', 'y_shape', 'h_shape', 'states_shape', 'ws_forward',
                 'ws_backward', 'native', 'forward')


def _plan_loop(name, qkva, tokens, state, lengths, resets):
    plan = _LoopPlan()
    fused = plan.fused = isinstance(qkva, torch.Tensor)
    parts = (qkva,) if fused else qkva
    _need(fused or (isinstance(qkva, (tuple, list)) and len(qkva) == 3 and all(isinstance(t, torch.Tensor) for t in qkva)),
          f'{name}: expected a tensor [q | kv | a] or the three tensors (q, kv, a)')
    _strided(name, *parts, state, lengths, resets)
    first = parts[0]
    rank = 3 if tokens else 2
    shape, dev = first.shape, first.device
    _need(len(shape) in (rank, rank + 1), f'{name}: expected {"(B, T[, P], C)" if tokens else "(B[, P], C)"} tensors, got {tuple(shape)}')
    if fused:
        _need(shape[-1] % 3 == 0 and shape[-1] > 0, f'{name}: the last axis holds [q | kv | a], three equal parts; got {shape[-1]}')
        C = shape[-1] // 3
    else:
        _need(all(t.shape == shape and t.dtype == first.dtype and t.device == dev for t in parts), f'{name}: q, kv and a differ in shape, type or device')
        C = shape[-1]
        _need(C > 0, f'{name}: no channels')
    dtype = _row_dtype(first, name)
    B, T = shape[0], shape[1] if tokens else 1
    pixels = len(shape) == rank + 1
    P = shape[rank - 1] if pixels else 1
    if max(B, T, P, C) > 1 << 30:                         # descriptors hold 32 bits
        raise NotImplementedError(f'{name}: {B} samples, {T} tokens, {P} pixels, {C} channels; up to 2^30 of each are built')
    h_shape = (B, P, C) if pixels else (B, C)
    if state is not None:
        _check_state(state, h_shape, dev, name)
    if lengths is not None:
        _need(isinstance(lengths, torch.Tensor) and tuple(lengths.shape) == (B,) and lengths.dtype in (torch.int32, torch.int64) and lengths.device == dev,
              f'{name}: lengths must be int32 / int64 ({B},) on {dev}')
    if resets is not None:
        _need(isinstance(resets, torch.Tensor) and tuple(resets.shape) == (B, T) and resets.dtype in (torch.bool, torch.uint8) and resets.device == dev,
              f'{name}: resets must be bool / uint8 {(B, T)} on {dev}')
    plan.ops = _ops(dev)
    plan.T, plan.C, plan.part_shape, plan.y_shape, plan.h_shape = T, C, tuple(shape), tuple(shape[:-1]) + (C,), h_shape
    plan.empty = B * P == 0                               # no sequences: nothing to launch
    if plan.empty:
        return plan
    plan.copy = (first.stride(-1) != 1 and shape[-1] > 1) or any(t.stride() != first.stride() for t in parts) or \
        any(t is not None and t.is_neg() for t in (*parts, state))
    st = plan.stride = torch.empty(shape, device='meta').stride() if plan.copy else first.stride()
    row = (3 if fused else 1) * C                         # gradients: one dense (B, T, P, 3C) tensor, or three dense ones
    plan.desc = GateLoopDesc(dtype=dtype, B=B, T=T, P=P, C=C, in_b=st[0] if B > 1 else 0, in_t=st[1] if tokens and T > 1 else 0,
                             in_p=st[rank - 1] if P > 1 else 0, grad_b=T * P * row, grad_t=P * row, grad_p=row)
    states, plan.ws_forward, plan.ws_backward = plan.ops.gateloop_sizes(plan.desc)
    plan.states_shape = (B, states, P, C) if states else None
    plan.native, plan.forward = plan.ops.loop_plan(plan)
    return plan


def _check_state(state, shape, device, name, what='state'):
    _need(isinstance(state, torch.Tensor) and tuple(state.shape) == shape, f'{name}: {what} must be a tensor of shape {shape}')
    _need(state.dtype == torch.float32, f'{name}: {what} is {state.dtype}; states are fp32')
    _need(state.device == device, f'{name}: {what} is on {state.device}, the rows on {device}')


def gate_loop(qkva, *, state=None, lengths=None, resets=None, return_state=False):
    """Gated linear recurrence ``h_t = sigmoid(a_t) h_{t-1} + kv_t``, ``y_t = q_t h_t`` along the tokens, per sample, pixel and channel.

    ``qkva``: ``(B, T, 3C)`` or ``(B, T, P, 3C)``, the projections [q | kv | a] side by side, or the three ``(B, T[, P], C)`` tensors
    ``(q, kv, a)``; bf16 or fp32; any strides.  ``state``: fp32 ``(B[, P], C)``, the state before the first token (default: empty).
    ``lengths``: ``(B,)`` int32 / int64, tokens per sample in a padded batch (values are taken into ``[0, T]``): ``y`` and the gradients are zero
    behind them, whatever the rows hold there, and the last state is the one behind the last token that exists.  ``resets``: ``(B, T)`` bool /
    uint8, tokens that start a new document: no state and no gradient crosses them.
    An infinite state stays infinite while decays are above zero (``a`` above about -87) and is NaN behind a decay of zero; a document start ends it.
    Returns ``y`` (``(B, T[, P], C)``, dense), with ``return_state`` also the last state.  Gradients reach ``qkva`` and ``state``."""
    fused = isinstance(qkva, torch.Tensor)
    plan = _plan(_key('loop', qkva, state, lengths, resets), _plan_loop, 'gate_loop', qkva, True, state, lengths, resets)
    leaves = (qkva,) if fused else tuple(qkva)
    if plan.empty:
        return _empty_loop(plan, leaves, state, return_state)
    if plan.copy:
        leaves, state = tuple(map(_copied, leaves)), _copied(state)
    if state is not None:
        state = _dense(state)
    if lengths is not None:
        lengths = _dense(lengths if lengths.dtype == torch.int32 else lengths.clamp(0, plan.T).to(torch.int32))
    if resets is not None:
        resets = _dense(resets)
    train = torch.is_grad_enabled() and (any(t.requires_grad for t in leaves) or (state is not None and state.requires_grad))
    y, h = plan.forward(plan.native, leaves, state, lengths, resets, None, 2 if train else 1 if return_state else 0)
    return (y, h) if return_state else y


def _empty_loop(plan, leaves, state, return_state):
    """results without an element, tied to every input as those of the kernels are: a training step passes through a batch of no sequences"""
    q, kv, a = leaves[0].split(plan.C, -1) if plan.fused else leaves
    y = q + kv + a
    if state is not None:
        y = y + state.unsqueeze(1).to(y.dtype)
    return (y, y.sum(1, dtype=torch.float32)) if return_state else y


def gate_loop_step(qkva, state, *, state_out=None):
    """One token of ``gate_loop``: ``qkva`` ``(B[, P], 3C)`` or ``(q, kv, a)`` of ``(B[, P], C)``, ``state`` dense fp32 ``(B[, P], C)``.  The new state is
    written over ``state``, or into ``state_out`` (dense fp32, the same shape; apart from ``state``, or ``state`` itself).  Returns ``y`` ``(B[, P], C)``.
    For inference: it has no gradient."""
    fused = isinstance(qkva, torch.Tensor)
    plan = _plan(_key('step', qkva, state, state_out), _plan_step, qkva, state, state_out)
    parts = (qkva,) if fused else tuple(qkva)
    if torch.is_grad_enabled():
        _need(not (state.requires_grad or (state_out is not None and state_out.requires_grad) or any(t.requires_grad for t in parts)),
              'gate_loop_step has no gradient (it updates the state in place): use gate_loop, or torch.no_grad()')
    if state_out is None:
        state_out = state
    else:
        apart = abs(state_out.data_ptr() - state.data_ptr())
        _need(apart == 0 or apart >= 4 * state.numel(), 'gate_loop_step: state_out overlaps state')
    if plan.empty:
        return parts[0].new_empty(plan.y_shape)
    if plan.copy:
        parts = tuple(map(_copied, parts))
    y = plan.forward(plan.native, parts, state, None, None, state_out, 0)[0]
    if not state_out.is_inference():                      # written behind autograd's back: what saved it must not use it any more
        torch.autograd.graph.increment_version(state_out)
    return y


def _plan_step(qkva, state, state_out):
    _need(isinstance(state, torch.Tensor), 'gate_loop_step: state must be a tensor')
    _strided('gate_loop_step', state_out)
    plan = _plan_loop('gate_loop_step', qkva, False, state, None, None)
    _need(state.is_contiguous() and not state.is_neg(), 'gate_loop_step: the state is updated in place and must be dense')
    if state_out is not None:
        _check_state(state_out, plan.h_shape, state.device, 'gate_loop_step', 'state_out')
        _need(state_out.is_contiguous() and not state_out.is_neg(), 'gate_loop_step: state_out must be dense')
    return plan


# ----------------------------------------------------------------------------------------------------------------- norms around a block
class _NormPlan:
    __slots__ = ('ops', 'desc', 'copy', 'cast', 'strides', 'shape', 'rows', 'branch', 'normed', 'keeps', 'ws_backward', 'native', 'forward')


def _row_stride(shape, stride):
    """elements between rows, where (..., C) is rows of C contiguous elements at one distance; None where it is not"""
    if shape[-1] > 1 and stride[-1] != 1:
        return None
    rows = [(n, s) for n, s in zip(shape[:-1], stride[:-1]) if n != 1]
    for (_, outer), (n, inner) in zip(rows, rows[1:]):
        if outer != n * inner:
            return None
    step = rows[-1][1] if rows else shape[-1]
    return step if step <= 1 << 20 else None


def _plan_norm(x, branch, gate, gate_act, *params):
    plan = _NormPlan()
    _need(isinstance(x, torch.Tensor) and x.dim() >= 1 and x.shape[-1] > 0, 'block_norm: x must have rows of at least one channel')
    _strided('block_norm', x, branch, gate, *params)
    _need(gate_act in _ACTS, f'block_norm: unknown gate_act {gate_act!r}; silu, sigmoid or none')
    C, dev = x.shape[-1], x.device
    dtype = _row_dtype(x, 'block_norm')
    if C > 16384:
        raise NotImplementedError(f'block_norm: rows of {C} channels; up to 16384 are built')
    post, scale, pre = params
    if branch is None:
        _need(gate is None and post is None and scale is None, 'block_norm: gate, post_gamma and scale act on a branch, and there is none')
        _need(pre is not None, 'block_norm: nothing to do without a branch and without pre_gamma')
    for name, t in (('branch', branch), ('gate', gate)):
        _need(t is None or (isinstance(t, torch.Tensor) and t.shape == x.shape and t.dtype == x.dtype and t.device == dev),
              f'block_norm: {name} and x differ in shape, type or device')
    for name, t in zip(('post_gamma', 'scale', 'pre_gamma'), params):
        _need(t is None or (isinstance(t, torch.Tensor) and tuple(t.shape) == (C,) and t.is_floating_point() and t.device == dev),
              f'block_norm: {name} must be a floating-point ({C},) tensor on {dev}')
    plan.ops = _ops(dev)
    plan.cast = any(t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.is_neg()) for t in params)
    steps = [None if t is None else _row_stride(t.shape, t.stride()) for t in (x, branch, gate)]
    plan.copy = any(t is not None and (s is None or t.is_neg()) for t, s in zip((x, branch, gate), steps))
    if plan.copy:
        steps = [C, C, C]
    plan.strides = None if plan.copy else tuple(None if t is None else t.stride() for t in (x, branch, gate))      # None: all dense
    plan.shape, plan.rows = tuple(x.shape), x.numel() // C
    plan.branch, plan.normed, plan.keeps = branch is not None, pre is not None, post is not None or pre is not None
    plan.desc = BlockNormDesc(dtype=dtype, C=C, rows=plan.rows, x_stride=steps[0] or 0, branch_stride=steps[1] or 0, gate_stride=steps[2] or 0,
                              gate_act=_ACTS[gate_act] if gate is not None else 0, reserved=0)
    plan.ws_backward = plan.ops.block_norm_workspace_bytes(plan.desc)
    plan.native, plan.forward = plan.ops.norm_plan(plan)
    return plan


def block_norm(x, branch=None, *, gate=None, gate_act='silu', post_gamma=None, scale=None, pre_gamma=None):
    """Closes a residual block and opens the next in one pass over the rows:

        out = x + scale * act(gate) * N(branch; post_gamma)          normed = N(out; pre_gamma)
        N(v; gamma) = v / max(|v|, 1e-12) * sqrt(C) * gamma          (the framework's RMSNorm, reference magvit2_pytorch.py:258-276)

    ``x``, ``branch``, ``gate``: ``(..., C)``, one shape, bf16 or fp32, any strides (a third of a fused projection is read where it lies);
    ``post_gamma``, ``scale``, ``pre_gamma``: ``(C,)``, computed with in fp32.  ``gate_act``: 'silu', 'sigmoid' or 'none' (the gate as it is).
    Left out: ``branch`` - no add, ``out`` is ``x``; ``post_gamma`` - the branch enters as it is; ``gate``, ``scale`` - ones; ``pre_gamma`` - no second
    norm, ``normed`` is None.  C <= 16384.  Sums of squares are fp32: N of a row with ``|v| >= 1.8e19`` is zero.
    Returns ``(out, normed)``.  Gradients reach every tensor; the parameters' are bitwise reproducible."""
    plan = _plan(_key('norm', x, branch, gate, gate_act, post_gamma, scale, pre_gamma), _plan_norm, x, branch, gate, gate_act, post_gamma, scale, pre_gamma)
    args = (x, branch, gate, post_gamma, scale, pre_gamma)
    if plan.copy:
        args = tuple(map(_copied, args[:3])) + args[3:]
    if plan.cast:
        args = args[:3] + tuple(None if t is None else _copied(t.to(torch.float32)) for t in args[3:])
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args)
    out, normed = plan.forward(plan.native, *args, train)
    return (out if plan.branch else x), normed
