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
Gradients are first order.  To capture a backward pass, capture the forward pass that belongs to it in the same graph (torch ties the
gradient nodes of a leaf to the stream of its first use: a leaf that an eager graph still holds must not be captured).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .ops_hip import BlockNormDesc, GateLoopDesc, HipOps, Mv2Error

__all__ = ['gate_loop', 'gate_loop_step', 'block_norm']

_DTYPES = {torch.bfloat16: 0, torch.float32: 1}
_ACTS = {'none': 0, 'silu': 2, 'sigmoid': 5}
_backends = {}                       # device -> launcher (tests put the kernel emulation here for the CPU)
_geometries = {}                     # sizes and strides -> filled descriptor and buffer sizes (a function of the shapes alone)
_MAX_GEOMETRIES = 512


def _ops(device):
    ops = _backends.get(device)
    if ops is None:
        if device.type != 'cuda':
            raise Mv2Error(f'tensors on {device}: these operators run on a HIP device and have no CPU fallback')
        ops = _backends[device] = HipOps(device)
    return ops


def _launch(ops, step):
    """on the current stream of the operator's device, which need not be the current device"""
    if ops.device.type == 'cuda' and ops.device.index != torch.cuda.current_device():
        with torch.cuda.device(ops.device):
            step(ops.current_stream())
    else:
        step(ops.current_stream())


def _need(cond, what):
    if not cond:
        raise ValueError(what)


def _row_dtype(t, name):
    if t.dtype not in _DTYPES:
        raise NotImplementedError(f'{name}: rows of {t.dtype}; bf16 and fp32 are built')
    return _DTYPES[t.dtype]


def _bytes(ops, n):
    return ops.empty((n,), torch.uint8) if n else None


# ----------------------------------------------------------------------------------------------------------------- gated recurrence
class _LoopGeometry:
    __slots__ = ('desc', 'B', 'T', 'P', 'C', 'states', 'ws_forward', 'ws_backward')


def _loop_geometry(ops, dtype, dims, strides, fused):
    key = (ops.device, dtype, dims, strides, fused)
    geo = _geometries.get(key)
    if geo is None:
        if len(_geometries) >= _MAX_GEOMETRIES:
            _geometries.clear()
        B, T, P, C = dims
        row = (3 if fused else 1) * C                     # gradients: one dense (B, T, P, 3C) tensor, or three dense ones
        geo = _LoopGeometry()
        geo.desc = GateLoopDesc(dtype=dtype, B=B, T=T, P=P, C=C, in_b=strides[0], in_t=strides[1], in_p=strides[2],
                                grad_b=T * P * row, grad_t=P * row, grad_p=row)
        geo.B, geo.T, geo.P, geo.C = dims
        geo.states, geo.ws_forward, geo.ws_backward = ops.gateloop_sizes(geo.desc)
        _geometries[key] = geo
    return geo


def _loop_parts(qkva, C):
    return qkva if isinstance(qkva, (tuple, list)) else qkva.split(C, dim=-1)


def _loop_layout(qkva, tokens):
    """checks (q, kv, a) or the tensor that holds them side by side; returns it in a layout the kernels address, with
    (B, T, P, C), the strides of (b, t, p) and the shapes of y and of the state.  tokens: is there a token axis?"""
    fused = torch.is_tensor(qkva)
    first = qkva if fused else qkva[0]
    _need(torch.is_tensor(first), 'gate_loop: expected a tensor [q | kv | a] or the three tensors (q, kv, a)')
    rank = 3 if tokens else 2
    _need(first.dim() in (rank, rank + 1), f'gate_loop: expected {"(B, T[, P], C)" if tokens else "(B[, P], C)"} tensors, got {tuple(first.shape)}')
    shape = first.shape
    if fused:
        _need(shape[-1] % 3 == 0 and shape[-1] > 0, f'gate_loop: the last axis holds [q | kv | a], three equal parts; got {shape[-1]}')
        C = shape[-1] // 3
        if first.stride(-1) != 1:
            qkva = first = first.contiguous()
    else:
        _need(len(qkva) == 3 and all(torch.is_tensor(t) for t in qkva), 'gate_loop: expected the three tensors (q, kv, a)')
        _need(all(t.shape == shape and t.dtype == first.dtype and t.device == first.device for t in qkva),
              'gate_loop: q, kv and a differ in shape, type or device')
        C = shape[-1]
        _need(C > 0, 'gate_loop: no channels')
        if first.stride(-1) != 1 or any(t.stride() != first.stride() for t in qkva):
            qkva = tuple(t.contiguous() for t in qkva)
            first = qkva[0]
    st = first.stride()
    B, T = shape[0], shape[1] if tokens else 1
    P = shape[rank - 1] if first.dim() == rank + 1 else 1
    strides = (st[0] if B > 1 else 0, st[1] if tokens and T > 1 else 0, st[rank - 1] if P > 1 else 0)
    lead = tuple(shape[:-1])
    return qkva, (B, T, P, C), strides, lead + (C,), ((B, P, C) if first.dim() == rank + 1 else (B, C)), first


def _check_state(state, shape, device, name='state'):
    _need(torch.is_tensor(state) and tuple(state.shape) == shape, f'gate_loop: {name} is {tuple(state.shape)}, expected {shape}')
    _need(state.dtype == torch.float32, f'gate_loop: {name} is {state.dtype}; states are fp32')
    _need(state.device == device, f'gate_loop: {name} is on {state.device}, the rows on {device}')


def _loop_forward(ops, geo, parts, state, lengths, resets, y_shape, h_shape, want_state, keep):
    y = ops.empty(y_shape, parts[0].dtype)
    h = ops.empty(h_shape, torch.float32) if want_state else None
    states = ops.empty((geo.B, geo.states, geo.P, geo.C), torch.float32) if keep and geo.states else None
    _launch(ops, ops.gateloop_forward(geo.desc, *parts, state, lengths, resets, y, h, states, _bytes(ops, geo.ws_forward)))
    return y, h, states


class _GateLoop(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, geo, shapes, lengths, resets, state, *qkva):
        parts = _loop_parts(qkva[0] if len(qkva) == 1 else qkva, geo.C)
        y, h, states = _loop_forward(ops, geo, parts, state, lengths, resets, *shapes, True, True)
        ctx.save_for_backward(state, lengths, resets, states, *qkva)
        ctx.ops, ctx.geo = ops, geo
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        state, lengths, resets, states, *qkva = ctx.saved_tensors
        ops, geo = ctx.ops, ctx.geo
        none = (None,) * 5
        if dy is None and dh is None:
            return none + (None,) * (1 + len(qkva))
        fused = len(qkva) == 1
        parts = _loop_parts(qkva[0] if fused else qkva, geo.C)
        dy = ops.zeros(tuple(parts[0].shape), parts[0].dtype) if dy is None else dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        grads = (ops.empty(tuple(qkva[0].shape), dy.dtype),) if fused else tuple(ops.empty(tuple(t.shape), dy.dtype) for t in qkva)
        dstate = ops.empty(tuple(state.shape), torch.float32) if state is not None and ctx.needs_input_grad[5] else None
        _launch(ops, ops.gateloop_backward(geo.desc, *parts, state, lengths, resets, states, dy, dh,
                                           *_loop_parts(grads[0] if fused else grads, geo.C), dstate, _bytes(ops, geo.ws_backward)))
        return none + (dstate,) + grads


def gate_loop(qkva, *, state=None, lengths=None, resets=None, return_state=False):
    """Gated linear recurrence ``h_t = sigmoid(a_t) h_{t-1} + kv_t``, ``y_t = q_t h_t`` along the tokens, per sample, pixel and channel.

    ``qkva``: ``(B, T, 3C)`` or ``(B, T, P, 3C)``, the projections [q | kv | a] side by side, or the three ``(B, T[, P], C)`` tensors
    ``(q, kv, a)``; bf16 or fp32; any strides.  ``state``: fp32 ``(B[, P], C)``, the state before the first token (default: empty).
    ``lengths``: ``(B,)`` int32 / int64, tokens per sample in a padded batch (values are taken into ``[0, T]``): ``y`` and the gradients are zero
    behind them, whatever the rows hold there, and the last state is the one behind the last token that exists.  ``resets``: ``(B, T)`` bool /
    uint8, tokens that start a new document: no state and no gradient crosses them.
    Returns ``y`` (``(B, T[, P], C)``, dense), with ``return_state`` also the last state.  Gradients reach ``qkva`` and ``state``."""
    qkva, dims, strides, y_shape, h_shape, first = _loop_layout(qkva, True)
    B, T, P, C = dims
    dtype, dev = _row_dtype(first, 'gate_loop'), first.device
    if state is not None:
        _check_state(state, h_shape, dev)
        state = state.contiguous()
    if lengths is not None:
        _need(torch.is_tensor(lengths) and tuple(lengths.shape) == (B,) and lengths.dtype in (torch.int32, torch.int64) and lengths.device == dev,
              f'gate_loop: lengths must be int32 / int64 ({B},) on {dev}')
        lengths = (lengths if lengths.dtype == torch.int32 else lengths.clamp(0, T).to(torch.int32)).contiguous()
    if resets is not None:
        _need(torch.is_tensor(resets) and tuple(resets.shape) == (B, T) and resets.dtype in (torch.bool, torch.uint8) and resets.device == dev,
              f'gate_loop: resets must be bool / uint8 {(B, T)} on {dev}')
        resets = resets.contiguous()
    ops = _ops(dev)
    if B * P == 0:                                        # no sequences: nothing to launch, and nothing that a gradient could reach
        y = first.new_empty(y_shape)
        return (y, first.new_empty(h_shape, dtype=torch.float32)) if return_state else y
    fused = torch.is_tensor(qkva)
    geo = _loop_geometry(ops, dtype, dims, strides, fused)
    leaves = (qkva,) if fused else qkva
    if torch.is_grad_enabled() and (any(t.requires_grad for t in leaves) or (state is not None and state.requires_grad)):
        y, h = _GateLoop.apply(ops, geo, (y_shape, h_shape), lengths, resets, state, *leaves)
    else:
        y, h, _ = _loop_forward(ops, geo, _loop_parts(qkva, C), state, lengths, resets, y_shape, h_shape, return_state, False)
    return (y, h) if return_state else y


def gate_loop_step(qkva, state, *, state_out=None):
    """One token of ``gate_loop``: ``qkva`` ``(B[, P], 3C)`` or ``(q, kv, a)`` of ``(B[, P], C)``, ``state`` dense fp32 ``(B[, P], C)``.  The new state is
    written over ``state``, or into ``state_out`` (dense fp32, the same shape; apart from ``state``, or ``state`` itself).  Returns ``y`` ``(B[, P], C)``.
    For inference: it has no gradient."""
    qkva, dims, strides, y_shape, h_shape, first = _loop_layout(qkva, False)
    dtype, dev = _row_dtype(first, 'gate_loop_step'), first.device
    _check_state(state, h_shape, dev)
    _need(state.is_contiguous(), 'gate_loop_step: the state is updated in place and must be dense')
    if state_out is None:
        state_out = state
    elif state_out is not state:
        _check_state(state_out, h_shape, dev, 'state_out')
        _need(state_out.is_contiguous(), 'gate_loop_step: state_out must be dense')
        apart = abs(state_out.data_ptr() - state.data_ptr())
        _need(apart == 0 or apart >= 4 * state.numel(), 'gate_loop_step: state_out overlaps state')
    fused = torch.is_tensor(qkva)
    if torch.is_grad_enabled():
        _need(not (state.requires_grad or state_out.requires_grad or any(t.requires_grad for t in ((qkva,) if fused else qkva))),
              'gate_loop_step has no gradient (it updates the state in place): use gate_loop, or torch.no_grad()')
    ops = _ops(dev)
    y = ops.empty(y_shape, first.dtype)
    if dims[0] * dims[2] == 0:
        return y
    geo = _loop_geometry(ops, dtype, dims, strides, fused)
    _launch(ops, ops.gateloop_forward(geo.desc, *_loop_parts(qkva, geo.C), state, None, None, y, state_out, None, _bytes(ops, geo.ws_forward)))
    return y


# ----------------------------------------------------------------------------------------------------------------- norms around a block
def _rows(t, C):
    """t as rows of C contiguous elements one stride apart, copied only where it has no such view"""
    r = t.reshape(-1, C)
    if r.stride(1) != 1 or (r.shape[0] > 1 and r.stride(0) > 1 << 20):
        r = r.contiguous()
    return r


def _stride(r):
    return 0 if r is None else (r.stride(0) if r.shape[0] > 1 else r.shape[1])


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, act, keep, x, branch, gate, post, scale, pre):
        C = x.shape[-1]
        rx, rb, rg = (None if t is None else _rows(t, C) for t in (x, branch, gate))
        d = BlockNormDesc(dtype=_DTYPES[x.dtype], C=C, rows=rx.shape[0], x_stride=_stride(rx), branch_stride=_stride(rb), gate_stride=_stride(rg),
                          gate_act=act, reserved=0)
        shape = tuple(x.shape)
        out = ops.empty(shape, x.dtype) if branch is not None else None
        normed = ops.empty(shape, x.dtype) if pre is not None else None
        rstd = ops.empty((2, rx.shape[0]), torch.float32) if keep and (post is not None or pre is not None) else None
        _launch(ops, ops.block_norm_forward(d, rx, rb, rg, post, scale, pre, out, normed, rstd))
        if keep:
            ctx.save_for_backward(rx, rb, rg, post, scale, pre, rstd)
            ctx.ops, ctx.desc, ctx.shape = ops, d, shape
            ctx.set_materialize_grads(False)
        return out, normed

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dn):
        x, branch, gate, post, scale, pre, rstd = ctx.saved_tensors
        if dout is None and dn is None:
            return (None,) * 9
        ops, d, need = ctx.ops, ctx.desc, ctx.needs_input_grad
        dout = None if dout is None else dout.contiguous()
        dn = None if dn is None else dn.contiguous()
        dx, dbranch, dgate = (ops.empty(ctx.shape, x.dtype) if n else None for n in need[3:6])
        dpost, dscale, dpre = (ops.empty((d.C,), torch.float32) if n else None for n in need[6:9])
        cols = dpost is not None or dscale is not None or dpre is not None
        ws = _bytes(ops, ops.block_norm_workspace_bytes(d)) if cols else None
        _launch(ops, ops.block_norm_backward(d, x, branch, gate, post, scale, pre, rstd, dout, dn, dx, dbranch, dgate, dpost, dscale, dpre, ws))
        return None, None, None, dx, dbranch, dgate, dpost, dscale, dpre


class _NoGrad:
    """stands in for the autograd context of a call without gradients"""


def block_norm(x, branch=None, *, gate=None, gate_act='silu', post_gamma=None, scale=None, pre_gamma=None):
    """Closes a residual block and opens the next in one pass over the rows:

        out = x + scale * act(gate) * N(branch; post_gamma)          normed = N(out; pre_gamma)
        N(v; gamma) = v / max(|v|, 1e-12) * sqrt(C) * gamma          (the framework's RMSNorm, reference magvit2_pytorch.py:258-276)

    ``x``, ``branch``, ``gate``: ``(..., C)``, one shape, bf16 or fp32, any strides (a third of a fused projection is read where it lies);
    ``post_gamma``, ``scale``, ``pre_gamma``: ``(C,)``, computed with in fp32.  ``gate_act``: 'silu', 'sigmoid' or 'none' (the gate as it is).
    Left out: ``branch`` - no add, ``out`` is ``x``; ``post_gamma`` - the branch enters as it is; ``gate``, ``scale`` - ones; ``pre_gamma`` - no second
    norm, ``normed`` is None.  C <= 16384.  Returns ``(out, normed)``.  Gradients reach every tensor; the parameters' are bitwise reproducible."""
    _need(torch.is_tensor(x) and x.dim() >= 1 and x.shape[-1] > 0, 'block_norm: x must have rows of at least one channel')
    _need(gate_act in _ACTS, f'block_norm: unknown gate_act {gate_act!r}; silu, sigmoid or none')
    C, dev = x.shape[-1], x.device
    _row_dtype(x, 'block_norm')
    if C > 16384:
        raise NotImplementedError(f'block_norm: rows of {C} channels; up to 16384 are built')
    if branch is None:
        _need(gate is None and post_gamma is None and scale is None, 'block_norm: gate, post_gamma and scale act on a branch, and there is none')
        _need(pre_gamma is not None, 'block_norm: nothing to do without a branch and without pre_gamma')
    for name, t in (('branch', branch), ('gate', gate)):
        if t is not None:
            _need(torch.is_tensor(t) and t.shape == x.shape and t.dtype == x.dtype and t.device == dev,
                  f'block_norm: {name} and x differ in shape, type or device')
    params = []
    for name, t in (('post_gamma', post_gamma), ('scale', scale), ('pre_gamma', pre_gamma)):
        if t is not None:
            _need(torch.is_tensor(t) and tuple(t.shape) == (C,) and t.is_floating_point() and t.device == dev,
                  f'block_norm: {name} must be a floating-point ({C},) tensor on {dev}')
            t = t.to(torch.float32).contiguous()
        params.append(t)
    ops = _ops(dev)
    args = (ops, _ACTS[gate_act] if gate is not None else 0)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, branch, gate, *params)):
        out, normed = _BlockNorm.apply(*args, True, x, branch, gate, *params)
    else:
        out, normed = _BlockNorm.forward(_NoGrad, *args, False, x, branch, gate, *params)
    return (x if branch is None else out), normed
