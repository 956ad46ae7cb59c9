"""The gated linear recurrence, the norms around its block, and the layer that joins them (csrc/gated_scan.hip,
csrc/block_norm.hip): autograd nodes and the single-step forms.  Public through mdmm.ops.

One layer of a recurrent residual block (models.common.GatedLinearRNN stacks them):

    n    = rms_norm(x, w_0)                                         the norm before the first block
    proj = n W^T + b            (T, B, 3H) = [f | c | g]            one time-parallel product
    h_t  = a_t h_{t-1} + (1 - a_t) c_t,  a = sigmoid(f)             gated_scan
    x'   = x + s silu(g) rms_norm(h, w);  n' = rms_norm(x', w')     block_norm (w': the next block's norm)

States, row statistics and sums are fp32 whatever the tensors' type; every stored tensor is rounded once.
"""
import ctypes as C

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import native

_TYPES = (torch.float32, torch.bfloat16)


def _check_type(name, *tensors):
    for t in tensors:
        if t is not None and t.dtype not in _TYPES:
            raise ValueError('%s: fp32 or bf16 tensors, got %s' % (name, t.dtype))


def _check_device(name, first, *tensors):
    """Every tensor on first's GPU -> its index."""
    i = first.get_device()
    if i < 0:
        ops._need_gpu(first)
    for t in tensors:
        if t is not None and t.get_device() != i:
            ops._need_gpu(t)
            raise ValueError('%s: tensors on %s and %s' % (name, first.device, t.device))
    return i


def _apply(device, fn, *args):
    """fn(*args) with `device` as the current one (a caller may have another one current)."""
    if device == torch._C._cuda_getDevice():
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


def _tangent(tensors):
    """Whether one of them carries a forward-mode tangent (which the kernels, reading addresses, would drop)."""
    return forward_ad._current_level >= 0 and any([t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors])


def _grad_wanted(*tensors):
    """Whether the call goes through its autograd node (which refuses tangents)."""
    return torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in tensors]) or _tangent(tensors)


_FN = {}


def _launch(name, tag, *structs):
    """ops._call on the current stream, without its look-ups (they cost as much as the launch itself)."""
    if ops.TIMER is not None:
        ops._call(name, *(C.byref(a) for a in structs), tag=tag)
        return
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(native.lib(), name)
    rc = fn(*structs, torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()))
    if rc:
        native.check(rc, name)


def _vector(name, what, t, H):
    """An fp32 weight vector of H elements as the kernels read it."""
    if t is None:
        return None
    if not torch.is_tensor(t) or t.dim() != 1 or t.shape[0] != H:
        raise ValueError('%s: %s must be a vector of %d elements, got %s'
                         % (name, what, H, tuple(t.shape) if torch.is_tensor(t) else t))
    if t.dtype != torch.float32:
        raise ValueError('%s: %s must be fp32, got %s' % (name, what, t.dtype))
    return t if t.is_contiguous() else t.contiguous()


def _vectors(name, weight, scale, next_weight, H):
    if weight is None:
        raise ValueError('%s: weight is not optional' % name)
    return [_vector(name, k, t, H) for k, t in (('weight', weight), ('scale', scale), ('next_weight', next_weight))]


def _mask_bytes(name, mask, lead):
    """(T,B[,1]) mask (bool, bytes or floats; 0 = left out) as a byte tensor."""
    if mask is None:
        return None
    if mask.dim() == len(lead) + 1 and mask.shape[-1] == 1:
        mask = mask.squeeze(-1)
    if tuple(mask.shape) != tuple(lead):
        raise ValueError('%s: mask must be %s, got %s' % (name, tuple(lead), tuple(mask.shape)))
    return mask if mask.dtype in (torch.bool, torch.uint8) else mask.detach() != 0


def _check_sizes(name, *sizes):
    if max(sizes) > 2 ** 31 - 1:
        raise ValueError('%s: dimensions below 2^31, got %s' % (name, sizes))


def _unit_cols(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_h0(name, h0, B, H):
    if h0 is None:
        return None
    if tuple(h0.shape) not in ((H,), (B, H)):
        raise ValueError('%s: h0 must be (%d,) or (%d, %d), got %s' % (name, H, B, H, tuple(h0.shape)))
    return _unit_cols(h0.float())


def _fill_scan(a, x, H, h0, mask, reverse):
    T, B = x.shape[:2]
    a.T, a.B, a.H, a.reverse, a.gates_bf16 = T, B, H, reverse, x.dtype is torch.bfloat16
    a.gates = x.data_ptr()
    a.gates_st, a.gates_sb = x.stride()[:2]
    if h0 is not None:
        a.h0, a.h0_sb = h0.data_ptr(), (h0.stride(0) if h0.dim() == 2 else 0)
    if mask is not None:
        a.mask, a.mask_st, a.mask_sb = mask.data_ptr(), mask.stride(0), mask.stride(1)


def _size(name, *args):
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(native.lib(), name)
    return fn(*args)


def _scan_ws(a, bwd, dev):
    """Scratch of a call, to be held until it is launched."""
    n = _size('mdmm_gated_scan_ws', a, bwd)
    if n <= 0:
        return None
    ws = torch.empty(n, dtype=torch.float32, device=dev)
    a.ws = ws.data_ptr()
    return ws


def _scan_forward(a, x, H, h0, mask, reverse, h, keep):
    """Fills the struct of a forward call over h.shape -> (h_last, states, scratch)."""
    T, B = x.shape[:2]
    dev = x.device
    last = torch.empty((B, H), device=dev, dtype=torch.float32)
    _fill_scan(a, x, H, h0, mask, reverse)
    a.h, a.h_last, a.h_bf16 = h.data_ptr(), last.data_ptr(), h.dtype is torch.bfloat16
    states = None
    if keep:
        n = _size('mdmm_gated_scan_states', a)
        if n:
            states = torch.empty(n, device=dev, dtype=torch.float32)
            a.states = states.data_ptr()
    return last, states, _scan_ws(a, 0, dev)


def _scan_backward(a, x, H, h0, mask, reverse, h_dtype, states, g_h, g_last, g_x, need_h0):
    """Fills the struct of a backward call that writes columns [0, 2H) of g_x -> (gradient of h0 in its shape or None,
    tensors to hold until the launch)."""
    B, dev = x.shape[1], x.device
    _fill_scan(a, x, H, h0, mask, reverse)
    a.h_bf16 = h_dtype is torch.bfloat16
    a.states, a.g_h, a.g_last = ops._ptr(states), ops._ptr(g_h), ops._ptr(g_last)
    a.g_gates, a.g_gates_st, a.g_gates_sb = g_x.data_ptr(), g_x.stride(0), g_x.stride(1)
    g0 = per = None
    if need_h0:
        g0 = per = torch.empty((B, H), device=dev, dtype=torch.float32)
        a.g_h0 = per.data_ptr()
        if h0.dim() == 1:
            g0 = torch.empty(H, device=dev, dtype=torch.float32)
            a.g_h0_sum = g0.data_ptr()
    return g0, (per, _scan_ws(a, 1, dev))


def _no_steps_last(h0, B, H, dev):
    return torch.zeros(B, H, device=dev) if h0 is None else h0.detach().expand(B, H).clone()


def _no_steps_grad(h0, g_last):
    """Gradient of h0 where nothing was launched: T = 0 hands g_last on, B or H = 0 has none."""
    if h0 is None:
        return None
    if g_last is None or h0.numel() == 0 or g_last.shape[0] == 0:
        return torch.zeros_like(h0)
    return g_last if h0.dim() == 2 else ops.colsum(g_last)


def _run_scan(gates, h0, mask, reverse, keep=False):
    """-> (h, h_last, states kept for the backward pass)."""
    T, B, H2 = gates.shape
    H = H2 // 2
    h = torch.empty((T, B, H), device=gates.device, dtype=gates.dtype)
    if h.numel() == 0:
        return h, _no_steps_last(h0, B, H, gates.device), None
    a = native.GatedScan()
    last, states, ws = _scan_forward(a, gates, H, h0, mask, reverse, h, keep)
    _launch('mdmm_gated_scan_fwd', 'gated_scan_fwd', a)
    del ws
    return h, last, states


class _GatedScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gates, h0, mask, reverse):
        ctx.set_materialize_grads(False)
        h, last, states = _run_scan(gates, h0, mask, reverse, True)
        ctx.save_for_backward(gates, h0, mask, states)
        ctx.reverse = reverse
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, g_h, g_last):
        if g_h is None and g_last is None:
            return None, None, None, None
        gates, h0, mask, states = ctx.saved_tensors
        g_h = None if g_h is None else g_h.contiguous()
        g_last = None if g_last is None else g_last.contiguous()
        g_x = _new(gates, gates.dtype)
        if g_x.numel() == 0:
            return g_x, _no_steps_grad(h0, g_last if gates.shape[0] == 0 else None), None, None
        a = native.GatedScan()
        g0, hold = _scan_backward(a, gates, gates.shape[2] // 2, h0, mask, ctx.reverse, gates.dtype, states, g_h, g_last, g_x,
                                  h0 is not None and ctx.needs_input_grad[1])
        _launch('mdmm_gated_scan_bwd', 'gated_scan_bwd', a)
        del hold
        return g_x, g0, None, None


def gated_scan(gates, h0=None, mask=None, reverse=False):
    """h_t = a_t h_{t-1} + (1 - a_t) c_t with a = sigmoid(f) over dim 0 of gates (T,B,2H) = [f | c], fp32 or bf16.

    h0: the state in front of the first step, (H,) for every sequence or (B,H); zeros by default.  mask (T,B): a step with
    0 leaves the state as it is, its f and c are not used (they may be NaN) and get zero gradients.  reverse: from the last
    step to the first.  -> (h (T,B,H) in the gates' type, the state behind the last step taken (B,H) in fp32).
    Differentiable in gates and h0, once."""
    if gates.dim() != 3 or gates.shape[2] % 2:
        raise ValueError('gated_scan: gates must be (T, B, 2H), got %s' % (tuple(gates.shape),))
    _check_type('gated_scan', gates)
    T, B, H2 = gates.shape
    _check_sizes('gated_scan', T, B, H2)
    h0, mask = _check_h0('gated_scan', h0, B, H2 // 2), _mask_bytes('gated_scan', mask, (T, B))
    dev = _check_device('gated_scan', gates, h0, mask)
    gates, reverse = _unit_cols(gates), bool(reverse)
    if _grad_wanted(gates, h0):
        return _apply(dev, _GatedScanFn.apply, gates, h0, mask, reverse)
    return _apply(dev, _run_scan, gates, h0, mask, reverse)[:2]


def _no_grad_only(name, *tensors):
    if _grad_wanted(*tensors):
        raise ValueError('%s has no gradient: call it under torch.no_grad(), or %s for training'
                         % (name, name.replace('_step', '')))


def _check_state(name, state, new_state, B, H):
    for what, t in (('state', state), ('new_state', new_state)):
        if t is None and what == 'new_state':
            continue
        if not torch.is_tensor(t) or t.dtype != torch.float32 or tuple(t.shape) != (B, H) or not t.is_contiguous():
            raise ValueError('%s: %s must be contiguous fp32 (%d, %d), got %s'
                             % (name, what, B, H, (t.dtype, tuple(t.shape)) if torch.is_tensor(t) else t))


def gated_scan_step(gates, state, mask=None, new_state=None):
    """One time step of gated_scan for streams whose state the caller keeps: gates (B,2H), state (B,H) fp32, mask (B,).
    -> (h (B,H) in the gates' type, new state (B,H) fp32).  new_state: where the state goes; `state` itself updates it in
    place, None allocates; it shares memory with no other input.  No gradient."""
    if gates.dim() != 2 or gates.shape[1] % 2:
        raise ValueError('gated_scan_step: gates must be (B, 2H), got %s' % (tuple(gates.shape),))
    _check_type('gated_scan_step', gates)
    B, H = gates.shape[0], gates.shape[1] // 2
    _check_sizes('gated_scan_step', B, 2 * H)
    mask = _mask_bytes('gated_scan_step', mask, (B,))
    _no_grad_only('gated_scan_step', gates, state)
    _check_state('gated_scan_step', state, new_state, B, H)
    dev = _check_device('gated_scan_step', gates, state, mask, new_state)
    return _apply(dev, _scan_step, _unit_cols(gates), state, mask, new_state)


def _scan_step(gates, state, mask, new_state):
    B, H = state.shape
    new_state = torch.empty_like(state) if new_state is None else new_state
    h = torch.empty((B, H), device=gates.device, dtype=gates.dtype)
    if h.numel():
        a = native.GatedScan()
        _fill_step(a, gates, H, state, mask, new_state)
        a.h, a.h_bf16 = h.data_ptr(), a.gates_bf16
        _launch('mdmm_gated_scan_fwd', 'gated_scan_step', a)
    return h, new_state


def _fill_step(a, x, H, state, mask, new_state):
    a.T, a.B, a.H, a.gates_bf16 = 1, x.shape[0], H, x.dtype is torch.bfloat16
    a.gates, a.gates_sb, a.h0, a.h0_sb, a.h_last = x.data_ptr(), x.stride(0), state.data_ptr(), H, new_state.data_ptr()
    if mask is not None:
        a.mask, a.mask_sb = mask.data_ptr(), mask.stride(0)


# ---- norms -------------------------------------------------------------------------------------------------------

def _as_rows(t, H):
    """(rows, H) view with unit column stride: rows of any one stride without a copy."""
    return _unit_cols(t.reshape(-1, H))


def _row(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _flat(t, H):
    """(t, or a view or copy of it, whose rows of H have one stride; that stride), None for None."""
    if t is None or t.is_contiguous():          # (no view: one costs as much as a launch)
        return None if t is None else (t, H)
    t = _as_rows(t, H)
    return t, _row(t)


def _new(like, dtype):
    """A new contiguous tensor of like's shape."""
    if like.dtype is dtype and like.is_contiguous():
        return torch.empty_like(like)
    return torch.empty(like.shape, device=like.device, dtype=dtype)


def _combo(name, y, branch, res):
    key = tuple(d == torch.bfloat16 for d in (y, branch, res))
    if key not in ((False, False, False), (True, True, True), (True, True, False), (False, True, False), (False, True, True)):
        raise ValueError('%s: types (y, gate / norm output, residual) = (%s, %s, %s) are not supported together' % (name, y, branch, res))
    return key


def _fill_norm(p, rows, H, y, gate, res, w, s, w_next, branch, eps):
    """y, gate, res: _flat()'s pairs."""
    p.rows, p.H, p.eps = rows, H, eps
    t, p.res_st = res
    p.res, p.branch_bf16, p.res_bf16 = t.data_ptr(), branch is torch.bfloat16, t.dtype is torch.bfloat16
    if y is not None:
        t, p.y_st = y
        p.y, p.y_bf16 = t.data_ptr(), t.dtype is torch.bfloat16
    if gate is not None:
        t, p.gate_st = gate
        p.gate = t.data_ptr()
    if w is not None:
        p.w = w.data_ptr()
    if s is not None:
        p.scale = s.data_ptr()
    if w_next is not None:
        p.w_next = w_next.data_ptr()


def _norm_backward(p, like, g_out, g_n, d_y, d_gate, d_res, want):
    """Fills in the gradients of a backward call: g_out, g_n _flat()'s pairs, d_y, d_gate, d_res contiguous tensors (None: not
    wanted), want = (d_w, d_scale, d_w_next) flags, like: a vector of H -> (the three column sums, None where not wanted;
    scratch to hold until the launch)."""
    H = p.H
    if g_out is not None:
        p.g_out, p.g_out_st = g_out[0].data_ptr(), g_out[1]
    if g_n is not None:
        p.g_n, p.g_n_st = g_n[0].data_ptr(), g_n[1]
    if d_y is not None:
        p.d_y, p.d_y_st = d_y.data_ptr(), H
    if d_gate is not None:
        p.d_gate, p.d_gate_st = d_gate.data_ptr(), H
    if d_res is not None:
        p.d_res, p.d_res_st = d_res.data_ptr(), H
    sums = [torch.empty_like(like) if k else None for k in want]
    if p.rows == 0:
        return [None if t is None else t.zero_() for t in sums], None
    p.d_w, p.d_scale, p.d_w_next = [ops._ptr(t) for t in sums]
    ws = like.new_empty(_size('mdmm_block_norm_ws', p))
    p.ws = ws.data_ptr()
    return sums, ws


def _run_norm(y, gate, res, w, s, w_next, branch, eps, H):
    """y, gate, res: tensors of one shape, or None for the first two -> (out or None, n or None)."""
    p = native.BlockNorm()
    flat = _flat(y, H), _flat(gate, H), _flat(res, H)             # (held until the launch)
    _fill_norm(p, res.numel() // H, H, *flat, w, s, w_next, branch, eps)
    out = n = None
    if y is not None:
        out = _new(res, res.dtype)
        p.out, p.out_st = out.data_ptr(), H
    if w_next is not None:
        n = _new(res, branch)
        p.n, p.n_st = n.data_ptr(), H
    _launch('mdmm_block_norm_fwd', 'block_norm_fwd', p)
    return out, n


class _RmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps, dtype):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, w)
        ctx.eps, ctx.branch = eps, dtype
        return _run_norm(None, None, x, None, None, w, dtype, eps, w.shape[0])[1]

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        if g is None:
            return None, None, None, None
        x, w = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        H = w.shape[0]
        d_x = _new(g, x.dtype) if need_x else None
        p = native.BlockNorm()
        res, g_n = _flat(x, H), _flat(g, H)
        _fill_norm(p, x.numel() // H, H, None, None, res, None, None, w, ctx.branch, ctx.eps)
        sums, ws = _norm_backward(p, w, None, g_n, None, None, d_x, (False, False, need_w))
        if ws is not None:
            _launch('mdmm_block_norm_bwd', 'rms_norm_bwd', p)
        del ws, res, g_n
        return d_x, sums[2], None, None


def _check_width(name, H):
    if not 1 <= H <= native.NORM_MAX_H:
        raise ValueError('%s: rows of 1 to %d columns, got %d' % (name, native.NORM_MAX_H, H))


def rms_norm(x, weight, eps=1e-6, dtype=None):
    """x rsqrt(mean(x^2) + eps) weight over the last dimension: the norm before a block.  x fp32 or bf16 (below 1e19, whose
    squares fp32 holds), weight (H,) fp32;
    dtype: the output's type (x's by default; bf16 from fp32 is the other one there is).  Differentiable, once."""
    if x.dim() < 1:
        raise ValueError('rms_norm: a tensor with rows, got a scalar')
    H = x.shape[-1]
    dtype = x.dtype if dtype is None else dtype
    _check_type('rms_norm', x)
    _check_width('rms_norm', H)
    if dtype not in _TYPES or (x.dtype == torch.bfloat16 and dtype != torch.bfloat16):
        raise ValueError('rms_norm: %s rows to %s' % (x.dtype, dtype))
    weight = _vector('rms_norm', 'weight', weight, H)
    dev = _check_device('rms_norm', x, weight)
    if _grad_wanted(x, weight):
        return _apply(dev, _RmsNormFn.apply, x, weight, float(eps), dtype)
    return _apply(dev, _run_norm, None, None, x, None, None, weight, dtype, float(eps), H)[1]


class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, res, w, gate, s, w_next, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(y, gate, res, w, s, w_next)
        ctx.eps = eps
        out, n = _run_norm(y, gate, res, w, s, w_next, y.dtype, eps, w.shape[0])
        return out if n is None else (out, n)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_out, g_n=None):
        if g_out is None and g_n is None:
            return (None,) * 7
        y, gate, res, w, s, w_next = ctx.saved_tensors
        need = ctx.needs_input_grad                     # y, res, w, gate, s, w_next
        H, like = w.shape[0], g_n if g_out is None else g_out
        d_y = _new(like, y.dtype) if need[0] else None
        d_gate = _new(like, gate.dtype) if need[3] else None
        d_res = _new(like, res.dtype) if need[1] and g_n is not None else None
        p = native.BlockNorm()
        flat = _flat(y, H), _flat(gate, H), _flat(res, H), _flat(g_out, H), _flat(g_n, H)
        _fill_norm(p, res.numel() // H, H, *flat[:3], w, s, w_next, y.dtype, ctx.eps)
        sums, ws = _norm_backward(p, w, *flat[3:], d_y, d_gate, d_res, (need[2], need[4], need[5]))
        if ws is not None:
            _launch('mdmm_block_norm_bwd', 'block_norm_bwd', p)
        del ws, flat
        if need[1] and d_res is None:                    # (without a next norm it is g_out itself)
            d_res = g_out
        return d_y, d_res, sums[0], d_gate, sums[1], sums[2], None


def block_norm(y, residual, weight, gate=None, scale=None, next_weight=None, eps=1e-6):
    """The end of a residual block and the norm of the next one in one pass each way:

        out = residual + scale * silu(gate) * rms_norm(y, weight)          (gate, scale: None = 1)
        n   = rms_norm(out, next_weight)

    -> out, or (out, n) with next_weight.  y, gate and n fp32 or bf16 (one type), residual and out that type or fp32; weight,
    scale and next_weight (H,) fp32; any leading dimensions.  Differentiable in every tensor, once."""
    name = 'block_norm'
    if y.shape != residual.shape or (gate is not None and gate.shape != y.shape) or y.dim() < 1:
        raise ValueError('%s: y %s, residual %s and gate %s must have one shape'
                         % (name, tuple(y.shape), tuple(residual.shape), None if gate is None else tuple(gate.shape)))
    H = y.shape[-1]
    _check_type(name, y, residual, gate)
    _check_width(name, H)
    if gate is not None and gate.dtype != y.dtype:
        raise ValueError('%s: gate %s beside y %s' % (name, gate.dtype, y.dtype))
    _combo(name, y.dtype, y.dtype, residual.dtype)
    weight, scale, next_weight = _vectors(name, weight, scale, next_weight, H)
    dev = _check_device(name, y, residual, weight, gate, scale, next_weight)
    if _grad_wanted(y, residual, weight, gate, scale, next_weight):
        return _apply(dev, _BlockNormFn.apply, y, residual, weight, gate, scale, next_weight, float(eps))
    out, n = _apply(dev, _run_norm, y, gate, residual, weight, scale, next_weight, y.dtype, float(eps), H)
    return out if n is None else (out, n)


# ---- the layer ---------------------------------------------------------------------------------------------------

def _up4(n):
    return (n + 3) & ~3


def _fill_block(p, proj, res, rows, H, h, w, s, w_next, eps):
    """The norm's struct on the states at address h and the gate's columns of proj -> tensors to hold until the launch (proj's
    and the residual's copies, where their rows have no one stride)."""
    res, (flat, st) = _flat(res, H), _flat(proj, 3 * H)
    _fill_norm(p, rows, H, None, None, res, w, s, w_next, proj.dtype, eps)
    p.y, p.y_st = h, H
    p.gate, p.gate_st = flat.data_ptr() + 2 * H * flat.element_size(), st
    return res, flat


def _run_block(proj, res, h0, w, s, w_next, mask, reverse, eps, keep=False):
    """-> (out, n or None, h_last, one buffer: the states of every step, then those kept for the backward pass)."""
    T, B, H = res.shape
    dev = proj.device
    out = _new(res, res.dtype)
    n = _new(res, proj.dtype) if w_next is not None else None
    if out.numel() == 0:
        return out, n, _no_steps_last(h0, B, H, dev), None
    last = torch.empty((B, H), device=dev, dtype=torch.float32)
    a, p = native.GatedScan(), native.BlockNorm()
    _fill_scan(a, proj, H, h0, mask, reverse)
    kept = _size('mdmm_gated_scan_states', a) if keep else 0
    size = _up4(T * B * H)
    states = torch.empty(size + kept, device=dev, dtype=torch.float32)
    a.h, a.h_last = states.data_ptr(), last.data_ptr()
    if kept:
        a.states = a.h + 4 * size
    flat = _fill_block(p, proj, res, T * B, H, a.h, w, s, w_next, eps)
    p.out, p.out_st = out.data_ptr(), H
    if n is not None:
        p.n, p.n_st = n.data_ptr(), H
    ws = _scan_ws(a, 0, dev)
    _launch('mdmm_gated_block_fwd', 'gated_block_fwd', a, p)
    del ws, flat
    return out, n, last, states


class _GatedBlockFn(torch.autograd.Function):
    """gated_scan and block_norm on one projection: the state stays fp32 between them, and their gradients land in one
    (T,B,3H) buffer instead of being joined by copies."""

    @staticmethod
    def forward(ctx, proj, res, h0, w, s, w_next, mask, reverse, eps):
        ctx.set_materialize_grads(False)
        out, n, last, states = _run_block(proj, res, h0, w, s, w_next, mask, reverse, eps, True)
        ctx.save_for_backward(proj, res, h0, w, s, w_next, mask, states)
        ctx.reverse, ctx.eps = reverse, eps
        return (out, last) if n is None else (out, n, last)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        proj, res, h0, w, s, w_next, mask, states = ctx.saved_tensors
        g_out, g_last = grads[0], grads[-1]
        g_n = grads[1] if len(grads) == 3 else None
        need = ctx.needs_input_grad                    # proj, res, h0, w, s, w_next
        T, B, H3 = proj.shape
        H, dev = H3 // 3, proj.device
        if g_out is None and g_n is None and g_last is None:
            return (None,) * 9
        d_res = None
        if need[1]:                                    # (without a next norm it is g_out itself)
            d_res = g_out if g_n is None else _new(g_n, res.dtype)
        g_out, g_n = _flat(g_out, H), _flat(g_n, H)
        g_last = None if g_last is None else g_last.contiguous()
        g_x = _new(proj, proj.dtype)
        through = g_out is not None or g_n is not None
        sums = [torch.empty_like(w) if k and through else None for k in need[3:6]]
        if g_x.numel() == 0:
            return (g_x, d_res, _no_steps_grad(h0, g_last if T == 0 else None),
                    *(None if t is None else t.zero_() for t in sums), None, None, None)
        a, p = native.GatedScan(), native.BlockNorm()
        _fill_scan(a, proj, H, h0, mask, ctx.reverse)
        size = _up4(T * B * H)
        base = states.data_ptr()
        if states.numel() > size:
            a.states = base + 4 * size
        a.g_last = ops._ptr(g_last)
        a.g_gates, a.g_gates_st, a.g_gates_sb = g_x.data_ptr(), B * H3, H3
        p.rows, p.H = T * B, H
        flat = _fill_block(p, proj, res, T * B, H, base, w, s, w_next, ctx.eps) if through else None
        # one scratch: the states' gradient | the norms' slabs | each sequence's gradient of h0 | the scan's splits
        slabs = _size('mdmm_block_norm_ws', p) if through else 0
        per = _up4(B * H) if h0 is not None and need[2] else 0
        splits = _size('mdmm_gated_scan_ws', a, 1)
        lead = size if through else 0
        scratch = w.new_empty(lead + _up4(slabs) + per + splits)
        at = scratch.data_ptr()
        g0 = None
        if through:
            if g_out is not None:
                p.g_out, p.g_out_st = g_out[0].data_ptr(), g_out[1]
            if g_n is not None:
                p.g_n, p.g_n_st = g_n[0].data_ptr(), g_n[1]
                if d_res is not None:
                    p.d_res, p.d_res_st = d_res.data_ptr(), H
            p.d_y, p.d_y_st, p.ws = at, H, at + 4 * lead
            p.d_gate, p.d_gate_st = g_x.data_ptr() + 2 * H * g_x.element_size(), H3
            p.d_w, p.d_scale, p.d_w_next = [ops._ptr(t) for t in sums]
            a.g_h = at
        else:
            g_x[..., 2 * H:].zero_()
        at += 4 * (lead + _up4(slabs))
        if per:
            g0 = torch.empty(h0.shape, device=dev, dtype=torch.float32)
            if h0.dim() == 1:
                a.g_h0, a.g_h0_sum = at, g0.data_ptr()
            else:
                a.g_h0 = g0.data_ptr()
        if splits:
            a.ws = at + 4 * per
        _launch('mdmm_gated_block_bwd', 'gated_block_bwd', a, p)
        del scratch, flat
        return (g_x, d_res, g0, *sums, None, None, None)


def _check_block(name, proj, residual, lead):
    H = residual.shape[-1]
    if tuple(proj.shape[:-1]) != tuple(residual.shape[:-1]) or proj.shape[-1] != 3 * H or proj.dim() != lead + 1:
        raise ValueError('%s: proj %s must be %s with three times the residual\'s columns, residual %s'
                         % (name, tuple(proj.shape), '(T, B, 3H)' if lead == 2 else '(B, 3H)', tuple(residual.shape)))
    _check_type(name, proj, residual)
    _check_width(name, H)
    _check_sizes(name, *residual.shape)
    _combo(name, torch.float32, proj.dtype, residual.dtype)
    return H


def gated_block(proj, residual, h0, weight, scale=None, next_weight=None, mask=None, reverse=False, eps=1e-6):
    """A recurrent residual block behind its projection proj (T,B,3H) = [f | c | g]:

        h   = gated_scan([f | c], h0, mask, reverse)                        kept in fp32
        out = residual + scale * silu(g) * rms_norm(h, weight);  n = rms_norm(out, next_weight)

    -> (out, h_last) or, with next_weight, (out, n, h_last).  The mask concerns the state alone: a step that is left out
    still gives an output, from the state it leaves unchanged, so its g must be finite.  proj and n fp32 or bf16, residual
    and out that type or fp32.  Differentiable in every floating tensor, once."""
    name = 'gated_block'
    H = _check_block(name, proj, residual, 2)
    T, B = proj.shape[:2]
    weight, scale, next_weight = _vectors(name, weight, scale, next_weight, H)
    h0, mask = _check_h0(name, h0, B, H), _mask_bytes(name, mask, (T, B))
    dev = _check_device(name, proj, residual, h0, weight, scale, next_weight, mask)
    proj, reverse = _unit_cols(proj), bool(reverse)
    if _grad_wanted(proj, residual, h0, weight, scale, next_weight):
        return _apply(dev, _GatedBlockFn.apply, proj, residual, h0, weight, scale, next_weight, mask, reverse, float(eps))
    out, n, last = _apply(dev, _run_block, proj, residual, h0, weight, scale, next_weight, mask, reverse, float(eps))[:3]
    return (out, last) if n is None else (out, n, last)


def gated_block_step(proj, residual, state, weight, scale=None, next_weight=None, mask=None, eps=1e-6, new_state=None):
    """One time step of gated_block in one launch: proj (B,3H), residual (B,H), state (B,H) fp32, mask (B,) ->
    (out, new state) or (out, n, new state).  new_state as in gated_scan_step.  No gradient."""
    name = 'gated_block_step'
    H = _check_block(name, proj, residual, 1)
    B = proj.shape[0]
    w, s, w_next = _vectors(name, weight, scale, next_weight, H)
    mask = _mask_bytes(name, mask, (B,))
    _no_grad_only(name, proj, residual, state, w, s, w_next)
    _check_state(name, state, new_state, B, H)
    dev = _check_device(name, proj, residual, state, w, s, w_next, mask, new_state)
    return _apply(dev, _block_step, _unit_cols(proj), _unit_cols(residual), state, w, s, w_next, mask, float(eps), new_state)


def _block_step(proj, residual, state, w, s, w_next, mask, eps, new_state):
    H = state.shape[1]
    new_state = torch.empty_like(state) if new_state is None else new_state
    a, p = native.GatedScan(), native.BlockNorm()
    _fill_norm(p, proj.shape[0], H, None, None, (residual, _row(residual)), w, s, w_next, proj.dtype, eps)
    out, n = _new(residual, residual.dtype), None
    p.out, p.out_st = out.data_ptr(), H
    if w_next is not None:
        n = _new(residual, proj.dtype)
        p.n, p.n_st = n.data_ptr(), H
    p.gate, p.gate_st = proj.data_ptr() + 2 * H * proj.element_size(), _row(proj)
    if out.numel():
        _fill_step(a, proj, H, state, mask, new_state)
        _launch('mdmm_gated_block_step', 'gated_block_step', a, p)
    return (out, new_state) if n is None else (out, n, new_state)


from . import ops  # noqa: E402  (last: ops re-exports this module's functions, whichever of the two is imported first)
