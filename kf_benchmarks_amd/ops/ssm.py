"""Selective state space layers on time-major sequences [T, B, D], next to the
recurrences of ops.rnn: a recurrence that is linear in its state, so that it
runs in parallel over time, and that goes on token by token from a state of
constant size (csrc/ssm.hip, csrc/causal_conv.hip).

  * ``causal_conv``     - the short convolution over time in front of it;
  * ``selective_scan``  - the recurrence, its skip and its gate;
  * ``causal_conv_step`` / ``selective_scan_step`` - one token, the state
    updated in place;
  * ``ssm_layer``       - one layer: projections, convolution, scan, group norm;
  * ``mask_rows``       - zero past each sequence's length, in front of a product.

Activations may be fp32, bf16 or fp16 and column slices of a wider
[T, B, ...] tensor (a projection's output): they are read in place.  Parameters
and scan states are fp32; all sums are.  Sequences of a padded batch are given
by ``lengths`` (int32 [B]; values are clamped to [0, T]): rows at or past a
sequence's length come out as zero, take no gradient and leave the state as it
is, whatever they hold.  ``reverse`` runs every sequence from its last row to its
first.  Gradients are the same on every run (no atomics).

On CPU tensors the same math runs as plain PyTorch autograd (the numerics
oracle of the GPU tests).
"""

from __future__ import annotations

import torch
from torch.autograd.graph import increment_version  # (a kernel's change of a tensor is torch's to know)

from . import _native as N
from . import nn as F_ops

_I, _L, _P = N.I, N.L, N.P
N.register_optional("kfb_ssm_floats", [_I] * 5, _L)
N.register_optional("kfb_ssm_furthest_state", [_I] * 4, _L)
N.register_optional("kfb_ssm_scan_fwd", [_I, _I] + [_P, _L] * 5 + [_P] * 9 + [_I] * 7 + [_P])
N.register_optional("kfb_ssm_scan_bwd", [_I, _I] + [_P, _L] * 4 + [_P] * 16 + [_I] * 3 + [_P] +
                    [_I] * 7 + [_P])
N.register_optional("kfb_ssm_step", [_I] + [_P, _L] * 5 + [_P] * 5 + [_I] * 5 + [_P])
N.register_optional("kfb_cconv_bwd_ws", [_I] * 4, _L)
N.register_optional("kfb_cconv_fwd", [_I, _I, _P, _L] + [_P] * 6 + [_I] * 6 + [_P])
N.register_optional("kfb_cconv_bwd", [_I, _I] + [_P, _L] * 2 + [_P] * 9 + [_I] * 2 + [_P] + [_I] * 6
                    + [_P])
N.register_optional("kfb_cconv_step", [_I, _I, _P, _L] + [_P] * 4 + [_I] * 4 + [_P])
N.register_optional("kfb_mask_rows", [_I, _I, _P, _L, _P, _P] + [_I] * 3 + [_P])

MAX_STATES, MAX_TAPS = 64, 8


# ------------------------------------------------------------------- arguments
def _rows(t):
    """(t, elements from one row to the next) of [T, B, K] read as rows in
    order, copied only if its rows are not evenly spaced."""
    if t.is_contiguous():
        return t, t.shape[2]
    T, B, K = t.shape
    s0, s1, s2 = t.stride()
    if (s2 != 1 and K != 1) or (T != 1 and B != 1 and s0 != B * s1):
        return t.contiguous(), K
    return t, (s1 if B != 1 else s0 if T != 1 else K)


def _vec(width, elems, *rows):
    """Whether every (tensor, row stride) and a width allow ``elems``-wide loads."""
    if width % elems:
        return False
    at = lds = 0
    size = 1
    for t, ld in rows:
        if t is not None:
            at |= t.data_ptr()
            lds |= ld
            size = t.element_size()
    return lds % elems == 0 and at % (elems * size) == 0  # (powers of two)


def _same(x, shape, **tensors):
    for name, t in tensors.items():
        if t is None:
            continue
        if tuple(t.shape) != tuple(shape) or t.dtype != x.dtype or t.device != x.device:
            raise ValueError("%s: %s %s on %s expected, got %s %s on %s" % (
                name, x.dtype, tuple(shape), x.device, t.dtype, tuple(t.shape), t.device))


def _check_lengths(x, lengths):
    if lengths is None:
        return
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (x.shape[1],) or \
            lengths.device != x.device or not lengths.is_contiguous():
        raise ValueError("lengths: a contiguous int32 [%d] tensor on %s expected" % (x.shape[1],
                                                                                   x.device))


def _needs_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return F_ops.has_tangent(*tensors)


def _fits(t, shape, dtype, dev):
    return t is None or (t.shape == shape and t.dtype is dtype and t.device == dev)


def _rows2(t):
    """_rows of a [B, K] tensor."""
    s0, s1 = t.stride()
    return (t, s0) if s1 == 1 or t.shape[1] == 1 else (t.contiguous(), t.shape[1])


def _positions(x, lengths, reverse):
    """[T, B] row of each position (its own inverse) and [T, B, 1] whether the
    position is inside its sequence."""
    T, B = x.shape[:2]
    s = torch.arange(T, device=x.device)[:, None].expand(T, B)
    n = torch.full((B,), T, device=x.device) if lengths is None else lengths.long().clamp(0, T)
    inside = s < n
    return (torch.where(inside, n - 1 - s, s) if reverse else s), inside[..., None], n


def _take(x, pos):
    return torch.gather(x, 0, pos[..., None].expand(-1, -1, x.shape[2]))


# ----------------------------------------------------------------- causal conv
def causal_conv_reference(x, w, b=None, activation=None, lengths=None, initial_state=None,
                          reverse=False):
    """Plain PyTorch (y, state) in w's precision: the oracle of the kernels."""
    T, B, D = x.shape
    K = w.shape[0]
    pos, inside, n = _positions(x, lengths, reverse)
    xs = torch.where(inside, _take(x.to(w.dtype), pos), torch.zeros((), dtype=w.dtype,
                                                                    device=x.device))
    head = xs.new_zeros((K - 1, B, D)) if initial_state is None else initial_state.to(w.dtype)
    seen = torch.cat([head, xs])
    u = sum(w[k] * seen[k:k + T] for k in range(K))
    if b is not None:
        u = u + b
    y = torch.where(inside, F_ops.apply_act(u, activation), torch.zeros_like(u))
    at = n[None, :] + torch.arange(K - 1, device=x.device)[:, None]
    return _take(y, pos).to(x.dtype), _take(seen, at).to(x.dtype)


def _cconv_forward(x, w, b, act, lengths, initial, reverse, state):
    T, B, D = x.shape
    K = w.shape[0]
    x, ld = _rows(x)
    y = torch.empty((T, B, D), dtype=x.dtype, device=x.device)
    last = torch.empty((K - 1, B, D), dtype=x.dtype, device=x.device) if state else None
    ve = 16 // x.element_size()
    N.call("kfb_cconv_fwd", N.dt(x), int(_vec(D, ve, (x, ld), (initial, D))), x.data_ptr(), ld,
           N.ptr(initial), w.data_ptr(), N.ptr(b), N.ptr(lengths), y.data_ptr(), N.ptr(last), T, B,
           D, K, act, int(reverse), N.stream(x.device))
    return y, last


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, initial, lengths, act, reverse, state):
        y, last = _cconv_forward(x, w, b, act, lengths, initial, reverse, state)
        ctx.save_for_backward(x, w, b, initial, lengths)
        ctx.args = (act, reverse, state)
        ctx.params = (w, b)
        ctx.set_materialize_grads(False)
        return (y, last) if state else y

    @staticmethod
    @F_ops.first_order
    def backward(ctx, dy, dlast=None):
        x, w, b, initial, lengths = ctx.saved_tensors
        act, reverse, state = ctx.args
        T, B, D = x.shape
        K, dev = w.shape[0], x.device
        if dy is None:
            dy = x.new_zeros((T, B, D))
        x, ldx = _rows(x)
        dy, ldy = _rows(dy)
        dlast = dlast.contiguous() if dlast is not None else None
        dx = torch.empty((T, B, D), dtype=x.dtype, device=dev)
        dinit = torch.empty_like(initial) if initial is not None and ctx.needs_input_grad[3] else None
        grads, acc = F_ops.grad_buffers(ctx.params)
        ws = torch.empty((F_ops.size_query("kfb_cconv_bwd_ws", T, B, D, K),), dtype=torch.float32, device=dev)
        N.call("kfb_cconv_bwd", N.dt(x),
               int(_vec(D, 4, (x, ldx), (dy, ldy), (initial, D), (dlast, D))), dy.data_ptr(), ldy,
               x.data_ptr(), ldx, N.ptr(initial), w.data_ptr(), N.ptr(b), N.ptr(lengths),
               N.ptr(dlast), dx.data_ptr(), N.ptr(dinit), N.ptr(grads[0]), N.ptr(grads[1]), acc[0],
               acc[1], ws.data_ptr(), T, B, D, K, act, int(reverse), N.stream(dev))
        grads = F_ops.grads_out(ctx.params, grads, acc)
        return dx, grads[0], grads[1], dinit, None, None, None, None


def _check_conv(x, w, b):
    D = x.shape[-1]
    if w.dim() != 2 or not 1 <= w.shape[0] <= MAX_TAPS:
        raise ValueError("causal_conv: filters [K, %d] with K = 1..%d expected, got %s" % (
            D, MAX_TAPS, tuple(w.shape)))
    F_ops.check_params(x, (w.shape[0], D), w=w)
    F_ops.check_params(x, (D,), b=b)


def causal_conv(x, w, b=None, activation=None, lengths=None, initial_state=None,
                return_state=False, reverse=False):
    """y_t = act(b + sum_k w[k] x_{t-K+1+k}) per channel of x [T, B, D]; w [K, D]
    (K = 1..8), b [D] fp32; ``activation`` as ops.nn.group_norm's.
    ``initial_state`` [K-1, B, D] (x's type): the inputs before the first row
    (zero if None).  ``return_state``: also the last K-1 inputs of each sequence,
    [K-1, B, D], from which causal_conv or causal_conv_step goes on.
    Differentiable once in x, w, b and initial_state."""
    act = F_ops.fused_act_code(activation)
    if x.dim() != 3 or x.numel() == 0:
        raise ValueError("causal_conv: a non-empty [T, B, D] tensor expected, got %s" %
                         (tuple(x.shape),))
    _check_conv(x, w, b)
    _check_lengths(x, lengths)
    T, B, D = x.shape
    K = w.shape[0]
    _same(x, (K - 1, B, D), initial_state=initial_state)
    if not x.is_cuda:
        y, last = causal_conv_reference(x, w, b, activation, lengths, initial_state, reverse)
        return (y, last) if return_state else y
    N.dt(x)
    if T > 1 << 20:
        raise ValueError("causal_conv: at most 2^20 rows, got %d" % T)
    if initial_state is not None:
        initial_state = initial_state.contiguous()  # (of one tap: empty, and its gradient too)
    with F_ops.on_device(x):
        if _needs_grad(x, w, b, initial_state):
            return _CausalConv.apply(x, w, b, initial_state, lengths, act, bool(reverse),
                                     bool(return_state))
        y, last = _cconv_forward(x, w, b, act, lengths, initial_state, reverse, return_state)
        return (y, last) if return_state else y


def causal_conv_step(x, state, w, b=None, activation=None):
    """One token x [B, D] after ``state`` [K-1, B, D] (x's type, contiguous, sharing
    no memory with x), which is moved on in place: y [B, D].  No gradient."""
    act = F_ops.fused_act_code(activation)
    if x.dim() != 2 or x.numel() == 0:
        raise ValueError("causal_conv_step: a non-empty [B, D] tensor expected, got %s" %
                         (tuple(x.shape),))
    B, D = x.shape
    K, dt, dev = w.shape[0] if w.dim() else 0, x.dtype, x.device
    # (one token: the checks are a good part of the call, so the messages are left
    # to the slow ones)
    if not (1 <= K <= MAX_TAPS and F_ops.fits_param(w, (K, D), dev) and F_ops.fits_param(b, (D,), dev)
            and _fits(state, (K - 1, B, D), dt, dev) and state is not None):
        _check_conv(x, w, b)
        if state is None:
            raise ValueError("causal_conv_step: a state expected")
        _same(x, (K - 1, B, D), state=state)
    if not state.is_contiguous():
        raise ValueError("causal_conv_step: a contiguous state expected")
    if _needs_grad(x, state, w, b):
        raise ValueError("causal_conv_step updates its state in place and has no gradient: "
                         "call it under torch.no_grad()")
    if not x.is_cuda:
        y, last = causal_conv_reference(x[None], w, b, activation, None, state)
        state.copy_(last)
        return y[0]
    x, ld = _rows2(x)
    y = x.new_empty((B, D))
    px, ps, ve = x.data_ptr(), state.data_ptr(), 4 if dt is torch.float32 else 8
    with F_ops.on_device(x):
        N.call("kfb_cconv_step", N.dt(x), int(D % ve == 0 and ld % ve == 0 and (px | ps) % 16 == 0),
               px, ld, ps, w.data_ptr(), N.ptr(b), y.data_ptr(), B, D, K, act, N.stream(dev))
    increment_version(state)
    return y


# -------------------------------------------------------------- selective scan
def selective_scan_reference(x, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=True,
                             lengths=None, initial_state=None, reverse=False, log_A=False):
    """Plain PyTorch (y, state) in A's precision: the oracle of the kernels."""
    if log_A:
        A = -torch.exp(A)
    T, Bn, Dn = x.shape
    pos, inside, _ = _positions(x, lengths, reverse)
    zero = torch.zeros((), dtype=A.dtype, device=x.device)

    def take(t):
        return torch.where(inside, _take(t.to(A.dtype), pos), zero)

    xs, dt, bs, cs = take(x), take(delta), take(B), take(C)
    if delta_bias is not None:
        dt = dt + delta_bias
    if softplus:
        dt = torch.nn.functional.softplus(dt, threshold=100.0)
    dt = torch.where(inside, dt, zero)
    h = xs.new_zeros((Bn, A.shape[0], Dn)) if initial_state is None else initial_state.to(A.dtype)
    ys = []
    for t in range(T):
        on = inside[t][:, :, None]  # (a gradient of zero times an infinite state is not zero)
        new = torch.exp(dt[t][:, None] * A) * torch.where(on, h, zero) + \
            (dt[t] * xs[t])[:, None] * bs[t][:, :, None]
        h = torch.where(on, new, h)
        ys.append((torch.where(on, h, zero) * cs[t][:, :, None]).sum(1))
    y = torch.stack(ys)
    if D is not None:
        y = y + D * xs
    if z is not None:
        y = y * torch.nn.functional.silu(take(z))
    y = torch.where(inside, y, zero)
    return _take(y, pos).to(x.dtype), h


def _scan_forward(x, delta, A, B, C, D, z, bias, lengths, h0, softplus, reverse, log_A, state,
                  train):
    T, Bn, Dn = x.shape
    Ns, dev = A.shape[0], x.device
    (x, ldx), (delta, ldd), (B, ldb), (C, ldc) = _rows(x), _rows(delta), _rows(B), _rows(C)
    z, ldz = _rows(z) if z is not None else (None, 0)
    y = torch.empty((T, Bn, Dn), dtype=x.dtype, device=dev)
    f32 = dict(dtype=torch.float32, device=dev)
    hT = torch.empty((Bn, Ns, Dn), **f32) if state else None
    bc = torch.empty((F_ops.size_query("kfb_ssm_floats", 0, T, Bn, Dn, Ns),), **f32)
    hs = torch.empty((F_ops.size_query("kfb_ssm_floats", 1, T, Bn, Dn, Ns),), **f32) if train else None
    V = 4 if _vec(Dn, 4, (x, ldx), (delta, ldd), (z, ldz)) else 1
    N.call("kfb_ssm_scan_fwd", N.dt(x), V, x.data_ptr(), ldx, delta.data_ptr(), ldd, N.ptr(z), ldz,
           B.data_ptr(), ldb, C.data_ptr(), ldc, A.data_ptr(), N.ptr(D), N.ptr(bias),
           N.ptr(lengths), N.ptr(h0), N.ptr(hT), N.ptr(hs), bc.data_ptr(), y.data_ptr(), T, Bn, Dn,
           Ns, int(softplus), int(reverse), int(log_A), N.stream(dev))
    return y, hT, bc, hs


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, z, bias, h0, lengths, softplus, reverse, log_A, state):
        y, hT, bc, hs = _scan_forward(x, delta, A, B, C, D, z, bias, lengths, h0, softplus,
                                      reverse, log_A, state, True)
        ctx.save_for_backward(x, delta, A, D, z, bias, lengths, bc, hs)
        ctx.args = (softplus, reverse, log_A, h0 is not None)
        ctx.params = (A, D, bias)
        ctx.set_materialize_grads(False)
        return (y, hT) if state else y

    @staticmethod
    @F_ops.first_order
    def backward(ctx, dy, dhT=None):
        x, delta, A, D, z, bias, lengths, bc, hs = ctx.saved_tensors
        softplus, reverse, log_A, has_h0 = ctx.args
        T, Bn, Dn = x.shape
        Ns, dev, dt = A.shape[0], x.device, x.dtype
        if dy is None:
            dy = x.new_zeros((T, Bn, Dn))
        (x, ldx), (delta, ldd), (dy, ldy) = _rows(x), _rows(delta), _rows(dy)
        z, ldz = _rows(z) if z is not None else (None, 0)
        dhT = dhT.contiguous() if dhT is not None else None
        f32 = dict(dtype=torch.float32, device=dev)
        dh0 = torch.empty((Bn, Ns, Dn), **f32) if has_h0 and ctx.needs_input_grad[8] else None
        dx, ddelta = (torch.empty((T, Bn, Dn), dtype=dt, device=dev) for _ in range(2))
        dz = torch.empty((T, Bn, Dn), dtype=dt, device=dev) if z is not None else None
        dB, dC = (torch.empty((T, Bn, Ns), dtype=dt, device=dev) for _ in range(2))
        grads, acc = F_ops.grad_buffers(ctx.params)
        ws = torch.empty((F_ops.size_query("kfb_ssm_floats", 2, T, Bn, Dn, Ns),), **f32)
        V = 4 if _vec(Dn, 4, (x, ldx), (delta, ldd), (z, ldz), (dy, ldy)) else 1
        N.call("kfb_ssm_scan_bwd", N.dt(x), V, dy.data_ptr(), ldy, x.data_ptr(), ldx,
               delta.data_ptr(), ldd, N.ptr(z), ldz, A.data_ptr(), N.ptr(D), N.ptr(bias),
               N.ptr(lengths), hs.data_ptr(), bc.data_ptr(), N.ptr(dhT), N.ptr(dh0), dx.data_ptr(),
               ddelta.data_ptr(), N.ptr(dz), dB.data_ptr(), dC.data_ptr(), N.ptr(grads[0]),
               N.ptr(grads[1]), N.ptr(grads[2]), acc[0], acc[1], acc[2], ws.data_ptr(), T, Bn, Dn,
               Ns, int(softplus), int(reverse), int(log_A), N.stream(dev))
        dA, dD, dbias = F_ops.grads_out(ctx.params, grads, acc)
        return dx, ddelta, dA, dB, dC, dD, dz, dbias, dh0, None, None, None, None, None


def _check_scan(x, delta, A, B, C, D, z, bias):
    lead, Dn = tuple(x.shape[:-1]), x.shape[-1]
    if A.dim() != 2 or not 1 <= A.shape[0] <= MAX_STATES:
        raise ValueError("selective_scan: A [N, %d] with N = 1..%d expected, got %s" % (
            Dn, MAX_STATES, tuple(A.shape)))
    _same(x, x.shape, delta=delta, z=z)
    _same(x, lead + (A.shape[0],), B=B, C=C)
    F_ops.check_params(x, (A.shape[0], Dn), A=A)
    F_ops.check_params(x, (Dn,), D=D, delta_bias=bias)


def _check_state(x, B, n, Dn, **states):
    for name, t in states.items():
        F_ops.check_params(x, (B, n, Dn), **{name: t})


def selective_scan(x, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=True, lengths=None,
                   initial_state=None, return_state=False, reverse=False, log_A=False):
    """The selective scan of x [T, B, D] with step sizes ``delta`` [T, B, D], input
    and output maps B, C [T, B, N] (all of one type) and decays A [N, D] (N = 1..64):

        dt = softplus(delta + delta_bias)        (softplus=False: delta + delta_bias)
        h_t = exp(dt A) h_{t-1} + dt x B_t,   h [B, N, D] fp32
        y   = (sum_n C_t h_t + D x) silu(z)

    A, D [D], delta_bias [D] fp32; D, z, delta_bias may be None.  dt A is meant to be
    finite and not positive; ``log_A``: A is given as log(-A), the form that training
    keeps negative (its gradient is that of the logarithm).  ``initial_state``: h
    before the first row (zero if None); ``return_state``: also h after each
    sequence's last row, from which selective_scan or selective_scan_step goes on.
    Differentiable once in every tensor but ``lengths``."""
    if x.dim() != 3 or x.numel() == 0:
        raise ValueError("selective_scan: a non-empty [T, B, D] tensor expected, got %s" %
                         (tuple(x.shape),))
    T, Bn, Dn = shape = x.shape
    dt, dev, Ns = x.dtype, x.device, A.shape[0] if A.dim() else 0
    if not (1 <= Ns <= MAX_STATES and _fits(delta, shape, dt, dev) and _fits(z, shape, dt, dev)
            and _fits(B, (T, Bn, Ns), dt, dev) and _fits(C, (T, Bn, Ns), dt, dev)
            and F_ops.fits_param(A, (Ns, Dn), dev) and F_ops.fits_param(D, (Dn,), dev)
            and F_ops.fits_param(delta_bias, (Dn,), dev)):
        _check_scan(x, delta, A, B, C, D, z, delta_bias)
    _check_lengths(x, lengths)
    _check_state(x, Bn, A.shape[0], Dn, initial_state=initial_state)
    if not x.is_cuda:
        y, h = selective_scan_reference(x, delta, A, B, C, D, z, delta_bias, softplus, lengths,
                                        initial_state, reverse, log_A)
        return (y, h) if return_state else y
    N.dt(x)
    if Bn > 65535:
        raise ValueError("selective_scan: at most 65535 sequences, got %d" % Bn)
    with F_ops.on_device(x):
        if _needs_grad(x, delta, A, B, C, D, z, delta_bias, initial_state):
            return _SelectiveScan.apply(x, delta, A, B, C, D, z, delta_bias, initial_state, lengths,
                                        bool(softplus), bool(reverse), bool(log_A),
                                        bool(return_state))
        y, h, _, _ = _scan_forward(x, delta, A, B, C, D, z, delta_bias, lengths, initial_state,
                                   softplus, reverse, log_A, return_state, False)
        return (y, h) if return_state else y


def selective_scan_step(x, delta, A, B, C, state, D=None, z=None, delta_bias=None, softplus=True,
                        log_A=False):
    """One token: x, delta, z [B, D], B, C [B, N] after ``state`` [B, N, D] (fp32,
    contiguous), which is moved on in place: y [B, D].  No gradient."""
    if x.dim() != 2 or x.numel() == 0:
        raise ValueError("selective_scan_step: a non-empty [B, D] tensor expected, got %s" %
                         (tuple(x.shape),))
    shape, dt, dev = x.shape, x.dtype, x.device
    Bn, Dn = shape
    Ns = A.shape[0] if A.dim() else 0
    if not (1 <= Ns <= MAX_STATES and Bn <= 65535 and _fits(delta, shape, dt, dev)
            and _fits(z, shape, dt, dev) and _fits(B, (Bn, Ns), dt, dev)
            and _fits(C, (Bn, Ns), dt, dev) and F_ops.fits_param(A, (Ns, Dn), dev)
            and F_ops.fits_param(D, (Dn,), dev) and F_ops.fits_param(delta_bias, (Dn,), dev)
            and state is not None and F_ops.fits_param(state, (Bn, Ns, Dn), dev)):
        _check_scan(x, delta, A, B, C, D, z, delta_bias)
        if state is None:
            raise ValueError("selective_scan_step: a state expected")
        _check_state(x, Bn, Ns, Dn, state=state)
        if x.is_cuda:
            raise ValueError("selective_scan_step: at most 65535 sequences, got %d" % Bn)
    if _needs_grad(x, delta, A, B, C, state, D, z, delta_bias):
        raise ValueError("selective_scan_step updates its state in place and has no gradient: "
                         "call it under torch.no_grad()")
    if not x.is_cuda:
        y, h = selective_scan_reference(x[None], delta[None], A, B[None], C[None], D,
                                        z[None] if z is not None else None, delta_bias, softplus,
                                        None, state, False, log_A)
        state.copy_(h)
        return y[0]
    (x, ldx), (delta, ldd), (B, ldb), (C, ldc) = _rows2(x), _rows2(delta), _rows2(B), _rows2(C)
    z, ldz = _rows2(z) if z is not None else (None, 0)
    y = x.new_empty((Bn, Dn))
    with F_ops.on_device(x):
        N.call("kfb_ssm_step", N.dt(x), x.data_ptr(), ldx, delta.data_ptr(), ldd, N.ptr(z), ldz,
               B.data_ptr(), ldb, C.data_ptr(), ldc, A.data_ptr(), N.ptr(D), N.ptr(delta_bias),
               state.data_ptr(), y.data_ptr(), Bn, Dn, Ns, int(softplus), int(log_A), N.stream(dev))
    increment_version(state)
    return y


# ----------------------------------------------------------------------- layer
class _SplitColumns(torch.autograd.Function):
    """Column slices of x [..., C], read in place; the backward puts their
    gradients side by side in one native launch."""

    @staticmethod
    def forward(ctx, x, widths):
        ctx.shape, ctx.widths = x.shape, widths
        ctx.set_materialize_grads(False)
        out, at = [], 0
        for w in widths:
            out.append(x[..., at:at + w])
            at += w
        return tuple(out)

    @staticmethod
    @F_ops.first_order
    def backward(ctx, *grads):
        offs = [0]
        for w in ctx.widths:
            offs.append(offs[-1] + w)
        some = next(g for g in grads if g is not None)
        dx = some.new_empty(ctx.shape)
        F_ops._concat_call(dx, [g.contiguous() if g is not None else None for g in grads], offs,
                           dx.numel() // offs[-1], split=False)
        return dx, None


def split_columns(x, widths):
    """x [..., sum(widths)] as slices of its last dim (GPU: no copy forward, one
    native concatenation of the gradients backward)."""
    if sum(widths) != x.shape[-1]:
        raise ValueError("split_columns: %d columns do not split into %s" % (x.shape[-1],
                                                                           tuple(widths)))
    if len(widths) > F_ops._CAT_MAX:
        raise ValueError("split_columns: at most %d slices" % F_ops._CAT_MAX)
    if not x.is_cuda or not x.requires_grad:
        return torch.split(x, list(widths), dim=-1)
    return _SplitColumns.apply(x.contiguous(), tuple(widths))


def _masked(x, lengths):
    x, ld = _rows(x)
    T, B, D = x.shape
    y = torch.empty((T, B, D), dtype=x.dtype, device=x.device)
    N.call("kfb_mask_rows", N.dt(x), int(_vec(D, 16 // x.element_size(), (x, ld))), x.data_ptr(), ld,
           lengths.data_ptr(), y.data_ptr(), T, B, D, N.stream(x.device))
    return y


class _MaskRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, lengths):
        ctx.save_for_backward(lengths)
        return _masked(x, lengths)

    @staticmethod
    @F_ops.first_order
    def backward(ctx, dy):
        return _masked(dy, ctx.saved_tensors[0]), None


def mask_rows(x, lengths):
    """x [T, B, D] with the rows at or past each sequence's length zero, whatever
    they hold (a product's weight gradient would multiply them by zero, which NaN
    and infinities survive)."""
    if x.dim() != 3 or x.numel() == 0:
        raise ValueError("mask_rows: a non-empty [T, B, D] tensor expected, got %s" % (tuple(x.shape),))
    _check_lengths(x, lengths)
    if lengths is None:
        return x
    if not x.is_cuda:
        inside = torch.arange(x.shape[0], device=x.device)[:, None] < lengths
        return torch.where(inside[..., None], x, torch.zeros((), dtype=x.dtype, device=x.device))
    N.dt(x)
    with F_ops.on_device(x):
        return _MaskRows.apply(x, lengths) if _needs_grad(x) else _masked(x, lengths)


def ssm_layer(x, w_in, conv_w, conv_b, w_rank, w_delta, w_bc, delta_bias, A_log, D, norm_w,
              groups=1, lengths=None, reverse=False, low=None):
    """One selective state space layer of x [T, B, din] -> [T, B, E]:

        u, z = x w_in;  u = silu(causal_conv(u))
        delta = u w_rank w_delta;  B, C = u w_bc
        y = group_norm(selective_scan(u, delta, -exp(A_log), B, C, D, z), groups of a row)

    w_in [din, 2 E], conv_w [K, E], w_rank [E, R], w_delta [R, E], w_bc [E, 2 N], A_log
    [N, E] (fp32 masters in the TF layout); ``low``: compute-type copies of the
    four matrices by name.  Rows past ``lengths`` count nowhere and give zero."""
    x = mask_rows(x, lengths)
    T, B, din = x.shape
    E, Ns = conv_w.shape[1], A_log.shape[0]
    low = low or {}

    def matmul(t, w, name):
        return F_ops.linear(t, w, None, w_lp=low.get(name))

    u, z = split_columns(matmul(x.reshape(T * B, din), w_in, "w_in").view(T, B, 2 * E), (E, E))
    u = causal_conv(u, conv_w, conv_b, "silu", lengths, reverse=reverse)
    # read by three consumers: their gradients are summed natively
    us, ur, ub = F_ops.fanout(u, 3)
    delta = matmul(matmul(ur.reshape(T * B, E), w_rank, "w_rank"), w_delta, "w_delta")
    Bm, C = split_columns(matmul(ub.reshape(T * B, E), w_bc, "w_bc").view(T, B, 2 * Ns), (Ns, Ns))
    y = selective_scan(us, delta.view(T, B, E), A_log, Bm, C, D, z, delta_bias, lengths=lengths,
                       reverse=reverse, log_A=True)
    return F_ops.group_norm(y.view(T * B, E), norm_w, None, groups).view(T, B, E)
