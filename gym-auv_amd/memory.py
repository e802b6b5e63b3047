"""Memory over an episode: the sequence operators of a recurrent feature extractor.

A single scan shows no obstacle's velocity; the reference's loader stacks earlier
scans behind each scan for that (utils/dataloader.py:123-137).  Here a vessel carries
a state instead: a short causal convolution and a selective state space scan, with
norms round the block.  Each operator works on whole rollouts (training) and, where
it has a state, on one token per vessel (stepping):

    causal_conv     causal_conv_step        last `width` tokens, channel by channel
    selective_scan  selective_scan_step     N states per channel, decays chosen by the token
    residual_norm   rms_norm                norm after a block, gate, scale, residual sum, norm before the next

Rollouts are [batch, length, channels] views with adjacent channels and any other
strides, so `rollout.transpose(0, 1)` of a time-major [steps, vessels, channels]
store needs no copy; results come back in the layout of the first argument.
`start` [batch, length] marks the first token of an episode (`sim.tensor("t_step") == 0`
on the step's observation): nothing before it is seen by it or by what follows.
`lengths` int32 [batch]: tokens a padded row really holds; the ones behind are not
used, and their outputs and gradients are 0.

Activations are float32, bfloat16 or float16, parameters and the scan's states
float32; arithmetic is in 32 bits and every output is rounded once.  Calls run on
torch's current stream of the tensors' device, never synchronise, and give the same
bits on every call.  They can be captured into a graph.  A captured backward pass is
refused while an eager graph of the same parameters is still alive: drop the outputs of
earlier eager passes first.

`EpisodeMemory` strings them together; `cnn.PerceptionNavigationExtractor(memory=...)`
steps one behind the scan's features.
"""
from __future__ import annotations

import ctypes as C
import math

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib

TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
GATES = {None: _lib.GATE_PLAIN, "silu": _lib.GATE_SILU, "sigmoid": _lib.GATE_SIGMOID}
MAX_STATES = 64
WIDTHS = (2, 3, 4)


# ----------------------------------------------------------------------------
# checks
# ----------------------------------------------------------------------------
def _activation(name, t, shape=None, like=None):
    """`t` is a float CUDA tensor with adjacent channels, of `shape`, and of `like`'s type and device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if like is not None:
        if t.dtype != like.dtype:
            raise TypeError(f"{name} must be {like.dtype}, got {t.dtype}")
        if t.device != like.device:
            raise ValueError(f"{name} is on {t.device}, the call's other tensors on {like.device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be adjacent in memory (call .contiguous())")


def _dense(name, t, shape, like, dtype=torch.float32):
    """An optional contiguous tensor of `dtype` (parameters, states, lengths)."""
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on {like.device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _marks(name, t, shape, like):
    if t is None:
        return
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"{name} must be a bool or uint8 tensor")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on {like.device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")


def _written(name, t, *others):
    """`t` is written element by element: no two of its elements may share memory, and none may lie in `others`."""
    if t.numel() and any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{name} is written and must not be an expanded tensor")
    lo, hi = _span(t)
    for other_name, o in others:
        if o is not None and o.numel() and t.numel():
            a, b = _span(o)
            if lo < b and a < hi:
                raise ValueError(f"{name} overlaps {other_name}")


def _span(t):
    """First byte and the byte behind the last of a tensor's elements."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _no_grad_here(who, *tensors):
    if _wants_grad(*tensors):
        raise RuntimeError(f"{who} keeps no gradients: call it under torch.no_grad(), or use the form for whole rollouts")


def _guard_capture(*leaves):
    """Refuse to record a graph whose backward pass would end in gradient accumulators that an eager graph made: torch
    runs those on the eager graph's stream, and joining that stream to a capture ends the process.  An accumulator lives
    as long as some graph uses it and carries a note of ours when that graph was made eagerly.  The caller holds what
    this returns until its own graph does."""
    capturing = torch.cuda.is_current_stream_capturing()
    nodes = [torch.autograd.graph.get_gradient_edge(t).node for t in leaves if t is not None and t.requires_grad and t.is_leaf]
    for node in nodes:
        if not capturing:
            node.metadata["auv_eager"] = True
        elif "auv_eager" in node.metadata:
            raise RuntimeError("a graph that records gradients is being captured while the outputs of an earlier eager pass "
                               "over the same parameters are alive: drop those first")
    return nodes


def _ptr(t):
    return None if t is None else t.data_ptr()


def _strides(name, t, *dims):
    """{name: pointer, name_row: stride, ...} of an activation; a dimension of one element has no stride to heed."""
    if t is None:
        return {}
    out = {name: t.data_ptr()}
    for k, d in enumerate(dims):
        out[f"{name}_{('row', 'token', 'group')[k]}"] = t.stride(d) if t.shape[d] > 1 else 0
    return out


def _call(name, args, what, device):
    """Runs entry point `name` on the current stream with the scratch memory it asks for."""
    lib = _lib.load()
    ref = C.byref(args)
    room = 0
    if what == _lib.SEQ_BACKWARD or (what == _lib.SEQ_FORWARD and name == "auv_selective_scan"):
        room = getattr(lib, name + "_workspace")(ref, what)
        if room < 0:
            raise _lib.AuvError(room, lib.auv_seq_last_error().decode())
    scratch = None
    if room:
        scratch = torch.empty(room, dtype=torch.uint8, device=device)   # the stream's own: free for it again on return
        args.workspace, args.workspace_bytes = scratch.data_ptr(), room
    rc = getattr(lib, name)(ref, what, torch.cuda.current_stream(device).cuda_stream)
    if rc != 0:
        raise _lib.AuvError(rc, lib.auv_seq_last_error().decode())


def _adjacent(t):
    return t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


# ----------------------------------------------------------------------------
# short causal convolution
# ----------------------------------------------------------------------------
def _conv_args(x, weight, bias, start, lengths, state, silu):
    B, L, D = x.shape
    return _lib.AuvConvArgs(device=x.device.index, dtype=TYPES[x.dtype], batch=B, length=L, channels=D, width=weight.shape[1],
                            silu=bool(silu), weight=weight.data_ptr(), bias=_ptr(bias), lengths=_ptr(lengths), state=_ptr(state),
                            **_strides("x", x, 0, 1), **_strides("start", start, 0, 1))


def _conv_forward(x, weight, bias, start, lengths, state, silu, return_state):
    B, L, D = x.shape
    y = torch.empty_like(x)
    new_state = torch.empty((B, weight.shape[1] - 1, D), dtype=x.dtype, device=x.device) if return_state else None
    if x.numel() == 0:
        if return_state:
            new_state.copy_(state) if state is not None else new_state.zero_()
        return y, new_state
    a = _conv_args(x, weight, bias, start, lengths, state, silu)
    a.y, a.y_row, a.y_token, a.new_state = y.data_ptr(), y.stride(0), y.stride(1), _ptr(new_state)
    _call("auv_causal_conv", a, _lib.SEQ_FORWARD, x.device)
    return y, new_state


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, start, lengths, silu, return_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, start, lengths)
        ctx.silu = silu
        return _conv_forward(x, weight, bias, start, lengths, state, silu, return_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dnew):
        x, weight, bias, state, start, lengths = ctx.saved_tensors
        want_x, want_w, want_b, want_s = ctx.needs_input_grad[:4]
        if x.numel() == 0:
            zeros = lambda t, want: torch.zeros_like(t) if want else None   # noqa: E731
            ds = None if not want_s else torch.zeros_like(state) if dnew is None else dnew.clone()
            return zeros(x, want_x), zeros(weight, want_w), zeros(bias, want_b), ds, None, None, None, None
        dy = torch.zeros_like(x) if dy is None else _adjacent(dy)
        dnew = None if dnew is None else dnew.contiguous()
        dx = torch.empty_like(x)
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        ds = torch.empty_like(state) if want_s else None
        a = _conv_args(x, weight, bias, start, lengths, state, ctx.silu)
        a.d_y, a.d_y_row, a.d_y_token = dy.data_ptr(), dy.stride(0), dy.stride(1)
        a.d_x, a.d_x_row, a.d_x_token = dx.data_ptr(), dx.stride(0), dx.stride(1)
        a.d_new_state, a.d_weight, a.d_bias, a.d_state = _ptr(dnew), _ptr(dw), _ptr(db), _ptr(ds)
        _call("auv_causal_conv", a, _lib.SEQ_BACKWARD, x.device)
        return dx if want_x else None, dw, db, ds, None, None, None, None


def _check_conv(x, weight, bias):
    D = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[1] not in WIDTHS:
        raise ValueError(f"weight must be [channels, width] with a width of {WIDTHS}")
    _dense("weight", weight, (D, weight.shape[1]), x)
    _dense("bias", bias, (D,), x)


def causal_conv(x, weight, bias=None, *, start=None, lengths=None, state=None, silu=True, return_state=False):
    """y[b,l,d] = act(bias[d] + sum_j weight[d,j] x[b,l-(width-1)+j,d]), act = SiLU or nothing.

    x [batch, length, channels]; weight float32 [channels, width], width 2 to 4, its last tap
    the current token's; bias float32 [channels].  `state` [batch, width-1, channels] of x's
    type holds the tokens before the row (None: zeros).  With return_state also the state
    behind each row's last token, which `causal_conv_step` goes on from.  Differentiable in
    x, weight, bias and state."""
    _activation("x", x)
    if x.dim() != 3:
        raise ValueError(f"x must be [batch, length, channels], got {tuple(x.shape)}")
    B, L, D = x.shape
    _check_conv(x, weight, bias)
    _marks("start", start, (B, L), x)
    _dense("lengths", lengths, (B,), x, torch.int32)
    _dense("state", state, (B, weight.shape[1] - 1, D), x, x.dtype)
    if _wants_grad(x, weight, bias, state):
        held = _guard_capture(x, weight, bias, state)   # noqa: F841
        y, new = _Conv.apply(x, weight, bias, state, start, lengths, bool(silu), bool(return_state))
    else:
        y, new = _conv_forward(x, weight, bias, start, lengths, state, silu, return_state)
    return (y, new) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, start=None, silu=True, new_state=None):
    """`causal_conv` of one token per row: x [batch, channels] -> y [batch, channels].  `state`
    [batch, width-1, channels] moves up by the token, in place or into `new_state`."""
    _activation("x", x)
    if x.dim() != 2:
        raise ValueError(f"x must be [batch, channels], got {tuple(x.shape)}")
    B, D = x.shape
    _check_conv(x, weight, bias)
    if state is None:
        raise TypeError("state must be a tensor, got None")
    shape = (B, weight.shape[1] - 1, D)
    _dense("state", state, shape, x, x.dtype)
    _marks("start", start, (B,), x)
    _no_grad_here("causal_conv_step", x, state, weight, bias)
    if new_state is None:
        new_state = state
    elif new_state is not state:
        _dense("new_state", new_state, shape, x, x.dtype)
        _written("new_state", new_state, ("state", state), ("x", x))
    y = torch.empty((B, D), dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return y
    a = _lib.AuvConvArgs(device=x.device.index, dtype=TYPES[x.dtype], batch=B, length=1, channels=D, width=shape[1] + 1,
                         silu=bool(silu), weight=weight.data_ptr(), bias=_ptr(bias), state=state.data_ptr(),
                         new_state=new_state.data_ptr(), y=y.data_ptr(), y_row=D, **_strides("x", x, 0), **_strides("start", start, 0))
    _call("auv_causal_conv", a, _lib.SEQ_STEP, x.device)
    return y


# ----------------------------------------------------------------------------
# selective state space scan
# ----------------------------------------------------------------------------
def _scan_args(u, delta, A, Bm, Cm, D, z, delta_bias, start, lengths, state, softplus):
    B, L, Dc = u.shape
    return _lib.AuvScanArgs(device=u.device.index, dtype=TYPES[u.dtype], batch=B, length=L, channels=Dc, states=A.shape[1],
                            groups=Bm.shape[2], softplus=bool(softplus), A=A.data_ptr(), D=_ptr(D), delta_bias=_ptr(delta_bias),
                            lengths=_ptr(lengths), state=_ptr(state), **_strides("u", u, 0, 1), **_strides("delta", delta, 0, 1),
                            **_strides("z", z, 0, 1), **_strides("B", Bm, 0, 1, 2), **_strides("C", Cm, 0, 1, 2),
                            **_strides("start", start, 0, 1))


def _scan_forward(u, delta, A, Bm, Cm, D, z, delta_bias, start, lengths, state, softplus, return_state, keep):
    y = torch.empty_like(u)
    new_state = torch.empty((u.shape[0],) + tuple(A.shape), dtype=torch.float32, device=u.device) if return_state else None
    if u.numel() == 0:
        if return_state:
            new_state.copy_(state) if state is not None else new_state.zero_()
        return y, new_state, None
    a = _scan_args(u, delta, A, Bm, Cm, D, z, delta_bias, start, lengths, state, softplus)
    a.y, a.y_row, a.y_token, a.new_state = y.data_ptr(), y.stride(0), y.stride(1), _ptr(new_state)
    segments = None
    if keep:
        n = _lib.load().auv_selective_scan_segments(C.byref(a))
        if n < 0:
            raise _lib.AuvError(n, _lib.load().auv_seq_last_error().decode())
        segments = torch.empty(n // 4, dtype=torch.float32, device=u.device)
        a.segments = segments.data_ptr()
    _call("auv_selective_scan", a, _lib.SEQ_FORWARD, u.device)
    return y, new_state, segments


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, Bm, Cm, D, z, delta_bias, state, start, lengths, softplus, return_state):
        ctx.set_materialize_grads(False)
        y, new_state, segments = _scan_forward(u, delta, A, Bm, Cm, D, z, delta_bias, start, lengths, state, softplus,
                                               return_state, True)
        ctx.save_for_backward(u, delta, A, Bm, Cm, D, z, delta_bias, state, start, lengths, segments)
        ctx.softplus = softplus
        return y, new_state

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dnew):
        u, delta, A, Bm, Cm, D, z, delta_bias, state, start, lengths, segments = ctx.saved_tensors
        want = ctx.needs_input_grad
        if u.numel() == 0:
            out = [torch.zeros_like(t) if w else None
                   for t, w in zip((u, delta, A, Bm, Cm, D, z, delta_bias, state), want)]
            if want[8] and dnew is not None:
                out[8] = dnew.clone()
            return (*out, None, None, None, None)
        dy = torch.zeros_like(u) if dy is None else _adjacent(dy)
        dnew = None if dnew is None else dnew.contiguous()
        a = _scan_args(u, delta, A, Bm, Cm, D, z, delta_bias, start, lengths, state, ctx.softplus)
        du, ddelta, dB, dC = (torch.empty_like(t) for t in (u, delta, Bm, Cm))
        dz = None if z is None else torch.empty_like(z)
        dA, dD, dbias, dstate = (torch.empty_like(t) if w else None
                                 for t, w in ((A, want[2]), (D, want[5]), (delta_bias, want[7]), (state, want[8])))
        for name, t, dims in (("d_y", dy, (0, 1)), ("d_u", du, (0, 1)), ("d_delta", ddelta, (0, 1)), ("d_z", dz, (0, 1)),
                              ("d_B", dB, (0, 1, 2)), ("d_C", dC, (0, 1, 2))):
            for k, v in _strides(name, t, *dims).items():
                setattr(a, k, v)
        a.segments, a.d_new_state = segments.data_ptr(), _ptr(dnew)
        a.d_A, a.d_D, a.d_delta_bias, a.d_state = _ptr(dA), _ptr(dD), _ptr(dbias), _ptr(dstate)
        _call("auv_selective_scan", a, _lib.SEQ_BACKWARD, u.device)
        first = [g if w else None for g, w in zip((du, ddelta, dA, dB, dC, dD, dz, dbias, dstate), want)]
        return (*first, None, None, None, None)


def _check_scan(u, delta, A, Bm, Cm, D, z, delta_bias):
    lead, Dc = tuple(u.shape[:-1]), u.shape[-1]
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"A must be [channels, states] with 1 to {MAX_STATES} states")
    _dense("A", A, (Dc, A.shape[1]), u)
    _activation("delta", delta, tuple(u.shape), u)
    if z is not None:
        _activation("z", z, tuple(u.shape), u)
    if not isinstance(Bm, torch.Tensor) or Bm.dim() != u.dim() + 1 or Bm.shape[-2] < 1 or Dc % Bm.shape[-2]:
        raise ValueError("B must be [..., groups, states] with a number of groups that divides the channels")
    shape = lead + (Bm.shape[-2], A.shape[1])
    _activation("B", Bm, shape, u)
    _activation("C", Cm, shape, u)
    _dense("D", D, (Dc,), u)
    _dense("delta_bias", delta_bias, (Dc,), u)


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, *, delta_softplus=True, start=None, lengths=None,
                   state=None, return_state=False):
    """Per channel d of a row, with N states h:

        dt = softplus(delta + delta_bias)      (delta_softplus False: the sum itself)
        h[n] <- exp(dt A[d,n]) h[n] + dt u B[g,n],    y = (sum_n C[g,n] h[n] + D[d] u) silu(z)

    u, delta, z [batch, length, channels]; B, C [batch, length, groups, N], adjacent channels
    sharing a group's; A float32 [channels, N], 1 to 64 states; D, delta_bias float32
    [channels]; D, z and delta_bias may be None.  `state` float32 [batch, channels, N] before
    the row (None: zeros).  With return_state also the state behind each row's last token,
    which `selective_scan_step` goes on from.  Differentiable in every float argument; for
    the backward pass the states before every 16th token are kept, N/4 bytes per element of u
    (N rounded up to 4, 8, 16, 32 or 64)."""
    _activation("u", u)
    if u.dim() != 3:
        raise ValueError(f"u must be [batch, length, channels], got {tuple(u.shape)}")
    _check_scan(u, delta, A, B, C, D, z, delta_bias)
    _marks("start", start, tuple(u.shape[:2]), u)
    _dense("lengths", lengths, (u.shape[0],), u, torch.int32)
    _dense("state", state, (u.shape[0],) + tuple(A.shape), u)
    tensors = (u, delta, A, B, C, D, z, delta_bias, state)
    if _wants_grad(*tensors):
        held = _guard_capture(*tensors)   # noqa: F841
        y, new = _Scan.apply(*tensors, start, lengths, bool(delta_softplus), bool(return_state))
    else:
        y, new, _ = _scan_forward(*tensors[:8], start, lengths, state, delta_softplus, return_state, False)
    return (y, new) if return_state else y


def selective_scan_step(u, delta, state, A, B, C, D=None, z=None, delta_bias=None, *, delta_softplus=True, start=None,
                        new_state=None):
    """`selective_scan` of one token per row: u, delta, z [batch, channels]; B, C [batch, groups, N];
    `state` [batch, channels, N] moves on by the token, in place or into `new_state`."""
    _activation("u", u)
    if u.dim() != 2:
        raise ValueError(f"u must be [batch, channels], got {tuple(u.shape)}")
    _check_scan(u, delta, A, B, C, D, z, delta_bias)
    if state is None:
        raise TypeError("state must be a tensor, got None")
    Bn, Dc = u.shape
    shape = (Bn,) + tuple(A.shape)
    _dense("state", state, shape, u)
    _marks("start", start, (Bn,), u)
    _no_grad_here("selective_scan_step", u, delta, state, A, B, C, D, z, delta_bias)
    if new_state is None:
        new_state = state
    elif new_state is not state:
        _dense("new_state", new_state, shape, u)
        _written("new_state", new_state, ("state", state), ("A", A))
    y = torch.empty((Bn, Dc), dtype=u.dtype, device=u.device)
    if u.numel() == 0:
        return y
    row = lambda t: t.stride(0) if Bn > 1 else 0   # noqa: E731
    group = lambda t: t.stride(1) if t.shape[1] > 1 else 0   # noqa: E731
    a = _lib.AuvScanArgs(device=u.device.index, dtype=TYPES[u.dtype], batch=Bn, length=1, channels=Dc, states=A.shape[1],
                         groups=B.shape[1], softplus=bool(delta_softplus), u=u.data_ptr(), u_row=row(u), delta=delta.data_ptr(),
                         delta_row=row(delta), B=B.data_ptr(), B_row=row(B), B_group=group(B), C=C.data_ptr(), C_row=row(C),
                         C_group=group(C), A=A.data_ptr(), D=_ptr(D), delta_bias=_ptr(delta_bias), state=state.data_ptr(),
                         new_state=new_state.data_ptr(), y=y.data_ptr(), y_row=Dc)
    if z is not None:
        a.z, a.z_row = z.data_ptr(), row(z)
    if start is not None:
        a.start, a.start_row = start.data_ptr(), row(start)
    _call("auv_selective_scan", a, _lib.SEQ_STEP, u.device)
    return y


# ----------------------------------------------------------------------------
# norms round a block
# ----------------------------------------------------------------------------
def _as_rows(t):
    """[..., channels] as [rows or batch, length, channels], without a copy where the strides allow one."""
    if t is None or t.dim() == 3:
        return t
    return t.reshape(1, -1, t.shape[-1]) if t.dim() != 2 else t[None]


def _norm_args(x, y, post_weight, pre_weight, gate, scale, gate_act, eps, dtype):
    B, L, D = x.shape
    return _lib.AuvNormArgs(device=x.device.index, dtype=TYPES[dtype], residual_dtype=TYPES[x.dtype], batch=B, length=L, channels=D,
                            gate_act=GATES[gate_act], eps=eps, post_weight=_ptr(post_weight), pre_weight=_ptr(pre_weight),
                            scale=_ptr(scale), **_strides("x", x, 0, 1), **_strides("y", y, 0, 1), **_strides("gate", gate, 0, 1))


def _norm_forward(x, y, post_weight, pre_weight, gate, scale, gate_act, eps, dtype):
    out = torch.empty_like(x) if y is not None else None
    h = None
    if pre_weight is not None:
        h = torch.empty_like(x if y is None else y, dtype=dtype)
    if x.numel():
        a = _norm_args(x, y, post_weight, pre_weight, gate, scale, gate_act, eps, dtype)
        for name, t in (("x_out", out), ("h", h)):
            for k, v in _strides(name, t, 0, 1).items():
                setattr(a, k, v)
        _call("auv_residual_norm", a, _lib.SEQ_FORWARD, x.device)
    return out, h


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, post_weight, pre_weight, gate, scale, gate_act, eps, dtype):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, y, post_weight, pre_weight, gate, scale)
        ctx.how = (gate_act, eps, dtype)
        return _norm_forward(x, y, post_weight, pre_weight, gate, scale, gate_act, eps, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_h):
        x, y, post_weight, pre_weight, gate, scale = ctx.saved_tensors
        want = ctx.needs_input_grad
        none = (None, None, None)
        if d_out is None and d_h is None or x.numel() == 0:
            return tuple(torch.zeros_like(t) if w else None
                         for t, w in zip((x, y, post_weight, pre_weight, gate, scale), want)) + none
        d_out, d_h = _adjacent(d_out), _adjacent(d_h)
        dx = torch.empty_like(x)
        dy, dgate = (None if t is None else torch.empty_like(t) for t in (y, gate))
        dpost, dpre, dscale = (torch.empty_like(t) if w else None
                               for t, w in ((post_weight, want[2]), (pre_weight, want[3]), (scale, want[5])))
        a = _norm_args(x, y, post_weight, pre_weight, gate, scale, *ctx.how)
        for name, t in (("d_x_out", d_out), ("d_h", d_h), ("d_x", dx), ("d_y", dy), ("d_gate", dgate)):
            for k, v in _strides(name, t, 0, 1).items():
                setattr(a, k, v)
        a.d_post_weight, a.d_pre_weight, a.d_scale = _ptr(dpost), _ptr(dpre), _ptr(dscale)
        _call("auv_residual_norm", a, _lib.SEQ_BACKWARD, x.device)
        return tuple(g if w else None for g, w in zip((dx, dy, dpost, dpre, dgate, dscale), want)) + none


def _norm(x, y, post_weight, pre_weight, gate, scale, gate_act, eps, dtype):
    D = x.shape[-1]
    if D < 1 or D > _lib.NORM_MAX_CHANNELS:
        raise ValueError(f"1 to {_lib.NORM_MAX_CHANNELS} channels, got {D}")
    if not eps > 0.0:
        raise ValueError("eps must be positive")
    if gate_act not in GATES:
        raise ValueError(f"gate_act must be one of {tuple(GATES)}, got {gate_act!r}")
    for name, t in (("post_weight", post_weight), ("pre_weight", pre_weight), ("scale", scale)):
        _dense(name, t, (D,), x)
    shape = x.shape
    xs, ys, gs = _as_rows(x), _as_rows(y), _as_rows(gate)
    args = (xs, ys, post_weight, pre_weight, gs, scale)
    if _wants_grad(x, y, post_weight, pre_weight, gate, scale):
        held = _guard_capture(x, y, post_weight, pre_weight, gate, scale)   # noqa: F841
        out, h = _Norm.apply(*args, gate_act, float(eps), dtype)
    else:
        out, h = _norm_forward(*args, gate_act, float(eps), dtype)
    return tuple(t if t is None else t.reshape(shape) for t in (out, h))


def rms_norm(x, weight, *, eps=1e-6, dtype=None):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension, x [..., channels] (at most 8,192),
    as `dtype` (x's own by default; float32 x may give bfloat16 or float16): the norm before a
    first block.  Differentiable in x and weight."""
    _activation("x", x)
    if x.dim() < 1 or weight is None:
        raise ValueError("x must have a channel dimension and weight be given")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in TYPES or (x.dtype != torch.float32 and x.dtype != dtype):
        raise TypeError(f"a norm of {x.dtype} cannot be {dtype}")
    return _norm(x, None, None, weight, None, None, None, eps, dtype)[1]


def residual_norm(x, y, post_weight=None, pre_weight=None, gate=None, scale=None, *, gate_act="silu", eps=1e-6):
    """What lies between a block's output y and the next block's input, in one pass:

        n = y / sqrt(mean(y^2) + eps) * post_weight       (post_weight None: n = y)
        x' = x + scale * act(gate) * n                    (scale, gate None: 1)
        h = x' / sqrt(mean(x'^2) + eps) * pre_weight      (pre_weight None: h is None)

    Returns (x', h).  x [..., channels] (at most 8,192) is the residual stream, float32 or of
    y's type; y and gate have x's shape and one type, which h gets too; post_weight, pre_weight
    and scale are float32 [channels]; gate_act is "silu", "sigmoid" or None.  A gate that is the
    same for several tokens is given expanded (`gate.expand_as(y)`).  Differentiable in every
    float argument."""
    _activation("x", x)
    _activation("y", y, tuple(x.shape))
    if y.device != x.device:
        raise ValueError(f"y is on {y.device}, x on {x.device}")
    if x.dtype not in (torch.float32, y.dtype):
        raise TypeError(f"x must be float32 or y's {y.dtype}, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("x must have a channel dimension")
    if gate is not None:
        _activation("gate", gate, tuple(x.shape), y)
    return _norm(x, y, post_weight, pre_weight, gate, scale, gate_act, eps, y.dtype)


# ----------------------------------------------------------------------------
# the operators strung together
# ----------------------------------------------------------------------------
class _Layer(nn.Module):
    def __init__(self, channels, inner, states, width, dtype):
        super().__init__()
        self.inner, self.states, self.rank = inner, states, max(1, math.ceil(channels / 16))
        lin = lambda i, o: nn.Linear(i, o, bias=False, dtype=dtype)   # noqa: E731
        self.widen = lin(channels, 2 * inner + channels)              # u, z and the block's gate
        self.choose = lin(inner, self.rank + 2 * states)              # delta (low rank), B, C
        self.delta = lin(self.rank, inner)
        self.narrow = lin(inner, channels)
        self.conv_weight = nn.Parameter(torch.randn(inner, width) / math.sqrt(width))
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.log_A = nn.Parameter(torch.log(torch.arange(1, states + 1, dtype=torch.float32)).repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner))
        # steps of 0.001 to 0.1 at first: softplus(delta_bias) spread evenly over their logarithm
        dt = torch.exp(torch.rand(inner) * math.log(100.0) + math.log(1e-3))
        self.delta_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.pre_weight = nn.Parameter(torch.ones(channels))
        self.post_weight = nn.Parameter(torch.ones(channels))
        self.scale = nn.Parameter(torch.ones(channels))

    def _mix(self, h, conv, scan):
        """Block output and gate of normed input h [..., channels]."""
        u, z, gate = self.widen(h).split((self.inner, self.inner, h.shape[-1]), dim=-1)
        u = conv(u)
        low, B, C = self.choose(u).split((self.rank, self.states, self.states), dim=-1)
        y = scan(u, self.delta(low), -torch.exp(self.log_A), B.unsqueeze(-2), C.unsqueeze(-2), z)
        return self.narrow(y), gate


class EpisodeMemory(nn.Module):
    """Features of a token and everything before it in its episode: a linear layer onto `channels`,
    `layers` blocks of convolution and scan between gated norms, and a last norm.

    `forward(features, start=None, lengths=None, state=None)` takes [batch, length, features]
    and gives ([batch, length, channels], state behind the rows); `step(features, state,
    start=None)` takes [batch, features], gives [batch, channels] and moves `state`
    (`new_state(batch)`, or one that forward gave) on in place.  Both compute the same
    function: a rollout stepped token by token and the rollout at once agree to rounding."""

    def __init__(self, features: int, channels: int = 64, layers: int = 1, *, inner: int | None = None, states: int = 16,
                 width: int = 4, dtype=torch.float32):
        super().__init__()
        if dtype not in TYPES:
            raise TypeError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        if not 1 <= states <= MAX_STATES or width not in WIDTHS or layers < 1:
            raise ValueError(f"states must be in 1..{MAX_STATES}, width in {WIDTHS}, layers at least 1")
        self.features, self.channels, self.dtype, self.width, self.states = features, channels, dtype, width, states
        self.inner = 2 * channels if inner is None else inner
        self.enter = nn.Linear(features, channels)
        self.layers = nn.ModuleList(_Layer(channels, self.inner, states, width, dtype) for _ in range(layers))
        self.last_weight = nn.Parameter(torch.ones(channels))

    def new_state(self, batch: int):
        """The state before an episode's first token."""
        dev = self.last_weight.device
        return [(torch.zeros(batch, self.width - 1, self.inner, dtype=self.dtype, device=dev),
                 torch.zeros(batch, self.inner, self.states, device=dev)) for _ in self.layers]

    def _run(self, features, mixers):
        x = self.enter(features)                       # the residual stream, in 32 bits
        h = rms_norm(x, self.layers[0].pre_weight, dtype=self.dtype)
        for i, (layer, (conv, scan)) in enumerate(zip(self.layers, mixers)):
            y, gate = layer._mix(h, conv, scan)
            after = self.layers[i + 1].pre_weight if i + 1 < len(self.layers) else self.last_weight
            x, h = residual_norm(x, y, layer.post_weight, after, gate, layer.scale)
        return h

    def forward(self, features, start=None, lengths=None, state=None):
        out = []

        def mixer(layer, s):
            def conv(u):
                u, new = causal_conv(u, layer.conv_weight, layer.conv_bias, start=start, lengths=lengths,
                                     state=None if s is None else s[0], return_state=True)
                out.append([new])
                return u

            def scan(u, delta, A, B, C, z):
                y, new = selective_scan(u, delta, A, B, C, layer.D, z, layer.delta_bias, start=start, lengths=lengths,
                                        state=None if s is None else s[1], return_state=True)
                out[-1].append(new)
                return y
            return conv, scan

        h = self._run(features, [mixer(layer, None if state is None else state[i]) for i, layer in enumerate(self.layers)])
        return h, [tuple(s) for s in out]

    @torch.no_grad()
    def step(self, features, state, start=None):
        def mixer(layer, s):
            def conv(u):
                return causal_conv_step(u, s[0], layer.conv_weight, layer.conv_bias, start=start)

            def scan(u, delta, A, B, C, z):
                return selective_scan_step(u, delta, s[1], A, B, C, layer.D, z, layer.delta_bias, start=start)
            return conv, scan

        return self._run(features, [mixer(layer, state[i]) for i, layer in enumerate(self.layers)])
