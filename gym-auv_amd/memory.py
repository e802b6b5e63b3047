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
earlier eager passes first.  A backward pass is captured together with its forward pass.
Forward-mode derivatives and traces (torch.jit.trace, make_fx) are refused; torch.compile
breaks its graph at these calls and runs them.

`EpisodeMemory` strings them together; `cnn.PerceptionNavigationExtractor(memory=...)`
steps one behind the scan's features.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
import threading
import weakref

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _lib

TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
GATES = {None: _lib.GATE_PLAIN, "silu": _lib.GATE_SILU, "sigmoid": _lib.GATE_SIGMOID}
MAX_STATES = 64
WIDTHS = (2, 3, 4)
_LEAST = torch.finfo(torch.float32).smallest_normal


# ----------------------------------------------------------------------------
# checks
# ----------------------------------------------------------------------------
# A call on a single vessel takes the GPU some 3 us, so the host's part counts: each check returns what the call goes on
# to use, and the argument blocks (include/auvsim.h: 64-bit fields only) are packed in one go.

# What torch tells of itself, by its own shortest ways where this torch has them: a step of one vessel is host time.
_jit_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)
_increment_version = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)
try:
    _modes = torch._C._len_torch_dispatch_stack
    _modes_before_dispatch = torch._ops.mode_stack_state_for_pre_dispatch().get      # of 0: a proxy mode
    _modes(), _modes_before_dispatch(0)
except (AttributeError, TypeError):
    _modes = _modes_before_dispatch = lambda *_: True


def _no_trace():
    """A trace would record the memory for the results, and not the kernels that fill it: outputs that nothing has written
    whenever it is run."""
    if _jit_tracing() or get_proxy_mode() is not None:
        raise RuntimeError("the sequence operators cannot be traced: call them outside of the trace")


def _first(name, t, dims, what):
    """The tensor that fixes a call's type and device: (shape, strides, device number)."""
    if _jit_tracing() or _modes() or _modes_before_dispatch(0):
        _no_trace()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    shape, strides = tuple(t.shape), t.stride()
    if dims is not None and len(shape) != dims:
        raise ValueError(f"{name} must be {what}, got {shape}")
    if not shape:
        raise ValueError(f"{name} must have a channel dimension")
    if shape[-1] > 1 and strides[-1] != 1:
        raise ValueError(f"{name}: the last dimension must be adjacent in memory (call .contiguous())")
    return shape, strides, t.get_device()


def _like(name, t, shape, dtype, dev):
    """Strides of another activation of the call."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on cuda:{dev}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    strides = t.stride()
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name}: the last dimension must be adjacent in memory (call .contiguous())")
    return strides


def _dense(name, t, shape, dev, dtype=torch.float32):
    """Address of an optional contiguous tensor (parameters, states, lengths); 0 for None."""
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on cuda:{dev}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _marks(t, shape, dev):
    """(address, row stride, token stride) of the optional start marks."""
    if t is None:
        return 0, 0, 0
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.bool, torch.uint8):
        raise TypeError("start must be a bool or uint8 tensor")
    if t.get_device() != dev:
        raise ValueError(f"start is on {t.device}, the call's other tensors on cuda:{dev}")
    if t.shape != shape:
        raise ValueError(f"start must be {tuple(shape)}, got {tuple(t.shape)}")
    strides = t.stride()
    return t.data_ptr(), strides[0], strides[1] if len(strides) > 1 else 0


def _apart(name, t, other_name, o):
    """`t`, contiguous and about to be written, shares no memory with `o`."""
    lo, hi = t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()
    first = o.data_ptr()
    last = first + (sum((n - 1) * s for n, s in zip(o.shape, o.stride())) + 1) * o.element_size() if o.numel() else first
    if lo < last and first < hi:
        raise ValueError(f"{name} overlaps {other_name}")


def _in_place(name, lo, t, others):
    """A step's new state, t's worth of memory from address lo on, shares none with the step's inputs, each given as its
    address and its length up to the last byte."""
    hi = lo + t.numel() * t.element_size()
    for p, n in others:
        if p < hi and lo < p + n:
            raise ValueError(f"{name} holds an input of the step")


def _written(t):
    """A kernel has written t: a graph that keeps t for its backward pass has to know, as after torch's own operations."""
    _increment_version((t,))


def _no_tangents(tensors):
    """Forward-mode derivatives end at these calls: refused, for they would end in silence (a tensor with a tangent need not
    require a gradient)."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the sequence operators have no forward-mode derivatives")


def _wants_grad(tensors):
    """Whether the call has to be recorded for a backward pass."""
    if getattr(forward_ad, "_current_level", 0) >= 0:        # within a dual_level, as far as this torch tells
        _no_tangents(tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_grad_here(who, tensors):
    if _wants_grad(tensors):
        raise RuntimeError(f"{who} keeps no gradients: call it under torch.no_grad(), or use the form for whole rollouts")


_eager_nodes = weakref.WeakSet()     # the graph nodes of eager calls, as long as their graphs live
_eager_lock = threading.Lock()


def _leaves_of(nodes):
    """The leaves whose gradient accumulators lie behind these graph nodes."""
    leaves, seen, todo = set(), set(), list(nodes)
    while todo:
        node = todo.pop()
        if node is None or node in seen:
            continue
        seen.add(node)
        leaf = getattr(node, "variable", None)       # an accumulator's
        if leaf is not None:
            leaves.add(id(leaf))
        todo.extend(n for n, _ in node.next_functions)
    return leaves


def _check_capture(tensors):
    """Refuse to record a graph whose backward pass would end in gradient accumulators that an eager graph made: torch
    runs those on the eager graph's stream, and joining that stream to a capture ends the process."""
    if not torch.cuda.is_current_stream_capturing():
        return
    with _eager_lock:
        alive = _leaves_of(_eager_nodes)
    if not alive:
        return
    wanted = [t for t in tensors if t is not None and t.requires_grad]
    leaves = {id(t) for t in wanted if t.grad_fn is None}
    if (leaves | _leaves_of(t.grad_fn for t in wanted)) & alive:
        raise RuntimeError("a graph that records gradients is being captured while the outputs of an earlier eager pass "
                           "over the same parameters are alive: drop those first")


def _note_node(ctx):
    if not torch.cuda.is_current_stream_capturing():
        with _eager_lock:
            _eager_nodes.add(ctx)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _rows(t):
    """(address, row stride, token stride) of an activation of our own making or known to be in order."""
    if t is None:
        return 0, 0, 0
    s = t.stride()
    return t.data_ptr(), s[0], s[1]


def _groups(t):
    s = t.stride()
    return t.data_ptr(), s[0], s[1], s[2]


def _new(t, dtype=None):
    """Memory for a result of t's shape, in t's layout where that leaves the channels adjacent (a sliding window over a
    signal has two strides of 1, and may come back the other way round)."""
    r = torch.empty_like(t, dtype=dtype)
    return r if r.stride(-1) == 1 or t.shape[-1] <= 1 else torch.empty(t.shape, dtype=r.dtype, device=t.device)


def _adjacent(t):
    return t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _packer(cls):
    """Packs an argument block without its last two fields, the workspace's."""
    kinds = {C.c_void_p: "q", C.c_int64: "q", C.c_double: "d"}
    return struct.Struct("<" + "".join(kinds[k] for _, k in cls._fields_[:-2])).pack


_pack_conv, _pack_scan, _pack_norm = _packer(_lib.AuvConvArgs), _packer(_lib.AuvScanArgs), _packer(_lib.AuvNormArgs)
_pack_room = struct.Struct("<2q").pack
_NO_ROOM = _pack_room(0, 0)


# the current stream's handle without the Stream object round it, where this torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _call(name, block, what, dev, scratch=True):
    """Runs entry point `name` on the current stream, with the scratch memory it asks for."""
    lib = _lib.load()
    tail = _NO_ROOM
    if scratch:
        room = getattr(lib, name + "_workspace")(block + _NO_ROOM, what)
        if room < 0:
            raise _lib.AuvError(room, lib.auv_seq_last_error().decode())
        if room:
            held = torch.empty(room, dtype=torch.uint8, device=dev)   # the stream's own: free for it again on return
            tail = _pack_room(held.data_ptr(), room)
    rc = getattr(lib, name)(block + tail, what, _raw_stream(dev))
    if rc != 0:
        raise _lib.AuvError(rc, lib.auv_seq_last_error().decode())


# ----------------------------------------------------------------------------
# short causal convolution
# ----------------------------------------------------------------------------
def _conv_head(x, weight, bias, start, lengths, state, silu):
    """The argument block up to state."""
    B, L, D = x.shape
    return (x.get_device(), TYPES[x.dtype], B, L, D, weight.shape[1], silu, *_rows(x), weight.data_ptr(), _ptr(bias), *_rows(start),
            _ptr(lengths), _ptr(state))


def _conv_forward(x, weight, bias, start, lengths, state, silu, return_state):
    y = _new(x)
    new = torch.empty((x.shape[0], weight.shape[1] - 1, x.shape[2]), dtype=x.dtype, device=x.device) if return_state else None
    if x.numel() == 0:
        if return_state:
            new.copy_(state) if state is not None else new.zero_()
        return y, new
    head = _conv_head(x, weight, bias, start, lengths, state, silu)
    _call("auv_causal_conv", _pack_conv(*head, _ptr(new), *_rows(y), *(0,) * 10), _lib.SEQ_FORWARD, head[0], scratch=False)
    return y, new


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, start, lengths, silu, return_state):
        _note_node(ctx)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, start, lengths)
        ctx.silu = silu
        return _conv_forward(x, weight, bias, start, lengths, state, silu, return_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dnew):
        x, weight, bias, state, start, lengths = ctx.saved_tensors
        want_x, want_w, want_b, want_s = ctx.needs_input_grad[:4]
        rest = (None,) * 4
        if x.numel() == 0:
            zeros = lambda t, want: torch.zeros_like(t) if want else None   # noqa: E731
            ds = None if not want_s else torch.zeros_like(state) if dnew is None else dnew.clone()
            return (zeros(x, want_x), zeros(weight, want_w), zeros(bias, want_b), ds) + rest
        dy = _new(x).zero_() if dy is None else _adjacent(dy)
        dnew = None if dnew is None else dnew.contiguous()
        dx = _new(x)
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        ds = torch.empty_like(state) if want_s else None
        head = _conv_head(x, weight, bias, start, lengths, state, ctx.silu)
        block = _pack_conv(*head, 0, 0, 0, 0, *_rows(dy), _ptr(dnew), *_rows(dx), _ptr(dw), _ptr(db), _ptr(ds))
        _call("auv_causal_conv", block, _lib.SEQ_BACKWARD, head[0])
        return (dx if want_x else None, dw, db, ds) + rest


def _taps(weight, bias, D, dev):
    """The width, of taps in order."""
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[1] not in WIDTHS:
        raise ValueError(f"weight must be [channels, width] with a width of {WIDTHS}")
    W = weight.shape[1]
    _dense("weight", weight, (D, W), dev)
    _dense("bias", bias, (D,), dev)
    return W


def causal_conv(x, weight, bias=None, *, start=None, lengths=None, state=None, silu=True, return_state=False):
    """y[b,l,d] = act(bias[d] + sum_j weight[d,j] x[b,l-(width-1)+j,d]), act = SiLU or nothing.

    x [batch, length, channels]; weight float32 [channels, width], width 2 to 4, its last tap
    the current token's; bias float32 [channels].  `state` [batch, width-1, channels] of x's
    type holds the tokens before the row (None: zeros).  With return_state also the state
    behind each row's last token, which `causal_conv_step` goes on from.  Differentiable in
    x, weight, bias and state."""
    (B, L, D), _, dev = _first("x", x, 3, "[batch, length, channels]")
    W = _taps(weight, bias, D, dev)
    _marks(start, (B, L), dev)
    _dense("lengths", lengths, (B,), dev, torch.int32)
    _dense("state", state, (B, W - 1, D), dev, x.dtype)
    silu, tensors = 1 if silu else 0, (x, weight, bias, state)
    if _wants_grad(tensors):
        _check_capture(tensors)
        y, new = _Conv.apply(*tensors, start, lengths, silu, bool(return_state))
    else:
        y, new = _conv_forward(x, weight, bias, start, lengths, state, silu, return_state)
    return (y, new) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, start=None, silu=True, new_state=None):
    """`causal_conv` of one token per row: x [batch, channels] -> y [batch, channels].  `state`
    [batch, width-1, channels] moves up by the token, in place or into `new_state`.  (A state that a
    rollout's backward pass still needs is cloned first, or stepped into a `new_state`.)"""
    (B, D), strides, dev = _first("x", x, 2, "[batch, channels]")
    W = _taps(weight, bias, D, dev)
    if state is None:
        raise TypeError("state must be a tensor, got None")
    s = _dense("state", state, (B, W - 1, D), dev, x.dtype)
    marks = _marks(start, (B,), dev)
    _no_grad_here("causal_conv_step", (x, state, weight, bias))
    to = s
    if new_state is not None and new_state is not state:
        to = _dense("new_state", new_state, (B, W - 1, D), dev, x.dtype)
        _apart("new_state", new_state, "state", state)
    last, pb = B - 1 if B else 0, _ptr(bias)
    _in_place("the new state", to, state, ((x.data_ptr(), (last * strides[0] + D) * x.element_size()), (weight.data_ptr(), 4 * D * W),
                                           (pb, 4 * D), (marks[0], last * marks[1] + 1)))
    y = _new(x)
    if B and D:
        block = _pack_conv(dev, TYPES[x.dtype], B, 1, D, W, 1 if silu else 0, x.data_ptr(), strides[0], 0, weight.data_ptr(),
                           pb, *marks, 0, s, to, y.data_ptr(), y.stride(0), 0, *(0,) * 10)
        _call("auv_causal_conv", block, _lib.SEQ_STEP, dev, scratch=False)
        _written(state if new_state is None else new_state)
    return y


# ----------------------------------------------------------------------------
# selective state space scan
# ----------------------------------------------------------------------------
def _scan_forward(u, A, state, head, return_state, keep):
    """`head`: the argument block up to state."""
    y = _new(u)
    new = torch.empty((u.shape[0],) + tuple(A.shape), dtype=torch.float32, device=u.device) if return_state else None
    if u.numel() == 0:
        if return_state:
            new.copy_(state) if state is not None else new.zero_()
        return y, new, None
    segments = None
    if keep:
        lib = _lib.load()
        n = lib.auv_selective_scan_segments(_pack_scan(*head, *(0,) * 30) + _NO_ROOM)
        if n < 0:
            raise _lib.AuvError(n, lib.auv_seq_last_error().decode())
        segments = torch.empty(n // 4, dtype=torch.float32, device=u.device)
    block = _pack_scan(*head, _ptr(new), *_rows(y), _ptr(segments), *(0,) * 25)
    _call("auv_selective_scan", block, _lib.SEQ_FORWARD, head[0])
    return y, new, segments


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, Bm, Cm, D, z, delta_bias, state, start, lengths, head, return_state):
        _note_node(ctx)
        ctx.set_materialize_grads(False)
        y, new, segments = _scan_forward(u, A, state, head, return_state, True)
        ctx.save_for_backward(u, delta, A, Bm, Cm, D, z, delta_bias, state, start, lengths, segments)
        ctx.softplus = head[7]
        return y, new

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dnew):
        u, delta, A, Bm, Cm, D, z, delta_bias, state, start, lengths, segments = ctx.saved_tensors
        want = ctx.needs_input_grad
        rest = (None,) * 4
        if u.numel() == 0:
            out = [torch.zeros_like(t) if w else None
                   for t, w in zip((u, delta, A, Bm, Cm, D, z, delta_bias, state), want)]
            if want[8] and dnew is not None:
                out[8] = dnew.clone()
            return (*out, *rest)
        dy = _new(u).zero_() if dy is None else _adjacent(dy)
        dnew = None if dnew is None else dnew.contiguous()
        du, ddelta, dB, dC = _new(u), _new(delta), _new(Bm), _new(Cm)
        dz = None if z is None else _new(z)
        dA = torch.empty_like(A) if want[2] else None
        dD = torch.empty_like(D) if want[5] else None
        dbias = torch.empty_like(delta_bias) if want[7] else None
        dstate = torch.empty_like(state) if want[8] else None
        dev = u.get_device()
        block = _pack_scan(dev, TYPES[u.dtype], *u.shape, A.shape[1], Bm.shape[2], ctx.softplus, *_rows(u), *_rows(delta), *_rows(z),
                           *_groups(Bm), *_groups(Cm), A.data_ptr(), _ptr(D), _ptr(delta_bias), *_rows(start), _ptr(lengths), _ptr(state),
                           0, 0, 0, 0, segments.data_ptr(), *_rows(dy), _ptr(dnew), *_rows(du), *_rows(ddelta), *_rows(dz),
                           *_groups(dB), *_groups(dC), _ptr(dA), _ptr(dD), _ptr(dbias), _ptr(dstate))
        _call("auv_selective_scan", block, _lib.SEQ_BACKWARD, dev)
        return (*(g if w else None for g, w in zip((du, ddelta, dA, dB, dC, dD, dz, dbias, dstate), want)), *rest)


def _scan_head(u, shape, u_strides, dev, delta, A, Bm, Cm, D, z, delta_bias, start, lengths, state, softplus, state_needed):
    """The argument block up to state, in order, for rollouts [batch, length, channels] and for steps [batch, channels]."""
    lead, Dc, dtype = shape[:-1], shape[-1], u.dtype
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"A must be [channels, states] with 1 to {MAX_STATES} states")
    N = A.shape[1]
    a = _dense("A", A, (Dc, N), dev)
    ds = _like("delta", delta, shape, dtype, dev)
    zs = None if z is None else _like("z", z, shape, dtype, dev)
    if not isinstance(Bm, torch.Tensor) or Bm.dim() != len(shape) + 1 or Bm.shape[-2] < 1 or Dc % Bm.shape[-2]:
        raise ValueError("B must be [..., groups, states] with a number of groups that divides the channels")
    G = Bm.shape[-2]
    bs = _like("B", Bm, lead + (G, N), dtype, dev)
    cs = _like("C", Cm, lead + (G, N), dtype, dev)
    skip, bias = _dense("D", D, (Dc,), dev), _dense("delta_bias", delta_bias, (Dc,), dev)
    marks = _marks(start, lead, dev)
    n = _dense("lengths", lengths, lead[:1], dev, torch.int32)
    if state is None and state_needed:
        raise TypeError("state must be a tensor, got None")
    h = _dense("state", state, (lead[0], Dc, N), dev)
    if len(lead) == 2:
        row = lambda p, s: (p, s[0], s[1])            # noqa: E731
        group = lambda p, s: (p, s[0], s[1], s[2])    # noqa: E731
    else:
        row = lambda p, s: (p, s[0], 0)               # noqa: E731
        group = lambda p, s: (p, s[0], 0, s[1])       # noqa: E731
    return (dev, TYPES[dtype], lead[0], lead[1] if len(lead) == 2 else 1, Dc, N, G, 1 if softplus else 0,
            *row(u.data_ptr(), u_strides), *row(delta.data_ptr(), ds), *(row(z.data_ptr(), zs) if zs else (0, 0, 0)),
            *group(Bm.data_ptr(), bs), *group(Cm.data_ptr(), cs), a, skip, bias, *marks, n, h)


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
    shape, strides, dev = _first("u", u, 3, "[batch, length, channels]")
    head = _scan_head(u, shape, strides, dev, delta, A, B, C, D, z, delta_bias, start, lengths, state, delta_softplus, False)
    tensors = (u, delta, A, B, C, D, z, delta_bias, state)
    if _wants_grad(tensors):
        _check_capture(tensors)
        y, new = _Scan.apply(*tensors, start, lengths, head, bool(return_state))
    else:
        y, new, _ = _scan_forward(u, A, state, head, return_state, False)
    return (y, new) if return_state else y


def selective_scan_step(u, delta, state, A, B, C, D=None, z=None, delta_bias=None, *, delta_softplus=True, start=None,
                        new_state=None):
    """`selective_scan` of one token per row: u, delta, z [batch, channels]; B, C [batch, groups, N];
    `state` [batch, channels, N] moves on by the token, in place or into `new_state`.  (A state that a
    rollout's backward pass still needs is cloned first, or stepped into a `new_state`.)"""
    shape, strides, dev = _first("u", u, 2, "[batch, channels]")
    head = _scan_head(u, shape, strides, dev, delta, A, B, C, D, z, delta_bias, start, None, state, delta_softplus, True)
    _no_grad_here("selective_scan_step", (u, delta, state, A, B, C, D, z, delta_bias))
    to = head[-1]
    if new_state is not None and new_state is not state:
        to = _dense("new_state", new_state, state.shape, dev)
        _apart("new_state", new_state, "state", state)
    # (addresses and row strides as they lie in the block; an absent tensor's address is 0, below any state)
    (_, _, rows, _, chans, N, G, _, pu, su, _, pd, sd, _, pz, sz, _, pB, sB, _, gB, pC, sC, _, gC, pA, pD, pb, ps, ss) = head[:30]
    last, size, more = rows - 1 if rows else 0, u.element_size(), G - 1
    _in_place("the new state", to, state, (
        (pu, (last * su + chans) * size), (pd, (last * sd + chans) * size), (pz, (last * sz + chans) * size),
        (pB, (last * sB + more * gB + N) * size), (pC, (last * sC + more * gC + N) * size),
        (pA, 4 * chans * N), (pD, 4 * chans), (pb, 4 * chans), (ps, last * ss + 1)))
    y = _new(u)
    if shape[0] and shape[1]:
        block = _pack_scan(*head, to, y.data_ptr(), y.stride(0), 0, *(0,) * 26)
        _call("auv_selective_scan", block, _lib.SEQ_STEP, dev, scratch=False)
        _written(state if new_state is None else new_state)
    return y


# ----------------------------------------------------------------------------
# norms round a block
# ----------------------------------------------------------------------------
def _as_rows(t):
    """[..., channels] as [rows or batch, length, channels], without a copy where the strides allow one."""
    if t is None or t.dim() == 3:
        return t
    return t[None] if t.dim() == 2 else t.reshape(1, -1, t.shape[-1])


def _norm_head(x, y, post_weight, pre_weight, gate, scale, act, eps, dtype):
    """The argument block up to scale."""
    return (x.get_device(), TYPES[dtype], TYPES[x.dtype], *x.shape, act, eps, *_rows(x), *_rows(y), *_rows(gate), _ptr(post_weight),
            _ptr(pre_weight), _ptr(scale))


def _norm_forward(x, y, post_weight, pre_weight, gate, scale, act, eps, dtype):
    out = _new(x) if y is not None else None
    h = _new(x if y is None else y, dtype) if pre_weight is not None else None
    if x.numel():
        head = _norm_head(x, y, post_weight, pre_weight, gate, scale, act, eps, dtype)
        _call("auv_residual_norm", _pack_norm(*head, *_rows(out), *_rows(h), *(0,) * 18), _lib.SEQ_FORWARD, head[0], scratch=False)
    return out, h


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, post_weight, pre_weight, gate, scale, act, eps, dtype):
        _note_node(ctx)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, y, post_weight, pre_weight, gate, scale)
        ctx.how = (act, eps, dtype)
        return _norm_forward(x, y, post_weight, pre_weight, gate, scale, act, eps, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_h):
        x, y, post_weight, pre_weight, gate, scale = ctx.saved_tensors
        want = ctx.needs_input_grad
        rest = (None,) * 3
        if d_out is None and d_h is None or x.numel() == 0:
            return tuple(torch.zeros_like(t) if w else None
                         for t, w in zip((x, y, post_weight, pre_weight, gate, scale), want)) + rest
        d_out, d_h = _adjacent(d_out), _adjacent(d_h)
        dx = _new(x)
        dy = None if y is None else _new(y)
        dgate = None if gate is None else _new(gate)
        dpost = torch.empty_like(post_weight) if want[2] else None
        dpre = torch.empty_like(pre_weight) if want[3] else None
        dscale = torch.empty_like(scale) if want[5] else None
        head = _norm_head(x, y, post_weight, pre_weight, gate, scale, *ctx.how)
        block = _pack_norm(*head, 0, 0, 0, 0, 0, 0, *_rows(d_out), *_rows(d_h), *_rows(dx), *_rows(dy), *_rows(dgate),
                           _ptr(dpost), _ptr(dpre), _ptr(dscale))
        _call("auv_residual_norm", block, _lib.SEQ_BACKWARD, head[0])
        return tuple(g if w else None for g, w in zip((dx, dy, dpost, dpre, dgate, dscale), want)) + rest


def _norm(x, dev, y, post_weight, pre_weight, gate, scale, gate_act, eps, dtype):
    D = x.shape[-1]
    if D < 1 or D > _lib.NORM_MAX_CHANNELS:
        raise ValueError(f"1 to {_lib.NORM_MAX_CHANNELS} channels, got {D}")
    if not eps >= _LEAST:
        raise ValueError("eps must be positive in 32 bits")
    if gate_act not in GATES:
        raise ValueError(f"gate_act must be one of {tuple(GATES)}, got {gate_act!r}")
    _dense("post_weight", post_weight, (D,), dev)
    _dense("pre_weight", pre_weight, (D,), dev)
    _dense("scale", scale, (D,), dev)
    shape, act, eps = x.shape, GATES[gate_act], float(eps)
    tensors = (x, y, post_weight, pre_weight, gate, scale)
    if len(shape) != 3:
        x, y, gate = _as_rows(x), _as_rows(y), _as_rows(gate)
    if _wants_grad(tensors):
        _check_capture(tensors)
        out, h = _Norm.apply(x, y, post_weight, pre_weight, gate, scale, act, eps, dtype)
    else:
        out, h = _norm_forward(x, y, post_weight, pre_weight, gate, scale, act, eps, dtype)
    if len(shape) != 3:
        out, h = (t if t is None else t.reshape(shape) for t in (out, h))
    return out, h


def rms_norm(x, weight, *, eps=1e-6, dtype=None):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension, x [..., channels] (at most 8,192),
    as `dtype` (x's own by default; float32 x may give bfloat16 or float16): the norm before a
    first block.  Differentiable in x and weight."""
    _, _, dev = _first("x", x, None, None)
    if weight is None:
        raise TypeError("weight must be a tensor, got None")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in TYPES or (x.dtype != torch.float32 and x.dtype != dtype):
        raise TypeError(f"a norm of {x.dtype} cannot be {dtype}")
    return _norm(x, dev, None, None, weight, None, None, None, eps, dtype)[1]


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
    shape, _, dev = _first("x", x, None, None)
    if not isinstance(y, torch.Tensor):
        raise TypeError(f"y must be a tensor, got {type(y).__name__}")
    if y.dtype not in TYPES or x.dtype not in (torch.float32, y.dtype):
        raise TypeError(f"x must be float32 or of y's type, got {x.dtype} and {y.dtype}")
    _like("y", y, shape, y.dtype, dev)
    if gate is not None:
        _like("gate", gate, shape, y.dtype, dev)
    return _norm(x, dev, y, post_weight, pre_weight, gate, scale, gate_act, eps, y.dtype)


# ----------------------------------------------------------------------------
# the operators strung together
# ----------------------------------------------------------------------------
class _Layer(nn.Module):
    # What is learned per channel, the rank of the step width and the first values are those of the published method (A. Gu
    # and T. Dao, Linear-Time Sequence Modeling with Selective State Spaces, 2023), whose arguments selective_scan takes.
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
    and gives ([batch, length, channels], state behind the rows), zeros behind each row's
    last token (`lengths`); `step(features, state,
    start=None)` takes [batch, features], gives [batch, channels] and moves `state`
    (`new_state(batch)`, or one that forward gave) on in place: clone one that a backward
    pass still needs.  Both compute the same function: a rollout stepped token by token and
    the rollout at once agree to rounding.  Types are those of `dtype` under torch.autocast too."""

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
        if torch.is_autocast_enabled():                # the types are the module's own
            with torch.autocast("cuda", enabled=False):
                return self._run(features.to(self.enter.weight.dtype), mixers)
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

        real = None
        if lengths is not None:
            # the layers between the operators know no lengths: what lies behind a row's last token goes in as zeros, so that
            # no gradient of a parameter sees it, and comes out as zeros
            real = (torch.arange(features.shape[1], device=features.device) < lengths[:, None])[..., None]
            features = torch.where(real, features, 0)
        h = self._run(features, [mixer(layer, None if state is None else state[i]) for i, layer in enumerate(self.layers)])
        return h if real is None else torch.where(real, h, 0), [tuple(s) for s in out]

    @torch.no_grad()
    def step(self, features, state, start=None):
        def mixer(layer, s):
            def conv(u):
                return causal_conv_step(u, s[0], layer.conv_weight, layer.conv_bias, start=start)

            def scan(u, delta, A, B, C, z):
                return selective_scan_step(u, delta, s[1], A, B, C, layer.D, z, layer.delta_bias, start=start)
            return conv, scan

        return self._run(features, [mixer(layer, state[i]) for i, layer in enumerate(self.layers)])
