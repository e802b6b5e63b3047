"""The sequence operators' refusals, before any GPU is touched: the C entry points check their
arguments first, and the Python side refuses what the kernels cannot take.  Also the oracle itself:
its gradients against differences of its values."""
import ctypes as C

import numpy as np
import pytest
import torch

from gym_auv_amd import _lib, memory
from oracle import seq_oracle as O

FAKE = 1 << 20    # a non-null address: every call here is refused before anything is read


def conv_args(**kw):
    a = _lib.AuvConvArgs(device=0, dtype=_lib.BF16, batch=2, length=3, channels=8, width=4, x=FAKE, weight=FAKE, y=FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def scan_args(**kw):
    a = _lib.AuvScanArgs(device=0, dtype=_lib.F32, batch=2, length=3, channels=8, states=4, groups=1, u=FAKE, delta=FAKE, B=FAKE,
                         C=FAKE, A=FAKE, y=FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def norm_args(**kw):
    a = _lib.AuvNormArgs(device=0, dtype=_lib.BF16, residual_dtype=_lib.F32, batch=2, length=3, channels=8, eps=1e-6, x=FAKE,
                         y=FAKE, x_out=FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_argument_blocks_have_the_headers_fields():
    """Names and order of every member of the three argument structs, and their kinds, from the header text."""
    import os
    import re

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "auvsim.h")).read()
    for name, cls in (("auv_conv_args", _lib.AuvConvArgs), ("auv_scan_args", _lib.AuvScanArgs), ("auv_norm_args", _lib.AuvNormArgs)):
        body = re.search(r"typedef struct %s\s*\{(.*?)\}\s*%s;" % (name, name), text, flags=re.S).group(1)
        want = []
        for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
            m = re.match(r"\s*(const\s+)?(\w+)\s*(\*?)\s*(.*)$", decl.strip(), flags=re.S)
            if not m or not m.group(4):
                continue
            kind = C.c_void_p if m.group(3) else {"int64_t": C.c_int64, "double": C.c_double}[m.group(2)]
            want += [(f.strip(), kind) for f in m.group(4).split(",")]
        assert cls._fields_ == want, name


@pytest.mark.parametrize("fn,args,what,match", [
    ("auv_causal_conv", conv_args(width=5), _lib.SEQ_FORWARD, "width"),
    ("auv_causal_conv", conv_args(width=1), _lib.SEQ_FORWARD, "width"),
    ("auv_causal_conv", conv_args(dtype=_lib.F64), _lib.SEQ_FORWARD, "f32, bf16 or f16"),
    ("auv_causal_conv", conv_args(channels=0), _lib.SEQ_FORWARD, "bad shape"),
    ("auv_causal_conv", conv_args(batch=-1), _lib.SEQ_FORWARD, "bad shape"),
    ("auv_causal_conv", conv_args(batch=1 << 39, length=1 << 39), _lib.SEQ_FORWARD, "bad shape"),
    ("auv_causal_conv", conv_args(weight=None), _lib.SEQ_FORWARD, "null weight"),
    ("auv_causal_conv", conv_args(x=None), _lib.SEQ_FORWARD, "null x"),
    ("auv_causal_conv", conv_args(y=None), _lib.SEQ_FORWARD, "null y"),
    ("auv_causal_conv", conv_args(), 7, "unknown pass"),
    ("auv_causal_conv", conv_args(), _lib.SEQ_STEP, "one token per row"),
    ("auv_causal_conv", conv_args(length=1), _lib.SEQ_STEP, "state and new_state"),
    ("auv_causal_conv", conv_args(state=FAKE, new_state=FAKE), _lib.SEQ_FORWARD, "state's memory"),
    ("auv_causal_conv", conv_args(), _lib.SEQ_BACKWARD, "d_y or d_x"),
    ("auv_causal_conv", conv_args(d_y=FAKE, d_x=FAKE, d_weight=FAKE), _lib.SEQ_BACKWARD, "workspace"),
    ("auv_selective_scan", scan_args(states=65), _lib.SEQ_FORWARD, "states"),
    ("auv_selective_scan", scan_args(states=0), _lib.SEQ_FORWARD, "states"),
    ("auv_selective_scan", scan_args(groups=3), _lib.SEQ_FORWARD, "divide"),
    ("auv_selective_scan", scan_args(groups=0), _lib.SEQ_FORWARD, "divide"),
    ("auv_selective_scan", scan_args(A=None), _lib.SEQ_FORWARD, "null argument"),
    ("auv_selective_scan", scan_args(y=None), _lib.SEQ_FORWARD, "null y"),
    ("auv_selective_scan", scan_args(length=1), _lib.SEQ_STEP, "state and new_state"),
    ("auv_selective_scan", scan_args(state=FAKE, new_state=FAKE), _lib.SEQ_FORWARD, "state's memory"),
    ("auv_selective_scan", scan_args(segments=FAKE + 4), _lib.SEQ_FORWARD, "aligned"),
    ("auv_selective_scan", scan_args(), _lib.SEQ_BACKWARD, "gradient or segments"),
    ("auv_selective_scan", scan_args(length=4096), _lib.SEQ_FORWARD, "workspace"),
    ("auv_selective_scan", scan_args(batch=1 << 36, length=1, state=FAKE, new_state=FAKE + 4096), _lib.SEQ_STEP, "too large"),
    ("auv_residual_norm", norm_args(), _lib.SEQ_STEP, "unknown pass"),
    ("auv_residual_norm", norm_args(channels=8193), _lib.SEQ_FORWARD, "at most 8192"),
    ("auv_residual_norm", norm_args(eps=0.0), _lib.SEQ_FORWARD, "eps"),
    ("auv_residual_norm", norm_args(eps=float("nan")), _lib.SEQ_FORWARD, "eps"),
    ("auv_residual_norm", norm_args(residual_dtype=_lib.F16), _lib.SEQ_FORWARD, "residual"),
    ("auv_residual_norm", norm_args(gate_act=3), _lib.SEQ_FORWARD, "activation"),
    ("auv_residual_norm", norm_args(x=None), _lib.SEQ_FORWARD, "null x"),
    ("auv_residual_norm", norm_args(x_out=None), _lib.SEQ_FORWARD, "x_out"),
    ("auv_residual_norm", norm_args(pre_weight=FAKE), _lib.SEQ_FORWARD, "h goes with"),
    ("auv_residual_norm", norm_args(y=None, x_out=None, gate=FAKE), _lib.SEQ_FORWARD, "belong to y"),
    ("auv_residual_norm", norm_args(y=None, x_out=None), _lib.SEQ_FORWARD, "neither"),
    ("auv_residual_norm", norm_args(), _lib.SEQ_BACKWARD, "null gradient"),
    ("auv_residual_norm", norm_args(d_x=FAKE, d_y=FAKE), _lib.SEQ_BACKWARD, "neither"),
    ("auv_residual_norm", norm_args(d_x=FAKE, d_y=FAKE, d_x_out=FAKE, d_scale=FAKE), _lib.SEQ_BACKWARD, "workspace"),
])
def test_c_entry_points_refuse(lib, fn, args, what, match):
    rc = getattr(lib, fn)(C.byref(args), what, None)
    assert rc < 0 and match in lib.auv_seq_last_error().decode()


def test_an_eps_that_vanishes_in_32_bits_is_refused(lib):
    """A row of zeros would divide by it."""
    assert lib.auv_residual_norm(C.byref(norm_args(eps=1e-60)), _lib.SEQ_FORWARD, None) < 0
    assert b"eps" in lib.auv_seq_last_error()
    assert lib.auv_residual_norm_workspace(C.byref(norm_args(eps=1e-60)), _lib.SEQ_BACKWARD) < 0


def test_c_entry_points_refuse_null_blocks(lib):
    for fn in ("auv_causal_conv", "auv_selective_scan", "auv_residual_norm"):
        assert getattr(lib, fn)(None, 0, None) == -1
        assert getattr(lib, fn + "_workspace")(None, 0) == -1
    assert lib.auv_selective_scan_segments(None) == -1


def test_workspaces_and_segments(lib):
    # 16 states kept before tokens 0, 16, 32: 3 x 2 rows x 8 channels x 16 x 4 bytes
    assert lib.auv_selective_scan_segments(C.byref(scan_args(length=33, states=13))) == 3 * 2 * 8 * 16 * 4
    assert lib.auv_selective_scan_workspace(C.byref(scan_args()), _lib.SEQ_FORWARD) == 0
    assert lib.auv_selective_scan_workspace(C.byref(scan_args(length=4096)), _lib.SEQ_FORWARD) > 0
    assert lib.auv_selective_scan_workspace(C.byref(scan_args()), _lib.SEQ_BACKWARD) > 0
    assert lib.auv_causal_conv_workspace(C.byref(conv_args()), _lib.SEQ_FORWARD) == 0
    assert lib.auv_causal_conv_workspace(C.byref(conv_args()), _lib.SEQ_BACKWARD) > 0
    assert lib.auv_residual_norm_workspace(C.byref(norm_args()), _lib.SEQ_BACKWARD) > 0
    # a batch without rows or tokens needs none and is no error forwards
    assert lib.auv_causal_conv(C.byref(conv_args(batch=0)), _lib.SEQ_FORWARD, None) == 0
    assert lib.auv_selective_scan(C.byref(scan_args(length=0)), _lib.SEQ_FORWARD, None) == 0
    assert lib.auv_residual_norm(C.byref(norm_args(batch=0)), _lib.SEQ_FORWARD, None) == 0


def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 3, 8), torch.zeros(8, 4)
    with pytest.raises(ValueError, match="CUDA"):
        memory.causal_conv(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        memory.causal_conv_step(x[:, 0], x[:, :3], w)
    with pytest.raises(ValueError, match="CUDA"):
        memory.selective_scan(x, x, w, x, x)
    with pytest.raises(ValueError, match="CUDA"):
        memory.selective_scan_step(x[:, 0], x[:, 0], x, w, x, x)
    with pytest.raises(ValueError, match="CUDA"):
        memory.residual_norm(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        memory.rms_norm(x, w[:, 0])
    with pytest.raises(TypeError, match="tensor"):
        memory.causal_conv(None, w)
    with pytest.raises(ValueError, match="width"):
        memory.EpisodeMemory(18, width=5)
    with pytest.raises(TypeError, match="dtype"):
        memory.EpisodeMemory(18, dtype=torch.float64)


def _difference(f, x, gy, eps=1e-6):
    """d (sum gy f(x)) / dx by central differences, over every element of x."""
    g = np.zeros_like(x)
    flat, out = x.reshape(-1), g.reshape(-1)
    for i in range(flat.size):
        keep = flat[i]
        flat[i] = keep + eps
        hi = sum((a * b).sum() for a, b in zip(f(), gy))
        flat[i] = keep - eps
        lo = sum((a * b).sum() for a, b in zip(f(), gy))
        flat[i] = keep
        out[i] = (hi - lo) / (2 * eps)
    return g


def test_oracle_gradients_against_differences():
    """Central differences of 64-bit sums of magnitude M: off by M (2^-53 / 1e-6 + third derivative 1e-12) < 1e-8 M."""
    rng = np.random.default_rng(0)
    B, L, D, W, N, G = 2, 5, 4, 3, 3, 2
    start = rng.random((B, L)) < 0.3
    lengths = np.array([5, 3])
    x, w, b, s = rng.normal(size=(B, L, D)), rng.normal(size=(D, W)), rng.normal(size=D), rng.normal(size=(B, W - 1, D))
    gy, gs = rng.normal(size=(B, L, D)), rng.normal(size=(B, W - 1, D))
    run = lambda: [O.conv(x, w, b, start, lengths, s)[k][0] for k in ("y", "new_state")]   # noqa: E731
    got = O.conv(x, w, b, start, lengths, s, dy=gy, dnew=gs)
    for name, t in (("x", x), ("weight", w), ("bias", b), ("state", s)):
        assert np.abs(got[name][0] - _difference(run, t, (gy, gs))).max() < 1e-7, name
    u, delta, z = (rng.normal(size=(B, L, D)) for _ in range(3))
    Bm, Cm = rng.normal(size=(B, L, G, N)), rng.normal(size=(B, L, G, N))
    A, Dv, db, h0 = -np.exp(rng.normal(size=(D, N))), rng.normal(size=D), rng.normal(size=D), rng.normal(size=(B, D, N))
    gh = rng.normal(size=(B, D, N))
    run = lambda: [O.scan(u, delta, A, Bm, Cm, Dv, z, db, True, start, lengths, h0)[k][0] for k in ("y", "new_state")]   # noqa: E731
    got = O.scan(u, delta, A, Bm, Cm, Dv, z, db, True, start, lengths, h0, dy=gy, dnew=gh)
    for name, t in (("u", u), ("delta", delta), ("A", A), ("B", Bm), ("C", Cm), ("D", Dv), ("z", z), ("delta_bias", db), ("state", h0)):
        assert np.abs(got[name][0] - _difference(run, t, (gy, gh))).max() < 1e-7, name
    r, y, g = (rng.normal(size=(3, D)) for _ in range(3))
    w1, w2, sc = (rng.normal(size=D) for _ in range(3))
    g1, g2 = rng.normal(size=(3, D)), rng.normal(size=(3, D))
    for act in ("silu", "sigmoid", None):
        run = lambda: [O.norm(r, y, w1, w2, g, sc, act)[k][0] for k in ("x_out", "h")]   # noqa: E731
        got = O.norm(r, y, w1, w2, g, sc, act, dx_out=g1, dh=g2)
        for name, t in (("x", r), ("y", y), ("post_weight", w1), ("pre_weight", w2), ("gate", g), ("scale", sc)):
            assert np.abs(got[name][0] - _difference(run, t, (g1, g2))).max() < 1e-7, (act, name)
