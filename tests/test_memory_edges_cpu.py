"""The sequence operators at the edges of what they take, as far as no GPU is needed to see it."""
import ctypes as C

import pytest
import torch

from gym_auv_amd import _lib, memory
from tests.test_memory_cpu import FAKE, conv_args, norm_args, scan_args


def test_tracing_is_refused():
    """Before anything else is looked at: a trace would hold no kernel."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x, w = torch.zeros(2, 3, 8), torch.zeros(8, 4)
    for call in (lambda t: memory.causal_conv(t, w), lambda t: memory.causal_conv_step(t[:, 0], t, w),
                 lambda t: memory.selective_scan(t, t, w, t, t), lambda t: memory.selective_scan_step(t[:, 0], t[:, 0], t, w, t, t),
                 lambda t: memory.residual_norm(t, t), lambda t: memory.rms_norm(t, w[:, 0])):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (x,), check_trace=False)
        for pre in (False, True):
            with pytest.raises(RuntimeError, match="traced"):
                make_fx(call, pre_dispatch=pre)(x)
        with pytest.raises(ValueError, match="CUDA"):
            call(x)


@pytest.mark.parametrize("shape", [dict(batch=0), dict(length=0), dict(batch=0, length=0)], ids=str)
def test_empty_batches_at_the_c_entry(lib, shape):
    """A planned launch of nothing: sizes of 0 and, backwards, a refusal, in every pass that takes them."""
    for fn, args in (("auv_causal_conv", conv_args), ("auv_selective_scan", scan_args), ("auv_residual_norm", norm_args)):
        a = args(**shape, d_y=FAKE, d_x=FAKE) if fn != "auv_selective_scan" else args(
            **shape, segments=FAKE, d_y=FAKE, d_u=FAKE, d_delta=FAKE, d_B=FAKE, d_C=FAKE)
        for what in (_lib.SEQ_FORWARD, _lib.SEQ_BACKWARD):
            assert getattr(lib, fn + "_workspace")(C.byref(a), what) == 0
        assert getattr(lib, fn)(C.byref(a), _lib.SEQ_FORWARD, None) == 0
        assert getattr(lib, fn)(C.byref(a), _lib.SEQ_BACKWARD, None) == -1
        assert b"empty batch" in lib.auv_seq_last_error()
    assert lib.auv_selective_scan_segments(C.byref(scan_args(**shape))) == 0


def test_launches_stay_within_a_grid(tmp_path):
    """The spread of workgroups over launches (csrc/auv_slices.hpp), built for the host and checked there."""
    import os
    import shutil
    import subprocess

    if shutil.which("g++") is None:
        pytest.skip("no g++")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "slices_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(root, "gym-auv_amd", "csrc"), "-o", exe,
                    os.path.join(root, "tests", "native", "slices_check.cpp")], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout.startswith("slices ok"), run.stdout + run.stderr
