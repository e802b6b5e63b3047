"""The sequence operators at the edges of what they take, as far as no GPU is needed to see it."""
import pytest
import torch

from gym_auv_amd import memory


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
