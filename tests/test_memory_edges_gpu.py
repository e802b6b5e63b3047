"""The sequence operators at the edges of what they take: values that are not finite, states that vanish or
grow, sizes beyond one launch, and calls that other torch machinery makes."""
import numpy as np
import pytest

from oracle import seq_oracle as O
from tests.test_memory_gpu import TYPES, Maker, check, host, hostb, lengths_of, scan_case, torch_

pytestmark = pytest.mark.gpu

SCAN_ARGS = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")


def finite_alike(name, got, want, K):
    """`got` is finite exactly where the definition is a number that got's type holds, and within its bound there.  (A state
    that grows by 2^134 hands back gradients beyond 2^128, which 64 bits hold and 32 do not.)"""
    import torch

    value, magnitude = want
    fin = np.abs(value) <= torch.finfo(got.dtype).max           # (false for NaN)
    have = torch.isfinite(got.detach()).cpu().numpy()
    same = np.array_equal(have, fin)
    assert same, (name, "finite:", int(have.sum()), "should be:", int(fin.sum()), "of", fin.size, "first at",
                                       tuple(int(i) for i in np.argwhere(have != fin)[0]))
    keep = torch.from_numpy(fin).to(got.device)
    check(name, torch.where(keep, got.detach(), torch.zeros_like(got)),
          (np.where(fin, value, 0.0), np.where(fin, np.nan_to_num(magnitude, nan=0.0, posinf=0.0), 0.0)), K)


def raw_scan(t, start, n, gy, gs, softplus):
    """The oracle on the values as they are, with nothing cleaned."""
    v = {k: host(x) for k, x in t.items()}
    with np.errstate(all="ignore"):
        return O.scan(*(v[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")), softplus, hostb(start),
                      None if n is None else n.cpu().numpy(), v["state"], host(gy), host(gs))


def run_scan(t, start, n, gy, gs, softplus):
    torch = torch_()
    from gym_auv_amd import memory

    t = {k: None if v is None else v.detach().requires_grad_(True) for k, v in t.items()}
    y, new = memory.selective_scan(*(t[k] for k in SCAN_ARGS), delta_softplus=softplus, start=start, lengths=n, state=t["state"],
                                   return_state=True)
    names = [k for k, v in t.items() if v is not None]
    return dict(y=y, new_state=new, **dict(zip(names, torch.autograd.grad([y, new], [t[k] for k in names], [gy, gs]))))


# ----------------------------------------------------------------------------
# rows cut into chunks: what one chunk hands to the next
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("where", ["u", "state", "d_y", "d_state"])
def test_what_is_not_finite_goes_on_to_the_next_start(where, bad):
    """A decays every state by e^-8 a token, by e^-128 (0 in 32 bits) over 16 tokens: a value that is not finite still
    stays until an episode starts, forwards, and back to the episode's first token, backwards."""
    torch = torch_()
    m = Maker(31, "float32", "time")
    B, L, D, N = 2, 700, 20, 16
    t, _, _ = scan_case(m, B, L, D, N, 1, None, None, True, True)
    t["A"] = torch.full_like(t["A"], -16.0)
    t["delta"], t["delta_bias"] = torch.full_like(t["delta"], 0.5), None
    t = {k: None if v is None else v.detach() for k, v in t.items()}
    gy, gs = m.rows(B, L, D), m.par(B, D, N)
    start = torch.zeros(B, L, dtype=torch.bool, device="cuda")
    start[0, 400], start[1, 200] = True, True
    put = {"u": t["u"], "state": t["state"], "d_y": gy, "d_state": gs}[where]
    if where == "u":
        put[0, 3, 5] = float(bad)
    elif where == "d_y":
        put[0, 650, 5] = float(bad)
    else:
        put[0, 5, 2] = float(bad)
    got, want = run_scan(t, start, None, gy, gs, False), raw_scan(t, start, None, gy, gs, False)
    K = 10 * (L + N + 12)
    assert not np.isfinite(want["y" if where in ("u", "state") else "u"][0][0]).all()
    for name in ("y", "new_state"):
        finite_alike(name, got[name], want[name], K)
    for name in ("u", "delta", "z", "B", "C", "A", "D", "state"):
        finite_alike("d_" + name, got[name], want[name], 2 * K + (B * L if name in ("A", "D") else D))


@pytest.mark.parametrize("B,L", [(2, 700), (1, 4200)])
def test_states_that_grow(B, L):
    """e^8 a token, beyond 32 bits over 16 tokens: states that are 0 stay 0, backwards too, until something feeds them."""
    torch = torch_()
    m = Maker(32, "float32", "time")
    D, N = 20, 16
    t, _, _ = scan_case(m, B, L, D, N, 1, None, None, False, True)
    t = {k: None if v is None else v.detach() for k, v in t.items()}
    t["A"], t["delta"], t["delta_bias"] = torch.full_like(t["A"], 16.0), torch.full_like(t["delta"], 0.5), None
    t["u"][:, :-3] = 0
    gy, gs = m.rows(B, L, D), torch.zeros(B, D, N, device="cuda")
    gy[:, 3:] = 0
    got, want = run_scan(t, None, None, gy, gs, False), raw_scan(t, None, None, gy, gs, False)
    # (three tokens that grow: each exponent 8 log2(e) = 11.5 rounded twice, a relative 2 x 8 of a step each)
    K = 10 * (L + N + 12) + 3 * 16
    for name in got:
        assert np.isfinite(want[name][0]).all()
        finite_alike(name, got[name], want[name], 2 * K + B * L)


def test_a_state_that_grows_by_more_than_32_bits_hold():
    """By 2^134 within a chunk, from 1e-30 to 2e10: the product of the decays alone is no number."""
    torch = torch_()
    m = Maker(33, "float32", "time")
    B, L, D, N = 1, 100, 20, 16
    t, _, _ = scan_case(m, B, L, D, N, 1, None, None, True, True)
    t = {k: None if v is None else v.detach() for k, v in t.items()}
    t["A"], t["delta"], t["delta_bias"] = torch.full_like(t["A"], 11.6), torch.zeros_like(t["delta"]), None
    t["delta"][:, :16] = 0.5
    t["u"][:] = 0
    t["state"] = torch.full_like(t["state"], 1e-30)
    gy, gs = m.rows(B, L, D), m.par(B, D, N)
    gy[:, 16:] *= 1e-20
    gs *= 1e-20
    got, want = run_scan(t, None, None, gy, gs, False), raw_scan(t, None, None, gy, gs, False)
    # sixteen tokens whose exponents, 8.4 each, are rounded twice; over a chunk one exponent of 134, rounded 18 times
    K = 10 * (L + N + 12) + 16 * 2 * 8 + 18 * 134
    # (one term of dA is d_state times the state before the row: nothing where 32 bits do not hold d_state)
    held = np.abs(want["state"][0]) <= np.finfo(np.float32).max
    assert held.any() and not held.all()
    want["A"] = tuple(np.where(held[0], v, np.nan) for v in want["A"])
    for name in ("y", "new_state", "state", "A", "C"):
        finite_alike(name, got[name], want[name], 2 * K + B * L)


# ----------------------------------------------------------------------------
# behind a row's last token
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [3, 7, 16, 20, 64])
@pytest.mark.parametrize("bad", ["state", "d_state"])
def test_padding_takes_no_gradient_of_states_that_are_not_finite(bad, N, dtype):
    torch = torch_()
    m = Maker(34, dtype, "time")
    B, L, D = 3, 37, 24
    t, _, _ = scan_case(m, B, L, D, N, 2, None, None, True, True)
    t = {k: None if v is None else v.detach() for k, v in t.items()}
    gy, gs = m.rows(B, L, D), m.par(B, D, N)
    n = torch.tensor([L, 5, 18], dtype=torch.int32, device="cuda")
    {"state": t["state"], "d_state": gs}[bad][:, ::5, 1] = float("inf")
    got = run_scan(t, None, n, gy, gs, True)
    for b, k in enumerate(n.tolist()):
        for name in ("y", "u", "delta", "z", "B", "C"):
            assert not got[name][b, k:].any(), (name, b)        # (NaN is true)


@pytest.mark.parametrize("L,ragged", [(20, False), (33, False), (40, True), (32, False)])
def test_a_state_that_overflows_with_the_rows_last_token(L, ragged):
    """The gradients of what came before are finite, A's among them: nothing behind the row's end adds to them."""
    torch = torch_()
    m = Maker(35, "float32", "time")
    B, D, N = 2, 20, 16
    t, _, _ = scan_case(m, B, L, D, N, 1, None, None, True, True)
    t = {k: None if v is None else v.detach() for k, v in t.items()}
    n = torch.tensor([23, L], dtype=torch.int32, device="cuda") if ragged else None
    last = 22 if ragged else L - 1
    t["delta"][0, last, 5], t["delta_bias"][5] = 3.0, 0.0
    t["u"][0, last, 5], t["B"][0, last, 0, 2] = 3e38, 100.0
    gy, gs = m.rows(B, L, D), m.par(B, D, N)
    got, want = run_scan(t, None, n, gy, gs, True), raw_scan(t, None, n, gy, gs, True)
    assert np.isfinite(want["A"][0]).all() and np.abs(want["A"][0]).max() < 1e30
    K = 10 * (L + N + 12)
    # (the ones that are not a product with dt u of that token, 9e38)
    for name in ("A", "u", "delta", "D", "delta_bias", "state"):
        finite_alike(name, got[name], want[name], 2 * K + B * L)


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_last_token_that_is_not_finite_meets_its_own_taps_only(W, dtype):
    """Without the SiLU the weight gradient is a sum of d_y x: the last token of a row meets the last tap only."""
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(36, dtype, "time")
    B, L, D = 3, 21, 24
    x = m.rows(B, L, D)
    n = torch.tensor([L, 9, 16], dtype=torch.int32, device="cuda")
    for b, k in enumerate(n.tolist()):
        x[b, k - 1, 3 + b] = float("inf")
    x.requires_grad_(True)
    w, b = m.par(D, W).requires_grad_(True), m.par(D).requires_grad_(True)
    gy = m.rows(B, L, D)
    y = memory.causal_conv(x, w, b, lengths=n, silu=False)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], gy)
    with np.errstate(all="ignore"):
        want = O.conv(host(x), host(w), host(b), None, n.cpu().numpy(), None, False, host(gy))
    assert np.isfinite(want["weight"][0][:, :-1]).all() and not np.isfinite(want["weight"][0][:, -1]).all()
    # (the oracle's magnitudes of gradients hold those of the pre-activations, which without the SiLU the gradients do not
    # depend on: they are taken from the row with zeros in place of its infinities)
    clean = O.conv(np.where(np.isinf(host(x)), 0.0, host(x)), host(w), host(b), None, n.cpu().numpy(), None, False, host(gy))
    for name in ("x", "weight", "bias"):
        want[name] = (want[name][0], clean[name][1])
    K = W + 2 + 8
    for name, g in (("y", y), ("x", dx), ("weight", dw), ("bias", db)):
        finite_alike(name, g, want[name], 2 * K + W + B * L)


# ----------------------------------------------------------------------------
# calls that other torch machinery makes
# ----------------------------------------------------------------------------
def test_a_state_that_was_stepped_on_is_no_good_for_backward_any_more():
    """A rollout from a state keeps it for its backward pass; a step that moves it on in place is such a change as
    torch's own in-place operations make, and backward says so."""
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(37, "float32")
    B, L, D, N = 2, 5, 8, 4
    t, _, _ = scan_case(m, B, L, D, N, 1, None, None, True, True)
    t = {k: None if v is None else v.detach() for k, v in t.items()}
    u, w = t["u"].requires_grad_(True), m.par(D, 4)
    scan = [u] + [t[k] for k in SCAN_ARGS[1:]]
    token = [v.detach()[:, 0] if v.dim() > 2 else v for v in scan]
    conv_state, conv_other, scan_state, scan_other = m.rows(B, 3, D), m.rows(B, 3, D), t["state"], m.par(B, D, N)
    conv = lambda s: memory.causal_conv(u, w, state=s).sum()                                            # noqa: E731
    rows = lambda s: memory.selective_scan(*scan, state=s).sum()                                        # noqa: E731
    step_conv = lambda s, to: memory.causal_conv_step(u.detach()[:, 0], s, w, new_state=to)             # noqa: E731
    step_rows = lambda s, to: memory.selective_scan_step(*token[:2], s, *token[2:], new_state=to)       # noqa: E731
    for call, step, state, other in ((conv, step_conv, conv_state, conv_other), (rows, step_rows, scan_state, scan_other)):
        for s, to in ((state, None), (other, other)):        # moved on in place; written as the new state of another
            y = call(s)
            before = s._version
            step(state if to is not None else s, to)
            assert s._version > before
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
        y = call(state)
        step(state, other)                                   # the old state is left as it was
        y.backward()
    net = memory.EpisodeMemory(6, 8, states=4).cuda()
    x = torch.randn(B, L, 6, device="cuda")
    with torch.no_grad():
        _, s = net(x)
    h, _ = net(x, state=s)
    net.step(x[:, 0], s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def _calls():
    """Each public call with a first argument of our choice: (name, shape of that argument, call)."""
    from gym_auv_amd import memory

    m = Maker(38, "float32")
    B, L, D, N = 2, 5, 8, 4
    w, wn, A = m.par(D, 4), m.par(D), -m.par(D, N).abs()
    x, bc = m.rows(B, L, D), m.rows(B, L, 1, N)
    return [
        ("causal_conv", (B, L, D), lambda t: memory.causal_conv(t, w)),
        ("causal_conv weight", (D, 4), lambda t: memory.causal_conv(x, t)),
        ("causal_conv_step", (B, D), lambda t: memory.causal_conv_step(t, m.rows(B, 3, D), w)),
        ("selective_scan", (B, L, D), lambda t: memory.selective_scan(t, x, A, bc, bc)),
        ("selective_scan z", (B, L, D), lambda t: memory.selective_scan(x, x, A, bc, bc, z=t)),
        ("selective_scan_step", (B, D), lambda t: memory.selective_scan_step(t, x[:, 0], m.par(B, D, N), A, bc[:, 0], bc[:, 0])),
        ("residual_norm", (B, L, D), lambda t: memory.residual_norm(t, x, wn)),
        ("residual_norm of rows", (B, D), lambda t: memory.residual_norm(x[:, 0], t, wn)),
        ("rms_norm", (B, L, D), lambda t: memory.rms_norm(t, wn)),
        ("rms_norm weight", (D,), lambda t: memory.rms_norm(x, t)),
    ]


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(grad):
    """None of the calls has them; without an error the tangent would be gone in silence."""
    torch = torch_()
    import torch.autograd.forward_ad as fwd

    for name, shape, call in _calls():
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            call(torch.ones(shape, device="cuda"))                                    # nothing has a tangent: computed
            dual = fwd.make_dual(torch.ones(shape, device="cuda"), torch.ones(shape, device="cuda"))
            with pytest.raises(NotImplementedError, match="forward"):
                call(dual)
                raise AssertionError(name)


def test_tracing_is_refused():
    """A trace would record the memory for the results and not the kernels that fill it."""
    torch = torch_()
    from torch.fx.experimental.proxy_tensor import make_fx

    for name, shape, call in _calls():
        x = torch.ones(shape, device="cuda")
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (x,), check_trace=False)
            raise AssertionError(name)
        for pre in (False, True):
            with pytest.raises(RuntimeError, match="traced"):
                make_fx(call, pre_dispatch=pre)(x)
                raise AssertionError(name)
        call(x)


def test_compiled_code_runs_the_calls():
    """torch.compile cannot look into them: it breaks its graph there, and the results are the eager ones."""
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(39, "float32")
    x, w = m.rows(2, 5, 8), m.par(8, 4)
    fn = lambda t: memory.causal_conv(t * 2.0, w) + 1.0          # noqa: E731
    a, b = (x.clone().requires_grad_(True) for _ in range(2))
    got, want = torch.compile(fn, backend="eager")(a), fn(b)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got.sum(), a)[0], torch.autograd.grad(want.sum(), b)[0])


# ----------------------------------------------------------------------------
# sizes beyond one launch
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("rows,D", [(4_194_303 + 70, 2056), (16_777_215 + 90, 520), ((1 << 30) + 130, 4)])
def test_norm_of_more_rows_than_one_launch_takes(rows, D):
    """A row takes a workgroup of 1,024 or 256 threads, or a 64th of one: 2^32 threads and more."""
    torch = torch_()
    from gym_auv_amd import memory

    torch.manual_seed(8)
    x = torch.zeros(rows, D, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(D, device="cuda")
    at = [0, rows - 131, rows - 100, rows - 71, rows - 70, rows - 69, rows - 5, rows - 1]
    at = torch.tensor([i for i in at if 0 <= i], device="cuda")
    x[at] = torch.randn(len(at), D, device="cuda").bfloat16()
    h = memory.rms_norm(x, w)
    assert torch.equal(h[at], memory.rms_norm(x[at], w))
    assert int(torch.count_nonzero(h[-200:].any(1))) == len(at) - 1 and not h[1:1000].any()


def test_scan_of_more_waves_than_one_launch_takes():
    """A group of one channel takes a wave of its own: 2^26 of them and more."""
    torch = torch_()
    from gym_auv_amd import memory

    torch.manual_seed(9)
    B, D = (1 << 20) + 33, 64
    u, delta, bc = torch.zeros(B, 1, D, device="cuda"), torch.zeros(B, 1, D, device="cuda"), torch.zeros(B, 1, D, 1, device="cuda")
    at = torch.tensor([0, 1, (1 << 20) - 2, (1 << 20) - 1, 1 << 20, B - 1], device="cuda")
    for t in (u, delta, bc):
        t[at] = torch.randn(t[at].shape, device="cuda")
    A = -torch.rand(D, 1, device="cuda")
    y, h = memory.selective_scan(u, delta, A, bc, bc, return_state=True)
    few = [t[at] for t in (u, delta, bc)]
    # (few rows take another form of the kernel where a channel has more than 4 states: not here)
    ys, hs = memory.selective_scan(few[0], few[1], A, few[2], few[2], return_state=True)
    assert torch.equal(y[at], ys) and torch.equal(h[at], hs)
    assert int(torch.count_nonzero(y.any(2))) == len(at)


def test_scan_gradients_of_more_sums_than_one_launch_takes():
    """dB and dC of a group wider than a workgroup are summed over its workgroups by a launch of their own: 2^32 numbers."""
    torch = torch_()
    from gym_auv_amd import memory

    torch.manual_seed(10)
    B, L, D, N, bf = (1 << 18) + 5, 128, 32, 64, torch.bfloat16
    at = torch.tensor([0, (1 << 18) - 1, 1 << 18, B - 1], device="cuda")
    rows = lambda *tail: torch.zeros(B, L, *tail, device="cuda", dtype=bf)          # noqa: E731
    u, delta, Bm, Cm, gy = rows(D), rows(D), rows(1, N), rows(1, N), rows(D)
    for t in (u, delta, Bm, Cm, gy):
        t[at] = torch.randn(len(at), *t.shape[1:], device="cuda").to(bf)
    A = -torch.rand(D, N, device="cuda")
    few = [t[at].requires_grad_(True) for t in (u, delta, Bm, Cm)]
    Bm.requires_grad_(True), Cm.requires_grad_(True)
    y = memory.selective_scan(u, delta, A, Bm, Cm)
    dB, dC = torch.autograd.grad(y, [Bm, Cm], gy)
    ys = memory.selective_scan(few[0], few[1], A, few[2], few[3])
    wB, wC = torch.autograd.grad(ys, few[2:], gy[at])
    assert torch.equal(y.detach()[at], ys.detach()) or float((y.detach()[at].float() - ys.detach().float()).abs().max()) <= 2 ** -7 * float(ys.detach().float().abs().max())
    for got, want in ((dB, wB), (dC, wC)):
        # a few rows are split over time: other orders of the same sums, then one rounding to bfloat16, half a step (2^-8) each
        assert float((got[at].float() - want.float()).abs().max()) <= 2 ** -7 * float(want.float().abs().max())
        assert not got[1:1000].any() and int(torch.count_nonzero(got[-100:].flatten(1).any(1))) == 3


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_memory_of_padded_rows(dtype):
    """What lies behind a row's last token, NaN and infinities included, has no part in outputs, states and gradients; the
    outputs there are 0."""
    torch = torch_()
    from gym_auv_amd import memory

    torch.manual_seed(6)
    B, L, F = 4, 21, 18
    net = memory.EpisodeMemory(F, 16, layers=2, dtype=getattr(torch, dtype)).cuda()
    x = torch.randn(B, L, F, device="cuda")
    n = torch.tensor([L, 0, 7, 16], dtype=torch.int32, device="cuda")
    weight = torch.randn(B, L, 16, device="cuda")
    params = list(net.parameters())

    def run(fill):
        v = x.clone()
        for b, k in enumerate(n.tolist()):
            v[b, k:] = fill
        v.requires_grad_(True)
        h, state = net(v, lengths=n)
        return h.detach(), [t.detach() for s in state for t in s], torch.autograd.grad((h.float() * weight).sum(), [v] + params)

    h0, s0, g0 = run(0.0)
    assert all(bool(torch.isfinite(g).all()) for g in g0)
    for b, k in enumerate(n.tolist()):
        assert not h0[b, k:].any() and not g0[0][b, k:].any()
        if k:        # and the row is the row by itself
            alone, s = net(x[b:b + 1, :k])
            tol = (2e-5 if dtype == "float32" else 0.08) * float(alone.float().abs().max())
            assert float((alone - h0[b:b + 1, :k]).float().abs().max()) <= tol
    for fill in (float("nan"), float("inf")):
        h1, s1, g1 = run(fill)
        assert torch.equal(h0, h1)
        for a, c in zip(s0 + list(g0), s1 + list(g1)):
            assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("under", ["bfloat16", "float16"])
def test_memory_under_autocast_keeps_its_own_types(dtype, under):
    torch = torch_()
    from gym_auv_amd import memory

    torch.manual_seed(7)
    net = memory.EpisodeMemory(18, 16, layers=2, dtype=getattr(torch, dtype)).cuda()
    x = torch.randn(3, 9, 18, device="cuda")
    want, _ = net(x)
    got_state, want_state = net.new_state(3), net.new_state(3)
    wants = net.step(x[:, 0], want_state)
    with torch.autocast("cuda", dtype=getattr(torch, under)):
        got, _ = net(x)
        gots = net.step(x[:, 0], got_state)
        low, _ = net(x.to(getattr(torch, under)))          # what an autocast layer in front hands over
        assert torch.is_autocast_enabled()
    assert got.dtype == want.dtype and torch.equal(got, want) and torch.equal(gots, wants)
    assert low.dtype == want.dtype and bool(torch.isfinite(low).all())
    g0, g1 = torch.autograd.grad(want.sum(), net.enter.weight), torch.autograd.grad(got.sum(), net.enter.weight)
    assert torch.equal(g0[0], g1[0])


# ----------------------------------------------------------------------------
# the extractor's tokens
# ----------------------------------------------------------------------------
def test_the_extractor_hands_out_what_its_memory_is_trained_on():
    """Two rollouts of one batch, the second in the middle of episodes: the memory over the kept tokens, from the state
    kept before, gives the features that the policy saw, and gradients."""
    import os

    torch = torch_()
    from gym_auv_amd import cnn, memory, scenarios
    from gym_auv_amd.env import VecAuvEnv
    from oracle import cnn_oracle

    gold = np.load(os.path.join(os.path.dirname(__file__), "golden", "cnn_golden.npz"))
    cfg, scene = scenarios.make_workload("cfg3_65536_moving", n_envs=64)
    cfg["max_steps"] = 9
    env = VecAuvEnv(cfg, scene, auto_reset="device")
    torch.manual_seed(11)
    net = memory.EpisodeMemory(18, 16, layers=2).cuda()
    weights = cnn_oracle.golden_weights(gold, "shallow")
    ext, whole = (cnn.PerceptionNavigationExtractor("shallow", weights, memory=net) for _ in range(2))
    assert ext.state is None
    obs, acts = env.reset(), torch.from_numpy(scenarios.random_actions(64, 20, seed=2)).cuda()
    for first, steps in ((0, 6), (6, 14)):
        tokens, starts = torch.zeros(steps, 64, 18, device="cuda"), torch.zeros(steps, 64, dtype=torch.bool, device="cuda")
        before = None if ext.state is None else [tuple(t.clone() for t in s) for s in ext.state]
        seen = []
        for k in range(steps):
            starts[k] = env.sim.tensor("t_step") == 0
            tokens[k] = ext.tokens(obs)
            seen.append(ext.remember(tokens[k], starts[k]))
            assert torch.equal(seen[-1], whole(obs, starts[k]))
            obs, _, _, _ = env.step(acts[first + k].t())
        h, _ = net(tokens.transpose(0, 1), start=starts.transpose(0, 1), state=before)
        seen = torch.stack(seen, 1)
        assert float((h - seen).abs().max()) <= 2e-5 * float(seen.abs().max())
        grads = torch.autograd.grad(h.square().sum(), list(net.parameters()))
        assert all(bool(torch.isfinite(g).all()) and bool(g.any()) for g in grads)
    assert starts.any() and not starts[0].all()
    plain = cnn.PerceptionNavigationExtractor("shallow", weights)
    assert torch.equal(plain(obs), ext.tokens(obs))
    with pytest.raises(ValueError, match="no memory"):
        plain.remember(tokens[0])
    with pytest.raises(ValueError, match="none"):
        plain(obs, starts[0])
    env.close()


# ----------------------------------------------------------------------------
# many rows a workgroup: sums carried from one to the next
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,residual", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("B,L,D", [(531, 131, 18), (251, 37, 250), (101, 13, 600), (67, 11, 2050)])
def test_norm_gradients_of_many_rows_a_workgroup(B, L, D, dtype, residual):
    """512 workgroups (256 above 2,048 channels) of 64, 8, 1 and 1 rows each go two to three times over; the last time not
    all of them.  A column's sum goes through its thread's rows, a workgroup's threads and 16 records in each of 32 parts."""
    torch = torch_()
    from gym_auv_amd import memory

    m, r = Maker(40, dtype, "time"), Maker(41, residual, "time")
    at_once = {18: 64 * 512, 250: 8 * 512, 600: 512, 2050: 256}[D]
    assert 2 * at_once < B * L < 4 * at_once and B * L % at_once
    named = dict(x=r.rows(B, L, D), y=m.rows(B, L, D), post_weight=m.par(D), pre_weight=m.par(D), gate=m.rows(B, L, D), scale=m.par(D))
    named = {k: v.requires_grad_(True) for k, v in named.items()}
    gx, gh = r.rows(B, L, D), m.rows(B, L, D)
    outs = memory.residual_norm(*named.values())
    grads = torch.autograd.grad(outs, list(named.values()), [gx, gh])
    flat = lambda t: host(t).reshape(-1, D) if t.dim() == 3 else host(t)     # noqa: E731
    want = O.norm(*(flat(t) for t in named.values()), dx_out=flat(gx), dh=flat(gh))
    K = 4 * (D + 24) + 4 + 64 + 16 + 32
    for (name, leaf), g in zip(named.items(), grads):
        check("d_" + name, g, tuple(v.reshape(leaf.shape) for v in want[name]), K)


@pytest.mark.parametrize("B,L,D,W,dtype", [(300, 20, 2100, 4, "float32"), (200, 23, 4100, 3, "bfloat16"), (2100, 20, 520, 4, "float16"),
                                           (2100, 20, 260, 2, "float32")])
def test_conv_gradients_of_many_runs_a_thread(B, L, D, W, dtype):
    """More runs than the records of a backward pass have threads for: a thread goes over several, from row to row."""
    torch = torch_()
    from gym_auv_amd import memory

    V = 4 if dtype == "float32" else 8
    slots = 256 // min(256, -(-D // V))
    assert B * -(-L // 8) > min(2048, 2 ** 20 // D) * slots
    m = Maker(42, dtype, "time")
    start, n = m.starts(B, L, 0.1), lengths_of("ragged", B, L, m.rng)
    x, w, b = m.rows(B, L, D), m.par(D, W), m.par(D)
    m.layout = "rows"
    s = m.rows(B, W - 1, D)
    leaves = [t.requires_grad_(True) for t in (x, w, b, s)]
    gy, gs = m.rows(B, L, D), m.rows(B, W - 1, D)
    y, new = memory.causal_conv(x, w, b, start=start, lengths=n, state=s, return_state=True)
    grads = torch.autograd.grad([y, new], leaves, [gy, gs])
    want = O.conv(host(x), host(w), host(b), hostb(start), n.cpu().numpy(), host(s), True, host(gy), host(gs))
    # a sum goes through a thread's runs of 8 tokens, a workgroup's threads and 64 records in each of 32 parts
    K = 2 * (W + 10) + W + 8 * 4 + slots + 64 + 32
    for name, g in zip(("x", "weight", "bias", "state"), grads):
        check("d_" + name, g, want[name], K)


@pytest.mark.parametrize("B,D,N,G,dtype", [(4200, 64, 16, 1, "float32"), (4200, 64, 16, 1, "bfloat16"), (4200, 40, 4, 2, "float16"), (4200, 64, 8, 1, "bfloat16"),
                                           (2100, 40, 20, 1, "float32"), (1100, 24, 64, 1, "bfloat16")])
def test_scan_gradients_of_many_rows_a_workgroup(B, D, N, G, dtype):
    """More rows than the workgroups of a backward pass take at once: sums of A, D and delta_bias carried from row to row."""
    torch = torch_()
    L = 5
    m = Maker(43, dtype, "time")
    t, start, n = scan_case(m, B, L, D, N, G, 0.2, "ragged", True, True)
    t = {k: None if v is None else v.detach() for k, v in t.items()}
    for k in ("u", "delta", "B", "C", "z"):                # (what the padding may hold is not at stake here)
        t[k] = torch.nan_to_num(t[k], nan=0.0, posinf=0.0)
    gy, gs = m.rows(B, L, D), m.par(B, D, N)
    got, want = run_scan(t, start, n, gy, gs, True), raw_scan(t, start, n, gy, gs, True)
    K = 10 * (L + N + 12)
    for name in got:
        # a thread's tokens of up to five rows, then 64 records in each of 32 parts; dB and dC: a group's channels
        more = 25 + 64 + 32 if name in ("A", "D", "delta_bias") else D // G if name in ("B", "C") else 0
        check("d_" + name, got[name], want[name], 2 * K + more)
