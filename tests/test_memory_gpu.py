"""The sequence operators on the GPU against the 64-bit oracle (oracle/seq_oracle.py), within the
rounding bounds it derives; and how they are called: strides, streams, graphs, refusals."""
import numpy as np
import pytest

from gym_auv_amd import _lib
from oracle import seq_oracle as O

pytestmark = pytest.mark.gpu

TYPES = ("float32", "bfloat16", "float16")


def torch_():
    import torch

    return torch


def check(name, got, want, K):
    """got within K u magnitude + half a step of its type, everywhere."""
    import torch

    value, magnitude = want
    half = torch.finfo(got.dtype).eps / 2
    tiny = float(torch.finfo(got.dtype).smallest_normal) if got.dtype == torch.float16 else 1e-30
    err = np.abs(got.detach().double().cpu().numpy() - value)
    tol = K * O.U32 * magnitude + half * np.abs(value) + half * tiny + 1e-30
    bad = ~(err <= tol)
    assert not bad.any(), (name, "values outside:", int(bad.sum()), "of", bad.size, "worst", float((err / tol)[bad].max()),
                           "at", tuple(int(i) for i in np.argwhere(bad)[0]))


class Maker:
    """Tensors of one case: values rounded to the type first, so that oracle and kernel see the same."""

    def __init__(self, seed, dtype, layout="rows"):
        self.rng, self.layout = np.random.default_rng(seed), layout
        self.dtype = getattr(torch_(), dtype)

    def rows(self, B, L, *tail, scale=1.0):
        """[B, L, *tail] on the GPU: as stored ("rows"), time-major ("time"), or a slice of a wider tensor whose
        channels start at an odd place ("slice")."""
        torch = torch_()
        v = torch.from_numpy(scale * self.rng.normal(size=(B, L) + tail)).to(self.dtype)
        if self.layout == "time":
            return v.transpose(0, 1).contiguous().cuda().transpose(0, 1)
        if self.layout == "slice":
            wide = torch.zeros((B, L) + tail[:-1] + (tail[-1] + 5,), dtype=self.dtype)
            wide[..., 3:3 + tail[-1]] = v
            return wide.cuda()[..., 3:3 + tail[-1]]
        return v.cuda()

    def par(self, *shape, scale=1.0, of=None):
        v = scale * self.rng.normal(size=shape) if of is None else of
        return torch_().from_numpy(v.astype(np.float32)).cuda()

    def starts(self, B, L, share):
        torch = torch_()
        if share is None:
            return None
        m = torch.from_numpy(self.rng.random((L, B)) < share).cuda()
        return m.transpose(0, 1)     # as the flags of a rollout are stored


def host(t):
    return None if t is None else t.detach().double().cpu().numpy()


def hostb(t):
    return None if t is None else t.cpu().numpy().astype(bool)


def lengths_of(kind, B, L, rng):
    torch = torch_()
    if kind is None:
        return None
    n = rng.integers(0, L + 1, B)
    n[0], n[-1] = L, 0                      # a full row and an empty one
    if B > 2:
        n[1] = L + 7                        # clamped
    if B > 3:
        n[2] = -1
    return torch.from_numpy(n.astype(np.int32)).cuda()


def spoil(t, lengths):
    """NaN and infinities behind every row's last token: nothing of them may be seen."""
    if lengths is None:
        return t
    for b, n in enumerate(lengths.clamp(0, t.shape[1]).tolist()):
        t[b, n:] = float("nan")
        t[b, n:n + 1] = float("inf")
    return t


# ----------------------------------------------------------------------------
# convolution
# ----------------------------------------------------------------------------
CONV = [  # B, L, D, W, start share, lengths, state, bias, silu, layout
    (1, 1, 1, 2, None, None, False, False, False, "rows"),
    (3, 1, 8, 4, 0.5, None, True, True, True, "rows"),
    (2, 2, 3, 4, 0.5, None, True, True, True, "time"),
    (4, 3, 18, 4, 0.3, "ragged", True, True, True, "time"),
    (5, 33, 90, 3, 0.1, "ragged", True, False, True, "rows"),
    (5, 70, 64, 4, 0.05, None, False, True, True, "time"),
    (4, 65, 130, 2, 1.0, "ragged", True, True, False, "rows"),
    (3, 40, 20, 4, 0.0, None, True, True, True, "slice"),
    (2, 9, 2100, 4, 0.2, "ragged", True, True, True, "rows"),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CONV, ids=lambda c: "x".join(map(str, c[:4])))
def test_conv_and_gradients_against_the_oracle(case, dtype):
    torch = torch_()
    from gym_auv_amd import memory

    B, L, D, W, share, ragged, with_state, with_bias, silu, layout = case
    m = Maker(1, dtype, layout)
    start, n = m.starts(B, L, share), lengths_of(ragged, B, L, m.rng)
    x = spoil(m.rows(B, L, D), n).requires_grad_(True)
    w = m.par(D, W, scale=0.7).requires_grad_(True)
    b = m.par(D).requires_grad_(True) if with_bias else None
    m.layout = "rows"
    s = m.rows(B, W - 1, D).requires_grad_(True) if with_state else None
    gy, gs = m.rows(B, L, D), m.rows(B, W - 1, D)
    y, new = memory.causal_conv(x, w, b, start=start, lengths=n, state=s, silu=silu, return_state=True)
    assert y.dtype == x.dtype and y.shape == x.shape and new.shape == (B, W - 1, D)
    leaves = [t for t in (x, w, b, s) if t is not None]
    grads = torch.autograd.grad([y, new], leaves, [gy, gs])
    xv = np.nan_to_num(host(x), nan=0.0, posinf=0.0)
    want = O.conv(xv, host(w), host(b), hostb(start), host(n), host(s), silu, host(gy), host(gs)) if n is None else \
        O.conv(xv, host(w), host(b), hostb(start), n.cpu().numpy(), host(s), silu, host(gy), host(gs))
    K = W + 2 + 8
    check("y", y, want["y"], K)
    check("new_state", new, want["new_state"], 0)
    names = [k for k, t in (("x", x), ("weight", w), ("bias", b), ("state", s)) if t is not None]
    for name, g in zip(names, grads):
        check("d_" + name, g, want[name], 2 * K + W + (B * L if name in ("weight", "bias") else 0))
    # without gradients, and without a state handed on: the same numbers
    with torch.no_grad():
        assert torch.equal(memory.causal_conv(x, w, b, start=start, lengths=n, state=s, silu=silu), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D,W", [(1, 1, 2), (3, 18, 4), (130, 64, 4), (7, 90, 3)])
def test_conv_token_by_token_equals_the_row_at_once(B, D, W, dtype):
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(2, dtype)
    L = 9
    x, w, b, s, start = m.rows(B, L, D), m.par(D, W), m.par(D), m.rows(B, W - 1, D), m.starts(B, L, 0.3)
    y, new = memory.causal_conv(x, w, b, start=start, state=s, return_state=True)
    state, other = s.clone(), torch.full_like(s, float("nan"))
    for t in range(L):
        if t % 2:
            yt = memory.causal_conv_step(x[:, t], state, w, b, start=start[:, t])
        else:                                       # into another buffer, the old state left as it was
            before = state.clone()
            yt = memory.causal_conv_step(x[:, t], state, w, b, start=start[:, t], new_state=other)
            assert torch.equal(state, before)
            state.copy_(other)
        assert torch.equal(yt, y[:, t]), t          # the same operations in the same order: the same bits
    assert torch.equal(state, new)


# ----------------------------------------------------------------------------
# scan
# ----------------------------------------------------------------------------
SCAN = [  # B, L, D, N, G, start share, lengths, state, optional (D, z, bias), layout
    (1, 1, 1, 1, 1, None, None, False, False, "rows"),
    (3, 1, 18, 4, 1, 0.5, None, True, True, "rows"),
    (2, 2, 16, 16, 1, 0.5, None, True, True, "time"),
    (4, 15, 18, 16, 1, 0.1, "ragged", True, True, "time"),
    (5, 17, 90, 7, 2, 0.1, "ragged", True, True, "time"),
    (3, 33, 64, 16, 1, 0.05, None, True, True, "slice"),
    (3, 40, 30, 8, 3, 1.0, None, True, True, "rows"),
    (2, 50, 40, 20, 2, 0.1, "ragged", False, True, "rows"),
    (2, 20, 24, 64, 2, 0.1, None, True, False, "rows"),
    (2, 20, 10, 33, 1, 0.1, None, True, True, "rows"),
    (1, 300, 32, 16, 1, 0.01, None, True, True, "time"),       # split into chunks
    (3, 200, 18, 5, 1, 0.02, "ragged", True, True, "rows"),    # likewise, rows that end in every chunk
    (1, 100, 600, 16, 1, 0.02, None, True, True, "rows"),      # a group wider than a workgroup
    (2, 70, 300, 40, 2, 0.02, "ragged", True, True, "rows"),
]


def scan_case(m, B, L, D, N, G, share, ragged, with_state, full):
    torch = torch_()
    start, n = m.starts(B, L, share), lengths_of(ragged, B, L, m.rng)
    t = dict(u=spoil(m.rows(B, L, D), n), delta=spoil(m.rows(B, L, D, scale=0.7), n), A=m.par(D, N, of=-np.exp(m.rng.uniform(-1, 2.5, (D, N)))),
             B=spoil(m.rows(B, L, G, N), n), C=spoil(m.rows(B, L, G, N), n), D=m.par(D) if full else None,
             z=spoil(m.rows(B, L, D), n) if full else None, delta_bias=m.par(D, of=m.rng.uniform(-4, 0, D)) if full else None,
             state=m.par(B, D, N) if with_state else None)
    return {k: None if v is None else v.requires_grad_(True) for k, v in t.items()}, start, n


def scan_oracle(t, start, n, gy=None, gs=None, softplus=True):
    clean = {k: None if v is None else np.nan_to_num(host(v), nan=0.0, posinf=0.0) for k, v in t.items()}
    return O.scan(clean["u"], clean["delta"], clean["A"], clean["B"], clean["C"], clean["D"], clean["z"], clean["delta_bias"],
                  softplus, hostb(start), None if n is None else n.cpu().numpy(), clean["state"], host(gy), host(gs))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", SCAN, ids=lambda c: "x".join(map(str, c[:5])))
def test_scan_and_gradients_against_the_oracle(case, dtype):
    torch = torch_()
    from gym_auv_amd import memory

    B, L, D, N, G, share, ragged, with_state, full, layout = case
    m = Maker(3, dtype, layout)
    t, start, n = scan_case(m, B, L, D, N, G, share, ragged, with_state, full)
    m.layout = "time"
    gy, gs = m.rows(B, L, D), m.par(B, D, N)
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")]
    y, new = memory.selective_scan(*args, start=start, lengths=n, state=t["state"], return_state=True)
    assert y.dtype == t["u"].dtype and new.dtype == torch.float32 and new.shape == (B, D, N)
    names = [k for k, v in t.items() if v is not None]
    grads = torch.autograd.grad([y, new], [t[k] for k in names], [gy, gs])
    want = scan_oracle(t, start, n, gy, gs)
    K = 10 * (L + N + 12)
    check("y", y, want["y"], K)
    check("new_state", new, want["new_state"], K)
    for name, g in zip(names, grads):
        more = B * L if name in ("A", "D", "delta_bias") else D // G if name in ("B", "C") else 0
        check("d_" + name, g, want[name], 2 * K + more)
    with torch.no_grad():
        again, _ = memory.selective_scan(*args, start=start, lengths=n, state=t["state"], return_state=True)
    assert torch.equal(again, y)


@pytest.mark.parametrize("N,D", [(16, 64), (8, 64), (32, 40), (3, 70), (50, 20)])
def test_scan_of_many_rows_against_the_oracle(N, D):
    """Enough rows for a whole channel per lane (the small cases above split it over lanes)."""
    torch = torch_()
    from gym_auv_amd import memory

    B, L = 4200, 5
    m = Maker(4, "float32", "time")
    t, start, n = scan_case(m, B, L, D, N, 1, 0.2, "ragged", True, True)
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")]
    gy = m.rows(B, L, D)
    y, new = memory.selective_scan(*args, start=start, lengths=n, state=t["state"], return_state=True)
    grads = torch.autograd.grad(y, [t["u"], t["delta"], t["B"], t["C"], t["z"]], gy)
    rows = np.r_[0:40, B - 40:B]
    idx = torch.from_numpy(rows).cuda()
    sub = {k: v if k in ("A", "D", "delta_bias") else v.detach()[idx] for k, v in t.items()}
    want = scan_oracle(sub, start[idx], n[idx], gy[idx])
    K = 10 * (L + N + 12)
    check("y", y[idx], want["y"], K)
    check("new_state", new[idx], want["new_state"], K)
    for name, g in zip(("u", "delta", "B", "C", "z"), grads):
        check("d_" + name, g[idx], want[name], 2 * K + D)


@pytest.mark.parametrize("softplus", [True, False])
def test_scan_of_extreme_steps(softplus):
    """Widths of nothing and of very much, as softplus makes them of -100 and 80 (or as given): decays of 1 and 0."""
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(5, "float32")
    B, L, D, N = 2, 24, 16, 16
    t, start, n = scan_case(m, B, L, D, N, 1, None, None, True, False)
    v = m.rng.choice([-100.0, -20.0, 0.0, 20.0, 80.0] if softplus else [0.0, 1e-6, 1.0, 80.0], (B, L, D))
    t["delta"] = torch.from_numpy(v.astype(np.float32)).cuda().requires_grad_(True)
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")]
    gy = m.rows(B, L, D)
    y, new = memory.selective_scan(*args, delta_softplus=softplus, state=t["state"], return_state=True)
    grads = torch.autograd.grad(y, [t["u"], t["delta"], t["A"]], gy)
    want = scan_oracle(t, start, n, gy, None, softplus)
    K = 10 * (L + N + 12) + 100 * 12          # |raw| up to 100 in place of 8
    check("y", y, want["y"], K)
    check("new_state", new, want["new_state"], K)
    for name, g in zip(("u", "delta", "A"), grads):
        check("d_" + name, g, want[name], 2 * K + B * L)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (3, 18, 4, 1), (130, 64, 16, 1), (7, 90, 7, 2), (5, 20, 32, 2), (3, 12, 64, 3), (2, 8, 50, 1)])
def test_scan_token_by_token_against_the_row_at_once(B, D, N, G, dtype):
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(6, dtype, "time")
    L = 7
    t, start, _ = scan_case(m, B, L, D, N, G, 0.3, None, True, True)
    t = {k: v.detach() for k, v in t.items()}
    want = scan_oracle(t, start, None)
    state, K = t["state"].clone(), 10 * (L + N + 12)
    other = torch.empty_like(state)
    for l in range(L):
        row = [t[k][:, l] for k in ("u", "delta")]
        rest = [t["A"], t["B"][:, l], t["C"][:, l], t["D"], t["z"][:, l], t["delta_bias"]]
        if l % 2:
            yt = memory.selective_scan_step(*row, state, *rest, start=start[:, l])
        else:
            before = state.clone()
            yt = memory.selective_scan_step(*row, state, *rest, start=start[:, l], new_state=other)
            assert torch.equal(state, before)
            state.copy_(other)
        check(f"y {l}", yt, (want["y"][0][:, l], want["y"][1][:, l]), K)
    check("state", state, want["new_state"], K)


def test_an_episode_does_not_see_what_came_before():
    """What lies before a start may be anything, infinities and NaN included: outputs after it are bit for bit those of
    the episode alone, forwards and, as long as what came before is finite, backwards."""
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(7, "float32", "time")
    B, L, D, N = 3, 40, 48, 16
    for cut in (1, 15, 16, 17, 31):
        t, _, _ = scan_case(m, B, L, D, N, 1, None, None, True, True)
        start = torch.zeros(L, B, dtype=torch.uint8, device="cuda").t()
        start[:, cut] = 1
        names = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")
        whole = [t[k].detach().clone() for k in names]
        for i in (0, 6):
            whole[i][:, :cut] = float("nan")
        y = memory.selective_scan(*whole, start=start, state=torch.full_like(t["state"], float("inf")))
        alone = [v if v.dim() < 3 else v[:, cut:] for v in whole]
        check("scan", y[:, cut:], (host(memory.selective_scan(*alone)), np.abs(host(y[:, cut:])) + 1.0), 10 * (L + N + 12))
        w, b, x = m.par(D, 4), m.par(D), m.rows(B, L, D)
        x[:, :cut] = float("nan")
        yc = memory.causal_conv(x, w, b, start=start, state=torch.full((B, 3, D), float("inf"), device="cuda"))
        assert torch.equal(yc[:, cut:], memory.causal_conv(x[:, cut:], w, b))


@pytest.mark.parametrize("B,L,cut", [(2, 900, 700), (2, 900, 16), (3, 700, 333), (1, 1500, 1300)])
def test_what_a_start_parts_in_a_row_of_many_chunks(B, L, cut):
    """Rows cut into chunks, one episode before `cut` and one from there on: neither sees NaN or infinities in any of the
    other's tokens, widths and gradients included."""
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(17, "float32", "time")
    D, N = 20, 16
    t, _, _ = scan_case(m, B, L, D, N, 1, None, None, True, True)
    gy = m.rows(B, L, D)
    start = torch.zeros(B, L, dtype=torch.uint8, device="cuda")
    start[:, cut] = 1
    rows, names = ("u", "delta", "B", "C", "z"), ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")
    K = 10 * (L + N + 12)
    for part in (slice(cut, None), slice(0, cut)):
        first = part.start == 0
        spoilt = {k: v if v is None else v.detach().clone() for k, v in t.items()}
        hole = slice(cut, None) if first else slice(0, cut)
        g = gy.clone()
        for i, v in enumerate([*(spoilt[k] for k in rows), g]):
            v[:, hole] = float("nan") if i % 2 == 0 else float("inf")
        spoilt["delta"][:, hole] = float("nan")
        if not first:
            spoilt["state"].fill_(float("inf"))
        given = [spoilt[k].requires_grad_(True) for k in names]
        y = memory.selective_scan(*given, start=start, state=spoilt["state"])
        grads = torch.autograd.grad(y, [spoilt[k] for k in rows], g)
        alone = {k: v if v is None or k not in rows else v[:, part] for k, v in t.items()}
        if not first:
            alone["state"] = None
        want = scan_oracle(alone, None, None, gy[:, part])
        check("y", y[:, part], want["y"], K)
        for k, d in zip(rows, grads):
            check("d_" + k, d[:, part], want[k], 2 * K + D)


@pytest.mark.parametrize("B,L,D,N,ragged,share", [(2, 4200, 12, 16, None, 0.002), (1, 4128, 30, 7, None, 0.0), (3, 4100, 5, 20, "ragged", 0.001)])
def test_scan_of_a_few_long_rows_against_the_oracle(B, L, D, N, ragged, share):
    """Hundreds of chunks a row, joined forwards and backwards, from a state and to the gradient of one."""
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(19, "float32", "time")
    t, start, n = scan_case(m, B, L, D, N, 1, share, ragged, True, True)
    gy, gs = m.rows(B, L, D), m.par(B, D, N)
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")]
    y, new = memory.selective_scan(*args, start=start, lengths=n, state=t["state"], return_state=True)
    names = list(t)
    grads = torch.autograd.grad([y, new], [t[k] for k in names], [gy, gs])
    want = scan_oracle(t, start, n, gy, gs)
    # (a decay carried over C chunks takes C products where the oracle takes L: no more roundings than the bound counts)
    K = 10 * (L + N + 12)
    check("y", y, want["y"], K)
    check("new_state", new, want["new_state"], K)
    for name, g in zip(names, grads):
        more = B * L if name in ("A", "D", "delta_bias") else D if name in ("B", "C") else 0
        check("d_" + name, g, want[name], 2 * K + more)


def test_windows_that_overlap():
    """Sliding windows over a signal: channels adjacent, and the next token one element on."""
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(18, "float32")
    D, N, L = 30, 4, 11
    signal = m.par(2, L + D - 1)
    x = signal.unfold(1, D, 1)
    assert x.shape == (2, L, D) and x.stride()[1:] == (1, 1)
    w, wn, A = m.par(D, 4), m.par(D), -m.par(D, N).abs()
    bc = m.rows(2, L, 1, N)
    gy = m.rows(2, L, D)

    def run(x):
        x = x.detach().requires_grad_(True)
        outs = [memory.causal_conv(x, w), memory.selective_scan(x, x, A, bc, bc, z=x)]
        return outs + [torch.autograd.grad(o, x, gy)[0] for o in outs]

    for a, b in zip(run(x), run(x.contiguous())):
        assert torch.equal(a, b)
    x, y = x.detach().requires_grad_(True), x.detach().requires_grad_(True)      # (two leaves over the same memory)
    outs = memory.residual_norm(x, y, wn, wn)
    grads = torch.autograd.grad(outs, [x, y], [gy, gy])
    flat = lambda t: host(t).reshape(-1, D)                                       # noqa: E731
    want = O.norm(flat(x), flat(y), host(wn), host(wn), dx_out=flat(gy), dh=flat(gy))
    for name, t in (("x_out", outs[0]), ("h", outs[1]), ("x", grads[0]), ("y", grads[1])):
        check(name, t, tuple(v.reshape(t.shape) for v in want[name]), 4 * (D + 24) + 2 * L)


# ----------------------------------------------------------------------------
# norms
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("D", [1, 6, 18, 64, 128, 129, 250, 512, 600, 2048, 2050, 8192])
@pytest.mark.parametrize("dtype,residual", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float16"), ("bfloat16", "bfloat16")])
def test_residual_norm_and_gradients_against_the_oracle(D, dtype, residual):
    torch = torch_()
    from gym_auv_amd import memory

    B, L = (3, 7) if D < 1000 else (2, 3)
    m, r = Maker(8, dtype, "time"), Maker(9, residual, "rows" if D % 2 else "time")
    x, y, gate = r.rows(B, L, D, scale=2.0), m.rows(B, L, D), m.rows(B, L, D)
    y[0, 0] = 0.0                                  # a row of zeros: its norm rests on eps
    w1, w2, sc = (m.par(D) for _ in range(3))
    gx, gh = r.rows(B, L, D), m.rows(B, L, D)
    flat = lambda t: None if t is None else host(t).reshape(-1, D)   # noqa: E731
    K = D + 24
    for act, use_gate, use_post, use_scale, use_pre in (("silu", True, True, True, True), ("sigmoid", True, False, True, True),
                                                        (None, True, True, False, True), ("silu", False, True, True, False)):
        named = dict(x=x, y=y, post_weight=w1 if use_post else None, pre_weight=w2 if use_pre else None, gate=gate if use_gate else None,
                     scale=sc if use_scale else None)
        named = {k: None if v is None else v.detach().requires_grad_(True) for k, v in named.items()}
        out, h = memory.residual_norm(*named.values(), gate_act=act)
        assert out.dtype == x.dtype and (h is None) == (not use_pre)
        leaves = {k: v for k, v in named.items() if v is not None}
        outs, gs = ([out, h], [gx, gh]) if use_pre else ([out], [gx])
        grads = torch.autograd.grad(outs, list(leaves.values()), gs)
        want = O.norm(flat(x), flat(y), *(flat(t) if t is not None and t.dim() == 3 else host(t) for t in list(named.values())[2:]),
                      gate_act=act, dx_out=flat(gx), dh=flat(gh) if use_pre else None)
        shaped = lambda p, t: tuple(v.reshape(t.shape) for v in p)   # noqa: E731
        check("x'", out, shaped(want["x_out"], out), K)
        if use_pre:
            check("h", h, shaped(want["h"], h), K)
        for (name, leaf), g in zip(leaves.items(), grads):
            check(f"{act} d_{name}", g, shaped(want[name], g), 4 * K + B * L)


@pytest.mark.parametrize("shape", [(5,), (4, 18), (2, 3, 64), (2, 3, 4, 10)])
def test_rms_norm_of_any_rows(shape):
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(10, "float32")
    x = torch.from_numpy(m.rng.normal(size=shape).astype(np.float32)).cuda().requires_grad_(True)
    w, g = m.par(shape[-1]).requires_grad_(True), torch.from_numpy(m.rng.normal(size=shape).astype(np.float32)).cuda()
    y = memory.rms_norm(x, w)
    D = shape[-1]
    want = O.norm(host(x).reshape(-1, D), pre_weight=host(w), dh=host(g).reshape(-1, D))
    check("y", y, tuple(v.reshape(shape) for v in want["h"]), D + 24)
    dx, dw = torch.autograd.grad(y, [x, w], g)
    check("dx", dx, tuple(v.reshape(shape) for v in want["x"]), 4 * (D + 24))
    check("dw", dw, want["pre_weight"], 4 * (D + 24) + 30)
    assert memory.rms_norm(x, w, dtype=torch.bfloat16).dtype == torch.bfloat16


def test_norm_of_an_expanded_gate():
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(11, "float32")
    B, L, D = 3, 6, 32
    x, y, w, g = m.rows(B, L, D), m.rows(B, L, D), m.par(D), m.rows(B, 1, D)
    g.requires_grad_(True)
    out, _ = memory.residual_norm(x, y, w, None, g.expand(B, L, D))
    (dg,) = torch.autograd.grad(out, g, torch.ones_like(out))
    wide = g.detach().expand(B, L, D).contiguous().requires_grad_(True)
    out2, _ = memory.residual_norm(x, y, w, None, wide)
    (dw,) = torch.autograd.grad(out2, wide, torch.ones_like(out))
    assert torch.equal(out, out2) and torch.allclose(dg, dw.sum(1, keepdim=True), rtol=1e-6, atol=1e-6)


# ----------------------------------------------------------------------------
# how they are called
# ----------------------------------------------------------------------------
def test_empty_batches_and_rows():
    torch = torch_()
    from gym_auv_amd import memory

    for B, L in ((0, 5), (3, 0)):
        x = torch.zeros(B, L, 8, device="cuda", requires_grad=True)
        w, s = torch.ones(8, 4, device="cuda", requires_grad=True), torch.ones(B, 3, 8, device="cuda", requires_grad=True)
        y, new = memory.causal_conv(x, w, state=s, return_state=True)
        assert y.shape == (B, L, 8) and torch.equal(new, s)
        gx, gw, gs = torch.autograd.grad([y, new], [x, w, s], [y, 2 * new])
        assert gx.shape == x.shape and float(gw.abs().sum()) == 0 and torch.equal(gs, 2 * new)
        bc = torch.zeros(B, L, 1, 16, device="cuda")
        A, h = torch.ones(8, 16, device="cuda", requires_grad=True), torch.ones(B, 8, 16, device="cuda", requires_grad=True)
        y, new = memory.selective_scan(x, x, A, bc, bc, state=h, return_state=True)
        assert y.shape == x.shape and torch.equal(new, h)
        gA, gh = torch.autograd.grad([y, new], [A, h], [y, 3 * new])
        assert float(gA.abs().sum()) == 0 and torch.equal(gh, 3 * new)
        out, hh = memory.residual_norm(x, x, w[:, 0].contiguous(), w[:, 1].contiguous())
        assert out.shape == hh.shape == x.shape
    e = torch.zeros(0, 8, device="cuda")
    assert memory.causal_conv_step(e, torch.zeros(0, 3, 8, device="cuda"), torch.ones(8, 4, device="cuda")).shape == (0, 8)


def test_refusals():
    torch = torch_()
    from gym_auv_amd import memory

    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)   # noqa: E731
    x, w, A, bc = z(2, 3, 8), z(8, 4), z(8, 16), z(2, 3, 1, 16)
    for call, err in [
        (lambda: memory.causal_conv(x[0], w), ValueError),
        (lambda: memory.causal_conv(x.double(), w), TypeError),
        (lambda: memory.causal_conv(x, w.bfloat16()), TypeError),
        (lambda: memory.causal_conv(x, z(8, 5)), ValueError),
        (lambda: memory.causal_conv(x, z(7, 4)), ValueError),
        (lambda: memory.causal_conv(x.transpose(1, 2), z(3, 4)), ValueError),
        (lambda: memory.causal_conv(x, w, start=z(2, 3)), TypeError),
        (lambda: memory.causal_conv(x, w, start=z(3, 2, dtype=torch.bool)), ValueError),
        (lambda: memory.causal_conv(x, w, lengths=z(2, dtype=torch.int64)), TypeError),
        (lambda: memory.causal_conv(x, w, state=z(2, 4, 8)), ValueError),
        (lambda: memory.causal_conv(x, w.t().contiguous().t()), ValueError),
        (lambda: memory.causal_conv(x, w, z(8).cpu()), ValueError),
        (lambda: memory.causal_conv_step(x[:, 0], z(2, 3, 8), w, new_state=z(2, 3, 8).bfloat16()), TypeError),
        (lambda: memory.causal_conv_step(x[:, 0], None, w), TypeError),
        (lambda: memory.selective_scan(x, x[:, :2], A, bc, bc), ValueError),
        (lambda: memory.selective_scan(x, x.half(), A, bc, bc), TypeError),
        (lambda: memory.selective_scan(x, x, z(8, 65), z(2, 3, 1, 65), z(2, 3, 1, 65)), ValueError),
        (lambda: memory.selective_scan(x, x, A, z(2, 3, 3, 16), z(2, 3, 3, 16)), ValueError),
        (lambda: memory.selective_scan(x, x, A, bc, z(2, 3, 2, 16)), ValueError),
        (lambda: memory.selective_scan(x, x, A, bc, bc, state=z(2, 8, 15)), ValueError),
        (lambda: memory.selective_scan_step(x[:, 0], x[:, 0], z(2, 8, 16)[:, :, ::2], z(8, 8), bc[:, 0, :, :8], bc[:, 0, :, :8]), ValueError),
        (lambda: memory.residual_norm(x, x[:, :2]), ValueError),
        (lambda: memory.residual_norm(x.half(), x), TypeError),
        (lambda: memory.residual_norm(x, x, gate=x[:, :1]), ValueError),
        (lambda: memory.residual_norm(x, x, gate=x, gate_act="tanh"), ValueError),
        (lambda: memory.residual_norm(x, x, z(8), eps=0.0), ValueError),
        (lambda: memory.rms_norm(z(2, 8193), z(8193)), ValueError),
        (lambda: memory.rms_norm(x.half(), z(8), dtype=torch.float32), TypeError),
    ]:
        with pytest.raises(err):
            call()
    state = z(2, 3, 8)
    with pytest.raises(ValueError, match="overlaps"):
        memory.causal_conv_step(x[:1, 0], state[:1], w, new_state=state.view(-1)[8:32].view(1, 3, 8))
    h = z(4, 8, 16)
    with pytest.raises(ValueError, match="overlaps"):
        memory.selective_scan_step(x[:, 0], x[:, 0], h[:2], A, bc[:, 0], bc[:, 0], new_state=h[1:3])
    with pytest.raises(RuntimeError, match="no gradients"):
        memory.causal_conv_step(x[:, 0].requires_grad_(True), state, w)
    with pytest.raises(RuntimeError, match="no gradients"):
        memory.selective_scan_step(x[:, 0], x[:, 0], h[:2], A.requires_grad_(True), bc[:, 0], bc[:, 0])


def test_a_step_does_not_read_what_it_writes():
    torch = torch_()
    from gym_auv_amd import memory

    h, A = torch.zeros(2, 8, 16, device="cuda"), torch.zeros(8, 16, device="cuda")
    x, bc = torch.zeros(2, 8, device="cuda"), torch.zeros(2, 1, 16, device="cuda")
    with pytest.raises(ValueError, match="holds an input"):
        memory.selective_scan_step(x, x, h, A, h[:, :1], bc)
    with pytest.raises(ValueError, match="holds an input"):
        memory.selective_scan_step(h[:, 0, :8], x, h, A, bc, bc)
    s = torch.zeros(2, 3, 8, device="cuda")
    with pytest.raises(ValueError, match="holds an input"):
        memory.causal_conv_step(s[:, 1], s, torch.zeros(8, 4, device="cuda"))


def test_a_step_does_not_read_what_it_writes_from_an_earlier_start():
    """Inputs that begin before the state's memory and reach into it, and ones that end where it begins."""
    torch = torch_()
    from gym_auv_amd import memory

    buf = torch.zeros(2048, device="cuda")
    h, A, bc = buf[256:512].view(2, 8, 16), torch.zeros(8, 16, device="cuda"), torch.zeros(2, 1, 16, device="cuda")
    x = torch.zeros(2, 8, device="cuda")
    for bad in (buf[200:].as_strided((2, 8), (56, 1)), buf[255:263].expand(2, 8), buf[252:268].view(2, 8)):
        with pytest.raises(ValueError, match="holds an input"):
            memory.selective_scan_step(bad, x, h, A, bc, bc)
        with pytest.raises(ValueError, match="holds an input"):
            memory.causal_conv_step(bad, buf[256:304].view(2, 3, 8), torch.zeros(8, 4, device="cuda"))
    with pytest.raises(ValueError, match="holds an input"):
        memory.selective_scan_step(x, x, h, buf[200:328].view(8, 16), bc, bc)
    with pytest.raises(ValueError, match="holds an input"):
        memory.selective_scan_step(x, x, h, A, bc, buf[226:258].view(2, 1, 16))
    with pytest.raises(ValueError, match="holds an input"):
        memory.causal_conv_step(x, buf[256:304].view(2, 3, 8), buf[225:257].view(8, 4))
    ahead = buf[240:256].view(2, 8)
    memory.selective_scan_step(ahead, ahead, h, A, bc, bc)
    memory.causal_conv_step(ahead, buf[256:304].view(2, 3, 8), torch.zeros(8, 4, device="cuda"))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows, computed within the whole and by themselves.  (Rows of the same shape go
    through the same kernels with the same bits.)"""
    torch = torch_()
    from gym_auv_amd import memory

    D, L = 520, 64
    B = 2 ** 31 // (D * L) + 3
    dev, bf = "cuda", torch.bfloat16
    torch.manual_seed(0)
    x = torch.zeros(B, L, D, device=dev, dtype=bf)
    x[-2:] = torch.randn(2, L, D, device=dev).to(bf)
    w, b = torch.randn(D, 4, device=dev), torch.randn(D, device=dev)
    y = memory.causal_conv(x, w, b)
    assert torch.equal(y[-2:], memory.causal_conv(x[-2:], w, b))
    (dx,) = torch.autograd.grad(memory.causal_conv(x.requires_grad_(True), w, b), x, y)
    part = x.detach()[-2:].clone().requires_grad_(True)
    (dp,) = torch.autograd.grad(memory.causal_conv(part, w, b), part, y[-2:])
    assert torch.equal(dx[-2:], dp)
    del dx, y
    x = x.detach()
    N = 4
    A, Bm, Cm = -torch.rand(D, N, device=dev), torch.randn(B, L, 1, N, device=dev).to(bf), torch.randn(B, L, 1, N, device=dev).to(bf)
    u = x.requires_grad_(True)
    y, h = memory.selective_scan(u, x.detach(), A, Bm, Cm, return_state=True)
    (du,) = torch.autograd.grad(y, u, y.detach())
    part = x.detach()[-2:].clone().requires_grad_(True)
    yp, hp = memory.selective_scan(part, part.detach(), A, Bm[-2:], Cm[-2:], return_state=True)
    (dp,) = torch.autograd.grad(yp, part, yp.detach())
    same = lambda a, c, k: float((a.float() - c.float()).abs().max()) <= k * float(c.float().abs().max())   # noqa: E731
    # a few rows alone are split over lanes and time: other orders of the same sums, then one rounding to bfloat16
    assert same(h[-2:], hp, 1e-5) and same(y[-2:].detach(), yp.detach(), 2 ** -8) and same(du[-2:], dp, 2 ** -7)
    del u, y, h, du
    rows = 2 ** 31 // D + 5
    flat = torch.zeros(rows, D, device=dev, dtype=bf)
    flat[-3:] = torch.randn(3, D, device=dev).to(bf)
    one = torch.ones(D, device=dev)
    o, hn = memory.residual_norm(flat, flat, one, one)
    po, ph = memory.residual_norm(flat[-3:], flat[-3:], one, one)
    assert torch.equal(o[-3:], po) and torch.equal(hn[-3:], ph)
    del flat, o, hn, x
    Bs, Ns = 2 ** 31 // (512 * 64) + 2, 64
    s = torch.zeros(Bs, 512, Ns, device=dev)
    s[-1] = torch.randn(512, Ns, device=dev)
    xs, bc = torch.randn(Bs, 512, device=dev), torch.randn(Bs, 1, Ns, device=dev)
    As = -torch.rand(512, Ns, device=dev)
    last = s[-1:].clone()
    ys = memory.selective_scan_step(xs, xs, s, As, bc, bc)
    yl = memory.selective_scan_step(xs[-1:], xs[-1:], last, As, bc[-1:], bc[-1:])
    assert torch.equal(ys[-1:], yl) and torch.equal(s[-1:], last)


def _training_pass(t, names, start):
    torch = torch_()
    from gym_auv_amd import memory

    x = memory.causal_conv(t["u"], t["w"], t["D"], start=start)
    y = memory.selective_scan(x, t["delta"], t["A"], t["B"], t["C"], t["D"], t["z"], t["delta_bias"], start=start)
    out, h = memory.residual_norm(t["x"], y, t["D"], t["delta_bias"], t["z"], t["D"])
    return [out.detach(), h.detach(), *torch.autograd.grad([out, h], [t[k] for k in names], [t["gx"], t["gh"]])]


def _training_tensors(seed=12, B=6, L=50, D=32, N=16):
    m = Maker(seed, "bfloat16", "time")
    t, start, _ = scan_case(m, B, L, D, N, 1, 0.1, None, False, True)
    names = [k for k, v in t.items() if v is not None]
    t["w"] = m.par(D, 4).requires_grad_(True)
    f = Maker(seed + 1, "float32")
    t["x"], t["gx"], t["gh"] = f.rows(B, L, D).requires_grad_(True), f.rows(B, L, D), m.rows(B, L, D)
    return t, names + ["w", "x"], start


def test_the_same_bits_on_every_call_and_on_another_stream():
    torch = torch_()
    t, names, start = _training_tensors()
    first = _training_pass(t, names, start)
    for a, b in zip(first, _training_pass(t, names, start)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _training_pass(t, names, start)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)


def test_two_calls_at_once_on_two_streams():
    torch = torch_()
    sets = [_training_tensors(seed) for seed in (12, 22)]
    want = [_training_pass(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _training_pass(*sets[i])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for a, b in zip(w, g):
            assert torch.equal(a, b)


def test_training_pass_captured_and_replayed():
    """Forward and backward recorded into two graphs that share a memory pool; replayed with new inputs and with eager
    work in between, against eager passes."""
    torch = torch_()
    t, names, start = _training_tensors()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _training_pass(t, names, start)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    pool = None
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            out = _training_pass(t, names, start)
        pool = pool or g.pool()
        graphs.append((g, out))
    for k in range(4):
        fresh, _, _ = _training_tensors(seed=40 + k)
        with torch.no_grad():
            for name in t:
                if t[name] is not None:
                    t[name].copy_(fresh[name])
        want = [v.clone() for v in _training_pass(fresh, names, start)]
        torch.cuda.synchronize()
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(want, out):
                assert torch.equal(a, b), k


def test_capturing_gradients_beside_a_live_eager_graph_is_refused():
    torch = torch_()
    from gym_auv_amd import memory

    x, w = torch.zeros(2, 3, 8, device="cuda"), torch.ones(8, 4, device="cuda", requires_grad=True)
    alive = memory.causal_conv(x, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="drop those first"):
        with torch.cuda.graph(g):
            memory.causal_conv(x, w)
    torch.cuda.synchronize()
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):                 # nothing eager is left: recorded
        y = memory.causal_conv(x, w)
        (gw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    g.replay()
    torch.cuda.synchronize()
    assert float(gw.abs().sum()) == 0.0


def test_capturing_beside_a_live_eager_graph_of_the_leaves_behind_the_arguments():
    torch = torch_()
    from gym_auv_amd import memory

    u, bc = torch.zeros(2, 5, 8, device="cuda"), torch.zeros(2, 5, 1, 4, device="cuda")
    log_A, w = torch.zeros(8, 4, device="cuda", requires_grad=True), torch.ones(8, 4, device="cuda", requires_grad=True)
    alive = memory.selective_scan(u, u, -torch.exp(log_A), bc, bc)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="drop those first"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            memory.selective_scan(u, u, -torch.exp(log_A), bc, bc)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="drop those first"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            memory.causal_conv(u, log_A)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):       # other leaves: recorded
        memory.causal_conv(u, w)
    torch.cuda.synchronize()
    del alive


def test_step_captured_with_its_state_in_place():
    torch = torch_()
    from gym_auv_amd import memory

    m = Maker(13, "bfloat16")
    B, D, N = 33, 24, 16
    t, start, _ = scan_case(m, B, 1, D, N, 1, 0.3, None, True, True)
    t = {k: v.detach() for k, v in t.items()}
    w, cs = m.par(D, 4), m.rows(B, 3, D)
    mark = start[:, 0].contiguous()

    def step(conv_state, state):
        u = memory.causal_conv_step(t["u"][:, 0], conv_state, w, start=mark)
        return memory.selective_scan_step(u, t["delta"][:, 0], state, t["A"], t["B"][:, 0], t["C"][:, 0], t["D"], t["z"][:, 0], t["delta_bias"],
                                          start=mark)

    a, b = (cs.clone(), t["state"].clone()), (cs.clone(), t["state"].clone())
    step(cs.clone(), t["state"].clone())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step(*a)
    for k in range(5):
        mark.copy_(torch.from_numpy(m.rng.random(B) < 0.3).cuda())
        want = step(*b)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), k


# ----------------------------------------------------------------------------
# together
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,tol", [("float32", 2e-5), ("bfloat16", 0.08)])
def test_memory_of_a_rollout_equals_its_steps(dtype, tol):
    """Two blocks: a rollout with restarts at once, its two halves with the state handed over, and token by token.
    Per block some 400 products of 32 bits stand between the forms, each sum in its own order (a step of 2^-24 each:
    2.4e-5 of values near 1 if all went one way, a tenth in practice); in bfloat16 the four roundings of each block's
    activations, 2^-9 each way, through two blocks with gains near 2: 0.03."""
    torch = torch_()
    from gym_auv_amd import memory

    torch.manual_seed(3)
    B, L, F = 37, 24, 18
    net = memory.EpisodeMemory(F, 32, layers=2, dtype=getattr(torch, dtype)).cuda()
    x = torch.randn(L, B, F, device="cuda").transpose(0, 1)
    start = (torch.rand(L, B, device="cuda") < 0.1).t()
    with torch.no_grad():
        y, state = net(x, start)
        a, s = net(x[:, :11], start[:, :11])
        b, s = net(x[:, 11:], start[:, 11:], state=s)
        halves = torch.cat([a, b], 1)
    live = net.new_state(B)
    steps = torch.stack([net.step(x[:, t], live, start[:, t]) for t in range(L)], 1)
    scale = float(y.float().abs().max())
    assert float((halves - y).float().abs().max()) <= tol * scale
    assert float((steps - y).float().abs().max()) <= tol * scale
    for (c0, h0), (c1, h1), (c2, h2) in zip(state, s, live):
        for p, q, r in ((c0, c1, c2), (h0, h1, h2)):
            top = max(1.0, float(p.float().abs().max()))
            assert float((p - q).float().abs().max()) <= tol * top and float((p - r).float().abs().max()) <= tol * top


def test_memory_gradients_against_differences():
    """Directional differences of a scalar of the whole module, in 32 bits.  A central difference with step e is off by
    e^2 / 6 times the third derivative, and the direction, 0.3 in each of some 8,000 parameters, is 27 long, so that the
    third derivative goes with 27^3: the differences for e and e/2 are combined, (4 d(e/2) - d(e)) / 3, which takes that
    term out.  What is left of the rounding: outputs of size S in 32 bits, S 2^-22 / e = 1.2e-4 S, some three times that
    in the combination."""
    torch = torch_()
    from gym_auv_amd import memory

    torch.manual_seed(4)
    net = memory.EpisodeMemory(18, 16, layers=2).cuda()
    x = torch.randn(5, 20, 18, device="cuda")
    start = torch.rand(5, 20, device="cuda") < 0.1
    weight = torch.randn(5, 20, 16, device="cuda", dtype=torch.float64) / 40
    value = lambda: (net(x, start)[0].double() * weight).sum()   # noqa: E731
    params = list(net.parameters())
    grads = torch.autograd.grad(value(), params)
    assert all(g is not None and bool(torch.isfinite(g).all()) for g in grads)
    at = [p.detach().clone() for p in params]

    @torch.no_grad()
    def difference(way, eps):
        ends = []
        for sign in (1, -1):
            for p, p0, d in zip(params, at, way):
                p.copy_(p0 + sign * eps * d)
            ends.append(float(value()))
        return (ends[0] - ends[1]) / (2 * eps)

    for seed in range(3):
        torch.manual_seed(10 + seed)
        way = [torch.randn_like(p) * 0.3 for p in params]
        eps = 2e-3
        want = (4 * difference(way, eps / 2) - difference(way, eps)) / 3
        got = sum(float((g.double() * d.double()).sum()) for g, d in zip(grads, way))
        assert abs(want - got) <= 5e-3 * max(1.0, abs(got)), seed


def test_extractor_with_memory_follows_the_vessels():
    """A batch stepped with in-step restarts: the memory behind the scan's features, one token per step, equals the
    module over the recorded rollout, with the starts taken from the step counters."""
    import os

    torch = torch_()
    from gym_auv_amd import cnn, memory, scenarios
    from gym_auv_amd.env import VecAuvEnv
    from oracle import cnn_oracle as N

    gold = np.load(os.path.join(os.path.dirname(__file__), "golden", "cnn_golden.npz"))
    cfg, scene = scenarios.make_workload("cfg3_65536_moving", n_envs=256)
    cfg["max_steps"] = 7
    env = VecAuvEnv(cfg, scene, auto_reset="device")
    torch.manual_seed(5)
    net = memory.EpisodeMemory(18, 32).cuda()
    plain = cnn.PerceptionNavigationExtractor("shallow", N.golden_weights(gold, "shallow"))
    ext = cnn.PerceptionNavigationExtractor("shallow", N.golden_weights(gold, "shallow"), memory=net)
    assert ext.features_dim == 32 and plain.features_dim == 18
    obs = env.reset()
    steps = env.sim.tensor("t_step")
    acts = torch.from_numpy(scenarios.random_actions(256, 20, seed=1)).cuda()
    feats, marks, outs = [], [], []
    for k in range(20):
        mark = steps == 0
        feats.append(plain(obs).clone())
        marks.append(mark)
        outs.append(ext(obs, mark))
        obs, _, _, _ = env.step(acts[k].t())
    marks = torch.stack(marks)
    assert bool(marks[0].all()) and bool(marks[1:].any())
    with torch.no_grad():
        want, _ = net(torch.stack(feats).transpose(0, 1), marks.t())
    got = torch.stack(outs, 1)
    assert float((got - want).abs().max()) <= 2e-5 * float(want.abs().max())
    ext.reset()
    assert torch.equal(ext(obs), ext.memory.step(plain(obs), net.new_state(256)))
    env.close()
