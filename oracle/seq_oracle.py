"""The sequence operators in float64, token by token, with their gradients.

Everything is written out for one token after another (numpy, no vectorisation over
time).  Beside each value stands its magnitude: the same sum with every term's absolute
value, which is what a rounding error is relative to.  An output of the library's kernels
is right if it lies within

    K u magnitude + half a step of its type * |value|,     u = 2^-24

with K counting the roundings on the longest way into one term (each function's docstring).
"""
import numpy as np

U32 = 2.0 ** -24


def sigmoid(x):
    return 1.0 / (1.0 + np.exp(-x))


def softplus(x):
    return np.maximum(x, 0.0) + np.log1p(np.exp(-np.abs(x)))


def _rows(lengths, B, L):
    return np.full(B, L) if lengths is None else np.clip(lengths, 0, L)


def conv(x, weight, bias=None, start=None, lengths=None, state=None, silu=True, dy=None, dnew=None):
    """Values and magnitudes: dict name -> (value, magnitude).  K: W + 2 for pre; the SiLU and its
    slope are Lipschitz with constant 1.1 and cost 6 roundings more; sums over T tokens add T."""
    x, weight = np.asarray(x, np.float64), np.asarray(weight, np.float64)
    B, L, D = x.shape
    W = weight.shape[1]
    bias = np.zeros(D) if bias is None else np.asarray(bias, np.float64)
    first = np.zeros((B, W - 1, D)) if state is None else np.asarray(state, np.float64)
    start = np.zeros((B, L), bool) if start is None else np.asarray(start, bool)
    n = _rows(lengths, B, L)
    y, ym = np.zeros((B, L, D)), np.zeros((B, L, D))
    new = np.zeros_like(first)
    out = {}
    grads = dy is not None
    dx, dxm = np.zeros_like(x), np.zeros_like(x)
    dw, dwm = np.zeros_like(weight), np.zeros_like(weight)
    db, dbm = np.zeros(D), np.zeros(D)
    ds, dsm = np.zeros_like(first), np.zeros_like(first)
    for b in range(B):
        window = [(first[b, i], ("s", i)) for i in range(W - 1)]        # (value, where it came from)
        for l in range(n[b]):
            if start[b, l]:
                window = [(np.zeros(D), None)] * (W - 1)
            row = window + [(x[b, l], ("x", l))]
            pre = bias + sum(v * weight[:, j] for j, (v, _) in enumerate(row))
            mag = np.abs(bias) + sum(np.abs(v * weight[:, j]) for j, (v, _) in enumerate(row))
            s = sigmoid(pre)
            y[b, l], ym[b, l] = (pre * s, mag) if silu else (pre, mag)
            window = row[1:]
            if grads:
                slope = s * (1.0 + pre * (1.0 - s)) if silu else np.ones(D)
                g = dy[b, l] * slope
                gm = np.abs(dy[b, l]) * (1.1 + mag)
                db += g
                dbm += gm
                for j, (v, source) in enumerate(row):
                    dw[:, j] += g * v
                    dwm[:, j] += gm * np.abs(v)
                    if source is not None:
                        to, tom = (dx, dxm) if source[0] == "x" else (ds, dsm)
                        to[b, source[1]] += g * weight[:, j]
                        tom[b, source[1]] += gm * np.abs(weight[:, j])
        for i, (v, source) in enumerate(window):
            new[b, i] = v
            if grads and dnew is not None and source is not None:
                to, tom = (dx, dxm) if source[0] == "x" else (ds, dsm)
                to[b, source[1]] += dnew[b, i]
                tom[b, source[1]] += np.abs(dnew[b, i])
    out.update(y=(y, ym), new_state=(new, np.abs(new)))
    if grads:
        out.update(x=(dx, dxm), weight=(dw, dwm), bias=(db, dbm), state=(ds, dsm))
    return out


def scan(u, delta, A, Bm, Cm, D=None, z=None, delta_bias=None, softplus_on=True, start=None, lengths=None, state=None,
         dy=None, dnew=None):
    """Values and magnitudes.  A term of a state goes through at most one decay e^-x per token, x = dt |A|:
    the product and the exponential round once each, the exponent twice (which moves the decay by
    2 x e^-x < 0.8), and dt itself is off by up to (|raw| + 8) u (by 0.37 of that: 6 for |raw| <= 8).
    With N + 12 other roundings K = 10 (L + N + 12); sums over T more terms add T."""
    f = lambda t: None if t is None else np.asarray(t, np.float64)   # noqa: E731
    u, delta, A, Bm, Cm, D, z, delta_bias, state, dy, dnew = map(f, (u, delta, A, Bm, Cm, D, z, delta_bias, state, dy, dnew))
    B, L, Dc = u.shape
    G, N = Bm.shape[2:]
    chan = np.arange(Dc) // (Dc // G)
    skip = np.zeros(Dc) if D is None else D
    start = np.zeros((B, L), bool) if start is None else np.asarray(start, bool)
    n = _rows(lengths, B, L)
    raw = delta + (0.0 if delta_bias is None else delta_bias)
    dt = softplus(raw) if softplus_on else raw
    slope = sigmoid(raw) if softplus_on else np.ones_like(raw)
    sz = np.ones_like(u) if z is None else z * sigmoid(z)
    y, ym = np.zeros_like(u), np.zeros_like(u)
    new = np.zeros((B, Dc, N)) if state is None else state.copy()
    newm = np.abs(new)
    grads = dy is not None
    shapes = dict(u=u, delta=u, z=u, A=A, B=Bm, C=Cm, D=skip, delta_bias=skip, state=new)
    g = {k: np.zeros_like(v) for k, v in shapes.items()}
    m = {k: np.zeros_like(v) for k, v in shapes.items()}
    for b in range(B):
        h, hm = new[b].copy(), newm[b].copy()
        hist = []
        for l in range(n[b]):
            if start[b, l]:
                h, hm = np.zeros_like(h), np.zeros_like(h)
            before = (h, hm)
            e = np.exp(dt[b, l][:, None] * A)
            x = (dt[b, l] * u[b, l])[:, None] * Bm[b, l, chan]
            h, hm = e * h + x, e * hm + np.abs(x)
            c = Cm[b, l, chan]
            yy, yym = (h * c).sum(1) + skip * u[b, l], (hm * np.abs(c)).sum(1) + np.abs(skip * u[b, l])
            y[b, l], ym[b, l] = yy * sz[b, l], yym * np.abs(sz[b, l])
            hist.append((before, (h, hm), e, yy, yym))
        new[b], newm[b] = h, hm
        if not grads:
            continue
        carry = np.zeros_like(h) if dnew is None else dnew[b].copy()
        cm = np.abs(carry)
        for l in range(n[b] - 1, -1, -1):
            (h0, h0m), (h1, h1m), e, yy, yym = hist[l]
            bb, cc = Bm[b, l, chan], Cm[b, l, chan]
            gy, gym = dy[b, l] * sz[b, l], np.abs(dy[b, l] * sz[b, l])
            if z is not None:
                s = sigmoid(z[b, l])
                dz = s * (1.0 + z[b, l] * (1.0 - s))
                g["z"][b, l] = dy[b, l] * yy * dz
                m["z"][b, l] = np.abs(dy[b, l]) * yym * (1.1 + np.abs(z[b, l]))
            d, a = dt[b, l][:, None], np.abs(dt[b, l])[:, None]
            uu = u[b, l][:, None]
            dh, dhm = carry + gy[:, None] * cc, cm + gym[:, None] * np.abs(cc)
            for name, t, tm in (("C", gy[:, None] * h1, gym[:, None] * h1m), ("B", dh * d * uu, dhm * a * np.abs(uu))):
                for k in range(G):
                    g[name][b, l, k] += t[chan == k].sum(0)
                    m[name][b, l, k] += tm[chan == k].sum(0)
            s1, s1m = (dh * bb).sum(1), (dhm * np.abs(bb)).sum(1)
            through, thm = dh * e * h0, dhm * e * h0m
            g["u"][b, l] = s1 * dt[b, l] + gy * skip
            m["u"][b, l] = s1m * a[:, 0] + gym * np.abs(skip)
            dr = (s1 * u[b, l] + (through * A).sum(1)) * slope[b, l]
            drm = (s1m * np.abs(u[b, l]) + (thm * np.abs(A)).sum(1)) * slope[b, l]
            g["delta"][b, l], m["delta"][b, l] = dr, drm
            g["delta_bias"] += dr
            m["delta_bias"] += drm
            g["D"] += gy * u[b, l]
            m["D"] += gym * np.abs(u[b, l])
            g["A"] += through * d
            m["A"] += thm * a
            carry, cm = (np.zeros_like(dh), np.zeros_like(dh)) if start[b, l] else (dh * e, dhm * e)
        g["state"][b], m["state"][b] = carry, cm
    out = {"y": (y, ym), "new_state": (new, newm)}
    if grads:
        out.update({k: (g[k], m[k]) for k in g})
    return out


def norm(x, y=None, post_weight=None, pre_weight=None, gate=None, scale=None, gate_act="silu", eps=1e-6, dx_out=None, dh=None):
    """Values and magnitudes over rows [R, D].  K: D + 24 (the sums over a row, and the elementwise products)."""
    f = lambda t: None if t is None else np.asarray(t, np.float64)   # noqa: E731
    x, y, post_weight, pre_weight, gate, scale, dx_out, dh = map(f, (x, y, post_weight, pre_weight, gate, scale, dx_out, dh))
    R, D = x.shape
    out = {}
    one = np.ones(D)
    w1, w2, sc = (one if t is None else t for t in (post_weight, pre_weight, scale))
    act, slope = np.ones_like(x), np.zeros_like(x)
    if gate is not None:
        s = sigmoid(gate)
        act, slope = {"silu": (gate * s, s * (1 + gate * (1 - s))), "sigmoid": (s, s * (1 - s)), None: (gate, np.ones_like(gate))}[gate_act]
    r, rm = x, np.abs(x)
    if y is not None:
        r1 = 1 / np.sqrt((y * y).mean(1, keepdims=True) + eps) if post_weight is not None else np.ones((R, 1))
        n = y * r1 * w1
        r = x + sc * act * n
        rm = np.abs(x) + np.abs(sc * act * n)
        out["x_out"] = (r, rm)
    r2 = 1 / np.sqrt((r * r).mean(1, keepdims=True) + eps)
    if pre_weight is not None:
        out["h"] = (r * r2 * w2, rm * r2 * np.abs(w2))
    if dx_out is None and dh is None:
        return out
    dr = np.zeros_like(x) if dx_out is None else dx_out
    drm = np.abs(dr)
    # the norm's factor is itself off by what x' is off by, relative to the row's mean magnitude
    q = (rm * rm).mean(1, keepdims=True) * r2 ** 2
    if dh is not None:
        t = dh * w2
        dr = dr + r2 * t - r * r2 ** 3 * (t * r).mean(1, keepdims=True)
        drm = drm + (r2 * np.abs(t) + rm * r2 ** 3 * (np.abs(t) * rm).mean(1, keepdims=True)) * (1 + q)
        out["pre_weight"] = ((dh * r * r2).sum(0), (np.abs(dh) * rm * r2 * (1 + q)).sum(0))
    out["x"] = (dr, drm)
    if y is not None:
        out["scale"] = ((dr * act * n).sum(0), (drm * np.abs(act * n)).sum(0))
        if gate is not None:
            out["gate"] = (dr * sc * n * slope, drm * np.abs(sc * n) * (1.1 + np.abs(gate)))
        dn, dnm = dr * sc * act, drm * np.abs(sc * act)
        if post_weight is not None:
            t, tm = dn * w1, dnm * np.abs(w1)
            out["y"] = (r1 * t - y * r1 ** 3 * (t * y).mean(1, keepdims=True),
                        r1 * tm + np.abs(y) * r1 ** 3 * (tm * np.abs(y)).mean(1, keepdims=True))
            out["post_weight"] = ((dn * y * r1).sum(0), (dnm * np.abs(y) * r1).sum(0))
        else:
            out["y"] = (dn, dnm)
    return out
