"""Plain 64-bit statements of the tree-verification calls, node by node along the parents, and tree shapes."""
import numpy as np

SHAPES = ["chain", "star", "random", "forest", "padded"]


def parents(shape: str, nt: int, seed: int = 0) -> np.ndarray:
    """int32 [nt]: -1 follows the last committed token, anything else outside 0 .. t-1 is padding."""
    r = np.random.default_rng(seed)
    if shape == "chain":
        p = [t - 1 for t in range(nt)]
    elif shape == "star":
        p = [-1] + [0] * (nt - 1)
    elif shape == "forest":                    # several first candidates
        p = [-1 if t % 3 == 0 else t - 1 for t in range(nt)]
    else:
        p = [-1] + [int(r.integers(max(-1, t - 9), t)) for t in range(1, nt)]
    if shape == "padded" and nt > 1:           # padding of every kind, in the middle and at the end
        p[nt - 1] = -2
        if nt > 4:
            p[nt // 2] = nt                    # after its own place
            p[nt // 3] = nt // 3               # its own parent
    return np.array(p[:nt], np.int32)


def path(par: np.ndarray, t: int):
    """Ancestors of node t and t itself, first first; None for a padding node."""
    out = []
    while t != -1:
        if not -1 <= par[t] < t:
            return None
        out.append(int(t))
        t = int(par[t])
    return out[::-1]


def masks(par: np.ndarray) -> np.ndarray:
    """int64 [nt] ancestor masks."""
    out = np.zeros(len(par), np.uint64)
    for t in range(len(par)):
        for a in path(par, t) or []:
            out[t] |= np.uint64(1) << np.uint64(a)
    return out.view(np.int64)


def norm_rotate(x, w, eps, pos, freq, mscale, pairs):
    """x [nt, heads, hd] -> (rotated rows, |a| + |b| of each element's pair before the rotation), float64."""
    x = x.astype(np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 if w is None else w.astype(np.float64))
    n = len(freq)
    i = np.arange(n)
    a, b = (2 * i, 2 * i + 1) if pairs else (i, i + n)
    ang = pos.astype(np.float64)[:, None] * freq.astype(np.float64)[None]
    c, s = np.cos(ang)[:, None] * mscale, np.sin(ang)[:, None] * mscale
    y, size = x.copy(), np.abs(x)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * abs(mscale)
    return y, size


def attn(q, k, v, pos0, nh, nkv, anc, scale):
    """f64 attention of tree nodes: q [nt, nh, 2*hd], k / v [rows, nkv*hd] (hidden rows are not looked at). Returns out
    [nt, nh, hd] and a bound of an f32 computation's error from it, element by element."""
    nt, hd = q.shape[0], q.shape[2] // 2
    rows = len(k)
    q = q.astype(np.float64)
    k, v = (x.reshape(rows, nkv, hd) for x in (k, v))
    out, tol = np.zeros((nt, nh, hd)), np.zeros((nt, nh, hd))
    for kh in range(nkv):
        heads = np.arange(nh // nkv) + kh * (nh // nkv)
        kp, vp = k[:pos0, kh].astype(np.float64), v[:pos0, kh].astype(np.float64)
        for t in range(nt):
            own = [j for j in range(nt) if int(anc[t]) >> j & 1]
            if not own:
                continue
            kk = np.concatenate([kp, k[pos0 + np.array(own), kh].astype(np.float64)])
            vv = np.concatenate([vp, v[pos0 + np.array(own), kh].astype(np.float64)])
            qt = q[t, heads, :hd]
            s = scale * qt @ kk.T
            p = np.exp(s - s.max(-1, keepdims=True))
            l = p.sum(-1, keepdims=True)
            o = p @ vv / l
            gate = 1 / (1 + np.exp(-q[t, heads, hd:]))
            # scores: q as two f16 (2^-22), 256 additions of independent roundings (16 steps of 2^-24); weights: two
            # f16 of the largest weight's size (2^-25 a key) and the exponentials (4 steps); the sums alike 16, the
            # division, the gate and the products 8
            size = scale * (np.abs(qt) @ np.abs(kk).T).max(-1, keepdims=True)
            vmax = np.abs(vv).max(0)
            rel = 2 * (20 * size + 4) + 32
            out[t, heads] = o * gate
            tol[t, heads] = (rel * 2.0 ** -24 + len(kk) * 2.0 ** -25 / l) * vmax * gate
    return out, tol


def gdn(x, w, conv, beta, alpha, dt, a, state, par, nv, nk, eps):
    """f64 recurrent layer node by node: out [nt, nv, 128] and a bound of an f32 computation's error, and per node the
    state and its error bound (scalars per head), and the conv window."""
    S, nt = 128, len(par)
    x, w, conv, state = (z.astype(np.float64) for z in (x, w, conv, state))
    K = w.shape[1]
    out, tol = np.zeros((nt, nv, S)), np.zeros((nt, nv, S))
    head = np.arange(nv) % nk
    states, errs, windows = {-1: state}, {-1: np.zeros(nv)}, {-1: conv}
    sig = lambda z: 1 / (1 + np.exp(-z))
    for t in range(nt):
        if path(par, t) is None:
            continue
        p = int(par[t])
        win = np.concatenate([windows[p], x[t:t + 1]])
        windows[t] = win[1:]
        y = (win * w.T).sum(0)
        size = (np.abs(win) * np.abs(w.T)).sum(0).reshape(-1, S).max(-1)     # of the sums that the conv rounds
        y = (y * sig(y)).reshape(-1, S)
        q, k, v = y[:nk], y[nk:2 * nk], y[2 * nk:]
        norms = [np.maximum(np.linalg.norm(z, axis=-1, keepdims=True), eps) for z in (q, k)]
        # relative error of a normalised row: conv and SiLU 6 steps of the sums' size, the norm 12
        rq, rk = (6 * size[i * nk:(i + 1) * nk] * np.sqrt(S) / n[:, 0] + 12 for i, n in enumerate(norms))
        q, k = (q / norms[0])[head], (k / norms[1])[head]
        rq, rk = rq[head], rk[head]
        b = sig(beta[t].astype(np.float64))
        g = np.log1p(np.exp(alpha[t].astype(np.float64) + dt)) * a.astype(np.float64)
        d = np.exp(g)
        s = states[p] * d[:, None, None]
        u = (v - np.einsum("hij,hi->hj", s, k)) * b[:, None]
        states[t] = s + k[:, :, None] * u[:, None, :]
        col = np.linalg.norm(s, axis=1).max(-1)                              # largest column norm of each head
        # the update's error: v (6 steps of its sums, 8 more), S^T k (k's error, 16 steps of the sum, the decays 12, and
        # what the state's columns are off by already), beta 6
        vmax = np.abs(v).max(-1)
        eu = 2.0 ** -24 * (6 * size[2 * nk:] + 14 * vmax + (rk + 34) * col) + errs[p] * d
        umax = np.abs(u).max(-1)
        # a column's error grows by the update's (|k| = 1), k's own error and the decays
        errs[t] = errs[p] * d + eu + 2.0 ** -24 * (rk * umax + 12 * col + 4 * (col + umax))
        col = np.linalg.norm(states[t], axis=1).max(-1)
        out[t] = np.einsum("hij,hi->hj", states[t], q) / np.sqrt(S)
        tol[t] = ((errs[t] + 2.0 ** -24 * (rq + 20) * col) / np.sqrt(S))[:, None]
    return out, tol, states, errs, windows
