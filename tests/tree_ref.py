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
