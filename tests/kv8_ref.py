"""Plain 64-bit statements of the paged 8-bit cache's calls, sequence by sequence and row by row."""
import numpy as np

PAGE, BLOCK = 64, 16


def k_elem(hd):
    """Element of a page and KV head that holds (row, dim) of K: [64, hd] indices."""
    r, d = np.arange(PAGE)[:, None], np.arange(hd)[None]
    return ((r // 16 * (hd // 64) + d // 64) * 64 + d // 8 % 4 * 16 + r % 16) * 16 + d // 32 % 2 * 8 + d % 8


def v_elem(hd):
    r, d = np.arange(PAGE)[:, None], np.arange(hd)[None]
    return (d // 16 * 64 + r // 4 % 4 * 16 + d % 16) * 16 + r // 16 * 4 + r % 4


def finite(x):
    """f16 rows as the cache takes them."""
    return np.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0).astype(np.float16)


def scale_of(amax):
    """amax / 127 up to the next number of four significant bits or multiple of 2^-24, at least 2^-24; exact in float64."""
    t = float(amax) / 127.0
    unit = 2.0 ** -24
    while 16 * unit < t:          # four bits: 8 .. 16 units
        unit *= 2
    n = int(np.ceil(float(amax) / (127.0 * unit)))
    return max(n, 1) * unit


def codes_of(x, s):
    """Codes (0 .. 255) of f16 values x at scale s: nearest, ties to even."""
    most = 113.0 if s > 512 else 127.0
    return (np.clip(np.rint(x.astype(np.float64) / s), -most, most) + 128).astype(np.uint8)


class Sequence:
    """What a sequence holds: its f16 rows, and the values that stand for them in the cache."""

    def __init__(self, nkv, hd):
        self.nkv, self.hd = nkv, hd
        self.k = np.zeros((0, nkv, hd), np.float16)
        self.v = np.zeros((0, nkv, hd), np.float16)

    def append(self, k, v):
        self.k = np.concatenate([self.k, finite(k).reshape(-1, self.nkv, self.hd)])
        self.v = np.concatenate([self.v, finite(v).reshape(-1, self.nkv, self.hd)])

    def cut(self, rows):
        self.k, self.v = self.k[:rows], self.v[:rows]

    @property
    def rows(self):
        return len(self.k)

    def page(self, p):
        """(K codes, V codes [nkv, 64*hd], scales [nkv, 8]) of full page p, in the page's order."""
        out, sc = [], np.zeros((self.nkv, 8))
        for i, (x, at) in enumerate(((self.k, k_elem(self.hd)), (self.v, v_elem(self.hd)))):
            c = np.zeros((self.nkv, PAGE * self.hd), np.uint8)
            for h in range(self.nkv):
                for a in range(4):
                    r = slice(p * PAGE + 16 * a, p * PAGE + 16 * a + 16)
                    s = sc[h, 4 * i + a] = scale_of(np.abs(x[r, h].astype(np.float64)).max())
                    c[h, at[16 * a:16 * a + 16]] = codes_of(x[r, h], s)
            out.append(c)
        return out[0], out[1], sc

    def values(self):
        """K, V [rows, nkv, hd] float64 as the calls see them."""
        full = self.rows // PAGE * PAGE
        out = []
        for x in (self.k, self.v):
            y = x.astype(np.float64)
            for a in range(0, full, BLOCK):
                for h in range(self.nkv):
                    s = scale_of(np.abs(y[a:a + BLOCK, h]).max())
                    y[a:a + BLOCK, h] = (codes_of(x[a:a + BLOCK, h], s).astype(np.float64) - 128) * s
            out.append(y)
        return out


def attention(q, k, v, before, scale, f16=False):
    """q [n, nh, 2*hd] (query | gate), k, v [rows, nkv, hd] float64, token t sees rows 0 .. before + t -> (out [n, nh, hd]
    float64, bound of an f32 or f16 evaluation's error).

    The bound, with u = 2^-24 (f32), for q in fixed point of its row's largest (three 8-bit digits: half a step is at most 2^-23
    of it; two, for an f16 output: 2^-15) or as an f16 pair (open rows: 2^-22 of the value), and weights as f16 pairs (2^-22)
    or one f16 (2^-11; their sums take them as rounded): with e = 2^-21 or 2^-11, a score is off by ds <= scale sum |q||k| (e + hd u) + 4 u |s|, |q| counted as a quarter or
    a sixteenth of the row's largest at least; a weight by 2 ds + e + 4 u of itself; sums over n keys by n u; so the output
    by 2 (2 ds + e + n u + 8 u) max |v| sigmoid(gate) at most, plus its own rounding. Weights below 2^-31 (2^-24 for one f16) of
    the largest may be lost: n of those times max |v|."""
    n, nh, hd2 = q.shape
    hd, nkv = hd2 // 2, k.shape[1]
    out, tol = np.zeros((n, nh, hd)), np.zeros((n, nh, hd))
    u, e, lost = 2.0 ** -24, (2.0 ** -11 if f16 else 2.0 ** -21), (2.0 ** -24 if f16 else 2.0 ** -31)
    q = q.astype(np.float64)
    for h in range(nh):
        kh, vh = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
        for t in range(n):
            m = before + t + 1
            x = q[t, h, :hd]
            s = scale * (kh[:m] @ x)
            w = np.exp(s - s.max())
            gate = 1 / (1 + np.exp(-q[t, h, hd:]))
            out[t, h] = (w @ vh[:m]) / w.sum() * gate
            size = np.maximum(np.abs(x), np.abs(x).max() / (16 if f16 else 4))
            ds = (abs(scale) * (np.abs(kh[:m]) @ size).max() * (e + hd * u) + 4 * u * np.abs(s).max())
            top = np.abs(vh[:m]).max(0)
            tol[t, h] = 2 * (2 * ds + e + (m + 8) * u + m * lost) * top * gate + 4 * u * np.abs(out[t, h])
            if f16:
                tol[t, h] += 2.0 ** -11 * np.abs(out[t, h]) + 2.0 ** -25
    return out, tol + 1e-30


def attention_rms(q, k, v, before, scale, f16=False, full=None):
    """As `attention`, with how far errors of the documented precisions carry in the mean: (out [n, nh, hd] float64, spread of an
    element's error [n, nh, hd], its own roundings [n, nh, hd]). full: rows before this one stand in full pages (all rows, if none
    is given). An output's error is at most SIGMAS spreads and the roundings.

    out = sum_j p_j v_j. A relative error e_j of weight j moves it by p_j e_j (v_j - out), where the sum of the weights has the same
    errors (one f16: its sum takes it as rounded), and by p_j e_j v_j else. The e_j of different keys are
    independent as far as K and V are; so the spread is the root of the sum of p_j^2 e_j^2 (v_j - out)^2, with e_j^2 the sum of
    - the score's error by q: half a step is h = 2^-15 (f16) or 2^-23 of the row's largest |q|, times 128/127 (the highest digit
      ends at 127), even in +-h: scale |k_j| h / sqrt 3; against open rows 2^-22 of each q_d, where that is more
    - the score's f32 roundings: 4 of |s_j - s_max| + |s_max| + 1 at 2^-24, and the open rows' sum of hd products in f32
    - the weight's: 2^-11 (one f16) or 2^-22 (a pair) / sqrt 3 of itself, or 2^-31 of the largest.
    The sum over m keys in f32 adds 2^-24 / sqrt 3 of a partial sum, page after page or of a split (so at most twice the largest page
    after page), at each of m / 16 products of matrix instructions and 16 more; and inside those, over 8 values, three times the root of
    the sum of (p_j v_j)^2.
    The roundings: 6 * 2^-24 of the result for the division and the gate, and half a step of f16 for such an output."""
    n, nh, hd2 = q.shape
    hd, nkv = hd2 // 2, k.shape[1]
    G = nh // nkv
    out, spread = np.zeros((n, nh, hd)), np.zeros((n, nh, hd))
    u, h0, ew = 2.0 ** -24, 2.0 ** (-15 if f16 else -23) * 128 / 127, 2.0 ** (-11 if f16 else -22)
    full = k.shape[0] if full is None else full
    q = q.astype(np.float64)
    for kh in range(nkv):
        key, val = np.ascontiguousarray(k[:, kh]), np.ascontiguousarray(v[:, kh])
        key2, val2 = key * key, val * val
        for t in range(n):
            m = before + t + 1
            x, kk, vv, k2, v2 = q[t, kh * G:kh * G + G, :hd], key[:m], val[:m], key2[:m], val2[:m]
            s = scale * (x @ kk.T)                                    # [G, m]
            most = s.max(1, keepdims=True)
            w = np.exp(s - most)
            p = w / w.sum(1, keepdims=True)
            o = p @ vv
            h = np.abs(x).max(1, keepdims=True) * h0
            e2 = scale * scale * k2.sum(1) * h * h / 3
            open_ = np.arange(m) >= full
            if open_.any():
                e2 = e2 + open_ * scale * scale * (2.0 ** -44 / 3 + hd * u * u) * ((x * x) @ k2.T)
            e2 = e2 + (4 * u * (np.abs(s - most) + np.abs(most) + 1)) ** 2
            a2 = p * p * (e2 + ew * ew / 3) + (2.0 ** -31 * p.max(1, keepdims=True)) ** 2 / 3
            # sum_j a2_j (v_j - o)^2 or, for pairs, of v_j^2 + o^2 at most
            var = a2 @ v2 + (0 if f16 else 1) * a2.sum(1, keepdims=True) * o * o
            if f16:
                var = var - 2 * o * (a2 @ vv) + a2.sum(1, keepdims=True) * o * o
            ends = np.stack([p[:, a:a + PAGE] @ vv[a:a + PAGE] for a in range(0, m, PAGE)])
            part = np.abs(np.cumsum(ends, 0)).max(0)
            var = np.maximum(var, 0) + u * u * ((m / 16 + 16) / 3 * (2 * part) ** 2 + 9 * (p * p) @ v2)
            gate = 1 / (1 + np.exp(-np.clip(q[t, kh * G:kh * G + G, hd:], -700, 700)))
            out[t, kh * G:kh * G + G] = o * gate
            spread[t, kh * G:kh * G + G] = np.sqrt(var) * gate
    own = 6 * u * np.abs(out)
    if f16:
        own = own + 2.0 ** -11 * np.abs(out) + 2.0 ** -25
    return out, spread, own


SIGMAS = 6.0


def too_far(got, want, spread, own):
    """Whether a row [.., hd] of outputs has an element further off than `attention_rms` allows."""
    return ~(np.abs(got - want) <= SIGMAS * spread + own + 1e-30).all(-1)


class Cuts:
    """To which lengths a sequence may be cut by its length alone: to a page's end, or into page `lowest` or a later one."""

    def __init__(self):
        self.rows = self.lowest = 0

    def append(self, n):
        self.rows += n
        self.lowest = max(self.lowest, (self.rows - 1) // PAGE - 1)

    def may(self, to):
        return 0 <= to <= self.rows and (to % PAGE == 0 or to // PAGE >= self.lowest)

    def cut(self, to):
        assert self.may(to)
        self.rows, self.lowest = to, min(self.lowest, to // PAGE)
