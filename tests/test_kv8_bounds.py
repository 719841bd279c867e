"""The error bound that the paged 8-bit cache's attention is held to lets the documented arithmetic through and nothing much
worse: an evaluation of it in numpy passes, and one that has lost a digit, a page or the right values does not, at the shapes of the
GPU tests. No device work."""
import numpy as np
import pytest

from tests import kv8_ref as ref


def rows(rng, n, nkv, hd):
    k = rng.standard_normal((n, nkv, hd))
    k /= np.sqrt((k * k).mean(-1, keepdims=True))
    return k.astype(np.float16), rng.standard_normal((n, nkv, hd)).astype(np.float16)


def half(x):
    return x.astype(np.float16).astype(np.float64)


def evaluate(q, k, v, before, scale, f16, digits, full, without=()):
    """The attention with q in `digits` signed digits of 8 bits for the rows of full pages (f16 pairs for the open ones), weights of
    a reference 7 below the row's maximum as f16 or f16 pairs, sums in float64, without the rows named."""
    n, nh, hd2 = q.shape
    hd, nkv = hd2 // 2, k.shape[1]
    out = np.zeros((n, nh, hd))
    for h in range(nh):
        kh = h // (nh // nkv)
        for t in range(n):
            m = before + t + 1
            x = q[t, h, :hd].astype(np.float64)
            ex = np.frexp(np.abs(x).max())[1]
            top = 127.0 * 256 ** (digits - 1)
            coarse = np.rint(np.ldexp(x * top, -ex)) * np.ldexp(1 / top, ex)
            y = np.ldexp(x, 14 - ex)
            fine = np.ldexp(half(y) + half(y - half(y)), ex - 14)
            s = scale * np.where(np.arange(m) < full, k[:m, kh] @ coarse, k[:m, kh] @ fine) * np.log2(np.e)
            s[[r for r in without if r < m]] = -np.inf
            w = np.exp2(s - s.max() + 7)
            hi = half(w)
            p, total = (hi, hi.sum()) if f16 else (hi + half(w - hi), w.sum())
            gate = 1 / (1 + np.exp(-q[t, h, hd:].astype(np.float64)))
            out[t, h] = (p @ v[:m, kh] / total * gate).astype(np.float16 if f16 else np.float32)
    return out


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("before,n,nh,nkv,hd", [(9000, 2, 8, 1, 256), (4103, 2, 6, 1, 256), (8190, 1, 8, 1, 256), (20000, 1, 2, 1, 128), (2900, 2, 8, 1, 128),
                                                (1000, 2, 8, 2, 256), (300, 3, 8, 1, 128), (8384, 2, 8, 1, 256), (130, 5, 4, 2, 256)])
def test_the_bound_passes_the_arithmetic_and_nothing_worse(before, n, nh, nkv, hd, f16):
    rng = np.random.default_rng(before + n)
    seq = ref.Sequence(nkv, hd)
    seq.append(*rows(rng, before + n, nkv, hd))
    k, v = seq.values()
    q = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32)
    full, scale, digits = seq.rows // 64 * 64, hd ** -0.5, 2 if f16 else 3
    bound = ref.attention_rms(q, k, v, before, scale, f16, full)
    assert np.allclose(bound[0], ref.attention(q, k, v, before, scale, f16)[0], rtol=0, atol=1e-12)
    run = lambda k=k, v=v, digits=digits, **kw: evaluate(q, k, v, before, scale, f16, digits, full, **kw)
    assert not ref.too_far(run(), *bound).any()
    page = full // 128 * 64                                       # a full page in the middle
    swapped, other = v.copy(), 0 if page else 64
    swapped[page:page + 64] = v[other:other + 64]
    wrong = dict(zeros=np.zeros_like(bound[0]), digit=run(digits=digits - 1), page=run(without=range(page, page + 64)), values=run(v=swapped))
    for name, got in wrong.items():
        assert ref.too_far(got, *bound).all(), (name, ref.too_far(got, *bound).mean())


@pytest.mark.parametrize("f16", [False, True])
def test_the_bound_with_single_large_dims(f16):
    """Queries with a dim far above the rest, whose fixed point is of that dim, and V in blocks of very different size."""
    rng = np.random.default_rng(4)
    seq = ref.Sequence(1, 256)
    k, v = rows(rng, 700, 1, 256)
    k[:, :, 5] = k[:, :, 5] * np.float16(0.1)
    v *= np.float16(2.0) ** (np.arange(700) // 16 % 9 - 6).astype(np.float16)[:, None, None]
    seq.append(k, v)
    k, v = seq.values()
    q = rng.standard_normal((2, 8, 512)).astype(np.float32)
    q[..., 5] *= 100
    bound = ref.attention_rms(q, k, v, 698, 1 / 16, f16, 640)
    digits = 2 if f16 else 3
    assert not ref.too_far(evaluate(q, k, v, 698, 1 / 16, f16, digits, 640), *bound).any()
    assert ref.too_far(evaluate(q, k, v, 698, 1 / 16, f16, digits - 1, 640), *bound).all()
