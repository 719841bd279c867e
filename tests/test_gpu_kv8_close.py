"""The 8-bit cache's attention against the bound of its documented precisions (kv8_ref.attention_rms), which zeros, a lost digit, a
lost page or another page's values pass nowhere (test_kv8_bounds.py)."""
import numpy as np
import pytest
import torch

from irontimber_amd import ops
from tests import kv8_ref as ref
from tests.gpu_util import announce, dev_f32, host
from tests.test_gpu_kv8 import Engine

pytestmark = pytest.mark.gpu


class Close(Engine):
    def attend(self, q, start, length, counts, nh, scale=None, f16=False, some=None):
        """As Engine.attend, for the sequences `some` (all, if none are given)."""
        n, sc, at = sum(counts), 1 / self.hd ** 0.5 if scale is None else scale, 0
        out = ops.attn_kv8(self.cache, dev_f32(q.reshape(n, -1), self.dev), start, length, self.table, nh, max(counts), scale=scale,
                           out_dtype=torch.float16 if f16 else torch.float32)
        got = host(out).astype(np.float64).reshape(n, nh, self.hd)
        for i, (s, c) in enumerate(zip(self.seqs, counts)):
            if c and (some is None or i in some):
                k, v = s.values()
                want, spread, own = ref.attention_rms(q[at:at + c], k, v, s.rows - c, sc, f16, s.rows // 64 * 64)
                far = ref.too_far(got[at:at + c], want, spread, own)
                worst = float((np.abs(got[at:at + c] - want) / (ref.SIGMAS * spread + own + 1e-30)).max())
                assert not far.any(), (i, c, s.rows, f16, worst, np.argwhere(far)[:5].tolist())
            at += c


@pytest.mark.parametrize("before,n,nh,nkv,hd,wide", [
    (8190, 1, 16, 2, 256, 0), (20000, 1, 4, 2, 128, 0), (4103, 4, 24, 4, 256, 0), (9000, 8, 16, 2, 256, 600), (4103, 4, 16, 2, 256, 600),
    (5000, 33, 2, 1, 128, 0), (1000, 90, 16, 2, 256, 0), (2000, 40, 24, 4, 256, 0), (130, 5, 34, 1, 128, 0), (63, 66, 8, 8, 128, 0)])
def test_lengths(dev, before, n, nh, nkv, hd, wide):
    announce(f"kv8 close {before} + {n} {nh}/{nkv} {hd} wide {wide}")
    e = Close(dev, 1, nkv, hd, (before + n) // 64 + 1, wide=wide)
    e.append([before])
    start, length = e.append([n])
    q = e.queries(n, nh)
    for f16 in (False, True):
        e.attend(q, start, length, [n], nh, f16=f16)


@pytest.mark.parametrize("lens,counts,nh,nkv,hd", [
    ([2000 + (i * 379) % 1000 for i in range(68)], [0 if i in (5, 64) else 1 + i % 2 for i in range(68)], 16, 2, 128),
    ([9000, 700, 200, 130], [20, 20, 20, 20], 16, 2, 256),
    ([61 + 37 * i for i in range(16)], [5] * 16, 16, 2, 256),
    ([37 * i for i in range(9)], [16] * 9, 32, 4, 256),
    ([1000, 0, 63], [129, 64, 65], 16, 2, 256),
    ([0, 300, 63, 0, 128], [1, 203, 97, 0, 5], 24, 4, 256),
    ([0, 300], [600, 200], 128, 16, 128)])
def test_batches(dev, lens, counts, nh, nkv, hd):
    announce(f"kv8 close batch {len(lens)} {sum(counts)} {nh}/{nkv} {hd}")
    e = Close(dev, len(lens), nkv, hd, max(a + b for a, b in zip(lens, counts)) // 64 + 1)
    e.append(lens)
    start, length = e.append(counts)
    q = e.queries(sum(counts), nh)
    for f16 in (False, True):
        e.attend(q, start, length, counts, nh, f16=f16, some=None if len(lens) < 20 else (0, 1, 6, 63, 65, 67))


@pytest.mark.parametrize("n", [1, 4, 20])
def test_many_pages_of_one_split(dev, n):
    """130 sequences that share a beginning of 131 pages, a split each: the page numbers and scales are read anew twice."""
    nseq, nkv, hd, before = 130, 2, 256, 64 * 131 + 3
    e = Close(dev, nseq, nkv, hd, 2, spare=140)
    base = np.random.default_rng(2).permutation(140)[:132].astype(np.int32)
    e.table_np = np.repeat(base[None], nseq, 0)
    e.table = torch.from_numpy(e.table_np.copy()).to(dev)
    e.append([before] + [0] * (nseq - 1))
    ops.kv8_copy(e.cache, seq_src=e.ints([0] * (nseq - 1)), seq_dst=e.ints(list(range(1, nseq))))
    for s in e.seqs[1:]:
        s.k, s.v = e.seqs[0].k, e.seqs[0].v
    start, length = e.append([n] * nseq)
    q = e.queries(n * nseq, 8)
    for f16 in (False, True):
        e.attend(q, start, length, [n] * nseq, 8, f16=f16, some=(0, 101))


@pytest.mark.parametrize("before,n", [(698, 2), (8000, 4), (300, 60)])
@pytest.mark.parametrize("large", [30.0, 1000.0])
def test_single_large_dims(dev, before, n, large):
    """Queries with a dim far above the rest, whose fixed point is of that dim, and V in blocks of very different size."""
    e = Close(dev, 1, 2, 256, (before + n) // 64 + 1)
    k, v = e.rows(before + n)
    k[:, [5, 261]] *= np.float16(0.1)
    v *= (2.0 ** (np.arange(before + n) // 16 % 9 - 6)).astype(np.float16)[:, None]
    e.append([before], rows=(k[:before], v[:before]))
    start, length = e.append([n], rows=(k[before:], v[before:]))
    q = e.queries(n, 16)
    q[:, :, 5] *= large
    q[:, 3, 200] = large
    for f16 in (False, True):
        e.attend(q, start, length, [n], 16, f16=f16)


@pytest.mark.parametrize("lens,counts,nh,nkv,hd", [
    ([600], [1], 16, 2, 256), ([9000, 64, 131, 0], [1, 2, 0, 1], 16, 2, 256), ([5000], [4], 8, 2, 128), ([37 * i for i in range(70)], [1] * 70, 64, 4, 128)])
def test_few_rows_are_as_exact_in_f16(dev, lens, counts, nh, nkv, hd):
    """At most 16 query rows of a KV head: an f16 output is the f32 one, rounded to nearest."""
    e = Engine(dev, len(lens), nkv, hd, max(a + b for a, b in zip(lens, counts)) // 64 + 1)
    e.append(lens)
    start, length = e.append(counts)
    q = dev_f32(e.queries(sum(counts), nh).reshape(sum(counts), -1), dev)
    run = lambda t: ops.attn_kv8(e.cache, q, start, length, e.table, nh, max(counts), out_dtype=t)
    assert torch.equal(run(torch.float16), run(torch.float32).half())
