"""The paged 8-bit cache: appending, reading, copying and attention, against the 64-bit statements of tests/kv8_ref.py."""
import numpy as np
import pytest
import torch

from irontimber_amd import _lib, ops
from tests import kv8_ref as ref
from tests.gpu_util import announce, dev_f32, host
from tests.test_gpu_guard_bands import assert_bands, banded

pytestmark = pytest.mark.gpu


class Engine:
    """A cache with its tables on the device, and the same sequences in the reference. Pages come from a shuffled list."""

    def __init__(self, dev, nseq, nkv, hd, max_pages, seed=0, spare=2, wide=0):
        self.dev, self.nkv, self.hd, self.nseq = dev, nkv, hd, nseq
        npages = nseq * max_pages + spare
        self.cache = ops.kv8_cache(npages, nseq, nkv, hd, dev)
        for t in self.cache[:2]:
            t.fill_(0xA5)
        for t in self.cache[2:]:        # what was never written is never used
            t.fill_(float("nan"))
        order = np.random.default_rng(seed).permutation(npages)
        self.table_np = order[:nseq * max_pages].reshape(nseq, max_pages).astype(np.int32)
        self.table = torch.from_numpy(np.pad(self.table_np, ((0, 0), (0, wide)), constant_values=-1)).to(dev)
        self.seqs = [ref.Sequence(nkv, hd) for _ in range(nseq)]
        self.rng = np.random.default_rng(seed + 1)

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def batch(self, counts):
        start = np.concatenate([[0], np.cumsum(counts)])
        return self.ints(start.tolist()), self.ints([s.rows for s in self.seqs])

    def rows(self, n, scale=1.0):
        k = self.rng.standard_normal((n, self.nkv, self.hd))
        k /= np.sqrt((k * k).mean(-1, keepdims=True))
        v = self.rng.standard_normal((n, self.nkv, self.hd))
        return (k * scale).astype(np.float16).reshape(n, -1), (v * scale).astype(np.float16).reshape(n, -1)

    def append(self, counts, rows=None, max_nt=None):
        """Appends rows to every sequence in one call; returns (start, length before) for the attention."""
        n = sum(counts)
        k, v = self.rows(n) if rows is None else rows
        start, length = self.batch(counts)
        ops.kv8_append(self.cache, torch.from_numpy(k).to(self.dev), torch.from_numpy(v).to(self.dev), start, length, self.table,
                       max_nt or max(counts))
        at = 0
        for s, c in zip(self.seqs, counts):
            s.append(k[at:at + c], v[at:at + c])
            at += c
        return start, length

    def check_buffers(self):
        """Every full page's codes and scales, bit by bit, and the open rows."""
        kp, vp, sc, tk, tv = (host(t) for t in self.cache)
        ke, ve = ref.k_elem(self.hd), ref.v_elem(self.hd)
        for i, s in enumerate(self.seqs):
            for p in range(s.rows // 64):
                k, v, scales = s.page(p)
                id = self.table_np[i, p]
                assert np.array_equal(sc[id].astype(np.float64), scales), (i, p)
                assert np.array_equal(kp[id], k) and np.array_equal(vp[id], v), (i, p)
            p = s.rows // 64
            for r in range(p * 64, s.rows):
                for h in range(self.nkv):
                    assert np.array_equal(tk[i, p & 1, h][ke[r % 64]], s.k[r, h]), (i, r, h)
                    assert np.array_equal(tv[i, p & 1, h][ve[r % 64]], s.v[r, h]), (i, r, h)

    def attend(self, q, start, length, counts, nh, scale=None, f16=False, max_nt=None, **kw):
        """Runs the attention of the tokens of the last append and checks every output; returns it."""
        n = sum(counts)
        out = torch.full((n + 3, nh * self.hd), 7.0, device=self.dev, dtype=torch.float16 if f16 else torch.float32)
        qd = dev_f32(q.reshape(n, -1), self.dev)
        ops.attn_kv8(self.cache, qd, start, length, self.table, nh, max_nt or max(counts), scale=scale, out=out[:n], **kw)
        got = host(out).astype(np.float64)
        assert (got[n:] == 7.0).all()
        sc, at = 1 / self.hd ** 0.5 if scale is None else scale, 0
        for s, c in zip(self.seqs, counts):
            if c:
                k, v = s.values()
                want, tol = ref.attention(q[at:at + c], k, v, s.rows - c, sc, f16)
                err = np.abs(got[at:at + c].reshape(want.shape) - want)
                assert (err <= tol).all(), (c, s.rows, float(np.nanmax(err - tol)), float(np.nanmax(err)))
                assert np.isfinite(err).all()
            at += c
        return got[:n]

    def queries(self, n, nh, scale=1.0):
        return (self.rng.standard_normal((n, nh, 2 * self.hd)) * scale).astype(np.float32)


@pytest.mark.parametrize("nkv,hd", [(2, 256), (1, 128), (3, 128)])
def test_append_codes_and_open_rows(dev, nkv, hd):
    """Any split of the rows over calls leaves the same codes, scales and open rows."""
    announce(f"kv8 append {nkv} {hd}")
    e = Engine(dev, 3, nkv, hd, 9)
    for counts in ([1, 0, 63], [62, 64, 1], [1, 1, 1], [2, 128, 0], [65, 7, 200], [0, 56, 127], [130, 1, 57]):
        e.append(counts)
        e.check_buffers()
    one = Engine(dev, 3, nkv, hd, 9)
    at = [np.concatenate([x.reshape(len(x), -1) for x in (getattr(s, name) for s in e.seqs)]) for name in ("k", "v")]
    one.append([s.rows for s in e.seqs], rows=at)
    one.check_buffers()


def test_append_token_by_token(dev):
    e = Engine(dev, 2, 2, 256, 4)
    for t in range(131):
        e.append([1, t % 2])
    e.check_buffers()


def test_append_special_values(dev):
    """Zeros, the smallest and the largest f16, infinities, NaN, and quotients that are ties."""
    e = Engine(dev, 1, 2, 256, 8)
    k, v = e.rows(448)
    for x in (k, v):
        x[:16] = 0
        x[16:32] = np.float16(6e-8)
        x[17, ::2] = np.float16(-6e-8)
        x[32:48] *= np.float16(1e-6)
        x[48:64] *= np.float16(3e-5)
        x[64:80] = np.float16(65504)
        x[65, ::3] = np.float16(-65504)
        x[66, ::3] = np.float16(288)          # half a step of 576: to even
        x[67, ::3] = np.float16(864)
        x[80:96, 5] = np.float16(np.inf)
        x[97, 9] = np.float16(-np.inf)
        x[112:128, ::7] = np.float16(np.nan)
        x[128:144] = np.arange(-127, 129, dtype=np.float16)[None, :].repeat(2, 0).reshape(1, -1)[:, :512] / 2
        x[128, 0] = 127                       # scale 1: halves are ties
        x[144:160] *= np.float16(500)
        x[160:176] *= np.float16(15000)
        x[440, 3] = np.float16(np.nan)        # an open row
        x[441, 4] = np.float16(-np.inf)
    e.append([448 - 5], rows=(k[:443], v[:443]))
    e.check_buffers()
    e.append([5], rows=(k[443:], v[443:]))
    e.check_buffers()


def test_rows_taken_back(dev):
    """Drafts that cross a page's end are taken back by a smaller length alone; the page is quantised again."""
    e = Engine(dev, 2, 2, 256, 6)
    e.append([62, 120])
    for keep, n in ((1, 4), (3, 4), (0, 8), (1, 64), (2, 3), (1, 60)):
        before = [s.rows for s in e.seqs]
        counts = [n, n]
        start, length = e.append(counts)
        e.check_buffers()
        q = e.queries(2 * n, 4)
        e.attend(q, start, length, counts, 4)
        for s, b in zip(e.seqs, before):
            s.cut(b + keep)
    e.append([5, 6])
    e.check_buffers()


@pytest.mark.parametrize("nkv,hd", [(2, 256), (3, 128)])
def test_read(dev, nkv, hd):
    """Any range of rows comes back as the values the cache holds; rows of no sequence and rows past a sequence's end stay."""
    e = Engine(dev, 4, nkv, hd, 6)
    e.append([200, 64, 0, 301])
    first, counts = [3, 0, 0, 250], [197, 64, 0, 60]      # (the last range is nine rows too long)
    start = e.ints(np.concatenate([[0], np.cumsum(counts)]).tolist())
    total = e.ints([s.rows for s in e.seqs])
    out = tuple(torch.full((330, nkv * hd), 9.0, device=dev, dtype=torch.float16) for _ in range(2))
    ops.kv8_read(e.cache, start, e.ints(first), total, e.table, 197, 330, out)
    for got, i in zip(out, range(2)):
        got, at = host(got), 0
        for s, f, c in zip(e.seqs, first, counts):
            want = s.values()[i].reshape(s.rows, nkv * hd)[f:f + c]
            assert np.array_equal(got[at:at + len(want)].astype(np.float64), want)
            assert (got[at + len(want):at + c] == 9.0).all()
            at += c
        assert (got[at:] == 9.0).all()
    k, v = ops.kv8_read(e.cache, start, e.ints(first), total, e.table, 5, 330)     # at most five rows a sequence
    assert np.array_equal(host(k)[:5].astype(np.float64), e.seqs[0].values()[0].reshape(200, -1)[3:8])
    wide = torch.zeros(330, 2 * nkv * hd + 16, device=dev, dtype=torch.float16)    # rows inside wider ones
    kv = wide[:, :nkv * hd], wide[:, nkv * hd + 16:]
    ops.kv8_read(e.cache, start, e.ints(first), total, e.table, 197, 330, kv)
    assert torch.equal(kv[0][:300], out[0][:300]) and torch.equal(kv[1][:300], out[1][:300])
    assert (wide[:, nkv * hd:nkv * hd + 16] == 0).all()


@pytest.mark.parametrize("nkv,hd", [(2, 256), (3, 128)])
def test_copy_forks_and_moves(dev, nkv, hd):
    """A fork reads its source's rows and goes on alone; pages moved elsewhere read the same under the new names."""
    e = Engine(dev, 3, nkv, hd, 6, spare=8)
    e.append([150, 0, 77])
    e.table_np[1, :2] = e.table_np[0, :2]                  # the full pages are shared
    e.table.copy_(torch.from_numpy(e.table_np))
    ops.kv8_copy(e.cache, seq_src=e.ints([0, 9, 2]), seq_dst=e.ints([1, 2, -1]))   # (no sequence 9, none -1)
    e.seqs[1].append(e.seqs[0].k, e.seqs[0].v)
    start, length = e.append([3, 60, 1])
    e.check_buffers()
    e.attend(e.queries(64, 2 * nkv), start, length, [3, 60, 1], 2 * nkv)
    used = set(e.table_np.reshape(-1).tolist())
    free = [p for p in range(e.cache.kp.shape[0]) if p not in used]
    src, dst = e.table_np[[0, 2, 1], [1, 0, 2]].tolist(), free[:3]
    others = [p for p in range(e.cache.kp.shape[0]) if p not in dst]
    before = [host(t)[others] for t in e.cache[:3]]
    ops.kv8_copy(e.cache, e.ints(src + [10 ** 6, src[0]]), e.ints(dst + [free[4], -5]))   # (neither is a page: skipped)
    for t, b in zip(e.cache[:3], before):
        assert np.array_equal(host(t)[others], b, equal_nan=t.dtype == torch.float16)
    for a, b in zip(src, dst):
        e.table_np[e.table_np == a] = b
    e.table.copy_(torch.from_numpy(e.table_np))
    e.check_buffers()
    ops.kv8_copy(e.cache)                                  # nothing to do


@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 256), (24, 4, 256), (8, 8, 128), (7, 1, 256), (32, 2, 128), (34, 1, 128)])
@pytest.mark.parametrize("f16", [False, True])
def test_attention_geometries(dev, nh, nkv, hd, f16):
    announce(f"kv8 attn {nh}/{nkv} {hd} f16={f16}")
    e = Engine(dev, 4, nkv, hd, 8)
    for counts in ([100, 64, 1, 0], [1, 1, 0, 1], [3, 4, 5, 1], [17, 2, 90, 128], [1, 1, 1, 1]):
        start, length = e.append(counts)
        e.attend(e.queries(sum(counts), nh), start, length, counts, nh, f16=f16)


@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 256), (24, 4, 256), (8, 8, 128), (7, 1, 256), (32, 2, 128), (34, 1, 128)])
@pytest.mark.parametrize("f16", [False, True])
def test_geometries_over_wide_tables(dev, nh, nkv, hd, f16):
    """Tables that could name long contexts call for row blocks of more rows."""
    announce(f"kv8 wide {nh}/{nkv} {hd} f16={f16}")
    e = Engine(dev, 4, nkv, hd, 8, wide=600)
    for counts in ([100, 64, 1, 0], [3, 4, 5, 1], [17, 2, 90, 128], [2, 1, 2, 3], [8, 8, 8, 8]):
        start, length = e.append(counts)
        e.attend(e.queries(sum(counts), nh), start, length, counts, nh, f16=f16)


@pytest.mark.parametrize("before,n", [(0, 2), (63, 4), (64, 3), (4103, 4), (9000, 8), (200, 8)])
def test_lengths_over_wide_tables(dev, before, n):
    e = Engine(dev, 1, 2, 256, before // 64 + 2, wide=600)
    if before:
        e.append([before])
    start, length = e.append([n])
    for f16 in (False, True):
        e.attend(e.queries(n, 16), start, length, [n], 16, f16=f16)


@pytest.mark.parametrize("before", [0, 1, 15, 62, 63, 64, 65, 127, 128, 191, 319, 640])
@pytest.mark.parametrize("n", [1, 2, 5, 66])
def test_attention_lengths(dev, before, n):
    e = Engine(dev, 1, 2, 256, 12)
    if before:
        e.append([before])
    start, length = e.append([n])
    e.attend(e.queries(n, 16), start, length, [n], 16, f16=before % 2 == 1)


@pytest.mark.parametrize("before,n,nh,nkv,hd", [(8190, 1, 16, 2, 256), (20000, 1, 4, 2, 128), (4103, 4, 24, 4, 256), (5000, 33, 2, 1, 128),
                                                (64 * 129, 1, 8, 1, 128)])
def test_long_contexts(dev, before, n, nh, nkv, hd):
    """More pages than are looked up at once, and many splits."""
    e = Engine(dev, 1, nkv, hd, before // 64 + 2)
    e.append([before])
    start, length = e.append([n])
    e.attend(e.queries(n, nh), start, length, [n], nh)


def test_one_split_of_many_pages(dev):
    """Enough sequences that each is one split, of more pages than are looked up at once."""
    nseq, nkv, hd = 70, 4, 128
    e = Engine(dev, nseq, nkv, hd, 72)
    lens = [4300 if i % 23 == 0 else (i * 37) % 300 for i in range(nseq)]
    e.append(lens)
    counts = [0 if i == 11 else 1 for i in range(nseq)]
    start, length = e.append(counts)
    e.attend(e.queries(sum(counts), 8), start, length, counts, 8)
    counts = [40 if i % 23 == 0 else 0 for i in range(nseq)]
    start, length = e.append(counts)
    e.attend(e.queries(sum(counts), 8), start, length, counts, 8, f16=True)


@pytest.mark.parametrize("alike", [True, False])
def test_many_sequences_of_many_pages(dev, alike):
    """A batch past one wave's 64 sequences, whose splits are chosen by counting them."""
    nseq, nkv, hd = 68, 2, 128
    e = Engine(dev, nseq, nkv, hd, 48)
    lens = [2900 if alike else 2000 + (i * 379) % 1000 for i in range(nseq)]
    e.append(lens)
    counts = [0 if i in (5, 64) else 1 + i % 2 for i in range(nseq)]
    start, length = e.append(counts)
    for f16 in (False, True):
        e.attend(e.queries(sum(counts), 16), start, length, counts, 16, f16=f16)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("f16", [False, True])
def test_forms_over_many_pages_of_one_split(dev, hd, f16):
    """Every number of row blocks over more than twice 64 pages in one workgroup: 130 sequences that share a beginning."""
    nseq, nkv, before = 130, 2, 64 * 131 + 3
    e = Engine(dev, nseq, nkv, hd, 2, spare=140)
    base = np.random.default_rng(2).permutation(140)[:132].astype(np.int32)
    e.table_np = np.repeat(base[None], nseq, 0)
    e.table = torch.from_numpy(e.table_np.copy()).to(dev)
    k, v = e.rows(before)
    for p in (64, 128):                              # the first pages of the second and third 64: a third of the weight
        k.reshape(before, nkv, hd)[64 * p:64 * p + 64] = np.float16(1)
    e.append([before] + [0] * (nseq - 1), rows=(k, v))
    ops.kv8_copy(e.cache, seq_src=e.ints([0] * (nseq - 1)), seq_dst=e.ints(list(range(1, nseq))))
    for s in e.seqs[1:]:
        s.k, s.v = e.seqs[0].k, e.seqs[0].v
    for n in (1, 4, 5, 8):                           # 8, 32, 40 and 64 rows; no page gets full
        start, length = e.append([n] * nseq)
        q = e.queries(n * nseq, 16)
        q[:, :, :hd] += np.float32(4 / hd ** 0.5)
        out = torch.empty(n * nseq, 16 * hd, device=dev, dtype=torch.float16 if f16 else torch.float32)
        got = host(ops.attn_kv8(e.cache, dev_f32(q.reshape(n * nseq, -1), dev), start, length, e.table, 16, n, out=out))
        for i in (0, 101):
            want, tol = ref.attention(q[i * n:i * n + n], *e.seqs[i].values(), e.seqs[i].rows - n, 1 / hd ** 0.5, f16)
            err = np.abs(got[i * n:i * n + n].reshape(want.shape).astype(np.float64) - want)
            assert (err <= tol).all(), (n, i, float((err - tol).max()))


def test_whole_prompts(dev):
    """Prompts long enough that no row block is split."""
    for f16 in (False, True):
        e = Engine(dev, 2, 4, 128, 20)
        counts = [1100, 203]
        start, length = e.append(counts)
        e.attend(e.queries(sum(counts), 32), start, length, counts, 32, f16=f16)


@pytest.mark.parametrize("before,counts,nh,nkv,hd,f16", [
    ([9000, 700, 200, 130], [20, 20, 20, 20], 16, 2, 256, False),       # one of many splits, others of few and of one
    ([9000, 700, 200, 130], [20, 20, 20, 20], 8, 1, 128, False),
    ([61 + 37 * i for i in range(16)], [5] * 16, 16, 2, 256, False),    # 40 rows each, many sequences
    ([61 + 37 * i for i in range(16)], [5] * 16, 8, 1, 128, True),
    ([0, 300], [600, 200], 128, 16, 128, False),                        # enough row blocks for the largest of each type
    ([0, 300, 63, 0, 128], [1, 203, 97, 0, 5], 24, 4, 256, True),
    ([1000, 0, 63], [129, 64, 65], 16, 2, 256, True),
    ([37 * i for i in range(9)], [16] * 9, 24, 4, 256, True),           # full batches: 96 rows in two blocks of 48, 128 in two of 64
    ([37 * i for i in range(9)], [16] * 9, 32, 4, 256, True),
    ([37 * i for i in range(17)], [8] * 17, 64, 8, 128, True),
])
def test_forms(dev, before, counts, nh, nkv, hd, f16):
    """Batches whose sizes call for each number of row blocks and each way of joining splits."""
    announce(f"kv8 forms {len(counts)} {sum(counts)} {nh}/{nkv} {hd} f16={f16}")
    e = Engine(dev, len(counts), nkv, hd, max(b + c for b, c in zip(before, counts)) // 64 + 1)
    e.append(before)
    start, length = e.append(counts)
    e.attend(e.queries(sum(counts), nh), start, length, counts, nh, f16=f16)


@pytest.mark.parametrize("before,n", [(60, 10), (0, 70), (128, 3), (190, 4), (1000, 90), (0, 1)])
@pytest.mark.parametrize("nh", [2, 16, 64])
def test_scores_far_below_zero(dev, before, n, nh):
    """Every score is some -150 in log2 units, so that weights under no reference would vanish: also for the rows of a block that
    see none of the open page, which comes first, and where the full pages' scores are far above the open page's."""
    e = Engine(dev, 1, 2, 256, 20)
    base = np.random.default_rng(11).standard_normal(512)
    base /= np.sqrt((base * base).mean())
    k, v = e.rows(before + n)
    low = 1.0 if nh > 2 else 2.0 - (np.arange(before + n) < (before + n) // 64 * 64)[:, None]     # (twice as low in the open page)
    k = (k.astype(np.float32) * 0.1 - base * low).astype(np.float16)
    if before:
        e.append([before], rows=(k[:before], v[:before]))
    start, length = e.append([n], rows=(k[before:], v[before:]))
    q = e.queries(n, nh)
    for h in range(nh):
        q[:, h, :256] = q[:, h, :256] * 0.1 + 6.5 * base[:256] * (1 if h < nh // 2 else 0) + 6.5 * base[256:] * (0 if h < nh // 2 else 1)
    for f16 in (False, True):
        e.attend(q, start, length, [n], nh, f16=f16)


@pytest.mark.parametrize("nkv,hd", [(4, 128), (2, 256)])
def test_full_pages_far_above_the_open_page(dev, nkv, hd):
    """Enough sequences that a workgroup has the open page and full ones; rows that see both, whose reference is raised between
    them, beside rows that see the full pages alone."""
    nseq, G = 48, 8
    e = Engine(dev, nseq, nkv, hd, 4)
    base = np.random.default_rng(13).standard_normal(hd)
    base /= np.sqrt((base * base).mean())
    def append(counts):
        k, v = e.rows(sum(counts))
        rows = np.concatenate([s.rows + np.arange(c) for s, c in zip(e.seqs, counts)])
        last = np.concatenate([np.full(c, (s.rows + c) // 64 * 64 if s.rows else 128) for s, c in zip(e.seqs, counts)])
        low = np.where(rows < last, 0.5, 2.0)[:, None, None]
        k = (k.reshape(-1, nkv, hd).astype(np.float32) * 0.2 - base * low).astype(np.float16).reshape(len(k), -1)
        return e.append(counts, rows=(k, v))
    append([40 + i % 31 if i % 2 else 100 + i for i in range(nseq)])
    counts = [30 + i % 7 for i in range(nseq)]
    start, length = append(counts)
    q = e.queries(sum(counts), nkv * G)
    q[:, :, :hd] = q[:, :, :hd] * 0.1 + 1.5 * base
    for f16 in (False, True):
        e.attend(q, start, length, counts, nkv * G, f16=f16)


def test_a_pool_past_32_bits(dev):
    """Pages whose bytes lie past 2^32 in a pool, through every call."""
    nkv, hd, far = 8, 256, 36000                     # 128 KiB a page: 4.7e9 bytes of K and of V
    e = Engine(dev, 2, nkv, hd, 6, spare=far)
    order = np.random.default_rng(1).permutation(12)
    e.table_np = (far + order).reshape(2, 6).astype(np.int32)
    e.table_np[0, 1] = 3
    e.table.copy_(torch.from_numpy(e.table_np))
    e.append([200, 130])
    start, length = e.append([3, 70])
    e.attend(e.queries(73, 16), start, length, [3, 70], 16)
    def check():
        k, v = ops.kv8_read(e.cache, e.ints([0, 203, 403]), e.ints([0, 0]), e.ints([203, 200]), e.table, 203, 403)
        at = 0
        for s in e.seqs:
            wk, wv = (x.reshape(len(x), -1).astype(np.float16) for x in s.values())
            assert np.array_equal(host(k[at:at + s.rows]), wk) and np.array_equal(host(v[at:at + s.rows]), wv)
            at += s.rows
    check()
    ops.kv8_copy(e.cache, src=e.ints([int(e.table_np[0, 1]), int(e.table_np[1, 0])]), dst=e.ints([far - 1, 5]))
    e.table_np[0, 1], e.table_np[1, 0] = far - 1, 5
    e.table.copy_(torch.from_numpy(e.table_np))
    check()


@pytest.mark.parametrize("f16", [False, True])
def test_idle_slots_and_padding(dev, f16):
    """A captured engine's shapes: more slots than sequences, token arrays longer than the batch, a bound above what comes."""
    e = Engine(dev, 70, 2, 256, 40)
    lens = [0] * 70
    lens[3], lens[68] = 2300, 77
    e.append(lens)
    counts = [0] * 70
    counts[3], counts[68] = 5, 1
    k, v = e.rows(6)
    pad = np.full((34, 512), np.nan, np.float16)
    start, length = e.batch(counts)
    ops.kv8_append(e.cache, *(torch.from_numpy(np.concatenate([x, pad])).to(dev) for x in (k, v)), start, length, e.table, 8)
    e.seqs[3].append(k[:5], v[:5])
    e.seqs[68].append(k[5:], v[5:])
    e.check_buffers()
    q = e.queries(40, 16)
    q[6:] = np.nan
    out = torch.full((40, 4096), 7.0, device=dev, dtype=torch.float16 if f16 else torch.float32)
    ops.attn_kv8(e.cache, dev_f32(q.reshape(40, -1), dev), start, length, e.table, 16, 8, out=out)
    assert (host(out)[6:] == 7.0).all()
    for i, at, n in ((3, 0, 5), (68, 5, 1)):
        want, tol = ref.attention(q[at:at + n], *e.seqs[i].values(), e.seqs[i].rows - n, 1 / 16, f16)
        assert (np.abs(host(out)[at:at + n].reshape(want.shape) - want) <= tol).all()


def test_sharp_flat_and_odd_scores(dev):
    """One key takes nearly all the weight, in the last or the first page; all keys the same; scales of any sign and size."""
    for kscale, qscale, scale in ((20.0, 1.0, None), (0.0, 1.0, None), (1.0, 1.0, -0.07), (1.0, 1e-30, None), (1.0, 1e4, 1e-5),
                                  (1.0, 1.0, 0.0), (1e-3, 1.0, 50.0)):
        e = Engine(dev, 1, 2, 256, 12)
        k, v = e.rows(500)
        k = (k.astype(np.float32) * kscale).astype(np.float16)
        start, length = None, None
        e.append([495], rows=(k[:495], v[:495]))
        start, length = e.append([5], rows=(k[495:], v[495:]))
        for f16 in (False, True):
            e.attend(e.queries(5, 16, qscale), start, length, [5], 16, scale=scale, f16=f16)


def test_a_late_large_score_and_a_lost_one(dev):
    """The reference is raised at every page (each page's keys larger), and a zero query row."""
    e = Engine(dev, 1, 2, 256, 24)
    k, v = e.rows(1400)
    ramp = np.linspace(0.0, 30.0, 1400)[:, None].astype(np.float32)
    base = np.random.default_rng(5).standard_normal(512).astype(np.float32)
    k = (k.astype(np.float32) * 0.1 + ramp * base / 16).astype(np.float16)
    e.append([1390], rows=(k[:1390], v[:1390]))
    start, length = e.append([10], rows=(k[1390:], v[1390:]))
    q = e.queries(10, 16)
    q[:, 0, :256] = base[:256]
    q[:, 1, :256] = -base[:256]
    q[3] = 0
    for f16 in (False, True):
        e.attend(q, start, length, [10], 16, f16=f16)


def test_small_and_large_values(dev):
    """Rows near the smallest normal f16 and rows near the largest."""
    for scale in (1e-4, 3000.0):
        e = Engine(dev, 1, 2, 256, 6)
        k, v = e.rows(200)
        v = (v.astype(np.float32) * scale).astype(np.float16)
        start, length = e.append([200], rows=(k, v))
        for f16 in (False, True):
            if scale > 1 or not f16:
                e.attend(e.queries(200, 16), start, length, [200], 16, f16=f16)


def test_rows_that_are_not_seen_do_not_matter(dev):
    """Infinities and NaN in the buffers behind a sequence's rows, in pages of others and in later tokens' rows (which the
    cache holds as finite values) leave an output bit by bit as it is; so do the other sequences of a call."""
    def run(poison, alone):
        e = Engine(dev, 2, 2, 256, 6, seed=3)
        e.append([70, 100])
        counts = [30, 0 if alone else 40]
        k, v = e.rows(70)
        k, v = k[:sum(counts)].copy(), v[:sum(counts)].copy()
        if poison:
            k[20:30] = np.float16(np.inf)
            v[20:30] = np.float16(np.nan)
        start, length = e.append(counts, rows=(k, v))
        if poison:      # rows at and after the length
            for t, x in ((e.cache.tk, float("nan")), (e.cache.tv, float("inf"))):
                for i, s in enumerate(e.seqs):
                    at = ref.k_elem(256) if t is e.cache.tk else ref.v_elem(256)
                    free = torch.from_numpy(at[s.rows % 64:].reshape(-1)).to(dev)
                    t[i, s.rows // 64 % 2][:, free] = x
        q = np.random.default_rng(9).standard_normal((70, 16, 512)).astype(np.float32)
        out = torch.empty(sum(counts), 16 * 256, device=dev)
        ops.attn_kv8(e.cache, dev_f32(q[:sum(counts)].reshape(sum(counts), -1), dev), start, length, e.table, 16, 40, out=out)
        return host(out)
    base = run(False, False)
    poisoned = run(True, False)
    # rows 70 .. 89 see none of the poisoned rows: their block (rows 80 .. 95) shares its scale with them, so compare those before
    assert np.isfinite(poisoned).all()
    assert np.array_equal(base[30:], poisoned[30:])
    assert np.array_equal(base[:30], run(False, True)[:30])


def test_bad_lengths_and_pages(dev):
    """A sequence whose length cannot be, or whose table cannot name its rows, gives NaN and is not appended to; a page outside
    the pool makes what reads it NaN and is not written; bounds outside the tokens are no tokens. The others are as always."""
    e = Engine(dev, 5, 2, 256, 4)
    e.append([100, 100, 100, 250, 90])
    good = [s.rows for s in e.seqs]
    start, length = e.batch([2, 2, 2, 8, 2])
    length[1] = -3
    table = e.table.clone()
    table[2, 0] = e.cache.kp.shape[0]
    table[4, 1] = -1
    k, v = e.rows(16)
    before = [host(t) for t in e.cache]
    ops.kv8_append(e.cache, torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), start, length, table, 8)
    after = [host(t) for t in e.cache]
    for i in (1, 3):        # 250 + 8 rows are more than four pages
        assert np.array_equal(before[3][i], after[3][i], equal_nan=True)
    e.seqs[0].append(k[:2], v[:2])
    q = np.random.default_rng(9).standard_normal((16, 16, 512)).astype(np.float32)
    for f16 in (torch.float32, torch.float16):
        out = host(ops.attn_kv8(e.cache, dev_f32(q.reshape(16, -1), dev), start, length, table, 16, 8, out_dtype=f16)).astype(np.float64)
        kk, vv = e.seqs[0].values()
        want, tol = ref.attention(q[:2], kk, vv, good[0], 1 / 16, f16 == torch.float16)
        assert (np.abs(out[:2].reshape(want.shape) - want) <= tol).all()
        assert np.isnan(out[2:6]).all() and np.isnan(out[6:14]).all()
        assert np.isfinite(out[14:]).all()              # (page 1 is open: its number is not needed yet)
    start2 = e.ints([0, 2, 2, -1, 99, 3])               # 2, 0, none, none, none
    out = torch.full((16, 16 * 256), 5.0, device=dev)
    length2 = e.ints(good)
    ops.attn_kv8(e.cache, dev_f32(q.reshape(16, -1), dev), start2, length2, e.table, 16, 8, out=out)
    got = host(out)
    assert (np.abs(got[:2].reshape(2, 16, 256) - ref.attention(q[:2], kk, vv, good[0], 1 / 16)[0]) <=
            ref.attention(q[:2], kk, vv, good[0], 1 / 16)[1]).all()
    assert (got[2:] == 5.0).all()


def test_nonfinite_queries_stay_in_their_rows(dev):
    e = Engine(dev, 1, 2, 256, 4)
    start, length = e.append([130])
    q = e.queries(130, 16)
    for f16 in (torch.float32, torch.float16):
        base = host(ops.attn_kv8(e.cache, dev_f32(q.reshape(130, -1), dev), start, length, e.table, 16, 130, out_dtype=f16))
        bad = q.copy()
        bad[7, 3, 5], bad[100, 9, 200], bad[129, 0, 0] = np.nan, np.inf, -np.inf
        got = host(ops.attn_kv8(e.cache, dev_f32(bad.reshape(130, -1), dev), start, length, e.table, 16, 130, out_dtype=f16))
        got, base = got.reshape(130, 16, 256), base.reshape(130, 16, 256)
        for t, h in ((7, 3), (100, 9), (129, 0)):
            assert np.isnan(got[t, h]).all()
            got[t, h] = base[t, h]
        assert np.array_equal(got, base)


def test_max_nt_leaves_later_tokens_out(dev):
    e = Engine(dev, 2, 2, 256, 4)
    k, v = e.rows(20)
    start, length = e.batch([12, 8])
    ops.kv8_append(e.cache, torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), start, length, e.table, 5)
    for s, a in zip(e.seqs, (0, 12)):
        s.append(k[a:a + 5], v[a:a + 5])
    e.check_buffers()
    q = e.queries(20, 16)
    out = torch.full((20, 4096), 3.0, device=dev)
    ops.attn_kv8(e.cache, dev_f32(q.reshape(20, -1), dev), start, length, e.table, 16, 5, out=out)
    got = host(out).reshape(20, 16, 256)
    for s, a in zip(e.seqs, (0, 12)):
        want, tol = ref.attention(q[a:a + 5], *s.values(), 0, 1 / 16)
        assert (np.abs(got[a:a + 5] - want) <= tol).all()
    assert (got[5:12] == 3.0).all() and (got[17:] == 3.0).all()


def test_strides_through_the_c_abi(dev):
    """Token strides of q, out, k and v wider than a row, through the C ABI."""
    e = Engine(dev, 1, 2, 256, 4)
    k, v = e.rows(90)
    kw = torch.full((90, 1040), 99.0, device=dev, dtype=torch.float16)
    kw[:, :512], kw[:, 528:] = torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev)
    start, length = e.batch([90])
    ops.kv8_append(e.cache, kw[:, :512], kw[:, 528:], start, length, e.table, 90)
    e.seqs[0].append(k, v)
    e.check_buffers()
    q = e.queries(90, 4)
    qw = torch.full((90, 4 * 512 + 12), float("nan"), device=dev)
    qw[:, :4 * 512] = dev_f32(q.reshape(90, -1), dev)
    out = torch.full((90, 1024 + 8), 4.0, device=dev)
    args = ops._kv8(e.cache)[-1]
    scratch = torch.empty(ops.attn_kv8_scratch_bytes(90, 4, 2), dtype=torch.uint8, device=dev)
    import ctypes
    _lib.call("it_attn_kv8", ctypes.addressof(args), qw.data_ptr(), qw.shape[1], 90, start.data_ptr(), length.data_ptr(),
              e.table.data_ptr(), 4, 90, 4, 1 / 16, out.data_ptr(), out.shape[1], 0, scratch.data_ptr(), scratch.numel(),
              torch.cuda.current_stream().cuda_stream)
    got = host(out)
    want, tol = ref.attention(q, *e.seqs[0].values(), 0, 1 / 16)
    assert (np.abs(got[:, :1024].reshape(want.shape) - want) <= tol).all()
    assert (got[:, 1024:] == 4.0).all()


@pytest.mark.parametrize("before,counts,nh,nkv,hd,f16", [
    ([8200], [1], 16, 2, 256, False), ([3, 0, 4000], [3, 4, 2], 24, 4, 256, False), ([500, 2100], [60, 9], 16, 2, 256, False),
    ([700], [300], 16, 2, 256, True), ([300] * 40, [5] * 40, 8, 1, 128, True), ([9000], [16], 8, 1, 128, False)])
def test_scratch_and_cache_bands(dev, before, counts, nh, nkv, hd, f16):
    """Scratch of exactly the bytes asked for, and a cache whose buffers are exactly as long as its sizes say, between bands of a
    sentinel byte: nothing is written outside them."""
    announce(f"kv8 bands {sum(counts)} {nh}/{nkv} {hd} f16={f16}")
    e = Engine(dev, len(counts), nkv, hd, max(b + c for b, c in zip(before, counts)) // 64 + 1, spare=0)
    held = [banded(t.nbytes, dev) for t in e.cache]
    e.cache = ops.Kv8Cache(*(view.view(t.dtype).view(t.shape) for (_, view), t in zip(held, e.cache)))
    for t in e.cache[2:]:
        t.fill_(float("nan"))
    e.append(before)
    start, length = e.append(counts)
    n = ops.attn_kv8_scratch_bytes(max(counts), nh, nkv, hd)
    buf, scratch = banded(n, dev)
    e.attend(e.queries(sum(counts), nh), start, length, counts, nh, f16=f16, scratch=scratch)
    assert_bands(buf, n)
    ops.kv8_copy(e.cache, e.ints([0]), e.ints([int(e.cache.kp.shape[0]) - 1]), e.ints([0]), e.ints([len(counts) - 1]))
    for (whole, _), t in zip(held, e.cache):
        assert_bands(whole, t.nbytes)


def test_the_same_call_gives_the_same_bits(dev):
    e = Engine(dev, 3, 4, 256, 20)
    e.append([900, 33, 600])
    counts = [4, 1, 3]
    start, length = e.append(counts)
    q = dev_f32(e.queries(8, 24).reshape(8, -1), dev)
    a = ops.attn_kv8(e.cache, q, start, length, e.table, 24, 4)
    for _ in range(4):
        assert torch.equal(a, ops.attn_kv8(e.cache, q, start, length, e.table, 24, 4))


def test_steps_captured_and_side_by_side(dev):
    """Whole steps (pre-pass, append, attention, length) captured once and replayed as the lengths advance over pages, on two
    streams at once with a graph each, against the same steps run eagerly."""
    nh, nkv, hd, steps = 16, 2, 256, 70
    freq, _ = ops.rope_freqs(64, device=dev)

    class Step:
        def __init__(self, seed):
            self.e = Engine(dev, 2, nkv, hd, 6, seed=seed)
            self.e.append([60, 100])
            g = torch.Generator(device=dev).manual_seed(seed)
            self.q0 = torch.randn(steps, 2, nh * 2 * hd, device=dev, generator=g)
            self.k0, self.v0 = (torch.randn(steps, 2, nkv * hd, device=dev, generator=g) for _ in range(2))
            self.q, self.k, self.v = self.q0[0].clone(), self.k0[0].clone(), self.v0[0].clone()
            self.length = torch.tensor([60, 100], dtype=torch.int32, device=dev)
            self.start = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
            self.kr, self.vr = (torch.empty(2, nkv * hd, dtype=torch.float16, device=dev) for _ in range(2))
            self.out = torch.empty(2, nh * hd, device=dev)
            self.scratch = torch.empty(ops.attn_kv8_scratch_bytes(1, nh, nkv), dtype=torch.uint8, device=dev)

        def feed(self, i):
            self.q.copy_(self.q0[i]); self.k.copy_(self.k0[i]); self.v.copy_(self.v0[i])

        def run(self):
            ops.attn_prep_pos_f16(self.q, self.k, self.v, self.kr, self.vr, self.length, 0, nh, nkv, freq)
            ops.kv8_append(self.e.cache, self.kr, self.vr, self.start, self.length, self.e.table, 1)
            ops.attn_kv8(self.e.cache, self.q, self.start, self.length, self.e.table, nh, 1, out=self.out, scratch=self.scratch)
            self.length.add_(1)

    want = []
    for seed in (1, 2):
        s = Step(seed)
        outs = []
        for i in range(steps):
            s.feed(i)
            s.run()
            outs.append(s.out.clone())
        want.append(outs)
    both = []
    for seed in (1, 2):
        s = Step(seed)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            s.run()
        both.append((s, st, graph))
    torch.cuda.synchronize()
    for i in range(steps):
        for s, st, graph in both:
            with torch.cuda.stream(st):
                s.feed(i)
                graph.replay()
        if i % 7 == 0:
            torch.cuda.synchronize()
        for (s, st, _), outs in zip(both, want):
            st.synchronize()
            assert torch.equal(s.out, outs[i]), i


def test_agrees_with_the_f16_cache(dev):
    """Rows read back into an f16 cache give it_attn_f16 the same keys and values: the two attentions agree to f16."""
    e = Engine(dev, 1, 2, 256, 20)
    e.append([1000])
    start, length = e.append([1])
    q = dev_f32(e.queries(1, 16).reshape(1, -1), dev)
    out = ops.attn_kv8(e.cache, q, start, length, e.table, 16, 1)
    k, v = ops.kv8_read(e.cache, e.ints([0, 1001]), e.ints([0]), e.ints([1001]), e.table, 1001, 1001)
    assert (ops.attn_f16(q, k, v, 1000, 16, 2) - out).abs().max() <= 2e-3


def test_reading_and_appending_anew_cuts_inside_a_page(dev):
    """A sequence cut back further than the open rows reach: the rest of its last page is read and appended anew."""
    e = Engine(dev, 1, 2, 256, 6)
    e.append([330])
    k, v = ops.kv8_read(e.cache, e.ints([0, 20]), e.ints([128]), e.ints([330]), e.table, 20, 20)
    vals = [x[128:148].astype(np.float16).reshape(20, -1) for x in e.seqs[0].values()]
    assert np.array_equal(host(k), vals[0]) and np.array_equal(host(v), vals[1])
    e.seqs[0].cut(128)
    e.append([20], rows=(host(k), host(v)))
    start, length = e.append([3])
    e.check_buffers()
    e.attend(e.queries(3, 16), start, length, [3], 16)


def test_front_end_refusals(dev):
    c = ops.kv8_cache(4, 2, 2, 256, dev)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    start, length, table = i(0, 1, 2), i(0, 0), torch.zeros(2, 2, dtype=torch.int32, device=dev)
    q, k = torch.zeros(2, 2048, device=dev), torch.zeros(2, 512, dtype=torch.float16, device=dev)
    ok = dict(start=start, length=length, table=table)
    for bad in (dict(start=i(0, 2)), dict(length=i(0)), dict(table=i(0, 0)), dict(start=start.long()), dict(table=table[:, :1].t()),
                dict(length=length.cpu())):
        a = dict(ok, **bad)
        with pytest.raises(ValueError):
            ops.kv8_append(c, k, k, a["start"], a["length"], a["table"], 1)
        with pytest.raises(ValueError):
            ops.attn_kv8(c, q, a["start"], a["length"], a["table"], 4, 1)
        with pytest.raises(ValueError):
            ops.kv8_read(c, a["start"], length, a["length"], a["table"], 1, 2)
    for kk, vv in ((k.float(), k), (k[:, :256], k), (k.t(), k.t()), (k, k[:1]), (k.cpu(), k)):
        with pytest.raises(ValueError):
            ops.kv8_append(c, kk, vv, start, length, table, 1)
    with pytest.raises(ValueError):
        ops.kv8_append(c._replace(vp=c.vp[:2]), k, k, start, length, table, 1)
    with pytest.raises(ValueError):
        ops.kv8_append(c._replace(sc=c.sc.float()), k, k, start, length, table, 1)
    for kw in (dict(out=torch.zeros(2, 1024, device=dev, dtype=torch.float64)), dict(out=torch.zeros(3, 1024, device=dev)),
               dict(scratch=torch.zeros(64, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            ops.attn_kv8(c, q, start, length, table, 4, 1, **kw)
    with pytest.raises(ValueError):
        ops.attn_kv8(c, q[:, :1024], start, length, table, 4, 1)
    with pytest.raises(_lib.ItError, match="scratch"):
        ops.attn_kv8(c, q, start, length, table, 4, 1, scratch=torch.zeros(64, dtype=torch.uint8, device=dev))
    for a in ((i(0), i(0, 1)), (i(0), None)):
        with pytest.raises(ValueError):
            ops.kv8_copy(c, *a)
    with pytest.raises(_lib.ItError, match="page copies"):
        ops.kv8_copy(c, i(0, 1, 2, 3, 0), i(1, 2, 3, 0, 1))
