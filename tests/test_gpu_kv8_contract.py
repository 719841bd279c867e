"""What the 8-bit cache's calls promise at the edge of their contract."""
import numpy as np
import pytest
import torch

from irontimber_amd import ops
from tests.gpu_util import announce, dev_f32, host
from tests.test_gpu_kv8 import Engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("before,n,nh,nkv,hd,page", [
    (50, 90, 16, 2, 256, 1), (60, 6, 16, 2, 256, 1), (62, 68, 4, 2, 128, 1), (120, 300, 16, 2, 256, 3), (4080, 100, 16, 2, 256, 64),
    (0, 700, 24, 4, 256, 6), (4090, 8, 8, 1, 128, 64)])
@pytest.mark.parametrize("f16", [torch.float32, torch.float16])
def test_an_unknown_page_is_lost_to_what_reads_it_alone(dev, before, n, nh, nkv, hd, page, f16):
    """A full page whose number is outside the pool: tokens before it, that share a block of rows with later ones, keep their
    outputs bit by bit; those that see it are NaN."""
    announce(f"kv8 unknown page {page} after {before} + {n} {nh}/{nkv} {hd}")
    for bad in (-1, 10 ** 6):
        e = Engine(dev, 1, nkv, hd, (before + n) // 64 + 3)
        if before:
            e.append([before])
        start, length = e.append([n + (64 - (before + n) % 64)])          # the page is full for all of these tokens
        m = int(start[1])
        q = dev_f32(e.queries(m, nh).reshape(m, -1), dev)
        run = lambda table: host(ops.attn_kv8(e.cache, q, start, length, table, nh, m, out_dtype=f16))
        good = run(e.table)
        table = e.table.clone()
        table[0, page] = bad
        got = run(table)
        first = max(page * 64 - before, 0)
        assert 0 < first < m and np.isfinite(good).all()
        assert np.array_equal(got[:first], good[:first])
        assert np.isnan(got[first:]).all()


def test_an_unknown_page_beside_an_open_one(dev):
    """Rows that see neither, the unknown page alone, and both."""
    e = Engine(dev, 1, 2, 256, 4)
    e.append([60])
    start, length = e.append([80])                                        # page 1 full, 12 open rows
    q = dev_f32(e.queries(80, 16).reshape(80, -1), dev)
    table = e.table.clone()
    table[0, 1] = -7
    for f16 in (torch.float32, torch.float16):
        good = host(ops.attn_kv8(e.cache, q, start, length, e.table, 16, 80, out_dtype=f16))
        got = host(ops.attn_kv8(e.cache, q, start, length, table, 16, 80, out_dtype=f16))
        assert np.array_equal(got[:4], good[:4]) and np.isnan(got[4:]).all()


def test_reading_rows_that_cannot_be(dev):
    """A sequence with more rows than its table can name, or with a negative length or first row, is read as NaN; a page outside
    the pool too; the others as always, and rows of no sequence stay."""
    e = Engine(dev, 6, 2, 256, 3)
    e.append([100, 150, 70, 80, 192, 130])
    first, counts = [0, 90, 3, -5, 128, 60], [100, 60, 30, 70, 64, 70]
    total = e.ints([100, 193, -1, 80, 192, 130])
    table = e.table.clone()
    table[5, 1] = e.cache.kp.shape[0]
    start = e.ints(np.concatenate([[0], np.cumsum(counts)]).tolist())
    n = sum(counts)
    out = tuple(torch.full((n + 5, 512), 9.0, device=dev, dtype=torch.float16) for _ in range(2))
    ops.kv8_read(e.cache, start, e.ints(first), total, table, max(counts), n + 5, out)
    for i in range(2):
        got, at = host(out[i]), 0
        for j, (s, f, c) in enumerate(zip(e.seqs, first, counts)):
            here = got[at:at + c]
            if j in (1, 2, 3):
                assert np.isnan(here).all(), j
            else:
                want = s.values()[i].reshape(s.rows, 512)[f:f + c].astype(np.float16)
                if j == 5:
                    want[64 - f:128 - f] = np.nan
                assert np.array_equal(here, want, equal_nan=True), j
            at += c
        assert (got[at:] == 9.0).all()
    at = e.ints([0, 0, 50, 50, 50, 50, 50])               # at most 20 of its 50 rows
    out = torch.full((50, 512), 9.0, device=dev, dtype=torch.float16), torch.full((50, 512), 9.0, device=dev, dtype=torch.float16)
    ops.kv8_read(e.cache, at, e.ints(first), total, table, 20, 50, out)
    for x in out:
        assert np.isnan(host(x)[:20]).all() and (host(x)[20:] == 9.0).all()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_a_scale_that_is_no_number(dev, scale):
    e = Engine(dev, 2, 2, 256, 3)
    e.append([70, 0])
    start, length = e.append([3, 30])
    q = dev_f32(e.queries(33, 16).reshape(33, -1), dev)
    for f16 in (torch.float32, torch.float16):
        assert np.isnan(host(ops.attn_kv8(e.cache, q, start, length, e.table, 16, 30, scale=scale, out_dtype=f16))).all()


def test_rows_taken_back_twice(dev):
    """126 rows, four drafts that cross a page's end, three of them taken back: the drafts' page has taken the open rows of the
    page two before it, so a cut into that page reads its rows and appends them anew."""
    e = Engine(dev, 1, 2, 256, 4)
    e.append([126])
    e.append([4])
    e.seqs[0].cut(127)
    e.append([1])
    e.seqs[0].cut(100)                                   # page 1 still stands in the open buffer
    start, length = e.append([2])
    e.check_buffers()
    e.attend(e.queries(2, 16), start, length, [2], 16)
    k, v = ops.kv8_read(e.cache, e.ints([0, 63]), e.ints([0]), e.ints([102]), e.table, 63, 63)
    want = [x[:63].astype(np.float16).reshape(63, -1) for x in e.seqs[0].values()]
    assert np.array_equal(host(k), want[0]) and np.array_equal(host(v), want[1])
    e.seqs[0].cut(0)
    e.append([63], rows=(host(k), host(v)))
    start, length = e.append([4])
    e.check_buffers()
    e.attend(e.queries(4, 16), start, length, [4], 16)


def test_cuts_by_the_rule(dev):
    """Appends and cuts at random: a length may fall to a page's end, or into a page from the lowest that stands in the open buffer
    on (kv8_ref.Cuts)."""
    from tests.kv8_ref import Cuts
    e, rng, cuts = Engine(dev, 1, 1, 128, 9), np.random.default_rng(8), Cuts()
    for turn in range(40):
        room = 9 * 64 - cuts.rows
        n = int(min(rng.choice([1, 3, 30, 63, 64, 65, 130, 300]), room))
        if n:
            start, length = e.append([n])
            cuts.append(n)
            e.check_buffers()
            if turn % 4 == 0:
                e.attend(e.queries(n, 8), start, length, [n], 8)
        to = int(rng.choice([x for x in range(cuts.rows + 1) if cuts.may(x)]))
        cuts.cut(to)
        e.seqs[0].cut(to)
