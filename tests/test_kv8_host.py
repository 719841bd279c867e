"""The paged 8-bit cache's host side: index arithmetic, sizes and refusals. No device work."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from irontimber_amd import _lib, ops
from tests import kv8_ref as ref

ROOT = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
F = 1 << 20      # an aligned address that is never followed


def test_index_sweep(tmp_path):
    exe = tmp_path / "kv8_sweep"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-o", str(exe),
                    os.path.join(ROOT, "tests", "csrc", "kv8_sweep.cpp")], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.startswith("ok"), res.stdout + res.stderr


def test_scales_make_every_value_an_f16_number():
    """code * scale is exact in f16 for every f16 that can be a block's largest, and the largest keeps its place."""
    bits = np.arange(0, 0x7C00, 1, dtype=np.uint16)
    amax = bits.view(np.float16).astype(np.float64)
    t = amax / 127
    unit = np.exp2(np.maximum(np.ceil(np.log2(np.maximum(t, 1e-30) / 16)), -24))
    s = np.maximum(np.ceil(amax / (127 * unit)), 1) * unit
    for i in range(0, len(bits), 97):
        assert s[i] == ref.scale_of(amax[i])
    steps = np.arange(0, 128)[:, None]
    most = np.where(s > 512, 113, 127)
    values = np.minimum(steps, most) * s
    assert np.array_equal(values.astype(np.float16).astype(np.float64), values)
    assert (s * 127 >= amax).all() and np.array_equal(s.astype(np.float16).astype(np.float64), s)
    assert (s <= np.maximum(t * 1.125, 2.0 ** -24 + t)).all()


def cache(**kw):
    a = dict(kp=F, vp=2 * F, sc=3 * F, tk=4 * F, tv=5 * F, npages=10, nseq=3, nkv=2, hd=256)
    a.update(kw)
    return _lib.Kv8CacheArgs(*a.values())


def refused(name, *args, text=""):
    assert getattr(_lib.lib(), name)(*args) != 0
    assert text in _lib.last_error(), _lib.last_error()


CACHES = [(dict(hd=64), "head_dim"), (dict(hd=512), "head_dim"), (dict(nkv=0), "n_head_kv"), (dict(nkv=1025), "n_head_kv"),
          (dict(npages=0), "pages"), (dict(npages=-1), "pages"), (dict(nseq=0), "nseq"), (dict(nseq=65536), "nseq"),
          (dict(kp=None), "null"), (dict(tv=None), "null"), (dict(sc=F + 8), "aligned"), (dict(tk=F + 2), "aligned")]
BATCHES = [(dict(ntok=0), "ntok"), (dict(ntok=-5), "ntok"), (dict(max_nt=0), "bound"), (dict(max_nt=-1), "bound"),
           (dict(max_pages=0), "max_pages"), (dict(max_pages=1 << 25), "max_pages"), (dict(start=None), "null"),
           (dict(len=None), "null"), (dict(table=None), "null")]


def addr(c):
    return ctypes.byref(c)      # (keeps it alive)


@pytest.mark.parametrize("kw,text", CACHES)
def test_cache_refusals(kw, text):
    c = cache(**kw)
    refused("it_kv8_append", addr(c), F, F, 512, 8, F, F, F, 4, 8, None, text=text)
    refused("it_kv8_read", addr(c), F, 2 * F, 512, 8, F, F, F, F, 4, 8, None, text=text)
    refused("it_kv8_copy", addr(c), F, F, 1, F, F, 1, None, text=text)
    refused("it_attn_kv8", addr(c), F, 16384, 8, F, F, F, 4, 8, 16, 0.1, F, 8192, 0, F, 1 << 30, None, text=text)


@pytest.mark.parametrize("kw,text", BATCHES)
def test_batch_refusals(kw, text):
    c, a = cache(), dict(ntok=8, start=F, len=F, table=F, max_pages=4, max_nt=8)
    a.update(kw)
    refused("it_kv8_append", addr(c), F, F, 512, *a.values(), None, text=text)
    refused("it_kv8_read", addr(c), F, 2 * F, 512, a["ntok"], a["start"], F, a["len"], a["table"], a["max_pages"], a["max_nt"], None,
            text=text)
    refused("it_attn_kv8", addr(c), F, 16384, *a.values(), 16, 0.1, F, 8192, 0, F, 1 << 30, None, text=text)


def test_null_cache():
    refused("it_kv8_append", None, F, F, 512, 8, F, F, F, 4, 8, None, text="null cache")


@pytest.mark.parametrize("kw,text", [(dict(k=None), "null"), (dict(v=None), "null"), (dict(k=F + 8), "aligned"), (dict(kts=508), "multiple"),
                                     (dict(kts=504), "overlap"), (dict(kts=-512), "overlap")])
def test_row_refusals(kw, text):
    c, a = cache(), dict(k=F, v=2 * F, kts=512)
    a.update(kw)
    refused("it_kv8_append", addr(c), *a.values(), 8, F, F, F, 4, 8, None, text=text)
    refused("it_kv8_read", addr(c), *a.values(), 8, F, F, F, F, 4, 8, None, text=text)


def test_read_refusals():
    refused("it_kv8_read", addr(cache()), F, F, 512, 8, F, F, F, F, 4, 8, None, text="two buffers")
    refused("it_kv8_read", addr(cache()), F, 2 * F, 512, 8, F, None, F, F, 4, 8, None, text="null")


@pytest.mark.parametrize("args,text", [((F, F, -1, F, F, 0), "page copies"), ((F, F, 11, F, F, 0), "page copies"),
                                       ((F, F, 0, F, F, 4), "sequence copies"), ((F, F, 0, F, F, -1), "sequence copies"),
                                       ((None, F, 1, None, None, 0), "null"), ((None, None, 0, F, None, 1), "null")])
def test_copy_refusals(args, text):
    refused("it_kv8_copy", addr(cache()), *args, None, text=text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(nh=5), "n_head"), (dict(nh=0), "n_head"), (dict(q=F + 4), "aligned"),
    (dict(out=F + 8), "aligned"), (dict(qts=16382), "strides"), (dict(ots=8190), "strides"), (dict(ots=8196, f16=1), "strides"),
    (dict(qts=8188), "overlap"), (dict(ots=1024), "overlap"), (dict(qts=-16384), "overlap"), (dict(ntok=1 << 23), "rows"),
    (dict(scratch=None), "scratch"), (dict(scratch=F + 8), "scratch"), (dict(nbytes=1000), "scratch")])
def test_attention_refusals(kw, text):
    a = dict(q=F, qts=16384, ntok=8, start=F, len=F, table=F, pages=4, max_nt=8, nh=16, scale=0.1, out=F, ots=8192, f16=0,
             scratch=F, nbytes=1 << 30)
    a.update(kw)
    refused("it_attn_kv8", addr(cache()), *a.values(), None, text=text)


@pytest.mark.parametrize("kw,text", [(dict(nh=1 << 24, ntok=2, qts=1 << 30), "overlap"), (dict(nh=1 << 24, ntok=2, ots=1 << 20, qts=0x7ffffff0), "overlap"),
                                     (dict(nh=1 << 18, ntok=1, qts=0, ots=0), "share"),
                                     (dict(nh=1024, ntok=65535, qts=1 << 20, ots=1 << 19), "sequences")])
def test_attention_refusals_of_sizes_past_32_bits(kw, text):
    """Widths of a token's row that pass an int, and more row blocks than a launch has room for."""
    many = cache(nkv=1024, nseq=65535) if text == "sequences" else cache()
    a = dict(q=F, qts=16384, ntok=8, start=F, len=F, table=F, pages=4, max_nt=8, nh=16, scale=0.1, out=F, ots=8192, f16=0,
             scratch=F, nbytes=1 << 62)
    a.update(kw)
    refused("it_attn_kv8", addr(many), *a.values(), None, text=text)


def test_scratch_sizes():
    f = _lib.lib().it_attn_kv8_scratch_bytes
    for args in ((0, 256, 16, 2), (1, 64, 16, 2), (1, 256, 16, 3), (1, 256, 0, 2), (1, 256, 16, 0), (-1, 256, 16, 2)):
        assert f(*args) == 0
    sizes = [f(n, 256, 16, 2) for n in (1, 2, 3, 4, 5, 8, 16, 64, 8192)]
    assert sizes == sorted(sizes)         # scratch for the bound given is enough for fewer tokens
    assert all(s % 16 == 0 and 0 < s <= 160 << 20 for s in sizes)
    assert ops.attn_kv8_scratch_bytes(4, 16, 2) == f(4, 256, 16, 2)
