"""Refusals of the tree-verification calls, and the rotation tables: host code only."""
import ctypes
import math

import numpy as np
import pytest
import torch

from irontimber_amd import _lib, ops

F = 1 << 20      # an aligned address that is never followed


def refused(name, *args, text=""):
    assert getattr(_lib.lib(), name)(*args) != 0
    assert text in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(nt=-1), "nt"), (dict(row0=-1), "pos0"), (dict(row0=1 << 22), "pos0"), (dict(hd=64), "head_dim"),
    (dict(nh=5), "n_head"), (dict(kvd=256), "kvd"), (dict(n_rot=3), "n_rot"), (dict(n_rot=258), "n_rot"),
    (dict(n_rot=4), "n_rot"), (dict(n_rot=-2), "n_rot"), (dict(freq=None), "freq"), (dict(mscale=math.inf), "mscale"),
    (dict(mscale=math.nan), "mscale"), (dict(layout=2), "layout"), (dict(mode=2), "round_mode"), (dict(q=None), "null"),
    (dict(q=F + 4), "aligned"), (dict(kc=F + 2), "aligned"), (dict(qts=4 * 512 - 4), "strides"),
    (dict(qts=4 * 512 + 2), "strides"), (dict(kts=508), "strides"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
    (dict(pos=None, pos0=-1), "pos0"), (dict(pos=None, pos0=2**31 - 4), "pos0")])
def test_prep_pos_refusals(kw, text):
    a = dict(q=F, qts=4 * 512, k=F, v=F, kts=512, qn=None, kn=None, eps=1e-6, kc=F, vc=F, kvd=512, pos=F, pos0=0, row0=0,
             hd=256, nh=4, nkv=2, nt=8, n_rot=64, freq=F, mscale=1.0, layout=0, mode=0)
    a.update(kw)
    refused("it_attn_prep_pos_f16", *a.values(), None, text=text)
    if "mode" not in kw:
        a.pop("mode")
        refused("it_attn_prep_pos_f32kv", *a.values(), None, text=text)


@pytest.mark.parametrize("args", [(F, 0, 0, F, F), (F, 65, 0, F, F), (F, 3, -1, F, F), (None, 3, 0, F, F),
                                  (F, 3, 0, None, F), (F, 3, 2**31 - 3, F, F)])
def test_tree_plan_refusals(args):
    refused("it_tree_plan", *args, None, text="it_tree_plan")


@pytest.mark.parametrize("kw", [dict(kc=None), dict(vc=None), dict(anc=None), dict(kc=F + 8), dict(kvd=0), dict(kvd=4),
                                dict(pos0=-1), dict(pos0=1 << 22), dict(nt=0), dict(nt=65), dict(leaf=-2), dict(leaf=5)])
def test_kv_tree_commit_refusals(kw):
    a = dict(kc=F, vc=F, kvd=512, pos0=9, nt=5, anc=F, leaf=2)
    a.update(kw)
    for name in ("it_kv_tree_commit_f16", "it_kv_tree_commit_f32"):
        refused(name, *a.values(), None, text=name)
        if "kc" not in kw and "vc" not in kw:
            assert getattr(_lib.lib(), name)(F, F, 512, 9, 5, F, -1, None) == 0     # nothing kept: nothing runs


@pytest.mark.parametrize("kw", [dict(q=None), dict(kc=None), dict(vc=None), dict(anc=None), dict(out=None), dict(q=F + 8),
                                dict(out=F + 4), dict(scratch=F + 8), dict(scratch=None), dict(nbytes=5 * 4 * 1040 - 1),
                                dict(hd=128), dict(nh=5), dict(kvd=256), dict(nt=0), dict(nt=65), dict(pos0=-1),
                                dict(rows=0), dict(rows=65), dict(pos0=(1 << 22) - 4), dict(qts=4 * 512 - 4),
                                dict(ots=1020), dict(qts=2050)])
@pytest.mark.parametrize("name", ["it_attn_tree_f16", "it_attn_tree_f32kv"])
def test_attn_tree_refusals(name, kw):
    a = dict(q=F, qts=4 * 512, kc=F, vc=F, kvd=512, pos0=700, hd=256, nh=4, nkv=2, nt=5, rows=5, anc=F, scale=0.0625, out=F,
             ots=4 * 256, scratch=F, nbytes=1 << 30)
    a.update(kw)
    refused(name, *a.values(), None, text=name)


def test_attn_tree_f32kv_refuses_wide_groups():
    refused("it_attn_tree_f32kv", F, 17 * 512, F, F, 256, 700, 256, 17, 1, 5, 5, F, 0.0625, F, 17 * 256, F, 1 << 30, None,
            text="16 q heads")


@pytest.mark.parametrize("nh,nkv", [(16, 2), (24, 4), (4, 4), (16, 1)])
def test_attn_tree_scratch(nh, nkv):
    """The preferred scratch holds whole records, is never below one per (node, head), and stays below 128 MiB."""
    for f in (_lib.lib().it_attn_tree_scratch_bytes, _lib.lib().it_attn_tree_f32kv_scratch_bytes):
        for nt in (1, 2, 5, 17, 64):
            assert f(0, nt, 256, nh, nkv) == 0
            for pos0 in (1, 63, 64, 65, 1000, 8128, 131072, (1 << 22) - nt):
                got = f(pos0, nt, 256, nh, nkv)
                assert got % (nt * nh * 1040) == 0 and nt * nh * 1040 <= got <= 128 << 20
        for bad in ((100, 0, 256, nh, nkv), (100, 65, 256, nh, nkv), (-1, 3, 256, nh, nkv), (100, 3, 256, nh, 0)):
            assert f(*bad) == 0


@pytest.mark.parametrize("kw", [dict(x=None), dict(conv=None), dict(state=None), dict(anc=None), dict(trace=None),
                                dict(x=F + 4), dict(conv=F + 4), dict(state=F + 8), dict(trace=F + 8), dict(nt=0),
                                dict(nt=65), dict(K=1), dict(K=5), dict(S=64), dict(nv=5), dict(nk=0), dict(xts=1020),
                                dict(xts=1026), dict(nbytes=5 * 6 * 512 + 5 * 4 * 8 - 1)])
def test_gdn_tree_refusals(kw):
    a = dict(x=F, xts=1024, w=F, K=4, conv=F, beta=F, alpha=F, bts=4, dt=F, a=F, state=F, anc=F, out=F, ots=512, nt=5, nv=4,
             nk=2, S=128, eps=1e-6, trace=F, nbytes=5 * 6 * 512 + 5 * 4 * 8)
    a.update(kw)
    refused("it_gdn_tree", *a.values(), None, text="it_gdn_tree")
    commit = ("x", "xts", "K", "conv", "state", "anc", 2, "nt", "nv", "nk", "S", "trace", "nbytes")
    refused("it_gdn_tree_commit", *(a.get(k, k) for k in commit), None, text="it_gdn_tree_commit")


@pytest.mark.parametrize("kw", [dict(w=None), dict(beta=None), dict(alpha=None), dict(dt=None), dict(a=None), dict(out=None),
                                dict(ots=508), dict(bts=3), dict(eps=math.nan)])
def test_gdn_tree_layer_refusals(kw):
    a = dict(x=F, xts=1024, w=F, K=4, conv=F, beta=F, alpha=F, bts=4, dt=F, a=F, state=F, anc=F, out=F, ots=512, nt=5, nv=4,
             nk=2, S=128, eps=1e-6, trace=F, nbytes=1 << 20)
    a.update(kw)
    refused("it_gdn_tree", *a.values(), None, text="it_gdn_tree")


def test_gdn_tree_commit_leaf():
    f = _lib.lib().it_gdn_tree_commit
    for leaf in (-2, 5):
        assert f(F, 1024, 4, F, F, F, leaf, 5, 4, 2, 128, F, 1 << 20, None) != 0 and "leaf" in _lib.last_error()
    assert f(F, 1024, 4, F, F, F, -1, 5, 4, 2, 128, F, 1 << 20, None) == 0     # nothing kept: nothing runs
    trace = _lib.lib().it_gdn_tree_trace_bytes
    assert trace(5, 4, 2, 128) == 5 * 6 * 512 + 5 * 4 * 8
    assert trace(0, 4, 2, 128) == trace(65, 4, 2, 128) == trace(5, 5, 2, 128) == trace(5, 4, 2, 64) == 0


def freqs(*args):
    f, m = (ctypes.c_float * max(args[0] // 2, 1))(), ctypes.c_float()
    assert _lib.lib().it_rope_freqs(*args, f, ctypes.byref(m)) == 0, _lib.last_error()
    return np.array(f, np.float64), m.value


def test_rope_freqs():
    step = 2.0 ** -24        # one rounding to f32
    i = np.arange(32)
    plain = 1e7 ** (-2 * i / 64)
    f, m = freqs(64, 1e7, 0, 5.0, 0)
    assert m == 1 and (np.abs(f - plain) <= step * plain).all()
    f, m = freqs(64, 1e7, 1, 8.0, 0)
    assert m == 1 and (np.abs(f - plain / 8) <= step * plain).all()
    f, m = freqs(64, 1e7, 2, 8.0, 0)
    assert m == 1 and f[0] == 1 and abs(f[31] * 8 / plain[31] - 1) <= 2 * step     # slowest stretched, fastest kept
    f, m = freqs(64, 1e7, 3, 16.0, 8192)
    assert abs(m - (0.1 * math.log(16) + 1)) <= step * 2
    turns = 8192 * plain / (2 * math.pi)
    # outside the blend (whose ends are rounded outwards to whole pairs) exactly kept and exactly stretched
    kept, slow = turns >= 32 * 1e7 ** (2 / 64), turns <= 1e7 ** (-2 / 64)
    assert kept.sum() >= 4 and slow.sum() >= 4
    assert (np.abs(f - plain)[kept] <= step * plain[kept]).all()
    assert (np.abs(f * 16 - plain)[slow] <= step * plain[slow]).all()
    assert (f <= plain * (1 + step)).all() and (f * 16 >= plain * (1 - step)).all() and (np.diff(f) < 0).all()
    assert np.array_equal(freqs(64, 1e7, 3, 1.0, 8192)[0], freqs(64, 1e7, 0, 1.0, 0)[0])
    assert np.array_equal(freqs(2, 1e4, 0, 1.0, 0)[0], [1.0])


@pytest.mark.parametrize("args", [(0, 1e7, 0, 1.0, 0), (3, 1e7, 0, 1.0, 0), (258, 1e7, 0, 1.0, 0), (64, 1.0, 0, 1.0, 0),
                                  (64, math.nan, 0, 1.0, 0), (64, math.inf, 0, 1.0, 0), (64, 1e7, 4, 1.0, 0),
                                  (64, 1e7, -1, 1.0, 0), (64, 1e7, 1, 0.5, 0), (64, 1e7, 2, math.inf, 0),
                                  (64, 1e7, 3, math.nan, 8192), (64, 1e7, 3, 2.0, 0), (2, 1e7, 2, 2.0, 0)])
def test_rope_freqs_refusals(args):
    f, m = (ctypes.c_float * 128)(), ctypes.c_float()
    refused("it_rope_freqs", *args, f, ctypes.byref(m), text="it_rope_freqs")


def test_front_end_refuses_host_tensors():
    z = torch.zeros(2, 1024)
    with pytest.raises(ValueError, match="device"):
        ops.attn_prep_pos_f16(z, z, z, z.half(), z.half(), None, 0, 1, 1, z[0])
    with pytest.raises(ValueError, match="device"):
        ops.tree_plan(torch.zeros(3, dtype=torch.int32), 0)
    with pytest.raises(ValueError, match="device"):
        ops.kv_tree_commit_f16(z.half(), z.half(), 0, 2, torch.zeros(2, dtype=torch.int64), 0)
    with pytest.raises(ValueError, match="kind"):
        ops.rope_freqs(64, kind="other", device="cpu")
