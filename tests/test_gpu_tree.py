"""Tree plan, pre-pass at given positions and the kept cache rows on the GPU, against 64-bit statements."""
import numpy as np
import pytest
import torch

from irontimber_amd import _lib, ops
from tests import tree_ref as ref
from tests.gpu_util import announce, dev_f32, host

pytestmark = pytest.mark.gpu

# norm_rotate's error relative to |a| + |b| of the pair, in steps of 2^-24: the sum of squares 8, its square
# root and division 2, the two factors 2; the reduced angle (half a step of a value below 4) 2, sincosf 2, the
# factor of cos and sin 1; two products and a sum 3
PREP_TOL = 20 * 2.0 ** -24


@pytest.mark.parametrize("nt", [1, 2, 7, 33, 63, 64])
@pytest.mark.parametrize("shape", ref.SHAPES)
def test_tree_plan(dev, shape, nt):
    par = ref.parents(shape, nt, seed=nt)
    anc, pos = ops.tree_plan(torch.from_numpy(par).to(dev), 1000)
    want = ref.masks(par)
    depth = np.array([len(ref.path(par, t) or [0]) - 1 for t in range(nt)])
    assert np.array_equal(host(anc), want)
    assert np.array_equal(host(pos), 1000 + depth)


def test_tree_plan_rejects_every_foreign_parent(dev):
    par = np.array([-1, 0, 2, 7, -3, -2**31, 2**31 - 1, 2, 1, 8], np.int32)
    anc, _ = ops.tree_plan(torch.from_numpy(par).to(dev), 0)
    assert host(anc).tolist() == [1, 3, 0, 0, 0, 0, 0, 0, 0b100000011, 0b1100000011]


def prep_case(dev, seed, nt, nh, nkv, hd, n_rot, layout, kv, row0, pos, weights=True, mscale=1.0, rows=None):
    r = np.random.default_rng(seed)
    f = lambda *s: r.standard_normal(s).astype(np.float32)
    kvd = nkv * hd
    q, k, v = 2 * f(nt, nh * 2 * hd), 2 * f(nt, kvd), f(nt, kvd)
    qn, kn = (1 + 0.1 * f(hd), 1 + 0.1 * f(hd)) if weights else (None, None)
    freq = (1e6 ** (-2 * np.arange(n_rot // 2) / max(n_rot, 1))).astype(np.float32)
    rows = row0 + nt + 3 if rows is None else rows
    dt = torch.float16 if kv == "f16" else torch.float32
    kc, vc = (torch.from_numpy(f(rows, kvd)).to(dev).to(dt) for _ in range(2))
    kc0, vc0 = host(kc).copy(), host(vc).copy()
    qd = dev_f32(q, dev)
    call = ops.attn_prep_pos_f16 if kv == "f16" else ops.attn_prep_pos_f32kv
    call(qd, dev_f32(k, dev), dev_f32(v, dev), kc, vc,
         None if pos is None else torch.from_numpy(pos.astype(np.int32)).to(dev), row0, nh, nkv, dev_f32(freq, dev),
         mscale=mscale, layout=layout, q_norm=None if qn is None else dev_f32(qn, dev),
         k_norm=None if kn is None else dev_f32(kn, dev), eps=1e-6, **({"pos0": 77} if pos is None else {}))
    p = 77 + np.arange(nt) if pos is None else pos
    q3 = q.reshape(nt, nh, 2 * hd)
    want, size = ref.norm_rotate(q3[..., :hd], qn, 1e-6, p, freq, mscale, layout == "interleaved")
    got = host(qd).reshape(nt, nh, 2 * hd)
    assert np.array_equal(got[..., hd:], q3[..., hd:]), "gates changed"
    assert (np.abs(got[..., :hd] - want) <= PREP_TOL * size + 1e-30).all()
    want, size = ref.norm_rotate(k.reshape(nt, nkv, hd), kn, 1e-6, p, freq, mscale, layout == "interleaved")
    half_step = 2.0 ** -11 if kv == "f16" else 0.0      # of the stored value; 2^-25 among the smallest f16
    tol = PREP_TOL * size + half_step * np.abs(want) * (1 + PREP_TOL) + (2.0 ** -25 if kv == "f16" else 1e-30)
    gk, gv = host(kc), host(vc)
    assert (np.abs(gk[row0:row0 + nt].reshape(nt, nkv, hd).astype(np.float64) - want) <= tol).all()
    assert np.array_equal(gv[row0:row0 + nt], v.astype(gv.dtype))
    for got, old in ((gk, kc0), (gv, vc0)):             # the other cache rows
        assert np.array_equal(got[:row0], old[:row0]) and np.array_equal(got[row0 + nt:], old[row0 + nt:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("nh,nkv,hd,n_rot", [(16, 2, 256, 64), (24, 4, 256, 256), (24, 4, 128, 128), (3, 3, 128, 64),
                                             (1, 1, 256, 0), (5, 1, 128, 8)])
def test_prep_pos_geometries(dev, layout, kv, nh, nkv, hd, n_rot):
    announce(f"prep_pos {layout} {kv} {nh}/{nkv} hd {hd} n_rot {n_rot}")
    r = np.random.default_rng(5)
    prep_case(dev, 1, 13, nh, nkv, hd, n_rot, layout, kv, 5, r.integers(0, 100_000, 13))


@pytest.mark.parametrize("n_rot", [2, 6, 30, 254])
def test_prep_pos_pairs_of_any_count(dev, n_rot):
    prep_case(dev, 2, 3, 4, 2, 256, n_rot, "interleaved", "f16", 0, np.array([0, 1, 4095]))


@pytest.mark.parametrize("pos", [[0], [2**31 - 1], [-5], [1, 0, 2**22, 2**30, 7, 7, 7]])
def test_prep_pos_positions(dev, pos):
    """Far, negative and repeated positions, in any order."""
    prep_case(dev, 3, len(pos), 16, 2, 256, 64, "half", "f16", 2, np.array(pos))


@pytest.mark.parametrize("nt", [1, 64, 501])
def test_prep_pos_consecutive(dev, nt):
    """No position array: pos0 + t; no norm weights; cos and sin scaled."""
    prep_case(dev, 4, nt, 16, 2, 256, 64, "half", "f16", 31, None, weights=False, mscale=1.277)


def test_prep_pos_agrees_with_the_models_own_rotation(dev):
    """freq = theta_scale^i at positions pos0 + t is attn_prep_f16's rotation, but for the f32 rounding of the
    table (2^-24 relative in the angle, at most 200 * 2^-24 rad here)."""
    from irontimber_amd.synth import rope_theta_scale
    r = np.random.default_rng(6)
    nt, nh, nkv, hd, pos0 = 9, 16, 2, 256, 190
    q, k, v = (torch.from_numpy(r.standard_normal(s).astype(np.float32)).to(dev)
               for s in ((nt, nh * 512), (nt, 512), (nt, 512)))
    caches = [torch.zeros(pos0 + nt, 512, device=dev, dtype=torch.float16) for _ in range(4)]
    q2 = q.clone()
    ops.attn_prep_f16(q, k, v, caches[0], caches[1], pos0, nh, nkv)
    ts = np.float64(np.float32(rope_theta_scale(1e7, 64)))
    ops.attn_prep_pos_f16(q2, k, v, caches[2], caches[3], None, pos0, nh, nkv,
                          dev_f32(ts ** np.arange(32), dev), pos0=pos0)
    a, b = host(q), host(q2)
    assert np.abs(a - b).max() <= (200 * 2.0 ** -24 + 2 * PREP_TOL) * 2 * np.abs(a).max()
    assert np.array_equal(host(caches[1]), host(caches[3]))


def test_prep_pos_strides(dev):
    """Token strides wider than the rows, and the words between them left alone."""
    r = np.random.default_rng(8)
    nt, nh, nkv, hd, n_rot = 6, 4, 2, 256, 64
    qts, kts = nh * 2 * hd + 12, nkv * hd + 8
    q, k, v = (r.standard_normal((nt, s)).astype(np.float32) for s in (qts, kts, kts))
    freq = (1e4 ** (-2 * np.arange(n_rot // 2) / n_rot)).astype(np.float32)
    pos = np.array([3, 4, 4, 5, 5, 5], np.int32)
    qd, kd, vd, fd, pd = dev_f32(q, dev), dev_f32(k, dev), dev_f32(v, dev), dev_f32(freq, dev), torch.from_numpy(pos).to(dev)
    kc, vc = (torch.zeros(nt, nkv * hd, device=dev, dtype=torch.float16) for _ in range(2))
    _lib.call("it_attn_prep_pos_f16", qd.data_ptr(), qts, kd.data_ptr(), vd.data_ptr(), kts, None, None, 1e-6,
              kc.data_ptr(), vc.data_ptr(), nkv * hd, pd.data_ptr(), 0, 0, hd, nh, nkv, nt, n_rot, fd.data_ptr(), 1.0, 0, 0,
              torch.cuda.current_stream().cuda_stream)
    got = host(qd)
    assert np.array_equal(got[:, nh * 2 * hd:], q[:, nh * 2 * hd:])
    want, size = ref.norm_rotate(q[:, :nh * 2 * hd].reshape(nt, nh, 2 * hd)[..., :hd], None, 1e-6, pos, freq, 1.0, False)
    assert (np.abs(got[:, :nh * 2 * hd].reshape(nt, nh, 2 * hd)[..., :hd] - want) <= PREP_TOL * size).all()
    assert np.array_equal(host(vc), v[:, :nkv * hd].astype(np.float16))


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("kvd", [8, 512, 1000, 1024])
@pytest.mark.parametrize("shape,nt", [("chain", 64), ("random", 41), ("padded", 20), ("star", 64), ("forest", 10),
                                      ("chain", 1)])
def test_kv_tree_commit(dev, kv, kvd, shape, nt):
    announce(f"kv_tree_commit {kv} kvd {kvd} {shape} {nt}")
    r = np.random.default_rng(nt + kvd)
    dt, pos0 = np.float16 if kv == "f16" else np.float32, 37
    k, v = (r.standard_normal((pos0 + nt + 2, kvd)).astype(dt) for _ in range(2))
    call = ops.kv_tree_commit_f16 if kv == "f16" else ops.kv_tree_commit_f32
    # a chain that starts over: its path skips the first nodes, and the moved rows overlap
    par = ref.parents(shape, nt, seed=nt)
    if shape == "chain" and nt > 8:
        par[3] = -1
    anc = torch.from_numpy(ref.masks(par)).to(dev)
    for leaf in {-1, 0, nt // 2, nt - 1}:
        kd, vd = torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev)
        call(kd, vd, pos0, nt, anc, leaf)
        kept = ref.path(par, leaf) or [] if leaf >= 0 else []
        for got, old in ((host(kd), k), (host(vd), v)):
            want = old.copy()
            for i, t in enumerate(kept):
                want[pos0 + i] = old[pos0 + t]
            assert np.array_equal(got, want), f"leaf {leaf}"


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_kv_tree_commit_keeps_nothing_of_a_padding_node(dev, kv):
    """A node whose own bit is clear is padding whatever else its mask holds, as it is to the recurrent layer's commit."""
    r = np.random.default_rng(9)
    dt = np.float16 if kv == "f16" else np.float32
    k, v = (r.standard_normal((9, 512)).astype(dt) for _ in range(2))
    anc = torch.tensor([1, 2, 0b10, 0b1000], dtype=torch.int64, device=dev)   # node 2: its ancestor's bit alone
    kd, vd = torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev)
    (ops.kv_tree_commit_f16 if kv == "f16" else ops.kv_tree_commit_f32)(kd, vd, 5, 4, anc, 2)
    assert np.array_equal(host(kd), k) and np.array_equal(host(vd), v)
