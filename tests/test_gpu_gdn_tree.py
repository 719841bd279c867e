"""The recurrent layer over a drafted tree, and the commit of a node's states, against the f64 statement."""
import numpy as np
import pytest
import torch

from irontimber_amd import _lib, ops
from tests import tree_ref as ref
from tests.gpu_util import announce, dev_f32, host

pytestmark = pytest.mark.gpu
EPS = 1e-6


def inputs(seed, nt, nv, nk, K=4, decay=1.0, sscale=0.05):
    r = np.random.default_rng(seed)
    f = lambda *s: r.standard_normal(s).astype(np.float32)
    cd = (2 * nk + nv) * 128
    return dict(x=f(nt, cd), w=0.5 * f(cd, K), conv=f(K - 1, cd), beta=f(nt, nv), alpha=f(nt, nv), dt=0.1 * f(nv),
                a=-decay * np.exp(r.uniform(-1, 1, nv)).astype(np.float32), state=sscale * f(nv, 128, 128))


def run(dev, d, anc, nv, nk, leaf=None):
    t = {k: dev_f32(z, dev) for k, z in d.items()}
    nt = len(d["x"])
    anc = torch.from_numpy(anc).to(dev)
    out = torch.full((nt, nv * 128), float("nan"), device=dev)
    trace = ops.gdn_tree_trace(nt, nv, nk, dev)
    trace.fill_(0xFF)
    ops.gdn_tree(t["x"], t["w"], t["conv"], t["beta"], t["alpha"], t["dt"], t["a"], t["state"], anc, nv, nk, trace, EPS,
                 out=out)
    for name in ("state", "conv"):      # the layer only reads them
        assert np.array_equal(host(t[name]), d[name], equal_nan=True)
    done = {}
    for k in () if leaf is None else leaf:
        c, s = t["conv"].clone(), t["state"].clone()
        ops.gdn_tree_commit(t["x"], c, s, anc, k, nv, nk, trace)
        done[k] = (host(c), host(s))
    return host(out).reshape(nt, nv, 128), done


def check(dev, seed, nt, nv, nk, shape, K=4, **kw):
    announce(f"gdn_tree nt={nt} {nv}/{nk} {shape} K={K} {kw}")
    d = inputs(seed, nt, nv, nk, K, **kw)
    par = ref.parents(shape, nt, seed)
    want, tol, states, errs, windows = ref.gdn(d["x"], d["w"], d["conv"], d["beta"], d["alpha"], d["dt"], d["a"], d["state"],
                                               par, nv, nk, EPS)
    leaves = {-1, 0, nt // 2, nt - 1}
    got, done = run(dev, d, ref.masks(par), nv, nk, leaves)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / np.maximum(tol, 1e-30)).max())
    for t in leaves:
        keep = -1 if t < 0 or ref.path(par, t) is None else t
        conv, state = done[t]
        assert np.array_equal(conv, windows[keep].astype(np.float32)), f"conv state after {t}"
        assert (np.abs(state - states[keep]) <= errs[keep][:, None, None]).all(), f"state after {t}"


@pytest.mark.parametrize("nv,nk", [(32, 16), (48, 16), (4, 4), (3, 1)])
@pytest.mark.parametrize("nt,shape", [(1, "chain"), (2, "forest"), (3, "star"), (15, "random"), (16, "chain"), (17, "padded"),
                                      (32, "star"), (33, "random"), (48, "forest"), (49, "padded"), (64, "chain"),
                                      (64, "padded")])
def test_geometries(dev, nv, nk, nt, shape):
    check(dev, nt, nt, nv, nk, shape)


@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("nt", [1, 2, 3, 4, 20])
def test_conv_sizes(dev, K, nt):
    check(dev, 3, nt, 4, 2, "chain", K=K)
    check(dev, 4, nt, 4, 2, "random", K=K)


@pytest.mark.parametrize("K", [2, 3])
@pytest.mark.parametrize("nt", [1, 16, 20, 41, 64])
def test_conv_sizes_of_many_heads(dev, K, nt):
    """48 heads: workgroups of 32 state columns."""
    check(dev, 5, nt, 48, 16, "random", K=K)


@pytest.mark.parametrize("decay", [0.0, 1e-3, 30.0, 1e4])
@pytest.mark.parametrize("shape", ["chain", "padded"])
def test_decays(dev, decay, shape):
    """No decay at all, and decays whose path sums leave the range of e^x (and, summed in f32, their own digits)."""
    check(dev, 5, 64, 4, 2, shape, decay=decay)


@pytest.mark.parametrize("sscale", [0.0, 1e-4, 1e3])
def test_state_sizes(dev, sscale):
    check(dev, 6, 40, 4, 2, "random", sscale=sscale)


def test_zero_rows(dev):
    """q and k rows of length zero: the norm's floor, no division by zero."""
    d = inputs(8, 5, 4, 2)
    d["x"][:] = 0
    d["conv"][:] = 0
    got, done = run(dev, d, ref.masks(ref.parents("chain", 5)), 4, 2, [4])
    assert (got == 0).all()
    g = np.log1p(np.exp(d["alpha"].astype(np.float64) + d["dt"])) * d["a"]
    want = d["state"] * np.exp(g.sum(0))[:, None, None]
    assert (np.abs(done[4][1] - want) <= 32 * 2.0 ** -24 * np.abs(want)).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38])
@pytest.mark.parametrize("name", ["x", "beta", "alpha"])
def test_other_branches_do_not_matter(dev, bad, name):
    """Whatever a padding node's or another branch's inputs hold, a node's output and states are those without them: to
    rounding where its own products run in another order, and bit for bit beside padding."""
    nt, nv, nk = 30, 4, 2
    d = inputs(9, nt, nv, nk)
    par = ref.parents("padded", nt, 9)
    anc = ref.masks(par)
    dead = [t for t in range(nt) if anc[t] == 0]
    leaf = max(t for t in range(nt) if anc[t])
    base, done = run(dev, d, anc, nv, nk, [leaf])
    d[name][dead] = bad
    got, again = run(dev, d, anc, nv, nk, [leaf])
    assert np.array_equal(got, base) and all(np.array_equal(a, b) for a, b in zip(done[leaf], again[leaf]))
    spoilt = next(t for t in range(2, nt) if anc[t] and not int(anc[leaf]) >> t & 1)
    d[name][spoilt] = bad
    got, again = run(dev, d, anc, nv, nk, [leaf])
    want, tol, states, errs, _ = ref.gdn(*(np.nan_to_num(d[k], nan=0.0, posinf=0.0) if k == name else d[k] for k in
                                           ("x", "w", "conv", "beta", "alpha", "dt", "a", "state")), par, nv, nk, EPS)
    keep = [t for t in range(nt) if anc[t] and not int(anc[t]) >> spoilt & 1]
    assert (np.abs(got - want)[keep] <= tol[keep]).all()
    assert (np.abs(again[leaf][1] - states[leaf]) <= errs[leaf][:, None, None]).all()


@pytest.mark.parametrize("nt", [14, 30, 60])
def test_other_branches_do_not_matter_to_many_heads(dev, nt):
    """The same with 32 state columns a workgroup: one branch's infinities reach no other node."""
    nv, nk = 48, 16
    d = inputs(12, nt, nv, nk)
    par = ref.parents("random", nt, 12)
    anc = ref.masks(par)
    spoilt = nt - 1
    d["x"][spoilt, ::3] = np.inf
    got, _ = run(dev, d, anc, nv, nk)
    d["x"][spoilt] = 0
    want, tol, *_ = ref.gdn(d["x"], d["w"], d["conv"], d["beta"], d["alpha"], d["dt"], d["a"], d["state"], par, nv, nk, EPS)
    assert (np.abs(got - want)[:spoilt] <= tol[:spoilt]).all()
    assert not np.isfinite(got[spoilt]).all()


def test_bits_that_are_no_ancestors(dev):
    """Later nodes' bits are ignored, and a node whose own bit is clear is padding."""
    nt, nv, nk = 6, 4, 2
    d = inputs(10, nt, nv, nk)
    par = np.array([-1, 0, -2, 1, 0, 4], np.int32)
    anc = ref.masks(par)
    base, done = run(dev, d, anc, nv, nk, [5, 2])
    loose = anc | np.array([-2, -4, 3, -16, -32, -64], np.int64)
    got, again = run(dev, d, loose, nv, nk, [5, 2])
    assert np.array_equal(got, base) and (got[2] == 0).all()
    for k in (5, 2):
        assert all(np.array_equal(a, b) for a, b in zip(done[k], again[k]))


def test_chain_agrees_with_the_decode_layer(dev):
    """Four tokens one after the other: it_gdn_decode_fused's outputs and states, to both sides' bound."""
    nt, nv, nk = 4, 32, 16
    d = inputs(11, nt, nv, nk)
    par = ref.parents("chain", nt)
    want, tol, states, errs, windows = ref.gdn(d["x"], d["w"], d["conv"], d["beta"], d["alpha"], d["dt"], d["a"], d["state"],
                                               par, nv, nk, EPS)
    got, done = run(dev, d, ref.masks(par), nv, nk, [3])
    t = {k: dev_f32(z, dev) for k, z in d.items()}
    conv2 = torch.empty_like(t["conv"])
    o = ops.gdn_decode_fused(t["x"], t["w"], t["conv"], conv2, t["beta"], t["alpha"], t["dt"], t["a"], t["state"], nv, nk, EPS)
    assert (np.abs(got - host(o).reshape(nt, nv, 128)) <= 2 * tol).all()
    assert (np.abs(done[3][1] - host(t["state"])) <= 2 * errs[3][:, None, None]).all()
    assert np.array_equal(done[3][0], host(conv2))


def test_strides_and_streams(dev):
    nt, nv, nk = 9, 4, 2
    cd = (2 * nk + nv) * 128
    d = inputs(12, nt, nv, nk)
    par = ref.parents("random", nt, 12)
    want, tol, states, errs, windows = ref.gdn(d["x"], d["w"], d["conv"], d["beta"], d["alpha"], d["dt"], d["a"], d["state"],
                                               par, nv, nk, EPS)
    wide = lambda z, n: np.concatenate([z, np.full((nt, n), np.nan, np.float32)], 1)
    x, br, ar = dev_f32(wide(d["x"], 8), dev), dev_f32(wide(d["beta"], 3), dev), dev_f32(wide(d["alpha"], 3), dev)
    t = {k: dev_f32(d[k], dev) for k in ("w", "conv", "dt", "a", "state")}
    anc = torch.from_numpy(ref.masks(par)).to(dev)
    out = torch.full((nt, nv * 128 + 5), 7.0, device=dev)
    nbytes = _lib.lib().it_gdn_tree_trace_bytes(nt, nv, nk, 128)
    trace = torch.full((nbytes + 64,), 0x55, device=dev, dtype=torch.uint8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    _lib.call("it_gdn_tree", x.data_ptr(), cd + 8, t["w"].data_ptr(), 4, t["conv"].data_ptr(), br.data_ptr(), ar.data_ptr(),
              nv + 3, t["dt"].data_ptr(), t["a"].data_ptr(), t["state"].data_ptr(), anc.data_ptr(), out.data_ptr(),
              nv * 128 + 5, nt, nv, nk, 128, EPS, trace.data_ptr(), nbytes, s.cuda_stream)
    _lib.call("it_gdn_tree_commit", x.data_ptr(), cd + 8, 4, t["conv"].data_ptr(), t["state"].data_ptr(), anc.data_ptr(),
              nt - 1, nt, nv, nk, 128, trace.data_ptr(), nbytes, s.cuda_stream)
    got = host(out)
    assert (got[:, nv * 128:] == 7.0).all() and (host(trace)[nbytes:] == 0x55).all()
    assert (np.abs(got[:, :nv * 128].reshape(nt, nv, 128) - want) <= tol).all()
    assert np.array_equal(host(t["conv"]), windows[nt - 1].astype(np.float32))
    assert (np.abs(host(t["state"]) - states[nt - 1]) <= errs[nt - 1][:, None, None]).all()
