"""Values at the ends of their range in the tree-verification calls, against the f64 statements."""
import numpy as np
import pytest
import torch

from irontimber_amd import ops
from tests import tree_ref as ref
from tests.gpu_util import announce, dev_f32, host
from tests.test_gpu_attn_tree import inputs as attn_inputs, run as attn_run
from tests.test_gpu_gdn_tree import EPS, inputs as gdn_inputs, run as gdn_run
from tests.test_tree_plans import MERGES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nv,nk", [(4, 2), (48, 16)])
@pytest.mark.parametrize("nt", [14, 30, 60])
def test_updates_that_overflow_stay_on_their_path(dev, nt, nv, nk):
    """Nodes 1 and 2, its child, have finite inputs and right-hand sides near the end of f32's range, and k rows that point
    against each other: node 2's update passes the range inside the solve. No node beside their path sees it, in its
    output or in the states committed after it."""
    announce(f"gdn_tree nt={nt} {nv}/{nk} overflow in the solve")
    d = gdn_inputs(nt, nt, nv, nk)
    par = ref.parents("random", nt, nt)
    par[1:3] = 0, 1
    par[3:][(par[3:] == 1) | (par[3:] == 2)] = 0
    d["w"][:, :-1], d["w"][:, -1] = 0, 1            # a node's own input alone
    qk = 2 * nk * 128
    d["x"][1:3, qk:] = 3.3e38
    d["x"][1:3, qk // 2:qk] = 0                     # k rows e0 and -e0 of every head
    d["x"][1, qk // 2:qk:128], d["x"][2, qk // 2:qk:128] = 10, -1.278
    d["beta"][1:3], d["alpha"][1:3] = 30, -30       # nothing damped
    want, tol, states, errs, _ = ref.gdn(*(d[k] for k in ("x", "w", "conv", "beta", "alpha", "dt", "a", "state")), par, nv, nk,
                                         EPS)
    anc = ref.masks(par)
    keep = [t for t in range(nt) if not int(anc[t]) >> 1 & 1]
    assert len(keep) == nt - 2
    got, done = gdn_run(dev, d, anc, nv, nk, keep[1:])
    assert (np.abs(got - want)[keep] <= tol[keep]).all()
    for t in keep[1:]:
        assert (np.abs(done[t][1] - states[t]) <= errs[t][:, None, None]).all(), t


def silu(x):
    return x / (1 + np.exp(-x))


@pytest.mark.parametrize("nv,nk", [(4, 2), (48, 16)])
@pytest.mark.parametrize("nt,size", [(1, 0.3), (3, 1e-3), (20, 1e-3), (5, 1e-6), (40, 1e-9)])
def test_rows_below_the_norms_floor(dev, nt, size, nv, nk):
    """q rows of norm `size` * eps come out at length `size`, to the accuracy that full rows have: the output is `size` times
    that of the same rows without a floor, and so is its bound. (k rows are full ones, so the states are too.)"""
    announce(f"gdn_tree nt={nt} {nv}/{nk} q rows of {size} eps")
    d = gdn_inputs(nt, nt, nv, nk)
    par = ref.parents("random", nt, nt)
    d["w"][:, :-1], d["w"][:, -1] = 0, 1
    q = slice(0, nk * 128)
    d["x"][:, q] *= size * EPS / 5.66               # |silu(z)| = |z| / 2 of 128 small normal values: 5.66 times their size
    args = [d[k] for k in ("x", "w", "conv", "beta", "alpha", "dt", "a", "state")]
    want, _, states, errs, _ = ref.gdn(*args, par, nv, nk, EPS)
    _, tol, *_ = ref.gdn(*args, par, nv, nk, 1e-30)
    row = np.linalg.norm(silu(d["x"][:, q].astype(np.float64)).reshape(nt, nk, 128), axis=-1) / EPS
    assert (row < 1).all()
    tol = tol * row[:, np.arange(nv) % nk, None]
    got, done = gdn_run(dev, d, ref.masks(par), nv, nk, [nt - 1])
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
    assert (np.abs(done[nt - 1][1] - states[nt - 1]) <= errs[nt - 1][:, None, None]).all()


@pytest.mark.parametrize("nv,nk", [(4, 2), (48, 16)])
@pytest.mark.parametrize("nt,size", [(1, 0.3), (3, 1e-3), (20, 1e-3), (5, 1e-6), (40, 1e-9)])
def test_updates_of_rows_below_the_norms_floor(dev, nt, size, nv, nk):
    """k rows of norm `size` * eps on an empty state: what a chain leaves is `size` times a sum of updates, and as accurate."""
    announce(f"gdn_tree nt={nt} {nv}/{nk} k rows of {size} eps")
    d = gdn_inputs(nt, nt, nv, nk)
    par = ref.parents("chain", nt)
    d["w"][:, :-1], d["w"][:, -1] = 0, 1
    d["state"][:] = 0
    k = slice(nk * 128, 2 * nk * 128)
    d["x"][:, k] *= size * EPS / 5.66
    _, _, states, _, _ = ref.gdn(*(d[n] for n in ("x", "w", "conv", "beta", "alpha", "dt", "a", "state")), par, nv, nk, EPS)
    x = d["x"].astype(np.float64)
    row = np.linalg.norm(silu(x[:, k]).reshape(nt, nk, 128), axis=-1) / EPS
    assert (row < 1).all()
    # Each update k u^T: k relative to its row as in the layer's statement (the conv's sums here are one product: 6 steps of
    # the largest element over the row's mean one, 12 of the norm, 4 of the pair), u = beta (v - what `size`^2 leaves): v and
    # beta 20 steps, the decays 16 and the sum over the path 64.
    z = np.abs(x[:, k]).reshape(nt, nk, 128)
    rel = 6 * z.max(-1) * np.sqrt(128) / (row * EPS) + 16 + 20 + 16 + 64
    u = np.abs(silu(x[:, 2 * nk * 128:])).reshape(nt, nv, 128).max(-1)
    head = np.arange(nv) % nk
    tol = (2.0 ** -24 * rel * row)[:, head] * u * (1 + size)
    _, done = gdn_run(dev, d, ref.masks(par), nv, nk, [0, nt - 1])
    for t in (0, nt - 1):
        bound = tol[:t + 1].sum(0)[:, None, None]
        assert (np.abs(done[t][1] - states[t]) <= bound).all(), float((np.abs(done[t][1] - states[t]) / bound).max())


@pytest.mark.parametrize("qscale,scale,kscale", [(1.0, 1 / 16, 6.0), (1.0, 1e-3, 375.0), (1.0, 1e-4, 3750.0), (0.02, 1 / 16, 300.0),
                                                 (1.0, -1e-4, 3750.0), (1.0, 0.0, 1.0), (3e4, 1 / 16, 2e-4)])
@pytest.mark.parametrize("nt,pos0", [(3, 700), (16, 1100), (64, 700), (64, 2100), (64, 4200)])
def test_sizes_of_queries_keys_and_scale(dev, nt, pos0, qscale, scale, kscale):
    """Scores of the same spread (6, so that few keys carry a row) from queries, keys and scales of other sizes, in every form of
    the context."""
    announce(f"attn_tree nt={nt} pos0={pos0} q {qscale} scale {scale} k {kscale}")
    q, k, v = attn_inputs(nt, nt, pos0, 16, 2, kscale)
    q[..., :256] *= qscale
    anc = ref.masks(ref.parents("random", nt, nt))
    # (the statement's bound takes a size from the scale: a negative one is given as the queries' sign)
    sign = np.where(np.arange(512) < 256, np.float32(np.sign(scale)), np.float32(1))
    want, tol = ref.attn(q * sign, k, v, pos0, 16, 2, anc, abs(scale))
    got = attn_run(dev, q, k, v, pos0, 16, 2, anc, scale=scale)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("ramp", ["up", "down"])
@pytest.mark.parametrize("f32,nt,pos0,nh,nkv", MERGES)
def test_merges_of_every_form(dev, f32, nt, pos0, nh, nkv, ramp):
    """Records joined by every form of the merge, with scores that grow or fall along the context: the largest are in the last
    records, or in the first."""
    announce(f"attn_tree merge f32={f32} nt={nt} pos0={pos0} {nh}/{nkv} {ramp}")
    q, k, v = attn_inputs(pos0 + nt, nt, pos0, nh, nkv)
    size = np.linspace(0.2, 6, pos0)[:, None].astype(np.float32)
    k[:pos0] = (k[:pos0] * (size if ramp == "up" else size[::-1])).astype(np.float16)
    kind = np.float32 if f32 else np.float16
    k, v = k.astype(kind), v.astype(kind)
    anc = ref.masks(ref.parents("random", nt, nt))
    want, tol = ref.attn(q, k, v, pos0, nh, nkv, anc, 1 / 16)
    call = ops.attn_tree_f32kv if f32 else ops.attn_tree_f16
    got = host(call(dev_f32(q.reshape(nt, -1), dev), torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), pos0, nh, nkv,
                    torch.from_numpy(anc).to(dev))).reshape(nt, nh, 256)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
