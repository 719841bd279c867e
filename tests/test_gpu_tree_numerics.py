"""Values at the ends of their range in the tree-verification calls, against the f64 statements."""
import numpy as np
import pytest

from tests import tree_ref as ref
from tests.gpu_util import announce
from tests.test_gpu_gdn_tree import EPS, inputs as gdn_inputs, run as gdn_run

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
