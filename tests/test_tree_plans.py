"""The splits of the tree attentions' contexts: host code only."""
import pytest

from irontimber_amd import _lib

CUS = 256
RECORD = 1040


@pytest.mark.parametrize("G", range(1, 17))
@pytest.mark.parametrize("nkv", [1, 2, 4])
def test_f32kv_splits_are_planned_by_the_workgroups_launched(G, nkv):
    """A split's cost is the rounds of its workgroups over the CUs times the tiles each takes and one. The workgroups are
    those of the launch: whole nodes, as many as fit 32 rows. No other split costs less than the chosen one."""
    f = _lib.lib().it_attn_tree_f32kv_scratch_bytes
    nh = G * nkv
    for nt in range(1, 65):
        per = (32 if nt * G > 16 else 16) // G
        groups = nkv * -(-nt // per)
        for pos0 in (600, 1000, 2048, 4096, 8128, 12000, 20000, 32768):
            tiles = -(-pos0 // 64)
            smax = f(pos0, nt, 256, nh, nkv) // (nt * nh * RECORD)
            cost = lambda s: -(-s * groups // CUS) * (-(-tiles // s) + 1)
            best = min(cost(-(-tiles // k)) for k in range(1, tiles + 1))
            assert cost(smax) == best, (nt, pos0, smax)


@pytest.mark.parametrize("nh,nkv", [(16, 2), (24, 4)])
@pytest.mark.parametrize("nt", [1, 5, 64])
def test_sizes_of_any_context(nh, nkv, nt):
    """Scratch sizes up to the largest int are those of a plan: whole records, and at most twice the longest context's (a split a
    round of the CUs, however long)."""
    f = _lib.lib().it_attn_tree_scratch_bytes
    longest = f((1 << 22) - 64, nt, 256, nh, nkv)
    for pos0 in (1 << 24, (1 << 31) - 65, (1 << 31) - 64, (1 << 31) - 63, (1 << 31) - 2, (1 << 31) - 1):
        got = f(pos0, nt, 256, nh, nkv)
        assert got % (nt * nh * RECORD) == 0 and got <= 2 * longest, pos0
