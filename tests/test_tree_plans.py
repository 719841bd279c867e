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


# (f32 cache, nodes, context, q heads, KV heads) whose merges take each form: 4 or 16 split lanes, one batch of records or more
MERGES = [(False, 3, 700, 16, 2), (False, 16, 8128, 16, 2), (False, 9, 8100, 24, 4), (False, 20, 20000, 16, 2),
          (False, 4, 16000, 16, 2), (False, 1, 20000, 16, 1), (True, 16, 4000, 16, 2), (True, 13, 16000, 16, 1),
          (True, 1, 8128, 16, 2), (True, 8, 8128, 16, 2), (True, 1, 20000, 16, 1)]


def merge_form(f32, nt, pos0, nh, nkv):
    """(split lanes, whether there is more than one batch of records), as the launch chooses them."""
    f = _lib.lib().it_attn_tree_f32kv_scratch_bytes if f32 else _lib.lib().it_attn_tree_scratch_bytes
    smax = f(pos0, nt, 256, nh, nkv) // (nt * nh * RECORD)
    lanes = 16 if smax > 32 and nt * nh <= 192 else 4
    return lanes, smax > 8 * lanes


def test_merge_cases_take_every_form():
    for f32 in (False, True):
        assert {merge_form(*c) for c in MERGES if c[0] == f32} == {(4, False), (4, True), (16, False), (16, True)}
