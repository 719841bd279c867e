"""Refusals of the tree calls beside those of single arguments: host code only."""
import pytest

from irontimber_amd import _lib

F = 1 << 20      # an aligned address that is never followed


@pytest.mark.parametrize("name", ["it_kv_tree_commit_f16", "it_kv_tree_commit_f32"])
def test_one_cache_for_both_is_refused(name):
    """Both caches' rows are moved at once: one cache given twice would be read while it is overwritten."""
    assert getattr(_lib.lib(), name)(F, F, 512, 9, 5, F, 2, None) != 0
    assert "two caches" in _lib.last_error()
