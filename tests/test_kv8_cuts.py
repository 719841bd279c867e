"""When a smaller length alone takes rows back from the 8-bit cache: the rule of it_attn.h (kv8_ref.Cuts) against a model of which
rows stand in the open buffer. No device work."""
import numpy as np
import pytest

from tests.kv8_ref import Cuts


class Open:
    """The open buffer of one sequence: half[p % 2][row of the page] = the row that was written there last, -1 before. A call that
    appends writes its new rows of the last two pages (kv8_append_kernel)."""

    def __init__(self):
        self.half = np.full((2, 64), -1)
        self.rows = 0

    def append(self, n):
        total = self.rows + n
        for p in range(max((total - 1) // 64 - 1, 0), (total - 1) // 64 + 1):
            r = np.arange(max(self.rows, 64 * p), min(total, 64 * p + 64))
            self.half[p % 2][r % 64] = r
        self.rows = total

    def whole(self, to):
        """Whether the rows of the page that is open at length `to` stand in its half."""
        p = to // 64
        return (self.half[p % 2][:to % 64] == 64 * p + np.arange(to % 64)).all()


def test_a_cut_after_a_cut_may_find_its_page_gone():
    """126 rows, four drafts, three of them rejected, then 64 more rows taken back: the drafts stand where page 0 stood."""
    model, cuts = Open(), Cuts()
    for m in (model, cuts):
        m.append(126)
        m.append(4)
    cuts.cut(127)
    model.rows = 127
    assert not model.whole(63) and not cuts.may(63)
    assert model.whole(64) and cuts.may(64) and cuts.may(0)
    for to in range(65, 127):
        assert model.whole(to) and cuts.may(to)


@pytest.mark.parametrize("seed", range(40))
def test_the_rule_never_allows_a_cut_into_rows_that_are_gone(seed):
    rng = np.random.default_rng(seed)
    model, cuts, refused = Open(), Cuts(), 0
    for _ in range(300):
        n = int(rng.choice([1, 2, 4, 31, 63, 64, 65, 127, 200]))
        model.append(n)
        cuts.append(n)
        most = cuts.rows
        for to in range(max(most - 300, 0), most + 1):
            assert not cuts.may(to) or model.whole(to), (most, to)
            refused += not cuts.may(to)
        assert all(cuts.may(to) for to in range(max((most - 1) // 64 - 1, cuts.lowest, 0) * 64, most + 1))
        if rng.integers(2):
            to = int(rng.integers(max(most - int(rng.choice([8, 64, 300])), 0), most + 1))
            if cuts.may(to):
                cuts.cut(to)
                model.rows = to
    assert refused
    assert not cuts.may(cuts.rows + 1) and not cuts.may(-1)
