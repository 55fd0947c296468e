"""What a page plan says of the pages that it lacks, by every way that a plan takes: d_missing against the plain form and
against the plan's own rows without a slot."""
import numpy as np
import pytest

import test_gpu_long_context as base
from test_page_plan_lacks import lost

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(oracle):
    from oracle import long_context

    return long_context


# tables that are wide enough for several launches, and not
@pytest.mark.parametrize("width", [5, 20000])
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("back", [True, False])
def test_a_shortage_is_told_until_the_page_is_passed(hip, L, width, decode, back):
    """Sequences whose next page is not there for some steps; pages come free in between, and one whose page was begun
    without it has its later tokens dropped, and told, up to the page's end."""
    page, lengths = 16, np.array([16, 11, 0, 32, 79], np.int64)
    S, count = len(lengths), 12
    pages = np.full((S, width), -1, np.int32)
    pages[0, 0], pages[1, 0], pages[3, :2], pages[4, :5] = 0, 1, (2, 3), (4, 5, 6, 7, 8)
    free, free_count = np.array([9, 10, 11] + [-1] * 9, np.int32), 0
    told = []
    for step in range(24):
        new = None if decode else (lengths > 0).astype(np.int32)
        keep = np.where(lengths < 0, -1, 0) if back else None
        got = base.run_plan(L, pages, lengths, new, keep, free, free_count, page, count, S + 2 if new is not None else S)
        assert np.array_equal(got["missing"], lost(got, S, page))
        told.append(list(got["missing"]))
        pages, lengths, free, free_count = got["pages"], got["lengths"], got["free"], int(got["free_count"])
        if step == 9:
            free_count = 2
    told = np.array(told)
    assert (told[:16, 0] == 1).all() and (told[:16, 3] == 1).all()  # (their pages were begun without an entry)
    assert not told[:5, 1].any() and (told[5:21, 1] == 1).all()
    assert not told[:, 2].any()
    # one that comes to the end of a table of five pages, or lacks its sixth
    assert not told[0, 4].any() and (told[1:17, 4] == 1).all()
    # what came free: two pages, for the first two that open one
    assert not told[16:, 0].any() and not told[16:, 3].any()


@pytest.mark.parametrize("S,width,rows", [(7, 6, 300), (7, 12000, 300), (60, 20, 9000), (1500, 4, 4000)])
def test_missing_is_what_the_rows_lack(hip, L, S, width, rows):
    """Gaps, begun pages without an entry, too few pages, tokens past the table's end."""
    rng = np.random.default_rng(S + width)
    lengths = rng.integers(0, 16 * min(width, 8) + 20, S)
    pages, free, count = base.table(rng, lengths, 16, width, rows // 40)
    pages[rng.random(pages.shape) < 0.2] = -1
    keep = np.where(rng.random(S) < 0.1, -1, rng.integers(0, 60, S))
    new = rng.multinomial(rows, np.full(S, 1.0 / S)) * (rng.random(S) < 0.8)
    for k in (None, keep):
        for n in (None, new):
            got = base.run_plan(L, pages, lengths, n, k, free, rows // 40, 16, count, S if n is None else int(n.sum()) + 3)
            assert np.array_equal(got["missing"], lost(got, S, 16))
            assert got["missing"].any() and not got["missing"].all()
            begun = (lengths % 16 != 0) & (pages[np.arange(S), np.minimum(lengths // 16, width - 1)] < 0)
            assert (got["missing"] > 0)[begun & (lengths < 16 * width)].any()


def test_missing_of_lengths_near_the_largest(hip, L):
    pages = np.full((3, 4), -1, np.int32)
    got = base.run_plan(L, pages, [2 ** 31 - 40, 50, 64], [30, 20, 70], None, np.zeros(4, np.int32), 0, 16, 4, 125)
    assert list(got["missing"]) == [3, 2, 5]
