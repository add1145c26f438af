"""What the AdamW step's library refuses of a table, asked before anything is launched."""
from array import array

import pytest

from superfloat.python_b200 import _lib, build
from superfloat.python_b200._errors import SFShapeError

A = 1 << 20                                    # addresses that no launch ever sees
GOOD = [A, 2 * A, 3 * A, 4 * A, 0, 0, 1000, 0]
OTHER = [5 * A, 6 * A, 7 * A, 8 * A, 0, 0, 1000, 0]


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()
    return _lib.load()


def check(*rows, dtype=0, sf8=0):
    words = array("q", [w for r in rows for w in r])
    _lib.adamw_check(words.buffer_info()[0], len(rows), dtype, sf8)


def test_good_tables():
    check()
    check(GOOD)
    check(GOOD, OTHER)
    check(GOOD, [5 * A, 2 * A] + OTHER[2:])                          # a gradient may be shared
    check(GOOD, GOOD[:6] + [0, 0])                                   # no elements, no place in memory
    check(GOOD[:4] + [9 * A, 10 * A, 1000, 0], sf8=1)


@pytest.mark.parametrize("rows,kw", [
    ([GOOD, GOOD], {}), ([GOOD, [A + 3996] + OTHER[1:]], {}), ([GOOD, OTHER[:2] + [A + 3996] + OTHER[3:]], {}),
    ([GOOD], dict(dtype=1)), ([GOOD], dict(sf8=1)), ([[0] + GOOD[1:]], {}), ([[A + 2] + GOOD[1:]], {}),
    ([GOOD[:6] + [-1, 0]], {}), ([GOOD[:4] + [9 * A, 9 * A + 12, 1000, 0]], dict(sf8=1)),
    ([GOOD, [A + 1998] + OTHER[1:]], dict(dtype=2))])
def test_refusals(rows, kw):
    with pytest.raises(SFShapeError):
        check(*rows, **kw)
