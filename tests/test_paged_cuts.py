"""Cuts of a sequence in a cache without room, on the CPU."""
import re

import pytest

from test_paged import Quiet, check, rows


def test_a_cut_without_room_for_its_copy_says_which_comes_first():
    c = Quiet(1, 1, 1, max_tokens=64 * 6)  # 2 blocks, 6 pages of 16 bits
    a = c.add()
    c.step(a, 64 * 4 + 63)
    (d,) = c.fork(a)
    for length in (10, 70, 200):
        before = (c.accounting(), c.pages(d))
        with pytest.raises(ValueError, match='full') as e:
            c.truncate(d, length)
        first = int(re.search(r'cut to (\d+) first', str(e.value)).group(1))
        assert first == -(-length // 64) * 64 and (c.accounting(), c.pages(d)) == before
    c.truncate(d, 64)
    c.truncate(d, 10)
    assert rows(c, d) == [10] and c.pages(d)[0][2] == 1 and c.length(a) == 64 * 4 + 63
    check(c, [a, d])


def test_a_page_that_is_not_full_in_the_middle():
    """The end of such a page that others hold would be copied too: a cut behind it comes first, if there is one."""
    c = Quiet(1, 1, 1, max_tokens=64 * 6)
    a = c.add()
    c.step(a, 30, 16)
    c.step(a, 64 * 5, 8)  # the other block
    (d,) = c.fork(a)
    e = c.add()
    c.step(e, 64, 16)
    c.step(e, 64, 16)  # the first block is full
    with pytest.raises(ValueError, match=r'full') as error:
        c.truncate(d, 10)
    assert 'cut to 94 first' in str(error.value)
    c.truncate(d, 94)  # shared pages: nothing is free yet
    with pytest.raises(ValueError, match='full'):
        c.truncate(d, 10)
    c.truncate(a, 94)
    with pytest.raises(ValueError, match='full'):
        c.truncate(d, 10)
    c.free(e)
    c.truncate(d, 10)
    assert rows(c, d) == [10] and rows(c, a) == [30, 64]
    check(c, [a, d])


def test_the_last_page_alone():
    c = Quiet(1, 1, 1, max_tokens=64 * 3)
    a = c.add()
    c.step(a, 64 * 3)
    (d,) = c.fork(a)
    with pytest.raises(ValueError, match='full') as error:
        c.truncate(d, 180)
    assert 'others hold)' in str(error.value) and c.length(d) == 192
    c.truncate(d, 128)
    check(c, [a, d])
