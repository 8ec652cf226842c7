"""shared_attention where a page among the shared ones is none: its number is read from the group's first row that has a token, and whatever it is, it is not followed."""
import pytest
import torch

from test_gpu_shared_attention import Batch

pytestmark = pytest.mark.gpu
GROUPS = [(3, 13, 50), (4, 12, 40), (2, 9, 30)]


@pytest.mark.parametrize("bad", [-1, "n_pages", 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("at", [0, 4, 8])
@pytest.mark.parametrize("hs", [64, 128])
def test_every_kind_of_number(bad, at, hs):
    for which in range(3):
        b = Batch(41, GROUPS, 8, 1 if hs == 128 else 4, hs)
        begin, end, _ = b.ranges[which]
        b.table[b.slot[begin], at] = b.n_pages if bad == "n_pages" else bad
        y = b.run()
        assert torch.isnan(y[begin:end]).all()
        b.check(y, rows=[m for m in range(b.M) if not begin <= m < end])


@pytest.mark.parametrize("bad", [-1, "n_pages", 2 ** 31 - 1])
def test_the_first_row_with_a_token_tells(bad):
    """A group that begins with rows without a token: the next one's table counts, and theirs and the later ones' are not looked at for what is shared."""
    for none in (0, 1, 2):
        for hit in range(4):
            b = Batch(43, GROUPS, 8, 2, 128)
            begin, end, _ = b.ranges[1]
            for m in range(begin, begin + none):
                b.pos[m] = -1
            b.table[b.slot[begin + hit], 5] = b.n_pages if bad == "n_pages" else bad
            y = b.run()
            live = range(begin + none, end)
            assert (y[begin:begin + none] == 0).all()
            if hit == none:
                assert torch.isnan(y[list(live)]).all()
            else:
                c = Batch(43, GROUPS, 8, 2, 128)                   # (the same without the number, whose rows' values are these ones')
                c.pos = b.pos
                c.check(y, rows=live)
            b.check(y, rows=[m for m in range(b.M) if not begin <= m < end])


@pytest.mark.parametrize("bad", [-1, "n_pages", 2 ** 31 - 1])
def test_a_row_of_its_own_pages(bad):
    """Every place of a row behind the shared pages that its positions reach: that row alone; a place behind them: no row."""
    b = Batch(45, GROUPS, 8, 2, 64)
    for m in (0, 5, 8):
        shared = next(p for begin, end, p in b.ranges if begin <= m < end)
        for k in range(shared, b.pos[m] // 32 + 2):
            c = Batch(45, GROUPS, 8, 2, 64)
            c.table[c.slot[m], k] = c.n_pages if bad == "n_pages" else bad
            y = c.run()
            reached = k <= b.pos[m] // 32
            assert torch.isnan(y[m]).all() == reached
            b.check(y, rows=[r for r in range(b.M) if r != m or not reached])
