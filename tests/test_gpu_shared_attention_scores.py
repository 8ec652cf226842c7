"""shared_attention where scores are very large: finite queries and keys give finite rows, the largest score's value where it stands alone and the mean of those that are equal.

Scores are sums in f32: of 128 products each exact in f32, they are off by at most 2^-16 of sum |q k| (127 additions of half a step, 2^-24, and as much again for terms cut off inside an MMA).  The
largest score here is at least three quarters of that sum above every other one (where scores grow, half a percent), and in the log2 domain some 2^10 or more above it, so that all other weights are 0 and
a row is the value of its largest score.  What multiplies that value is the weight in fp16, what it is divided by the weight in f32, from the polynomial for some: off by 2^-11 and 8e-5 of the value.
Where n scores are equal they are so bit for bit (the same operands in the same places of one kind of MMA: all of them stand among the shared pages, or all behind them), and all weights are: the
same 2^-11 and 8e-5 of the mean of |v|.  2^-20 beside it for the sums."""
import pytest
import torch

from test_gpu_shared_attention import PAGE, Batch

pytestmark = pytest.mark.gpu
OFF = 2.0 ** -11 + 8e-5 + 2.0 ** -20


def _lines(b, m):
    """Where the keys of a row stand: pages and places of its positions."""
    t = torch.arange(b.pos[m] + 1)
    return b.table[b.slot[m]][t // PAGE].cuda(), (t % PAGE).cuda()


def _large(seed, groups, heads, kv, hs, size, sign):
    """Keys that are all one random direction times a factor: some places of the shared pages and of each row's own have `sign` times the largest factor, the other ones a quarter of it or less.  Queries
    point along the direction, each head with a length of its own."""
    b = Batch(seed, groups, heads, kv, hs)
    g = torch.Generator(device="cuda").manual_seed(seed)
    way = torch.randn(kv, 1, hs, generator=g, device="cuda")
    factor = 0.25 * (2 * torch.rand(b.n_pages, kv, PAGE, 1, generator=g, device="cuda") - 1)
    b.k = (factor * size * way).half()
    length = torch.exp(torch.rand(b.M, heads, 1, generator=g, device="cuda"))
    b.q = (sign * size * length * way.repeat_interleave(heads // kv, 0).transpose(0, 1)).reshape(b.M, heads * hs).contiguous()
    b.way = way
    return b


SHAPES = [([(40, 20, 60)], 8, 2, 128), ([(9, 33, 40), (30, 7, 90), (1, 0, 50)], 16, 4, 64), ([(3, 16, 60)], 32, 8, 128), ([(70, 25, 50)], 8, 1, 128)]


@pytest.mark.parametrize("size", [40.0, 700.0, 2000.0, 9000.0])
@pytest.mark.parametrize("groups,heads,kv,hs", SHAPES)
def test_the_largest_score_alone(groups, heads, kv, hs, size):
    """In the shared part, in a row's own, early and late."""
    for seed, where in enumerate(("shared", "own", "first", "last")):
        b = _large(seed + 1, groups, heads, kv, hs, size, 1)
        want = torch.empty(b.M, kv, hs, dtype=torch.float64, device="cuda")
        for begin, end, pages in b.ranges:
            gen = torch.Generator().manual_seed(seed + begin)
            at = int(torch.randint(0, max(1, pages * PAGE), (1,), generator=gen)) if where != "first" else 0
            for m in range(begin, end):
                page, place = _lines(b, m)
                t = {"shared": at, "first": 0, "last": b.pos[m], "own": int(torch.randint(pages * PAGE, b.pos[m] + 1, (1,), generator=gen))}[where]
                t = min(t, b.pos[m])
                b.k[page[t], :, place[t]] = (size * b.way)[:, 0].half()
                want[m] = b.v[page[t], :, place[t]].double()
        y = b.run().double().view(b.M, kv, heads // kv, hs)
        assert torch.isfinite(y).all()
        assert ((y - want[:, :, None]).abs() <= OFF * want[:, :, None].abs()).all()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [700.0, 9000.0])
@pytest.mark.parametrize("groups,heads,kv,hs", SHAPES)
def test_scores_that_are_all_the_same(groups, heads, kv, hs, size, sign):
    b = _large(9, groups, heads, kv, hs, size, sign)
    b.k = (size * b.way).half()[None].expand(b.n_pages, kv, PAGE, hs).contiguous()
    for begin, end, pages in b.ranges:                           # a row's own keys, where its group has some: far below
        for m in range(begin, end if pages else begin):
            page, place = _lines(b, m)
            b.k[page[pages * PAGE:], :, place[pages * PAGE:]] = 0 if sign > 0 else (1.5 * size * b.way)[:, 0].half()
    y = b.run().double().view(b.M, kv, heads // kv, hs)
    for begin, end, pages in b.ranges:
        for m in range(begin, end):
            page, place = _lines(b, m)
            n = pages * PAGE if pages else len(page)
            v = b.v[page[:n], :, place[:n]].double()
            assert ((y[m] - v.mean(0)[:, None]).abs() <= OFF * v.abs().mean(0)[:, None]).all()


def test_scores_that_grow_from_small_to_very_large():
    """A row whose scores are small for the first pages and very large for later ones, and the other way round: the value of the largest."""
    for order in (1, -1):
        b = _large(21, [(20, 60, 40)], 8, 2, 128, 1.0, 1)
        lead = b.table[b.slot[0]][:60]
        factor = torch.exp2(torch.linspace(-6, 11, 60 * PAGE))
        if order < 0:
            factor = factor.flip(0)
        b.k = torch.zeros_like(b.k)
        b.k[lead.cuda()] = (factor.view(60, 1, PAGE, 1).cuda() * b.way).half()
        b.q *= 2000
        y = b.run().double().view(b.M, 2, 4, 128)
        t = 60 * PAGE - 1 if order > 0 else 0
        want = b.v[lead[t // PAGE], :, t % PAGE].double()
        assert ((y - want[None, :, None]).abs() <= OFF * want[None, :, None].abs()).all()


@pytest.mark.parametrize("hs", [64, 128])
def test_scores_beyond_f32(hs):
    """A row with a score that f32 does not hold is NaN, whichever part of the positions has it and whatever its sign is where there are no others; its neighbours keep their values."""
    b = Batch(31, [(6, 12, 60), (2, 0, 40)], 8, 2, hs)
    q = b.q.view(b.M, 8, hs)
    q[2], q[7] = torch.sign(q[2]) * 3e38, torch.sign(q[7]) * 3e38
    y = b.run().view(b.M, 8, hs)
    for m in range(b.M):
        page, place = _lines(b, m)
        s = torch.matmul(q[m].double().view(2, 4, hs), b.k[page, :, place].double().permute(1, 2, 0)) * 1.4426950408889634 / hs ** 0.5
        beyond = (s > 3.5e38).any(-1).flatten() | (s < -3.5e38).all(-1).flatten()
        assert beyond.all() == (m in (2, 7)) and torch.isnan(y[m]).all(-1)[beyond].all()
    b.check(y.reshape(b.M, -1), rows=[0, 1, 3, 4, 5, 6])
