"""shared_attention against the formula in 64 bits.

What may be off: queries and softmax weights are rounded to fp16 (uniform errors of up to half a step, 2^-11 of the value: standard deviation 2^-11 / sqrt 3), a quarter of the weights come from a
polynomial that is off by 8e-5.  A score is then off by a standard deviation of at most s = 2^-11 / sqrt 3 * sqrt(sum q^2 k^2) / sqrt(d), which both the weights and their sum follow: an output
sum w_t v_t by s sqrt(sum w_t^2 (v_t - y)^2).  The sum of the weights is that of the ones in f32, what multiplies the values are the rounded ones: an error r_t of a weight, relative to it, adds
sum w_t r_t v_t, and nothing of it cancels however close the values are to y (two tokens of the same value v: y = v (1 + (r_1 + r_2) / 2), although every v_t - y is 0): r sqrt(sum w_t^2 v_t^2)
with r = sqrt(2^-22 / 3 + 8e-5^2).  EIGHT of both together, beside 2^-20 of sum w |v| for the sums in f32 and half a step of the output's type.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE = 32
EIGHT = 8.0
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def K():
    from dllama_b200.ops import kernels
    return kernels


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int64), dtype=torch.int32).cuda()


class Batch:
    """groups: (rows, shared pages, tokens of their own at most); their rows lie one behind the other."""

    def __init__(self, seed, groups, heads, kv, hs, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv, self.hs = heads, kv, hs
        self.pos, self.ranges = [], []
        for rows, pages, own in groups:
            b = len(self.pos)
            self.pos += [pages * PAGE + int(x) for x in torch.randint(0, own, (rows,), generator=g)]
            self.ranges.append((b, b + rows, pages))
        M = self.M = len(self.pos)
        need = [p // PAGE + 1 for p in self.pos]
        self.n_pages = sum(need) - sum((e - b - 1) * p for b, e, p in self.ranges) + spare
        perm = torch.randperm(self.n_pages, generator=g)
        self.slot = torch.randperm(M, generator=g).tolist()
        self.table = torch.full((M, max(need) + 1), -7, dtype=torch.int64)       # places behind a sequence's pages are not to be followed
        at = 0
        for b, e, p in self.ranges:
            lead = perm[at:at + p]
            at += p
            for m in range(b, e):
                row = self.table[self.slot[m]]
                row[:p] = lead
                row[p:need[m]] = perm[at:at + need[m] - p]
                at += need[m] - p
        gc = torch.Generator(device="cuda").manual_seed(seed)
        shape = (self.n_pages, kv, PAGE, hs)
        self.k = (torch.randn(shape, generator=gc, device="cuda") * torch.exp(0.5 * torch.randn(kv, 1, hs, generator=gc, device="cuda"))).half()
        self.v = (torch.randn(shape, generator=gc, device="cuda") * torch.exp(0.3 * torch.randn(self.n_pages, kv, PAGE, 1, generator=gc, device="cuda"))).half()
        self.q = torch.randn(M, heads * hs, generator=gc, device="cuda")
        self.meta = [len(self.ranges)] + [x for r in self.ranges for x in r]

    def run(self, dtype=torch.float32, y=None, meta=None, q=None, **kw):
        k = K()
        work = k.shared_attention_workspace(self.M, self.heads, self.kv, self.hs, "cuda")
        work.fill_(255)                                            # whatever it holds before: NaN
        if y is None:
            y = torch.full((self.M, self.heads * self.hs), 77.0, device="cuda", dtype=dtype)
        k.shared_attention(self.q if q is None else q, self.M, self.heads, i32(self.pos), i32(self.slot), i32(self.table.numpy()), i32(self.meta if meta is None else meta), self.k, self.v, work,
                           y_out=y, **kw)
        return y

    def want(self, m, q=None):
        """f64 output of a row, and what it may be off by."""
        p = self.pos[m]
        q = (self.q if q is None else q)[m].double().view(self.kv, -1, self.hs)
        pages = self.table[self.slot[m]][:p // PAGE + 1].cuda()
        k, v = (x[pages].double().transpose(0, 1).flatten(1, 2)[:, :p + 1] for x in (self.k, self.v))
        w = torch.softmax(torch.matmul(q, k.transpose(1, 2)) / math.sqrt(self.hs), -1)
        y = torch.matmul(w, v)
        s = 2.0 ** -11 / math.sqrt(3) * torch.matmul(q ** 2, k.transpose(1, 2) ** 2).amax(-1, keepdim=True).sqrt() / math.sqrt(self.hs)
        squares = torch.matmul(w ** 2, v ** 2)
        spread = (squares - 2 * y * torch.matmul(w ** 2, v) + (w ** 2).sum(-1, keepdim=True) * y ** 2).clamp(min=0)
        off = torch.sqrt(s ** 2 * spread + (2.0 ** -22 / 3 + 8e-5 ** 2) * squares)
        return y.reshape(-1), (EIGHT * off + 2.0 ** -20 * torch.matmul(w, v.abs())).reshape(-1)

    def check(self, y, rows=None, q=None):
        for m in range(self.M) if rows is None else rows:
            want, off = self.want(m, q)
            got = y[m].double()
            worst = ((got - want).abs() - off - STEP[y.dtype] * want.abs()).max()
            assert worst <= 0, (m, float(worst), float((got - want).abs().max()), float(off.max()))


CASES = [
    ([(3, 16, 60)], 32, 8, 128), ([(1, 5, 40)], 32, 8, 128), ([(2, 1, 1)], 4, 4, 128), ([(7, 3, 33), (5, 4, 70)], 32, 8, 64), ([(32, 25, 100)], 32, 8, 128), ([(33, 130, 40)], 32, 8, 128),
    ([(70, 9, 50)], 64, 8, 64), ([(4, 40, 900), (1, 0, 500), (9, 6, 20)], 16, 8, 128), ([(11, 300, 300)], 8, 2, 128), ([(40, 17, 64)], 16, 1, 128), ([(40, 17, 64)], 16, 1, 64), ([(5, 7, 10)], 6, 2, 64),
    ([(70, 9, 50)], 128, 8, 64), ([(60, 5, 40)], 128, 8, 128), ([(23, 4, 40)], 18, 2, 128), ([(230, 4, 40)], 18, 2, 64),
    ([(130, 30, 45)], 8, 1, 128), ([(2, 2, 5)] * 8, 8, 4, 64), ([(9, 0, 200)], 32, 8, 128), ([(20, 64, 32), (20, 65, 32), (20, 66, 32), (20, 67, 32)], 16, 8, 64), ([(300, 12, 40)], 32, 8, 128),
]


@pytest.mark.parametrize("groups,heads,kv,hs", CASES)
def test_rows_of_groups(groups, heads, kv, hs):
    b = Batch(len(groups) * 100 + heads, groups, heads, kv, hs)
    b.check(b.run())
    b.check(b.run(torch.bfloat16), rows=range(0, b.M, 3))
    b.check(b.run(torch.float16, pdl=True), rows=range(0, b.M, 5))


def test_it_is_what_attention_gives():
    k = K()
    b = Batch(3, [(6, 20, 100), (3, 30, 50)], 32, 8, 128)
    y, ya = b.run(), torch.zeros(b.M, b.heads * b.hs, device="cuda")
    table = b.table.clamp(min=0)
    k.attention(b.q, b.M, b.heads, b.kv, b.hs, b.k, b.v, i32(b.pos), i32(b.slot), i32(table.numpy()), table.shape[1], 1, None, None, None, 0, y_out=ya)
    b.check(ya)
    assert (y - ya).abs().max() < 2e-3


def test_lists_of_groups_that_are_not_in_order():
    """Groups that overlap, that end behind the rows, more than eight, none, fewer than said: the answers are the same."""
    b = Batch(5, [(6, 20, 100), (5, 9, 50), (4, 13, 30)], 32, 8, 64)
    full = b.meta
    for meta in ([0], [3], full[:7], [2] + full[1:], [100] + full[1:], [-3] + full[1:], [3, 0, 6, 20, 3, 11, 9, 11, 15, 13], [2, 6, 11, 9, 0, 6, 20], [1, 11, 4000, 13], [1, -5, 6, 20], [1, 3, 3, 4],
                 [1, 6, 2, 4], [10] + [0, 0, 9] * 8 + [0, 6, 20], [1, 0, 6, -4], [1, 1, 4, 3]):
        b.check(b.run(meta=meta))


def test_rows_that_do_not_see_all_of_the_shared_pages():
    """A row that ends inside of what is shared, at its end, one without a token: zeros there, the others as they should be."""
    b = Batch(7, [(6, 20, 100)], 32, 8, 128)
    for ends in ((5 * 32 + 3,), (20 * 32 - 1,), (20 * 32,), (-1,), (0,), (31,), (-1, 40), (-9, -9, -9, -9, -9), (-1,) * 6):
        c = Batch(7, [(6, 20, 100)], 32, 8, 128)
        c.pos[:len(ends)] = ends
        y = c.run()
        c.check(y, rows=[m for m in range(6) if c.pos[m] >= 0])
        for m in range(6):
            if c.pos[m] < 0:
                assert (y[m] == 0).all()
    assert b.M == 6


@pytest.mark.parametrize("hs", [64, 128])
def test_what_lies_behind_the_ends_is_not_looked_at(hs):
    """NaN and infinities in places that no row sees: behind the last token of a page, behind the last shared page of a step, in pages of nobody."""
    b = Batch(9, [(6, 21, 100), (3, 2, 40), (2, 0, 5)], 16, 4, hs)
    seen = torch.zeros(b.n_pages, PAGE, dtype=torch.bool)
    for m, p in enumerate(b.pos):
        t = torch.arange(p + 1)
        seen[b.table[b.slot[m]][t // PAGE], t % PAGE] = True
    for bad in (math.nan, math.inf, -math.inf):
        for x in (b.k, b.v):
            x.transpose(1, 2)[~seen.cuda()] = bad
        b.check(b.run())
        b.check(b.run(meta=[0]))


def test_what_is_not_finite_reaches_the_rows_that_see_it():
    for bad in (math.nan, math.inf):
        b = Batch(11, [(5, 6, 50), (4, 9, 50)], 16, 4, 128)
        b.v[b.table[b.slot[0]][3], :, 7, 5] = bad                  # of the first group's pages
        b.v[b.table[b.slot[6]][9], :, 0, 9] = bad                  # of row 6 alone
        y = b.run().view(9, 16, 128)
        for m in range(9):
            hit = torch.zeros(128, dtype=torch.bool)
            hit[5], hit[9] = m < 5, m == 6
            assert (~torch.isfinite(y[m])).any(0).cpu().equal(hit) and (~torch.isfinite(y[m][:, hit])).all()
        b = Batch(11, [(5, 6, 50), (4, 9, 50)], 16, 4, 128)
        b.k[b.table[b.slot[0]][3], 1, 7, 5] = math.nan             # a key of one key/value head
        y = b.run().view(9, 16, 128)
        assert torch.isnan(y[:5, 4:8]).all() and torch.isfinite(y[:5, :4]).all() and torch.isfinite(y[:5, 8:]).all() and torch.isfinite(y[5:]).all()


@pytest.mark.parametrize("hs", [64, 128])
def test_queries_of_any_size(hs):
    b = Batch(13, [(9, 10, 60)], 8, 2, hs)
    q = b.q.clone()
    for m, f in enumerate([1e-3, 1e3, 0.0, 1e-20, 3e4, 30.0, 1.0, 1e-38]):
        q[m] *= f
    c = Batch(13, [(9, 10, 60)], 8, 2, hs)
    c.k *= 0.01
    y = c.run(q=q)
    c.check(y, q=q)
    q[3, 5], q[5, hs + 1], q[7, 0] = math.nan, math.inf, -math.inf
    y = c.run(q=q).view(9, 8, hs)
    bad = torch.isnan(y).all(-1).cpu()
    want = torch.zeros(9, 8, dtype=torch.bool)
    want[3, 0] = want[5, 1] = want[7, 0] = True
    assert bad.equal(want)
    keep = [m for m in range(9) if m not in (3, 5, 7)]
    c.check(y.reshape(9, -1), rows=keep, q=q)


def test_scores_far_apart():
    """Maxima that grow from step to step and pieces whose weights vanish beside others'."""
    b = Batch(15, [(40, 120, 60)], 8, 2, 128)
    ramp = torch.linspace(0, 3, b.n_pages, device="cuda")[torch.argsort(torch.randperm(b.n_pages, generator=torch.Generator().manual_seed(1))).cuda()]
    b.k = (b.k.float() * ramp[:, None, None, None]).half()
    b.q *= 3
    b.check(b.run())


@pytest.mark.parametrize("what", ["page", "own_page", "slot", "position"])
def test_what_is_not_in_the_tables_is_not_followed(what):
    b = Batch(17, [(5, 12, 50), (4, 9, 50)], 16, 4, 64)
    hit = []
    if what == "page":
        for m in range(5):
            b.table[b.slot[m], 7] = b.n_pages if m % 2 == 0 else b.n_pages
        hit = range(5)
    if what == "own_page":
        b.table[b.slot[2], 12] = -1
        hit = [2]
    if what == "slot":
        b.slot[0] = b.M
        hit = [0]
    if what == "position":
        b.pos[8] = b.table.shape[1] * PAGE
        hit = [8]
    y = b.run()
    for m in range(b.M):
        if m in hit:
            assert torch.isnan(y[m]).all()
    b.check(y, rows=[m for m in range(b.M) if m not in hit])


@pytest.mark.parametrize("pages", [5, 9, 13, 21])
def test_a_page_that_is_none_stays_in_its_group(pages):
    """Shares of the work that end in one group and begin the next one: what is wrong in one reaches no row of another."""
    for which in range(3):
        b = Batch(18, [(3, pages, 50), (4, 12, 40), (2, pages, 30)], 8, 1, 128)
        first = sum((3, 4, 2)[:which])
        hit = range(first, first + (3, 4, 2)[which])
        for m in hit:
            b.table[b.slot[m], 4] = b.n_pages
        y = b.run()
        assert torch.isnan(y[list(hit)]).all()
        b.check(y, rows=[m for m in range(9) if m not in hit])


def test_strides_and_rows_behind():
    b = Batch(19, [(6, 8, 40)], 16, 4, 128)
    wide = torch.zeros(9, 16 * 128 + 12, device="cuda")
    wide[:6, 4:4 + 2048] = b.q
    out = torch.full((9, 16 * 128 + 5), 5.0, device="cuda", dtype=torch.bfloat16)
    K().shared_attention(wide[:, 4:4 + 2048], 6, 16, i32(b.pos), i32(b.slot), i32(b.table.numpy()), i32(b.meta), b.k, b.v, K().shared_attention_workspace(6, 16, 4, 128, "cuda"), y_out=out[:, 3:3 + 2048])
    b.check(out[:6, 3:3 + 2048].contiguous())
    out[:6, 3:3 + 2048] = 5
    assert (out == 5).all()


@pytest.mark.parametrize("hs", [64, 128])
def test_into_the_slabs(hs):
    from test_gpu_kernels import _decode_xh, _decode_xq
    from dllama_b200.ops import quant
    k = K()
    b = Batch(21, [(5, 8, 40)], 16, 4, hs)
    xq, xh = k.alloc_xq(16 * hs, 8, "cuda"), k.alloc_xh(16 * hs, 8, "cuda")
    y = b.run(xq_out=xq, xh_out=xh, out_mcap=8)
    b.check(y)
    dq = _decode_xq(xq, 16 * hs, 8, 5)[0]
    np.testing.assert_array_equal(dq, quant.q80_roundtrip(y.cpu().numpy()))
    np.testing.assert_allclose(_decode_xh(xh, 16 * hs, 8, 5), dq, rtol=2e-3, atol=1e-7)


def test_pages_beyond_32_bits():
    """A cache of more than 4 GB of keys: the pages in use lie at its end."""
    b = Batch(23, [(6, 40, 90)], 32, 8, 128)
    far = 4 * 2 ** 30 // (8 * PAGE * 128 * 2) + 4000
    for x in ("k", "v"):
        big = torch.zeros(far + b.n_pages, 8, PAGE, 128, dtype=torch.float16, device="cuda")
        big[far:] = getattr(b, x)
        setattr(b, x, big)
    b.table = torch.where(b.table >= 0, b.table + far, b.table)
    b.check(b.run())


def test_two_graphs_at_once_on_new_rows():
    """Each with a workspace of its own; queries, positions and groups change between replays."""
    k = K()
    batches = [Batch(25 + i, [(12, 30 + 9 * i, 60), (7, 11, 40)], 32, 8, 128) for i in range(2)]
    runs = []
    for b in batches:
        t = [b.q, i32(b.pos), i32(b.slot), i32(b.table.numpy()), i32(b.meta)]
        work, y = k.shared_attention_workspace(b.M, 32, 8, 128, "cuda"), torch.zeros(b.M, 4096, device="cuda")
        call = lambda pdl, t=t, b=b, work=work, y=y: k.shared_attention(t[0], b.M, 32, t[1], t[2], t[3], t[4], b.k, b.v, work, y_out=y, pdl=pdl)
        call(False)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(False)
            call(True)
            call(True)
        runs.append((t, y, s, g, work))                            # (a graph does not keep its tensors alive)
    for turn in range(3):
        for b, (t, y, s, g, _) in zip(batches, runs):
            b.q = torch.randn(b.M, 4096, generator=torch.Generator(device="cuda").manual_seed(turn), device="cuda")
            b.pos = [max(0, p - 3 * turn) for p in b.pos]
            meta = b.meta if turn != 1 else [1] + b.meta[4:7] + [0, 0, 0]
            t[0].copy_(b.q)
            t[1].copy_(i32(b.pos))
            t[4].copy_(i32(meta))
        torch.cuda.synchronize()
        for t, y, s, g, _ in runs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for b, (t, y, s, g, _) in zip(batches, runs):
            b.check(y, rows=range(0, b.M, 4))
