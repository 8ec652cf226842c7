"""sample_tokens against the definition in 64 bits.

Tokens are whole numbers and have to be equal: the kernel's weights are off by 2^-29 of themselves at most and its sums exact, so a coin falls on another side of a border
between two tokens with a chance of some 2^-29 sqrt(vocabulary) < 1e-6 a row.  Probabilities: one rounding to f32 (2^-24) and 2^-29 of the total.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
PROB_REL = 2.0 ** -23


def K():
    from dllama_b200.ops import kernels
    return kernels


def oracle(x, t, k, p, min_p, u):
    """Token and probability of one row (f64)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64)) + 0.0
    m = x.max()
    if m == -np.inf:
        return 0, 0.0
    if not t > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == m, 1.0, np.exp(np.where(x == m, 0.0, x - m) / np.float64(t)))
    w = np.where(x == -np.inf, 0.0, w)
    order = np.argsort(-x, kind="stable")
    n = k if 0 < k < len(x) else len(x)
    sums = np.cumsum(w[order[:n]])
    if 0 < p < 1:
        n = min(n, int((sums - w[order[:n]] < np.float64(p) * sums[-1]).sum()))
    if min_p > 0:
        n = min(n, max(1, int((w >= min(np.float64(min_p), 1.0)).sum())))
    left = np.sort(order[:n])
    sums = np.cumsum(w[left])
    i = min(int(np.searchsorted(sums, np.float64(u) * sums[-1], side="right")), n - 1)
    while w[left[i]] == 0:                         # (a coin of one: the last that has a weight)
        i -= 1
    return int(left[i]), w[left[i]] / sums[-1]


def check(logits, t, k, p, min_p, u, M=None):
    M = logits.shape[0] if M is None else M
    n = len(t)
    dev = lambda v, d: None if v is None else torch.tensor(v, dtype=d, device="cuda")
    tokens, prob = torch.full((n + 1,), -9, dtype=torch.int32, device="cuda"), torch.full((n + 1,), -9.0, device="cuda")
    K().sample_tokens(logits, M, dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(min_p, torch.float32), dev(u, torch.float32), tokens, prob)
    x = logits.float().cpu().numpy()
    f32 = lambda v: [0.0] * n if v is None else np.asarray(v, np.float32)
    want = [oracle(x[m], f32(t)[m], 0 if k is None else k[m], f32(p)[m], f32(min_p)[m], f32(u)[m]) for m in range(M)]
    assert tokens[:M].tolist() == [w[0] for w in want]
    got = prob[:M].double().cpu().numpy()
    for g, (_, w) in zip(got, want):
        assert abs(g - w) <= PROB_REL * w + 2.0 ** -40
    assert (tokens[M:] == -9).all() and (prob[M:] == -9).all()      # what lies behind is as it was
    return tokens[:M]


def settings(rng, n):
    on = rng.random((4, n)) < 0.6
    return (np.where(rng.random(n) < 0.1, 0.0, rng.uniform(0.3, 2.0, n)).tolist(), (rng.integers(1, 300, n) * on[0]).tolist(), (rng.uniform(0.3, 0.999, n) * on[1]).tolist(),
            (rng.uniform(0.001, 0.4, n) * on[2]).tolist(), rng.random(n).astype(np.float32).tolist())


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 511, 4096, 4097, 8193, 32003, 50001, 128256, 327680, 524288])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_of_every_size(vocab, dtype):
    rng = np.random.default_rng(vocab)
    M = 37 if vocab < 100000 else 9
    x = rng.standard_normal((M, vocab)) * rng.uniform(0.5, 5, (M, 1))
    x[:, rng.integers(0, vocab, 20)] += rng.uniform(0, 12, 20)
    check(torch.from_numpy(x).to(dtype).cuda(), *settings(rng, M))


@pytest.mark.parametrize("vocab", [33, 5000, 128256])
def test_equal_logits(vocab):
    """Ties: the lowest indexes stay."""
    rng = np.random.default_rng(3)
    flat = np.full((8, vocab), 1.25)
    levels = rng.integers(-2, 3, (8, vocab)).astype(np.float64)
    levels[:, ::7] *= -0.0                                     # zeros of both signs are equal
    k = [1, 2, 17, vocab // 2, vocab - 1, vocab, vocab + 5, 0]
    for x in (flat, levels):
        for p in (None, [0.5, 0.9, 0.1, 0.3, 0.99, 1e-6, 0.25, 0.75]):
            check(torch.from_numpy(x).float().cuda(), [1.0, 0.7, 1.3, 1.0, 2.0, 1.0, 0.5, 1.0], k, p, None, rng.random(8).astype(np.float32).tolist())


def test_a_border_among_many_that_are_close():
    """More tokens in one bin than the list holds, all different."""
    rng = np.random.default_rng(5)
    x = 3 + rng.standard_normal((6, 100000)) * np.array([[1e-3], [1e-4], [1e-5], [1e-6], [0.2], [30.0]])
    check(torch.from_numpy(x).float().cuda(), [1.0] * 6, [40000, 0, 70000, 99999, 60000, 50000], [0.0, 0.5, 0.9, 0.2, 0.999, 0.99999], None, [0.1, 0.5, 0.999, 0.7, 0.3, 0.9])


def test_coins_and_settings_at_their_ends():
    rng = np.random.default_rng(7)
    x = rng.standard_normal((16, 2000)) * 3
    inf = math.inf
    t = [1e-30, 1e-45, 1e30, inf, 1e-3, 1.0, 1.0, 1.0, -1.0, math.nan, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0]
    k = [0, 5, 0, 0, 3, 1, 0, 0, 0, 0, -4, 2 ** 31 - 1, 50, 50, 0, 0]
    p = [0.9, 0.9, 0.5, 0.0, 0.9, 0.9, 1e-30, 1.0 - 2.0 ** -24, 0.5, 0.5, 1.5, -1.0, math.nan, 0.5, 0.0, 0.9]
    min_p = [0.0, 0.1, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.1, 0.0, 1.0, 7.0, 0.1, -1.0, math.nan, 1e-30]
    top = 1.0 - 2.0 ** -24
    u = [0.0, top, 0.5, 0.25, 0.0, top, 0.3, top, 0.5, 0.5, 0.5, 0.9, 0.5, 0.0, 2.0 ** -24, top]
    check(torch.from_numpy(x).float().cuda(), t, k, p, min_p, u)


def test_masked_tokens_and_what_is_not_finite():
    rng = np.random.default_rng(9)
    x = rng.standard_normal((9, 6000)) * 2
    inf = math.inf
    x[0, :5990] = -inf                                         # a mask that leaves ten
    x[1] = -inf                                                # ... nothing
    x[2, 100:] = -3.4e38                                       # masked by the type's lowest value
    x[3, [7, 4000]] = inf                                      # two that are infinite
    x[4, ::3] = math.nan
    x[5] = math.nan
    x[6, 5999], x[6, :5999] = -2.0, -inf                        # one token, the last one
    x[7] = 3.3e38
    x[7, 11] = 3.4e38
    x[8, 0], x[8, 1:] = 3e38, -3e38
    for k, p in (([0] * 9, None), ([20] * 9, [0.9] * 9), ([0] * 9, [0.6] * 9), ([5500] * 9, None)):
        check(torch.from_numpy(x).float().cuda(), [0.8] * 9, k, p, [0.05] * 9 if p else None, rng.random(9).astype(np.float32).tolist())
    check(torch.from_numpy(x).float().cuda(), [0.0] * 9, None, None, None, [0.5] * 9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_do_not_lie_side_by_side(dtype):
    rng = np.random.default_rng(11)
    wide = torch.from_numpy(rng.standard_normal((20, 2, 3001))).to(dtype).cuda()
    s = settings(rng, 20)
    check(wide[:, 1, 3:], *s)
    check(wide[:, 0, 1:], *[v[:7] for v in s], M=6)             # fewer rows than there are
    one = wide[3:4, 1, 5:]
    check(one, *[v[:1] for v in s])


def test_the_distribution():
    """Coins spread evenly give each token as often as its probability says."""
    n = 4096
    x = torch.tensor([0.0, 1.0, 2.0, 3.0, -1.0]).cuda().repeat(n, 1)
    u = ((torch.arange(n) + 0.5) / n).tolist()
    t = check(x, [1.0] * n, [4] * n, [0.99] * n, None, u)
    w = torch.exp(torch.tensor([0.0, 1.0, 2.0, 3.0, -math.inf], dtype=torch.float64))
    count = torch.bincount(t.cpu().long(), minlength=5).double()
    assert (count - n * w / w.sum()).abs().max() <= 1


def test_captured_and_replayed_and_beside_itself():
    """Two graphs at once on streams of their own, new coins in between."""
    k = K()
    rng = np.random.default_rng(13)
    x = torch.from_numpy(rng.standard_normal((24, 32000)) * 3).float().cuda()
    t, kk, p, mp, u = settings(rng, 24)
    args = [torch.tensor(v, dtype=d, device="cuda") for v, d in ((t, torch.float32), (kk, torch.int32), (p, torch.float32), (mp, torch.float32), (u, torch.float32))]
    sets = []
    for _ in range(2):
        a = [v.clone() for v in args]
        out = torch.zeros(24, dtype=torch.int32, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        k.sample_tokens(x, 24, *a, out)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            k.sample_tokens(x, 24, *a, out, pdl=True)
            k.sample_tokens(x, 24, *a, out, pdl=True)
        sets.append((a, out, s, g))
    for i in range(3):
        coins = [torch.from_numpy(rng.random(24).astype(np.float32)).cuda() for _ in sets]
        torch.cuda.synchronize()
        for (a, out, s, g), c in zip(sets, coins):
            with torch.cuda.stream(s):
                a[4].copy_(c)
                g.replay()
        torch.cuda.synchronize()
        xs = x.cpu().numpy()
        for (a, out, s, g), c in zip(sets, coins):
            cc = c.cpu().numpy()
            f = [v.cpu().numpy() for v in a]
            assert out.tolist() == [oracle(xs[m], f[0][m], f[1][m], f[2][m], f[3][m], cc[m])[0] for m in range(24)]


@pytest.mark.parametrize("left", [3, 200, 5000, 9000])
def test_rows_of_which_a_mask_leaves_few(left):
    """A grammar's mask over a large vocabulary: as many tokens as the list takes, and more; k below, at and above what is left."""
    rng = np.random.default_rng(left)
    x = np.full((8, 50000), -np.inf)
    for m in range(8):
        x[m, rng.choice(50000, left, replace=False)] = rng.standard_normal(left) * 3
    check(torch.from_numpy(x).float().cuda(), [0.8] * 8, [1, left - 1, left, left + 1, 40, 2000, 49999, 7], [0.0, 0.9, 0.5, 0.99, 0.0, 0.9, 0.3, 0.0], [0.0, 0.0, 0.1, 0.0] * 2, rng.random(8).astype(np.float32).tolist())


@pytest.mark.parametrize("order", [1, -1])
def test_sorted_rows(order):
    """The best tokens all in one place: the partial maxima say little."""
    rng = np.random.default_rng(21)
    x = np.sort(rng.standard_normal((9, 128256)) * 3, 1)[:, ::order].copy()
    check(torch.from_numpy(x).float().cuda(), [0.7, 1.0, 1.3] * 3, [50, 0, 300, 0, 1, 20, 0, 3000, 100000], [0.9, 0.95, 0.0, 0.5, 0.9, 0.99, 0.999, 0.9, 0.8], [0.0, 0.0, 0.05] * 3,
          rng.random(9).astype(np.float32).tolist())


def test_rows_with_large_nuclei_in_16_bits():
    """Nuclei of tens of thousands of tokens, whose logits have a few hundred values."""
    rng = np.random.default_rng(22)
    x = torch.from_numpy(rng.standard_normal((12, 128256)) * np.array([[0.3], [1.0], [2.2]] * 4)).cuda()
    for dtype in (torch.bfloat16, torch.float16):
        check(x.to(dtype), [1.0, 1.3, 0.7] * 4, [0] * 12, [0.9, 0.99, 0.999, 0.5] * 3, [0.0] * 9 + [0.01] * 3, rng.random(12).astype(np.float32).tolist())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_some_heavy_tokens_ahead_of_a_long_tail(dtype):
    """Borders among the heavy tokens, at the weight from which they count as such, and far behind them; rows in which all tokens are heavy."""
    rng = np.random.default_rng(31)
    x = rng.standard_normal((48, 128256)) * 2.2
    for m in range(48):
        x[m, rng.integers(0, 128256, 64)] += 6 + 8 * rng.random(64) ** 3
    x[:4] *= 0.2
    t = np.concatenate([[1.0, 5.0, 20.0, 0.3], rng.uniform(0.5, 1.4, 44)]).tolist()
    p = np.concatenate([[0.9, 0.5, 0.99, 0.95], 1 - 10 ** rng.uniform(-4, -0.3, 44)]).tolist()
    check(torch.from_numpy(x).to(dtype).cuda(), t, None, p, None, rng.random(48).astype(np.float32).tolist())
    check(torch.from_numpy(x[:5]).to(dtype).cuda(), t[:5], None, p[:5], [0.0, 0.01, 0.0, 0.0, 1e-4], rng.random(5).astype(np.float32).tolist())


@pytest.mark.parametrize("rows", [1, 3, 40, 160])
def test_as_many_tokens_as_there_are_partial_maxima(rows):
    """k at the numbers of groups whose maxima bound the list, and beside them, for clusters of every size."""
    rng = np.random.default_rng(rows)
    ks = sorted({b + d for n in (1, 3) for b in (n * 2 ** e for e in range(3, 13)) for d in (-1, 0, 1)})
    x = rng.standard_normal((rows, 33000)) * 2
    x[:, ::50] += 4
    logits = torch.from_numpy(x).to(torch.bfloat16).cuda()
    for i in range(0, len(ks), rows) if rows < 40 else [0]:
        k = (ks[i:] + ks)[:rows] if rows < 40 else (ks * (rows // len(ks) + 1))[:rows]
        check(logits, [0.9] * rows, k, [0.95] * rows, None, rng.random(rows).astype(np.float32).tolist())
