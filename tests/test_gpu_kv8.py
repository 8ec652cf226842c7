"""The 8-bit token cache against a plain implementation in 64 bits.

What may be off: codes and scales nothing (the same f32 numbers go through the same single roundings; keys are turned in 64 bits on both sides);
values read back half a step of their type; f32 attention what a sum in f32 gives, see ATT_REL; 16-bit outputs half a step more.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 32
# f32 results against 64 bits, relative to the largest magnitude that the row's sum of |weight * value| allows: a score of d products is off by some
# 2^-24 sqrt(d) of its size (up to ~8 in these tests, in units of log2: 12 * 2^-24 * 11 = 8e-6 at most), a weight by as much relatively, the sums by 2^-24 for
# each of ~log(T) steps.  Errors of many weights average out: 2e-6 for rows that see more than one token was the worst that this arithmetic allows on average;
# the bound is the one of a single weight.
ATT_REL = 1e-5
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def K():
    from dllama_b200.ops import kernels
    return kernels


def _table(rng, lens, spare=3):
    """Block table of sequences of these lengths, pages in a random order, and the number of pages."""
    need = [max(1, -(-t // PAGE)) for t in lens]
    perm = rng.permutation(sum(need) + spare).astype(np.int32)
    bt = np.full((len(lens), max(need) + 1), -7, dtype=np.int32)      # places behind a sequence's pages are not to be followed
    at = 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[at:at + n]
        at += n
    return bt, sum(need) + spare


def _cache(rng, n_pages, kv, hs):
    k, v = (torch.from_numpy(rng.integers(-127, 128, (n_pages, kv, PAGE, hs), dtype=np.int8)) for _ in range(2))
    ks, vs = (torch.from_numpy(np.exp(0.4 * rng.standard_normal((n_pages, kv, PAGE))).astype(np.float32) / 64) for _ in range(2))
    return k, v, ks, vs


def _values(codes, scales, bt_row, T):
    """f64 [T][kv][hs] of a sequence."""
    idx = torch.from_numpy(bt_row[:max(1, -(-T // PAGE))].astype(np.int64))
    x = codes[idx].double() * scales[idx].double()[..., None]
    return x.permute(0, 2, 1, 3).reshape(-1, codes.shape[1], codes.shape[3])[:T]


def _attention(q, k, v):
    """f64: q [H][hs] over k, v [T][kv][hs]."""
    H, hs = q.shape
    kv = k.shape[1]
    out = torch.zeros(H, hs, dtype=torch.float64)
    if k.shape[0]:
        s = torch.einsum("ghd,tgd->ght", q.double().view(kv, H // kv, hs), k) / math.sqrt(hs)
        out = torch.einsum("ght,tgd->ghd", torch.softmax(s, -1), v).reshape(H, hs)
    return out


def _dev(*ts):
    return [t.cuda() if isinstance(t, torch.Tensor) else torch.from_numpy(np.asarray(t)).cuda() for t in ts]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _code(x):
    """f32 lines [..., hs] -> (codes, scales) by the format's definition, products in 64 bits."""
    amax = x.abs().amax(-1)
    live = amax >= 2.0 ** -100
    bad = ~torch.isfinite(x).all(-1)
    most = torch.full_like(amax, 127.0)                         # (number / tensor is a reciprocal and a product: two roundings)
    factor = torch.where(live & ~bad, most / amax, torch.zeros_like(amax))
    scale = torch.where(live, amax / most, torch.zeros_like(amax))
    codes = torch.round(torch.nan_to_num(x.double(), 0.0, 0.0, 0.0) * factor.double()[..., None]).to(torch.int8)
    return torch.where(bad[..., None], torch.zeros_like(codes), codes), torch.where(bad, torch.full_like(scale, math.nan), scale)


def _turn(x, pos, freqs):
    a = pos.double()[:, None, None] * freqs.double()
    c, s = torch.cos(a), torch.sin(a)
    x0, x1 = x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), -1).flatten(-2)


# ---------------------------------------------------------------------------------------------------------------
# writing and reading back
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,hs,positions,ld,rope", [
    (32, 8, 128, [192], 0, True),                                       # one token
    (4, 2, 128, [0, 31, 32, 63, 64, -1, 5], 0, True),                   # page borders, a row without a token
    (8, 8, 64, list(range(100, 141)), 8, True),                         # wider rows
    (3, 1, 32, [7, 70000, 131071, 1], 3, True),                         # far positions, three heads, rows that are not aligned
    (5, 5, 32, list(range(33)), 0, False),
    (16, 3, 64, [2, 900], 1, False),
    (1, 1, 128, list(range(700)), 0, True),
])
def test_write_and_read(heads, kv, hs, positions, ld, rope):
    k = K()
    rng = np.random.default_rng(heads * 131 + hs)
    M, seq = len(positions), len(set(positions)) != len(positions) or M_is_scattered(positions)
    slots = list(range(M)) if seq else [0] * M
    lens = [max(p, 0) + 1 for p in positions] if seq else [max(positions) + 1]
    bt, n_pages = _table(rng, lens)
    host = _cache(rng, n_pages, kv, hs)
    width = (heads + 2 * kv) * hs
    wide = torch.from_numpy(rng.standard_normal((M + 2, width + ld)).astype(np.float32) * np.exp(rng.standard_normal((M + 2, 1))).astype(np.float32))
    freqs = torch.from_numpy((500000.0 ** (-np.arange(0, hs, 2) / hs)).astype(np.float32)) if rope else None
    # lines that are not ordinary: zeros, tiny, an infinity, a NaN, one that reaches past fp16
    x = wide[:, :width].view(M + 2, heads + 2 * kv, hs)
    if M > 1:
        x[0, heads + kv] = 0.0
        x[1, heads + kv] = 1e-33
        x[M - 1, heads + kv] *= 1e6
    if M > 4:
        x[2, heads + kv, 3] = math.inf
        x[3, heads, 5] = math.nan
        x[4, heads + kv] = 2.0 ** -100
    cache = k.Kv8Cache(*_dev(*host))
    qkv = wide.cuda()[:, :width]
    q_out = torch.full((M + 1, heads * hs), -5.0, device="cuda")
    where = (_i32(positions), _i32(slots), torch.from_numpy(bt).cuda())
    k.kv8_write(qkv, M, heads, freqs.cuda() if rope else None, *where, q_out, cache)
    pos = torch.tensor(positions)
    rows = x[:M]
    turned = _turn(rows[:, :heads + kv], pos, freqs) if rope else rows[:, :heads + kv].double()
    codes, scales = _code(torch.cat((turned[:, heads:].float(), rows[:, heads + kv:]), 1))
    want = [t.clone() for t in host]
    for m, p in enumerate(positions):
        if p >= 0:
            page = bt[slots[m], p // PAGE]
            want[0][page, :, p % PAGE], want[1][page, :, p % PAGE] = codes[m, :kv], codes[m, kv:]
            want[2][page, :, p % PAGE], want[3][page, :, p % PAGE] = scales[m, :kv], scales[m, kv:]
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):      # what was not written is as it was
        assert torch.equal(got.cpu().view(torch.uint8 if got.dtype == torch.int8 else torch.int32) if not got.is_floating_point() else torch.nan_to_num(got.cpu(), -1.0),
                           w.view(torch.uint8) if not w.is_floating_point() else torch.nan_to_num(w, -1.0))
    live = pos >= 0
    got = q_out[:M].cpu().double()
    ref = turned[:, :heads].reshape(M, -1)
    # f32 products of sines and cosines rounded to f32: three roundings of values below |x0| + |x1|
    size = rows[:, :heads].abs().reshape(M, heads, -1, 2).sum(-1, keepdim=True).expand(-1, -1, -1, 2).reshape(M, -1).double()
    assert ((got - ref).abs() <= 4 * 2.0 ** -24 * size + 1e-30)[live].all()
    assert (got[~live] == -5.0).all() and (q_out[M] == -5.0).all()
    for t in (torch.float32, torch.float16, torch.bfloat16):
        k_out, v_out = (torch.full((M + 1, kv * hs + 5), 9.0, dtype=t, device="cuda")[:, :kv * hs] for _ in range(2))
        k.kv8_read(M, *where, cache, k_out, v_out)
        for o, lo in ((k_out, 0), (v_out, kv)):
            r = codes[:, lo:lo + kv].double() * scales[:, lo:lo + kv].double()[..., None]
            r = torch.where(live[:, None, None], r, torch.zeros_like(r)).reshape(M, -1)
            r16 = r.to(t) if t != torch.float32 else r.float()
            assert torch.equal(torch.nan_to_num(o[:M].cpu(), -1.0), torch.nan_to_num(r16, -1.0))
            assert (o[M] == 9.0).all()


def M_is_scattered(positions):
    return positions != list(range(positions[0], positions[0] + len(positions)))


def test_codes_do_not_depend_on_the_batch():
    """A prompt in one batch, in pieces and row by row: the same bits in the cache."""
    k = K()
    rng = np.random.default_rng(5)
    heads, kv, hs, n = 4, 2, 128, 75
    bt, n_pages = _table(rng, [n])
    qkv = torch.from_numpy(rng.standard_normal((n, (heads + 2 * kv) * hs)).astype(np.float32)).cuda()
    freqs = torch.from_numpy((10000.0 ** (-np.arange(0, hs, 2) / hs)).astype(np.float32)).cuda()
    pos, slot, table = torch.arange(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.from_numpy(bt).cuda()
    held = []
    for cuts in ([0, n], [0, 16, 47, n], list(range(n + 1))):
        cache = k.alloc_kv8(n_pages, kv, hs, "cuda")
        q_out = torch.zeros(n, heads * hs, device="cuda")
        for b, e in zip(cuts, cuts[1:]):
            k.kv8_write(qkv[b:e], e - b, heads, freqs, pos[b:e].clone(), slot[b:e].clone(), table, q_out[b:e], cache)
        held.append((cache.k, cache.v, cache.k_scale, cache.v_scale, q_out))
    for other in held[1:]:
        assert all(torch.equal(a, b) for a, b in zip(held[0], other))


def test_rows_that_the_tables_do_not_hold():
    k = K()
    rng = np.random.default_rng(6)
    heads, kv, hs = 4, 2, 64
    n_pages = 4
    host = _cache(rng, n_pages, kv, hs)
    cache = k.Kv8Cache(*_dev(*host))
    bt = torch.tensor([[1, 4], [0, -3], [2, 3]], dtype=torch.int32, device="cuda")
    positions, slots = [40, 33, 64, 5, 5, 3, 2 ** 31 - 1], [0, 1, 2, 3, -1, 2, 2]      # two bad pages, behind the table, two bad sequences; one good row
    M = len(positions)
    qkv = torch.from_numpy(rng.standard_normal((M, (heads + 2 * kv) * hs)).astype(np.float32)).cuda()
    q_out = torch.zeros(M, heads * hs, device="cuda")
    where = (_i32(positions), _i32(slots), bt)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    k.kv8_write(qkv, M, heads, None, *where, q_out, cache)
    after = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    for a, b in zip(after, before):
        a[2, :, 3] = b[2, :, 3]
        assert torch.equal(a, b)
    k_out, v_out = (torch.zeros(M, kv * hs, device="cuda") for _ in range(2))
    k.kv8_read(M, *where, cache, k_out, v_out)
    good = [m == 5 for m in range(M)]
    for o in (k_out, v_out):
        assert [bool(torch.isfinite(o[m]).all()) for m in range(M)] == good and [bool(torch.isnan(o[m]).all()) for m in range(M)] == [not g for g in good]
    y = torch.zeros(M, heads * hs, device="cuda")
    for splits in (1, 3):
        y.zero_()
        scratch = torch.zeros(k.attention_scratch_bytes(M, heads, hs, splits), dtype=torch.uint8, device="cuda")
        k.kv8_attention(qkv[:, :heads * hs], M, heads, *where, cache, splits, scratch, y_out=y)
        assert [bool(torch.isfinite(y[m]).all()) for m in range(M)] == good and [bool(torch.isnan(y[m]).all()) for m in range(M)] == [not g for g in good]


# ---------------------------------------------------------------------------------------------------------------
# decode rows
# ---------------------------------------------------------------------------------------------------------------
def _decode_case(heads, kv, hs, positions, seed=0, ldq=0):
    rng = np.random.default_rng(seed + heads * 7 + hs)
    M = len(positions)
    bt, n_pages = _table(rng, [max(p, 0) + 1 for p in positions])
    host = _cache(rng, n_pages, kv, hs)
    for m, p in enumerate(positions):                        # what lies behind a sequence's last token is nobody's business
        if p >= 0 and (p + 1) % PAGE:
            page = bt[m, p // PAGE]
            for s in host[2:]:
                s[page, :, (p + 1) % PAGE:] = math.nan
    q = torch.from_numpy(rng.standard_normal((M, heads * hs + ldq)).astype(np.float32))
    ref = torch.stack([_attention(q[m, :heads * hs].view(heads, hs), _values(host[0], host[2], bt[m], p + 1), _values(host[1], host[3], bt[m], p + 1)).reshape(-1)
                       for m, p in enumerate(positions)])
    return bt, host, q, ref


def _near(got, ref, rel):
    got, ref = got.double().cpu(), ref.double()
    big = ref.abs().amax(-1, keepdim=True).clamp_min(1e-30)
    off = ((got - ref).abs() / big).max().item()
    assert off <= rel, off


@pytest.mark.parametrize("heads,kv,hs,positions,splits", [
    (32, 8, 128, [0], 1), (32, 8, 128, [191], 2), (4, 1, 128, [0, 1, 15, 16, 30, 31, 32, 33, 63, 64, 65, -1], 1),
    (8, 4, 32, [0, 5, 31, 32, 100], 1), (8, 8, 64, [63, 64, 65, 700], 2), (16, 2, 128, [300], 8), (16, 1, 128, [129, 1000], 32),
    (64, 8, 64, [1200, 3, 900], 6), (5, 1, 128, [777, 40], 4), (12, 2, 64, [2000], 5), (7, 7, 32, [900, 45], 3), (9, 1, 32, [801], 4),
    (3, 1, 128, [1000 - 1] * 3, 2), (20, 2, 128, [767, 768, 769], 7), (4, 1, 64, [20000], 32),
])
def test_attention(heads, kv, hs, positions, splits):
    k = K()
    M = len(positions)
    bt, host, q, ref = _decode_case(heads, kv, hs, positions)
    cache = k.Kv8Cache(*_dev(*host))
    where = (_i32(positions), _i32(list(range(M))), torch.from_numpy(bt).cuda())
    scratch = torch.zeros(k.attention_scratch_bytes(M, heads, hs, splits), dtype=torch.uint8, device="cuda")
    for t in (torch.float32, torch.float32, torch.bfloat16, torch.float16):          # f32 twice: the counters of the splits go back to zero
        y = torch.full((M + 1, heads * hs), 3.0, dtype=t, device="cuda")
        k.kv8_attention(q.cuda(), M, heads, *where, cache, splits, scratch, y_out=y)
        _near(y[:M], ref, ATT_REL + (STEP[t] if t != torch.float32 else 0.0))
        assert (y[M] == 3.0).all()


@pytest.mark.parametrize("heads,kv,hs,M,long,splits", [
    (4, 2, 64, 2, {1: 5000}, 32), (8, 2, 32, 5, {0: 9000, 4: 2600}, 64), (4, 1, 128, 32, {31: 6000}, 8), (16, 2, 64, 33, {32: 5000, 3: 900}, 16), (2, 1, 32, 70, {5: 12000, 40: 1000, 69: 3000}, 7),
    (4, 4, 32, 100, {7: 4000}, 2), (4, 4, 32, 3, {0: 800, 1: 800, 2: 800}, 16), (8, 8, 64, 3, {0: 16 * 32 * 8 - 1, 1: 255, 2: 768}, 32),
])
def test_attention_of_rows_of_unlike_lengths(heads, kv, hs, M, long, splits):
    """Rows take shares by their part of all pages; some are skipped, one has no token, one is in no table."""
    k = K()
    rng = np.random.default_rng(M)
    positions = [long.get(m, int(rng.integers(0, 70))) for m in range(M)]
    skip = [int(m not in long and rng.random() < 0.3) for m in range(M)]
    if M > 5:
        positions[2], skip[2] = -1, 0
    bt, host, q, ref = _decode_case(heads, kv, hs, positions)
    cache = k.Kv8Cache(*_dev(*host))
    slots = list(range(M))
    nowhere = [m for m in range(M) if M > 5 and m == 6]
    for m in nowhere:
        slots[m], skip[m] = M + 5, 0
    where = (_i32(positions), _i32(slots), torch.from_numpy(bt).cuda())
    scratch = torch.zeros(k.attention_scratch_bytes(M, heads, hs, splits), dtype=torch.uint8, device="cuda")
    live = [m for m in range(M) if not skip[m] and m not in nowhere]
    first = None
    for _ in range(2):                                          # twice: the counters of the splits go back to zero, and the sums' order is always the same
        y = torch.full((M, heads * hs), 3.0, device="cuda")
        k.kv8_attention(q.cuda(), M, heads, *where, cache, splits, scratch, y_out=y, row_skip=_i32(skip))
        _near(y[live], ref[live], ATT_REL)
        assert (y[[m for m in range(M) if skip[m]]] == 3.0).all() and torch.isnan(y[nowhere]).all()
        assert first is None or torch.equal(first[live], y[live])
        first = y
    assert not scratch[:65536].any()


def test_attention_strides_alignment_and_skipped_rows():
    k = K()
    heads, kv, hs, positions = 8, 2, 128, [100, 37, 900, 0]
    M = len(positions)
    bt, host, q, ref = _decode_case(heads, kv, hs, positions, ldq=5)
    cache = k.Kv8Cache(*_dev(*host))
    where = (_i32(positions), _i32(list(range(M))), torch.from_numpy(bt).cuda())
    scratch = torch.zeros(k.attention_scratch_bytes(M, heads, hs, 4), dtype=torch.uint8, device="cuda")
    y = torch.full((M, heads * hs + 3), 3.0, device="cuda")[:, 1:heads * hs + 1]
    skip = _i32([0, 1, 0, 0])
    k.kv8_attention(q.cuda()[:, :heads * hs], M, heads, *where, cache, 4, scratch, y_out=y, row_skip=skip)
    _near(y[[0, 2, 3]], ref[[0, 2, 3]], ATT_REL)
    assert (y[1] == 3.0).all()


def test_attention_of_unusual_numbers():
    """Large and tiny queries and scales, a sink whose value is small, lines of zeros, NaN where it is seen and where it is not."""
    k = K()
    heads, kv, hs = 4, 1, 128
    positions = [400] * 6
    M = len(positions)
    bt, host, q, _ = _decode_case(heads, kv, hs, positions, seed=3)
    q[0] *= 30.0                                   # nearly one-hot weights
    q[1] *= 1e-20                                  # weights alike
    host[3][bt[2, 0], :, 0] = 1e-5                 # a strong token whose value is small
    host[0][bt[2, 0], 0, 0] = 127 * torch.sign(q[2].view(heads, hs).sum(0)).to(torch.int8)
    host[3][bt[3, :5]] = 0.0                       # tokens whose values are zeros
    host[2][bt[4, 3], 0, 7] = math.nan
    host[3][bt[5, 2], 0, 9] = math.nan
    ref = torch.stack([_attention(q[m].view(heads, hs), _values(host[0], host[2], bt[m], 401), _values(host[1], host[3], bt[m], 401)).reshape(-1) for m in range(M)])
    cache = k.Kv8Cache(*_dev(*host))
    where = (_i32(positions), _i32(list(range(M))), torch.from_numpy(bt).cuda())
    y = torch.zeros(M, heads * hs, device="cuda")
    k.kv8_attention(q.cuda(), M, heads, *where, cache, 1, None, y_out=y)
    # scores of row 0 reach 30 times the size: so may the errors of its weights
    _near(y[:1], ref[:1], 30 * ATT_REL)
    _near(y[1:4], ref[1:4], ATT_REL)
    assert torch.isnan(y[4:]).all()
    q[0, 3] = math.inf
    q[1, 130] = math.nan
    k.kv8_attention(q.cuda(), M, heads, *where, cache, 1, None, y_out=y)
    bad = torch.isnan(y.view(M, heads, hs)).all(-1).cpu()
    assert bad[0].tolist() == [True, False, False, False] and bad[1].tolist() == [False, True, False, False]


@pytest.mark.parametrize("heads,hs", [(4, 128), (8, 64), (4, 32)])
def test_attention_into_the_slabs(heads, hs):
    from dllama_b200.ops import quant
    from test_gpu_kernels import _decode_xq
    k = K()
    positions = [70, 900, 3]
    M = len(positions)
    bt, host, q, ref = _decode_case(heads, 2, hs, positions)
    cache = k.Kv8Cache(*_dev(*host))
    where = (_i32(positions), _i32(list(range(M))), torch.from_numpy(bt).cuda())
    scratch = torch.zeros(k.attention_scratch_bytes(M, heads, hs, 3), dtype=torch.uint8, device="cuda")
    xq, y = k.alloc_xq(heads * hs, 8, "cuda"), torch.zeros(M, heads * hs, device="cuda")
    k.kv8_attention(q.cuda(), M, heads, *where, cache, 3, scratch, xq, None, 8, y)
    dq = _decode_xq(xq, heads * hs, 8, M)[0]
    got = y.cpu().numpy()
    np.testing.assert_allclose(dq, quant.q80_roundtrip(got), rtol=0, atol=np.abs(got).max() / 127 * 1.01)      # a code beside a border
    from test_gpu_kernels import _decode_xh
    xh = k.alloc_xh(heads * hs, 16, "cuda")
    k.kv8_attention(q.cuda(), M, heads, *where, cache, 3, scratch, None, xh, 16)
    np.testing.assert_allclose(_decode_xh(xh, heads * hs, 16, M), dq, rtol=2e-3, atol=1e-7)                      # the same codes, times the scale in fp16
    # a prompt chunk's rows take the same places
    n = 20
    bt2 = torch.from_numpy(bt[1:2].copy()).cuda()
    pos, slot, meta = torch.arange(700, 700 + n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), _i32([1, 0, n])
    qp = torch.randn(n, heads * hs, device="cuda")
    xh, y = k.alloc_xh(heads * hs, 32, "cuda"), torch.zeros(n, heads * hs, device="cuda")
    k.kv8_attention_prefill(qp, n, heads, pos, slot, bt2, meta, cache, xh_out=xh, out_mcap=32, y_out=y)
    got = y.cpu().numpy()
    np.testing.assert_allclose(_decode_xh(xh, heads * hs, 32, n), quant.q80_roundtrip(got), rtol=2e-3, atol=np.abs(got).max() / 127 * 1.01)


# ---------------------------------------------------------------------------------------------------------------
# prompt chunks
# ---------------------------------------------------------------------------------------------------------------
# 16-bit operands of the products: queries and weights rounded to 11 bits (2^-11 of a score of size ~6, of a weight), errors of hundreds of weights
# average out, those of a row that sees few tokens do not: 6 * 2^-11 + 2^-11
PROMPT_REL = 4e-3


@pytest.mark.parametrize("heads,kv,hs,segs", [
    (4, 1, 128, [(0, 0, 16)]), (8, 2, 128, [(0, 37, 100)]), (4, 4, 64, [(3, 5, 70)]), (2, 1, 128, [(62, 200, 130)]), (2, 2, 64, [(31, 31, 33)]),
    (4, 2, 128, [(2, 10, 40), (45, 0, 90)]), (8, 8, 128, [(0, 0, 700)]), (16, 1, 128, [(5, 900, 300)]), (8, 2, 128, [(0, 0, 257), (260, 130, 384)]),
    (5, 1, 128, [(1, 77, 900)]), (16, 1, 64, [(0, 3, 50)]), (6, 2, 32, [(1, 60, 45)]), (5, 1, 128, [(0, 100, 17), (20, 0, 1)]), (32, 8, 128, [(0, 1000, 100)]), (8, 1, 64, [(0, 2500, 31)]),
    (32, 8, 64, [(0, 10, 230)]), (5, 1, 64, [(1, 77, 1450)]), (8, 8, 64, [(0, 100, 930)]), (16, 2, 64, [(0, 0, 257), (260, 130, 200)]),
    # (few rows behind many tokens: several CTAs for an item)
    (16, 2, 128, [(0, 2500, 260), (300, 40, 100)]), (8, 8, 128, [(3, 2600, 530)]), (5, 1, 64, [(0, 3000, 1440)]), (4, 1, 128, [(1, 9000, 1100)]), (32, 8, 64, [(0, 5000, 129), (130, 2100, 120)]),
])
def test_attention_prefill(heads, kv, hs, segs):
    k = K()
    rng = np.random.default_rng(heads + hs)
    M = max(b + n for b, _, n in segs) + 2
    bt, n_pages = _table(rng, [p0 + n for _, p0, n in segs])
    host = _cache(rng, n_pages, kv, hs)
    positions, slots, meta, covered = [0] * M, [0] * M, [len(segs)], np.zeros(M, dtype=bool)
    for i, (b, p0, n) in enumerate(segs):
        if (p0 + n) % PAGE:
            for s in host[2:]:
                s[bt[i, (p0 + n) // PAGE], :, (p0 + n) % PAGE:] = math.nan
        positions[b:b + n], slots[b:b + n], covered[b:b + n] = range(p0, p0 + n), [i] * n, True
        meta += [b, b + n]
    q = torch.from_numpy(rng.standard_normal((M, heads * hs)).astype(np.float32))
    cache = k.Kv8Cache(*_dev(*host))
    where = (_i32(positions), _i32(slots), torch.from_numpy(bt).cuda())
    meta = _i32(meta + [0] * 8)
    work = k.kv8_prefill_workspace(n_pages, kv, hs, M, "cuda")
    ref = torch.zeros(M, heads * hs, dtype=torch.float64)
    for i, (b, p0, n) in enumerate(segs):
        kk, vv = _values(host[0], host[2], bt[i], p0 + n), _values(host[1], host[3], bt[i], p0 + n)
        for m in range(b, b + n):
            ref[m] = _attention(q[m].view(heads, hs), kk[:positions[m] + 1], vv[:positions[m] + 1]).reshape(-1)
    for w in ((work, None) if work is not None else (None,)):
        for t in (torch.float32, torch.bfloat16, torch.float16):
            y = torch.full((M, heads * hs), 7.0, dtype=t, device="cuda")
            k.kv8_attention_prefill(q.cuda(), M, heads, *where, meta, cache, workspace=w, y_out=y)
            _near(y[covered], ref[covered], PROMPT_REL + STEP[t])
            assert (y[~covered] == 7.0).all()                     # rows outside the segments are left alone


@pytest.mark.parametrize("heads,kv,hs,rows,context", [(16, 4, 128, 300, 700), (5, 5, 128, 830, 2600), (40, 8, 64, 200, 1500), (32, 8, 64, 250, 2500)])
def test_attention_prefill_into_the_cast_for_the_next_matmul(heads, kv, hs, rows, context):
    from dllama_b200.ops import quant
    from test_gpu_kernels import _decode_xh, _decode_xq
    k = K()
    rng = np.random.default_rng(rows)
    M, mcap = rows + 1, (rows + 8) // 8 * 8
    bt, n_pages = _table(rng, [context + rows])
    cache = k.Kv8Cache(*_dev(*_cache(rng, n_pages, kv, hs)))
    where = (_i32([0] + list(range(context, context + rows))), _i32([0] * M), torch.from_numpy(bt).cuda())
    q = torch.from_numpy(rng.standard_normal((M, heads * hs)).astype(np.float32)).cuda()
    assert k.kv8_widens(M, heads, hs)
    work = k.kv8_prefill_workspace(n_pages, kv, hs, M, "cuda")
    xq, xh, y = k.alloc_xq(heads * hs, mcap, "cuda"), k.alloc_xh(heads * hs, mcap, "cuda"), torch.zeros(M, heads * hs, device="cuda")
    k.kv8_attention_prefill(q, M, heads, *where, _i32([1, 1, M]), cache, work, xq, xh, mcap, y)
    got = y.cpu().numpy()[1:]
    dq = _decode_xq(xq, heads * hs, mcap, M)[0][1:]
    np.testing.assert_allclose(dq, quant.q80_roundtrip(got), rtol=0, atol=np.abs(got).max() / 127 * 1.01)          # a code beside a border
    np.testing.assert_allclose(_decode_xh(xh, heads * hs, mcap, M)[1:], dq, rtol=2e-3, atol=1e-7)
    assert not _decode_xq(xq, heads * hs, mcap, M)[0][0].any()                                                      # the row outside the segment


@pytest.mark.parametrize("workspace", [False, True])
def test_attention_prefill_looks_at_the_segments_that_are_there(workspace):
    """meta that promises more than its tensor holds: the segments that it holds are taken, what lies behind is not read."""
    k = K()
    rng = np.random.default_rng(3)
    heads, kv, hs, M = 32, 8, 128, 150
    bt, n_pages = _table(rng, [M])
    cache = k.Kv8Cache(*_dev(*_cache(rng, n_pages, kv, hs)))
    where = (_i32(list(range(M))), _i32([0] * M), torch.from_numpy(bt).cuda())
    q = torch.from_numpy(rng.standard_normal((M, heads * hs)).astype(np.float32)).cuda()
    work = k.kv8_prefill_workspace(n_pages, kv, hs, M, "cuda") if workspace else None
    holds = _i32([8, 0, 100, 100, 140, 140, 150])
    y, ref = torch.full((M, heads * hs), 7.0, device="cuda"), torch.full((M, heads * hs), 7.0, device="cuda")
    k.kv8_attention_prefill(q, M, heads, *where, holds[:5], cache, work, y_out=y)
    k.kv8_attention_prefill(q, M, heads, *where, _i32([2, 0, 100, 100, 140]), cache, work, y_out=ref)
    assert torch.equal(y, ref) and (y[140:] == 7.0).all() and not (y[:140] == 7.0).any()


@pytest.mark.parametrize("workspace,hs", [(False, 128), (True, 128), (False, 64), (True, 64)])
def test_attention_prefill_of_unusual_lines(workspace, hs):
    """A line with a NaN is seen by the rows from its token on, and by no other; a segment of a sequence, a position or a page that is not there is NaN;
    one without tokens gives zeros."""
    k = K()
    rng = np.random.default_rng(8)
    heads, kv = (16, 8) if hs == 128 else (32, 16)
    segs = [(0, 100, 60, 0), (60, 0, 40, 1), (100, 30, 20, 9), (120, 200, 30, 2), (150, -40, 20, 1), (170, 0, 33, 3), (203, 5, 50, 4)]      # begin, position, rows, sequence
    M = 260
    assert k.kv8_widens(M, heads, hs)                           # the widened pages, where there is a workspace
    bt, n_pages = _table(rng, [160, 40, 220, 33, 55])
    bt = bt[:, :7]                                              # the fourth segment ends behind the table: 7 pages are 224 tokens
    bt[3, 1] = n_pages                                          # a page that is not there
    host = _cache(rng, n_pages, kv, hs)
    host[2][bt[0, 4], 1, 2] = math.nan                          # token 130, keys of the second head
    host[3][bt[1, 0], 0, 20] = math.nan                         # token 20, values of the first one
    positions, slots, meta = [0] * M, [0] * M, [len(segs)]
    for b, p0, n, s in segs:
        positions[b:b + n], slots[b:b + n] = range(p0, p0 + n), [s] * n
        meta += [b, b + n]
    q = torch.from_numpy(rng.standard_normal((M, heads * hs)).astype(np.float32))
    cache = k.Kv8Cache(*_dev(*host))
    where = (_i32(positions), _i32(slots), torch.from_numpy(bt.copy()).cuda())
    y = torch.full((M, heads * hs), 7.0, device="cuda")
    k.kv8_attention_prefill(q.cuda(), M, heads, *where, _i32(meta), cache, workspace=k.kv8_prefill_workspace(n_pages, kv, hs, M, "cuda") if workspace else None, y_out=y)
    y = y.cpu().view(M, heads, hs)
    nan = torch.isnan(y)
    assert nan[30:60, 2:4].all() and not nan[:60, :2].any() and not nan[:60, 4:].any() and not nan[:30].any()
    assert nan[80:100, :2].all() and not nan[60:100, 2:].any() and not nan[60:80].any()
    assert nan[100:150].all() and (y[150:170] == 0).all()
    assert nan[202].all() and (y[253:] == 7.0).all()
    for b, p0, n, s in (segs[0], segs[1], segs[6]):
        kk, vv = _values(host[0], host[2], bt[s], p0 + n), _values(host[1], host[3], bt[s], p0 + n)
        kk, vv = torch.nan_to_num(kk), torch.nan_to_num(vv)
        for m in range(b, b + n):
            ref = _attention(q[m].view(heads, hs), kk[:positions[m] + 1], vv[:positions[m] + 1])
            for h in range(heads):
                if not nan[m, h].any():
                    _near(y[m, h], ref[h], PROMPT_REL)


# ---------------------------------------------------------------------------------------------------------------
# together, as they are used
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,hs", [(8, 2, 128), (16, 8, 64), (4, 2, 32)])
def test_a_conversation(heads, kv, hs):
    """A prompt in two chunks, tokens one by one beside another user's: what attention gives is the formula on what the cache reads back."""
    k = K()
    g = torch.Generator(device="cuda")
    g.manual_seed(hs)
    rng = np.random.default_rng(hs)
    n, n_pages = 90, 12
    bt = torch.from_numpy(rng.permutation(n_pages).astype(np.int32).reshape(2, 6)).cuda()
    cache, freqs = k.alloc_kv8(n_pages, kv, hs, "cuda"), torch.from_numpy((10000.0 ** (-np.arange(0, hs, 2) / hs)).astype(np.float32)).cuda()
    scratch = torch.zeros(k.attention_scratch_bytes(2, heads, hs, 2), dtype=torch.uint8, device="cuda")
    seen = {}                                                    # rotated queries and outputs by (sequence, position)

    def step(positions, slots, chunk):
        M = len(positions)
        qkv = torch.randn(M, (heads + 2 * kv) * hs, generator=g, device="cuda")
        q, y = torch.zeros(M, heads * hs, device="cuda"), torch.zeros(M, heads * hs, device="cuda")
        where = (_i32(positions), _i32(slots), bt)
        k.kv8_write(qkv, M, heads, freqs, *where, q, cache)
        if chunk:
            k.kv8_attention_prefill(q, M, heads, *where, _i32([1, 0, M]), cache, y_out=y)
        else:
            k.kv8_attention(q, M, heads, *where, cache, 2, scratch, y_out=y)
        for m, at in enumerate(zip(slots, positions)):
            seen[at] = (q[m].cpu(), y[m].cpu(), chunk)

    step(list(range(50)), [0] * 50, True)
    step(list(range(50, n)), [0] * (n - 50), True)
    step(list(range(17)), [1] * 17, True)
    for i in range(40):
        step([n + i, 17 + i], [0, 1], False)
    lens = [n + 40, 57]
    for s, T in enumerate(lens):
        pos, slot = torch.arange(T, dtype=torch.int32, device="cuda"), torch.full((T,), s, dtype=torch.int32, device="cuda")
        kk, vv = (torch.zeros(T, kv * hs, device="cuda") for _ in range(2))
        k.kv8_read(T, pos, slot, bt, cache, kk, vv)
        kk, vv = (x.double().cpu().view(T, kv, hs) for x in (kk, vv))
        for p in range(T):
            q, y, chunk = seen[s, p]
            _near(y[None], _attention(q.view(heads, hs), kk[:p + 1], vv[:p + 1]).reshape(1, -1), PROMPT_REL if chunk else ATT_REL)


def test_captured_replayed_and_on_other_streams():
    """Two graphs with scratches of their own, replayed side by side on two streams, then again on new inputs; and eager calls on a side stream."""
    k = K()
    heads, kv, hs, positions, splits = 16, 2, 128, [1500, 40, 901], 6
    M = len(positions)
    bt, host, q, ref = _decode_case(heads, kv, hs, positions)
    cache = k.Kv8Cache(*_dev(*host))
    where = (_i32(positions), _i32(list(range(M))), torch.from_numpy(bt).cuda())
    streams, graphs, qs, ys = [torch.cuda.Stream() for _ in range(2)], [], [], []
    torch.cuda.synchronize()
    for st in streams:
        qs.append(torch.zeros(M, heads * hs, device="cuda"))
        ys.append(torch.zeros(M, heads * hs, device="cuda"))
        scratch = torch.zeros(k.attention_scratch_bytes(M, heads, hs, splits), dtype=torch.uint8, device="cuda")
        with torch.cuda.stream(st):
            st.wait_stream(torch.cuda.default_stream())
            k.kv8_attention(qs[-1], M, heads, *where, cache, splits, scratch, y_out=ys[-1])       # (functions are loaded ahead of the capture)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            for _ in range(4):
                k.kv8_attention(qs[-1], M, heads, *where, cache, splits, scratch, y_out=ys[-1])
        graphs.append(graph)
    for f in (1.0, -0.5):
        for t in qs:
            t.copy_(q.cuda() * f)
        want = ref if f == 1.0 else torch.stack([_attention(f * q[m].view(heads, hs), _values(host[0], host[2], bt[m], p + 1), _values(host[1], host[3], bt[m], p + 1)).reshape(-1) for m, p in enumerate(positions)])
        torch.cuda.synchronize()
        for _ in range(3):
            for st, graph in zip(streams, graphs):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ys[0], ys[1])
        _near(ys[0], want, ATT_REL)
    st = streams[0]
    with torch.cuda.stream(st):
        kk, vv = (torch.zeros(M, kv * hs, dtype=torch.float16, device="cuda") for _ in range(2))
        k.kv8_read(M, *where, cache, kk, vv)
    st.synchronize()
    for m, p in enumerate(positions):
        assert torch.equal(kk[m].cpu().view(kv, hs), _values(host[0], host[2], bt[m], p + 1)[p].half())


def test_far_pages_of_a_large_cache():
    """Lines beyond 2^31 bytes of codes."""
    k = K()
    free, _ = torch.cuda.mem_get_info()
    n_pages, kv, hs = 70000, 8, 128                              # 2.3 GB of codes of the keys, as many of the values
    if free < 8 << 30:
        pytest.skip("8 GB of device memory")
    heads, T = 8, 100
    cache = k.alloc_kv8(n_pages, kv, hs, "cuda")
    bt = torch.tensor([[n_pages - 1, 5, n_pages - 2, n_pages - 7]], dtype=torch.int32, device="cuda")
    pos, slot = torch.arange(T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    qkv = torch.randn(T, (heads + 2 * kv) * hs, device="cuda")
    q, y = torch.zeros(T, heads * hs, device="cuda"), torch.zeros(1, heads * hs, device="cuda")
    k.kv8_write(qkv, T, heads, None, pos, slot, bt, q, cache)
    codes, scales = _code(qkv.cpu().view(T, -1, hs)[:, heads:])
    held = (codes.double() * scales.double()[..., None])
    kk, vv = (torch.zeros(T, kv * hs, device="cuda") for _ in range(2))
    k.kv8_read(T, pos, slot, bt, cache, kk, vv)
    assert torch.equal(kk.cpu().view(T, kv, hs), held[:, :kv].float()) and torch.equal(vv.cpu().view(T, kv, hs), held[:, kv:].float())
    k.kv8_attention(q[T - 1:], 1, heads, pos[T - 1:], slot[:1], bt, cache, 1, None, y_out=y)
    _near(y, _attention(q[T - 1].cpu().view(heads, hs), held[:, :kv], held[:, kv:]).reshape(1, -1), ATT_REL)
    n = 20
    yp = torch.zeros(n, heads * hs, device="cuda")
    k.kv8_attention_prefill(q[T - n:], n, heads, pos[T - n:], slot[:n], bt, _i32([1, 0, n]), cache, y_out=yp)
    for m in range(n):
        _near(yp[m:m + 1], _attention(q[T - n + m].cpu().view(heads, hs), held[:T - n + m + 1, :kv], held[:T - n + m + 1, kv:]).reshape(1, -1), PROMPT_REL)
