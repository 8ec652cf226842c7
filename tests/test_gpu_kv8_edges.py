"""The 8-bit token cache where lines are not ordinary: NaN lines at every place of a step, queries beyond fp16, weights of very
unlike sizes, scores beyond f32, pages beyond 2^32 bytes, calls in graphs side by side, lines read back beside queued work, users of unlike lengths.

Tolerances are those of test_gpu_kv8.py, which derives them.
"""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv8 import ATT_REL, K, PAGE, PROMPT_REL, _attention, _cache, _code, _dev, _i32, _near, _table, _values

pytestmark = pytest.mark.gpu


class _Prompt:
    """One segment of `rows` rows behind `context` tokens, `wide` pages more in the block table."""

    def __init__(self, heads, kv, hs, rows, context, seed=0, wide=0):
        rng = np.random.default_rng(seed + heads * 3 + hs + context)
        self.heads, self.kv, self.hs, self.rows, self.context = heads, kv, hs, rows, context
        bt, self.n_pages = _table(rng, [context + rows])
        self.bt = np.concatenate((bt, np.full((1, wide), -7, dtype=np.int32)), 1) if wide else bt
        self.host = _cache(rng, self.n_pages, kv, hs)
        self.q = torch.from_numpy(rng.standard_normal((rows, heads * hs)).astype(np.float32))

    def at(self, t):
        """Page and place of token t."""
        return int(self.bt[0, t // PAGE]), t % PAGE

    def run(self, workspace, dtype=torch.float32):
        k = K()
        if workspace:
            assert k.kv8_widens(self.rows, self.heads, self.hs)
        cache = k.Kv8Cache(*_dev(*self.host))
        where = (_i32(list(range(self.context, self.context + self.rows))), _i32([0] * self.rows), torch.from_numpy(self.bt).cuda())
        work = k.kv8_prefill_workspace(self.n_pages, self.kv, self.hs, self.rows, "cuda") if workspace else None
        y = torch.full((self.rows, self.heads * self.hs), 7.0, dtype=dtype, device="cuda")
        k.kv8_attention_prefill(self.q.cuda(), self.rows, self.heads, *where, _i32([1, 0, self.rows]), cache, workspace=work, y_out=y)
        return y.cpu().view(self.rows, self.heads, self.hs)

    def ref(self, m):
        """f64 [heads][hs] of row m."""
        T = self.context + m + 1
        return _attention(self.q[m].view(self.heads, self.hs), _values(self.host[0], self.host[2], self.bt[0], T), _values(self.host[1], self.host[3], self.bt[0], T))


@pytest.mark.parametrize("workspace", [False, True])
@pytest.mark.parametrize("heads,kv,hs,rows,context,wide,first", [
    (16, 8, 128, 300, 200, 0, 8), (16, 8, 128, 300, 200, 0, 136), (16, 8, 128, 300, 200, 0, 304), (16, 8, 128, 300, 200, 0, 488),
    (16, 8, 128, 300, 200, 60, 304),                                     # tables that may hold long sequences
    (16, 8, 128, 260, 2600, 0, 1400), (16, 8, 128, 260, 2600, 0, 2736),    # steps that go to several CTAs
    (8, 8, 128, 530, 0, 0, 264),                                         # heads that come alone: two tiles of rows side by side
    (32, 8, 64, 300, 200, 0, 8), (32, 8, 64, 300, 200, 60, 304), (32, 8, 64, 240, 3000, 0, 1704), (8, 8, 64, 930, 100, 0, 520),
])
def test_a_nan_line_is_seen_wherever_it_stands(heads, kv, hs, rows, context, wide, first, workspace):
    """Eight neighbouring tokens from `first` on, one for each key/value head: key of the even ones, value of the odd ones."""
    p = _Prompt(heads, kv, hs, rows, context, wide=wide)
    for h in range(kv):
        page, place = p.at(first + h)
        p.host[2 + h % 2][page, h, place] = math.nan
    nan = torch.isnan(p.run(workspace))
    sees = torch.tensor([[context + m >= first + h // (heads // kv) for h in range(heads)] for m in range(rows)])
    assert torch.equal(nan.all(-1), sees) and torch.equal(nan.any(-1), sees)


@pytest.mark.parametrize("workspace", [False, True])
@pytest.mark.parametrize("heads,kv,hs,rows,context", [(16, 4, 128, 300, 0), (16, 4, 128, 300, 90), (16, 8, 128, 260, 2600), (32, 8, 64, 240, 0), (32, 8, 64, 240, 3000), (8, 8, 64, 930, 0)])
def test_prompt_queries_beyond_fp16(heads, kv, hs, rows, context, workspace):
    """Finite ones count as they are, whatever their size beside the row's others; an infinity or a NaN makes the row of its head NaN, and no other."""
    p = _Prompt(heads, kv, hs, rows, context)
    p.host[0][..., 5] = 0                                          # a channel that no key has: queries may be large there
    q = p.q.view(rows, heads, hs)
    large = {0: 1e5, 1: -7e4, 33: 65519.0, 64: -3e6, 131: 4e5, rows - 1: 65536.0}
    for m, x in large.items():
        q[m, :, 5] = x
    q[2, 0, 5], q[40, 3, 7], q[rows - 2, 1, hs - 1], q[130, 2, 0] = math.inf, math.nan, -math.inf, math.inf
    y = p.run(workspace)
    bad = torch.zeros(rows, heads, dtype=torch.bool)
    bad[2, 0] = bad[40, 3] = bad[rows - 2, 1] = bad[130, 2] = True
    nan = torch.isnan(y)
    assert torch.equal(nan.all(-1), bad) and torch.equal(nan.any(-1), bad)
    for m in sorted(set(large) | {3, 32, 41, 129, rows - 3}):
        if workspace or m not in large:                            # (without one queries have 16 bits of the largest of them: the others are lost beside it here)
            _near(y[m].reshape(1, -1), p.ref(m).reshape(1, -1), PROMPT_REL)


@pytest.mark.parametrize("size", [2e5, 1e6, 4e6])                # scores of -3e6, -1.6e7, -6e7 in the log2 domain
@pytest.mark.parametrize("heads,kv,hs,rows", [(16, 4, 128, 300), (32, 8, 64, 240)])
def test_first_rows_of_large_queries(heads, kv, hs, rows, size):
    """One token is seen: its value, however far below zero its score is."""
    p = _Prompt(heads, kv, hs, rows, 0)
    q = p.q.view(rows, heads, hs)
    page, place = p.at(0)
    for h in range(heads):
        q[0, h] = -size * torch.sign(p.host[0][page, h // (heads // kv), place].float())
    for workspace in (False, True):
        _near(p.run(workspace)[0].reshape(1, -1), p.ref(0).reshape(1, -1), PROMPT_REL)


@pytest.mark.parametrize("heads,kv,hs", [(4, 1, 128), (8, 2, 64), (4, 2, 32)])
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 26, 2.0 ** 40, 2.0 ** 100])
def test_prompt_values_of_very_unlike_sizes(heads, kv, hs, size):
    """Early tokens whose values are huge and whose weights vanish beside those of later ones: what counts are the later ones' values, to the last digit."""
    p = _Prompt(heads, kv, hs, 40, 500)
    p.q = 1.0 + 0.1 * p.q                                          # queries of about one direction
    low = -(math.log(size) + 45.0)                                 # scores: the early weights are size * e^low = e^-45 of the others
    page = int(p.bt[0, 0])
    p.host[0][page], p.host[2][page] = -127, -low / math.sqrt(hs) / 127
    p.host[3][page] *= size
    page = int(p.bt[0, 4])                                         # (this one too: less low, less huge)
    p.host[0][page], p.host[2][page] = -127, 30.0 / math.sqrt(hs) / 127
    p.host[3][page] *= 2.0 ** 10
    y = p.run(False)
    for m in (0, 1, 17, 39):
        _near(y[m].reshape(1, -1), p.ref(m).reshape(1, -1), PROMPT_REL)


@pytest.mark.parametrize("heads,kv,hs", [(4, 1, 128), (4, 1, 64), (4, 2, 32)])
def test_scores_beyond_f32(heads, kv, hs):
    """Where every score of a row is below what f32 holds, no weight can be formed: NaN, and not the zeros of a row without tokens."""
    k = K()
    positions, M = [900, 3, -1, 40], 4
    rng = np.random.default_rng(hs)
    bt, n_pages = _table(rng, [max(p, 0) + 1 for p in positions])
    host = _cache(rng, n_pages, kv, hs)
    q = torch.from_numpy(rng.standard_normal((M, heads * hs)).astype(np.float32))
    for m in (0, 1):
        host[0][bt[m, :positions[m] // PAGE + 1]], host[2][bt[m, :positions[m] // PAGE + 1]] = -127, 1e18
        q[m] = 1e22
    cache = k.Kv8Cache(*_dev(*host))
    where = (_i32(positions), _i32(list(range(M))), torch.from_numpy(bt).cuda())
    for splits in (1, 8):
        scratch = torch.zeros(k.attention_scratch_bytes(M, heads, hs, splits), dtype=torch.uint8, device="cuda")
        y = torch.full((M, heads * hs), 3.0, device="cuda")
        k.kv8_attention(q.cuda(), M, heads, *where, cache, splits, scratch, y_out=y)
        assert torch.isnan(y[:2]).all() and (y[2] == 0).all()
        _near(y[3:], _attention(q[3].view(heads, hs), _values(host[0], host[2], bt[3], 41), _values(host[1], host[3], bt[3], 41)).reshape(1, -1), ATT_REL)


@pytest.mark.parametrize("heads,kv,hs,rows,context,workspace", [
    (16, 4, 128, 300, 40, True), (32, 8, 64, 240, 0, True), (16, 8, 128, 260, 2600, True), (32, 8, 64, 240, 3000, True), (4, 2, 32, 60, 10, False), (8, 1, 64, 33, 0, False), (4, 1, 128, 20, 700, False)])
def test_prompt_scores_beyond_f32(heads, kv, hs, rows, context, workspace):
    p = _Prompt(heads, kv, hs, rows, context)
    p.host[0][:], p.host[2][:] = -127, 60000.0 / 127 if workspace else 1e18
    q = p.q.view(rows, heads, hs)
    q[3] = q[rows - 1] = 3e38 if workspace else 1e22
    nan = torch.isnan(p.run(workspace))
    assert nan[3].all() and nan[rows - 1].all() and not nan[:3].any() and not nan[4:rows - 1].any()


def test_far_pages_of_a_larger_cache():
    """Pages beyond 2^32 bytes of codes, and of the fp16 pages of a workspace: written, read back, attended to by tokens and by prompts on both routes."""
    k = K()
    n_pages, kv, hs, heads, T, n = 135000, 8, 128, 8, 1200, 530    # 4.4 GB of codes of the keys, 8.8 GB of keys as fp16; as many of the values
    if torch.cuda.mem_get_info()[0] < 36 << 30:
        pytest.skip("36 GB of device memory")
    rng = np.random.default_rng(4)
    bt = np.concatenate([n_pages - 1 - 3 * rng.permutation(T // PAGE), [7]]).astype(np.int32)[None]
    cache, table = k.alloc_kv8(n_pages, kv, hs, "cuda"), torch.from_numpy(bt).cuda()
    pos, slot = torch.arange(T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    qkv, q = torch.from_numpy(rng.standard_normal((T, (heads + 2 * kv) * hs)).astype(np.float32)), torch.zeros(T, heads * hs, device="cuda")
    k.kv8_write(qkv.cuda(), T, heads, None, pos, slot, table, q, cache)
    codes, scales = _code(qkv.view(T, -1, hs)[:, heads:])
    held = codes.double() * scales.double()[..., None]
    kk, vv = (torch.zeros(T, kv * hs, device="cuda") for _ in range(2))
    k.kv8_read(T, pos, slot, table, cache, kk, vv)
    assert torch.equal(kk.cpu().view(T, kv, hs), held[:, :kv].float()) and torch.equal(vv.cpu().view(T, kv, hs), held[:, kv:].float())
    ref = {m: _attention(q[m].cpu().view(heads, hs), held[:m + 1, :kv], held[:m + 1, kv:]).reshape(1, -1) for m in (T - n, T - n + 127, T - 300, T - 1)}
    splits = k.kv8_attention_splits(1, heads, kv, bt.shape[1])
    y = torch.zeros(1, heads * hs, device="cuda")
    k.kv8_attention(q[T - 1:], 1, heads, pos[T - 1:], slot[:1], table, cache, splits, torch.zeros(k.attention_scratch_bytes(1, heads, hs, splits), dtype=torch.uint8, device="cuda"), y_out=y)
    _near(y, ref[T - 1], ATT_REL)
    assert k.kv8_widens(n, heads, hs)
    for work in (k.kv8_prefill_workspace(n_pages, kv, hs, n, "cuda"), None):
        y = torch.zeros(n, heads * hs, device="cuda")
        k.kv8_attention_prefill(q[T - n:], n, heads, pos[T - n:], slot[:n], table, _i32([1, 0, n]), cache, work, y_out=y)
        for m, r in ref.items():
            _near(y[m - T + n:m - T + n + 1], r, PROMPT_REL)



@pytest.mark.parametrize("heads,kv,hs,rows,context", [(16, 8, 128, 260, 2600), (32, 8, 64, 240, 10), (32, 8, 64, 240, 3000), (16, 4, 128, 100, 900)])
def test_prompts_captured_and_side_by_side(heads, kv, hs, rows, context):
    """A layer's calls -- rows written, one row of another user, the prompt -- twice over in two graphs with buffers of their own, replayed on two streams at once and
    again on new rows, each launch ahead of its predecessor's end where it may: what single calls give, bit for bit."""
    k = K()
    rng = np.random.default_rng(rows)
    bt, n_pages = _table(rng, [context + rows, 900])
    host, M = _cache(rng, n_pages, kv, hs), rows + 1
    where = (_i32([899] + list(range(context, context + rows))), _i32([1] + [0] * rows), torch.from_numpy(bt).cuda())
    meta, skip, splits = _i32([1, 1, M]), _i32([0] + [1] * rows), 3
    freqs = torch.from_numpy((10000.0 ** (-np.arange(0, hs, 2) / hs)).astype(np.float32)).cuda()

    class Side:
        def __init__(self):
            self.cache = k.Kv8Cache(*_dev(*host))
            self.qkv, self.q, self.y = (torch.zeros(M, n * hs, device="cuda") for n in (heads + 2 * kv, heads, heads))
            self.work = k.kv8_prefill_workspace(n_pages, kv, hs, M, "cuda")
            self.scratch = torch.zeros(k.attention_scratch_bytes(M, heads, hs, splits), dtype=torch.uint8, device="cuda")

        def run(self, pdl):
            k.kv8_write(self.qkv, M, heads, freqs, *where, self.q, self.cache, pdl=pdl)
            k.kv8_attention(self.q, M, heads, *where, self.cache, splits, self.scratch, y_out=self.y, row_skip=skip, pdl=pdl)
            k.kv8_attention_prefill(self.q, M, heads, *where, meta, self.cache, self.work, y_out=self.y, pdl=pdl)

    sides, plain, graphs, streams = [Side(), Side()], Side(), [], [torch.cuda.Stream() for _ in range(2)]
    plain.run(False)                                               # (functions are loaded ahead of the captures)
    torch.cuda.synchronize()
    for st, side in zip(streams, sides):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=st):
            for _ in range(2):
                side.run(True)
    for seed in (1, 2, 3):
        x = torch.from_numpy(np.random.default_rng(seed).standard_normal((M, (heads + 2 * kv) * hs)).astype(np.float32)).cuda()
        for s in sides + [plain]:
            s.qkv.copy_(x)
        plain.run(False)
        torch.cuda.synchronize()
        for _ in range(3):
            for st, graph in zip(streams, graphs):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for s in sides:
            assert torch.equal(s.y, plain.y) and torch.equal(s.cache.k, plain.cache.k) and torch.equal(s.cache.v_scale, plain.cache.v_scale)
    assert not torch.isnan(plain.y).any() and not any(s.scratch[:65536].any() for s in sides)



def _engine(path, **kw):
    from dllama_b200.models.llama import LlamaEngine
    return LlamaEngine(path, max_rows=64, n_slots=3, max_seq_len=512, kv_dtype=torch.int8, **kw)


def test_read_cache_ahead_of_the_next_user(tiny_tp_model_path):
    """A conversation is read out behind queued work, and its sequence and pages go to another user before the read has run."""
    rng = np.random.default_rng(1)
    e = _engine(tiny_tp_model_path)
    a = e.alloc_slot()
    e.prefill(a, rng.integers(1, 1024, 100).tolist(), 0)
    e.forward(rng.integers(1, 1024, 64).tolist(), list(range(64)), [e.alloc_slot()] * 64)      # (the shape's graph is captured)
    want = [t.clone() for t in e.read_cache(0, a, 100, torch.float32)]
    e.ensure_capacity(a, 140)                                      # the table that the read needs is on its way
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    got = e.read_cache(0, a, 100, torch.float32)
    e.free_slot(a)
    b = e.alloc_slot()
    assert a == b
    e.forward(rng.integers(1, 1024, 64).tolist(), list(range(64)), [b] * 64)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    e.close()


def test_read_cache_behind_a_queued_step(tiny_tp_model_path):
    """A step waits with the table that it was given; a conversation is read out when its sequence has been given to another user."""
    rng = np.random.default_rng(2)
    e = _engine(tiny_tp_model_path)
    a, b = e.alloc_slot(), e.alloc_slot()
    e.prefill(a, rng.integers(1, 1024, 100).tolist(), 0)
    e.prefill(b, rng.integers(1, 1024, 50).tolist(), 0)
    want = e.forward([7], [100], [a]).clone()
    held = [t.clone() for t in e.read_cache(1, b, 50, torch.float16)]
    e.ensure_capacity(b, 70)
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    got = e.forward([7], [100], [a])
    e.free_slot(a)
    assert e.alloc_slot() == a
    e.ensure_capacity(a, 128)                                      # its pages in another order
    again = e.read_cache(1, b, 50, torch.float16)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(again, held))
    e.close()


def test_users_of_unlike_lengths(tmp_path):
    """One user deep in a conversation beside others at its beginning: steps of few users, and of more than 32, with shares for the long one."""
    from dllama_b200.formats import mfile
    from dllama_b200.models.llama import LlamaEngine
    from dllama_b200.models.oracle import OracleLlama
    from test_gpu_kv8_model import TOL, _rel_err
    rng, path = np.random.default_rng(3), str(tmp_path / "m.m")
    mfile.write_random_model(path, dict(dim=512, hidden_dim=512, n_layers=2, n_heads=8, n_kv_heads=2, vocab_size=1024, max_seq_len=1024, rope_theta=500000, rope=(32, 1, 4, 8192)), exact=True, seed=6)
    e = LlamaEngine(path, max_rows=64, n_slots=40, max_seq_len=1024, kv_dtype=torch.int8)
    prompts = [rng.integers(1, 1024, 950).tolist()] + [rng.integers(1, 1024, 1 + i % 50).tolist() for i in range(36)]
    slots = [e.alloc_slot() for _ in prompts]
    for s, p in zip(slots, prompts):
        e.prefill(s, p[:-1], 0) if len(p) > 1 else None
    want = {}
    for i in (0, 1, 2, 17, 36):
        o = OracleLlama(mfile.ModelFile(path), n_nodes=1, max_seq_len=1024)
        want[i] = o.forward(prompts[i], 0).numpy()[-1]
    for users in (range(3), range(37)):
        order = list(rng.permutation(list(users)))
        got = e.forward([prompts[i][-1] for i in order], [len(prompts[i]) - 1 for i in order], [slots[i] for i in order]).float().cpu().numpy()
        for i in set(users) & set(want):
            assert _rel_err(got[order.index(i)], want[i]) < TOL
    e.close()
