"""sample_many's steps as they run in the end: behind a captured graph, on shared pages, with the tokens that it drew given to the engine's public calls."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kernels import _decode_xh, _decode_xq
from test_gpu_sample_many import _engine, wide_heads_path  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
PAGE = 32


@pytest.mark.parametrize("n", [2, 4])
def test_what_is_to_be_shared_is_shared_beside_the_persistent_kernel(wide_heads_path, n, monkeypatch):  # noqa: F811
    """share=True on an engine whose batches of a few rows run on the persistent decode kernel, which knows no groups."""
    from dllama_b200.ops import kernels as K
    e = _engine(wide_heads_path, use_mega=True)
    assert e._mega_usable(n, False)
    calls = []
    shared = K.shared_attention
    monkeypatch.setattr(K, "shared_attention", lambda *a, **kw: (calls.append(a[1]), shared(*a, **kw)))
    prompt = np.random.default_rng(n).integers(1, 1024, 100).tolist()
    t = e.sample_many(prompt, n, 3, 1.0, seed=2, share=True)
    assert calls == [n] * 4 and t.shape == (n, 3)                  # two layers, a step launched and one captured
    calls.clear()
    e.sample_many(prompt, n, 3, 1.0, seed=2)
    assert not e.shares_prompt(n, 3) and calls == []
    e.close()


def _replayed(e, prompt, tokens):
    """The logits behind tokens [n][count] (all but the last one of each are run), every sample a sequence of its own that the engine's public calls run."""
    n, count = tokens.shape
    slots = [e.alloc_slot() for _ in range(n)]
    for s in slots:
        e.prefill(s, prompt)
    for i in range(count - 1):
        logits = e.forward(tokens[:, i].tolist(), [len(prompt) + i] * n, slots)
    out = logits[:n].float().cpu().numpy().copy()
    for s in slots:
        e.free_slot(s)
    return out


def _lines(cache, table, pos):
    """Keys or values of positions 0 .. pos of a sequence with that row of the block table: [kv heads][positions][head size]."""
    pages = table[:pos // PAGE + 1].long()
    return cache[pages].transpose(0, 1).flatten(1, 2)[:, :pos + 1]


def _attention(q, k, v):
    """f64 attention of a row's heads [kv heads][heads of each][head size], and what shared_attention may be off by (head of test_gpu_shared_attention)."""
    q, k, v = q.double(), k.double(), v.double()
    hs = q.shape[-1]
    w = torch.softmax(torch.matmul(q, k.transpose(1, 2)) / math.sqrt(hs), -1)
    y = torch.matmul(w, v)
    s = 2.0 ** -11 / math.sqrt(3) * torch.matmul(q ** 2, k.transpose(1, 2) ** 2).amax(-1, keepdim=True).sqrt() / math.sqrt(hs)
    squares = torch.matmul(w ** 2, v ** 2)
    spread = (squares - 2 * y * torch.matmul(w ** 2, v) + (w ** 2).sum(-1, keepdim=True) * y ** 2).clamp(min=0)
    off = 8 * torch.sqrt(s ** 2 * spread + (2.0 ** -22 / 3 + 8e-5 ** 2) * squares) + 2.0 ** -20 * torch.matmul(w, v.abs())
    return y.flatten(), off.flatten()


@pytest.mark.parametrize("which", ["tp8", "wide"])
@pytest.mark.parametrize("n,length,count", [(2, 64, 110), (3, 97, 34), (5, 95, 110), (16, 200, 110), (20, 33, 66), (11, 31, 40), (4, 300, 140)])
def test_many_captured_steps(tiny_tp_model_path, wide_heads_path, which, n, length, count):  # noqa: F811
    """A run on shared pages whose steps come out of the captured graph, on the dp4a rows and on tcgen05, with tails of no token, one and 31 behind the shared pages (or nothing shared at all) and
    samples that grow over several pages.  Against the same tokens run through the engine's public calls, every sample a sequence of its own:

    * where the last step's rows stand, and the first layer's keys and values of every token, which hang on nothing but the token and its place: equal, bit for bit;
    * the last layer's attention of the last step, as it went into the next product, against 64 bits over that step's own queries, keys and values.  Q80: half a step, 1/254 of a block's largest
      value (and of what that may be off by), a scale in fp16 (2^-11), and for rows on tcgen05 the value in fp16 (2^-11);
    * the logits: queries and weights in fp16 beside Q80 activations in two layers, 1e-2 of the largest one, as for two steps in test_shared_pages_give_the_same_logits;
    * the last tokens are those that the last step's logits and the seed's coins give."""
    from dllama_b200.ops import kernels as K
    e = _engine({"tp8": tiny_tp_model_path, "wide": wide_heads_path}[which])
    prompt = np.random.default_rng(length).integers(1, 1024, length).tolist()
    tokens = e.sample_many(prompt, n, count, 1.0, 0, 0.95, 0.0, seed=n, share=True)
    last = length + count - 2
    logits = e.logits[:n].clone()
    assert e.pos[:n].tolist() == [last] * n and len(set(e.slot[:n].tolist())) == n
    table = [e.block_table[s].clone() for s in e.slot[:n].tolist()]
    first = [[_lines(c[0], t, last).clone() for t in table] for c in (e.k_cache, e.v_cache)]
    assert all(torch.equal(t[:length // PAGE], table[0][:length // PAGE]) for t in table)
    own = torch.cat([t[length // PAGE:last // PAGE + 1] for t in table])
    assert len(own.unique()) == len(own)
    # the last layer's attention
    cols = e.q_loc
    if n <= 3:
        got = _decode_xq(e.xq_att[:cols // 128 * n * 160], cols, n, n)[0]
    else:
        got = _decode_xh(e.xh_att, cols, e.ncap, n)
    for m in range(n):
        y, off = _attention(e.q[m].view(e.n_kv_loc, -1, e.hs), _lines(e.k_cache[-1], table[m], last), _lines(e.v_cache[-1], table[m], last))
        top = (y.abs() + off).view(-1, 32).amax(1, keepdim=True).expand(-1, 32).flatten()
        room = off + top / 254 * (1 + 2.0 ** -8) + (2.0 ** -11 + (2.0 ** -11 if n > 3 else 0)) * top
        assert ((torch.from_numpy(got[m]).double().cuda() - y).abs() <= room).all()
    # the draw
    coins = torch.rand(count, n, generator=torch.Generator().manual_seed(n))
    out, full = torch.zeros(n, dtype=torch.int32, device="cuda"), lambda v, d: torch.full((n,), v, dtype=d, device="cuda")
    K.sample_tokens(logits, n, full(1.0, torch.float32), full(0, torch.int32), full(0.95, torch.float32), full(0.0, torch.float32), coins[-1].cuda(), out)
    assert out.tolist() == tokens[:, -1].tolist()
    # the same tokens through the public calls
    slots = [e.alloc_slot() for _ in range(n)]
    for s in slots:
        e.prefill(s, prompt)
    for i in range(count - 1):
        want = e.forward(tokens[:, i].tolist(), [length + i] * n, slots)
    assert (logits - want[:n]).abs().max() <= 1e-2 * want[:n].abs().max()
    for m, s in enumerate(slots):
        for c, lines in zip((e.k_cache, e.v_cache), first):
            assert torch.equal(lines[m], _lines(c[0], torch.from_numpy(e.pages.table[s]).cuda(), last))
    e.close()
