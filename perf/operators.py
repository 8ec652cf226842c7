"""Performance cases of the 8-bit token cache: what a server with many users, or with long conversations, has it do.

The cache holds int8 keys and values in pages of 32 tokens, with one f32 scale for each token and key/value head:
``s = f32(amax / 127)``, ``code = rint(x * f32(127 / amax))``.

Kinds (a case is a dict of plain values; "kind" says which operator):

* ``write``   -- the merged q|k|v rows of a layer: rotary positions on queries and keys, keys and values quantised into their
                 pages; the rows' lines are then read back, so that what the pages hold can be compared.
* ``read``    -- lines of a conversation out of its pages, as fp16 or f32 (to keep it elsewhere while its owner is away).
* ``decode``  -- attention of one new token per sequence over its pages.
* ``prompt``  -- causal attention of a prompt chunk behind an earlier context.

Heads and head sizes are those of the repository's benchmark and tests (32 heads on 8 key/value heads of 128 and 64, tensor-parallel
shares of them, and 64 heads on 8).
"""
import math

import torch

own = False                   # True: run() calls the framework's operators

PAGE = 32
ROPE_BASE = 500000.0
TINY = 2.0 ** -100            # lines whose largest magnitude is below are held as zeros


def listed():
    return [
        # one user chatting: the smallest call, a token's row into the cache
        {"name": "write_1", "kind": "write", "rows": 1, "heads": 32, "kv_heads": 8, "head_size": 128, "context": 192, "prompt": False},
        # a token of each of 32 users
        {"name": "write_32", "kind": "write", "rows": 32, "heads": 32, "kv_heads": 8, "head_size": 128, "context": 500, "prompt": False},
        # a long prompt's chunk, an odd number of tokens behind 77 others
        {"name": "write_4001", "kind": "write", "rows": 4001, "heads": 32, "kv_heads": 8, "head_size": 128, "context": 77, "prompt": True},
        # a short conversation moved out of the cache, small heads
        {"name": "read_700", "kind": "read", "rows": 700, "kv_heads": 8, "head_size": 64, "out": "f32"},
        # a long one, as fp16
        {"name": "read_100003", "kind": "read", "rows": 100003, "kv_heads": 8, "head_size": 128, "out": "f16"},
        # one user chatting
        {"name": "decode_1", "kind": "decode", "rows": 1, "heads": 32, "kv_heads": 8, "head_size": 128, "context": 192},
        # 32 users deep in a conversation, each at a place of its own
        {"name": "decode_32", "kind": "decode", "rows": 32, "heads": 32, "kv_heads": 8, "head_size": 128, "context": 3000},
        # seven users, eight query heads for each key/value head, small heads
        {"name": "decode_7_group8", "kind": "decode", "rows": 7, "heads": 64, "kv_heads": 8, "head_size": 64, "context": 5000},
        # one user with a book in the context
        {"name": "decode_long", "kind": "decode", "rows": 1, "heads": 32, "kv_heads": 8, "head_size": 128, "context": 100003},
        # a user's next message behind a conversation
        {"name": "prompt_100", "kind": "prompt", "rows": 100, "heads": 32, "kv_heads": 8, "head_size": 128, "context": 1000},
        # a prompt of small heads
        {"name": "prompt_500_small", "kind": "prompt", "rows": 500, "heads": 32, "kv_heads": 8, "head_size": 64, "context": 0},
        # a long prompt as one chunk, an odd number of tokens behind 77 others
        {"name": "prompt_4001", "kind": "prompt", "rows": 4001, "heads": 32, "kv_heads": 8, "head_size": 128, "context": 77},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "prompt"])
    heads, kv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 8), (16, 4), (8, 1), (16, 1)])
    hs = rng.choice([64, 128, 128])
    c = {"kind": kind, "kv_heads": kv, "head_size": hs}
    if kind == "read":
        c.update(rows=_log(rng, 1, 100000), out=rng.choice(["f16", "f32", "bf16"]))
        if c["out"] == "f32":
            c["rows"] = (c["rows"] + 1) // 2
        return c
    c["heads"] = heads
    if kind == "write":
        c["prompt"] = rng.random() < 0.5
        c.update(rows=_log(rng, 16, 4000) if c["prompt"] else _log(rng, 1, 64), context=_log(rng, 1, 3000))
        if heads == 64:
            c["rows"] = (c["rows"] + 1) // 2
    elif kind == "decode":
        c.update(rows=_log(rng, 1, 48))
        c.update(context=_log(rng, 1, min(100000, 96000 // c["rows"])))
    else:
        c.update(rows=_log(rng, 16, 2800 if heads == 64 else 4000), context=rng.choice([0, _log(rng, 1, 1000), _log(rng, 16, 8000)]))
        c["context"] = min(c["context"], 8000000 * 32 // heads // c["rows"] // 2)
    return c


# ---------------------------------------------------------------------------------------------------------------
# inputs (made from the seed alone)
# ---------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rows(case, seed):
    """Position and sequence of every row, tokens of every sequence."""
    M = case["rows"]
    if case["kind"] == "read":
        return list(range(M)), [0] * M, [M]
    if case["kind"] == "prompt" or (case["kind"] == "write" and case["prompt"]):
        p0 = case["context"]
        return list(range(p0, p0 + M)), [0] * M, [p0 + M]
    g = torch.Generator()
    g.manual_seed(seed)
    top = case["context"]
    pos = [top - 1] if M == 1 else [int(x) for x in torch.randint(top // 2, top, (M,), generator=g)]
    return pos, list(range(M)), [p + 1 for p in pos]


def _page_table(g, lens):
    """Block table [sequences][pages], pages in a random order, and the number of pages."""
    need = [(t + PAGE - 1) // PAGE for t in lens]
    perm = torch.randperm(sum(need), generator=g, device="cuda", dtype=torch.int32)
    bt = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[at:at + n]
        at += n
    return bt, at


def _lines(g, n_pages, kv, hs, key):
    """Pages as a model leaves them: keys with some strong channels, values of differing lengths from token to token."""
    x = _randn(g, n_pages, kv, PAGE, hs)
    if key:
        x *= torch.exp(0.5 * _randn(g, kv, 1, hs))
    else:
        x *= torch.exp(0.3 * _randn(g, n_pages, kv, PAGE, 1))
    amax = x.abs().amax(-1, keepdim=True)
    return torch.round(x * (127.0 / amax)).to(torch.int8), (amax / 127.0).squeeze(-1)


def prepare(case, seed):
    g = _gen(seed)
    M, kv, hs = case["rows"], case["kv_heads"], case["head_size"]
    pos, slot, lens = _rows(case, seed)
    bt, n = _page_table(g, lens)
    s = {"case": dict(case), "pos": _i32(pos), "slot": _i32(slot), "bt": bt}
    (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = _lines(g, n, kv, hs, True), _lines(g, n, kv, hs, False)
    if own:
        from dllama_b200.ops import kernels as K
        s["cache"] = K.Kv8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if case["kind"] == "read":
        t = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[case["out"]]
        s["k_out"], s["v_out"] = (torch.zeros(M, kv * hs, dtype=t, device="cuda") for _ in range(2))
        return s
    H = case["heads"]
    if case["kind"] == "write":
        s["qkv"] = _randn(g, M, (H + 2 * kv) * hs)
        s["freqs"] = (ROPE_BASE ** (-torch.arange(0, hs, 2, device="cuda", dtype=torch.float64) / hs)).float()
        s["q_out"] = torch.zeros(M, H * hs, device="cuda")
        s["k_out"], s["v_out"] = (torch.zeros(M, kv * hs, dtype=torch.float16, device="cuda") for _ in range(2))
        return s
    s["q"] = _randn(g, M, H * hs)
    if case["kind"] == "decode":
        s["y"] = torch.zeros(M, H * hs, device="cuda")
        if own:
            s["splits"] = K.kv8_attention_splits(M, H, kv, bt.shape[1])
            s["scratch"] = torch.zeros(K.attention_scratch_bytes(M, H, hs, s["splits"]), dtype=torch.uint8, device="cuda")
    else:
        s["y"] = torch.zeros(M, H * hs, dtype=torch.bfloat16, device="cuda")      # what a 16-bit product reads next
        s["meta"] = _i32([1, 0, M])
        if own:
            s["work"] = K.kv8_prefill_workspace(n, kv, hs, M, "cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------------
def _run_own(s):
    from dllama_b200.ops import kernels as K
    c = s["case"]
    M, kind = c["rows"], c["kind"]
    where, cache = (s["pos"], s["slot"], s["bt"]), s["cache"]
    if kind == "read":
        K.kv8_read(M, *where, cache, s["k_out"], s["v_out"])
        return {"k": s["k_out"], "v": s["v_out"]}
    if kind == "write":
        K.kv8_write(s["qkv"], M, c["heads"], s["freqs"], *where, s["q_out"], cache)
        K.kv8_read(M, *where, cache, s["k_out"], s["v_out"])
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    if kind == "decode":
        K.kv8_attention(s["q"], M, c["heads"], *where, cache, s["splits"], s["scratch"], y_out=s["y"])
    else:
        K.kv8_attention_prefill(s["q"], M, c["heads"], *where, s["meta"], cache, workspace=s["work"], y_out=s["y"])
    return s["y"]


# ---------------------------------------------------------------------------------------------------------------
# their plain form
# ---------------------------------------------------------------------------------------------------------------
def _places(s):
    """Page and place in the page of every row."""
    return s["bt"][s["slot"].long(), (s["pos"] // PAGE).long()].long(), (s["pos"] % PAGE).long()


def _values(codes, scale):
    return codes.float() * scale[..., None]


def _plain_read(s, dtype):
    page, at = _places(s)
    M = page.shape[0]
    return tuple(_values(s[x][page, :, at], s[x + "_scale"][page, :, at]).to(dtype).reshape(M, -1) for x in ("k", "v"))


def _codes(x):
    """f32 lines [..., head size] -> codes and scales; products with the factor in 64 bits, as values may lie next to a border."""
    amax = x.abs().amax(-1)
    live = amax >= TINY
    factor = torch.where(live, 127.0 / amax, torch.zeros_like(amax))
    return torch.round(x.double() * factor.double()[..., None]).to(torch.int8), torch.where(live, amax / 127.0, torch.zeros_like(amax))


def _rotated(x, pos, freqs):
    """x [M][heads][head size] f32, pairs of neighbouring values turned by position * frequency (in 64 bits)."""
    a = pos.double()[:, None, None] * freqs.double()
    c, sn = torch.cos(a), torch.sin(a)
    x0, x1 = x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack((x0 * c - x1 * sn, x0 * sn + x1 * c), -1).flatten(-2).float()


def _plain_write(s):
    c = s["case"]
    M, H, kv, hs = c["rows"], c["heads"], c["kv_heads"], c["head_size"]
    x = s["qkv"].view(M, H + 2 * kv, hs)
    turned = _rotated(x[:, :H + kv], s["pos"], s["freqs"])
    page, at = _places(s)
    s["k"][page, :, at], s["k_scale"][page, :, at] = _codes(turned[:, H:])
    s["v"][page, :, at], s["v_scale"][page, :, at] = _codes(x[:, H + kv:])
    k, v = _plain_read(s, torch.float16)
    return {"q": turned[:, :H].reshape(M, -1), "k": k, "v": v}


def _weights(scores, seen):
    """Softmax over the last axis of what is seen."""
    scores = scores.masked_fill_(~seen, -math.inf)
    e = torch.exp_(scores - scores.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_decode(s):
    c = s["case"]
    M, H, kv, hs = c["rows"], c["heads"], c["kv_heads"], c["head_size"]
    pages = s["bt"][s["slot"].long()].long()                                          # [M][pages]
    k, v = (_values(s[x][pages], s[x + "_scale"][pages]).transpose(1, 2).reshape(M, kv, -1, hs) for x in ("k", "v"))
    seen = torch.arange(k.shape[2], device="cuda") <= s["pos"][:, None]
    w = _weights(torch.matmul(s["q"].view(M, kv, H // kv, hs), k.transpose(-1, -2)) / math.sqrt(hs), seen[:, None, None])
    return torch.matmul(w, v).reshape(M, H * hs)


def _plain_prompt(s):
    c = s["case"]
    M, H, kv, hs = c["rows"], c["heads"], c["kv_heads"], c["head_size"]
    pages = s["bt"][s["slot"][0].long()].long()
    k, v = (_values(s[x][pages], s[x + "_scale"][pages]).transpose(0, 1).reshape(kv, -1, hs) for x in ("k", "v"))
    q = s["q"].view(M, kv, H // kv, hs).permute(1, 2, 0, 3)                           # [kv][group][M][hs]
    seen = torch.arange(k.shape[1], device="cuda") <= s["pos"][:, None]
    w = _weights(torch.matmul(q, k[:, None].transpose(-1, -2)) / math.sqrt(hs), seen)
    return torch.matmul(w, v[:, None]).permute(2, 0, 1, 3).reshape(M, H * hs).to(torch.bfloat16)


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "read":
        k, v = _plain_read(state, state["k_out"].dtype)
        return {"k": k, "v": v}
    return {"write": _plain_write, "decode": _plain_decode, "prompt": _plain_prompt}[kind](state)


# ---------------------------------------------------------------------------------------------------------------
# the work that a case cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    M, kv, hs = case["rows"], case["kv_heads"], case["head_size"]
    line = 2 * kv * (hs + 4)                     # codes and scales of a token's key and value
    if case["kind"] == "read":
        return {"bytes": M * (line + 2 * kv * hs * (4 if case["out"] == "f32" else 2)), "flops": 2 * M * kv * hs}
    H = case["heads"]
    if case["kind"] == "write":                  # rows in, queries out, lines into the pages and back
        return {"bytes": M * (4 * (2 * H + 2 * kv) * hs + 2 * line + 4 * kv * hs), "flops": M * (H + 2 * kv) * hs * 6}
    pos, _, lens = _rows(case, 1)
    seen, out = sum(p + 1 for p in pos), 4 if case["kind"] == "decode" else 2
    return {"bytes": sum(lens) * line + M * H * hs * (4 + out), "flops": 4 * seen * H * hs}


def exact(case, seed):
    s = prepare(case, seed)
    M, kv, hs = case["rows"], case["kv_heads"], case["head_size"]
    page, at = s["bt"].long()[s["slot"].long(), s["pos"].long() // PAGE], s["pos"].long() % PAGE
    if case["kind"] == "read":
        return {x: (s[x][page, :, at].double() * s[x + "_scale"][page, :, at].double().unsqueeze(2)).flatten(1) for x in ("k", "v")}
    H = case["heads"]
    if case["kind"] == "write":
        q, k, v = s["qkv"].double().view(M, -1, hs).split([H, kv, kv], 1)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * s["freqs"].double()[None])[:, None]

        def turned(x):
            return torch.view_as_real(torch.view_as_complex(x.reshape(M, -1, hs // 2, 2)) * turn).flatten(2)

        def held(x):                             # scale and factor are f32 numbers, and so is what they are made of
            top = x.float().abs().max(2, keepdim=True).values
            return ((x.float().double() * (127.0 / top).double()).round() * (top / 127.0).double()).flatten(1)

        return {"q": turned(q).flatten(1), "k": held(turned(k)), "v": held(v)}
    y = torch.empty(M, H, hs, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(M, H, hs)
    one = case["kind"] == "prompt"               # all rows of one sequence
    for m in ([slice(0, M)] if one else [slice(i, i + 1) for i in range(M)]):
        seq = s["bt"][s["slot"][m][0].long()].long()
        last = int(s["pos"][m][-1])
        hide = torch.arange(last + 1, device="cuda")[None] > s["pos"][m][:, None]
        for h in range(kv):
            k, v = ((s[x][seq, h].double() * s[x + "_scale"][seq, h].double()[..., None]).flatten(0, 1)[:last + 1] for x in ("k", "v"))
            for u in range(h * (H // kv), (h + 1) * (H // kv)):
                z = q[m, u] @ k.T * hs ** -0.5
                y[m, u] = torch.softmax(z.masked_fill(hide, -math.inf), 1) @ v
    return y.flatten(1)
