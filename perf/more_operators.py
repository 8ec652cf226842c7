"""Performance cases of a serving step for many users of one prompt: where their rows lie, attention that reads the shared part once, the tokens drawn.

Token caches are fp16 pages of 32 tokens, [pages][key/value heads][32][head size]; a request's pages are a row of the block table.

Kinds (a case is a dict of plain values; "kind" says which operator):

* ``tables`` -- block tables and slot maps from the requests' lengths: pages for the tokens that come, off a list of free ones, the pages of a shared
                prompt ahead of them, and position, table row and cache line of every token row.
* ``shared`` -- attention of one new token per sequence, where groups of sequences begin with the same pages ("37x130 1x0": 37 sequences that
                share 130 pages, and one that shares none).
* ``sample`` -- a token for every row of logits: temperature, top-k, top-p and min-p, with given random numbers.

Heads, head sizes and vocabularies are those of the repository's benchmark and tests (32 heads on 8 key/value heads of 128 and 64, tensor-parallel shares of
them, 64 heads on 8; 128256 and 32000 tokens).
"""
import math

import torch

own = False                   # True: run() calls the framework's operators

PAGE = 32
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a step of 32 users deep in conversations of their own: a token each
        {"name": "tables_32", "kind": "tables", "requests": 32, "new": 1, "context": 3000, "shared": 0},
        # prompts and decoding users in one batch, all behind a system prompt of 1600 tokens
        {"name": "tables_50_prompts", "kind": "tables", "requests": 50, "new": 700, "context": 2500, "shared": 50},
        # a large batch of short prompts behind a long instruction
        {"name": "tables_2001_prompts", "kind": "tables", "requests": 2001, "new": 64, "context": 9000, "shared": 250},
        # three answers to a short question
        {"name": "shared_3", "kind": "shared", "groups": "3x16", "heads": 32, "kv_heads": 8, "head_size": 128, "own": 60},
        # 32 users behind a long system prompt
        {"name": "shared_32", "kind": "shared", "groups": "32x250", "heads": 32, "kv_heads": 8, "head_size": 128, "own": 300},
        # eight query heads for each key/value head, small heads; two prompts and a user without one
        {"name": "shared_55_group8", "kind": "shared", "groups": "37x130 17x333 1x0", "heads": 64, "kv_heads": 8, "head_size": 64, "own": 500},
        # a tensor-parallel share: two key/value heads, a book in the prompt, eleven readers
        {"name": "shared_11_book", "kind": "shared", "groups": "11x3001", "heads": 8, "kv_heads": 2, "head_size": 128, "own": 1000},
        # many samples of one long prompt
        {"name": "shared_200", "kind": "shared", "groups": "200x999", "heads": 32, "kv_heads": 8, "head_size": 128, "own": 400},
        # one user: top-p
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 128256, "dtype": "f32", "filters": "p"},
        # 32 users, each with settings of their own
        {"name": "sample_32", "kind": "sample", "rows": 32, "vocab": 128256, "dtype": "f32", "filters": "mixed"},
        # a smaller vocabulary, 16-bit logits
        {"name": "sample_75_bf16", "kind": "sample", "rows": 75, "vocab": 32000, "dtype": "bf16", "filters": "mixed"},
        # many samples of one prompt, all alike: top-k, then top-p
        {"name": "sample_200", "kind": "sample", "rows": 200, "vocab": 128256, "dtype": "f32", "filters": "kp"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "shared", "sample"])
    if kind == "tables":
        c = {"kind": kind, "requests": _log(rng, 1, 2000), "new": rng.choice([1, _log(rng, 2, 1000)]), "context": _log(rng, 40, 9000), "shared": 0}
        c["new"] = max(1, min(c["new"], 64000 // c["requests"]))
        if rng.random() < 0.6:
            c["shared"] = _log(rng, 1, max(1, c["context"] // 2 // PAGE))
        return c
    if kind == "sample":
        c = {"kind": kind, "rows": _log(rng, 1, 200), "vocab": rng.choice([128256, 128256, 32000, 32003, 50001, _log(rng, 500, 128000)]),
             "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "filters": rng.choice(["mixed", "mixed", "p", "k", "kp", "min", "none"])}
        return c
    heads, kv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 8), (16, 4), (8, 2), (8, 1)])
    c = {"kind": kind, "heads": heads, "kv_heads": kv, "head_size": rng.choice([64, 128, 128])}
    n = rng.choice([1, 1, 1, 2, 3])
    groups = []
    for _ in range(n):
        rows = _log(rng, 2, 200 // n)
        groups.append((rows, _log(rng, 4, min(3000, 180000 * 32 // heads // rows // n))))
    if rng.random() < 0.3:
        groups.append((rng.randint(1, 5), 0))
    c["groups"] = " ".join(f"{rows}x{pages}" for rows, pages in groups)
    c["own"] = _log(rng, 4, max(5, min(4000, 60000 // sum(rows for rows, _ in groups))))
    return c


# ---------------------------------------------------------------------------------------------------------------
# inputs (made from the seed alone)
# ---------------------------------------------------------------------------------------------------------------
def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pages(tokens):
    return (tokens + PAGE - 1) // PAGE


def _lengths(case, seed):
    """Tokens that every request holds and that it runs now."""
    n, lead = case["requests"], case["shared"]
    g = _gen(seed, "cpu")
    held = torch.randint(case["context"] // 2, case["context"] + 1, (n,), generator=g).clamp_(min=PAGE * lead)
    if case["new"] == 1:                          # users who decode; one in 16 waits
        return held, (torch.randperm(n, generator=g) % 16 != 15).long()
    # prompts, short ones the most, in another order with every seed; half of them have just come: nothing of their own in the cache
    new = torch.exp(torch.linspace(0, 1, n)[torch.randperm(n, generator=g)] * math.log(case["new"])).round().long()
    held[torch.rand(n, generator=g) < 0.5] = PAGE * lead
    return held, new


def _prepare_tables(case, seed):
    n, lead = case["requests"], case["shared"]
    held, new = _lengths(case, seed)
    have, need = _pages(held), _pages(held + new)
    g = _gen(seed)
    rows, taken = int(new.sum()), int((need - have).sum())
    n_pages = int((have - lead).sum()) + lead + taken + 40
    page = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int32)
    width = max(case["context"], PAGE * lead) // PAGE + case["new"] // PAGE + 4
    seq = torch.randperm(n, generator=g, device="cuda", dtype=torch.int32)                # table rows, in no order; the prompt's is the last one
    k = torch.arange(width, device="cuda")
    mine = (have - lead).cuda()
    at = lead + mine.cumsum(0) - mine
    table = torch.zeros(n + 1, width, dtype=torch.int32, device="cuda")
    own_pages = (k >= lead) & (k < have.cuda()[:, None])
    table[seq.long()] = torch.where(own_pages, page[(at[:, None] + k - lead).clamp_(0, n_pages - 1)], torch.zeros_like(page[0]))
    table[n, :lead] = page[:lead]
    used = lead + int(mine.sum())
    cap = (rows + 7) // 8 * 8 + 8                                                         # places for rows; those behind the last one stay empty
    s = {"case": dict(case), "held": _i32(held.tolist()), "new": _i32(new.tolist()), "seq": seq, "table": table, "free": page[used:].contiguous(),
         "taken": _i32([7]), "n_pages": n_pages, "lead_seq": None, "lead_pages": None}
    if lead:
        s["lead_seq"], s["lead_pages"] = torch.full_like(seq, n), torch.full_like(seq, lead)
    for x, size in (("pos", cap), ("slot", cap), ("line", cap), ("start", n + 1), ("held_out", n), ("taken_out", 1), ("status", 1)):
        s[x] = torch.zeros(size, dtype=torch.int32, device="cuda")
    return s


def _rows(case, seed):
    """Position of every row, and each group's range of rows and shared pages."""
    g = _gen(seed, "cpu")
    pos, groups = [], []
    for rows, pages in (map(int, x.split("x")) for x in case["groups"].split()):
        groups.append((len(pos), len(pos) + rows, pages))
        pos += (pages * PAGE + torch.randint(0, case["own"], (rows,), generator=g)).tolist()
    return pos, groups


def _prepare_shared(case, seed):
    H, kv, hs = case["heads"], case["kv_heads"], case["head_size"]
    pos, groups = _rows(case, seed)
    M = len(pos)
    need = [p // PAGE + 1 for p in pos]
    n_pages = sum(need) - sum((e - b - 1) * p for b, e, p in groups)
    g = _gen(seed)
    order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int32)
    table = torch.zeros(M, max(need) + 1, dtype=torch.int32, device="cuda")
    at = 0
    for b, e, p in groups:
        table[b:e, :p] = order[at:at + p]
        at += p
        for m in range(b, e):
            table[m, p:need[m]] = order[at:at + need[m] - p]
            at += need[m] - p
    meta = [len([1 for x in groups if x[2]])] + [v for x in groups if x[2] for v in x]
    # keys with some strong channels, values of differing lengths from token to token, as a model leaves them
    k = torch.randn(n_pages, kv, PAGE, hs, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(kv, 1, hs, generator=g, device="cuda"))
    v = torch.randn(n_pages, kv, PAGE, hs, generator=g, device="cuda") * torch.exp(0.3 * torch.randn(n_pages, kv, PAGE, 1, generator=g, device="cuda"))
    s = {"case": dict(case), "groups": groups, "pos": _i32(pos), "slot": torch.arange(M, dtype=torch.int32, device="cuda"), "table": table, "meta": _i32(meta),
         "k": k.half(), "v": v.half(), "q": torch.randn(M, H * hs, generator=g, device="cuda"),
         "y": torch.zeros(M, H * hs, dtype=torch.bfloat16, device="cuda")}                # what a 16-bit product reads next
    if own:
        from dllama_b200.ops import kernels as K
        s["work"] = K.shared_attention_workspace(M, H, kv, hs, "cuda")
    return s


def _prepare_sample(case, seed):
    M, V = case["rows"], case["vocab"]
    g = _gen(seed)
    x = torch.randn(M, V, generator=g, device="cuda") * 2.2
    # some dozens of tokens that fit, the better the fewer
    n = min(V, 64)
    at = torch.randint(0, V, (M, n), generator=g, device="cuda")
    x.scatter_add_(1, at, 6 + 8 * torch.rand(M, n, generator=g, device="cuda") ** 3)
    s = {"case": dict(case), "logits": x.to(TYPES[case["dtype"]])}

    def some(lo, hi):
        return lo + (hi - lo) * torch.rand(M, generator=g, device="cuda")

    f = case["filters"]
    off, k = torch.zeros(M, device="cuda"), torch.randint(5, 200, (M,), generator=g, device="cuda", dtype=torch.int32)
    s["temperature"], s["top_p"], s["min_p"], s["coin"] = some(0.5, 1.3), some(0.7, 0.99), some(0.01, 0.2), torch.rand(M, generator=g, device="cuda")
    if f == "mixed":                                                                      # each of the settings on or off, some users greedy
        on = torch.rand(4, M, generator=g, device="cuda") < 0.6
        s["temperature"] = torch.where(torch.rand(M, generator=g, device="cuda") < 0.1, off, s["temperature"])
        s["top_k"], s["top_p"], s["min_p"] = k * on[0], s["top_p"] * on[1], s["min_p"] * on[2]
    else:
        s["top_k"], s["top_p"], s["min_p"] = k * ("k" in f), s["top_p"] * ("p" in f), s["min_p"] * (f == "min")
        if f == "min":
            s["top_p"] = off
    s["tokens"], s["prob"] = torch.zeros(M, dtype=torch.int32, device="cuda"), torch.zeros(M, device="cuda")
    return s


def prepare(case, seed):
    return {"tables": _prepare_tables, "shared": _prepare_shared, "sample": _prepare_sample}[case["kind"]](case, seed)


# ---------------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------------
_TABLES = ("table", "pos", "slot", "line", "start", "held_out", "taken_out", "status")


def _run_own(s):
    from dllama_b200.ops import kernels as K
    c = s["case"]
    if c["kind"] == "tables":
        K.page_tables(c["requests"], s["held"], s["new"], s["seq"], s["table"], s["free"], s["taken"], s["n_pages"], s["pos"], s["slot"], s["status"],
                      line=s["line"], start=s["start"], held_out=s["held_out"], taken_out=s["taken_out"], lead_seq=s["lead_seq"], lead_pages=s["lead_pages"])
        return {x: s[x] for x in _TABLES}
    if c["kind"] == "shared":
        K.shared_attention(s["q"], len(s["slot"]), c["heads"], s["pos"], s["slot"], s["table"], s["meta"], s["k"], s["v"], s["work"], y_out=s["y"])
        return s["y"]
    K.sample_tokens(s["logits"], c["rows"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["coin"], s["tokens"], prob_out=s["prob"])
    return {"tokens": s["tokens"], "prob": s["prob"]}


# ---------------------------------------------------------------------------------------------------------------
# their plain form
# ---------------------------------------------------------------------------------------------------------------
def _plain_tables(s):
    n, cap = s["case"]["requests"], s["pos"].shape[0]
    held, new, seq, table = s["held"].long(), s["new"].long(), s["seq"].long(), s["table"]
    have, need = (held + PAGE - 1) // PAGE, (held + new + PAGE - 1) // PAGE
    pages = need - have
    first = s["taken"].long() + pages.cumsum(0) - pages
    k = torch.arange(table.shape[1], device="cuda")
    rows = table[seq]
    fresh = (k >= have[:, None]) & (k < need[:, None])
    rows = torch.where(fresh, s["free"][(first[:, None] + k - have[:, None]).clamp_(0, s["free"].shape[0] - 1)], rows)
    if s["lead_seq"] is not None:
        rows = torch.where(k < s["lead_pages"][:, None], table[s["lead_seq"].long()], rows)
    table[seq] = rows
    end = new.cumsum(0)
    start = torch.cat((end.new_zeros(1), end))
    r = torch.arange(cap, device="cuda")
    live = r < start[n]
    i = torch.searchsorted(end, r, right=True).clamp_(max=n - 1)
    pos, slot = held[i] + r - start[i], seq[i]
    line = table[slot, (pos // PAGE).clamp_(0, table.shape[1] - 1)].long() * PAGE + pos % PAGE
    none = torch.full_like(pos, -1)
    out = (table, torch.where(live, pos, none), torch.where(live, slot, torch.zeros_like(slot)), torch.where(live, line, none), start, held + new,
           s["taken"].long() + pages.sum(), torch.zeros_like(s["status"]))
    return {x: t.int() for x, t in zip(_TABLES, out)}


def _plain_shared(s):
    c = s["case"]
    H, kv, hs = c["heads"], c["kv_heads"], c["head_size"]
    q = s["q"].view(-1, kv, H // kv, hs) / math.sqrt(hs)
    y = torch.empty_like(q)
    for b, e, pages in s["groups"]:
        n = e - b
        mine = s["table"][b:e, pages:].long()                                             # [rows][pages of their own]
        k, v = (s[x][mine].float().transpose(1, 2).reshape(n, kv, -1, hs) for x in ("k", "v"))
        seen = torch.arange(k.shape[2], device="cuda") + pages * PAGE <= s["pos"][b:e, None]
        z = torch.matmul(q[b:e], k.transpose(-1, -2)).masked_fill_(~seen[:, None, None], -math.inf)
        top = z.amax(-1, keepdim=True)
        if pages:
            head = s["table"][b, :pages].long()                                           # the group's, read once
            ks, vs = (s[x][head].float().transpose(0, 1).reshape(kv, -1, hs) for x in ("k", "v"))
            zs = torch.matmul(q[b:e].transpose(0, 1).reshape(kv, -1, hs), ks.transpose(-1, -2)).view(kv, n, H // kv, -1)
            top = torch.maximum(top, zs.amax(-1, keepdim=True).transpose(0, 1))
        w = torch.exp_(z - top)
        total, sums = w.sum(-1, keepdim=True), torch.matmul(w, v)
        if pages:
            w = torch.exp_(zs - top.transpose(0, 1))
            total = total + w.sum(-1, keepdim=True).transpose(0, 1)
            sums = sums + torch.matmul(w.reshape(kv, -1, pages * PAGE), vs).view(kv, n, H // kv, hs).transpose(0, 1)
        y[b:e] = sums / total
    return y.reshape(-1, H * hs).to(torch.bfloat16)


def _plain_sample(s):
    x = s["logits"].double()                       # sums of a vocabulary, compared with a random number: in 64 bits
    M, V = x.shape
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    k, p, min_p = s["top_k"].long()[:, None], s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)                        # ties: the lowest index first
    w = torch.exp((xs - xs[:, :1]) / t)
    keep = (torch.arange(V, device="cuda") < k) | (k <= 0)
    w_k = w * keep
    ahead = w_k.cumsum(1) - w_k
    keep &= (ahead < p * w_k.sum(1, keepdim=True)) | (p <= 0) | (p >= 1)
    keep &= (w >= min_p) | (min_p <= 0)
    w = torch.zeros_like(w).scatter_(1, order, w * keep)                                  # drawn in the order of the vocabulary
    total = w.cumsum(1)
    want = s["coin"].double()[:, None] * total[:, -1:]
    token = (total <= want).sum(1).clamp_(max=V - 1)
    token = torch.where(greedy, order[:, 0], token)
    prob = torch.where(greedy, torch.ones_like(t[:, 0]), w.gather(1, token[:, None])[:, 0] / total[:, -1])
    return {"tokens": token.int(), "prob": prob.float()}


def run(state):
    if own:
        return _run_own(state)
    return {"tables": _plain_tables, "shared": _plain_shared, "sample": _plain_sample}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------------------
# the work that a case cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "tables":
        held, new = _lengths(case, 1)
        n, lead, rows = case["requests"], case["shared"], int(new.sum())
        pages = int((_pages(held + new) - _pages(held)).sum())
        # lengths, table rows, free pages and the shared prompt's in; pages, rows (position, table row, line), starts and lengths out
        return {"bytes": 12 * n + 4 * (pages + lead) + 4 * (pages + lead * n) + 12 * rows + 4 * n + 4 * n, "flops": 8 * n + 4 * rows}
    if case["kind"] == "sample":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": case["rows"] * case["vocab"] * 8}
    H, kv, hs = case["heads"], case["kv_heads"], case["head_size"]
    pos, groups = _rows(case, 1)
    tokens = sum(p + 1 for p in pos)
    lines = tokens - sum((e - b - 1) * p * PAGE for b, e, p in groups)                    # a group's shared part once
    return {"bytes": lines * kv * hs * 4 + len(pos) * H * hs * 6, "flops": 4 * tokens * H * hs}


def _exact_tables(case, seed):
    s = _prepare_tables(case, seed)
    table, free = s["table"].tolist(), s["free"].tolist()
    held, new, seq = s["held"].tolist(), s["new"].tolist(), s["seq"].tolist()
    cap, lead = len(s["pos"]), case["shared"]
    pos, slot, line, start, at = [], [], [], [0], 7
    for h, c, q in zip(held, new, seq):
        row = table[q]
        row[:lead] = table[-1][:lead]
        for p in range(-(-h // PAGE), -(-(h + c) // PAGE)):
            row[p] = free[at]
            at += 1
        for x in range(h, h + c):
            pos.append(x)
            slot.append(q)
            line.append(row[x // PAGE] * PAGE + x % PAGE)
        start.append(len(pos))
    gap = cap - len(pos)
    out = (table, pos + [-1] * gap, slot + [0] * gap, line + [-1] * gap, start, [h + c for h, c in zip(held, new)], [at], [0])
    return {x: _i32(v) for x, v in zip(_TABLES, out)}


def _exact_shared(case, seed):
    s = _prepare_shared(case, seed)
    H, kv, hs = case["heads"], case["kv_heads"], case["head_size"]
    y = torch.empty(len(s["pos"]), H, hs, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(-1, H, hs)
    for m, p in enumerate(s["pos"].tolist()):                                             # every row by itself, over its own table
        pages = s["table"][m, :p // PAGE + 1].long()
        k, v = (s[x][pages].double().transpose(0, 1).flatten(1, 2)[:, :p + 1] for x in ("k", "v"))
        a = torch.softmax(torch.einsum("hgd,htd->hgt", q[m].view(kv, -1, hs), k) * hs ** -0.5, -1)
        y[m] = torch.einsum("hgt,htd->hgd", a, v).reshape(H, hs)
    return y.flatten(1)


def _exact_sample(case, seed):
    import numpy as np
    s = _prepare_sample(case, seed)
    tokens, prob = [], []
    k, p, min_p, t, u = (s[x].cpu().numpy().astype(np.float64) for x in ("top_k", "top_p", "min_p", "temperature", "coin"))
    for m in range(case["rows"]):
        x = s["logits"][m].double().cpu().numpy()
        if t[m] <= 0:
            tokens.append(int(np.argmax(x)))
            prob.append(1.0)
            continue
        order = np.argsort(-x, kind="stable")
        w = np.exp((x - x.max()) / t[m])
        n = len(x) if k[m] <= 0 else min(len(x), int(k[m]))                               # what is kept is the front of the order
        sums = np.cumsum(w[order[:n]])
        if 0 < p[m] < 1:
            n = min(n, int(np.searchsorted(sums, p[m] * sums[-1], side="left")) + 1)
        if min_p[m] > 0:
            n = min(n, max(1, int((w >= min_p[m]).sum())))
        left = np.sort(order[:n])
        sums = np.cumsum(w[left])
        i = min(n - 1, int(np.searchsorted(sums, u[m] * sums[-1], side="right")))
        tokens.append(int(left[i]))
        prob.append(w[left[i]] / sums[-1])
    return {"tokens": _i32(tokens), "prob": torch.tensor(prob, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    return {"tables": _exact_tables, "shared": _exact_shared, "sample": _exact_sample}[case["kind"]](case, seed)
