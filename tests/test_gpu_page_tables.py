"""page_tables against a plain implementation: whole numbers, all of them equal."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE = 32


def K():
    from dllama_b200.ops import kernels
    return kernels


def oracle(c):
    """What a call leaves, from the arguments before it (dict of numpy arrays and lists)."""
    k = K()
    n, table, free, n_pages, M = len(c["held"]), c["table"].copy(), c["free"], c["n_pages"], c["M"]
    lead = c.get("lead")
    bad, seen, rows = 0, set(), 0
    need = [-(-(int(h) + int(x)) // PAGE) - -(-int(h) // PAGE) for h, x in zip(c["held"], c["new"])]
    has = {s: -(-int(h) // PAGE) for s, h, x in zip(c["seq"], c["held"], need) if x > 0}      # of rows that get pages
    led = {s for s, (t, l) in zip(c["seq"], lead) if l > 0 and t != s} if lead else set()
    for i, (h, x, s) in enumerate(zip(c["held"], c["new"], c["seq"])):
        if h < 0 or x < 0 or int(h) + int(x) > table.shape[1] * PAGE:
            bad |= k.TABLES_BAD_LENGTH
            continue
        if not 0 <= s < table.shape[0] or s in seen:
            bad |= k.TABLES_BAD_SEQ
        seen.add(s)
        if lead:
            t, l = lead[i]
            if l < 0 or l * PAGE > h or (l > 0 and (not 0 <= t < table.shape[0] or (t != s and (t in led or l > has.get(t, l))))):
                bad |= k.TABLES_BAD_LEAD
    ok_lengths = not bad & k.TABLES_BAD_LENGTH
    if ok_lengths:
        if sum(c["new"]) > M:
            bad |= k.TABLES_NO_ROWS
        if c["taken"] < 0 or c["taken"] + sum(need) > len(free):
            bad |= k.TABLES_NO_PAGES
        elif any(not 0 <= p < n_pages for p in free[c["taken"]:c["taken"] + sum(need)]):
            bad |= k.TABLES_BAD_PAGE
    out = {"pos": [], "slot": [], "line": [], "start": [0], "held": list(c["held"]), "taken": c["taken"], "status": bad}
    if not bad:
        before = table.copy()
        at = c["taken"]
        for i, (h, x, s) in enumerate(zip(c["held"], c["new"], c["seq"])):
            for q in range(need[i]):
                table[s, -(-h // PAGE) + q] = free[at]
                at += 1
        for i, s in enumerate(c["seq"]):
            if lead and lead[i][1]:
                table[s, :lead[i][1]] = before[lead[i][0], :lead[i][1]]
        for h, x, s in zip(c["held"], c["new"], c["seq"]):
            for p in range(h, h + x):
                page = int(table[s, p // PAGE])
                out["pos"].append(p)
                out["slot"].append(s)
                out["line"].append(page * PAGE + p % PAGE if 0 <= page < n_pages else -1)
            out["start"].append(len(out["pos"]))
        out["taken"], out["held"] = at, [h + x for h, x in zip(c["held"], c["new"])]
    else:
        out["start"] = [0] * (n + 1)
    gap = M - len(out["pos"])
    for x, fill in (("pos", -1), ("slot", 0), ("line", -1)):
        out[x] += [fill] * gap
    return {**out, "table": table}


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int64), dtype=torch.int32).cuda()


def run(c, in_place=False, line=True, start=True, pdl=False):
    n, M = len(c["held"]), c["M"]
    t = {x: i32(c[x]) for x in ("held", "new", "seq", "table", "free")}
    taken, status = i32([c["taken"]]), i32([77])
    pos, slot, ln, st = (torch.full((size,), -5, dtype=torch.int32, device="cuda") for size in (M, M, M, n + 1))
    held_out, taken_out = (t["held"], taken) if in_place else (i32([-5] * n), i32([-5]))
    lead = c.get("lead")
    K().page_tables(n, t["held"], t["new"], t["seq"], t["table"], t["free"], taken, c["n_pages"], pos, slot, status, line=ln if line else None, start=st if start else None,
                    held_out=None if in_place else held_out, taken_out=None if in_place else taken_out, lead_seq=i32([x[0] for x in lead]) if lead else None,
                    lead_pages=i32([x[1] for x in lead]) if lead else None, pdl=pdl)
    got = {"pos": pos, "slot": slot, "held": held_out, "taken": taken_out, "status": status, "table": t["table"]}
    if line:
        got["line"] = ln
    if start:
        got["start"] = st
    return {x: v.cpu().numpy() for x, v in got.items()}


def check(c, **how):
    want, got = oracle(c), run(c, **how)
    for x, v in got.items():
        assert np.array_equal(v.reshape(-1), np.asarray(want[x], dtype=np.int64).reshape(-1)), x
    return want


def case(rng, n, context, new, width=None, spare_rows=5, extra_seqs=3, taken=3, lead=0):
    held = rng.integers(0, context + 1, n)
    count = rng.integers(0, new + 1, n)
    if lead:
        held = np.maximum(held, lead * PAGE)
    width = width or int((held + count).max(initial=0)) // PAGE + 2
    pages = int(sum(-(-(h + x) // PAGE) - -(-h // PAGE) for h, x in zip(held, count)))
    seqs = n + extra_seqs
    n_pages = seqs * width + pages + taken + 4
    perm = rng.permutation(n_pages)
    table = perm[:seqs * width].reshape(seqs, width)
    free = perm[seqs * width:]
    c = {"held": held.tolist(), "new": count.tolist(), "seq": rng.permutation(seqs - 1)[:n].tolist(), "table": table, "free": free.tolist(), "taken": taken, "n_pages": n_pages,
         "M": int(count.sum()) + spare_rows}
    if lead:
        c["lead"] = [(seqs - 1, int(rng.integers(0, lead + 1))) for _ in range(n)]
    return c


@pytest.mark.parametrize("n,context,new", [(1, 0, 1), (1, 31, 1), (1, 32, 1), (1, 100, 5000), (3, 64, 0), (32, 3000, 1), (33, 500, 40), (200, 4000, 300), (1025, 200, 9), (5000, 60, 3), (8192, 40, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_tables(n, context, new, in_place):
    rng = np.random.default_rng(n * 7 + new)
    check(case(rng, n, context, new), in_place=in_place)
    check(case(rng, n, context, new, spare_rows=0, taken=0), in_place=in_place, line=False)
    check(case(rng, n, context, new, lead=3), in_place=in_place, start=False, pdl=True)


def test_long_shared_prompts():
    rng = np.random.default_rng(2)
    check(case(rng, 300, 9000, 20, lead=400))
    check(case(rng, 3, 100000, 40, lead=3000), in_place=True)


def test_a_lead_may_be_a_request_and_a_row_its_own():
    rng = np.random.default_rng(4)
    c = case(rng, 6, 300, 50)
    c["held"][0] = 320
    for i in range(1, 6):
        c["held"][i] = max(c["held"][i], 10 * PAGE)
    c["table"] = np.arange(c["table"].shape[0] * 20).reshape(-1, 20)
    c["n_pages"] = 10 ** 6
    c["free"] = list(range(500000, 501000))
    c["lead"] = [(c["seq"][0], 10)] * 6                        # the first one's own
    assert check(c)["status"] == 0


@pytest.mark.parametrize("n", [6, 2500])
def test_a_lead_that_gets_pages_leads_with_those_it_held(n):
    """Pages that a call takes for one request are no lead for another one: nothing says which of the two comes first."""
    rng = np.random.default_rng(6)
    for held, status in ((320, 0), (289, 0), (288, K().TABLES_BAD_LEAD), (0, K().TABLES_BAD_LEAD)):      # 10, 10, 9 and no pages
        c = case(rng, n, 300, 50)
        c["held"] = [max(h, 10 * PAGE) for h in c["held"]]
        i = n // 2
        c["held"][i], c["new"][i] = held, 350
        c["table"] = np.arange(c["table"].shape[0] * 24).reshape(-1, 24)
        c["n_pages"], c["free"], c["M"] = 10 ** 6, list(range(500000, 520000)), n * 50 + 400
        c["lead"] = [(c["seq"][i], 10 if j != i else 0) for j in range(n)]
        assert check(c)["status"] == status
        check(c, in_place=True)


def test_no_requests_and_no_rows():
    rng = np.random.default_rng(5)
    c = case(rng, 4, 100, 10)
    c.update(held=[], new=[], seq=[])
    assert check(c)["taken"] == 3
    c = case(rng, 4, 100, 0, spare_rows=0)
    check(c)
    c = case(rng, 4, 100, 0)
    c["free"] = []
    c["taken"] = 0
    check(c, in_place=True)


def test_a_page_that_is_none_has_no_lines():
    rng = np.random.default_rng(6)
    c = case(rng, 5, 100, 9)
    c["held"] = [5, 37, 64, 90, 1]
    c["new"] = [9, 3, 4, 8, 2]
    c["M"] = 40
    c["table"][:] = -1
    check(c)


@pytest.mark.parametrize("what", ["length", "negative", "negative_new", "huge", "seq", "twice", "seq_high", "lead", "lead_chain", "lead_seq", "lead_negative", "pages", "taken", "bad_page", "rows", "several"])
@pytest.mark.parametrize("n", [7, 3000])
def test_what_is_wrong_is_said_and_nothing_is_done(what, n):
    k = K()
    rng = np.random.default_rng(8)
    c = case(rng, n, 400, 12, lead=2)
    c["new"][n // 2] = 12
    c["M"] += 12
    c["n_pages"] += 1
    c["free"].append(c["n_pages"] - 1)
    i = n // 3
    want = {"length": k.TABLES_BAD_LENGTH, "negative": k.TABLES_BAD_LENGTH, "negative_new": k.TABLES_BAD_LENGTH, "huge": k.TABLES_BAD_LENGTH, "seq": k.TABLES_BAD_SEQ, "twice": k.TABLES_BAD_SEQ,
            "seq_high": k.TABLES_BAD_SEQ, "lead": k.TABLES_BAD_LEAD, "lead_chain": k.TABLES_BAD_LEAD, "lead_seq": k.TABLES_BAD_LEAD, "lead_negative": k.TABLES_BAD_LEAD, "pages": k.TABLES_NO_PAGES,
            "taken": k.TABLES_NO_PAGES, "bad_page": k.TABLES_BAD_PAGE, "rows": k.TABLES_NO_ROWS, "several": k.TABLES_BAD_SEQ | k.TABLES_NO_ROWS}[what]
    if what == "length":
        c["new"][i] = c["table"].shape[1] * PAGE
    if what == "negative":
        c["held"][i] = -1
    if what == "negative_new":
        c["new"][i] = -3
    if what == "huge":
        c["held"][i], c["new"][i] = 2 ** 31 - 1, 2 ** 31 - 1
    if what == "seq":
        c["seq"][i] = -1
    if what == "twice":
        c["seq"][i] = c["seq"][i + 1]
    if what == "seq_high":
        c["seq"][i] = c["table"].shape[0]
    if what == "lead":
        c["lead"][i] = (c["lead"][i][0], c["held"][i] // PAGE + 1)
    if what == "lead_chain":
        c["lead"][i], c["lead"][i + 1] = (c["lead"][i][0], 1), (c["seq"][i], 1)
    if what == "lead_seq":
        c["lead"][i] = (2 ** 31 - 1, 1)
    if what == "lead_negative":
        c["lead"][i] = (0, -1)
    if what == "pages":
        used = sum(-(-(h + x) // PAGE) - -(-h // PAGE) for h, x in zip(c["held"], c["new"]))
        c["free"] = c["free"][:c["taken"] + used - 1]
    if what == "taken":
        c["taken"] = -1
    if what == "bad_page":
        c["free"][c["taken"]] = c["n_pages"]
    if what in ("rows", "several"):
        c["M"] = sum(c["new"]) - 1
    if what == "several":
        c["seq"][i] = c["seq"][i + 1]
    assert check(c)["status"] == want
    check(c, in_place=True)


def test_a_loop_of_steps_in_a_graph():
    """Lengths and pages go on in place from replay to replay until the list is empty; the steps behind take nothing."""
    k = K()
    rng = np.random.default_rng(10)
    c = case(rng, 9, 100, 1, width=40)
    c["new"] = [1] * 9
    c["M"] = 16
    c["free"] = c["free"][:3 + 12]
    t = {x: i32(c[x]) for x in ("held", "new", "seq", "table", "free")}
    taken, status = i32([c["taken"]]), i32([0])
    pos, slot, line = (torch.zeros(16, dtype=torch.int32, device="cuda") for _ in range(3))
    args = (9, t["held"], t["new"], t["seq"], t["table"], t["free"], taken, c["n_pages"], pos, slot, status)
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        k.page_tables(*args, line=line, pdl=True)
    ran_dry = False
    for _ in range(60):
        want = oracle(c)
        g.replay()
        torch.cuda.synchronize()
        assert pos.tolist() == want["pos"] and slot.tolist() == want["slot"] and line.tolist() == want["line"]
        assert t["held"].tolist() == want["held"] and taken.tolist() == [want["taken"]] and status.tolist() == [want["status"]]
        assert np.array_equal(t["table"].cpu().numpy(), want["table"])
        c.update(held=want["held"], taken=want["taken"], table=want["table"])
        ran_dry |= want["status"] == k.TABLES_NO_PAGES
    assert ran_dry
