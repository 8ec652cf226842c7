"""What sample_tokens and page_tables refuse, without a GPU: from Python, and at the C entries."""
import pytest
import torch

from dllama_b200.ops import kernels as K
from dllama_b200.ops import lib


@pytest.fixture(autouse=True)
def _here(monkeypatch):
    """Tensors without a GPU stand on the current device, so that checks end ahead of a launch."""
    monkeypatch.setattr(K, "_launching", lambda t, what: -1)


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _sample(**change):
    a = {"logits": torch.zeros(4, 50), "M": 4, "temperature": torch.ones(4), "top_k": i32(4), "top_p": torch.zeros(4), "min_p": torch.zeros(4), "coin": torch.zeros(4), "tokens_out": i32(4),
         "prob_out": torch.zeros(4)}
    a.update(change)
    K.sample_tokens(**a)


@pytest.mark.parametrize("change", [
    {"logits": torch.zeros(4, 50, dtype=torch.float64)}, {"logits": torch.zeros(4, 50, 2)}, {"logits": torch.zeros(50, 4).t()}, {"M": 5}, {"M": -1}, {"logits": torch.zeros(4, 0)},
    {"logits": torch.zeros(1, 524289).expand(4, 524289)}, {"logits": torch.zeros(1, 50).expand(4, 50)}, {"temperature": None}, {"temperature": torch.ones(3)}, {"temperature": torch.ones(4).double()},
    {"temperature": torch.ones(8)[::2]}, {"top_k": torch.zeros(4)}, {"top_k": i32(3)}, {"top_p": i32(4)}, {"min_p": torch.zeros(2)}, {"coin": None}, {"coin": torch.zeros(4).half()},
    {"tokens_out": None}, {"tokens_out": torch.zeros(4, dtype=torch.int64)}, {"tokens_out": i32(3)}, {"prob_out": torch.zeros(4).double()}, {"prob_out": torch.zeros(3)}])
def test_sample_tokens_refuses(change):
    with pytest.raises(ValueError):
        _sample(**change)


def _tables(**change):
    a = {"n": 3, "held": i32(3), "new": i32(3), "seq": i32(3), "block_table": i32(5, 7), "free_pages": i32(9), "taken": i32(1), "n_pages": 40, "pos": i32(8), "slot": i32(8), "status": i32(1)}
    a.update(change)
    K.page_tables(**a)


@pytest.mark.parametrize("change", [
    {"n": -1}, {"n": 4}, {"n": 8193}, {"held": None}, {"new": None}, {"seq": i32(2)}, {"held": torch.zeros(3)}, {"new": torch.zeros(3, dtype=torch.int64)}, {"seq": i32(6)[::2]}, {"block_table": i32(35)}, {"block_table": None},
    {"block_table": torch.zeros(5, 7)}, {"block_table": i32(7, 5).t()}, {"block_table": i32(0, 7)}, {"block_table": i32(5, 0)}, {"block_table": i32(131073, 1)}, {"free_pages": None},
    {"free_pages": torch.zeros(9)}, {"taken": i32(0)}, {"n_pages": 0}, {"n_pages": (1 << 26) + 1}, {"pos": None}, {"slot": i32(7)}, {"line": i32(7)}, {"start": i32(3)}, {"held_out": i32(2)},
    {"taken_out": i32(0)}, {"status": None}, {"status": torch.zeros(1)}, {"lead_seq": i32(3)}, {"lead_pages": i32(3)}, {"lead_seq": i32(3), "lead_pages": i32(2)}])
def test_page_tables_refuses(change):
    with pytest.raises(ValueError):
        _tables(**change)


def test_the_c_entries_refuse():
    L = lib.cuda_lib()
    p = torch.zeros(64, dtype=torch.int32).data_ptr()
    assert L.dl_sample_tokens(p, 0, 2, 0, 8, p, p, p, p, p, p, p, 0, None) == -1
    assert L.dl_sample_tokens(p, 0, 2, 524289, 524289, p, p, p, p, p, p, p, 0, None) == -1
    assert L.dl_sample_tokens(p, 0, 2, 8, 7, p, p, p, p, p, p, p, 0, None) == -1
    assert L.dl_sample_tokens(p, 3, 2, 8, 8, p, p, p, p, p, p, p, 0, None) == -1
    assert L.dl_sample_tokens(None, 0, 2, 8, 8, p, p, p, p, p, p, p, 0, None) == -1
    assert L.dl_sample_tokens(p, 0, 0, 8, 8, p, p, p, p, p, p, p, 0, None) == 0      # no rows: nothing to do
    ok = dict(n=1, held=p, new=p, seq=p, table=p, n_seqs=1, max_pages=1, free=p, n_free=1, taken=p, n_pages=1, M=1, pos=p, slot=p, line=p, start=p, held_out=p, taken_out=p, status=p, ls=None, lp=None)
    for change in ({"n": -1}, {"n": 8193}, {"n_seqs": 0}, {"n_seqs": 131073}, {"max_pages": 0}, {"max_pages": (1 << 25) + 1}, {"n_free": -1}, {"n_free": (1 << 30) + 1}, {"n_pages": 0}, {"M": -1}, {"M": (1 << 30) + 1}, {"held": None}, {"table": None},
                   {"free": None}, {"taken": None}, {"pos": None}, {"held_out": None}, {"status": None}, {"ls": p}, {"lp": p}):
        assert L.dl_page_tables(*{**ok, **change}.values(), 0, None) == -1
    assert b"null" in L.dl_last_error()
    assert L.dl_page_tables_packed(None) == -1
    packed = lambda **kw: K._TABLES_ARGS.pack(*[v or 0 for v in {**ok, **kw}.values()], 0, 0)
    assert L.dl_page_tables_packed(packed(n=1 << 40)) == -1 and L.dl_page_tables_packed(packed(n=8193)) == -1 and L.dl_page_tables_packed(packed(table=None)) == -1


def _shared(monkeypatch, **change):
    monkeypatch.setattr(K, "_current_device", lambda: -1)
    monkeypatch.setattr(K, "_kv8_rows", lambda *a: (0, 0, 0, a[0], 4, 3))
    kv = torch.zeros(6, 2, 32, 64, dtype=torch.float16)
    a = {"q": torch.zeros(4, 4 * 64), "M": 4, "n_heads": 4, "pos": i32(4), "slot": i32(4), "block_table": i32(4, 3), "groups": i32(4), "k_cache": kv, "v_cache": kv.clone(),
         "workspace": torch.zeros(1 << 22, dtype=torch.uint8), "y_out": torch.zeros(4, 4 * 64)}
    monkeypatch.setattr(K, "_shared_bytes", lambda *a: 1 << 22)
    a.update(change)
    K.shared_attention(**a)


@pytest.mark.parametrize("change", [
    {"k_cache": torch.zeros(6, 2, 32, 64)}, {"k_cache": torch.zeros(6, 2, 32, 32).half()}, {"k_cache": torch.zeros(6, 2, 16, 64).half()}, {"v_cache": torch.zeros(5, 2, 32, 64).half()},
    {"v_cache": torch.zeros(6, 2, 32, 64)}, {"k_cache": torch.zeros(6, 32, 2, 64).half().transpose(1, 2)}, {"n_heads": 3}, {"n_heads": 0}, {"n_heads": 34, "q": torch.zeros(4, 34 * 64)},
    {"q": torch.zeros(4, 255)}, {"q": torch.zeros(3, 256)}, {"q": torch.zeros(4, 256).half()}, {"q": torch.zeros(4, 258)[:, 2:]}, {"q": torch.zeros(4, 257)[:, :256]}, {"q": None}, {"groups": None},
    {"groups": torch.zeros(4)}, {"groups": i32(0)}, {"groups": i32(8)[::2]}, {"workspace": None}, {"workspace": torch.zeros(100, dtype=torch.uint8)}, {"y_out": torch.zeros(4, 256).double()},
    {"y_out": torch.zeros(4, 255)}, {"M": 65536}, {"xq_out": torch.zeros(10, dtype=torch.uint8), "out_mcap": 4}, {"xh_out": torch.zeros(1 << 20, dtype=torch.uint8), "out_mcap": 3}])
def test_shared_attention_refuses(monkeypatch, change):
    with pytest.raises(ValueError):
        _shared(monkeypatch, **change)


def test_the_c_entry_of_shared_attention_refuses():
    L = lib.cuda_lib()
    p = torch.zeros(1 << 16, dtype=torch.int32).data_ptr() // 16 * 16
    ok = dict(q=p, ldq=256, H=4, kv=2, hs=64, k=p, v=p, n_pages=6, pos=p, slot=p, bt=p, M=2, n_slots=2, max_pages=4, groups=p, max_groups=1, scratch=p, bytes=1 << 40, xq=None, xh=None, mcap=0, y=p, ldy=256,
              yt=0)
    for change in ({"hs": 32}, {"H": 3}, {"kv": 0}, {"H": 34}, {"M": -1}, {"M": 65536}, {"n_slots": 0}, {"max_pages": 0}, {"max_pages": 1 << 26}, {"n_pages": 0}, {"n_pages": 1 << 26}, {"max_groups": -1},
                   {"q": None}, {"k": None}, {"pos": None}, {"groups": None}, {"scratch": None}, {"bytes": 100}, {"ldq": 255}, {"ldq": 258}, {"q": p + 4}, {"k": p + 2}, {"ldy": 255}, {"yt": 3},
                   {"max_pages": 1 << 25, "M": 60000}):
        assert L.dl_shared_attention(*{**ok, **change}.values(), 0, None) == -1, change
    assert L.dl_shared_attention(*{**ok, "M": 0}.values(), 0, None) == 0
