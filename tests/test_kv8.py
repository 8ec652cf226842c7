"""The 8-bit token cache without a GPU: what its entry points refuse, sizes, and the command line."""
import ctypes as C
import dataclasses

import pytest
import torch

from dllama_b200.ops import kernels as K
from dllama_b200.ops.lib import DlKv8Cache, NativeLibraryError, check


def _codes(n=3, kv=2, hs=64, **kw):
    return torch.zeros(n, kv, 32, hs, dtype=kw.get("dtype", torch.int8))


def _scales(n=3, kv=2, dtype=torch.float32):
    return torch.zeros(n, kv, 32, dtype=dtype)


def test_cache_checks_its_tensors():
    c = K.Kv8Cache(_codes(), _codes(), _scales(), _scales())
    assert (c.n_pages, c.n_kv_heads, c.head_size) == (3, 2, 64)
    assert c.nbytes() == 3 * K.kv8_page_bytes(2, 64) == sum(t.numel() * t.element_size() for t in (c.k, c.v, c.k_scale, c.v_scale))
    for bad in ((_codes(hs=48), _codes(hs=48), _scales(), _scales()), (_codes(), _codes(n=4), _scales(), _scales()), (_codes(), _codes(), _scales(n=2), _scales()),
                (_codes(dtype=torch.uint8), _codes(), _scales(), _scales()), (_codes(), _codes(), _scales(dtype=torch.float16), _scales()),
                (torch.zeros(3, 2, 16, 64, dtype=torch.int8), _codes(), _scales(), _scales()), (_codes(hs=128)[..., ::2], _codes(), _scales(), _scales()),
                (_codes(n=0), _codes(n=0), _scales(n=0), _scales(n=0)), (_codes()[0], _codes()[0], _scales()[0], _scales()[0])):
        with pytest.raises(ValueError):
            K.Kv8Cache(*bad)


def test_calls_refuse_a_cache_that_is_not_on_the_current_device():
    c = K.Kv8Cache(_codes(), _codes(), _scales(), _scales())
    i = torch.zeros(4, dtype=torch.int32)
    x, y, bt = torch.zeros(4, 8 * 64), torch.zeros(4, 4 * 64), torch.zeros(1, 3, dtype=torch.int32)
    with pytest.raises(ValueError):
        K.kv8_write(x, 4, 4, None, i, i, bt, y, c)
    with pytest.raises(ValueError):
        K.kv8_read(4, i, i, bt, c, x[:, :128], x[:, 128:256])
    with pytest.raises(ValueError):
        K.kv8_attention(y, 4, 4, i, i, bt, c, 1, None, y_out=y)
    with pytest.raises(ValueError):
        K.kv8_attention_prefill(y, 4, 4, i, i, bt, torch.tensor([1, 0, 4], dtype=torch.int32), c, y_out=y)


A = 4096                                                        # an aligned address that nothing follows: every call here ends ahead of a launch


def _cache(**kw):
    a = dict(k=A, v=A, k_scale=A, v_scale=A, n_pages=4, n_kv_heads=2, head_size=64)
    a.update(kw)
    return C.byref(DlKv8Cache(*a.values()))


def _rows(**kw):
    a = dict(pos=A, slot=A, table=A, M=4, n_slots=2, max_pages=3)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("cache,rows", [
    (dict(head_size=48), {}), (dict(head_size=256), {}), (dict(n_kv_heads=0), {}), (dict(n_pages=0), {}), (dict(k=None), {}), (dict(v_scale=None), {}), (dict(v=A + 8), {}),
    (dict(k_scale=A + 4), {}), ({}, dict(pos=None)), ({}, dict(slot=None)), ({}, dict(table=None)), ({}, dict(M=-1)), ({}, dict(n_slots=0)), ({}, dict(max_pages=0)),
    ({}, dict(max_pages=1 << 27)),
])
def test_library_refuses_caches_and_rows(cache, rows):
    L = K.cuda_lib()
    c, r = _cache(**cache), _rows(**rows)
    for rc in (L.dl_kv8_write(A, 512, 4, None, *r, A, 256, c, 0, None), L.dl_kv8_read(*r, c, A, A, 128, 0, 0, None),
               L.dl_kv8_attention(A, 256, 4, *r, c, 1, None, None, None, 0, A, 256, 0, None, 0, None),
               L.dl_kv8_attention_prefill(A, 256, 4, *r, A, 1, c, None, None, None, None, None, 0, A, 256, 0, 0, None)):
        with pytest.raises(NativeLibraryError):
            check(rc, "dl_kv8")


def test_library_refuses_arguments():
    L, c, r = K.cuda_lib(), _cache(), _rows()
    bad = [L.dl_kv8_write(A, 511, 4, None, *r, A, 256, c, 0, None), L.dl_kv8_write(A, 512, 4, None, *r, A, 255, c, 0, None), L.dl_kv8_write(None, 512, 4, None, *r, A, 256, c, 0, None),
           L.dl_kv8_write(A, 512, 4, None, *r, None, 256, c, 0, None), L.dl_kv8_write(A, 512, -1, None, *r, A, 256, c, 0, None),
           L.dl_kv8_read(*r, c, A, None, 128, 0, 0, None), L.dl_kv8_read(*r, c, A, A, 127, 0, 0, None), L.dl_kv8_read(*r, c, A, A, 128, 3, 0, None)]
    for heads, splits, scratch, xq, mcap, y, ldq, ldy, t in ((3, 1, None, None, 0, A, 256, 256, 0), (34, 1, None, None, 0, A, 4096, 4096, 0), (1, 1, None, None, 0, A, 256, 256, 0),
                                                             (4, 2, None, None, 0, A, 256, 256, 0), (4, 2, A + 4, None, 0, A, 256, 256, 0), (4, 65, A, None, 0, A, 256, 256, 0),
                                                             (4, 1, None, None, 0, None, 256, 256, 0), (4, 1, None, None, 0, A, 255, 256, 0), (4, 1, None, None, 0, A, 256, 255, 0),
                                                             (4, 1, None, None, 0, A, 256, 256, 5), (4, 1, None, A, 3, None, 256, 256, 0)):
        bad.append(L.dl_kv8_attention(A, ldq, heads, *r, c, splits, scratch, xq, None, mcap, y, ldy, t, None, 0, None))
    bad.append(L.dl_kv8_attention(A, 256, 4, *_rows(M=65536), c, 1, None, None, None, 0, A, 256, 0, None, 0, None))
    bad.append(L.dl_kv8_attention(A, 256, 4, *_rows(M=10000), c, 2, A, None, None, 0, A, 256, 0, None, 0, None))       # more units than there are counters
    bad.append(L.dl_kv8_attention_prefill(A, 256, 4, *r, A, 0, c, None, None, None, None, None, 0, A, 256, 0, 0, None))
    bad.append(L.dl_kv8_attention_prefill(A, 256, 4, *r, None, 1, c, None, None, None, None, None, 0, A, 256, 0, 0, None))
    bad.append(L.dl_kv8_attention_prefill(A, 256, 4, *r, A, 1, c, A, None, None, None, None, 0, A, 256, 0, 0, None))
    bad.append(L.dl_kv8_attention_prefill(A, 256, 4, *r, A, 1, c, None, None, A, None, None, 0, A, 256, 0, 0, None))
    assert all(rc != 0 for rc in bad), bad
    # nothing to do: no launch
    none = _rows(M=0)
    assert L.dl_kv8_write(A, 512, 4, None, *none, A, 256, c, 0, None) == 0 and L.dl_kv8_read(*none, c, A, A, 128, 0, 0, None) == 0
    assert L.dl_kv8_attention(A, 256, 4, *none, c, 1, None, None, None, 0, A, 256, 0, None, 0, None) == 0
    assert L.dl_kv8_attention_prefill(A, 256, 4, *none, A, 1, c, None, None, None, None, None, 0, A, 256, 0, 0, None) == 0


@pytest.mark.parametrize("M,heads,kv,pages,want", [(0, 32, 8, 6, 1), (1, 32, 8, 6, 1), (1, 32, 8, 125, 15), (1, 32, 8, 4000, 32), (16, 32, 8, 4000, 32), (32, 32, 8, 4000, 16), (7, 64, 8, 157, 19), (64, 32, 8, 100, 8), (65, 32, 8, 100, 1)])
def test_splits(M, heads, kv, pages, want):
    assert K.kv8_attention_splits(M, heads, kv, pages) == want


def test_workspace():
    w = K.kv8_prefill_workspace(3, 2, 128, 512, "cpu")
    assert w.k16.shape == w.v16.shape == (3, 2, 32, 128) and w.k16.dtype == torch.float16
    assert w.scratch.nbytes == K.cuda_lib().dl_kv8_prefill_scratch_bytes(128) > 17 * 4
    assert K.kv8_prefill_workspace(3, 2, 64, 512, "cpu").v16.shape == (3, 2, 32, 64)
    assert K.kv8_prefill_workspace(3, 2, 32, 512, "cpu") is None and K.kv8_prefill_workspace(3, 2, 128, 1, "cpu") is None
    assert [K.kv8_widens(128, 32, 128), K.kv8_widens(129, 32, 128), K.kv8_widens(129, 32, 64), K.kv8_widens(256, 32, 64), K.kv8_widens(4096, 32, 32)] == [False, True, False, True, False]


def test_command_line(tiny_model_path):
    from dllama_b200.cli.app import AppArgs, build_engine
    from dllama_b200.ops import quant
    base = ["dllama", "inference", "--model", "m", "--tokenizer", "t"]
    assert AppArgs.parse(base, True).kv_cache == "f16" and AppArgs.parse(base + ["--kv-cache", "q8"], True).kv_cache == "q8"
    with pytest.raises(ValueError):
        AppArgs.parse(base + ["--kv-cache", "int8"], True)
    with pytest.raises(ValueError):
        build_engine(tiny_model_path, 0, 1, 8, 2, 128, quant.Q80, "cpu", kv_cache="q8")


def test_required_memory_of_the_cache(tiny_model_path):
    from dllama_b200.formats.mfile import read_header
    from dllama_b200.models.memory import required_memory
    h = read_header(tiny_model_path, 0)
    f16, q8 = (required_memory(h, 1, n_slots=3, seq_len=64, kv_cache=t)["kv_cache"] for t in ("f16", "q8"))
    assert f16 == 2 * 2 * 3 * 64 * 4 * 32 * 2 and q8 == 2 * 3 * 2 * K.kv8_page_bytes(4, 32)
    wide = dataclasses.replace(h, dim=2048, n_heads=32, n_kv_heads=4)
    few, many = (required_memory(wide, 1, rows, n_slots=3, seq_len=64, kv_cache="q8")["kv_cache"] for rows in (64, 512))
    assert few == 2 * 3 * 2 * K.kv8_page_bytes(4, 64) and many == few + 3 * 64 * 2 * 256 * 2        # and fp16 pages of one layer
