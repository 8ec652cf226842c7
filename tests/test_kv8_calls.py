"""What the 8-bit token cache's Python calls give and refuse, without a GPU (beside test_kv8.py)."""
import pytest
import torch

from dllama_b200.ops import kernels as K


@pytest.mark.parametrize("M,heads,kv", [(64, 32, 8), (64, 256, 256), (64, 1024, 64), (64, 1040, 65), (64, 2048, 128), (33, 2048, 128), (32, 2048, 128), (31, 2064, 129), (1, 2048, 128), (64, 300, 300)])
def test_splits_that_the_library_takes(M, heads, kv):
    """A counter for each row, key/value head and four query heads of it: where they are more than the scratch has room for, rows have one share."""
    units = M * kv * ((heads // kv + 3) // 4)
    want = max(1, min(512 // M, 32)) if units <= 65536 // 4 else 1
    assert K.kv8_attention_splits(M, heads, kv, 4096) == want


class _Here:
    """A cache that stands on the current device, for checks that end ahead of a launch."""

    def __init__(self, monkeypatch):
        codes, scales = (torch.zeros(3, 2, 32, 64, dtype=torch.int8) for _ in range(2)), (torch.zeros(3, 2, 32) for _ in range(2))
        self.cache = K.Kv8Cache(*codes, *scales)
        self.cache.index = -1                                      # where tensors without a GPU are
        monkeypatch.setattr(K, "_kv8_rows", lambda *a: (0, 0, 0, 4, 1, 3))


@pytest.mark.parametrize("missing", ["qkv", "q_out", "k_out", "v_out", "q"])
def test_a_missing_tensor_is_a_value_error(monkeypatch, missing):
    c = _Here(monkeypatch).cache
    has = lambda name, *shape: None if name == missing else torch.zeros(*shape)
    with pytest.raises(ValueError):
        if missing in ("qkv", "q_out"):
            K.kv8_write(has("qkv", 4, 512), 4, 4, None, None, None, None, has("q_out", 4, 256), c)
        elif missing == "q":
            K.kv8_attention(None, 4, 4, None, None, None, c, 1, None, y_out=torch.zeros(4, 256))
        else:
            K.kv8_read(4, None, None, None, c, has("k_out", 4, 128), has("v_out", 4, 128))
    if missing == "q":
        with pytest.raises(ValueError):
            K.kv8_attention_prefill(None, 4, 4, None, None, None, torch.zeros(3, dtype=torch.int32), c, y_out=torch.zeros(4, 256))
