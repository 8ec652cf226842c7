"""What the 8-bit token cache's Python calls give and refuse, without a GPU (beside test_kv8.py)."""
import pytest

from dllama_b200.ops import kernels as K


@pytest.mark.parametrize("M,heads,kv", [(64, 32, 8), (64, 256, 256), (64, 1024, 64), (64, 1040, 65), (64, 2048, 128), (33, 2048, 128), (32, 2048, 128), (31, 2064, 129), (1, 2048, 128), (64, 300, 300)])
def test_splits_that_the_library_takes(M, heads, kv):
    """A counter for each row, key/value head and four query heads of it: where they are more than the scratch has room for, rows have one share."""
    units = M * kv * ((heads // kv + 3) // 4)
    want = max(1, min(512 // M, 32)) if units <= 65536 // 4 else 1
    assert K.kv8_attention_splits(M, heads, kv, 4096) == want
