"""What the calls of a serving step count as launches: no rows, none."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_rows_no_launch():
    from dllama_b200.ops import kernels as K
    f32, i32 = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    kv = torch.zeros(6, 2, 32, 64, dtype=torch.float16, device="cuda")
    work = K.shared_attention_workspace(4, 4, 2, 64, "cuda")
    for M, want in ((0, (0, 0, 1)), (3, (1, 2, 1))):
        counts = []
        before = K.lib.launch_count
        tokens = torch.full((4,), -9, dtype=torch.int32, device="cuda")
        K.sample_tokens(torch.zeros(4, 50, device="cuda"), M, f32, None, None, None, f32, tokens)
        counts.append(K.lib.launch_count - before)
        before = K.lib.launch_count
        y = torch.zeros(4, 256, device="cuda")
        K.shared_attention(torch.zeros(4, 256, device="cuda"), M, 4, i32, i32, torch.zeros(4, 3, dtype=torch.int32, device="cuda"), i32, kv, kv.clone(), work, y_out=y)
        counts.append(K.lib.launch_count - before)
        before = K.lib.launch_count
        status = torch.full((1,), 9, dtype=torch.int32, device="cuda")
        K.page_tables(0, i32, i32, i32, torch.zeros(4, 3, dtype=torch.int32, device="cuda"), i32, torch.zeros(1, dtype=torch.int32, device="cuda"), 4, i32[:M].clone(), i32[:M].clone(), status)
        counts.append(K.lib.launch_count - before)
        assert tuple(counts) == want
        assert tokens.tolist() == [0] * M + [-9] * (4 - M) and status.item() == 0
