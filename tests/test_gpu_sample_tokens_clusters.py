"""sample_tokens where the CTAs of a row start at unlike times: short rows on clusters of every size, beside work of other streams that takes the SMs as they come free.  Tokens equal to the definition
in 64 bits."""
import numpy as np
import pytest
import torch

from test_gpu_sample_tokens import K, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(1, 8192), (1, 65536), (3, 32768), (9, 16384), (40, 8192), (70, 8200)])
@pytest.mark.parametrize("pdl", [False, True])
def test_clusters_that_start_beside_other_work(rows, vocab, pdl):
    k, rng = K(), np.random.default_rng(rows + vocab)
    x = rng.standard_normal((rows, vocab)) * 3
    t, kk, p, mp = [0.8] * rows, [(0, 40, 0)[m % 3] for m in range(rows)], [(0.9, 0.95, 0.0)[m % 3] for m in range(rows)], [(0.0, 0.0, 0.02)[m % 3] for m in range(rows)]
    logits = torch.from_numpy(x).float().cuda()
    f32, i32 = (lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")), (lambda v: torch.tensor(v, dtype=torch.int32, device="cuda"))
    args = [f32(t), i32(kk), f32(p), f32(mp)]
    coins = rng.random((60, rows)).astype(np.float32)
    coin = torch.from_numpy(coins).cuda()
    out = torch.full((60, rows), -9, dtype=torch.int32, device="cuda")
    a = torch.randn(1500, 1500, device="cuda")
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for s in side:                                               # grids of some hundred blocks, one behind the other
        with torch.cuda.stream(s):
            for _ in range(40):
                b = a @ a
    for i in range(60):
        k.sample_tokens(logits, rows, *args, coin[i], out[i], pdl=pdl)
    torch.cuda.synchronize()
    got, xs = out.tolist(), x.astype(np.float32)
    for i in range(0, 60, 7):
        assert got[i] == [oracle(xs[m], np.float32(t[m]), kk[m], np.float32(p[m]), np.float32(mp[m]), coins[i][m])[0] for m in range(rows)]
    assert min(map(min, got)) >= 0
