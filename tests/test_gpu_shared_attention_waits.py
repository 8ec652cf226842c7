"""shared_attention whose waits run out: a limit that is over at once, under which no page is copied."""
import ctypes

import pytest
import torch

from test_gpu_shared_attention import Batch

pytestmark = pytest.mark.gpu


# one tile in both places, one step of it alone, two tiles, several items of a CTA, rows of no group among all of them
@pytest.mark.parametrize("groups,heads,kv,hs", [([(11, 60, 40), (2, 0, 90)], 8, 2, 128), ([(3, 3, 40), (1, 0, 50)], 32, 8, 128), ([(70, 25, 50), (3, 0, 70)], 8, 1, 128), ([(33, 20, 40), (5, 0, 40)], 64, 8, 64),
                                                ([(2, 1, 40), (3, 2, 30), (1, 0, 50), (2, 1, 40), (4, 5, 20), (2, 0, 20)], 16, 8, 64), ([(2, 1, 9)] * 8 + [(4, 0, 40)], 32, 8, 128)])
def test_waits_that_run_out_reach_the_caller(groups, heads, kv, hs):
    """The kernel ends, the rows of groups are NaN, those of no group what they were, and the status word changes for that launch and not for the next one, which is right."""
    from dllama_b200.ops import lib as B
    library = B.cuda_lib()
    b = Batch(len(groups) + heads, groups, heads, kv, hs)
    before = b.run()
    torch.cuda.synchronize()
    status = B.WaitStatus(library)
    status.check()
    library.dl_debug_set_wait_limit.argtypes = [ctypes.c_ulonglong]
    library.dl_debug_set_wait_limit(0)
    try:
        y = b.run()
        torch.cuda.synchronize()
    finally:
        library.dl_debug_set_wait_limit(4_000_000_000)
    with pytest.raises(B.NativeLibraryError, match="gave up"):
        status.check()
    shared = torch.zeros(b.M, dtype=torch.bool)
    for begin, end, pages in b.ranges:
        shared[begin:end] = pages > 0
    assert torch.isnan(y[shared]).all() and torch.equal(y[~shared], before[~shared])
    after = b.run()
    torch.cuda.synchronize()
    status.check()
    assert torch.equal(after, before)
    b.check(after, rows=range(0, b.M, 3))
