"""sample_many's steps as they run in the end: behind a captured graph, on shared pages, with the tokens that it drew given to the engine's public calls."""
import numpy as np
import pytest
import torch

from test_gpu_sample_many import _engine, wide_heads_path  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [2, 4])
def test_what_is_to_be_shared_is_shared_beside_the_persistent_kernel(wide_heads_path, n, monkeypatch):  # noqa: F811
    """share=True on an engine whose batches of a few rows run on the persistent decode kernel, which knows no groups."""
    from dllama_b200.ops import kernels as K
    e = _engine(wide_heads_path, use_mega=True)
    assert e._mega_usable(n, False)
    calls = []
    shared = K.shared_attention
    monkeypatch.setattr(K, "shared_attention", lambda *a, **kw: (calls.append(a[1]), shared(*a, **kw)))
    prompt = np.random.default_rng(n).integers(1, 1024, 100).tolist()
    t = e.sample_many(prompt, n, 3, 1.0, seed=2, share=True)
    assert calls == [n] * 4 and t.shape == (n, 3)                  # two layers, a step launched and one captured
    calls.clear()
    e.sample_many(prompt, n, 3, 1.0, seed=2)
    assert not e.shares_prompt(n, 3) and calls == []
    e.close()
