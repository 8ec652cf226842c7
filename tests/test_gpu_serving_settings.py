"""top_k and min_p of any size through the serving loop: a request whose settings do not fit 32 bits is answered like any other, and so are its neighbours."""
import math

import pytest

from dllama_b200.serving.batch_engine import BatchEngine, GenerationRequest


def _engine(path, tmp_path, **kw):
    from dllama_b200.formats import tfile
    from dllama_b200.models.llama import LlamaEngine
    from dllama_b200.text import native as T
    tfile.write_synthetic_tokenizer(str(tmp_path / "tiny.t"), 1024)
    e = LlamaEngine(path, max_rows=32, n_slots=8, max_seq_len=256, bucket_rows=True)
    return e, BatchEngine(e, T.Tokenizer(str(tmp_path / "tiny.t")))


def _answers(be, reqs):
    reqs = [be.submit(r) for r in reqs]
    for _ in range(200):
        be.step()
        if all(r.finish_reason for r in reqs):
            break
    return [r.tokens for r in reqs]


@pytest.mark.gpu
def test_settings_beyond_32_bits(tiny_model_path, tmp_path):
    e, be = _engine(tiny_model_path, tmp_path)
    ask = lambda i, **kw: GenerationRequest([1, 5 + i, 9], max_tokens=10, seed=20 + i, **{"temperature": 0.9, "top_p": 0.95, **kw})
    small = [{"top_k": 7}, {"min_p": 0.2}, {}, {"min_p": 1.0}, {"top_k": 7, "min_p": 0.2}]
    plain = _answers(be, [ask(i, **kw) for i, kw in enumerate(small)])
    # what takes nothing out, and as much as there is, written in numbers of any size
    large = [{"top_k": 7, "min_p": -1e300}, {"top_k": 10 ** 12, "min_p": 0.2}, {"top_k": -10 ** 12}, {"min_p": 1e300}, {"top_k": 7.0, "min_p": 0.2}]
    assert _answers(be, [ask(i, **kw) for i, kw in enumerate(large)]) == plain
    large = [{"top_k": 7, "min_p": math.nan}, {"top_k": math.inf, "min_p": 0.2}, {"top_k": 1024, "min_p": 0.0}, {"min_p": math.inf}, {"top_k": 7, "min_p": 0.2}]
    assert _answers(be, [ask(i, **kw) for i, kw in enumerate(large)]) == plain
    assert be.n_errors == 0
    e.close()


def test_what_the_settings_mean():
    from dllama_b200.serving.filters import settings
    for (k, p), want in (((0, 0.0), (0, 0.0)), ((40, 0.0625), (40, 0.0625)), ((999, 1.0), (999, 1.0)), ((1000, 2.0), (0, 1.0)), ((10 ** 30, 1e300), (0, 1.0)), ((-(10 ** 30), -1e300), (0, 0.0)),
                         ((math.nan, math.nan), (0, 0.0)), ((math.inf, math.inf), (0, 1.0)), ((0.5, 2.0 ** -100), (0, 2.0 ** -100)), ((2.7, 0.0), (2, 0.0)), ((0, 1e-60), (0, 0.0))):
        assert settings(k, p, 1000) == want


@pytest.mark.gpu
def test_sample_many_with_a_min_p_beyond_32_bits(tiny_model_path):
    """Above 1 it is 1, however large: the first of the largest logits, as top_k 1."""
    from dllama_b200.models.llama import LlamaEngine
    e = LlamaEngine(tiny_model_path, max_rows=32, n_slots=8, max_seq_len=256)
    want = e.sample_many([1, 5, 9], 3, 8, 1.3, top_k=1, top_p=0.0)
    for min_p in (1.0, 7.0, 1e300, math.inf):
        assert (e.sample_many([1, 5, 9], 3, 8, 1.3, top_p=0.0, min_p=min_p) == want).all()
    assert (e.sample_many([1, 5, 9], 3, 8, 1.3, top_k=10 ** 30, top_p=0.0, min_p=1e300) == want).all()
    e.close()
