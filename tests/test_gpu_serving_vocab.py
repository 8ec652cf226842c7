"""A vocabulary beyond what sample_tokens takes: requests with top_k or min_p are refused when they come, and end no batch; the other ones are served."""
import json
import urllib.error
import urllib.request

import pytest

from dllama_b200.serving import batch_engine, filters, native_server
from dllama_b200.serving import api_types as A


def test_the_largest_vocabulary_is_the_kernels():
    from dllama_b200.ops import kernels as K
    assert filters.MAX_VOCAB == K._max_vocab()


@pytest.mark.gpu
def test_a_vocabulary_that_is_too_large(tiny_model_path, tmp_path, monkeypatch):
    """The limit set below the model's 1024 tokens stands in for a model of more than 524288."""
    from dllama_b200.formats import tfile
    from dllama_b200.models.llama import LlamaEngine
    from dllama_b200.text import native as T
    for m in (batch_engine, native_server):
        monkeypatch.setattr(m, "MAX_VOCAB", 1023)
    tfile.write_synthetic_tokenizer(str(tmp_path / "tiny.t"), 1024)
    tok = T.Tokenizer(str(tmp_path / "tiny.t"))
    e = LlamaEngine(tiny_model_path, max_rows=32, n_slots=8, max_seq_len=256, bucket_rows=True)
    be = batch_engine.BatchEngine(e, tok)
    ask = lambda **kw: batch_engine.GenerationRequest([1, 5, 9], max_tokens=4, temperature=0.9, **kw)
    for kw in ({"top_k": 5}, {"min_p": 0.1}):
        with pytest.raises(ValueError):
            be.submit(ask(**kw))
    r = be.submit(ask(top_k=1024))
    for _ in range(20):
        be.step()
        if r.finish_reason:
            break
    assert len(r.tokens) >= 1 and r.error is None
    srv = native_server.NativeApiServer(e, tok, "tiny.m", A.InferenceParams(messages=[], temperature=0.8, top_p=0.9, seed=1), host="127.0.0.1", port=0, verbose=False)
    srv.start()
    try:
        def post(**kw):
            body = {"messages": [{"role": "user", "content": "hello"}], "max_tokens": 4, **kw}
            req = urllib.request.Request(f"http://127.0.0.1:{srv.port}/v1/chat/completions", data=json.dumps(body).encode(), method="POST")
            with urllib.request.urlopen(req, timeout=60) as r:
                return json.load(r)["usage"]["completion_tokens"]
        assert post() >= 1
        for kw in ({"top_k": 5}, {"min_p": 0.1}):
            with pytest.raises(urllib.error.HTTPError) as err:
                post(**kw)
            assert err.value.code == 400
        assert srv.stats()["engine_errors"] == 0
    finally:
        srv.close()
    e.close()
