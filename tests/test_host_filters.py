"""top_k and min_p where the host samples: what takes nothing out is served, by the Python loop and by the native server."""
import json
import urllib.error
import urllib.request

import pytest

from dllama_b200.formats import tfile
from dllama_b200.models.cpu_engine import CpuEngine
from dllama_b200.serving import api_types as A
from dllama_b200.serving.batch_engine import BatchEngine, GenerationRequest
from dllama_b200.serving.native_server import NativeApiServer
from dllama_b200.text import native as T

VOCAB = 1024


@pytest.fixture(scope="module")
def tok(tmp_path_factory):
    p = str(tmp_path_factory.mktemp("tok") / "tiny.t")
    tfile.write_synthetic_tokenizer(p, VOCAB)
    return T.Tokenizer(p)


def _engine(path):
    return CpuEngine(path, max_rows=8, n_slots=4, max_seq_len=128)


def _loop(be, **kw):
    r = be.submit(GenerationRequest([1, 2, 3], max_tokens=4, seed=5, temperature=0.8, **kw))
    for _ in range(20):
        be.step()
        if r.finish_reason:
            return r.tokens


class _Server:
    def __init__(self, engine, tok):
        self.srv = NativeApiServer(engine, tok, "tiny.m", A.InferenceParams(messages=[], temperature=0.8, top_p=0.9, seed=1), host="127.0.0.1", port=0, verbose=False)

    def __enter__(self):
        self.srv.start()
        return self

    def __exit__(self, *a):
        self.srv.close()

    def post(self, **kw):
        body = {"messages": [{"role": "user", "content": "hello"}], "max_tokens": 4, "seed": 5, **kw}
        req = urllib.request.Request(f"http://127.0.0.1:{self.srv.port}/v1/chat/completions", data=json.dumps(body).encode(), method="POST")
        with urllib.request.urlopen(req, timeout=60) as r:
            return json.load(r)["choices"][0]["message"]["content"]


def test_what_takes_nothing_out_is_served(tiny_model_path, tok):
    e = _engine(tiny_model_path)
    be = BatchEngine(e, tok)
    plain = _loop(be)
    for kw in ({"top_k": VOCAB}, {"top_k": 10 ** 12}, {"top_k": -3, "min_p": -0.5}):
        assert _loop(be, **kw) == plain
    for kw in ({"top_k": VOCAB - 1}, {"min_p": 1e-9}):
        with pytest.raises(ValueError):
            be.submit(GenerationRequest([1, 2, 3], max_tokens=2, **kw))
    with _Server(e, tok) as s:
        plain = s.post()
        for kw in ({"top_k": VOCAB}, {"top_k": 10 ** 12}, {"top_k": None, "min_p": None}, {"top_k": -3, "min_p": -0.5}):
            assert s.post(**kw) == plain
        for kw in ({"top_k": VOCAB - 1}, {"min_p": 1e-9}):
            with pytest.raises(urllib.error.HTTPError) as err:
                s.post(**kw)
            assert err.value.code == 400


def test_requests_are_served_without_them_where_that_is_said(tiny_model_path, tok, monkeypatch):
    """DLLAMA_HOST_FILTERS=ignore: clients that send top_k with every request keep their server, whatever its value's type."""
    e = _engine(tiny_model_path)
    monkeypatch.setenv("DLLAMA_HOST_FILTERS", "ignore")
    be = BatchEngine(e, tok)
    plain = _loop(be)
    for kw in ({"top_k": 5}, {"min_p": 0.1}, {"top_k": 40, "min_p": 0.5}):
        assert _loop(be, **kw) == plain
    with _Server(e, tok) as s:
        plain = s.post()
        for kw in ({"top_k": 5}, {"min_p": 0.1}, {"top_k": 40, "min_p": 0.5}, {"top_k": "many"}, {"min_p": [1]}):
            assert s.post(**kw) == plain


def test_the_python_front_end_leaves_them_out_as_well(tiny_model_path, tok, monkeypatch):
    import threading
    from http.server import ThreadingHTTPServer
    from dllama_b200.serving.api import ApiState, make_handler
    monkeypatch.setenv("DLLAMA_HOST_FILTERS", "ignore")
    be = BatchEngine(_engine(tiny_model_path), tok)
    be.start()
    state = ApiState(be, tok, "tiny.m", A.InferenceParams(messages=[], temperature=0.8, top_p=0.9, seed=1))
    srv = ThreadingHTTPServer(("127.0.0.1", 0), make_handler(state))
    threading.Thread(target=srv.serve_forever, daemon=True).start()
    try:
        def post(**kw):
            body = {"messages": [{"role": "user", "content": "hello"}], "max_tokens": 4, "seed": 5, **kw}
            req = urllib.request.Request(f"http://127.0.0.1:{srv.server_address[1]}/v1/chat/completions", data=json.dumps(body).encode(), method="POST")
            with urllib.request.urlopen(req, timeout=60) as r:
                return json.load(r)["choices"][0]["message"]["content"]
        plain = post()
        for kw in ({"top_k": 5}, {"min_p": 0.1}, {"top_k": "many"}):
            assert post(**kw) == plain
    finally:
        srv.shutdown()
        be.stop()
