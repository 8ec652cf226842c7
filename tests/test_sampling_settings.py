"""top_k and min_p on their way in: the API's parameters, the CLI's options, and what hosts without the device sampler answer."""
import json
import urllib.error
import urllib.request

import pytest

from dllama_b200.cli.app import AppArgs
from dllama_b200.formats import tfile
from dllama_b200.models.cpu_engine import CpuEngine
from dllama_b200.models.paging import PageAllocator
from dllama_b200.serving import api_types as A
from dllama_b200.serving.batch_engine import BatchEngine, GenerationRequest
from dllama_b200.serving.native_server import NativeApiServer
from dllama_b200.text import native as T


@pytest.fixture(scope="module")
def tok(tmp_path_factory):
    p = str(tmp_path_factory.mktemp("tok") / "tiny.t")
    tfile.write_synthetic_tokenizer(p, 1024)
    return T.Tokenizer(p)


def test_api_parameters():
    d = A.InferenceParams(messages=[])
    body = {"messages": [{"role": "user", "content": "x"}]}
    p = A.parse_inference_params(body, d)
    assert p.top_k == 0 and p.min_p == 0.0
    p = A.parse_inference_params({**body, "top_k": 40, "min_p": 0.05}, d)
    assert p.top_k == 40 and p.min_p == 0.05
    assert A.parse_inference_params({**body, "top_k": -1}, d).top_k == 0
    assert A.parse_inference_params({**body, "top_k": 10 ** 12}, d).top_k == (1 << 31) - 1
    for bad in (float("nan"), float("inf")):                     # (json.loads takes both; answered with 400)
        with pytest.raises((ValueError, OverflowError)):
            A.parse_inference_params({**body, "top_k": bad}, d)


def test_cli_options():
    a = AppArgs.parse(["dllama", "inference", "--samples", "8", "--topk", "40", "--minp", "0.1"], True)
    assert (a.samples, a.topk, a.minp) == (8, 40, 0.1)
    a = AppArgs.parse(["dllama", "inference"], True)
    assert (a.samples, a.topk, a.minp) == (1, 0, 0.0)


def test_without_the_device_sampler(tiny_model_path, tok):
    """The host samplers have neither: such a request is refused, others are served."""
    eng = CpuEngine(tiny_model_path, max_rows=8, n_slots=4, max_seq_len=128)
    be = BatchEngine(eng, tok)
    for kw in ({"top_k": 5}, {"min_p": 0.1}):
        with pytest.raises(ValueError):
            be.submit(GenerationRequest([1, 2, 3], max_tokens=2, **kw))
    srv = NativeApiServer(eng, tok, "tiny.m", A.InferenceParams(messages=[], temperature=0.0, top_p=0.9, seed=1), host="127.0.0.1", port=0, verbose=False)
    srv.start()
    try:
        def post(**kw):
            body = {"messages": [{"role": "user", "content": "hello"}], "max_tokens": 2, **kw}
            return urllib.request.urlopen(urllib.request.Request(f"http://127.0.0.1:{srv.port}/v1/chat/completions", data=json.dumps(body).encode(), method="POST"), timeout=60)
        for kw in ({"top_k": 5}, {"min_p": 0.1}, {"top_k": "many"}):
            with pytest.raises(urllib.error.HTTPError) as e:
                post(**kw)
            assert e.value.code == 400
        for kw in ({}, {"top_k": 0, "min_p": 0}, {"top_k": -1}):
            with post(**kw) as r:
                assert json.load(r)["usage"]["completion_tokens"] >= 1
    finally:
        srv.close()


def test_pages_of_no_sequence():
    p = PageAllocator(6, 2, 4)
    s = p.alloc_slot()
    p.ensure(s, 40)
    a = p.take(3)
    assert len(set(a)) == 3 and not set(a) & set(p.table[s, :2].tolist())
    with pytest.raises(RuntimeError):
        p.take(2)
    p.give(a)
    p.free_slot(s)
    assert sorted(p.free_pages) == list(range(6))
