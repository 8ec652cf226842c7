"""top_k and min_p on the default server's way to the sampler, and `dllama inference --samples`."""
import io
import json
import threading
import time
import urllib.request
from contextlib import redirect_stdout

import pytest

from dllama_b200.formats import tfile
from dllama_b200.serving import api_types as A
from dllama_b200.text import native as T

pytestmark = pytest.mark.gpu

# requests of one batch: settings of every kind side by side, and some that have none
ASKS = [dict(temperature=0.9, top_p=0.95), dict(temperature=0.9, top_p=0.95, top_k=5), dict(temperature=1.2, top_p=0.0, min_p=0.3), dict(temperature=0.0, top_k=3), dict(temperature=1.3, top_p=0.8, top_k=40, min_p=0.02),
        dict(temperature=1.5, top_k=1, top_p=0.9), dict(temperature=0.7, top_p=0.5), dict(temperature=1.0, top_p=0.9, top_k=1000000, min_p=0.001)]
TEXTS = ["hello world", "the of and", "token model fast", "hello", "world world world", "model", "fast gpu and the", "llama"]


def _tok(tmp_path):
    p = str(tmp_path / "tiny.t")
    tfile.write_synthetic_tokenizer(p, 1024)
    return T.Tokenizer(p)


def _llama(path):
    from dllama_b200.models.llama import LlamaEngine
    return LlamaEngine(path, max_rows=64, n_slots=8, max_seq_len=256, bucket_rows=True)


def _layers(tmp_path):
    from dllama_b200.models import registry
    from dllama_b200.models.layered import example_config, write_random_model
    d = str(tmp_path / "m")
    write_random_model(d, example_config(width=128, vocab=1024, blocks=3, heads=4), seed=23)
    return registry.engine_for_dir(d, max_rows=64, n_slots=8, max_seq_len=256, dtype="bfloat16")


def _by_the_python_loop(e, tok, asks):
    from dllama_b200.serving.api import ApiState
    from dllama_b200.serving.batch_engine import BatchEngine
    be = BatchEngine(e, tok)
    state = ApiState(be, tok, "m", A.InferenceParams(messages=[], temperature=0.8, top_p=0.9, seed=1))
    reqs = [be.submit(state.build_request(A.parse_inference_params(dict(a, messages=[{"role": "user", "content": TEXTS[i]}], max_tokens=12, seed=30 + i), state.defaults))) for i, a in enumerate(asks)]
    for _ in range(200):
        be.step()
        if all(r.finish_reason for r in reqs):
            break
    return [r.text for r in reqs], [len(r.tokens) for r in reqs]


def _by_the_native_server(e, tok, asks, monkeypatch):
    """All requests arrive ahead of the first step, in order, so that batches are those of the Python loop."""
    from dllama_b200.serving import filters
    from dllama_b200.serving.native_server import NativeApiServer
    drawn, draw = [], filters.Filters.draw
    monkeypatch.setattr(filters.Filters, "draw", lambda self, logits, n, n_on, *a: (drawn.append((n, n_on)), draw(self, logits, n, n_on, *a)))
    srv = NativeApiServer(e, tok, "m", A.InferenceParams(messages=[], temperature=0.8, top_p=0.9, seed=1), host="127.0.0.1", port=0, verbose=False)
    srv.listen()
    out = {}

    def post(i):
        body = dict(asks[i], messages=[{"role": "user", "content": TEXTS[i]}], max_tokens=12, seed=30 + i)
        req = urllib.request.Request(f"http://127.0.0.1:{srv.port}/v1/chat/completions", data=json.dumps(body).encode(), method="POST")
        with urllib.request.urlopen(req, timeout=120) as r:
            out[i] = json.load(r)
    threads = []
    try:
        for i in range(len(asks)):
            threads.append(threading.Thread(target=post, args=(i,)))
            threads[-1].start()
            end = time.time() + 60
            while srv.stats()["waiting"] <= i and time.time() < end:
                time.sleep(0.002)
            assert srv.stats()["waiting"] == i + 1
        for _ in range(200):
            srv.step()
            if srv.stats()["running"] + srv.stats()["waiting"] == 0:
                break
        [t.join(timeout=60) for t in threads]
        assert srv.stats()["engine_errors"] == 0
    finally:
        srv.close()
    return [out[i]["choices"][0]["message"]["content"] for i in range(len(asks))], [out[i]["usage"]["completion_tokens"] for i in range(len(asks))], drawn


@pytest.mark.parametrize("kind", ["llama", "layers"])
@pytest.mark.parametrize("which", [list(range(8)), [1, 2, 4], [0, 5], [2]])
def test_the_native_server_draws_what_the_python_loop_draws(kind, which, tiny_model_path, tmp_path, monkeypatch):
    tok = _tok(tmp_path)
    e = _llama(tiny_model_path) if kind == "llama" else _layers(tmp_path)
    asks = [ASKS[i] for i in which]
    want, lengths = _by_the_python_loop(e, tok, asks)
    got, n, drawn = _by_the_native_server(e, tok, asks, monkeypatch)
    assert got == want and n == lengths
    on = sum(bool(0 < a.get("top_k", 0) < 1024 or a.get("min_p", 0) > 0) for a in asks)
    assert (len(asks), on) in drawn and all(0 < k <= m for m, k in drawn)
    e.close()


def test_one_token_left_is_the_greedy_answer(tiny_model_path, tmp_path, monkeypatch):
    """Through HTTP, one request at a time: top_k 1 and min_p 1 at any temperature."""
    tok = _tok(tmp_path)
    e = _llama(tiny_model_path)
    answers = [_by_the_native_server(e, tok, [dict(temperature=t, top_p=0.0, **kw)], monkeypatch)[0] for t, kw in ((0.0, {}), (1.4, {"top_k": 1}), (5.0, {"min_p": 1.0}), (0.3, {"top_k": 1, "min_p": 1.0}))]
    assert answers[0] == answers[1] == answers[2] == answers[3]
    e.close()


@pytest.mark.parametrize("options,settings", [(["--samples", "5"], (0.8, 0, 0.9, 0.0)), (["--samples", "7", "--topk", "20", "--minp", "0.02", "--temperature", "1.1", "--topp", "0.7"], (1.1, 20, 0.7, 0.02)),
                                              (["--topk", "3"], (0.8, 3, 0.9, 0.0))])
def test_samples_of_the_command_line(options, settings, tiny_model_path, tmp_path):
    from dllama_b200.cli import dllama as cli
    from dllama_b200.models.llama import LlamaEngine
    tok = _tok(tmp_path)
    prompt, steps, seed = "hello world the of and", 40, 11
    buf = io.StringIO()
    with redirect_stdout(buf):
        rc = cli.main(["dllama", "inference", "--model", tiny_model_path, "--tokenizer", str(tmp_path / "tiny.t"), "--buffer-float-type", "q80", "--prompt", prompt, "--steps", str(steps),
                       "--max-seq-len", "128", "--device", "cuda", "--seed", str(seed), *options])
    assert rc == 0, buf.getvalue()
    n = int(options[options.index("--samples") + 1]) if "--samples" in options else 1
    e = LlamaEngine(tiny_model_path, max_rows=256, n_slots=64, max_seq_len=128)
    tokens = tok.encode(prompt, add_bos=True, add_special_tokens=False)
    want = e.sample_many(tokens, n, steps - len(tokens), *settings, seed)
    e.close()
    for i, row in enumerate(want.tolist()):
        tok.reset_decoder()
        stop = next((j for j, t in enumerate(row) if t in tok.eos_token_ids), len(row))
        text = "".join(tok.decode(t) or "" for t in row[:stop])
        assert f"Sample {i} | {prompt}{text}\n" in buf.getvalue()
    assert f"Sample {n} |" not in buf.getvalue() and f"nTokens: {want.size}" in buf.getvalue()


def test_what_the_command_line_refuses(tiny_model_path, tmp_path):
    from dllama_b200.cli import dllama as cli
    _tok(tmp_path)
    base = ["dllama", "inference", "--model", tiny_model_path, "--tokenizer", str(tmp_path / "tiny.t"), "--buffer-float-type", "q80", "--prompt", "hello world", "--max-seq-len", "128", "--seed", "1"]
    for more in (["--steps", "20", "--samples", "0", "--device", "cuda"], ["--steps", "20", "--samples", "2000", "--device", "cuda"], ["--steps", "20", "--samples", "2", "--device", "cpu"]):
        buf = io.StringIO()
        try:
            with redirect_stdout(buf):
                rc = cli.main(base + more)
        except (ValueError, SystemExit) as e:
            rc = 1 if isinstance(e, ValueError) else e.code
        assert rc != 0
