"""The Llama engine on the 8-bit token cache, against the oracle and against itself on fp16.

Tolerances: the fp16 engine is held to 3e-2 of the largest logit (test_gpu_model.py).  A value in 8 bits is off by at most 1/254 of its line's largest,
and so is what attention returns; scores move by as much relatively, weights by that times a score of ~3: 4/254 for a layer's attention output, which the
residual stream carries as one part of many.  1e-2 more for two layers.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TOL = 4e-2


@pytest.fixture(scope="module")
def wide_heads_path(tmp_path_factory):
    """Heads of 128: the tensor-core forms of prompts."""
    from dllama_b200.formats import mfile
    p = str(tmp_path_factory.mktemp("models") / "wide.m")
    shape = dict(dim=1024, hidden_dim=1024, n_layers=2, n_heads=8, n_kv_heads=2, vocab_size=1024, max_seq_len=1024, rope_theta=500000, rope=(32, 1, 4, 8192))
    mfile.write_random_model(p, shape, exact=True, seed=5)
    return p


def _oracle(path):
    from dllama_b200.formats.mfile import ModelFile
    from dllama_b200.models.oracle import OracleLlama
    return OracleLlama(ModelFile(path), n_nodes=1, max_seq_len=1024)


def _engine(path, **kw):
    from dllama_b200.models.llama import LlamaEngine
    kw.setdefault("max_seq_len", 1024)
    kw.setdefault("kv_dtype", torch.int8)
    return LlamaEngine(path, **kw)


def _rel_err(a, b):
    return float(np.abs(a - b).max() / (np.abs(b).max() + 1e-9))


@pytest.mark.parametrize("use_graphs,use_pdl", [(False, False), (True, True)])
@pytest.mark.parametrize("which", ["tiny", "tp8", "wide"])
def test_prompt_and_decode_match_the_oracle(tiny_model_path, tiny_tp_model_path, wide_heads_path, which, use_graphs, use_pdl):
    path = {"tiny": tiny_model_path, "tp8": tiny_tp_model_path, "wide": wide_heads_path}[which]
    o, rng = _oracle(path), np.random.default_rng(1)
    e = _engine(path, max_rows=64, n_slots=2, use_graphs=use_graphs, use_pdl=use_pdl, max_seq_len=512)
    prompt = rng.integers(1, 1024, 100).tolist()                     # two batches: 64 rows, then 36 behind them
    slot = e.alloc_slot()
    ref = o.forward(prompt, 0).numpy()
    got = e.prefill(slot, prompt, 0).float().cpu().numpy()
    assert _rel_err(got[0], ref[-1]) < TOL
    tok, pos = int(np.argmax(ref[-1])), len(prompt)
    for _ in range(5):
        ref = o.forward([tok], pos).numpy()
        got = e.forward([tok], [pos], [slot]).float().cpu().numpy()
        assert _rel_err(got[0], ref[0]) < TOL
        tok, pos = int(np.argmax(ref[0])), pos + 1
    e.close()


def test_long_prompt_on_widened_pages(wide_heads_path):
    """More than 4096 rows times heads: the tcgen05 kernel on pages widened once, then a short chunk and a token behind it."""
    o, rng = _oracle(wide_heads_path), np.random.default_rng(2)
    e = _engine(wide_heads_path, max_rows=640, n_slots=2)
    assert e.kv8_work is not None
    prompt = rng.integers(1, 1024, 600).tolist()
    slot = e.alloc_slot()
    ref = o.forward(prompt, 0).numpy()
    got = e.forward(prompt, list(range(600)), [slot] * 600, logits_from=0).float().cpu().numpy()
    for t in (0, 1, 31, 32, 127, 128, 400, 599):
        assert _rel_err(got[t], ref[t]) < TOL, t
    more = rng.integers(1, 1024, 30).tolist()
    ref = o.forward(more, 600).numpy()
    got = e.forward(more, list(range(600, 630)), [slot] * 30, logits_from=0).float().cpu().numpy()
    assert max(_rel_err(got[t], ref[t]) for t in range(30)) < TOL
    ref = o.forward([5], 630).numpy()
    assert _rel_err(e.forward([5], [630], [slot]).float().cpu().numpy()[0], ref[0]) < TOL
    e.close()


def test_chunk_beside_decode_rows_of_other_users(tiny_tp_model_path):
    e = _engine(tiny_tp_model_path, max_rows=64, n_slots=4, max_seq_len=512)
    rng = np.random.default_rng(9)
    pa, pb, chunk = (rng.integers(1, 1024, n).tolist() for n in (7, 3, 40))
    sa, sb, sc = e.alloc_slot(), e.alloc_slot(), e.alloc_slot()
    e.prefill(sa, pa, 0)
    e.prefill(sb, pb, 0)
    got = e.forward(chunk + [11, 12], list(range(40)) + [7, 3], [sc] * 40 + [sa, sb], logits_from=39).float().cpu().numpy().copy()
    for i, (before, tok) in enumerate(((chunk[:-1], chunk[-1]), (pa, 11), (pb, 12))):
        o = _oracle(tiny_tp_model_path)
        o.forward(before, 0)
        assert _rel_err(got[i], o.forward([tok], len(before)).numpy()[0]) < TOL
    e.close()


def test_cache_is_half_as_large_and_reads_back(wide_heads_path):
    """Keys and values of a prompt, out of the pages, against the fp16 engine's: half a step of a line's 127, and fp16's own 2^-11 of a value."""
    from dllama_b200.ops import kernels as K
    rng = np.random.default_rng(3)
    prompt = rng.integers(1, 1024, 90).tolist()
    held = {}
    for t in (torch.float16, torch.int8):
        e = _engine(wide_heads_path, max_rows=128, n_slots=2, kv_dtype=t)
        slot = e.alloc_slot()
        e.prefill(slot, prompt, 0)
        held[t] = [x.double().cpu().view(90, 2, 128) for x in e.read_cache(0, slot, 90, torch.float32 if t == torch.int8 else torch.float16)]
        if t == torch.int8:
            assert e.kv8_cache[0].nbytes() == e.n_pages * K.kv8_page_bytes(2, 128)
            assert e.kv8_cache[0].nbytes() * 2 < e.n_pages * 2 * 2 * 32 * 128 * 2 * 1.04
        e.close()
    for a, b in zip(held[torch.int8], held[torch.float16]):
        # layer 0 sees the same rows in both engines; the matmul's f32 sums come out of another epilogue, turned in f32 there
        top = b.abs().amax(-1, keepdim=True)
        assert ((a - b).abs() <= top * (0.5 / 127 + 2.0 ** -11 + 1e-5)).all()


def test_serving_on_it(tiny_model_path, tmp_path):
    """Continuous batching: buckets, captured graphs, packed prompts; greedy tokens are near the oracle's best."""
    from dllama_b200.formats import mfile
    from dllama_b200.models.oracle import OracleLlama
    from dllama_b200.serving.batch_engine import BatchEngine, GenerationRequest
    from dllama_b200.formats import tfile
    from dllama_b200.text import native as T
    tfile.write_synthetic_tokenizer(str(tmp_path / "tiny.t"), 1024)
    e = _engine(tiny_model_path, max_rows=32, n_slots=6, max_seq_len=256, bucket_rows=True)
    be = BatchEngine(e, T.Tokenizer(str(tmp_path / "tiny.t")))
    be.warmup()
    rng = np.random.default_rng(4)
    prompts = [[5, 6, 7, 8, 9, 10], [100, 200, 300], rng.integers(1, 1000, 40).tolist(), [42]]
    reqs = [be.submit(GenerationRequest(prompt_tokens=p, max_tokens=5, temperature=0.0)) for p in prompts]
    be.start()
    for r in reqs:
        r.result(timeout=120)
    be.stop()
    o = OracleLlama(mfile.ModelFile(tiny_model_path), max_seq_len=256)
    for r, p in zip(reqs, prompts):
        o.reset()
        lg = o.forward(p, 0).numpy()[-1]
        for i, t in enumerate(r.tokens):
            assert lg[t] >= lg.max() - TOL * max(1.0, float(abs(lg).max())), (p, i, t)
            lg = o.forward([t], len(p) + i).numpy()[0]
    e.close()


def test_device_loop_and_host_loop_agree(wide_heads_path):
    e = _engine(wide_heads_path, max_rows=16, n_slots=2, max_seq_len=256)
    slot = e.alloc_slot()
    lg = e.prefill(slot, [3, 4, 5, 6], 0)
    first = int(lg[-1].argmax())
    e.ensure_capacity(slot, 40)
    host, tok = [], first
    for i in range(8):
        tok = e.decode_greedy_host([tok], [4 + i], [slot])[0]
        host.append(tok)
    e.set_batch([first], [4], [slot])
    torch.cuda.synchronize()
    e.decode_greedy_device(8, 1)
    torch.cuda.synchronize()
    assert e.read_history(8, 1, e.current_step() - 8)[:, 0].tolist() == host
    e.close()
