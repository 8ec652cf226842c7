"""Many samples of one prompt: block tables from lengths, attention over the prompt's shared pages and drawing, as LlamaEngine.sample_many runs them one behind the other; and top-k and min-p
through the serving loop."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wide_heads_path(tmp_path_factory):
    """Heads of 128, four to a key/value head."""
    from dllama_b200.formats import mfile
    p = str(tmp_path_factory.mktemp("models") / "wide.m")
    shape = dict(dim=1024, hidden_dim=1024, n_layers=2, n_heads=8, n_kv_heads=2, vocab_size=1024, max_seq_len=1024, rope_theta=500000, rope=(32, 1, 4, 8192))
    mfile.write_random_model(p, shape, exact=True, seed=6)
    return p


def _engine(path, **kw):
    from dllama_b200.models.llama import LlamaEngine
    kw.setdefault("max_seq_len", 512)
    kw.setdefault("max_rows", 64)
    kw.setdefault("n_slots", 24)
    return LlamaEngine(path, **kw)


def _by_hand(e, prompt, n, count, coins, filters):
    """The same, every sample a sequence of its own that the engine's public calls run."""
    from dllama_b200.ops import kernels as K
    slots = [e.alloc_slot() for _ in range(n)]
    for s in slots:
        logits = e.prefill(s, prompt)
    args = [torch.full((n,), v, dtype=d, device="cuda") for v, d in zip(filters, (torch.float32, torch.int32, torch.float32, torch.float32))]
    out, tokens = [], torch.zeros(n, dtype=torch.int32, device="cuda")
    logits = logits[:1].expand(n, -1).contiguous()
    for i in range(count):
        K.sample_tokens(logits, n, *args, coins[i].cuda(), tokens)
        out.append(tokens.tolist())
        if i + 1 < count:
            logits = e.forward(out[-1], [len(prompt) + i] * n, slots)
    for s in slots:
        e.free_slot(s)
    return np.array(out).T


@pytest.mark.parametrize("kv_dtype", [torch.float16, torch.int8])
@pytest.mark.parametrize("use_graphs", [False, True])
@pytest.mark.parametrize("n,length", [(1, 5), (3, 64), (7, 100), (20, 31), (12, 33)])
def test_samples_are_those_of_sequences_by_themselves(tiny_model_path, n, length, use_graphs, kv_dtype):
    """Not shared: the same kernels run over the same values, wherever the pages lie: the same tokens."""
    e = _engine(tiny_model_path, use_graphs=use_graphs, kv_dtype=kv_dtype)
    rng = np.random.default_rng(n)
    prompt = rng.integers(1, 1024, length).tolist()
    free = len(e.pages.free_pages), len(e.pages.free_slots)
    coins = torch.rand(40, n, generator=torch.Generator().manual_seed(n))
    filters = (0.9, 50, 0.95, 0.01)
    got = e.sample_many(prompt, n, 40, *filters, coins=coins, share=False)
    assert (len(e.pages.free_pages), len(e.pages.free_slots)) == free
    assert np.array_equal(got, _by_hand(e, prompt, n, 40, coins, filters))
    again = e.sample_many(prompt, n, 40, *filters, coins=coins, share=False)
    assert np.array_equal(got, again)
    e.close()


@pytest.mark.parametrize("which", ["tp8", "wide"])
@pytest.mark.parametrize("n,length", [(2, 40), (5, 97), (16, 200), (23, 64)])
def test_shared_pages_give_the_same_logits(tiny_tp_model_path, wide_heads_path, which, n, length):
    """Heads of 64 and 128, on the dp4a rows (2), and on tcgen05: the logits of the last step, after the same tokens (the samples of a step are those of the step's logits: as long as the
    tokens of the steps ahead are the same).  Queries and weights in fp16 instead of f32: 2^-11 of an attention output, beside Q80 activations of 1/254; 1e-2 of the largest logit for two layers."""
    e = _engine({"tp8": tiny_tp_model_path, "wide": wide_heads_path}[which])
    prompt = np.random.default_rng(length).integers(1, 1024, length).tolist()
    coins = torch.rand(2, n, generator=torch.Generator().manual_seed(1))
    logits = []
    for share in (False, True):
        t = e.sample_many(prompt, n, 2, 1.0, 0, 0.0, 0.0, coins=coins, share=share)
        logits.append((t[:, 0].tolist(), e.logits[:n].float().cpu().numpy().copy()))
    assert logits[0][0] == logits[1][0]
    assert np.abs(logits[0][1] - logits[1][1]).max() <= 1e-2 * np.abs(logits[0][1]).max()
    e.close()


def test_a_long_run_on_shared_pages(wide_heads_path):
    """Samples that grow over several pages, behind the engine's usual work and ahead of it; the seed tells the samples."""
    e = _engine(wide_heads_path, max_seq_len=1024)
    prompt = np.random.default_rng(3).integers(1, 1024, 300).tolist()
    slot = e.alloc_slot()
    before = e.prefill(slot, prompt[:50]).clone()
    assert e.shares_prompt(16, 64) and not e.shares_prompt(2, 1000) and not e.shares_prompt(64, 8)
    a = e.sample_many(prompt, 16, 120, 1.0, seed=5, share=True)
    b = e.sample_many(prompt, 16, 120, 1.0, seed=5, share=True)
    c = e.sample_many(prompt, 16, 120, 1.0, seed=6, share=True)
    assert np.array_equal(a, b) and not np.array_equal(a, c) and a.shape == (16, 120) and a.min() >= 0 and a.max() < 1024
    assert len({tuple(r) for r in a.tolist()}) > 1
    greedy = e.sample_many(prompt, 16, 30, 0.0, share=True)
    assert (greedy == greedy[:1]).all()
    e.free_slot(slot)
    slot = e.alloc_slot()
    assert torch.equal(before, e.prefill(slot, prompt[:50]))              # the tables are the engine's own again
    e.close()


def test_refusals(tiny_model_path):
    e = _engine(tiny_model_path, n_slots=4, kv_dtype=torch.int8)
    for bad in (lambda: e.sample_many([], 1, 4), lambda: e.sample_many([1], 0, 4), lambda: e.sample_many([1], 4, 4), lambda: e.sample_many([1], 65, 4), lambda: e.sample_many([1], 1, 0),
                lambda: e.sample_many([1] * 500, 1, 13), lambda: e.sample_many([1], 2, 4, coins=torch.zeros(4, 3)), lambda: e.sample_many([1] * 40, 2, 4, share=True)):
        with pytest.raises(ValueError):
            bad()
    assert len(e.pages.free_slots) == 4
    e.world = 2
    with pytest.raises(NotImplementedError):
        e.sample_many([1], 1, 4)
    e.world = 1
    e.close()


def test_top_k_and_min_p_through_the_serving_loop(tiny_model_path, tmp_path):
    """top_k 1 gives the greedy answer at any temperature, beside requests that have neither."""
    from dllama_b200.serving.batch_engine import BatchEngine, GenerationRequest
    from dllama_b200.formats import tfile
    from dllama_b200.text import native as T
    tfile.write_synthetic_tokenizer(str(tmp_path / "tiny.t"), 1024)
    e = _engine(tiny_model_path, max_rows=32, n_slots=4, bucket_rows=True)
    be = BatchEngine(e, T.Tokenizer(str(tmp_path / "tiny.t")))
    prompts = [[1, 5, 9, 13], [1, 7, 7], [2, 3, 4, 5, 6]]
    answers = {}
    for name, kw in (("greedy", dict(temperature=0.0)), ("top_k", dict(temperature=1.3, top_k=1, top_p=0.0)), ("min_p", dict(temperature=0.7, min_p=1.0, top_p=0.0))):
        reqs = [be.submit(GenerationRequest(list(p), max_tokens=12, seed=3 + i, **kw)) for i, p in enumerate(prompts)]
        plain = be.submit(GenerationRequest([4, 4, 4], max_tokens=12, seed=9, temperature=0.8))
        for _ in range(200):
            be.step()
            if all(r.finish_reason for r in reqs + [plain]):
                break
        answers[name] = [r.tokens for r in reqs]
    assert answers["greedy"] == answers["top_k"] == answers["min_p"]
    e.close()


def test_neighbours_with_top_k_change_no_answer():
    """Rows without top_k and min_p are drawn as in a batch where nobody has them: by the sampler that they had before."""
    from dllama_b200.ops import kernels as K
    from dllama_b200.serving.filters import Filters
    g = torch.Generator(device="cuda").manual_seed(3)
    n, vocab = 24, 1024
    logits = torch.zeros(32, vocab, device="cuda")
    logits[:n] = 2 * torch.randn(n, vocab, generator=g, device="cuda")
    logits[5] = 0.0                                                # all tokens alike: both samplers agree on none of top_p's
    params = torch.stack([torch.full((32,), 0.9), torch.full((32,), 0.8), torch.rand(32, generator=torch.Generator().manual_seed(4))]).cuda()
    alone = torch.zeros(32, dtype=torch.int32, device="cuda")
    K.sample_rows(logits[:n], params[0], params[1], params[2], alone)
    f = Filters(32, logits.device)
    seen = []

    def rows(*a):
        seen.append(len(a[0]))
        K.sample_rows(*a)
    for on in ([], [0], [3, 17], list(range(n))):
        f.top_k.zero_()
        f.min_p.zero_()
        f.top_k[on[::2]], f.min_p[on[1::2]] = 7, 0.2
        f.top_k[n:] = 5                                            # (places behind the batch's rows)
        want = torch.full((32,), -9, dtype=torch.int32, device="cuda")
        K.sample_tokens(logits, n, params[0], f.top_k.cuda(), params[1], f.min_p.cuda(), params[2], want)
        got = torch.full((32,), -9, dtype=torch.int32, device="cuda")
        f.draw(logits, n, len(on), params, rows, got)
        for m in range(32):
            assert got[m] == (-9 if m >= n else want[m] if m in on else alone[m])
    assert seen == [n] * 3
