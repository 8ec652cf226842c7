"""The token cache's type on its way from the root's command line to a worker's engine (no GPU)."""
import socket
import threading

import pytest

from dllama_b200.cli import app


class _Built(Exception):
    pass


@pytest.mark.parametrize("kv_cache", ["f16", "q8"])
def test_a_worker_builds_the_cache_that_the_root_was_asked_for(tiny_model_path, monkeypatch, kv_cache):
    from dllama_b200.parallel import symm
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    asked = {}

    def build_engine(model, rank, world, max_batch, n_slots, max_seq_len, sync_type, device="auto", gpu_index=-1, workers=(), n_threads=0, dtype="bfloat16", kv_cache="f16"):
        asked.update(model=model, rank=rank, world=world, max_batch=max_batch, kv_cache=kv_cache)
        raise _Built

    monkeypatch.setattr(app, "use_cuda_device", lambda device: True)
    monkeypatch.setattr(app, "build_engine", build_engine)
    monkeypatch.setattr(symm, "init_distributed", lambda: (1, 2, None))
    for name in ("RANK", "WORLD_SIZE", "LOCAL_RANK", "MASTER_ADDR", "MASTER_PORT"):
        monkeypatch.setenv(name, "0")                            # (set by the worker; put back behind the test)

    def work():
        with pytest.raises(_Built):
            app.run_worker_app(app.AppArgs(port=port))

    worker = threading.Thread(target=work, daemon=True)
    worker.start()
    root = app.AppArgs.parse(["dllama", "inference", "--model", tiny_model_path, "--tokenizer", "t", "--max-batch", "16", "--kv-cache", kv_cache,
                              "--workers", f"127.0.0.1:{port}"], True)
    for _ in range(200):
        try:
            assert app.dial_workers(root, 23456) == 2
            break
        except ConnectionRefusedError:
            worker.join(0.05)
    worker.join(10)
    assert not worker.is_alive() and asked == dict(model=tiny_model_path, rank=1, world=2, max_batch=16, kv_cache=kv_cache)
