"""top_k and min_p of a batch's rows, for the loops that draw on the GPU."""
from __future__ import annotations

import os

import numpy as np
import torch

MAX_VOCAB = 1 << 19          # of sample_tokens (dl_sample_tokens_max_vocab)


def host_ignores() -> bool:
    """DLLAMA_HOST_FILTERS=ignore: loops that sample on the host leave top_k and min_p out of account, as they do with fields that they do not know."""
    return os.environ.get("DLLAMA_HOST_FILTERS", "refuse") == "ignore"


def settings(top_k, min_p, vocab: int) -> tuple:
    """top_k and min_p of a request as the kernel takes them: 0 where they take nothing out (a top_k below 1, or of the vocabulary or more; a min_p that is not above 0 in f32), a min_p of 1 at most."""
    return int(top_k) if 0 < top_k < vocab else 0, float(np.float32(min(min_p, 1.0))) if min_p > 0 else 0.0


class Filters:
    """Settings of up to `rows` rows: written into top_k (int32, 0: off) and min_p (f32, 0: off) on the host, pinned, and read by draw()."""

    def __init__(self, rows: int, device: torch.device):
        self.top_k, self.min_p = torch.zeros(rows, dtype=torch.int32).pin_memory(), torch.zeros(rows, dtype=torch.float32).pin_memory()
        self._top_k, self._min_p = self.top_k.to(device), self.min_p.to(device)
        self._drawn = torch.zeros(rows, dtype=torch.int32, device=device)

    def draw(self, logits: torch.Tensor, n: int, n_on: int, params: torch.Tensor, sample_rows, tokens: torch.Tensor):
        """tokens[:n] from params (temperature, top_p, coin); n_on rows have top_k or min_p on and are drawn by sample_tokens, the other ones by sample_rows: what a request without them is answered
        does not hang on its neighbours."""
        from ..ops import kernels as K
        self._top_k.copy_(self.top_k, non_blocking=True)
        self._min_p.copy_(self.min_p, non_blocking=True)
        drawn = tokens if n_on == n else self._drawn
        K.sample_tokens(logits, n, params[0], self._top_k, params[1], self._min_p, params[2], drawn)
        if n_on < n:
            sample_rows(logits[:n], params[0], params[1], params[2], tokens)
            tokens[:n] = torch.where((self._top_k[:n] > 0) | (self._min_p[:n] > 0), drawn[:n], tokens[:n])
