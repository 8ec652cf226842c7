"""Shared memory of another CTA of a cluster is there once that CTA has started, which only a barrier of the cluster tells: no kernel reaches for it ahead of one.  By reading the sources, as a
kernel that does may fault."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "distributed-llama-multiusers_b200", "csrc", "cuda")
KERNELS = [("sample_tokens.cu", "sample_tokens_kernel", r"z\.at\(|map_shared_rank", r"cluster_wait\(\)|cluster\.sync\(\)"),
           ("shared_attention.cu", "shared_own_kernel", r"map_shared_rank", r"cluster\.sync\(\)"),
           ("kv8_attention.cu", None, r"map_shared_rank", r"cluster\.sync\(\)")]


def _without_comments(text):
    return re.sub(r"//[^\n]*", "", text)


def _body(text, name):
    """From the kernel's parameters to the brace that ends it."""
    at = re.search(r"__global__[^;{]*\b" + name + r"\(", text).end()
    i = text.index("{", at)
    depth = 0
    for j in range(i, len(text)):
        depth += (text[j] == "{") - (text[j] == "}")
        if depth == 0:
            return text[i:j]


@pytest.mark.parametrize("file,kernel,reach,barrier", KERNELS)
def test_a_barrier_comes_ahead_of_other_ctas_memory(file, kernel, reach, barrier):
    text = _without_comments(open(os.path.join(CSRC, file)).read())
    body = _body(text, kernel) if kernel else text
    first, sync = re.search(reach, body), re.search(barrier, body)
    assert first and sync and sync.start() < first.start()
    # a wait belongs to an arrival ahead of it, by all threads
    if sync.group().startswith("cluster_wait"):
        arrive = re.search(r"\n    cluster_arrive_relaxed\(\);", body)
        assert arrive and arrive.start() < sync.start() and re.search(r"\n    cluster_wait\(\);", body)
