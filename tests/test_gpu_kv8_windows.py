"""Windows larger than any context, up to the largest int, beside rows of negative positions (needs a B200).
Tolerances: test_gpu_kv8.py."""
import numpy as np
import pytest
import torch

from kv8_helpers import Pool
from test_gpu_kv8 import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", ["few", "many"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 90, 89, 88])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_window_that_no_context_fills(pkg, monkeypatch, kernel, window, hd):
    monkeypatch.setenv("BZB_KV8_ATTENTION", kernel)
    seqs = [(-6, 9), (-40, 129), (87, 3), (0, 70)]  # (the longest context has 90 positions)
    lens, news = [a + b for a, b in seqs], [s[1] for s in seqs]
    pool = Pool(pkg, lens, 2, hd, seed=1, fill=lens)
    n = sum(news)
    q = torch.from_numpy(np.random.default_rng(hd).standard_normal((n, 4, hd)).astype(np.float32)).cuda().half()
    out, lse = torch.full_like(q, float("nan")), torch.full((n, 4), float("nan"), device="cuda")
    pool.cache.attention(pool.batch(news, lens), q, out, 0.125, window=window, lse=lse)
    pool.cache.check()
    check_attention(pool, q, out, lse, seqs, 0.125, window, True, "f16")
