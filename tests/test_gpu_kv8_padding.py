"""Padding rows (a negative position) of attention over all keys: zeros and a log-sum-exp of -inf, as in causal attention
(needs a B200). Tolerances: test_gpu_kv8.py."""
import numpy as np
import pytest
import torch

from kv8_helpers import Pool
from test_gpu_kv8 import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", ["few", "many"])
@pytest.mark.parametrize("H,KV,hd,seqs", [
    (4, 2, 64, [(-3, 5), (13, 3), (-4, 4), (0, 2)]),                 # a tile with both kinds of rows; no key at all
    (8, 1, 128, [(-9, 40), (-1, 1), (5, 4)]),
    (2, 1, 64, [(-200, 400), (-130, 131), (-128, 300), (7, 200)]),   # whole tiles of padding
])
def test_padding_rows_of_attention_over_all_keys(pkg, monkeypatch, kernel, H, KV, hd, seqs):
    monkeypatch.setenv("BZB_KV8_ATTENTION", kernel)
    lens, news = [a + b for a, b in seqs], [s[1] for s in seqs]
    pool = Pool(pkg, lens, KV, hd, seed=H, fill=lens)
    n = sum(news)
    x = np.random.default_rng(n).standard_normal((n, H, hd)).astype(np.float32)
    pad = np.concatenate([np.arange(a, a + b) < 0 for a, b in seqs])
    x[pad] = np.nan  # (append leaves these rows of its output as they were)
    q = torch.from_numpy(x).cuda().half()
    out, lse = torch.full_like(q, 7.0), torch.full((n, H), 7.0, device="cuda")
    pool.cache.attention(pool.batch(news, lens), q, out, 0.125, causal=False, lse=lse)
    pool.cache.check()
    assert not out[torch.from_numpy(pad)].any() and torch.isneginf(lse[torch.from_numpy(pad)]).all()
    check_attention(pool, q, out, lse, seqs, 0.125, 0, False, "f16")
