"""Contexts of which one CTA of the few-row kernel takes more blocks than it looks up at once (needs a B200): batches so
large that contexts are cut into a few ranges at most. Tolerances: test_gpu_kv8.py."""
import numpy as np
import pytest
import torch

from kv8_helpers import Pool
from test_gpu_kv8 import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,window", [(64, 0), (128, 0), (64, 20000)])
def test_long_contexts_of_many_sequences(pkg, monkeypatch, hd, window):
    """600 sequences of 14 lengths over the same pages, on both sides of every refill of a warp's table."""
    monkeypatch.setenv("BZB_KV8_ATTENTION", "few")
    lens = [33000, 8192, 8193, 8191, 8256, 10240, 10241, 10239, 2048, 2049, 16384, 24600, 1, 300]
    pool = Pool(pkg, [33000], 2, hd, 64, seed=hd, fill=[33000])
    n = 600
    kinds = torch.arange(n) % len(lens)
    q1 = torch.from_numpy(np.random.default_rng(5).standard_normal((len(lens), 4, hd)).astype(np.float32)).cuda().half()
    q = q1[kinds.cuda()].contiguous()
    table = pool.table[int(pool.slots_np[0])][None].expand(n, -1).contiguous()
    cache = pkg.KV8Cache(pool.pages, pool.scales, table)
    kv_len = torch.tensor(lens, dtype=torch.int32)[kinds].cuda()
    batch = pkg.KV8Batch(torch.arange(n + 1, dtype=torch.int32, device="cuda"), kv_len, n, 1, max(lens))
    out, lse = torch.zeros_like(q), torch.zeros((n, 4), device="cuda")
    cache.attention(batch, q, out, 0.1, window=window, lse=lse)
    cache.check()
    ranges = max((t.numel() for t in batch._workspaces.values()), default=0) / (n * 2 * 8 * (hd + 4) * 4)
    assert 33000 / 16 / max(1, ranges) > 512, "ranges shorter than these are in test_gpu_kv8.py"
    assert torch.equal(out, out[: len(lens)][kinds.cuda()]) and torch.equal(lse, lse[: len(lens)][kinds.cuda()])
    whole = pool.values[0], pool.exps[0]
    for i, L in enumerate(lens):
        pool.values[0], pool.exps[0] = whole[0][:, :L], whole[1][:, : -(-L // 16)]
        check_attention(pool, q1[i: i + 1], out[i: i + 1], lse[i: i + 1], [(L - 1, 1)], 0.1, window, True, "f16")
