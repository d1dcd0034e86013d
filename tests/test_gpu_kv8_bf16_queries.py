"""bf16 queries whose elements span more than f16's range in one row (needs a B200). Tolerances: test_gpu_kv8.py."""
import numpy as np
import pytest
import torch

from kv8_helpers import Pool
from test_gpu_kv8 import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", ["few", "many"])
@pytest.mark.parametrize("hd,new", [(64, 3), (128, 70)])
def test_small_elements_beside_a_large_one_in_bf16_queries(pkg, monkeypatch, kernel, hd, new):
    """A query element 2^26 times the others that meets keys of zero: the others' scores keep all their bits."""
    monkeypatch.setenv("BZB_KV8_ATTENTION", kernel)
    L = 90
    pool = Pool(pkg, [L], 1, hd, seed=3, fill=[L])
    pool.pages[:, 0, :, :, 5] = 0
    pool.values[0][0, :, :, 5] = 0
    x = np.random.default_rng(new).standard_normal((new, 2, hd)).astype(np.float32)
    x[..., 5] = 2.0 ** 26
    q = torch.from_numpy(x).cuda().bfloat16()
    out, lse = torch.full_like(q, float("nan")), torch.full((new, 2), float("nan"), device="cuda")
    pool.cache.attention(pool.batch([new], [L]), q, out, 0.125, lse=lse)
    pool.cache.check()
    check_attention(pool, q, out, lse, [(L - new, new)], 0.125, 0, True, "bf16")
