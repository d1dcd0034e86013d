"""Queries of any magnitude that their type holds (needs a B200)."""
import numpy as np
import pytest
import torch

from kv8_helpers import TYPES, UNIT, Pool, turned
from test_gpu_kv8 import rope_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
def test_norms_of_queries_whose_squares_leave_f32(pkg, kind, hd, eps):
    """Rows from 1e-37 to 3e38 beside ordinary ones: the normed row of the formula, also where the sum of the squares
    is beyond f32 or below it. Tolerance: the output's rounding and a few of f32's (the norm, two products, the turn)."""
    mags = [1.0, 1e25, 3e37, 1e19, 1e-25, 1e-37, 1e-12, 1.0, 2e18, 1e-16, 1e-20, 1.0, 1e38]
    n, H = len(mags), 3
    rng = np.random.default_rng(hd)
    x = rng.uniform(-3, 3, (n, H, hd)) * np.array(mags)[:, None, None]
    q = torch.from_numpy(x.astype(np.float32)).cuda().to(TYPES[kind])
    assert torch.isfinite(q).all()
    w = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
    table = rope_table(n, hd)
    pool = Pool(pkg, [n], 1, hd)
    k = torch.zeros((n, 1, hd), dtype=TYPES[kind], device="cuda")
    out = torch.full((n, H, hd), float("nan"), dtype=torch.bfloat16, device="cuda")
    pool.cache.append(pool.batch([n], [n]), q, k, k, out, q_norm=torch.from_numpy(w).cuda(), eps=eps, rope=torch.from_numpy(table).cuda())
    want = turned(q.double().cpu().numpy(), w, float(np.float32(eps)), table)
    got = out.double().cpu().numpy()
    top = np.abs(want).max(-1, keepdims=True)
    assert (np.abs(got - want) <= UNIT["bf16"] * np.abs(want) + 2e-6 * top + 2.0 ** -133).all()
