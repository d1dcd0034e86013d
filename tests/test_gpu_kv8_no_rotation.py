"""Appending without a rotation (needs a B200): every element stands for itself, an infinite one or a NaN included."""
import pytest
import torch

from kv8_helpers import Pool

pytestmark = pytest.mark.gpu


def special(n, heads, hd):
    x = torch.randn((n, heads, hd), device="cuda").clamp(0.1, 3.0)
    x[1, 0, 7], x[2, 0, hd - 3], x[3] = float("inf"), float("nan"), 0.0
    return x


@pytest.mark.parametrize("hd", [64, 128])
def test_norms_of_rows_with_infinities_nan_and_zeros(pkg, hd):
    """x / sqrt(mean x^2 + eps): an infinite element makes itself NaN and the others zero, a NaN all of its row, and
    a row of zeros stays zero."""
    q, k = special(5, 2, hd), special(5, 1, hd)
    pool = Pool(pkg, [5], 1, hd)
    out = torch.full((5, 2, hd), 7.0, dtype=torch.float16, device="cuda")
    one = torch.ones(hd, device="cuda")
    pool.cache.append(pool.batch([5], [5]), q, k, k.clone(), out, q_norm=one, k_norm=one)
    pool.cache.check()
    keys = torch.empty((5, 1, hd), device="cuda")
    pool.cache.read(pool.batch([5], [5]), keys, torch.empty_like(keys))
    for rows in (out[:, :1].float(), keys):
        assert torch.isnan(rows[1, 0, 7]) and not rows[1, 0, :7].any() and not rows[1, 0, 8:].any()
        assert torch.isnan(rows[2, 0]).all() and not rows[3].any()
        assert torch.isfinite(rows[[0, 4]]).all() and rows[[0, 4]].all()
    assert torch.isfinite(out[1:3, 1]).all()


@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_without_norm_and_rotation_are_unchanged(pkg, kind, hd):
    q = special(5, 3, hd).to(kind)
    pool = Pool(pkg, [5], 1, hd)
    k = torch.zeros((5, 1, hd), dtype=kind, device="cuda")
    out = torch.full((5, 3, hd), 7.0, dtype=torch.bfloat16 if kind == torch.bfloat16 else torch.float16, device="cuda")
    pool.cache.append(pool.batch([5], [5]), q, k, k, out)
    want = q.to(out.dtype)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(want))
