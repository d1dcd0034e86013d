"""Blocks whose scales lie far apart, in the same 128 positions of the cache: a loud block takes no precision from the
quiet ones beside it, for rows that see it and for rows that do not (needs a B200).

Tolerances as in test_gpu_kv8.py, but taken over the keys that a row sees, row by row: weights in f16 (2^-11 relative;
below 2^-14 of the largest 2^-25 absolute, in units of the largest value that the row sees), the result in the output
type, the scores' f32 products and sums 2^-20 of their magnitude.
"""
import numpy as np
import pytest
import torch

from kv8_helpers import UNIT, Pool, e4m3_table

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["few", "many"])
def kernel(request, monkeypatch):
    monkeypatch.setenv("BZB_KV8_ATTENTION", request.param)


def put_block(pool, plane, blk, codes, e):
    """Sets one block of 16 positions of sequence 0 (kv head 0): bytes [16][hd] and the scale's exponent."""
    hd = pool.hd
    pg, off = pool.table_np[pool.slots_np[0], blk * 16 // pool.page], blk * 16 % pool.page
    to = codes if plane == 0 else codes.reshape(4, 4, hd // 4, 4).transpose(2, 0, 3, 1).reshape(16, hd)
    pool.pages[pg, plane, 0, off: off + 16] = torch.from_numpy(np.ascontiguousarray(to)).cuda()
    pool.scales[pg, plane, 0, off // 16] = 2.0 ** e
    n = pool.values[0].shape[1]
    lo, hi = blk * 16, min(n, blk * 16 + 16)
    pool.values[0][plane, lo:hi, 0] = e4m3_table()[codes][: hi - lo]
    pool.exps[0][plane, blk, 0] = e


def check_rows(pool, q, out, lse, old, scale, window, kind):
    k, v = pool.dequantised(0, pool.values[0].shape[1])
    q, out, lse = (t.double().cpu().numpy() for t in (q, out, lse))
    for i in range(len(q)):
        p = old + i
        lo, hi = (max(0, p - window + 1) if window else 0), p + 1
        kk, vv = k[lo:hi, 0], v[lo:hi, 0]
        for h in range(q.shape[1]):
            s = scale * (kk @ q[i, h])
            w = np.exp(s - s.max())
            want, mag = w @ vv / w.sum(), w @ np.abs(vv) / w.sum()
            eps = abs(scale) * (np.abs(kk) @ np.abs(q[i, h])).max() * 2.0 ** -20
            bound = (mag * (2.0 ** -11 + 2 * eps + 2.0 ** -18) + np.abs(want) * UNIT[kind]
                     + (hi - lo) * 2.0 ** -24 * np.abs(vv).max() + 1e-7)
            # (what the output's type cannot hold is infinite)
            most = float(torch.finfo(getattr(torch, {"f16": "float16", "bf16": "bfloat16"}[kind])).max)
            over = np.abs(want) > most * (1 + UNIT[kind])
            assert (np.isinf(out[i, h][over]) & (np.sign(out[i, h][over]) == np.sign(want[over]))).all()
            near = np.abs(want) > most * (1 - UNIT[kind]) - bound  # (either side of the largest)
            ok = (np.abs(out[i, h] - want) <= bound) | near
            assert ok.all(), (i, h, np.max((np.abs(out[i, h] - want) / bound)[~near]))
            wl = s.max() + np.log(w.sum())
            assert abs(lse[i, h] - wl) <= eps + (hi - lo) * 2.0 ** -24 + 2.0 ** -20 + abs(wl) * 2.0 ** -21, (i, h)


@pytest.mark.parametrize("hd,kind", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("plane", [0, 1])
@pytest.mark.parametrize("apart", [10, 20, 30, 55])
@pytest.mark.parametrize("old,new,window,blk", [(0, 150, 0, 5), (149, 1, 0, 5), (60, 90, 20, 3), (60, 90, 20, 8)])
def test_a_loud_block_beside_quiet_ones(pkg, hd, kind, plane, apart, old, new, window, blk):
    L, quiet = old + new, -15
    pool = Pool(pkg, [L], 1, hd, 32, seed=blk + apart, fill=[L])
    for other in range(-(-L // 16)):
        for pl in (0, 1):
            pg, off = pool.table_np[pool.slots_np[0], other // 2], other % 2
            pool.scales[pg, pl, 0, off] = 2.0 ** (-8 if pl == 0 else quiet)
            pool.exps[0][pl, other, 0] = -8 if pl == 0 else quiet
    rng = np.random.default_rng(apart)
    codes = np.zeros((16, hd), np.uint8)
    if plane == 0:
        # keys that are loud in one element only, which the queries do not have: their scores are zero
        codes[:, 3] = rng.integers(0x70, 0x7F, 16) | (rng.integers(0, 2, 16) << 7)
    else:
        codes[:] = rng.integers(0x60, 0x7F, (16, hd)) | (rng.integers(0, 2, (16, hd)) << 7)
    put_block(pool, plane, blk, codes, min(40, (-8 if plane == 0 else quiet) + apart))
    x = rng.standard_normal((new, 2, hd)).astype(np.float32) * 1.5
    x[..., 3] = 0
    q = torch.from_numpy(x).cuda().to(torch.float16 if kind == "f16" else torch.bfloat16)
    out, lse = torch.full_like(q, float("nan")), torch.full((new, 2), float("nan"), device="cuda")
    pool.cache.attention(pool.batch([new], [L]), q, out, hd ** -0.5, window=window, lse=lse)
    pool.cache.check()
    check_rows(pool, q, out, lse, old, hd ** -0.5, window, kind)


@pytest.mark.parametrize("new", [1, 100, 700])
@pytest.mark.parametrize("values", ["alike", "apart"])
def test_every_block_at_another_scale(pkg, new, values):
    """Key scales over 26 powers of two in one stage, all of which count: each block's keys have an element of their own,
    which the queries have in the inverse magnitude, so every score is about one."""
    L, hd = 700, 64
    rng = np.random.default_rng(new)
    pool = Pool(pkg, [L], 1, hd, 64, seed=4, fill=[L])
    blocks = -(-L // 16)
    e = rng.integers(-13, 14, (2, blocks))
    if values == "alike":
        e[1] = -3
    x = np.zeros((new, 2, hd), np.float32)
    for blk in range(blocks):
        codes = np.zeros((16, hd), np.uint8)
        codes[:, blk] = rng.integers(0x28, 0x40, 16) | (rng.integers(0, 2, 16) << 7)  # magnitudes 0.25 to 1.9
        put_block(pool, 0, blk, codes, int(e[0, blk]))
        put_block(pool, 1, blk, rng.integers(0, 0x7F, (16, hd), dtype=np.uint8) | (rng.integers(0, 2, (16, hd), dtype=np.uint8) << 7), int(e[1, blk]))
        x[..., blk] = rng.uniform(-2, 2, (new, 2)) * 2.0 ** -float(e[0, blk])
    q = torch.from_numpy(x).cuda().half()
    out, lse = torch.full_like(q, float("nan")), torch.full((new, 2), float("nan"), device="cuda")
    pool.cache.attention(pool.batch([new], [L]), q, out, 1.0, lse=lse)
    pool.cache.check()
    check_rows(pool, q, out, lse, L - new, 1.0, 0, "f16")
