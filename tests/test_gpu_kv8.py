"""The 8-bit paged key/value cache on the GPU against a plain 64-bit restatement (needs a B200).

Tolerances, from the arithmetic: a value is stored as the nearest e4m3 of its block's scale, so values
(which are only scaled by a power of two) and rescaled older positions must match bit for bit, and keys
(normed and rotated first) within half a spacing, 2^-4 relative or 2^-10 scales. Attention rounds
its weights to f16 (2^-11 relative; below 2^-14 of the largest 2^-25 absolute) and its result to the
output type, and its scores carry f32 rounding of the products' sum.
"""
import numpy as np
import pytest
import torch

from kv8_helpers import E_MAX, E_MIN, TYPES, UNIT, Pool, attend, exponent, round_e4m3, turned

pytestmark = pytest.mark.gpu
EPS = 1e-5


def rope_table(n, hd):
    a = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)[None]
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def strided(x, kind, layout):
    """x [n][heads][hd] as a GPU tensor of a layout: packed, a column range of wider rows, an odd offset, head-major."""
    t = torch.from_numpy(x).to("cuda", TYPES[kind])
    n, H, hd = t.shape
    if layout == "packed":
        return t
    if layout == "heads":
        return t.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    width, at = (H * hd + 64, 32) if layout == "wide" else (H * hd + 5, 3)
    w = torch.full((n, width), float("nan"), dtype=t.dtype, device="cuda")
    v = w[:, at: at + H * hd].unflatten(1, (H, hd))
    v.copy_(t)
    return v


def append_expected(pool, b, k64, v64, start):
    """Updates the pool's expected content by appending rows at positions start.. (k64: already turned)."""
    old_v, old_e = pool.values[b][:, :start], pool.exps[b]
    end = start + len(k64)
    blocks = -(-end // 16)
    vals = np.concatenate([old_v, np.zeros((2, end - start) + old_v.shape[2:])], 1)
    exps = np.concatenate([old_e[:, : -(-start // 16)], np.zeros((2, blocks - -(-start // 16), pool.n_kv), np.int64)], 1)
    for i, x in enumerate((k64, v64)):
        x = np.where(np.isfinite(x), x, np.nan)
        for blk in range(start // 16, blocks):
            lo, hi = max(start, blk * 16), min(end, blk * 16 + 16)
            for h in range(pool.n_kv):
                new = x[lo - start: hi - start, h]
                e = exponent(np.nanmax(np.abs(new), initial=0.0))
                if blk * 16 < start:
                    was = old_e[i, blk, h]
                    e = max(e, was)
                    vals[i, blk * 16: start, h] = round_e4m3(vals[i, blk * 16: start, h] * 2.0 ** (was - e))
                exps[i, blk, h] = e
                vals[i, lo:hi, h] = new * 2.0 ** -float(e)  # (not rounded yet)
    pool.values[b], pool.exps[b] = vals, exps
    return vals, exps


def same(a, b):
    return np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.nan_to_num(a), np.nan_to_num(b))


def check_append(pool, b, start, n, tol_k=1e-5):
    end = start + n
    got, e, behind = pool.held(b, end)
    want, we = pool.values[b], pool.exps[b]
    first = start // 16 * 16
    assert np.array_equal(e, we), (e - we)
    assert not behind.any(), "positions behind the end are zero"
    assert same(got[:, :first], want[:, :first])
    assert same(got[:, first:start], want[:, first:start]), "older positions of a block: exact"
    assert same(got[1, start:], round_e4m3(want[1, start:])), "values: exact"
    w, g = want[0, start:], got[0, start:]
    assert np.array_equal(np.isnan(w), np.isnan(g))
    w, g = np.nan_to_num(w), np.nan_to_num(g)
    slack = tol_k * np.abs(want[0, start:][~np.isnan(want[0, start:])]).max(initial=0.0)
    assert (np.abs(g - np.clip(w, -448, 448)) <= np.maximum(np.abs(w) * 2.0 ** -4, 2.0 ** -10) + slack).all()
    pool.values[b][0, start:], pool.values[b][1, start:] = got[0, start:], round_e4m3(want[1, start:])


APPENDS = [
    # heads, kv, hd, type, page, layout, norm, rope, (old, new) of each sequence
    (4, 2, 64, "f32", 16, "packed", True, True, [(0, 1), (1, 1), (15, 1), (16, 1), (217, 1)]),
    (32, 8, 64, "f32", 16, "wide", True, True, [(0, 33), (7, 0), (9, 9), (40, 1), (0, 16), (15, 2)]),
    (6, 2, 128, "f16", 64, "wide", True, True, [(0, 200), (63, 66), (5, 17)]),
    (7, 1, 128, "bf16", 32, "odd", True, True, [(3, 50), (0, 31)]),
    (8, 8, 64, "f16", 128, "heads", False, True, [(130, 140), (0, 1)]),
    (5, 5, 64, "bf16", 256, "odd", True, False, [(250, 20), (16, 16)]),
    (0, 3, 128, "f32", 16, "odd", False, False, [(0, 40), (17, 15), (31, 1)]),
]


@pytest.mark.parametrize("H,KV,hd,kind,page,layout,norm,rope,seqs", APPENDS)
def test_append_and_read_match_64_bit(pkg, H, KV, hd, kind, page, layout, norm, rope, seqs):
    rng = np.random.default_rng(H * hd + page)
    olds, news = [s[0] for s in seqs], [s[1] for s in seqs]
    lens = [a + b for a, b in seqs]
    pool = Pool(pkg, lens, KV, hd, page, seed=page, fill=olds)
    before = pool.pages.clone()
    n = sum(news)
    xq, xk, xv = (rng.standard_normal((n, h, hd)).astype(np.float32) * 2 for h in (H, KV, KV))
    cast = lambda x: torch.from_numpy(x).to(TYPES[kind]).double().numpy()  # noqa: E731
    wq, wk = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32), (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
    table = rope_table(max(lens), hd)
    batch = pool.batch(news, lens)
    out_kind = "bf16" if kind == "bf16" else "f16"
    q_out = strided(np.zeros((n, H, hd), np.float32), out_kind, layout) if H else None
    g = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    pool.cache.append(batch, strided(xq, kind, layout) if H else None, strided(xk, kind, layout), strided(xv, kind, layout), q_out,
                      g(wq) if norm else None, g(wk) if norm else None, EPS, g(table) if rope else None)
    pool.cache.check()
    at = 0
    for b, (old, new) in enumerate(seqs):
        cs = table[old: old + new] if rope else None
        rows = slice(at, at + new)
        at += new
        if H:
            want = turned(cast(xq[rows]), wq if norm else None, EPS, cs)
            got = q_out[rows].double().cpu().numpy()
            if new:
                assert np.abs(got - want).max() <= UNIT[out_kind] * np.abs(want).max() + 2e-6 * np.abs(want).max()
        append_expected(pool, b, turned(cast(xk[rows]), wk if norm else None, EPS, cs), cast(xv[rows]), old)
        if new:
            check_append(pool, b, old, new)
    # pages of no sequence stay as they were
    spare = torch.from_numpy(pool.spare.astype(np.int64)).cuda()
    assert torch.equal(pool.pages[spare], before[spare])
    # and everything reads back as what it stands for, in each type
    for rk in ("f32", "f16", "bf16"):
        everything = pool.batch(lens, lens)
        ko, vo = (strided(np.zeros((sum(lens), KV, hd), np.float32), rk, layout) for _ in range(2))
        pool.cache.read(everything, ko, vo)
        at = 0
        for b, L in enumerate(lens):
            want = torch.from_numpy(pool.dequantised(b, L)).to(TYPES[rk])
            assert torch.equal(ko[at: at + L].cpu(), want[0]) and torch.equal(vo[at: at + L].cpu(), want[1])
            at += L


def test_append_one_by_one_gives_the_same_scales_as_at_once(pkg):
    """A block's scale depends on its values only, and older positions keep theirs wherever they stay normal numbers."""
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((2, 40, 2, 64)) * np.exp(rng.uniform(-1, 1, (2, 40, 1, 1)))).astype(np.float32)
    x = np.sign(x) * np.maximum(np.abs(x), 0.2)  # nothing subnormal: 448 / 2^-6 covers the range
    one, many = Pool(pkg, [40], 2, 64, seed=1), Pool(pkg, [40], 2, 64, seed=2)
    g = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    one.cache.append(one.batch([40], [40]), None, g(x[0]), g(x[1]), None)
    for i in range(40):
        many.cache.append(many.batch([1], [i + 1]), None, g(x[0, i: i + 1]), g(x[1, i: i + 1]), None)
    (a, ea, _), (b, eb, _) = one.held(0, 40), many.held(0, 40)
    assert np.array_equal(ea, eb)
    # (each value was rounded at the scale of its time and then only moved by powers of two)
    assert np.array_equal(a, b)


def test_append_twice_is_the_same_as_once(pkg):
    rng = np.random.default_rng(6)
    pool = Pool(pkg, [50, 9], 2, 128, 32, seed=3, fill=[21, 3])
    x = [torch.from_numpy(rng.standard_normal((35, h, 128)).astype(np.float32)).cuda() * 3 for h in (4, 2, 2)]
    out = torch.zeros((35, 4, 128), dtype=torch.float16, device="cuda")
    batch = pool.batch([29, 6], [50, 9])
    pool.cache.append(batch, *x, out)
    a, s, o = pool.pages.clone(), pool.scales.clone(), out.clone()
    pool.cache.append(batch, *x, out)
    assert torch.equal(a, pool.pages) and torch.equal(s, pool.scales) and torch.equal(o, out)


def test_append_extreme_values(pkg):
    """Zero blocks, the smallest and largest scales, exact boundaries, infinities and NaN."""
    hd = 64
    x = np.zeros((16 * 7, 1, hd), np.float32)
    x[16:32, 0, 3] = 448.0            # exactly 2^0
    x[32:48, 0, 5] = np.nextafter(np.float32(448.0), np.float32(1000))  # just above: 2^1
    x[48:64, 0] = 1e-30               # below the smallest scale: zero
    x[64:80, 0, 1] = 3e38             # above the largest: saturates
    x[64:80, 0, 2] = -1e10
    x[80:96, 0] = 1.5
    x[81, 0, 7], x[82, 0, 8], x[83, 0, 9] = np.inf, -np.inf, np.nan
    x[96:112, 0] = np.float32(1e-42)  # a subnormal float
    pool = Pool(pkg, [len(x)], 1, hd)
    g = torch.from_numpy(x).cuda()
    pool.cache.append(pool.batch([len(x)], [len(x)]), None, g, g.clone(), None)
    append_expected(pool, 0, x.astype(np.float64), x.astype(np.float64), 0)
    assert [int(e) for e in pool.exps[0][0, :, 0]] == [E_MIN, 0, 1, E_MIN, E_MAX, exponent(1.5), E_MIN]
    check_append(pool, 0, 0, len(x))


@pytest.mark.parametrize("hd", [64, 128])
def test_keys_are_the_correctly_rounded_ones(pkg, hd):
    """Normed and rotated keys are rounded once, from the exact value: byte for byte the 64-bit result's. Without eps
    too, in whole blocks and in one whose last positions are empty (and stay zero)."""
    rng = np.random.default_rng(hd)
    n = 16 * 900 + 5
    x = rng.standard_normal((n, 1, hd)).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
    table = rope_table(n, hd)
    pool = Pool(pkg, [n], 1, hd, 256, seed=1)
    g = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    pool.cache.append(pool.batch([n], [n]), None, g(x), g(x), None, k_norm=g(w), eps=0.0, rope=g(table))
    append_expected(pool, 0, turned(x, w, 0.0, table), x.astype(np.float64), 0)
    got, e, behind = pool.held(0, n)
    assert np.array_equal(e, pool.exps[0]) and not behind.any()
    assert np.array_equal(got, round_e4m3(pool.values[0]))


def test_padding_rows_and_empty_sequences(pkg):
    rng = np.random.default_rng(8)
    pool = Pool(pkg, [20, 20, 20, 20], 2, 64, seed=4, fill=[0, 0, 12, 0])
    news, lens = [3, 5, 4, 0], [0, 2, 16, 0]   # three padding rows; three and two real ones; plain; nothing
    k, v = (torch.from_numpy(rng.standard_normal((12, 2, 64)).astype(np.float32)).cuda() for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((12, 4, 64)).astype(np.float32)).cuda().half()
    q_out = torch.full((12, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    batch = pool.batch(news, lens)
    pool.cache.append(batch, q.float(), k, v, q_out)
    pool.cache.check()
    pad = [0, 1, 2, 3, 4, 5]
    assert (q_out[pad] == 7.0).all() and torch.equal(q_out[6:], q[6:])
    ko, vo = (torch.full((12, 2, 64), 7.0, device="cuda") for _ in range(2))
    pool.cache.read(batch, ko, vo)
    assert not ko[pad].any() and not vo[pad].any() and ko[6:].any()
    out, lse = torch.full((12, 4, 64), 7.0, dtype=torch.float16, device="cuda"), torch.zeros((12, 4), device="cuda")
    q[:6] = float("nan")
    pool.cache.attention(batch, q, out, 0.125, lse=lse)
    pool.cache.check()
    assert not out[pad].any() and torch.isneginf(lse[pad]).all() and torch.isfinite(out).all() and torch.isfinite(lse[6:]).all()


ATTENDS = [
    # heads, kv, hd, type, page, layout, window, causal, (old, new)
    (4, 2, 64, "f16", 16, "packed", 0, True, [(0, 1), (15, 1), (16, 1), (217, 1), (2030, 1)]),
    (32, 8, 64, "f16", 16, "wide", 0, True, [(90, 1), (700, 1), (0, 1), (33, 1)]),
    (32, 8, 64, "bf16", 64, "packed", 0, True, [(3000, 1)]),
    (28, 4, 128, "bf16", 32, "odd", 100, True, [(50, 5), (300, 5), (0, 5), (98, 5)]),
    (8, 8, 128, "f16", 16, "heads", 0, True, [(1500, 1), (3, 1)]),
    (12, 1, 64, "f16", 16, "packed", 7, True, [(40, 1), (2, 3), (0, 9)]),
    (5, 1, 128, "bf16", 256, "odd", 0, False, [(100, 4), (0, 3), (255, 2)]),
    (8, 2, 64, "f16", 16, "odd", 0, True, [(0, 1), (0, 17), (0, 70), (0, 129), (5, 0)]),
    (32, 8, 64, "bf16", 128, "packed", 0, True, [(0, 300), (128, 64), (77, 131)]),
    (16, 2, 128, "f16", 16, "wide", 50, True, [(30, 200), (0, 97)]),
    (4, 4, 128, "bf16", 64, "heads", 0, False, [(200, 140), (1, 65)]),
    (40, 8, 128, "f16", 64, "packed", 1, True, [(64, 90), (0, 33)]),
]


def check_attention(pool, q, out, lse, seqs, scale, window, causal, kind, used=None):
    at = 0
    for b, (old, new) in enumerate(seqs):
        L = old + new
        k, v = pool.dequantised(b, L)
        q64 = q[at: at + new].double().cpu().numpy()
        want, wl, mag, sc = attend(q64, k, v, scale, old, causal, window)
        got, gl = out[at: at + new].double().cpu().numpy(), lse[at: at + new].double().cpu().numpy()
        at += new
        if not new:
            continue
        eps = sc * 2.0 ** -20
        bound = (mag * (2.0 ** -11 + 2 * eps[..., None] + 2.0 ** -18) + np.abs(want) * UNIT[kind]
                 + L * 2.0 ** -25 * 2 * np.abs(v).max(initial=0) + 1e-7)
        assert (np.abs(got - want) <= bound).all(), (b, np.max(np.abs(got - want) / bound))
        bl = eps + L * 2.0 ** -24 + 2.0 ** -20 + np.abs(np.where(np.isfinite(wl), wl, 0)) * 2.0 ** -21
        fin = np.isfinite(wl)
        assert np.array_equal(fin, np.isfinite(gl))
        assert (np.abs(gl - wl)[fin] <= bl[fin]).all(), np.max((np.abs(gl - wl) / bl)[fin])


@pytest.mark.parametrize("H,KV,hd,kind,page,layout,window,causal,seqs", ATTENDS)
def test_attention_matches_64_bit(pkg, H, KV, hd, kind, page, layout, window, causal, seqs):
    rng = np.random.default_rng(H + hd + page)
    lens, news = [a + b for a, b in seqs], [s[1] for s in seqs]
    pool = Pool(pkg, lens, KV, hd, page, seed=window + 1, fill=lens)
    n = sum(news)
    q = strided(rng.standard_normal((n, H, hd)).astype(np.float32) * 1.5, kind, layout)
    out = strided(np.full((n, H, hd), np.nan, np.float32), kind, layout)
    lse = torch.full((n, H), float("nan"), device="cuda")
    scale = hd ** -0.5
    pool.cache.attention(pool.batch(news, lens), q, out, scale, causal=causal, window=window, lse=lse)
    pool.cache.check()
    check_attention(pool, q, out, lse, seqs, scale, window, causal, kind)


# rows of a kv head (tokens x group) on both sides of every change of kernel and tile, and contexts that are split
EDGES = [(1, 8, 70), (1, 9, 70), (3, 5, 300), (8, 8, 100), (13, 5, 500), (16, 4, 64), (21, 3, 40), (64, 1, 33), (65, 1, 200),
         (32, 4, 900), (129, 2, 129), (257, 1, 300), (43, 6, 2100), (2, 12, 6000), (90, 3, 5000)]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,group,L", EDGES)
def test_attention_at_the_edges_of_its_tiles(pkg, hd, new, group, L):
    new = min(new, L)
    pool = Pool(pkg, [L], 1, hd, 16, seed=L + new, fill=[L])
    q = torch.from_numpy(np.random.default_rng(new).standard_normal((new, group, hd)).astype(np.float32)).cuda().half()
    out, lse = torch.full_like(q, float("nan")), torch.full((new, group), float("nan"), device="cuda")
    pool.cache.attention(pool.batch([new], [L]), q, out, 0.1, lse=lse)
    pool.cache.check()
    check_attention(pool, q, out, lse, [(L - new, new)], 0.1, 0, True, "f16")


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 3.0])
def test_attention_scales(pkg, new, scale):
    """Any finite scale: a negative one, none, and one that leaves a single key."""
    pool = Pool(pkg, [90], 2, 64, seed=2, fill=[90])
    q = torch.from_numpy(np.random.default_rng(9).standard_normal((new, 4, 64)).astype(np.float32)).cuda().half()
    out, lse = torch.zeros_like(q), torch.zeros((new, 4), device="cuda")
    pool.cache.attention(pool.batch([new], [90]), q, out, scale, lse=lse)
    check_attention(pool, q, out, lse, [(90 - new, new)], scale, 0, True, "f16")
    with pytest.raises(RuntimeError, match="finite"):
        pool.cache.attention(pool.batch([new], [90]), q, out, float("inf"))


def test_contexts_longer_than_one_range_with_many_sequences(pkg):
    """More positions than a CTA's range may hold, in a batch that would otherwise not be split: sequences that
    share their pages all give the one answer."""
    L, n, KV, hd = 9000, 150, 8, 64
    pool = Pool(pkg, [L], KV, hd, 64, seed=3, fill=[L])
    q1 = torch.from_numpy(np.random.default_rng(5).standard_normal((1, 16, hd)).astype(np.float32)).cuda().half()
    q = q1.expand(n, 16, hd).contiguous()
    table = pool.table[int(pool.slots_np[0])][None].expand(n, -1).contiguous()
    cache = pkg.KV8Cache(pool.pages, pool.scales, table)
    batch = pkg.KV8Batch(torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.full((n,), L, dtype=torch.int32, device="cuda"),
                         n, 1, L)
    out, lse = torch.zeros_like(q), torch.zeros((n, 16), device="cuda")
    cache.attention(batch, q, out, 0.125, lse=lse)
    cache.check()
    assert torch.equal(out, out[:1].expand_as(out)) and torch.equal(lse, lse[:1].expand_as(lse))
    check_attention(pool, q1, out[:1], lse[:1], [(L - 1, 1)], 0.125, 0, True, "f16")


def test_ragged_rows_of_one_call(pkg):
    """Sequences with one row, with none and with hundreds in the same call, and bounds larger than any of them."""
    seqs = [(5, 1), (100, 0), (0, 260), (40, 7), (1000, 1), (3, 64)]
    lens, news = [a + b for a, b in seqs], [s[1] for s in seqs]
    pool = Pool(pkg, lens, 2, 64, 32, seed=21, fill=lens)
    n = sum(news)
    q = torch.from_numpy(np.random.default_rng(3).standard_normal((n, 6, 64)).astype(np.float32)).cuda().bfloat16()
    out, lse = torch.full_like(q, float("nan")), torch.full((n, 6), float("nan"), device="cuda")
    pool.cache.attention(pool.batch(news, lens, max_new=300, max_len=1024), q, out, 0.125, lse=lse)
    pool.cache.check()
    check_attention(pool, q, out, lse, seqs, 0.125, 0, True, "bf16")


def test_c_calls_with_a_workspace_of_any_content(pkg):
    """The C entry points on plain pointers: the workspace's content does not matter, its size does."""
    import ctypes
    from bz_ggml_b200.kv8 import _Batch, _Cache
    lib = pkg.lib().lib
    pool = Pool(pkg, [3000], 2, 128, seed=6, fill=[3000])

    class Rows(ctypes.Structure):
        _fields_ = [("data", ctypes.c_void_p), ("row", ctypes.c_longlong), ("head", ctypes.c_longlong), ("n", ctypes.c_int),
                    ("type", ctypes.c_int)]

    q = torch.from_numpy(np.random.default_rng(8).standard_normal((1, 4, 128)).astype(np.float32)).cuda().half()
    batch = pool.batch([1], [3000])
    c, b = ctypes.byref(pool.cache._c), ctypes.byref(batch._c)
    need = lib.bzb_kv8_attention_workspace(c, b, 4, 1, 0)
    assert need > 0
    stream = torch.cuda.current_stream().cuda_stream
    got = []
    for fill in (0, 255, 127):
        ws = torch.full((need + 64,), fill, dtype=torch.uint8, device="cuda")
        out = torch.zeros_like(q)
        rq, ro = (ctypes.byref(Rows(t.data_ptr(), 512, 128, 4, 1)) for t in (q, out))
        assert lib.bzb_kv8_attention(c, b, rq, ro, None, 0.09, 1, 0, ws.data_ptr(), need, stream) == 0
        torch.cuda.synchronize()
        assert (ws[need:] == fill).all(), "wrote past the workspace"
        got.append(out)
        assert lib.bzb_kv8_attention(c, b, rq, ro, None, 0.09, 1, 0, ws.data_ptr(), need - 1, stream) == -1
        assert b"workspace" in lib.breeze_last_error()
        assert lib.bzb_kv8_attention(c, b, rq, ro, None, 0.09, 1, 0, None, need, stream) == -1
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    lse = torch.zeros((1, 4), device="cuda")
    pool.cache.attention(batch, q, out, 0.09, lse=lse)
    assert torch.equal(out, got[0])
    check_attention(pool, q, out, lse, [(2999, 1)], 0.09, 0, True, "f16")
    assert isinstance(pool.cache._c, _Cache) and isinstance(batch._c, _Batch)


@pytest.mark.parametrize("new", [1, 3, 150])
def test_attention_with_value_scales_far_apart(pkg, new):
    """Blocks whose scales differ by 2^40: weights carry the values' scales, sums must not."""
    pool = Pool(pkg, [300], 2, 64, seed=9)
    pool.fill([300], spread=(-24, 16))
    q = torch.from_numpy(np.random.default_rng(1).standard_normal((new, 4, 64)).astype(np.float32)).cuda().half()
    pool.exps[0][0] = -8
    pool.scales[:, 0] = 2.0 ** -8
    out, lse = torch.zeros((new, 4, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((new, 4), device="cuda")
    pool.cache.attention(pool.batch([new], [300]), q.bfloat16(), out, 0.125, lse=lse)
    check_attention(pool, q.bfloat16(), out, lse, [(300 - new, new)], 0.125, 0, True, "bf16")


@pytest.mark.parametrize("hd,new", [(64, 4), (128, 3), (64, 40), (128, 70)])
def test_nan_reaches_only_the_rows_that_see_it(pkg, hd, new):
    """A NaN key or value of a position leaves every row that does not look at it alone."""
    L, W, KV = 100, 30, 2
    rng = np.random.default_rng(2)
    q = torch.from_numpy(rng.standard_normal((new, 4, hd)).astype(np.float32)).cuda().half()
    for plane, at in ((0, L - 2), (1, L - 2), (1, L - new - 20), (0, 40), (1, 47)):
        pool = Pool(pkg, [L], KV, hd, seed=at, fill=[L])
        pg, off = pool.table_np[pool.slots_np[0], at // 16], at % 16
        if plane == 0:
            pool.pages[pg, 0, 1, off, 5] = 0x7F
        else:
            pool.pages[pg, 1, 1].view(-1)[(9 // 4) * 64 + off // 4 * 16 + (9 % 4) * 4 + off % 4] = 0xFF
        out, lse = torch.zeros_like(q), torch.zeros((new, 4), device="cuda")
        pool.cache.attention(pool.batch([new], [L]), q, out, 0.1, window=W, lse=lse)
        bad = torch.isnan(out).cpu().numpy()
        for i in range(new):
            p = L - new + i
            sees = p - W < at <= p
            assert not bad[i, :2].any()
            if plane == 0:
                assert bad[i, 2:].all() == sees and bad[i, 2:].any() == sees, (plane, at, i)
            else:
                assert bad[i, 2:, 9].all() == sees and not np.delete(bad[i, 2:], 9, -1).any(), (plane, at, i)


def test_bf16_queries_outside_f16(pkg):
    pool = Pool(pkg, [70], 1, 64, seed=12, fill=[70])
    x = np.random.default_rng(3).standard_normal((2, 2, 64)).astype(np.float32)
    for f in (1e30, 1e-30):
        q = torch.from_numpy(x * f).cuda().bfloat16()
        out, lse = torch.zeros_like(q), torch.zeros((2, 2), device="cuda")
        pool.cache.attention(pool.batch([2], [70]), q, out, 0.125 / f, lse=lse)
        check_attention(pool, q, out, lse, [(68, 2)], 0.125 / f, 0, True, "bf16")


def test_a_layer_of_a_shared_pool(pkg):
    """Pages that hold several layers: one descriptor for each, the others' bytes untouched."""
    pool = Pool(pkg, [40, 17], 2, 64, seed=5, layers=3, layer=1)
    before = pool.pool.clone()
    x = [torch.randn((57, 2, 64), device="cuda") for _ in range(2)]
    pool.cache.append(pool.batch([40, 17], [40, 17]), None, *x, None)
    assert torch.equal(pool.pool[:, 0], before[:, 0]) and torch.equal(pool.pool[:, 2], before[:, 2])
    k = torch.empty((57, 2, 64), device="cuda")
    v = torch.empty_like(k)
    pool.cache.read(pool.batch([40, 17], [40, 17]), k, v)
    assert (k - x[0]).abs().max() < 0.3 and (v - x[1]).abs().max() < 0.3


def test_offsets_past_32_bits(pkg):
    """Pages beyond 4 GiB of a pool: the same results as in its first pages."""
    hd, KV, page = 128, 8, 256
    n_pages = (5 << 30) // (2 * KV * page * hd)
    pages = torch.empty((n_pages, 2, KV, page, hd), dtype=torch.uint8, device="cuda")
    scales = torch.empty((n_pages, 2, KV, page // 16), device="cuda")
    x = [torch.randn((300, h, hd), device="cuda") for h in (16, KV, KV)]
    got = []
    for ids in ([0, 1], [n_pages - 1, n_pages - 2]):
        cache = pkg.KV8Cache(pages, scales, torch.tensor([ids], dtype=torch.int32, device="cuda"))
        batch = pkg.KV8Batch(torch.tensor([0, 300], dtype=torch.int32, device="cuda"),
                             torch.tensor([300], dtype=torch.int32, device="cuda"), 300, 300, 300)
        q = torch.empty((300, 16, hd), dtype=torch.float16, device="cuda")
        cache.append(batch, *x, q)
        one = pkg.KV8Batch(torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                           torch.tensor([300], dtype=torch.int32, device="cuda"), 1, 1, 300)
        out, few, k, v = torch.empty_like(q), torch.empty_like(q[:1]), torch.empty_like(x[1]), torch.empty_like(x[1])
        cache.attention(batch, q, out, 0.09)
        cache.attention(one, q[299:], few, 0.09)
        cache.read(batch, k, v)
        cache.check()
        got.append((out, few, k, v))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_repeats_streams_and_graphs_give_the_same_bits(pkg):
    """Split ranges are joined in order: the same bits every time, on another stream, and replayed."""
    pool = Pool(pkg, [2500, 900, 40], 2, 64, seed=7, fill=[2500, 900, 40])
    q = torch.randn((3, 8, 64), device="cuda").half()
    batch, outs = pool.batch([1, 1, 1], [2500, 900, 40]), []
    for _ in range(20):
        o = torch.zeros_like(q)
        pool.cache.attention(batch, q, o, 0.125)
        outs.append(o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = torch.zeros_like(q)
        for _ in range(3):
            pool.cache.attention(batch, q, o, 0.125)
        outs.append(o)
    side.synchronize()
    o = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        pool.cache.attention(batch, q, o, 0.125)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            pool.cache.attention(batch, q, o, 0.125)
    o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    outs.append(o)
    assert all(torch.equal(outs[0], x) for x in outs[1:])


def test_device_side_errors_are_reported_and_the_rest_computed(pkg):
    """A page id, a slot or a length out of range is skipped and shows in the status; other sequences are right."""
    lens = [40, 40, 40]
    for what in ("page", "slot", "length", "rows"):
        pool = Pool(pkg, lens, 2, 64, seed=11, fill=lens)
        good = pool.batch([1, 1, 1], lens)
        q = torch.randn((3, 4, 64), device="cuda").half()
        want, got = torch.zeros_like(q), torch.zeros_like(q)
        pool.cache.attention(good, q, want, 0.125)
        pool.cache.check()
        bad = pool.batch([1, 1, 1], lens)
        if what == "page":
            pool.table[int(pool.slots_np[1]), 2] = 1 << 20
        elif what == "slot":
            bad._held[2][1] = -1
        elif what == "length":
            bad._held[1][1] = 41
        else:
            bad._held[0].copy_(torch.tensor([0, 1, 1 << 30, 3], dtype=torch.int32))
        pool.cache.attention(bad, q, got, 0.125)
        with pytest.raises(RuntimeError, match="out of range"):
            pool.cache.check()
        pool.cache.check()
        assert torch.equal(got[0], want[0]), what
        if what != "rows":
            assert torch.equal(got[2], want[2]), what
        before = pool.pages.clone()
        k = torch.randn((3, 2, 64), device="cuda")
        pool.cache.append(bad, None, k, k.clone(), None)
        pool.cache.read(bad, torch.empty_like(k), torch.empty_like(k))
        with pytest.raises(RuntimeError, match="out of range"):
            pool.cache.check()
        others = [p for p in range(before.shape[0]) if p not in pool.table_np[pool.slots_np[[0, 2]]]]
        assert torch.equal(pool.pages[others], before[others])


def test_refusals(pkg):
    pool = Pool(pkg, [20], 2, 64, fill=[20])
    b = pool.batch([2], [20])
    q, o = torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda"), torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda")
    k = torch.zeros((2, 2, 64), dtype=torch.float16, device="cuda")
    att, app = pool.cache.attention, pool.cache.append
    with pytest.raises(ValueError, match="q"):
        att(b, q[:1], o, 1.0)
    with pytest.raises(ValueError, match="contiguous heads"):
        att(b, q.transpose(1, 2).contiguous().transpose(1, 2), o, 1.0)
    with pytest.raises(RuntimeError, match="type"):
        att(b, q.float(), o.float(), 1.0)
    with pytest.raises(RuntimeError, match="one type"):
        att(b, q, o.bfloat16(), 1.0)
    with pytest.raises(RuntimeError, match="multiple of n_kv"):
        att(b, q[:, :3], o[:, :3], 1.0)
    with pytest.raises(RuntimeError, match="window"):
        att(b, q, o, 1.0, causal=False, window=4)
    with pytest.raises(RuntimeError, match="window"):
        att(b, q, o, 1.0, window=-1)
    with pytest.raises(RuntimeError, match="overlap"):
        att(b, q, o[:1].expand(2, 4, 64), 1.0)
    with pytest.raises(RuntimeError, match="max_len"):
        att(pool.batch([2], [20], max_len=1000), q, o, 1.0)
    with pytest.raises(RuntimeError, match="one type"):
        app(b, q, k, k.float(), o)
    with pytest.raises(RuntimeError, match="together"):
        app(b, q, k, k, None)
    with pytest.raises(RuntimeError, match="f16 or bf16"):
        app(b, q, k, k, o.float())
    with pytest.raises(RuntimeError, match="rope"):
        app(b, q, k, k, o, rope=torch.zeros((19, 32, 2), device="cuda"))
    with pytest.raises(ValueError, match="rope"):
        app(b, q, k, k, o, rope=torch.zeros((20, 64), device="cuda"))
    with pytest.raises(RuntimeError, match="heads"):
        app(b, q, k[:, :1], k, o)
    with pytest.raises(ValueError, match="q_norm"):
        app(b, q, k, k, o, q_norm=torch.ones(32, device="cuda"))
    with pytest.raises(RuntimeError, match="head_dim"):
        pages = torch.zeros((2, 2, 2, 16, 96), dtype=torch.uint8, device="cuda")
        c = pkg.KV8Cache(pages, torch.ones((2, 2, 2, 1), device="cuda"), pool.table)
        c.read(b, k[..., :1].expand(2, 2, 96).contiguous(), k[..., :1].expand(2, 2, 96).contiguous())
    with pytest.raises(ValueError, match="pages"):
        pkg.KV8Cache(pool.pages.int(), pool.scales, pool.table)
