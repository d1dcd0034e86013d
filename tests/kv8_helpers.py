"""A plain 64-bit restatement of the 8-bit paged cache and a small pool of sequences to test it with."""
import numpy as np
import torch

E_MIN, E_MAX = -24, 40
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half the spacing of a type's numbers, relative to them
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def e4m3_table():
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    x = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7.0), m / 8 * 2.0 ** -6)
    return np.where((b & 127) == 127, np.nan, x) * np.where(b >> 7, -1.0, 1.0)


def round_e4m3(x):
    """float64 -> the nearest e4m3 (ties to even), saturating; NaN stays."""
    x = np.asarray(x, np.float64)
    _, e = np.frexp(np.where(np.isfinite(x), x, 0.0))
    step = np.exp2(np.maximum(e - 4, -9))
    return np.clip(np.rint(x / step) * step, -448, 448)


def exponent(top):
    if top == 0:
        return E_MIN
    m, e = np.frexp(top / 448.0)
    return int(np.clip(e - (m == 0.5), E_MIN, E_MAX))


class Pool:
    """A cache of a few sequences on the GPU, the pages of each in any order, with bytes that are NaN
    wherever nothing was written."""

    def __init__(self, pkg, lens, n_kv, hd, page=16, seed=0, fill=None, layers=1, layer=0):
        self.rng = np.random.default_rng(seed)
        self.n_kv, self.hd, self.page = n_kv, hd, page
        self.cap = [max(1, -(-n // page)) for n in lens]
        n_pages = sum(self.cap) + 3
        order = self.rng.permutation(n_pages)
        self.table_np = np.zeros((len(lens) + 2, max(self.cap) + 1), np.int32)
        self.slots_np = self.rng.permutation(len(lens) + 2)[: len(lens)].astype(np.int32)
        at = 0
        for b, n in enumerate(self.cap):
            self.table_np[self.slots_np[b], :n] = order[at: at + n]
            at += n
        self.spare = order[at:]
        pool = torch.full((n_pages, layers, 2, n_kv, page, hd), 0xFF, dtype=torch.uint8, device="cuda")
        scales = torch.full((n_pages, layers, 2, n_kv, page // 16), 2.0 ** 30, device="cuda")
        self.pool, self.all_scales = pool, scales
        self.pages, self.scales = pool[:, layer], scales[:, layer]
        self.table = torch.from_numpy(self.table_np).cuda()
        self.slots = torch.from_numpy(self.slots_np).cuda()
        self.cache = pkg.KV8Cache(self.pages, self.scales, self.table)
        self.pkg = pkg
        # what the cache should hold: per sequence, bytes as values [K, V] and exponents of each block
        self.values = [np.zeros((2, 0, n_kv, hd)) for _ in lens]
        self.exps = [np.zeros((2, 0, n_kv), np.int64) for _ in lens]
        if fill is not None:
            self.fill(fill)

    def fill(self, lens, spread=1.0):
        """Sets the sequences' content directly: random bytes without NaN and scales."""
        t = e4m3_table()
        pages, scales = self.pages.cpu().numpy(), self.scales.cpu().numpy()
        for b, n in enumerate(lens):
            blocks = -(-n // 16)
            x = self.rng.standard_normal((2, blocks * 16, self.n_kv, self.hd)) * 90
            # magnitudes as they come out of an append: up to 448, in units of the block's scale
            vals = round_e4m3(np.clip(x, -448, 448))
            e = self.rng.integers(-9, -6, (2, blocks, self.n_kv)) if spread == 1.0 else self.rng.integers(*spread, (2, blocks, self.n_kv))
            vals[:, n:] = np.nan
            self.values[b], self.exps[b] = vals[:, :n].copy(), e
            order = np.argsort(t[:128], kind="stable")
            mag = np.abs(np.nan_to_num(vals))
            code = order[np.searchsorted(t[:128][order][:127], mag)].astype(np.uint8) | (np.signbit(vals) * 128).astype(np.uint8)
            code[np.isnan(vals)] = 0x7F
            for blk in range(blocks):
                pg, off = self.table_np[self.slots_np[b], blk * 16 // self.page], blk * 16 % self.page
                for h in range(self.n_kv):
                    pages[pg, 0, h, off: off + 16] = code[0, blk * 16: blk * 16 + 16, h]
                    v = code[1, blk * 16: blk * 16 + 16, h].reshape(4, 4, self.hd // 4, 4)
                    pages[pg, 1, h, off: off + 16] = v.transpose(2, 0, 3, 1).reshape(16, self.hd)
                    scales[pg, :, h, off // 16] = np.exp2(e[:, blk, h])
        self.pages.copy_(torch.from_numpy(pages))
        self.scales.copy_(torch.from_numpy(scales))

    def batch(self, new, lens, max_new=None, max_len=None):
        q_start = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
        return self.pkg.KV8Batch(q_start, torch.tensor(lens, dtype=torch.int32, device="cuda"), int(sum(new)),
                                 max(new) if max_new is None else max_new, max(lens) if max_len is None else max_len, self.slots)

    def held(self, b, n):
        """(bytes as values [2][n][kv][hd], exponents [2][blocks][kv]) of sequence b's first n positions in the device's pages."""
        t = e4m3_table()
        pages, scales = self.pages.cpu().numpy(), self.scales.cpu().numpy()
        blocks = -(-n // 16)
        out, e = np.zeros((2, blocks * 16, self.n_kv, self.hd)), np.zeros((2, blocks, self.n_kv), np.int64)
        for blk in range(blocks):
            pg, off = self.table_np[self.slots_np[b], blk * 16 // self.page], blk * 16 % self.page
            for h in range(self.n_kv):
                out[0, blk * 16: blk * 16 + 16, h] = t[pages[pg, 0, h, off: off + 16]]
                v = t[pages[pg, 1, h, off: off + 16]].reshape(self.hd // 4, 4, 4, 4).transpose(1, 3, 0, 2)
                out[1, blk * 16: blk * 16 + 16, h] = v.reshape(16, self.hd)
                s = scales[pg, :, h, off // 16]
                e[:, blk, h] = np.log2(s).round()
                assert np.array_equal(np.exp2(e[:, blk, h]), s)
        return out[:, :n], e, out[:, n:]

    def dequantised(self, b, n):
        """Keys and values [2][n][kv][hd] that the expected content stands for."""
        v, e = self.values[b][:, :n], self.exps[b]
        return v * np.repeat(np.exp2(e.astype(np.float64)), 16, 1)[:, : v.shape[1], :, None]


def turned(x, w, eps, cs):
    """norm and rotation of rows [n][heads][hd] in float64; cs [n][hd / 2][2] or None."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    if cs is None:
        return x
    h = x.shape[-1] // 2
    c, s = cs[:, None, :, 0].astype(np.float64), cs[:, None, :, 1].astype(np.float64)
    return np.concatenate([x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c], -1)


def attend(q, k, v, scale, first, causal, window):
    """out, lse, sum p|v|, the scores' magnitude bound of rows q [n][heads][hd] at positions first, first + 1, ...
    over keys k, values v [len][kv][hd]; NaN propagates only from keys that a row sees."""
    n, H, hd = q.shape
    L, KV = k.shape[:2]
    out, lse = np.zeros((n, H, hd)), np.full((n, H), -np.inf)
    mag, sc = np.zeros((n, H, hd)), np.zeros((n, H))
    for i in range(n):
        p = first + i
        lo, hi = (max(0, p - window + 1) if window else 0), (p + 1 if causal else L)
        if p < 0 or hi <= lo:
            continue
        for h in range(H):
            kk, vv = k[lo:hi, h * KV // H], v[lo:hi, h * KV // H]
            s = scale * (kk @ q[i, h])
            m = s.max()
            e = np.exp(s - m)
            out[i, h] = e @ vv / e.sum()
            lse[i, h] = m + np.log(e.sum())
            mag[i, h] = e @ np.abs(vv) / e.sum()
            sc[i, h] = abs(scale) * (np.abs(kk) @ np.abs(q[i, h])).max()
    return out, lse, mag, sc
