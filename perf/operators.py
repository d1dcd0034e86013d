"""What is measured of the 8-bit paged key/value cache: appending to it, reading it back, attention over it.

Each case is one call on buffers that a serving loop has in hand. `run` computes it in elementary torch
operations in 32 bits, or with the library's own kernels where `own` is true; `exact` restates each operator
in 64 bits.

The cache: a page of `page` positions is [K|V][kv head][position][head_dim] bytes of e4m3, with one f32 scale
(a power of two 2^e) for each block of 16 positions and head. Keys of a block are rows of head_dim bytes;
values of a block are 4 x 4 patches [head_dim / 4][4 position groups][4 of head_dim][4 positions]. e is the
smallest integer with 448 2^e >= the block's largest finite magnitude, clamped to [-24, 40].
"""
import math

import numpy as np
import torch

own = False

BLOCK = 16
E_MIN, E_MAX = -24, 40
EPS = 1e-6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def _case(name, op, n_seq, new_lo, new_hi, old_lo, old_hi, heads, kv, hd, dtype, page=16, window=0, causal=True, lse=False):
    c = dict(op=op, n_seq=n_seq, new_lo=new_lo, new_hi=new_hi, old_lo=old_lo, old_hi=old_hi, heads=heads, kv=kv,
             hd=hd, dtype=dtype, page=page, window=window, causal=causal, lse=lse)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one session's frame step: the new position's q/k/v row as the projection leaves it (f32)
        _case("append_step_1", "append", 1, 1, 1, 217, 217, 32, 8, 64, "f32"),
        # a full serving step: 64 sessions at contexts from just created to nearly full
        _case("append_step_64", "append", 64, 1, 1, 90, 2030, 32, 8, 64, "f32"),
        # prompts that arrived together, packed, each into its own fresh pages
        _case("append_prompts", "append", 24, 17, 301, 0, 0, 32, 8, 64, "f16"),
        # long inputs that continue sessions in the middle of a block, larger heads and pages
        _case("append_long", "append", 4, 4096, 4096, 1003, 1003, 32, 8, 128, "bf16", page=64),
        # a reference voice's positions taken out of the cache to be kept on the host
        _case("read_voice", "read", 1, 151, 151, 0, 0, 32, 8, 64, "f16"),
        # many sessions moved to another server: their whole contexts in 16 bits
        _case("read_sessions", "read", 16, 700, 4096, 0, 0, 32, 8, 128, "bf16", page=64),
        # one session's frame step: latency of a single short row
        _case("attend_step_1", "attend", 1, 1, 1, 217, 217, 32, 8, 64, "f16"),
        # a full serving step over ragged contexts
        _case("attend_step_64", "attend", 64, 1, 1, 90, 2030, 32, 8, 64, "f16"),
        # few sessions with very long contexts: the cache's bytes are the time
        _case("attend_step_long", "attend", 8, 1, 1, 32001, 32767, 32, 8, 128, "bf16", page=64, lse=True),
        # several guessed tokens of each session checked at once, sliding window, odd group of heads
        _case("attend_guesses", "attend", 16, 5, 5, 200, 4000, 28, 4, 128, "bf16", window=1000, lse=True),
        # prompts that arrived together
        _case("attend_prompts", "attend", 24, 17, 301, 0, 0, 32, 8, 64, "f16"),
        # a long document read in one piece behind a cached one
        _case("attend_long", "attend", 1, 8192, 8192, 4100, 4100, 32, 8, 128, "bf16", page=64),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "attend", "attend", "attend"])
    hd = rng.choice([64, 128])
    heads, kv = rng.choice([(32, 8), (28, 4), (8, 8), (16, 2), (12, 4), (5, 1), (40, 8), (8, 2)])
    dtype = rng.choice(["f16", "bf16"] if op == "attend" else ["f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "attend":
        kind = rng.choice(["step", "guesses", "prompts", "long"])
    else:
        kind = rng.choice(["step", "prompts", "long"])
    if kind == "step":
        n_seq, new, old = _spread(rng, 1, 200), 1, _spread(rng, 30, 8000)
        if n_seq < 12:
            old = _spread(rng, 30, 32000)
        old = min(old, 600_000 // n_seq)
        c = (n_seq, 1, 1, max(1, old // rng.choice([1, 2, 9])), old)
    elif kind == "guesses":
        new, old = rng.randint(2, 9), _spread(rng, 30, 6000)
        c = (_spread(rng, 1, 64), new, new, max(1, old // rng.choice([1, 3])), old)
    elif kind == "prompts":
        new = _spread(rng, 20, 700)
        old = rng.choice([0, 0, _spread(rng, 5, 900)])
        c = (_spread(rng, 2, 30), max(1, new // rng.choice([1, 2, 10])), new, old, old)
    else:
        new = _spread(rng, 900, 3500)
        c = (rng.randint(1, 2), new, new, 0, _spread(rng, 1, 2000))
    window = rng.choice([0, 0, 0, _spread(rng, 20, 2000)]) if op == "attend" else 0
    causal = op != "attend" or bool(window) or rng.random() < 0.85
    lse = op == "attend" and rng.random() < 0.4
    return _case(None, op, *c, heads, kv, hd, dtype, page, window, causal, lse)


def _lengths(case):
    """(new, total) positions of each sequence: spread evenly over the case's ranges, in a fixed shuffled order."""
    n = case["n_seq"]
    at = np.random.RandomState(n).permutation(n)
    f = at / max(1, n - 1)
    new = np.rint(case["new_lo"] + f * (case["new_hi"] - case["new_lo"])).astype(np.int64)
    old = np.rint(case["old_lo"] + f[::-1] * (case["old_hi"] - case["old_lo"])).astype(np.int64)
    return new, old + new


def _pairs(case):
    """(query, key) pairs that attention looks at, over one query head."""
    new, total = _lengths(case)
    pairs = 0
    for n, t in zip(new.tolist(), total.tolist()):
        if not case["causal"]:
            pairs += n * t
            continue
        seen = np.arange(t - n, t) + 1
        if case["window"]:
            seen = np.minimum(seen, case["window"])
        pairs += int(seen.sum())
    return pairs


def work(case):
    new, total = _lengths(case)
    T, H, KV, hd = int(new.sum()), case["heads"], case["kv"], case["hd"]
    size = 4 if case["dtype"] == "f32" else 2
    cached = 2 * KV * (hd + 4.0 / BLOCK)  # bytes of a position's keys and values with their scales
    back = int((new + (total - new) % BLOCK).sum())  # positions of the blocks that an append touches
    if case["op"] == "append":
        table = int(new.max()) * hd * 4
        rows = T * (H + 2 * KV) * hd
        old = back - T
        return {"bytes": rows * size + table + T * H * hd * 2 + (back + old) * cached + back * 2 * KV * hd * 2,
                "flops": T * (H + KV) * hd * 8}
    if case["op"] == "read":
        return {"bytes": T * cached + T * 2 * KV * hd * size, "flops": 0}
    keys = 0  # cached positions that any query of a sequence may look at
    for n, t in zip(new.tolist(), total.tolist()):
        keys += min(t, case["window"] + n - 1) if case["window"] else t
    return {"bytes": keys * cached + 2 * T * H * hd * size + (T * H * 4 if case["lse"] else 0),
            "flops": 4.0 * hd * H * _pairs(case)}


# ---------------------------------------------------------------- inputs

def _rope_table(n, hd):
    inv = 500000.0 ** (-np.arange(0, hd, 2) / hd)
    a = np.arange(n)[:, None] * inv[None, :]
    return torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)).cuda()


def prepare(case, seed):
    new, total = _lengths(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 31))
    n, H, KV, hd, page = case["n_seq"], case["heads"], case["kv"], case["hd"], case["page"]
    dt = DTYPES[case["dtype"]]
    T, max_new, max_len = int(new.sum()), int(new.max()), int(total.max())
    # each sequence holds pages of a shared pool in any order; its table row is one of a few more slots
    pages_of = -(-total // page)
    max_pages, n_slots, n_pages = int(pages_of.max()), n + 3, int(pages_of.sum()) + 5
    slots = r.permutation(n_slots)[:n]
    order, table, at = r.permutation(n_pages), np.zeros((n_slots, max_pages), np.int64), 0
    for b in range(n):
        table[slots[b], : pages_of[b]] = order[at: at + pages_of[b]]
        at += pages_of[b]
    q_start = np.concatenate([[0], np.cumsum(new)])
    ints = lambda v: torch.from_numpy(np.ascontiguousarray(v, dtype=np.int32)).cuda()  # noqa: E731
    # the pool's content: normal keys and values, a few channels of the keys several times the others
    e_k, e_v = (torch.randint(e, e + 2, (n_pages, 1, KV, page // BLOCK), device="cuda", generator=g) for e in (-5, -7))
    scales = torch.exp2(torch.cat([e_k, e_v], 1).float())
    loud = 1 + 3 * (torch.rand(hd, device="cuda", generator=g) < 0.05)
    pages = torch.empty((n_pages, 2, KV, page, hd), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (2 * KV * page * hd))
    for i in range(0, n_pages, step):
        x = torch.randn((min(step, n_pages - i), 2, KV, page // BLOCK, BLOCK, hd), device="cuda", generator=g)
        x[:, 0] *= loud
        x = (x / scales[i: i + step, :, :, :, None, None]).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        v = x[:, 1].view(-1, KV, page // BLOCK, 4, 4, hd // 4, 4).permute(0, 1, 2, 5, 3, 6, 4)
        pages[i: i + step, 0] = x[:, 0].reshape(-1, KV, page, hd)
        pages[i: i + step, 1] = v.reshape(-1, KV, page, hd)
    st = dict(case=case, pages=pages, scales=scales, table=ints(table), slots=ints(slots), q_start=ints(q_start),
              kv_len=ints(total), T=T, max_new=max_new, max_len=max_len)
    if case["op"] == "append":
        # q, k and v are column ranges of the fused projection's output rows
        qkv = torch.randn((T, (H + 2 * KV) * hd), device="cuda", generator=g).to(dt)
        st["q"] = qkv[:, : H * hd].unflatten(1, (H, hd))
        st["k"] = qkv[:, H * hd: (H + KV) * hd].unflatten(1, (KV, hd))
        st["v"] = qkv[:, (H + KV) * hd:].unflatten(1, (KV, hd))
        st["wq"], st["wk"] = (1 + 0.2 * torch.randn(hd, device="cuda", generator=g) for _ in range(2))
        st["wk"] = st["wk"] * loud
        st["rope"] = _rope_table(max_len, hd)
        st["q_out"] = torch.empty((T, H, hd), dtype=torch.float16 if dt == torch.float32 else dt, device="cuda")
        # the whole of every touched block is read back: what was there before the new positions too
        back = new + (total - new) % BLOCK
        st["back_start"], st["T_back"], st["max_back"] = ints(np.concatenate([[0], np.cumsum(back)])), int(back.sum()), int(back.max())
    if case["op"] == "attend":
        st["q"] = (torch.randn((T, H, hd), device="cuda", generator=g) * 1.3).to(dt)
        st["out"] = torch.empty((T, H, hd), dtype=dt, device="cuda")
        st["lse"] = torch.empty((T, H), device="cuda") if case["lse"] else None
    else:
        rows = st.get("T_back", T)
        kind = torch.float16 if case["op"] == "append" and dt == torch.float32 else dt
        st["k_out"], st["v_out"] = (torch.empty((rows, KV, hd), dtype=kind, device="cuda") for _ in range(2))
    if own:  # the handles that a program keeps beside its buffers
        import __graft_entry__ as entry
        lib = entry.load_package()
        st["cache"] = lib.KV8Cache(pages, scales, st["table"])
        st["batch"] = lib.KV8Batch(st["q_start"], st["kv_len"], T, max_new, max_len, st["slots"])
        if case["op"] == "append":
            st["back"] = lib.KV8Batch(st["back_start"], st["kv_len"], st["T_back"], st["max_back"], max_len, st["slots"])
    return st


# ---------------------------------------------------------------- the plain forms

def _grid(start, kv_len, n_grid):
    """Rows and positions of each sequence padded to n_grid: (row, position, whether there is one)."""
    start = start.long()
    n = start[1:] - start[:-1]
    t = torch.arange(n_grid, device=start.device)[None, :]
    pos = (kv_len.long() - n)[:, None] + t
    return start[:-1, None] + t, pos, (t < n[:, None]) & (pos >= 0)


def _place(st, pos):
    """(page, position in it) of positions [n_seq, m]; those outside a sequence's table row read page entry 0."""
    page = st["case"]["page"]
    table = st["table"].long()[st["slots"].long()]
    entry = (pos.clamp(min=0) // page).clamp(max=table.shape[1] - 1)
    return table.gather(1, entry), pos.clamp(min=0) % page


def _values_index(hd, device):
    """Byte of (position in block, element) within a block of values."""
    p, d = torch.arange(BLOCK, device=device)[:, None], torch.arange(hd, device=device)[None, :]
    return (d // 4) * 64 + (p // 4) * 16 + (d % 4) * 4 + p % 4


def _cached(st, pos):
    """Keys, values [n_seq, m, kv, hd] in f32 and the scales' exponents of both, at positions [n_seq, m]."""
    hd, KV = st["case"]["hd"], st["case"]["kv"]
    pg, at = _place(st, pos)
    pages, scales = st["pages"], st["scales"]
    heads = torch.arange(KV, device=pos.device)
    k = pages[:, 0][pg[..., None], heads, at[..., None]]
    blocks = pages[:, 1].reshape(pages.shape[0], KV, -1, BLOCK * hd)
    where = _values_index(hd, pos.device)[at % BLOCK]
    v = blocks[pg[..., None, None], heads[:, None], (at // BLOCK)[..., None, None], where[:, :, None, :]]
    sk = scales[:, 0][pg[..., None], heads, (at // BLOCK)[..., None]]
    sv = scales[:, 1][pg[..., None], heads, (at // BLOCK)[..., None]]
    f = lambda x, s: x.view(torch.float8_e4m3fn).float() * s[..., None]  # noqa: E731
    return f(k, sk), f(v, sv), sk, sv


def _norm_rotate(x, w, cs):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a, b = x.chunk(2, -1)
    c, s = cs[..., 0], cs[..., 1]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _exponent(amax):
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, e - 9 + (m > 0.875), E_MIN).clamp(E_MIN, E_MAX)


def _append_plain(st):
    hd, KV = st["case"]["hd"], st["case"]["kv"]
    start, kv_len = st["q_start"].long(), st["kv_len"].long()
    n = start[1:] - start[:-1]
    # positions of the packed rows
    row = torch.arange(st["T"], device=start.device)
    seq = torch.searchsorted(start[1:], row, right=True)
    pos = kv_len[seq] - n[seq] + row - start[seq]
    cs = st["rope"][pos][:, None]
    q = _norm_rotate(st["q"], st["wq"], cs)
    k = _norm_rotate(st["k"], st["wk"], cs)
    st["q_out"].copy_(q)
    # every touched block of 16 positions: older ones from the cache, new ones, zeros behind the end
    first = (kv_len - n) // BLOCK * BLOCK
    m = (st["max_new"] + 2 * BLOCK - 2) // BLOCK * BLOCK
    P = first[:, None] + torch.arange(m, device=start.device)[None, :]
    fresh = (P >= (kv_len - n)[:, None]) & (P < kv_len[:, None])
    older = P < (kv_len - n)[:, None]
    src = (start[:-1, None] + P - (kv_len - n)[:, None]).clamp(0, st["T"] - 1)
    ok, ov, sk, sv = _cached(st, P)
    live = (P < kv_len[:, None]).unflatten(1, (-1, BLOCK))[:, :, 0]
    pg, at = _place(st, P)
    pg, blk = pg[:, ::BLOCK][live], (at[:, ::BLOCK] // BLOCK)[live]
    out = []
    for x, o, s in ((k[src], ok, sk), (st["v"].float()[src], ov, sv)):
        new = torch.where(fresh[..., None, None], x, 0.0)
        new = torch.where(new.isfinite(), new, torch.nan).unflatten(1, (-1, BLOCK))
        e = _exponent(torch.nan_to_num(new, 0.0).abs().amax((2, 4)))
        e_old = torch.log2(s[:, ::BLOCK]).round().int()
        e = torch.where(older[:, ::BLOCK, None], torch.maximum(e, e_old), e)
        o = torch.where(older[..., None, None], o, 0.0).unflatten(1, (-1, BLOCK))
        scale = torch.exp2(e.float())
        q8 = ((new + o) / scale[:, :, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        out.append((q8[live].transpose(1, 2), scale[live]))
    heads = torch.arange(KV, device=start.device)[None, :]
    index = (pg[:, None], heads, blk[:, None])
    # (views of the state's own buffers: the pool is updated in place)
    pool = st["pages"].view(st["pages"].shape[0], 2, KV, -1, BLOCK * hd)
    pool[:, 0][index] = out[0][0].flatten(2)
    pool[:, 1][index] = out[1][0].unflatten(-1, (hd // 4, 4)).unflatten(2, (4, 4)).permute(0, 1, 4, 2, 5, 3).flatten(2)
    st["scales"][:, 0][index] = out[0][1]
    st["scales"][:, 1][index] = out[1][1]
    return _read_plain(st, st["back_start"], st["max_back"])


def _read_plain(st, start, most):
    row, pos, there = _grid(start, st["kv_len"], most)
    k, v, _, _ = _cached(st, pos)
    st["k_out"][row[there]] = k[there].to(st["k_out"].dtype)
    st["v_out"][row[there]] = v[there].to(st["v_out"].dtype)


def _attend_plain(st):
    c = st["case"]
    H, KV, hd = c["heads"], c["kv"], c["hd"]
    row, pos, there = _grid(st["q_start"], st["kv_len"], st["max_new"])
    key = torch.arange(st["max_len"], device=row.device)[None, :].expand(c["n_seq"], -1)
    k, v, _, _ = _cached(st, key)
    v = torch.where((key < st["kv_len"].long()[:, None])[..., None, None], v, 0.0)
    q = st["q"].float()[row.clamp(max=st["T"] - 1)].unflatten(2, (KV, H // KV))
    s = torch.matmul(q.permute(0, 2, 3, 1, 4), k.permute(0, 2, 3, 1)[:, :, None]).mul_(hd ** -0.5)
    sees = (key < st["kv_len"].long()[:, None])[:, None, :].expand(-1, st["max_new"], -1)
    if c["causal"]:
        sees = sees & (key[:, None, :] <= pos[:, :, None])
    if c["window"]:
        sees = sees & (key[:, None, :] > pos[:, :, None] - c["window"])
    s.masked_fill_(~sees[:, None, None], -torch.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s, v.transpose(1, 2)[:, :, None])
    o = torch.where(total > 0, o / total, 0.0)
    st["out"][row[there]] = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[there].to(st["out"].dtype)
    if c["lse"]:
        st["lse"][row[there]] = (top + total.log())[..., 0].permute(0, 3, 1, 2).flatten(2)[there]


# ---------------------------------------------------------------- one pass

def run(st):
    op = st["case"]["op"]
    if op == "append":
        if own:
            st["cache"].append(st["batch"], st["q"], st["k"], st["v"], st["q_out"], q_norm=st["wq"], k_norm=st["wk"], eps=EPS, rope=st["rope"])
            st["cache"].read(st["back"], st["k_out"], st["v_out"])
        else:
            _append_plain(st)
        return {"q": st["q_out"], "k": st["k_out"], "v": st["v_out"]}
    if op == "read":
        if own:
            st["cache"].read(st["batch"], st["k_out"], st["v_out"])
        else:
            _read_plain(st, st["q_start"], st["max_new"])
        return {"k": st["k_out"], "v": st["v_out"]}
    if own:
        st["cache"].attention(st["batch"], st["q"], st["out"], scale=st["case"]["hd"] ** -0.5, causal=st["case"]["causal"],
                              window=st["case"]["window"], lse=st["lse"])
    else:
        _attend_plain(st)
    return {"out": st["out"], "lse": st["lse"]} if st["case"]["lse"] else {"out": st["out"]}


# ---------------------------------------------------------------- the definition in 64 bits

def _e4m3_values():
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    x = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m / 8.0 * 2.0 ** -6)
    return torch.from_numpy(np.where((b & 127) == 127, np.nan, x) * np.where(b >> 7, -1.0, 1.0)).cuda()


def _power(e):
    """2^e in 64 bits from whole exponents, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _to_e4m3(x):
    """64-bit values of magnitude <= 448 rounded to the nearest e4m3, ties to even."""
    _, e = torch.frexp(x)
    step = _power((e - 4).clamp(min=-9))
    return (x / step).round() * step


def _sequence(st, b, values, n):
    """Keys and values [n, kv, hd] and their scales [n, kv] of sequence b's first n positions, in 64 bits."""
    c = st["case"]
    pages = st["table"][int(st["slots"][b])].long()[: -(-n // c["page"])]
    raw, sc = st["pages"][pages], st["scales"][pages].double()
    k = raw[:, 0].permute(0, 2, 1, 3)
    v = raw[:, 1].reshape(len(pages), c["kv"], c["page"] // BLOCK, c["hd"] // 4, 4, 4, 4)
    v = v.permute(0, 2, 4, 6, 1, 3, 5)
    k, v = (values[x.reshape(-1, c["kv"], c["hd"])[:n].long()] for x in (k, v))
    sk, sv = (sc[:, i].repeat_interleave(BLOCK, 2).permute(0, 2, 1).reshape(-1, c["kv"])[:n] for i in (0, 1))
    return k * sk[..., None], v * sv[..., None], sk, sv


def _turned(x, w, first, hd):
    x = x.double()
    x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    # the table's own 32-bit numbers are the operator's input
    t = first["rope"][first["at"]].double()[:, None]
    lo, hi = x[..., : hd // 2], x[..., hd // 2:]
    return torch.cat([lo * t[..., 0] - hi * t[..., 1], hi * t[..., 0] + lo * t[..., 1]], -1)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    new, total = _lengths(case)
    hd, H, KV, values = case["hd"], case["heads"], case["kv"], _e4m3_values()
    q_all, k_all, v_all, l_all, at = [], [], [], [], 0
    for b, (n, t) in enumerate(zip(new.tolist(), total.tolist())):
        rows = slice(at, at + n)
        at += n
        if case["op"] == "read":
            k, v, _, _ = _sequence(st, b, values, t)
            k_all.append(k[t - n:])
            v_all.append(v[t - n:])
        elif case["op"] == "append":
            old = t - n
            turn = {"rope": st["rope"], "at": torch.arange(old, t, device="cuda")}
            q_all.append(_turned(st["q"][rows], st["wq"], turn, hd))
            fresh = (_turned(st["k"][rows], st["wk"], turn, hd), st["v"][rows].double())
            kept = _sequence(st, b, values, old) if old else None
            head = old % BLOCK
            for i, (x, to) in enumerate(zip(fresh, (k_all, v_all))):
                x = torch.cat([kept[i][old - head:], x]) if head else x
                pad = torch.cat([x, x.new_zeros((-len(x) % BLOCK, KV, hd))]).view(-1, BLOCK, KV, hd)
                news = pad.clone()
                news[0, :head] = 0
                top = news.abs().amax((1, 3))
                m, e = torch.frexp(top / 448)  # the next power of two at or above top / 448
                e = torch.where(top > 0, e - (m == 0.5).int(), E_MIN).clamp(E_MIN, E_MAX)
                if head:
                    e[0] = torch.maximum(e[0], torch.frexp(kept[2 + i][old - 1])[1] - 1)
                s = _power(e)[:, None, :, None]
                to.append((_to_e4m3(pad / s) * s).view(-1, KV, hd)[: len(x)])
        else:
            k, v, _, _ = _sequence(st, b, values, t)
            q = st["q"][rows].double().view(n, KV, H // KV, hd)
            o, lse = torch.zeros((n, H, hd), device="cuda", dtype=torch.float64), torch.zeros((n, H), device="cuda", dtype=torch.float64)
            key = torch.arange(t, device="cuda")[None, :]
            for i in range(0, n, 1024):
                mine = torch.arange(t - n + i, min(t, t - n + i + 1024), device="cuda")[:, None]
                sees = (key <= mine) if case["causal"] else torch.ones_like(key <= mine)
                if case["window"]:
                    sees = sees & (mine - key < case["window"])
                for h in range(H):
                    s = (q[i: i + 1024, h // (H // KV), h % (H // KV)] @ k[:, h // (H // KV)].T) / math.sqrt(hd)
                    s = torch.where(sees, s, -torch.inf)
                    l = torch.logsumexp(s, -1, keepdim=True)
                    o[i: i + 1024, h] = torch.exp(s - l) @ v[:, h // (H // KV)]
                    lse[i: i + 1024, h] = l[:, 0]
            q_all.append(o)
            l_all.append(lse)
    cat = lambda v: torch.cat(v)  # noqa: E731
    if case["op"] == "read":
        return {"k": cat(k_all), "v": cat(v_all)}
    if case["op"] == "append":
        return {"q": cat(q_all), "k": cat(k_all), "v": cat(v_all)}
    return {"out": cat(q_all), "lse": cat(l_all)} if case["lse"] else {"out": cat(q_all)}
