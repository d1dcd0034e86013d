"""The 8-bit cache's C entry points without a GPU: what they refuse, and the workspace sizes they ask for. Every
check comes before the first CUDA call that needs a device, so no memory is touched."""
import ctypes

import pytest

F32, F16, BF16 = 0, 1, 2
FAKE = 1 << 20  # an aligned address that nothing reads


class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("pages", "scales", "page_table", "status")] + \
               [(n, ctypes.c_longlong) for n in ("page_stride", "scale_stride")] + \
               [(n, ctypes.c_int) for n in ("n_pages", "n_slots", "max_pages", "page_tokens", "n_kv", "head_dim", "device")]


class Batch(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q_start", "kv_len", "slots")] + \
               [(n, ctypes.c_int) for n in ("n_seq", "n_tok", "max_new", "max_len")]


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("row_stride", ctypes.c_longlong), ("head_stride", ctypes.c_longlong),
                ("n_head", ctypes.c_int), ("type", ctypes.c_int)]


def cache(**kw):
    d = dict(pages=FAKE, scales=FAKE, page_table=FAKE, status=None, page_stride=2 * 2 * 16 * 64, scale_stride=4, n_pages=9,
             n_slots=4, max_pages=8, page_tokens=16, n_kv=2, head_dim=64, device=0)
    d.update(kw)
    return Cache(**d)


def batch(**kw):
    d = dict(q_start=FAKE, kv_len=FAKE, slots=None, n_seq=3, n_tok=5, max_new=2, max_len=128)
    d.update(kw)
    return Batch(**d)


def rows(heads, kind=F16, **kw):
    d = dict(data=FAKE, row_stride=heads * 64, head_stride=64, n_head=heads, type=kind)
    d.update(kw)
    return Rows(**d)


@pytest.fixture
def lib(pkg):
    return pkg.lib().lib


def refused(lib, rc, word):
    assert rc == -1
    assert word in lib.breeze_last_error().decode(), lib.breeze_last_error()


def ref(x):
    return None if x is None else ctypes.byref(x)


@pytest.mark.parametrize("change,word", [
    (dict(pages=None), "null pages"), (dict(scales=None), "null pages"), (dict(page_table=None), "null pages"),
    (dict(head_dim=96), "head_dim"), (dict(page_tokens=24), "page_tokens"), (dict(page_tokens=512), "page_tokens"),
    (dict(n_kv=0), "n_kv"), (dict(n_pages=0), "positive"), (dict(max_pages=0), "positive"),
    (dict(page_stride=4095), "page_stride"), (dict(page_stride=4096 + 8), "page_stride"), (dict(scale_stride=3), "scale_stride"),
    (dict(pages=FAKE + 8), "16-byte"), (dict(scales=FAKE + 2), "4-byte"), (dict(max_pages=1 << 27), "too large"),
])
def test_caches_refused(lib, change, word):
    c, b, k = cache(**change), batch(max_len=min(128, 16)), rows(2)
    refused(lib, lib.bzb_kv8_read(ref(c), ref(b), ref(k), ref(k), None), word)
    refused(lib, lib.bzb_kv8_append(ref(c), ref(b), None, ref(k), ref(k), None, None, None, 1e-6, None, 0, None), word)
    refused(lib, lib.bzb_kv8_attention_workspace(ref(c), ref(b), 4, 1, 0), word)


@pytest.mark.parametrize("change,word", [
    (dict(q_start=None), "q_start"), (dict(kv_len=None), "kv_len"), (dict(n_seq=5), "page table rows"), (dict(n_tok=-1), "negative"),
    (dict(max_len=129), "max_len"), (dict(max_new=(1 << 24) + 1), "2^24"),
])
def test_batches_refused(lib, change, word):
    c, b, q = cache(), batch(**change), rows(4)
    refused(lib, lib.bzb_kv8_attention(ref(c), ref(b), ref(q), ref(q), None, 1.0, 1, 0, None, 0, None), word)


def test_row_tensors_and_arguments_refused(lib):
    c, b = cache(), batch()
    att = lambda q, o, scale=1.0, causal=1, window=0, lse=None: lib.bzb_kv8_attention(  # noqa: E731
        ref(c), ref(b), ref(q), ref(o), lse, scale, causal, window, None, 0, None)
    refused(lib, att(None, rows(4)), "null query")
    refused(lib, att(rows(4), rows(2)), "same heads")
    refused(lib, att(rows(3), rows(3)), "multiple of n_kv")
    refused(lib, att(rows(4, F32), rows(4, F32)), "f16 or bf16")
    refused(lib, att(rows(4), rows(4, BF16)), "one type")
    refused(lib, att(rows(4, data=None), rows(4)), "null data")
    refused(lib, att(rows(4, data=FAKE + 1), rows(4)), "aligned")
    refused(lib, att(rows(4), rows(4, row_stride=0)), "overlap")
    refused(lib, att(rows(4, head_stride=32), rows(4)), "overlap")
    refused(lib, att(rows(4), rows(4), causal=0, window=3), "window")
    refused(lib, att(rows(4), rows(4), window=-3), "window")
    refused(lib, att(rows(4), rows(4), scale=float("nan")), "finite")
    refused(lib, att(rows(4), rows(4), lse=FAKE + 2), "lse")
    app = lambda q, k, v, o, wq=None, eps=1e-6, rope=None, n=0: lib.bzb_kv8_append(  # noqa: E731
        ref(c), ref(b), ref(q), ref(k), ref(v), ref(o), wq, None, eps, rope, n, None)
    refused(lib, app(None, None, rows(2), None), "null key")
    refused(lib, app(rows(4), rows(2), rows(2), None), "together")
    refused(lib, app(rows(4), rows(2), rows(2, F32), rows(4)), "one type")
    refused(lib, app(rows(4), rows(3), rows(2), rows(4)), "heads")
    refused(lib, app(rows(4), rows(2), rows(2), rows(4, F32)), "f16 or bf16")
    refused(lib, app(rows(4), rows(2), rows(2), rows(4, row_stride=8)), "overlap")
    refused(lib, app(rows(4), rows(2), rows(2), rows(4), eps=-1.0), "eps")
    refused(lib, app(rows(4), rows(2), rows(2), rows(4), wq=FAKE + 1), "q_norm")
    refused(lib, app(rows(4), rows(2), rows(2), rows(4), rope=FAKE + 8, n=128), "rope")
    refused(lib, app(rows(4), rows(2), rows(2), rows(4), rope=FAKE, n=127), "rope")
    refused(lib, lib.bzb_kv8_read(ref(c), ref(b), ref(rows(2)), ref(rows(2, F32)), None), "one type")
    refused(lib, lib.bzb_kv8_read(ref(c), ref(b), None, ref(rows(2)), None), "null key")
    refused(lib, lib.bzb_kv8_read(None, ref(b), ref(rows(2)), ref(rows(2)), None), "null cache")


def test_nothing_to_do_is_no_error(lib):
    """Batches without sequences, rows or positions return before any launch."""
    for b in (batch(n_seq=0, n_tok=0, max_new=0, max_len=0), batch(n_tok=0), batch(max_new=0)):
        assert lib.bzb_kv8_attention(ref(cache()), ref(b), ref(rows(4)), ref(rows(4)), None, 1.0, 1, 0, None, 0, None) == 0
        assert lib.bzb_kv8_read(ref(cache()), ref(b), ref(rows(2)), ref(rows(2)), None) == 0
        assert lib.bzb_kv8_append(ref(cache()), ref(b), None, ref(rows(2)), ref(rows(2)), None, None, None, 0.0, None, 0, None) == 0


def test_workspace_sizes(lib):
    """None where nothing is split; for long contexts of few sequences some, and never more than a few ranges for each SM."""
    c = cache(max_pages=1 << 16, n_kv=8, page_stride=2 * 8 * 16 * 64, scale_stride=16, n_slots=1 << 16)
    for n_seq in (1, 2, 7, 64, 500, 5000, 60000):
        for max_new in (1, 3, 16, 64, 700):
            for max_len in (16, 300, 5000, 32768, 1 << 20):
                b = batch(n_seq=n_seq, n_tok=n_seq * max_new, max_new=max_new, max_len=max_len)
                n = lib.bzb_kv8_attention_workspace(ref(c), ref(b), 32, 1, 0)
                assert n >= 0 and n % 16 == 0
                if max_len <= 64:
                    assert n == 0
                if max_len == 1 << 20 and n_seq * max_new <= 2:
                    assert n > 0
