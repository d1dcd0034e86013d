"""Sizes at the ends of what the 8-bit cache's entry points take, without a GPU: indexes that would leave an int are
refused before any launch. max_new is a bound and costs no memory, so such calls need no large buffers."""
import pytest

from test_kv8_host import F16, batch, cache, lib, ref, refused, rows  # noqa: F401


def wide(n_kv=1, **kw):
    return cache(n_kv=n_kv, page_stride=2 * n_kv * 16 * 64, scale_stride=2 * n_kv, max_pages=1 << 20, n_slots=1 << 24, **kw)


@pytest.mark.parametrize("kernel", [None, "few", "many"])
@pytest.mark.parametrize("max_new,n_head", [(1 << 16, 1 << 16), (1 << 24, 256), ((1 << 24) - 1, 65), (1 << 24, 1 << 16)])
def test_rows_of_a_kv_head_past_2_30_are_refused(lib, monkeypatch, kernel, max_new, n_head):  # noqa: F811
    """(token, head) rows are numbered in an int: 2^32 of them wrapped, and tiles past 2^31 began at negative rows."""
    if kernel:
        monkeypatch.setenv("BZB_KV8_ATTENTION", kernel)
    c, b, q = wide(), batch(n_seq=1, n_tok=5, max_new=max_new, max_len=1 << 22), rows(n_head, F16)
    refused(lib, lib.bzb_kv8_attention_workspace(ref(c), ref(b), n_head, 1, 0), "too large")
    refused(lib, lib.bzb_kv8_attention(ref(c), ref(b), ref(q), ref(q), None, 1.0, 1, 0, None, 0, None), "too large")


@pytest.mark.parametrize("kernel", [None, "few", "many"])
def test_more_ctas_than_a_launch_takes_are_refused(lib, monkeypatch, kernel):  # noqa: F811
    if kernel:
        monkeypatch.setenv("BZB_KV8_ATTENTION", kernel)
    c = wide(4096)
    for n_seq, max_new, n_head in ((1 << 24, 1 << 24, 4096 * 16), (1 << 24, 1, 4096), (1 << 20, 1 << 10, 4096)):
        b, q = batch(n_seq=n_seq, n_tok=5, max_new=max_new, max_len=1 << 22), rows(n_head, F16)
        refused(lib, lib.bzb_kv8_attention_workspace(ref(c), ref(b), n_head, 1, 0), "too large")
        refused(lib, lib.bzb_kv8_attention(ref(c), ref(b), ref(q), ref(q), None, 1.0, 1, 0, None, 0, None), "too large")


def test_the_largest_counts_of_rows_are_planned(lib):  # noqa: F811
    c = wide()
    for max_new, n_head in ((1 << 24, 64), (1 << 14, 1 << 16), (1 << 24, 1)):
        b = batch(n_seq=1, n_tok=5, max_new=max_new, max_len=1 << 22)
        assert lib.bzb_kv8_attention_workspace(ref(c), ref(b), n_head, 1, 0) >= 0, lib.breeze_last_error()


@pytest.mark.parametrize("hd,most", [(64, 24 << 20), (128, 36 << 20)])
def test_workspaces_stay_small_whatever_the_bounds(lib, hd, most):  # noqa: F811
    """Ranges are made to fill the GPU and for no other reason: their results take tens of MB however many
    sequences and positions a batch may have. (A range held 512 blocks at most, which made 277 MB of 512 sequences
    bounded by 131072 positions and 11 GB of 5000 by 2^20.)"""
    c = cache(max_pages=1 << 16, n_kv=8, head_dim=hd, page_stride=2 * 8 * 16 * hd, scale_stride=16, n_slots=1 << 16)
    for n_seq in (1, 3, 17, 64, 200, 512, 5000, 60000):
        for max_new in (1, 2, 5, 40, 300):
            for max_len in (64, 2000, 8192, 8200, 131072, 1 << 20):
                for n_head in (8, 32, 64):
                    for window in (0, 500, 30000):
                        b = batch(n_seq=n_seq, n_tok=n_seq * max_new, max_new=max_new, max_len=max_len)
                        n = lib.bzb_kv8_attention_workspace(ref(c), ref(b), n_head, 1, window)
                        assert 0 <= n <= most, (n_seq, max_new, max_len, n_head, window, n)
