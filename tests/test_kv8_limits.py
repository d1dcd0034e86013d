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
