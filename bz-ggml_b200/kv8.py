"""The 8-bit paged key/value cache (bzb_kv8_* of include/bzb_ext.h) on PyTorch CUDA tensors.

A program keeps one KV8Cache for each layer's pages and one KV8Batch for each shape of step, refills the
batch's device arrays, and calls append() and attention() in turn. Every call enqueues on the current
stream of the cache's device and returns; nothing is copied, converted or allocated, but for the attention
workspace, which a batch allocates at its first use on a stream, and once in each CUDA graph that captures it. The
batch holds its workspaces as long as it lives, and has to outlive the graphs that captured it; one graph is not to be
launched again while it runs.
"""
from __future__ import annotations

import ctypes
import os

from . import lib

_p, _ll, _i = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int


class _Cache(ctypes.Structure):
    _fields_ = [("pages", _p), ("scales", _p), ("page_table", _p), ("status", _p), ("page_stride", _ll),
                ("scale_stride", _ll), ("n_pages", _i), ("n_slots", _i), ("max_pages", _i), ("page_tokens", _i),
                ("n_kv", _i), ("head_dim", _i), ("device", _i)]


class _Batch(ctypes.Structure):
    _fields_ = [("q_start", _p), ("kv_len", _p), ("slots", _p), ("n_seq", _i), ("n_tok", _i), ("max_new", _i),
                ("max_len", _i), ("device", _i)]  # (the device is for csrc/kv8_torch.cpp, behind the C struct)


_EXT = None


def _ext(library):
    """The compiled PyTorch side of the calls (csrc/kv8_torch.cpp), bound to the loaded libbreeze.so."""
    global _EXT
    if _EXT is None:
        import importlib.util
        import torch  # noqa: F401  (its libraries must be loaded first)
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_kv8_torch.so")
        if not os.path.exists(path):
            raise FileNotFoundError(f"_kv8_torch.so not found at {path}; run `make -C {os.path.dirname(path)}`")
        spec = importlib.util.spec_from_file_location("_kv8_torch", path)
        ext = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(ext)
        at = lambda name: ctypes.cast(getattr(library.lib, name), ctypes.c_void_p).value  # noqa: E731
        ext.bind(at("bzb_kv8_append"), at("bzb_kv8_read"), at("bzb_kv8_attention"), at("bzb_kv8_attention_workspace"),
                 at("breeze_last_error"))
        _EXT = ext
    return _EXT


def _check(t, name: str, dtype: str, dims: int, device: int, contiguous: bool = True) -> None:
    if str(t.dtype) != "torch." + dtype or t.dim() != dims or t.get_device() != device or (contiguous and not t.is_contiguous()):
        raise ValueError(f"{name}: {'contiguous ' if contiguous else ''}{dims}-d {dtype} tensor on cuda:{device} expected")


class KV8Batch:
    """The rows and positions of one call.

    q_start [n_seq + 1], kv_len [n_seq] and slots [n_seq] (page table rows, None: 0, 1, ...) are int32
    CUDA tensors, read when the work runs: sequence b has rows q_start[b]..q_start[b + 1] - 1 of n_tok,
    and its last row stands for position kv_len[b] - 1. max_new and max_len bound every sequence's
    rows and kv_len.
    """

    def __init__(self, q_start, kv_len, n_tok: int, max_new: int, max_len: int, slots=None):
        dev, n = q_start.get_device(), kv_len.numel()
        if dev < 0:
            raise ValueError("q_start: a CUDA tensor expected")
        _check(q_start, "q_start", "int32", 1, dev)
        _check(kv_len, "kv_len", "int32", 1, dev)
        if slots is not None:
            _check(slots, "slots", "int32", 1, dev)
        if q_start.numel() != n + 1 or (slots is not None and slots.numel() != n):
            raise ValueError("q_start must have one entry more than kv_len, slots as many")
        self.device, self.n_tok = dev, int(n_tok)
        self._held = (q_start, kv_len, slots)
        self._c = _Batch(q_start.data_ptr(), kv_len.data_ptr(), None if slots is None else slots.data_ptr(), n, n_tok,
                         max_new, max_len, dev)
        self._at = ctypes.addressof(self._c)
        self._workspaces: dict = {}  # attention's, one for each stream, size and capture


class KV8Cache:
    """One layer's cache: pages uint8 [n_pages, 2, n_kv, page_tokens, head_dim], scales f32
    [n_pages, 2, n_kv, page_tokens // 16] (both may be strided over pages, for pools that hold several
    layers in a page) and page_table int32 [n_slots, max_pages]."""

    def __init__(self, pages, scales, page_table):
        import torch
        dev = pages.get_device()
        if dev < 0:
            raise ValueError("pages: a CUDA tensor expected")
        _check(pages, "pages", "uint8", 5, dev, False)
        _check(scales, "scales", "float32", 4, dev, False)
        _check(page_table, "page_table", "int32", 2, dev)
        n_pages, two, n_kv, page_tokens, hd = pages.shape
        if two != 2 or tuple(scales.shape) != (n_pages, 2, n_kv, page_tokens // 16):
            raise ValueError("pages must be [n_pages, 2, n_kv, page_tokens, head_dim] and scales [n_pages, 2, n_kv, page_tokens // 16]")
        if n_pages == 0 or not pages[0].is_contiguous() or not scales[0].is_contiguous():
            raise ValueError("pages and scales must be contiguous within a page")
        self.device, self.n_kv, self.head_dim, self.page_tokens = dev, n_kv, hd, page_tokens
        self.status = torch.zeros(1, dtype=torch.int32, device=pages.device)
        self._held = (pages, scales, page_table)
        one = n_pages == 1  # (a single page's stride says nothing)
        self._c = _Cache(pages.data_ptr(), scales.data_ptr(), page_table.data_ptr(), self.status.data_ptr(),
                         2 * n_kv * page_tokens * hd if one else pages.stride(0),
                         2 * n_kv * (page_tokens // 16) if one else scales.stride(0), n_pages, page_table.shape[0],
                         page_table.shape[1], page_tokens, n_kv, hd, dev)
        self._at = ctypes.addressof(self._c)
        ext = _ext(lib())
        self._append, self._read, self._attention = ext.append, ext.read, ext.attention

    def append(self, batch: KV8Batch, q, k, v, q_out, q_norm=None, k_norm=None, eps: float = 1e-6, rope=None) -> None:
        """Norms (q_norm / k_norm [head_dim] f32) and rotates (rope [positions, head_dim / 2, 2] f32: cos,
        sin) the batch's queries q [n_tok, n_head, head_dim] into q_out and its keys k [n_tok, n_kv,
        head_dim], and appends the keys and the values v. q and q_out may both be None."""
        self._append(self._at, batch._at, q, k, v, q_out, q_norm, k_norm, eps, rope)

    def read(self, batch: KV8Batch, k_out, v_out) -> None:
        """The batch's positions back as rows k_out, v_out [n_tok, n_kv, head_dim] (f32, f16 or bf16)."""
        self._read(self._at, batch._at, k_out, v_out)

    def attention(self, batch: KV8Batch, q, out, scale: float, causal: bool = True, window: int = 0, lse=None) -> None:
        """out [n_tok, n_head, head_dim] = softmax(scale q k^T) v over each row's cached keys (those up to
        its own position when causal, of them the last `window` when that is positive); lse [n_tok, n_head]
        f32, when given, gets the rows' log-sum-exp."""
        self._attention(self._at, batch._at, batch._workspaces, q, out, scale, causal, window, lse)

    def check(self) -> None:
        """Waits for the device and raises if a call met a page, slot or length out of range, or a wait inside the
        attention ran out, since the last check."""
        status = int(self.status.item())
        if status:
            self.status.zero_()
            what = {1: "a page, slot or length was out of range; that sequence was skipped",
                    2: "a bounded wait inside the attention ran out; its rows are missing or wrong"}
            raise RuntimeError("kv8: " + "; ".join(text for bit, text in what.items() if status & bit))
