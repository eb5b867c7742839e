"""The paged KV cache of a batch of sequences (include/yalm_b200.h, yb_paged_batch) on torch tensors.

PagedBatch checks the tensors' types, shapes and strides once, keeps the batch descriptor, and launches
the two kernels of a serving step: append (per-head norm, rotation, store) and attend.  The tensors
stay the caller's: new lengths and page tables are written into them between steps, also between replays
of a captured graph.  No counterpart in yalm, which runs one sequence over one contiguous cache.
"""
from __future__ import annotations

import ctypes
import math

from . import _lib

_DTYPES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}
FLT_MAX = 3.4028234663852886e38


def _dtype(t, name: str) -> int:
    d = _DTYPES.get(str(t.dtype))
    if d is None:
        raise ValueError(f"{name}: unsupported type {t.dtype}")
    return d


class PagedBatch:
    """k_pages, v_pages [n_pages][n_kv_heads][page_size][head_dim] fp16 or bf16; page_table [n_seqs][max_pages],
    q_start [n_seqs + 1] and kv_len [n_seqs] int32; n_tokens: rows of the token-major tensors.  All on one
    GPU, contiguous."""

    def __init__(self, k_pages, v_pages, page_table, q_start, kv_len, n_heads: int, n_tokens: int):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
            raise ValueError("k_pages and v_pages must be [n_pages][n_kv_heads][page_size][head_dim] of one type")
        if page_table.dim() != 2 or tuple(q_start.shape) != (page_table.shape[0] + 1,) or \
                tuple(kv_len.shape) != (page_table.shape[0],):
            raise ValueError("page_table must be [n_seqs][max_pages], q_start [n_seqs + 1], kv_len [n_seqs]")
        for name, t in (("page_table", page_table), ("q_start", q_start), ("kv_len", kv_len)):
            if str(t.dtype) != "torch.int32":
                raise ValueError(f"{name} must be int32")
        keep = (k_pages, v_pages, page_table, q_start, kv_len)
        for t in keep:
            if not t.is_contiguous() or t.device != k_pages.device:
                raise ValueError("the batch's tensors must be contiguous and on one device")
        self._keep = keep
        self.device = k_pages.device
        self.head_dim, self.n_heads, self.n_kv_heads = int(k_pages.shape[3]), int(n_heads), int(k_pages.shape[1])
        self.n_tokens = int(n_tokens)
        self._dtype = k_pages.dtype
        self.c = _lib.yb_paged_batch(
            n_seqs=page_table.shape[0], n_tokens=self.n_tokens, n_heads=self.n_heads, n_kv_heads=self.n_kv_heads,
            head_dim=self.head_dim, dtype=_dtype(k_pages, "k_pages"), page_size=k_pages.shape[2],
            n_pages=k_pages.shape[0], max_pages=page_table.shape[1], q_start_dev=q_start.data_ptr(),
            kv_len_dev=kv_len.data_ptr(), page_table_dev=page_table.data_ptr(), k_pages=k_pages.data_ptr(),
            v_pages=v_pages.data_ptr())
        self._ref = ctypes.byref(self.c)
        self._q_width = self.n_heads * self.head_dim
        self._scratch = 0
        self._qkv_width = (self.n_heads + 2 * self.n_kv_heads) * self.head_dim

    def _rows(self, t, name: str, width: int) -> int:
        """Checks a token-major tensor and returns its row stride in elements."""
        if tuple(t.shape) != (self.n_tokens, width) or t.stride(1) != 1 or t.device != self.device:
            raise ValueError(f"{name} must be [{self.n_tokens}][{width}] with unit column stride on {self.device}")
        return t.stride(0) if self.n_tokens > 1 else max(t.stride(0), width)

    def append(self, qkv, q_out, inv_freq, rotary_dim: int, *, q_norm=None, k_norm=None, eps: float = 1e-5,
               half: bool = False, pos=None, clip: float = FLT_MAX, stream: int = 0) -> None:
        """yb_paged_append_dev: clip, norm and rotate qkv [n_tokens][(n_heads + 2 n_kv_heads) head_dim], queries to
        q_out, keys and values into their pages."""
        src = _dtype(qkv, "qkv")
        s_in, s_out = self._rows(qkv, "qkv", self._qkv_width), self._rows(q_out, "q_out", self._q_width)
        if q_out.dtype != self._dtype:
            raise ValueError("q_out must have the caches' type")
        for name, t, n, d in (("q_norm", q_norm, self.head_dim, "torch.float32"),
                              ("k_norm", k_norm, self.head_dim, "torch.float32"),
                              ("inv_freq", inv_freq if rotary_dim else None, rotary_dim // 2, "torch.float32"),
                              ("pos", pos, self.n_tokens, "torch.int32")):
            if t is not None and (t.numel() < n or not t.is_contiguous() or str(t.dtype) != d
                                  or t.device != self.device):
                raise ValueError(f"{name} must hold {n} contiguous {d} values on {self.device}")
        _lib.call("yb_paged_append_dev", self._ref, q_out.data_ptr(), s_out, qkv.data_ptr(), s_in, src,
                  q_norm.data_ptr() if q_norm is not None else None,
                  k_norm.data_ptr() if k_norm is not None else None, eps,
                  inv_freq.data_ptr() if inv_freq is not None else None, rotary_dim, 1 if half else 0,
                  pos.data_ptr() if pos is not None else None, clip, stream)

    def scratch_bytes(self) -> int:
        """Size of attend's workspace: zero-filled before its first use, one per stream of calls."""
        if not self._scratch:
            self._scratch = _lib.lib().yb_paged_attention_scratch_bytes(self._ref)
            if not self._scratch:
                raise _lib.YalmB200Error(_lib.YB_E_INVALID, _lib.last_error())
        return self._scratch

    def attend(self, q, out, scratch, *, scale: float | None = None, window: int = 0, stream: int = 0) -> None:
        """yb_paged_attention_dev: causal attention of q [n_tokens][n_heads * head_dim] over the caches."""
        s_q, s_out = self._rows(q, "q", self._q_width), self._rows(out, "out", self._q_width)
        if q.dtype != self._dtype or out.dtype != self._dtype:
            raise ValueError("q and out must have the caches' type")
        if scratch.device != self.device or not scratch.is_contiguous() or \
                scratch.numel() * scratch.element_size() < self.scratch_bytes():
            raise ValueError("scratch must hold scratch_bytes() contiguous bytes")
        _lib.call("yb_paged_attention_dev", self._ref, out.data_ptr(), s_out, q.data_ptr(), s_q,
                  1.0 / math.sqrt(self.head_dim) if scale is None else scale, window, scratch.data_ptr(), stream)
