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
    GPU, contiguous.  The calls launch on `stream`, a cudaStream_t as an integer (0: the legacy default stream), or
    without it on torch's current stream of that GPU."""

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
        self._append, self._attend = _lib.lib().yb_paged_append_dev, _lib.lib().yb_paged_attention_dev
        self._scratch = 0
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._codes = {}
        self._index = k_pages.get_device()
        import torch  # the caller's tensors are torch's; the package itself does not need it
        self._f32, self._i32 = torch.float32, torch.int32
        self._current = torch.cuda.current_stream
        self._q_shape = (self.n_tokens, self.n_heads * self.head_dim)
        self._qkv_shape = (self.n_tokens, (self.n_heads + 2 * self.n_kv_heads) * self.head_dim)

    def _rows(self, t, name: str, shape) -> int:
        """Checks a token-major tensor and returns its row stride in elements."""
        row, col = t.stride()
        if t.shape != shape or col != 1 or t.get_device() != self._index:
            raise ValueError(f"{name} must be [{shape[0]}][{shape[1]}] with unit column stride on {self.device}")
        return row if self.n_tokens > 1 else shape[1]

    def _stream(self) -> int:
        return self._current(self._index).cuda_stream if self._index >= 0 else 0

    def _vector(self, t, name: str, n: int, dtype):
        """Checks an optional vector and returns its address."""
        if t is None:
            return None
        if t.dtype is not dtype or t.numel() < n or t.get_device() != self._index or not t.is_contiguous():
            raise ValueError(f"{name} must hold {n} contiguous {dtype} values on {self.device}")
        return t.data_ptr()

    def append(self, qkv, q_out, inv_freq, rotary_dim: int, *, q_norm=None, k_norm=None, eps: float = 1e-5,
               half: bool = False, pos=None, clip: float = FLT_MAX, stream: int | None = None) -> None:
        """yb_paged_append_dev: clip, norm and rotate qkv [n_tokens][(n_heads + 2 n_kv_heads) head_dim], queries to
        q_out, keys and values into their pages."""
        src = self._codes.get(qkv.dtype)
        if src is None:
            src = self._codes[qkv.dtype] = _dtype(qkv, "qkv")
        s_in, s_out = self._rows(qkv, "qkv", self._qkv_shape), self._rows(q_out, "q_out", self._q_shape)
        if q_out.dtype != self._dtype:
            raise ValueError("q_out must have the caches' type")
        _lib.check(self._append(
            self._ref, q_out.data_ptr(), s_out, qkv.data_ptr(), s_in, src,
            self._vector(q_norm, "q_norm", self.head_dim, self._f32),
            self._vector(k_norm, "k_norm", self.head_dim, self._f32), eps,
            self._vector(inv_freq if rotary_dim else None, "inv_freq", rotary_dim // 2, self._f32), rotary_dim,
            1 if half else 0, self._vector(pos, "pos", self.n_tokens, self._i32), clip,
            self._stream() if stream is None else stream))

    def scratch_bytes(self) -> int:
        """Size of attend's workspace: one for each stream of calls.  Its first word collects status bits, so it is
        to start as zeros; the rest has no meaning between calls."""
        if not self._scratch:
            self._scratch = _lib.lib().yb_paged_attention_scratch_bytes(self._ref)
            if not self._scratch:
                raise _lib.YalmB200Error(_lib.YB_E_INVALID, _lib.last_error())
        return self._scratch

    def _check_scratch(self, scratch) -> None:
        if scratch.get_device() != self._index or not scratch.is_contiguous() or \
                scratch.numel() * scratch.element_size() < (self._scratch or self.scratch_bytes()):
            raise ValueError("scratch must hold scratch_bytes() contiguous bytes")

    def status(self, scratch) -> int:
        """Waits for the device and returns the status bits (as Model.status) of the attend calls in this workspace
        since the last look, or since it was made of zeros: 0, or their outputs are not complete.  Clears them.  Not
        for a stream that is being captured."""
        import torch
        self._check_scratch(scratch)
        if scratch.is_cuda:
            torch.cuda.synchronize(scratch.device)
        word = scratch.view(-1).view(torch.uint8)[:4].view(torch.int32)
        bits = int(word.item()) & 0xFFFFFFFF
        if bits:
            word.zero_()
            if scratch.is_cuda:  # before a call on any stream
                torch.cuda.synchronize(scratch.device)
        return bits

    def attend(self, q, out, scratch, *, scale: float | None = None, window: int = 0,
               stream: int | None = None) -> None:
        """yb_paged_attention_dev: causal attention of q [n_tokens][n_heads * head_dim] over the caches.  The launch
        is not waited for; a wait inside it that runs out is told by status()."""
        s_q, s_out = self._rows(q, "q", self._q_shape), self._rows(out, "out", self._q_shape)
        if q.dtype != self._dtype or out.dtype != self._dtype:
            raise ValueError("q and out must have the caches' type")
        self._check_scratch(scratch)
        window = max(-1, min(window, 0x7FFFFFFF))  # a C int; what is wider than any cache sees all of it
        _lib.check(self._attend(self._ref, out.data_ptr(), s_out, q.data_ptr(), s_q,
                                self._scale if scale is None else scale, window, scratch.data_ptr(),
                                self._stream() if stream is None else stream))
