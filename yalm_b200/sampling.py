"""A token for every row of a batch's logits (include/yalm_b200.h, yb_sample_rows_dev) on torch tensors: yalm's
Sampler (src/sampler.cpp:11-64) for rows with settings of their own, with top-k, top-p and min-p."""
from __future__ import annotations

from . import _lib
from .paged import _dtype, _raw_stream

_codes = {}  # element types that logits may have
_stream = None


def _vector(t, name: str, rows: int, dtype, index: int):
    """Checks a vector of a row's settings each and returns its address."""
    if t is None:
        return None
    if t.dtype is not dtype or t.dim() != 1 or t.numel() != rows or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must hold {rows} contiguous {dtype} values on the logits' device")
    return t.data_ptr()


def sample_rows(logits, coin, tokens, *, prob=None, temperature=None, top_k=None, top_p=None, min_p=None,
                stream: int | None = None) -> None:
    """logits [rows][vocab] fp32, fp16 or bf16, unit column stride; coin [rows] fp32 random numbers from 0 to 1; writes
    tokens [rows] int32 and, where given, prob [rows] fp32.  temperature, top_p, min_p [rows] fp32 and top_k [rows] int32:
    each row's settings, None for temperature 1 and no limit.  All on one GPU; launches on `stream`, a cudaStream_t as an
    integer (0: the legacy default stream), or without it on torch's current stream of that GPU."""
    global _stream
    if _stream is None:
        import torch
        _codes["f32"], _codes["i32"] = torch.float32, torch.int32
        _stream = _raw_stream()  # last: calls of other threads go by it
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows][vocab] with unit column stride")
    rows, vocab = logits.shape
    index, f32, i32 = logits.get_device(), _codes["f32"], _codes["i32"]
    code = _codes.get(logits.dtype)
    if code is None:
        code = _codes[logits.dtype] = _dtype(logits, "logits")
    if coin is None or tokens is None:
        raise ValueError("coin and tokens are needed")
    args = (_vector(tokens, "tokens", rows, i32, index), _vector(prob, "prob", rows, f32, index), logits.data_ptr(),
            logits.stride(0) if rows > 1 else vocab, code, rows, vocab, _vector(coin, "coin", rows, f32, index),
            _vector(temperature, "temperature", rows, f32, index), _vector(top_k, "top_k", rows, i32, index),
            _vector(top_p, "top_p", rows, f32, index), _vector(min_p, "min_p", rows, f32, index))
    if stream is None:
        stream = _stream(index) if index >= 0 else 0
    _lib.check(_lib.lib().yb_sample_rows_dev(*args, stream))
