"""A token for every row of a batch's logits (include/yalm_b200.h, yb_sample_rows_dev) on torch tensors: yalm's
Sampler (src/sampler.cpp:11-64) for rows with settings of their own, with top-k, top-p and min-p."""
from __future__ import annotations

from . import _lib
from .paged import _dtype


def sample_rows(logits, coin, tokens, *, prob=None, temperature=None, top_k=None, top_p=None, min_p=None,
                stream: int | None = None) -> None:
    """logits [rows][vocab] fp32, fp16 or bf16, unit column stride; coin [rows] fp32 random numbers from 0 to 1; writes
    tokens [rows] int32 and, where given, prob [rows] fp32.  temperature, top_p, min_p [rows] fp32 and top_k [rows] int32:
    each row's settings, None for temperature 1 and no limit.  All on one GPU; launches on `stream`, a cudaStream_t as an
    integer (0: the legacy default stream), or without it on torch's current stream of that GPU."""
    import torch
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows][vocab] with unit column stride")
    rows, vocab = logits.shape
    index = logits.get_device()

    def vector(t, name: str, dtype, needed: bool = False):
        if t is None and not needed:
            return None
        if t.dtype is not dtype or tuple(t.shape) != (rows,) or t.get_device() != index or not t.is_contiguous():
            raise ValueError(f"{name} must hold {rows} contiguous {dtype} values on {logits.device}")
        return t.data_ptr()

    f32, i32 = torch.float32, torch.int32
    args = (vector(tokens, "tokens", i32, True), vector(prob, "prob", f32), logits.data_ptr(),
            logits.stride(0) if rows > 1 else vocab, _dtype(logits, "logits"), rows, vocab,
            vector(coin, "coin", f32, True), vector(temperature, "temperature", f32), vector(top_k, "top_k", i32),
            vector(top_p, "top_p", f32), vector(min_p, "min_p", f32))
    if stream is None:
        stream = torch.cuda.current_stream(index).cuda_stream if index >= 0 else 0
    _lib.check(_lib.lib().yb_sample_rows_dev(*args, stream))
