"""Logits of the next token before sampling: penalties for repeated tokens,
biases and a grammar mask in one pass (``qmm_process_logits_dev``)."""
from __future__ import annotations

import contextlib

import torch

from . import _lib
from ._lib import MAX_BIAS

_HERE = contextlib.nullcontext()


def _ptr(t: torch.Tensor | None, name: str, dtype: torch.dtype, shape, index: int) -> int | None:
    """The pointer of a contiguous tensor of this type and shape on GPU ``index``."""
    if t is None:
        return None
    if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype:
        raise _lib.DTypeMismatch(_lib.ERR_DTYPE_MISMATCH, f"{name}: {t.dtype}, expected {dtype}")
    if t.shape != shape:
        raise _lib.ShapeMismatch(_lib.ERR_SHAPE_MISMATCH, f"{name}: shape {tuple(t.shape)}, expected {shape}")
    raise ValueError(f"{name} has to be contiguous and on cuda:{index}")


def process_logits(logits: torch.Tensor, *, tokens: torch.Tensor | None = None,
                   token_lengths: torch.Tensor | None = None, prompt_lengths: torch.Tensor | None = None,
                   repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                   bias_values: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                   mask_rows: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """f32 logits [rows][vocab] (rows may be strided) after, in this order:

    * repetition: a token among the row's first ``token_lengths`` ids of ``tokens``
      (int32 [rows][n]): x / r where x > 0, else x * r (``repetition`` f32 [rows])
    * frequency and presence (f32 [rows]): x - f * count - p for a token that
      comes count > 0 times after the first ``prompt_lengths`` ids
    * biases: ``bias_values`` f32 added at ``bias_ids`` int32 (both [rows][n], n <= 1024)
    * grammar: -inf where the token's bit (t % 32 of word t / 32) of state
      ``mask_rows[row]`` of ``mask`` (int32 [states][ceil(vocab / 32)]) is clear;
      state -1: no mask; without ``mask_rows`` row i uses state i

    ``out`` may be ``logits``. Ids outside the vocabulary are ignored: pad bias lists
    with -1."""
    if logits.dim() != 2:
        raise _lib.ShapeMismatch(_lib.ERR_SHAPE_MISMATCH, f"logits: {tuple(logits.shape)} is not [rows][vocab]")
    f32, i32 = torch.float32, torch.int32
    if logits.dtype is not f32:
        raise _lib.DTypeMismatch(_lib.ERR_DTYPE_MISMATCH, f"logits: {logits.dtype}, expected {f32}")
    dev = logits.get_device()
    if dev < 0:
        raise ValueError("logits have to be on a GPU")
    rows, vocab = logits.shape
    if (tokens is None) != (token_lengths is None) or (bias_ids is None) != (bias_values is None):
        raise ValueError("tokens and token_lengths, bias_ids and bias_values: both or neither")
    if tokens is None and (prompt_lengths is not None or repetition is not None or presence is not None
                           or frequency is not None):
        raise ValueError("penalties need tokens")
    if mask is None and mask_rows is not None:
        raise ValueError("mask_rows without mask")
    width = 0 if tokens is None else tokens.shape[-1]
    n_bias = 0 if bias_ids is None else bias_ids.shape[-1]
    n_masks = 0 if mask is None else mask.shape[0]
    if n_bias > MAX_BIAS:
        raise _lib.ShapeMismatch(_lib.ERR_SHAPE_MISMATCH, f"{n_bias} biases a row, at most {MAX_BIAS}")
    if out is not None and (out.shape != logits.shape or out.dtype is not f32 or out.get_device() != dev):
        raise _lib.ShapeMismatch(_lib.ERR_SHAPE_MISMATCH, "out differs from logits in shape, type or device")
    for t in (logits,) if out is None else (logits, out):
        if vocab > 1 and t.stride(1) != 1:
            raise ValueError("rows of logits and out have to be contiguous")
    one, bias = (rows,), (rows, n_bias)
    lib = _lib.lib()
    if out is None:
        out = logits.new_empty((rows, vocab))
    with _HERE if torch._C._cuda_getDevice() == dev else torch.cuda.device(dev):
        status = lib.qmm_process_logits_dev(
            logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab,
            _ptr(tokens, "tokens", i32, (rows, width), dev), width, width,
            _ptr(token_lengths, "token_lengths", i32, one, dev),
            _ptr(prompt_lengths, "prompt_lengths", i32, one, dev), _ptr(repetition, "repetition", f32, one, dev),
            _ptr(presence, "presence", f32, one, dev), _ptr(frequency, "frequency", f32, one, dev),
            _ptr(bias_ids, "bias_ids", i32, bias, dev), _ptr(bias_values, "bias_values", f32, bias, dev), n_bias,
            _ptr(mask, "mask", i32, (n_masks, (vocab + 31) // 32), dev), n_masks,
            _ptr(mask_rows, "mask_rows", i32, one, dev), out.data_ptr(), out.stride(0) if rows > 1 else vocab,
            torch._C._cuda_getCurrentRawStream(dev))
    if status:
        _lib.check(status)
    return out
