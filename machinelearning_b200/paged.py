"""Serving over a paged key/value cache: the cache of one layer and the three
steps of a decode step that touch it.

A ``PagedKVCache`` is a view of a pool of pages (K and V tensors
``[pages][kv heads][slots per page][head_dim]`` in f32, f16 or bf16) with a
block table: row ``s`` of ``block_table`` lists the pages of sequence ``s``.
Sequences have their own lengths, positions and pages; the table, lengths and
positions are device tensors, so a captured step can be replayed while they
advance in place.

* ``append``  the new tokens' q, k, v: per-head RMSNorm, rotation, k and v into
              their slots (``qmm_paged_append_dev``)
* ``attend``  attention of one new token per sequence over its slots
              (``qmm_paged_attention_dev``)
* ``evict``   keeps the slots with the most accumulated attention weight
              (``qmm_paged_evict_dev``)

All run on the current torch stream of the cache's device. The reference keeps
one dense f32 cache per sequence (layers/main/src/core/attention.rs:454-610).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import KV_BF16, KV_F16, KV_F32

KV_DTYPES = {torch.float32: KV_F32, torch.float16: KV_F16, torch.bfloat16: KV_BF16}


def _mismatch(message: str) -> _lib.ShapeMismatch:
    return _lib.ShapeMismatch(_lib.ERR_SHAPE_MISMATCH, message)


class PagedKVCache:
    """K and V pages of one layer and the block table (int32 [sequences][pages
    of a sequence]; an entry outside the pool names no page). ``k`` and ``v`` may
    be strided views (one pool for all layers, say) with contiguous rows."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor):
        if k.dim() != 4 or k.shape != v.shape or self._strides(k) != self._strides(v):
            raise _mismatch("k and v: [pages][kv heads][slots][head_dim], of equal shape and strides")
        if k.dtype not in KV_DTYPES or v.dtype != k.dtype:
            raise _lib.DTypeMismatch(_lib.ERR_DTYPE_MISMATCH, f"cache types {k.dtype}, {v.dtype}")
        if block_table.dim() != 2 or block_table.dtype != torch.int32:
            raise _mismatch("block_table: int32 [sequences][pages]")
        if not k.is_cuda or v.device != k.device or block_table.device != k.device:
            raise ValueError("k, v and block_table have to be on one GPU")
        if k.stride(3) != 1 or v.stride(3) != 1 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
            raise _mismatch("rows of the cache and of the block table have to be contiguous")
        self.k, self.v, self.block_table = k, v, block_table
        self.device = k.device
        self._index = k.device.index
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.n_seqs, self.max_pages = block_table.shape
        self.capacity = self.max_pages * self.page_size  # slots of one sequence
        self._desc = _lib.PagedKv(k.data_ptr(), v.data_ptr(), KV_DTYPES[k.dtype], self.n_kv_heads, self.head_dim,
                                  self.page_size, self.n_pages, *self._strides(k), block_table.data_ptr(), self.n_seqs,
                                  self.max_pages, block_table.stride(0) if self.n_seqs > 1 else self.max_pages)
        self._ref = ctypes.byref(self._desc)
        self._lib = _lib.lib()
        self._seqs_shape = (self.n_seqs,)
        self._slots_shape = (self.n_seqs, self.n_kv_heads, self.capacity)

    @staticmethod
    def _strides(t: torch.Tensor) -> list[int]:
        """Of pages, heads and slots; a dimension of size one has any stride."""
        return [t.shape[3] if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])]

    @classmethod
    def allocate(cls, n_seqs: int, capacity: int, n_kv_heads: int, head_dim: int, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: int = 0) -> "PagedKVCache":
        """A cache of its own with room for ``capacity`` slots of every sequence."""
        per = -(-capacity // page_size)
        dev = torch.device("cuda", device)
        k = torch.zeros(n_seqs * per, n_kv_heads, page_size, head_dim, dtype=dtype, device=dev)
        table = torch.arange(n_seqs * per, dtype=torch.int32, device=dev).view(n_seqs, per)
        return cls(k, torch.zeros_like(k), table)

    # ---- argument checks (a few attribute reads a tensor: small steps are bound by the host) ----
    def _check(self, t: torch.Tensor, name: str, dtype: torch.dtype, shape) -> int:
        """The pointer of a contiguous tensor of this type and shape on the cache's device."""
        if t.dtype is dtype and t.shape == shape and t.get_device() == self._index and t.is_contiguous():
            return t.data_ptr()
        if t.dtype is not dtype:
            raise _lib.DTypeMismatch(_lib.ERR_DTYPE_MISMATCH, f"{name}: {t.dtype}, expected {dtype}")
        if t.shape != shape:
            raise _mismatch(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
        raise ValueError(f"{name} has to be contiguous and on {self.device}")

    def _rows(self, t: torch.Tensor, name: str, row: int):
        """(pointer, row stride) of an f32 tensor of contiguous rows of ``row`` values."""
        if t.dtype is not torch.float32:
            raise _lib.DTypeMismatch(_lib.ERR_DTYPE_MISMATCH, f"{name}: {t.dtype}, expected torch.float32")
        if t.get_device() != self._index:
            raise ValueError(f"{name} has to be on {self.device}")
        if t.is_contiguous():
            return t.data_ptr(), row
        if t[0].is_contiguous():
            return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else row
        raise ValueError(f"{name}: rows have to be contiguous")

    def _call(self, fn, *args) -> None:
        """Calls a library function on the current stream of the cache's device (it launches on the
        current device, which is made the cache's)."""
        if torch._C._cuda_getDevice() == self._index:
            status = fn(self._ref, *args, torch._C._cuda_getCurrentRawStream(self._index))
        else:
            with torch.cuda.device(self.device):
                status = fn(self._ref, *args, torch._C._cuda_getCurrentRawStream(self._index))
        if status:
            _lib.check(status)

    # ---- operators ---------------------------------------------------------------------
    def append(self, qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, cos: torch.Tensor,
               sin: torch.Tensor, *, n_heads: int, q_norm: torch.Tensor | None = None,
               k_norm: torch.Tensor | None = None, offset: float = 0.0, eps: float = 1e-6,
               seqs: torch.Tensor | None = None, interleaved: bool = False,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """q [tokens][n_heads][head_dim] of the fused f32 rows ``qkv`` [tokens][(n_heads
        + 2 n_kv_heads) head_dim]; k and v of token i go to slot ``slots[i]`` of
        sequence ``seqs[i]`` (default: sequence i), on a page that no other sequence
        shares. ``positions[i]`` picks the row of the cos/sin tables [ctx][head_dim /
        2]. Rows with slot -1 store nothing."""
        tokens, hd = qkv.shape[0], self.head_dim
        row = (n_heads + 2 * self.n_kv_heads) * hd
        if qkv.numel() != tokens * row:
            raise _mismatch(f"qkv: {tuple(qkv.shape)} is not [tokens][({n_heads} + 2 * {self.n_kv_heads}) * {hd}]")
        ctx = cos.shape[0]
        if seqs is None and tokens > self.n_seqs:
            raise _mismatch(f"{tokens} tokens for {self.n_seqs} sequences: seqs is needed")
        if (q_norm is None) != (k_norm is None):
            raise ValueError("q_norm and k_norm: both or neither")
        i32, f32, check, one = torch.int32, torch.float32, self._check, (tokens,)
        ptr, ld = self._rows(qkv, "qkv", row)
        shape, table = (tokens, n_heads, hd), (ctx, hd // 2)
        if out is None:
            out = qkv.new_empty(shape)
            out_ptr = out.data_ptr()
        else:
            out_ptr = check(out, "out", f32, shape)
        self._call(self._lib.qmm_paged_append_dev, ptr, ld, tokens, n_heads,
                   None if q_norm is None else check(q_norm, "q_norm", f32, (hd,)),
                   None if k_norm is None else check(k_norm, "k_norm", f32, (hd,)), offset, eps,
                   check(cos, "cos", f32, table), check(sin, "sin", f32, table), ctx, interleaved,
                   check(positions, "positions", i32, one), check(slots, "slots", i32, one),
                   None if seqs is None else check(seqs, "seqs", i32, one), out_ptr)
        return out

    def attend(self, q: torch.Tensor, lengths: torch.Tensor, scale: float, *, window: int = 0,
               weights: torch.Tensor | None = None, weights_out: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """softmax(scale q . k) v [sequences][heads][head_dim] of f32 queries of that
        shape over each sequence's first ``lengths`` slots (the last ``window`` of
        them, 0: all); a sequence of length 0 gives zeros. ``weights`` f32
        [sequences][kv heads][capacity]: every slot's softmax weight, summed over
        the kv head's query heads, is added (into ``weights_out`` if given). The
        library's workspace then holds sequences * heads * capacity scores."""
        shape = q.shape
        if len(shape) != 3 or shape[0] != self.n_seqs or shape[2] != self.head_dim:
            raise _mismatch(f"q: {tuple(shape)} is not [{self.n_seqs}][heads][{self.head_dim}]")
        f32, check = torch.float32, self._check
        ptr, ld = self._rows(q, "q", shape[1] * shape[2])
        w = w_out = None
        if weights is not None:
            w = check(weights, "weights", f32, self._slots_shape)
            w_out = w if weights_out is None else check(weights_out, "weights_out", f32, self._slots_shape)
        elif weights_out is not None:
            raise ValueError("weights_out without weights")
        if out is None:
            out = q.new_empty(shape)
            out_ptr = out.data_ptr()
        else:
            out_ptr = check(out, "out", f32, shape)
        self._call(self._lib.qmm_paged_attention_dev, ptr, ld, shape[1],
                   check(lengths, "lengths", torch.int32, self._seqs_shape), scale, window, w, w_out, out_ptr)
        return out

    def evict(self, lengths: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor,
              next_positions: torch.Tensor, budget: int, recent: int):
        """(lengths, weights, positions) after every sequence is brought down to at
        most ``budget`` slots per kv head: the slots of the last ``recent`` positions
        before ``next_positions``, then those with the largest ``weights``, ties by
        the lowest slot. Kept slots at or above ``budget`` move (k and v in place)
        into the evicted ones below it, in slot order. ``weights`` f32 and
        ``positions`` int32 [sequences][kv heads][capacity] are not changed. A page
        below a sequence's length may be on no other sequence's row of the table (a
        shared prefix): rows would move under the other one."""
        i32, f32, check, slots = torch.int32, torch.float32, self._check, self._slots_shape
        args = (check(lengths, "lengths", i32, self._seqs_shape), check(weights, "weights", f32, slots),
                check(positions, "positions", i32, slots),
                check(next_positions, "next_positions", i32, self._seqs_shape), budget, recent)
        new = torch.empty_like(lengths), torch.empty_like(weights), torch.empty_like(positions)
        self._call(self._lib.qmm_paged_evict_dev, *args, new[0].data_ptr(), new[1].data_ptr(), new[2].data_ptr())
        return new

    def reserve(self, n_heads: int, weights: bool = False, budget: int = 0,
                stream: torch.cuda.Stream | None = None) -> None:
        """Grows the library's workspace of ``stream`` (default: the current one) to
        what ``attend`` (with ``weights``) and ``evict`` (``budget`` > 0) of this cache
        need; call it before capturing them in a CUDA graph."""
        need = self._lib.qmm_paged_attention_workspace_size(self._ref, int(n_heads), int(weights))
        if not need:
            raise _mismatch(f"{n_heads} query heads on {self.n_kv_heads} kv heads, or a cache that attend refuses")
        if budget < 0:
            raise ValueError(f"budget {budget}")
        if budget:
            need = max(need, self._lib.qmm_paged_evict_workspace_size(self._ref, int(budget)))
        stream = torch.cuda.current_stream(self.device) if stream is None else stream
        _lib.check(self._lib.qmm_reserve_workspace(self.device.index, ctypes.c_void_p(stream.cuda_stream), need))
