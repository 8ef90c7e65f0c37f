"""Paged KV cache in 8 bits: quantised as it is written, read back, and decoded over.

A row of the cache, the ``head_dim`` values of one token and kv head, is held as
8-bit codes and one fp32 scale (``code * scale``), so the cache takes
``head_dim + 4`` bytes per row where bf16 takes ``2 * head_dim``, and a decode
step reads about half as much.  Two formats:

* ``"int8"``: ``code = rint(127 x / a)``, ``scale = a / 127`` with ``a`` the row's
  largest magnitude (at least 2**-100); an error of at most ``a / 254``;
* ``"fp8_e4m3"``: the scale is the smallest power of two that brings the row under
  e4m3's largest value 448, the code ``e4m3(x / scale)``; an error of at most
  2**-4 of each value.

A row with a NaN or an infinity reads back as NaN.

``QuantPool`` holds the device buffers.  ``kvq_append``, ``kvq_append_qkv`` (with the
q/k norm and rotation of :func:`lara_b200.ops.qk_norm_rope` in the same launch),
``kvq_read`` and ``gqa_decode_kvq`` are the stateless calls (``include/lara_b200.h``:
lengths, block tables and results stay on the device, nothing synchronises, and the
calls can be captured in a CUDA graph); ``QuantKVCache`` adds the page allocator of
:class:`lara_b200.paged.PagedKVCache`.  The FPGA keeps one bf16 sequence in BRAM
(hw/rtl/mem/kv_cache_ram.sv); it has no quantised cache.
"""

from __future__ import annotations

import ctypes
import math

import torch

from ._native import LARA_KVQ_FP8_E4M3, LARA_KVQ_INT8, LaraKvqPool, check, lib
from .ops import _binding, _check_words, _strided, new_workspace
from .paged import PagedKVCache

_FORMATS = {torch.int8: LARA_KVQ_INT8, torch.float8_e4m3fn: LARA_KVQ_FP8_E4M3}
_DTYPES = {"int8": torch.int8, "fp8_e4m3": torch.float8_e4m3fn}


class QuantPool:
    """Device buffers of a paged 8-bit cache.

    ``k_codes``/``v_codes``: ``[num_pages, Hkv, page_size, D]`` int8 or float8_e4m3fn,
    ``k_scales``/``v_scales``: float32 ``[num_pages, Hkv, page_size]``; contiguous, on one
    CUDA device.  ``QuantPool.empty`` allocates them.
    """

    def __init__(self, k_codes, v_codes, k_scales, v_scales):
        if k_codes.dtype not in _FORMATS:
            raise TypeError(f"codes must be int8 or float8_e4m3fn, got {k_codes.dtype}")
        if k_codes.dim() != 4:
            raise ValueError("k_codes must be [num_pages, Hkv, page_size, D]")
        self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k_codes.shape
        for name, t, dt, shape in (("k_codes", k_codes, k_codes.dtype, k_codes.shape),
                                   ("v_codes", v_codes, k_codes.dtype, k_codes.shape),
                                   ("k_scales", k_scales, torch.float32, k_codes.shape[:3]),
                                   ("v_scales", v_scales, torch.float32, k_codes.shape[:3])):
            if t.dtype != dt:
                raise TypeError(f"{name} must be {dt}, got {t.dtype}")
            if tuple(t.shape) != tuple(shape):
                raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
            if not t.is_cuda or t.device != k_codes.device:
                raise ValueError(f"{name} must be on the CUDA device of k_codes")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.device, self.index = k_codes.device, k_codes.get_device()
        self._c = LaraKvqPool(k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                              _FORMATS[k_codes.dtype], self.num_pages, self.n_kv_heads, self.page_size, self.head_dim)
        self.address = ctypes.addressof(self._c)
        self.scale = 1.0 / math.sqrt(self.head_dim)  # of the scores, where a call gives none

    @classmethod
    def empty(cls, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, fmt: str = "int8",
              device="cuda:0") -> "QuantPool":
        if fmt not in _DTYPES:
            raise ValueError(f"fmt must be one of {sorted(_DTYPES)}, got {fmt!r}")
        shape = (int(num_pages), int(n_kv_heads), int(page_size), int(head_dim))
        codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(_DTYPES[fmt]) for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)


def kvq_append(pool: QuantPool, block_table, starts, k_new, v_new, *, counts=None, new_lens=None,
               workspace=None) -> None:
    """Quantise ``k_new``/``v_new[B, Hkv, n, D]`` (bf16, any strides over contiguous rows) into the pool.

    Row ``t`` of sequence ``b`` lands at token ``starts[b] + t`` for ``t < counts[b]`` (int32 device
    tensors; ``counts=None``: all ``n``).  ``starts`` stays as it is; ``new_lens`` (int32[B], another
    tensor) receives ``starts + counts``.  ``workspace`` (``ops.new_workspace(256, device)``) collects
    the status bits of dropped rows (``ops.workspace_status``).
    """
    rc = _binding.append(pool.address, pool.index, block_table, starts, k_new, v_new, counts, new_lens, workspace)
    if rc:
        check(rc, "lara_kvq_append")


def kvq_append_qkv(pool: QuantPool, block_table, starts, q, k, v, *, positions=None, cos_sin=None, q_weight=None,
                   k_weight=None, eps: float = 1e-5, interleaved: bool = True, counts=None, new_lens=None,
                   workspace=None, out=None):
    """A serving step's row work in one launch: q and k are normed and rotated, k and v quantised into the pool.

    q ``[B, n, Hq, D]``, k and v ``[B, n, Hkv, D]`` (bf16, any strides over contiguous heads: views of one
    projection output are taken as they are).  The words are those of :func:`lara_b200.ops.qk_norm_rope` followed
    by :func:`kvq_append`, whose arguments these are; ``positions`` (int32 ``[B, n]``) default to
    ``starts[b] + t``.  Returns the new q, ``[B, n, Hq, D]`` (``out``, which may be q itself).
    """
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    rc = _binding.append_qkv(pool.address, pool.index, block_table, starts, q, k, v, out, positions, cos_sin, q_weight,
                             k_weight, eps, interleaved, counts, new_lens, workspace)
    if rc:
        check(rc, "lara_kvq_append_qkv")
    return out


def kvq_read(pool: QuantPool, block_table, seq_lens, n_tokens: int, *, starts=None, out=None, workspace=None):
    """Tokens ``starts[b] .. starts[b] + n_tokens - 1`` of every sequence as bf16 ``(k, v)[B, Hkv, n, D]``.

    ``starts=None`` reads from token 0.  Tokens at or past ``seq_lens[b]`` read as zeros.  ``out`` may be
    two strided views, e.g. ``cache[:, :, :n]`` of a bf16 cache for :func:`lara_b200.ops.gqa_prefill`.
    """
    if out is None:
        shape = (seq_lens.numel(), pool.n_kv_heads, n_tokens, pool.head_dim)
        out = tuple(torch.empty(shape, dtype=torch.bfloat16, device=pool.device) for _ in range(2))
    k, v = out
    rc = _binding.read(pool.address, pool.index, block_table, seq_lens, n_tokens, starts, k, v, workspace)
    if rc:
        check(rc, "lara_kvq_read")
    return k, v


def decode_workspace(batch: int, n_q_heads: int, n_kv_heads: int, head_dim: int, device="cuda:0") -> torch.Tensor:
    """A zeroed workspace for :func:`gqa_decode_kvq` calls of any batch with these or fewer query heads per kv head.

    One stream at a time uses it.
    """
    dev = torch.device(device)
    with torch.cuda.device(dev):
        return new_workspace(int(lib.lara_kvq_decode_workspace_bytes(batch, n_q_heads, n_kv_heads, head_dim)), dev)


def gqa_decode_kvq(q, pool: QuantPool, block_table, seq_lens, *, scale=None, workspace=None, out=None):
    """One new token per sequence: ``q[B, Hq, D]`` (bf16) attends its cached tokens; returns ``o[B, Hq, D]``.

    ``Hq`` is any multiple of the pool's kv heads up to 16 per kv head.  A sequence of length 0 gives
    zeros.  ``workspace`` comes from :func:`decode_workspace` (``None`` allocates one for the call).  ``out`` may be
    ``q``.
    """
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        workspace = decode_workspace(max(q.shape[0], 1), q.shape[1], pool.n_kv_heads, pool.head_dim, pool.device)
    if scale is None:
        scale = pool.scale
    rc = _binding.decode(pool.address, pool.index, q, block_table, seq_lens, out, scale, workspace)
    if rc:
        check(rc, "lara_gqa_decode_kvq")
    return out


class QuantKVCache(PagedKVCache):
    """:class:`PagedKVCache` (pages, prefixes, slots, files) holding 8-bit rows.

    ``append`` quantises, ``decode`` attends the codes, ``gather`` and ``read`` return bf16.  ``save`` writes
    the values the cache stands for; ``load`` quantises them again, which gives the same values.
    """

    def __init__(self, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, max_seqs: int,
                 max_seq_len: int, device="cuda:0", fmt: str = "int8"):
        self._fmt = fmt
        super().__init__(num_pages, page_size, n_kv_heads, head_dim, max_seqs, max_seq_len, device)

    def _alloc_pages(self) -> None:
        self.pool = QuantPool.empty(self.num_pages, self.page_size, self.n_kv_heads, self.head_dim, self._fmt,
                                    self.device)

    def _rows(self, slots):
        idx = torch.as_tensor(slots, device=self.device)
        return idx, self.block_table.index_select(0, idx), self.lens.index_select(0, idx)

    def append(self, k_new, v_new, slots=None) -> None:
        """k/v_new ``[n_seq, Hkv, n, D]`` (bf16, any strides) for the given slots (default: all active, ascending)."""
        slots = self._slots(slots)
        n = int(k_new.shape[2])
        shape = (len(slots), self.n_kv_heads, n, self.head_dim)
        _strided("k_new", k_new, shape, self.pool.index)
        _strided("v_new", v_new, shape, self.pool.index)
        self.reserve(slots, n)
        idx, table, lens = self._rows(slots)
        new_lens = torch.empty_like(lens)
        kvq_append(self.pool, table, lens, k_new, v_new, new_lens=new_lens, workspace=self._status)
        self.lens.index_copy_(0, idx, new_lens)
        self._lens[slots] += n

    def append_qkv(self, q, k, v, slots=None, *, cos_sin=None, q_weight=None, k_weight=None, eps: float = 1e-5,
                   interleaved: bool = True):
        """:func:`kvq_append_qkv` for the given slots, at positions that follow their cached tokens; returns q."""
        slots = self._slots(slots)
        n = int(k.shape[1])
        shape = (len(slots), n, self.n_kv_heads, self.head_dim)
        _strided("k", k, shape, self.pool.index)
        _strided("v", v, shape, self.pool.index)
        self.reserve(slots, n)
        idx, table, lens = self._rows(slots)
        new_lens = torch.empty_like(lens)
        q = kvq_append_qkv(self.pool, table, lens, q, k, v, cos_sin=cos_sin, q_weight=q_weight, k_weight=k_weight,
                           eps=eps, interleaved=interleaved, new_lens=new_lens, workspace=self._status)
        self.lens.index_copy_(0, idx, new_lens)
        self._lens[slots] += n
        return q

    def decode(self, q, slots=None, scale=None):
        """q ``[n_seq, Hq, D]`` (bf16) -> o ``[n_seq, Hq, D]`` over each slot's cached tokens."""
        slots = self._slots(slots)
        _check_words("q", q, (len(slots), q.shape[1], self.head_dim))
        _, table, lens = self._rows(slots)
        need = int(lib.lara_kvq_decode_workspace_bytes(len(slots), q.shape[1], self.n_kv_heads, self.head_dim))
        self._ws = self._large_enough(self._ws, need)
        return gqa_decode_kvq(q, self.pool, table, lens, scale=scale, workspace=self._ws)

    def read(self, slots=None, out=None):
        """bf16 ``(k, v)[n_seq, Hkv, T, D]`` of the given slots, T the longest's length, zeros past each length."""
        slots = self._slots(slots)
        n = int(self._lens[slots].max()) if out is None else int(out[0].shape[2])
        _, table, lens = self._rows(slots)
        return kvq_read(self.pool, table, lens, n, out=out, workspace=self._status)

    def gather(self, slot: int):
        """(k, v) ``[Hkv, len, D]`` bf16 of one sequence."""
        if not self._active[slot]:
            raise ValueError("slots must name active sequences")
        k, v = self.read([slot])
        return k[0], v[0]
