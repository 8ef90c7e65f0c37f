"""Paged KV cache for many concurrent sequences (device pool + host page allocator).

The reference attends one sequence per transaction out of BRAM
(hw/rtl/mem/kv_cache_ram.sv); a B200 serving process holds thousands of
sequences of different lengths and cannot give each a max-length slab.  Here
K/V live in page pools ``[num_pages, Hkv, page_size, D]`` (bf16; the rows of
one (page, kv head) are contiguous, so the decode kernel still moves each
64-token tile with one or a few bulk copies) and a device block table
``int32[max_seqs, pages_per_seq]`` maps token ``t`` of sequence ``s`` to page
``block_table[s, t // page_size]``.  Pages are allocated on the host from a
free list with reference counts, so a common prefix can be shared between
sequences (``share_prefix``); an append never writes into a shared page.

The kernels are ``lara_gqa_decode_paged`` / ``lara_kv_append_paged``
(include/lara_b200.h); a decode over a paged cache returns the same words as
over a contiguous cache holding the same tokens.

For batches behind a common prefix and for contexts that outgrow their room there
are, as stateless calls on the same pages and as methods of the cache:

* :func:`gqa_decode_shared`: a decode that reads the pages which all sequences begin
  with once for the batch, instead of once for each sequence;
* :func:`gqa_decode_scored`: a decode that also adds to every cached slot's weight the
  attention it got, summed over the query heads of its kv head;
* :func:`kv_evict`: cuts sequences down to a number of slots for each kv head: the first
  ones, the last ones, and the heaviest of the rest.

``save`` / ``load`` use the ``lara-kv-v1`` file format of :mod:`lara_b200.kvfile`.
"""

from __future__ import annotations

import math

import numpy as np
import torch

from . import kvfile
from ._native import check, lib
from .ops import _binding, _check_words, _stream, new_workspace


def _workspace(nbytes: int, device) -> torch.Tensor:
    dev = torch.device(device)
    with torch.cuda.device(dev):
        return new_workspace(nbytes, dev)


def shared_workspace(batch: int, n_q_heads: int, n_kv_heads: int, head_dim: int, device="cuda:0") -> torch.Tensor:
    """A zeroed workspace for :func:`gqa_decode_shared` calls of this or a smaller batch and group of query heads.

    One stream at a time uses it.
    """
    return _workspace(int(lib.lara_decode_shared_workspace_bytes(batch, n_q_heads, n_kv_heads, head_dim)), device)


def gqa_decode_shared(q, k_pages, v_pages, block_table, seq_lens, shared_pages: int, *, scale=None, workspace=None,
                      out=None):
    """One new token per sequence, of a batch whose sequences begin with the same pages (``lara_gqa_decode_shared``).

    q ``[B, Hq, D]`` (bf16) attends the first ``seq_lens[b]`` tokens that ``block_table[b]`` names in ``k_pages`` and
    ``v_pages`` ``[num_pages, Hkv, page_size, D]``.  The first ``shared_pages`` columns of the table are the same for
    all sequences that are at least as long, and read once for them (a shorter sequence is read by itself).
    ``Hq`` is any multiple of ``Hkv`` up to 16 per kv head, ``D`` 64 or 128.  A sequence of length 0 gives zeros.
    ``workspace`` comes from :func:`shared_workspace` (``None`` allocates one for the call).  Returns ``o[B, Hq, D]``
    (``out``, which may be q).
    """
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        workspace = shared_workspace(max(q.shape[0], 1), q.shape[1], k_pages.shape[1], k_pages.shape[3], k_pages.device)
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    rc = _binding.decode_shared(q, k_pages, v_pages, block_table, seq_lens, shared_pages, out, sc, workspace)
    if rc:
        check(rc, "lara_gqa_decode_shared")
    return out


def scored_workspace(batch: int, n_q_heads: int, k_pages, pages_per_seq: int) -> torch.Tensor:
    """A zeroed workspace for :func:`gqa_decode_scored` calls over a pool and tables of these sizes, or smaller batches.

    It holds ``n_q_heads`` fp32 scores for every token that ``batch`` sequences can have in the pool.  One stream at a
    time uses it.
    """
    num_pages, hkv, page_size, d = k_pages.shape
    return _workspace(int(lib.lara_decode_scored_workspace_bytes(batch, n_q_heads, hkv, d, page_size, pages_per_seq,
                                                                 num_pages)), k_pages.device)


def gqa_decode_scored(q, k_pages, v_pages, weights, block_table, seq_lens, *, weights_out=None, scale=None,
                      workspace=None, out=None):
    """One new token per sequence, with the attention that every cached slot gets (``lara_gqa_decode_scored``).

    As :func:`gqa_decode_shared` without a shared part, and ``weights_out[slot] = weights[slot] + sum`` over the kv
    head's query heads of the slot's softmax weight: float32 ``[num_pages, Hkv, page_size]``, for the slots below
    ``seq_lens[b]`` alone (``weights_out=None``: in place).  The sequences of one call share no pages.  ``workspace``
    comes from :func:`scored_workspace`.
    """
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        workspace = scored_workspace(max(q.shape[0], 1), q.shape[1], k_pages, block_table.shape[1])
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    rc = _binding.decode_scored(q, k_pages, v_pages, weights, weights if weights_out is None else weights_out,
                                block_table, seq_lens, out, sc, workspace)
    if rc:
        check(rc, "lara_gqa_decode_scored")
    return out


def evict_workspace(batch: int, n_kv_heads: int, keep: int, device="cuda:0") -> torch.Tensor:
    """A zeroed workspace for :func:`kv_evict` calls of these or smaller sizes.  One stream at a time uses it."""
    return _workspace(int(lib.lara_kv_evict_workspace_bytes(batch, n_kv_heads, keep)), device)


def kv_evict(k_pages, v_pages, weights, block_table, seq_lens, keep: int, *, first: int = 0, last: int = 0,
             weights_out=None, new_lens=None, sources=None, workspace=None):
    """Cut every sequence of more than ``keep`` tokens down to ``keep``, each kv head by itself (``lara_kv_evict``).

    The first ``first`` slots stay, the last ``last``, and of the rest the heaviest by ``weights`` (ties to the lowest
    slot).  Kept rows from slot ``keep`` on move, in order, into the slots below it that are given up, in order, with
    their weights; weights from ``keep`` to the old length become 0 (``weights_out=None``: in place).  The order of the
    slots is no longer that of the positions, which a decode does not need.  ``seq_lens`` stays as it is; ``new_lens``
    (int32 ``[B]``, another tensor; ``None``: a new one) receives ``min(seq_lens, keep)`` and is returned.  ``sources``
    (int32 ``[B, Hkv, keep]``) receives the slot that each slot's row came from, -1 past the new length.  The sequences
    of one call share no pages.  How the work is laid out follows from the table's width: 16 sequences of 2049 slots
    are cut by one in 10 us from tables of 2112 slots, in 42 from tables of 131072, so pass the columns that are used.
    """
    if new_lens is None:
        new_lens = torch.empty_like(seq_lens)
    if workspace is None:
        workspace = evict_workspace(max(seq_lens.numel(), 1), k_pages.shape[1], max(int(keep), 1), k_pages.device)
    rc = _binding.evict(k_pages, v_pages, weights, weights if weights_out is None else weights_out, block_table,
                        seq_lens, new_lens, sources, keep, first, last, workspace)
    if rc:
        check(rc, "lara_kv_evict")
    return new_lens


class PagedKVCache:
    """Page pool, block tables and lengths of many sequences.

    ``scored=True`` also keeps a weight for every slot and kv head (``weights``, float32), the attention it has got from
    :meth:`decode_scored` since its token was appended, by which :meth:`evict` chooses.  (Files hold no weights, and
    a prompt's own queries add none: until a scored step all slots weigh the same, and the first ones stay.)  One
    stream at a time uses a cache.
    """

    def __init__(self, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, max_seqs: int,
                 max_seq_len: int, device="cuda:0", scored: bool = False):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two >= 16")
        self.device = torch.device(device)
        self.page_size, self.n_kv_heads, self.head_dim = int(page_size), int(n_kv_heads), int(head_dim)
        self.num_pages, self.max_seqs = int(num_pages), int(max_seqs)
        self.pages_per_seq = int(math.ceil(max_seq_len / page_size))
        self._alloc_pages()
        self.weights = None
        if scored:
            self.weights = torch.zeros((self.num_pages, self.n_kv_heads, self.page_size), dtype=torch.float32,
                                       device=self.device)
        self._table = np.full((self.max_seqs, self.pages_per_seq), -1, np.int32)
        self.block_table = torch.from_numpy(self._table).to(self.device)
        self._lens = np.zeros(self.max_seqs, np.int32)
        self.lens = torch.zeros(self.max_seqs, dtype=torch.int32, device=self.device)
        self._refs = np.zeros(self.num_pages, np.int32)
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._active = np.zeros(self.max_seqs, bool)
        self._cut = np.zeros(self.max_seqs, bool)  # slots no longer in the order of the positions
        self._ws = None
        self._serving_ws = {}  # of decode_shared, decode_scored and evict
        self._status = new_workspace(256, self.device)

    def _alloc_pages(self) -> None:
        shape = (self.num_pages, self.n_kv_heads, self.page_size, self.head_dim)
        self.k_pages = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)
        self.v_pages = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)

    # ------------------------------------------------------------ allocation
    @property
    def capacity(self) -> int:
        return self.pages_per_seq * self.page_size

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def seq_len(self, slot: int) -> int:
        return int(self._lens[slot])

    def new_sequence(self) -> int:
        idle = np.flatnonzero(~self._active)
        if idle.size == 0:
            raise RuntimeError("no free sequence slot")
        slot = int(idle[0])
        self._active[slot] = True
        self._cut[slot] = False
        self._lens[slot] = 0
        self._sync_rows([slot])
        return slot

    def free_sequence(self, slot: int) -> None:
        for j in range(self.pages_per_seq):
            page = int(self._table[slot, j])
            if page >= 0:
                self._release(page)
                self._table[slot, j] = -1
        self._lens[slot] = 0
        self._active[slot] = False
        self._sync_rows([slot])

    def share_prefix(self, src: int, dst: int, n_tokens: int) -> int:
        """Give ``dst`` the first full pages of ``src`` covering up to ``n_tokens``
        tokens (reference-counted, read-only); returns the tokens shared."""
        if self._lens[dst] != 0 or not self._active[src] or not self._active[dst]:
            raise ValueError("share_prefix needs an active source and an empty active destination")
        if self._cut[src]:
            raise ValueError(f"sequence {src} has been cut by evict: its first slots are not its first tokens")
        n_pages = min(int(n_tokens), int(self._lens[src])) // self.page_size
        for j in range(n_pages):
            page = int(self._table[src, j])
            self._refs[page] += 1
            self._table[dst, j] = page
        self._lens[dst] = n_pages * self.page_size
        self._sync_rows([dst])
        return n_pages * self.page_size

    def reserve(self, slots, n_new: int) -> None:
        """Make sure each slot has pages for n_new more tokens; a call that is refused takes none."""
        wanted = []
        for slot in dict.fromkeys(int(s) for s in slots):
            need_end = int(self._lens[slot]) + int(n_new)
            if need_end > self.capacity:
                raise ValueError(f"sequence {slot} would hold {need_end} tokens > capacity {self.capacity}")
            first = int(self._lens[slot]) // self.page_size
            last = (need_end - 1) // self.page_size if need_end > 0 else -1
            for j in range(first, last + 1):
                page = int(self._table[slot, j])
                if page >= 0 and self._refs[page] > 1:
                    raise ValueError(f"sequence {slot} would append into shared page {page}")
                if page < 0:
                    wanted.append((slot, j))
        if len(wanted) > len(self._free):
            raise MemoryError("page pool exhausted")
        if not wanted:
            return
        fresh = [self._free.pop() for _ in wanted]
        for (slot, j), page in zip(wanted, fresh):
            self._refs[page] = 1
            self._table[slot, j] = page
        if self.weights is not None:  # what an earlier sequence's tokens gathered
            self.weights.index_fill_(0, torch.as_tensor(np.asarray(fresh, np.int64), device=self.device), 0.0)
        self._sync_rows(sorted({slot for slot, _ in wanted}))

    def _release(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            self._free.append(page)

    def _sync_rows(self, slots) -> None:
        idx = torch.as_tensor(np.asarray(slots, np.int64), device=self.device)
        self.block_table.index_copy_(0, idx, torch.from_numpy(self._table[slots]).to(self.device))
        self.lens.index_copy_(0, idx, torch.from_numpy(self._lens[slots]).to(self.device))

    def _slots(self, slots):
        if slots is None:
            slots = np.flatnonzero(self._active)
        slots = np.asarray(slots, np.int64)
        if slots.size == 0 or not np.all(self._active[slots]):
            raise ValueError("slots must name active sequences")
        return slots

    # --------------------------------------------------------------- kernels
    def append(self, k_new, v_new, slots=None) -> None:
        """k/v_new ``[n_seq, Hkv, n, D]`` (bf16) for the given slots (default: all active, ascending)."""
        slots = self._slots(slots)
        n = int(k_new.shape[2])
        _check_words("k_new", k_new, (len(slots), self.n_kv_heads, n, self.head_dim))
        _check_words("v_new", v_new, (len(slots), self.n_kv_heads, n, self.head_dim))
        self.reserve(slots, n)
        idx = torch.as_tensor(slots, device=self.device)
        table = self.block_table.index_select(0, idx)
        lens = self.lens.index_select(0, idx)
        check(lib.lara_kv_append_paged(self.k_pages.data_ptr(), self.v_pages.data_ptr(), table.data_ptr(),
                                       lens.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), len(slots),
                                       self.n_kv_heads, self.head_dim, self.page_size, self.pages_per_seq,
                                       self.num_pages, n, self._status.data_ptr(), _stream(self.device)),
              "lara_kv_append_paged")
        self.lens.index_copy_(0, idx, lens)
        self._lens[slots] += n

    def decode(self, q, slots=None, scale=None):
        """q ``[n_seq, Hq, D]`` (bf16) -> o ``[n_seq, Hq, D]`` over each slot's cached tokens."""
        import ctypes

        slots = self._slots(slots)
        B, hq, d = q.shape
        _check_words("q", q, (len(slots), hq, self.head_dim))
        idx = torch.as_tensor(slots, device=self.device)
        table = self.block_table.index_select(0, idx)
        lens = self.lens.index_select(0, idx)
        lens_host = np.ascontiguousarray(self._lens[slots])
        ns, ch = ctypes.c_int(0), ctypes.c_int(0)
        check(lib.lara_decode_plan(B, hq, self.n_kv_heads, d, self.capacity, lens_host.ctypes.data,
                                   ctypes.byref(ns), ctypes.byref(ch)), "lara_decode_plan")
        nbytes = int(lib.lara_decode_workspace_bytes(B, hq, self.n_kv_heads, d, ns.value))
        self._ws = self._large_enough(self._ws, nbytes)
        o = torch.empty_like(q)
        sc = 1.0 / math.sqrt(d) if scale is None else float(scale)
        check(lib.lara_gqa_decode_paged(q.data_ptr(), self.k_pages.data_ptr(), self.v_pages.data_ptr(),
                                        table.data_ptr(), lens.data_ptr(), o.data_ptr(), B, hq, self.n_kv_heads, d,
                                        self.page_size, self.pages_per_seq, self.num_pages, sc, ns.value, ch.value,
                                        self._ws.data_ptr(), self._ws.numel(), _stream(self.device)),
              "lara_gqa_decode_paged")
        return o

    def _large_enough(self, ws, nbytes: int) -> torch.Tensor:
        """``ws``, or a larger workspace in its place; the status bits of the one that goes are kept."""
        if ws is not None:
            if ws.numel() >= nbytes:
                return ws
            self._status[:4].view(torch.int32).bitwise_or_(ws[:4].view(torch.int32))
            if ws.is_cuda:  # the last call that used it may still run
                ws.record_stream(torch.cuda.current_stream(ws.device))
        return _workspace(nbytes, self.device)

    def _serving(self, name: str, nbytes: int) -> torch.Tensor:
        ws = self._serving_ws[name] = self._large_enough(self._serving_ws.get(name), nbytes)
        return ws

    def _rows_of(self, slots):
        idx = torch.as_tensor(slots, device=self.device)
        return idx, self.block_table.index_select(0, idx), self.lens.index_select(0, idx)

    def _own_pages(self, slots, what: str) -> None:
        """Refuse slots whose pages another sequence has too."""
        pages = self._table[slots]
        if np.any(self._refs[pages[pages >= 0]] > 1):
            raise ValueError(f"{what}: a sequence has pages in common with another")
        if len(np.unique(slots)) != len(slots):
            raise ValueError(f"{what}: a slot is named twice")

    def _need_weights(self, what: str) -> None:
        if not hasattr(self, "k_pages"):
            raise ValueError(f"{what} needs a cache of bf16 rows")
        if self.weights is None:
            raise ValueError(f"{what} needs a cache with weights (scored=True)")

    def shared_pages(self, slots=None) -> int:
        """How many pages the slots begin with in common, those aside that end within them.

        Every sequence that holds that many whole pages begins with the same ones, and of such prefixes it is the one
        whose single reading spares the most pages.
        """
        slots = self._slots(slots)
        rows = self._table[slots]
        if len(slots) == 1:
            return int((rows[0] >= 0).cumprod().sum())
        whole = self._lens[slots] // self.page_size
        n = int(whole.max())
        if n == 0:
            return 0
        same = rows[:, :n] == rows[whole.argmax(), :n]
        same = np.where(same.all(1), n, same.argmin(1))  # pages that are also the longest sequence's, from the first
        ends = np.bincount(whole, minlength=n + 1)
        holders = len(slots) - ends.cumsum()[:n]  # sequences with 1, 2, .. n whole pages
        differ = (np.bincount(np.minimum(same, whole), minlength=n + 1) - ends)[:n].cumsum()  # of them, with other ones
        spared = np.where(differ == 0, (holders - 1) * np.arange(1, n + 1), 0)
        most = int(spared.argmax())
        return most + 1 if spared[most] > 0 else 0

    def decode_shared(self, q, slots=None, scale=None):
        """:meth:`decode`, reading the pages that all slots begin with (:meth:`share_prefix`) once for the batch."""
        if not hasattr(self, "k_pages"):
            raise ValueError("decode_shared needs a cache of bf16 rows")
        slots = self._slots(slots)
        _check_words("q", q, (len(slots), q.shape[1], self.head_dim))
        _, table, lens = self._rows_of(slots)
        ws = self._serving("shared", int(lib.lara_decode_shared_workspace_bytes(len(slots), q.shape[1],
                                                                                self.n_kv_heads, self.head_dim)))
        shared = self.shared_pages(slots) if len(slots) > 1 else 0
        return gqa_decode_shared(q, self.k_pages, self.v_pages, table, lens, shared, scale=scale, workspace=ws)

    def decode_scored(self, q, slots=None, scale=None):
        """:meth:`decode` that adds to each slot's weight what attention it gets (a cache with ``scored=True``)."""
        self._need_weights("decode_scored")
        slots = self._slots(slots)
        _check_words("q", q, (len(slots), q.shape[1], self.head_dim))
        self._own_pages(slots, "decode_scored")
        _, table, lens = self._rows_of(slots)
        ws = self._serving("scored", int(lib.lara_decode_scored_workspace_bytes(
            len(slots), q.shape[1], self.n_kv_heads, self.head_dim, self.page_size, self.pages_per_seq,
            self.num_pages)))
        return gqa_decode_scored(q, self.k_pages, self.v_pages, self.weights, table, lens, scale=scale, workspace=ws)

    def evict(self, keep: int, slots=None, *, first: int = 0, last: int = 0, sources=None) -> None:
        """:func:`kv_evict` of the given slots (default: all active); pages behind ``keep`` are free again.

        A sequence that was cut has its rows out of order: it decodes as before, but is nobody's prefix.
        """
        self._need_weights("evict")
        slots = self._slots(slots)
        self._own_pages(slots, "evict")
        _, table, lens = self._rows_of(slots)
        ws = self._serving("evict", int(lib.lara_kv_evict_workspace_bytes(len(slots), self.n_kv_heads,
                                                                          max(int(keep), 1))))
        kv_evict(self.k_pages, self.v_pages, self.weights, table, lens, keep, first=first, last=last,
                 sources=sources, workspace=ws)
        cut = slots[self._lens[slots] > keep]
        self._lens[cut] = keep
        self._cut[cut] = True
        for slot in cut:
            for j in range(-(-int(self._lens[slot]) // self.page_size), self.pages_per_seq):
                if self._table[slot, j] >= 0:
                    self._release(int(self._table[slot, j]))
                    self._table[slot, j] = -1
        if len(cut):
            self._sync_rows(cut)

    def status(self) -> int:
        """Device status bits of the last appends, decodes and evictions (read and cleared)."""
        from .ops import workspace_status

        bits = workspace_status(self._status)
        for ws in (self._ws, *self._serving_ws.values()):
            if ws is not None:
                bits |= workspace_status(ws)
        return bits

    # ------------------------------------------------------------ contents
    def gather(self, slot: int):
        """(k, v) ``[Hkv, len, D]`` of one sequence, read through its block table."""
        n = int(self._lens[slot])
        pages = self._table[slot, : (n + self.page_size - 1) // self.page_size]
        idx = torch.as_tensor(pages.astype(np.int64), device=self.device)
        k = self.k_pages.index_select(0, idx).permute(1, 0, 2, 3).reshape(self.n_kv_heads, -1, self.head_dim)
        v = self.v_pages.index_select(0, idx).permute(1, 0, 2, 3).reshape(self.n_kv_heads, -1, self.head_dim)
        return k[:, :n].contiguous(), v[:, :n].contiguous()

    def save(self, path, slots=None) -> None:
        slots = self._slots(slots)
        T = max(int(self._lens[slots].max()), 1)
        k = np.zeros((len(slots), self.n_kv_heads, T, self.head_dim), np.uint16)
        v = np.zeros_like(k)
        for i, s in enumerate(slots):
            ks, vs = self.gather(int(s))
            n = ks.shape[1]
            k[i, :, :n] = ks.view(torch.int16).cpu().numpy().view(np.uint16)
            v[i, :, :n] = vs.view(torch.int16).cpu().numpy().view(np.uint16)
        kvfile.save(path, k, v, self._lens[slots], self._cut[slots])

    def load(self, path) -> list[int]:
        """Create one new sequence per stored sequence; returns their slots."""
        k, v, lens, cut = kvfile.load_any(path)
        if k.shape[1] != self.n_kv_heads or k.shape[3] != self.head_dim:
            raise ValueError(f"{path}: geometry {k.shape} does not match this cache")
        slots = []
        for i in range(k.shape[0]):
            s = self.new_sequence()
            slots.append(s)
            n = int(lens[i])
            if n:
                t = lambda a: torch.from_numpy(np.ascontiguousarray(a[None, :, :n]).view(np.int16)).to(  # noqa: E731
                    self.device).view(torch.bfloat16)
                self.append(t(k[i]), t(v[i]), slots=[s])
            self._cut[s] = cut[i]
        return slots
