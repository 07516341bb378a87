"""Pages of a cache that several sequences share, and appends at each sequence's own position.

``PageTable`` keeps block table, lengths and reference counts of up to ``max_seqs`` sequences on the device and
changes them there (``ffa_pages_*``): ``fork`` lets a new sequence hold the pages of another one, ``extend`` makes
room for new tokens and gives a sequence a page of its own before it writes into a shared one, ``truncate`` and
``free`` give pages back, ``compact`` moves the live pages to the front of the pools.  Nothing here synchronises or
allocates on the device when the arguments are device tensors, so the calls may be captured in a CUDA graph.

The reference has no counterpart: its cache is one tensor per layer that grows by ``torch.cat``
(ffa-fp8fp8/e2e/fp8fp8_cache.py:74-121).
"""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from . import _lib

PAGE = 64
MAX_SEQS = 65536
BAD_ARGUMENT, NO_SPACE = 1, 2           # bits of PageTable.status()

Numbers = Union[torch.Tensor, Sequence[int]]


def upload(numbers: Sequence[int], device: torch.device) -> torch.Tensor:
    """An int32 vector on the device, without waiting for what the stream still has to do: through pinned memory, which
    the allocator keeps until the copy is over."""
    if torch.cuda.is_current_stream_capturing():
        raise ValueError("a graph would keep the numbers of a list: give a device tensor while a stream is captured")
    return torch.tensor(list(numbers), dtype=torch.int32).pin_memory().to(device, non_blocking=True)


class PageTable:
    """Block table ``[max_seqs, pages_per_seq]``, lengths and reference counts of the pages of ``pools``.

    ``pools``: the tensors ``[n_pages, 64, ...]`` whose page ``p`` belongs to cache page ``p`` (base, residual and V
    of every layer that shares the table); ``extend`` and ``compact`` copy pages in all of them.  Lists of sequence
    numbers and lengths are int32 device tensors or Python sequences (which are copied to the device first, without
    waiting for it).

    A call that cannot be carried out changes nothing and sets a bit of the status word: ``BAD_ARGUMENT`` or
    ``NO_SPACE``.  ``check()`` raises for it.  Calls on one table must not overlap on the GPU, nor with the table's
    own making (which zeroes its scratch): keep them on one stream, or order the streams."""

    def __init__(self, n_pages: int, max_seqs: int, pages_per_seq: int, *, pools: Sequence[torch.Tensor] = (),
                 device="cuda"):
        if n_pages <= 0 or max_seqs <= 0 or pages_per_seq <= 0:
            raise ValueError("n_pages, max_seqs and pages_per_seq must be positive")
        device = torch.device(device)
        self._setup(torch.full((max_seqs, pages_per_seq), -1, dtype=torch.int32, device=device),
                    torch.zeros(max_seqs, dtype=torch.int32, device=device),
                    torch.zeros(n_pages, dtype=torch.int32, device=device), pools)

    @classmethod
    def wrap(cls, block_table: torch.Tensor, seq_lens: torch.Tensor, refcount: torch.Tensor, *,
             pools: Sequence[torch.Tensor] = ()) -> "PageTable":
        """A table on state that exists already: ``block_table [max_seqs, pages_per_seq]`` (-1 where a sequence has no
        page), ``seq_lens [max_seqs]``, ``refcount [n_pages]``, all int32 device tensors, used in place."""
        self = cls.__new__(cls)
        self._setup(block_table, seq_lens, refcount, pools)
        return self

    def _setup(self, block_table, seq_lens, refcount, pools) -> None:
        for name, t, dim in (("block_table", block_table, 2), ("seq_lens", seq_lens, 1), ("refcount", refcount, 1)):
            if t.dtype != torch.int32 or t.dim() != dim or t.numel() == 0:
                raise ValueError(f"{name} must be a non-empty int32 tensor with {dim} dimension{'s' * (dim > 1)}")
            if not t.is_cuda:
                raise ValueError(f"{name} must be a CUDA tensor (this build has no CPU path)")
            if t.stride(-1) != 1 or t.device != block_table.device:
                raise ValueError(f"{name} must have unit stride in its last dimension and be on block_table's device")
        if seq_lens.shape[0] != block_table.shape[0]:
            raise ValueError("seq_lens must have one entry for each row of block_table")
        if block_table.shape[0] > MAX_SEQS:
            raise ValueError(f"a table holds at most {MAX_SEQS} sequences, got {block_table.shape[0]}")
        if block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]:
            raise ValueError("the rows of block_table must not overlap")
        self.block_table, self.seq_lens, self.refcount = block_table, seq_lens, refcount
        self.device = block_table.device
        self.max_seqs, self.pages_per_seq = block_table.shape
        self.n_pages = refcount.shape[0]
        self.pools = list(pools)
        for p in self.pools:
            if p.dim() < 3 or p.shape[0] != self.n_pages or p.shape[1] != PAGE:
                raise ValueError(f"pools must be [n_pages, 64, ...] with n_pages = {self.n_pages}, got {tuple(p.shape)}")
            if not p.is_contiguous() or p.device != self.device:
                raise ValueError("pools must be contiguous and on block_table's device")
            if p[0, 0].numel() * p.element_size() % 16 or p.data_ptr() % 16:
                raise ValueError("a token of a pool must take a multiple of 16 bytes, and the pool start on 16 bytes")
        token = [p[0, 0].numel() * p.element_size() for p in self.pools]
        # 62 zeroed ints ahead of the scratch keep the status word on a line of its own
        n_scratch = _lib.lib().ffa_pages_scratch_bytes(self.n_pages, self.max_seqs)
        self._scratch = torch.zeros(256 + n_scratch, dtype=torch.uint8, device=self.device)
        self.status_word = self._scratch[:4].view(torch.int32)
        self._bases = torch.tensor([p.data_ptr() for p in self.pools], dtype=torch.int64, device=self.device)
        self._token_bytes = torch.tensor(token, dtype=torch.int32, device=self.device)
        a = self._table = _lib.FfaPageTable()
        a.n_pages, a.max_seqs, a.cols = self.n_pages, self.max_seqs, self.pages_per_seq
        a.bt_stride = block_table.stride(0) if self.max_seqs > 1 else self.pages_per_seq
        a.block_table, a.seq_lens, a.refcount = block_table.data_ptr(), seq_lens.data_ptr(), refcount.data_ptr()
        a.status, a.scratch, a.scratch_bytes = self.status_word.data_ptr(), self._scratch.data_ptr() + 256, n_scratch
        b = self._pool_args = _lib.FfaPagePools()
        b.n_pools, b.max_token_bytes = len(self.pools), max(token, default=0)
        b.bases, b.token_bytes = self._bases.data_ptr(), self._token_bytes.data_ptr()

    def _list(self, x: Numbers, name: str) -> torch.Tensor:
        if not isinstance(x, torch.Tensor):
            x = upload(x, self.device)
        if x.dtype != torch.int32 or x.dim() != 1 or x.device != self.device or not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector on {self.device}")
        if x.numel() > self.max_seqs:
            raise ValueError(f"{name} lists {x.numel()} sequences, the table has {self.max_seqs}")
        return x

    def _pair(self, seqs: Numbers, name: str, values, value_name: str):
        if not isinstance(seqs, torch.Tensor) and not isinstance(values, (torch.Tensor, int)):
            seqs, values = list(seqs), list(values)
            both = upload([*seqs, *values], self.device)      # one copy for two lists
            seqs, values = both[:len(seqs)], both[len(seqs):]
        seqs = self._list(seqs, name)
        if isinstance(values, int):
            values = torch.full_like(seqs, values)
        values = self._list(values, value_name)
        n = seqs.numel()
        if values.numel() != n:
            raise ValueError(f"{name} and {value_name} must have the same length")
        return seqs, values, n

    def truncate(self, seqs: Numbers, new_lens: Union[Numbers, int]) -> None:
        """Shorten the sequences to ``new_lens`` tokens; a length above the present one changes nothing.  A sequence
        listed twice gets the smaller length."""
        seqs, new_lens, n = self._pair(seqs, "seqs", new_lens, "new_lens")
        if n:
            _lib.enqueue(self.device, _lib.lib().ffa_pages_truncate, "ffa_pages_truncate", self._table, seqs.data_ptr(),
                         new_lens.data_ptr(), n)

    def free(self, seqs: Numbers) -> None:
        """End the sequences: ``truncate`` to zero tokens."""
        self.truncate(seqs, 0)

    def fork(self, parents: Numbers, children: Numbers) -> None:
        """Let the empty sequences ``children[i]`` begin with all tokens of ``parents[i]``, on the same pages.  No
        child may be listed twice or be a parent in the same call."""
        parents, children, n = self._pair(parents, "parents", children, "children")
        if n:
            _lib.enqueue(self.device, _lib.lib().ffa_pages_fork, "ffa_pages_fork", self._table, parents.data_ptr(),
                         children.data_ptr(), n)

    def extend(self, seqs: Numbers, n_new: Union[Numbers, int]) -> None:
        """Make room for ``n_new`` more tokens in each sequence (none listed twice) and add them to ``seq_lens``; the
        caller then writes the tokens.  A partly filled last page that other sequences hold too is copied to a page
        of its own first, in every pool.  All or nothing: without enough free pages no sequence changes."""
        seqs, n_new, n = self._pair(seqs, "seqs", n_new, "n_new")
        if n:
            _lib.enqueue(self.device, _lib.lib().ffa_pages_extend, "ffa_pages_extend", self._table, self._pool_args,
                         seqs.data_ptr(), n_new.data_ptr(), n)

    def compact(self, *, block_table_out: Optional[torch.Tensor] = None, refcount_out: Optional[torch.Tensor] = None) -> None:
        """Move live pages into the free ones with lower numbers, in every pool, until the live pages are the first
        ones; block table and reference counts follow.  With ``block_table_out`` and ``refcount_out`` the new state
        is written there and the table itself stays as it is: it remains valid until the next ``extend``, since the
        moved pages' old contents are not touched."""
        if (block_table_out is None) != (refcount_out is None):
            raise ValueError("give both block_table_out and refcount_out, or neither")
        if block_table_out is None:
            block_table_out, refcount_out = self.block_table, self.refcount
        for name, t, like in (("block_table_out", block_table_out, self.block_table), ("refcount_out", refcount_out, self.refcount)):
            if t.dtype != torch.int32 or t.shape != like.shape or t.stride() != like.stride() or t.device != self.device:
                raise ValueError(f"{name} must be int32 with the shape, strides and device of the table's own")
        _lib.enqueue(self.device, _lib.lib().ffa_pages_compact, "ffa_pages_compact", self._table, self._pool_args,
                     block_table_out.data_ptr(), refcount_out.data_ptr())

    # ---- for the host (these synchronise) --------------------------------------------------------------
    def status(self) -> int:
        """Status word: 0, or the bits of the calls since the last ``check()`` that changed nothing."""
        return int(self.status_word.item())

    def check(self) -> None:
        """Raise for the calls since the last check that could not be carried out."""
        bits = self.status()
        if bits:
            self.status_word.zero_()
            raise RuntimeError("page table: " + " and ".join(
                text for bit, text in ((BAD_ARGUMENT, "a call with sequence numbers or lengths that are not allowed"),
                                       (NO_SPACE, "an extend without enough free pages")) if bits & bit)
                + " changed nothing")

    def free_pages(self) -> int:
        return int((self.refcount == 0).sum().item())


def append_ragged_fp8fp8(k: torch.Tensor, v: torch.Tensor, base_pool: torch.Tensor, residual_pool: torch.Tensor,
                         v_pool: torch.Tensor, block_table: torch.Tensor, positions: torch.Tensor,
                         counts: Optional[torch.Tensor] = None) -> None:
    """Quantise ``k [B, T_new, HKV, 128]`` (post-RoPE) to fp8 base and residual and write both, and ``v``, at
    positions ``positions[b] ..`` of sequence b's row of ``block_table [B, pages]`` in the pools
    ``[n_pages, 64, HKV, 128]``.  ``counts [B]``: tokens of each sequence that count, the rest of T_new is padding
    and is not written.  Nothing is written for positions without a page (an entry of -1, or past the table).  The
    codes are those of ``quantize_k_fp8_fp8_residual``."""
    shape = k.shape
    if not k.is_cuda or len(shape) != 4 or shape[3] != 128:
        raise ValueError(f"k must be a CUDA tensor [B, T, HKV, 128], got {tuple(shape)} on {k.device}")
    dtype, device, (B, T, HKV, _), pool_shape, pool_dtype = k.dtype, k.device, shape, base_pool.shape, base_pool.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"k must be float16 or bfloat16, got {dtype}")
    if v.shape != shape or v.dtype != dtype:
        raise ValueError("v must have the shape and type of k")
    if len(pool_shape) != 4 or pool_shape[1:] != (PAGE, HKV, 128):
        raise ValueError(f"pools must be [n_pages, 64, {HKV}, 128], got {tuple(pool_shape)}")
    fp8 = _lib.fp8_code(pool_dtype)
    if residual_pool.shape != pool_shape or residual_pool.dtype != pool_dtype:
        raise ValueError("residual_pool must have the shape and type of base_pool")
    if v_pool.shape != pool_shape or v_pool.dtype != dtype:
        raise ValueError("v_pool must have the shape of base_pool and v's type")
    table_shape = block_table.shape
    if block_table.dtype != torch.int32 or len(table_shape) != 2 or table_shape[0] != B:
        raise ValueError("block_table must be an int32 tensor [B, pages]")
    cols, table_stride = table_shape[1], block_table.stride(0) if B > 1 else table_shape[1]
    if block_table.stride(1) != 1 or table_stride < cols:
        raise ValueError("block_table must have unit stride in its last dimension and rows that do not overlap")
    for name, t in (("positions", positions), ("counts", counts)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (B,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous int32 vector of B = {B} entries")
    if not (base_pool.is_contiguous() and residual_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("pools must be contiguous")
    for t in (v, base_pool, residual_pool, v_pool, block_table, positions, counts):
        if t is not None and t.device != device:
            raise ValueError(f"all tensors must be on {device}")
    if B == 0 or T == 0:
        return
    k, v = k.contiguous(), v.contiguous()
    _lib.enqueue(device, _lib.lib().ffa_cache_append_ragged, "ffa_cache_append_ragged", k.data_ptr(), v.data_ptr(),
                 _lib.float_code(dtype), B, T, HKV, fp8, base_pool.data_ptr(), residual_pool.data_ptr(), v_pool.data_ptr(),
                 pool_shape[0], block_table.data_ptr(), table_stride, cols, positions.data_ptr(), _lib.ptr(counts))
