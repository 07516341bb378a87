"""Paged fp8 + fp8-residual cache in which sequences share the pages of a common prompt.

``PagedFP8Fp8Cache`` gives every sequence its own pages and all of them one length.  Here a :class:`PageTable`
hands pages out: ``fork`` lets a new sequence begin on the pages of a prompt, the first write into a shared open page
copies it, ``free`` gives the pages of an ended sequence back, ``compact`` moves the pages in use to the front.  One
table serves all layers.  A decode step appends every sequence's token at its own position and attends to shared
pages once per group of sequences (every token counts; nothing is pruned).

Sequences have numbers ``0 .. max_seqs - 1``.  ``activate`` names those that the next model calls are about, in batch
order; sequences that were forked from one another should be next to each other in it, since a group is a stretch of
the batch.  Lengths are known on the host as well, so that only ``check()`` waits for the device; for that reason model calls
cannot be captured in a graph.  A model call that runs out of pages writes no token; ``check()`` finds it and takes lengths
and shared pages from the device again.

The reference has no counterpart (ffa-fp8fp8/e2e/fp8fp8_cache.py appends a batch of one length with ``torch.cat``).
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
import torch

from ...pages import PageTable, append_ragged_fp8fp8, upload
from ..attn_kernel.attn_kernel_shared_prefix_fp8fp8 import SharedPrefixWorkspace, attn_forward_decode_shared_prefix_fp8fp8
from .fp8fp8_cache import PAGE, resolve_fp8_dtype


def _stretches(common: np.ndarray) -> tuple[list[int], list[int]]:
    """Cut a batch into groups.  ``common[i]``: pages that sequences i and i + 1 share.  The first sequence of every group
    and the batch's end, and the pages that all of a group have in common: the cut that saves the most reading of pages, a
    group of n with m pages in common saving (n - 1) * m.  One group for each stretch that shares the same number
    throughout (samples of one prompt); a stretch of forks of forks is cut by dynamic programming."""
    n = len(common) + 1
    cuts = [0, *(np.flatnonzero(common == 0) + 1).tolist(), n]
    start, pages = [], []
    for a, b in zip(cuts[:-1], cuts[1:]):
        c = common[a:b - 1]
        if b - a == 1 or (c == c[0]).all():
            start.append(a)
            pages.append(int(c[0]) if b - a > 1 else 0)
            continue
        best, first = np.zeros(b - a + 1, dtype=np.int64), np.zeros(b - a + 1, dtype=np.int64)
        for j in range(1, b - a + 1):                         # best cut of the first j; its last group is first[j] .. j - 1
            least = np.minimum.accumulate(np.append(c[:j - 1], 0)[::-1][1:])[::-1] if j > 1 else c[:0]
            saved = best[:j] + np.append(least * np.arange(j - 1, 0, -1), 0)
            first[j] = saved.argmax()
            best[j] = saved[first[j]]
        groups = []
        while b > a:
            i = a + int(first[b - a])
            groups.append((i, int(common[i:b - 1].min()) if b - i > 1 else 0))
            b = i
        for i, m in reversed(groups):
            start.append(i)
            pages.append(m)
    return [*start, n], pages


class SharedPrefixFP8Fp8Cache:
    def __init__(self, max_seqs: int, num_kv_heads: int, max_seq_len: int, *, num_layers: int, n_pages: Optional[int] = None,
                 head_dim: int = 128, fp8_dtype: Optional[torch.dtype] = None, dtype: torch.dtype = torch.bfloat16,
                 device="cuda"):
        if head_dim != 128:
            raise ValueError(f"this build supports head_dim 128, got {head_dim}")
        if num_layers <= 0:
            raise ValueError(f"num_layers must be positive, got {num_layers}")
        if num_kv_heads <= 0:
            raise ValueError(f"num_kv_heads must be positive, got {num_kv_heads}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
        self.num_kv_heads, self.head_dim, self.num_layers, self.dtype = num_kv_heads, head_dim, num_layers, dtype
        self.fp8_dtype = fp8_dtype or resolve_fp8_dtype(device)
        if self.fp8_dtype not in (torch.float8_e4m3fn, torch.float8_e5m2):
            raise ValueError(f"fp8_dtype must be float8_e4m3fn or float8_e5m2, got {self.fp8_dtype}")
        pages_per_seq = -(-max_seq_len // PAGE)
        self.max_seq_len = pages_per_seq * PAGE
        shape = (n_pages or max_seqs * pages_per_seq, PAGE, num_kv_heads, head_dim)
        self.key_base = [torch.zeros(shape, dtype=self.fp8_dtype, device=device) for _ in range(num_layers)]
        self.key_residual = [torch.zeros(shape, dtype=self.fp8_dtype, device=device) for _ in range(num_layers)]
        self.value = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.table = PageTable(shape[0], max_seqs, pages_per_seq, device=device,
                               pools=[*self.key_base, *self.key_residual, *self.value])
        self.device = self.table.device
        self.lengths = [0] * max_seqs
        # what is in every page of every sequence: equal numbers in a column are one page, a page gets a new number when
        # it is written to.  Known up to so many tokens of a sequence, what was written since is its own (`_note`)
        self._contents = np.full((max_seqs, pages_per_seq), -1, dtype=np.int64)
        self._known = [0] * max_seqs
        self._next_content = 0
        self._groups: Optional[tuple[torch.Tensor, torch.Tensor]] = None
        self._seqs: list[int] = []
        self._new = 0
        self._workspace: Optional[SharedPrefixWorkspace] = None
        self._gave_up = torch.zeros(1, dtype=torch.int32, device=self.device)         # of workspaces before the present one

    # ---- sequences ---------------------------------------------------------------------------------------
    def _numbers(self, seqs: Sequence[int]) -> list[int]:
        seqs = [int(s) for s in seqs]
        if any(s < 0 or s >= len(self.lengths) for s in seqs) or len(set(seqs)) != len(seqs):
            raise ValueError(f"sequence numbers must differ and be 0 to {len(self.lengths) - 1}, got {seqs}")
        return seqs

    def activate(self, seqs: Sequence[int]) -> None:
        """The sequences of the next model calls, in batch order."""
        seqs = self._numbers(seqs)
        if not seqs:
            raise ValueError("activate at least one sequence")
        self._seqs = seqs
        self._rows = upload(seqs, self.device)
        self._slice = slice(seqs[0], seqs[0] + len(seqs)) if seqs == list(range(seqs[0], seqs[0] + len(seqs))) else None
        self._new, self._groups = 0, None

    @property
    def active(self) -> tuple[int, ...]:
        """The sequences that ``activate`` named."""
        return tuple(self._seqs)

    def _written(self, seqs: list[int], first: np.ndarray, end: np.ndarray) -> None:
        """Columns first[i] .. end[i] - 1 of seqs[i] get contents of their own."""
        n = end - first
        at = np.arange(n.sum())
        self._contents[np.repeat(seqs, n), at - np.repeat(n.cumsum() - n - first, n)] = self._next_content + at
        self._next_content += len(at)

    def _note(self, seqs: Sequence[int]) -> None:
        """Give a number to what the sequences wrote since it was last asked for."""
        grown = [s for s in seqs if self.lengths[s] > self._known[s]]
        if grown:
            of = lambda x: np.array([x[s] for s in grown], dtype=np.int64)
            self._written(grown, of(self._known) // PAGE, -(-of(self.lengths) // PAGE))
            for s in grown:
                self._known[s] = self.lengths[s]

    def _group(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Stretches of the batch whose sequences have their first full pages in common, and how many: asked for by the next
        step, so that several changes in a row cost it once."""
        if self._groups is None:
            self._note(self._seqs)
            lens = np.array([self.lengths[s] for s in self._seqs], dtype=np.int64) // PAGE
            cols = max(1, int(lens.max()))
            rows = self._contents[self._seqs, :cols]
            same = (rows[1:] == rows[:-1]) & (np.arange(cols) < np.minimum(lens[1:], lens[:-1])[:, None])
            start, pages = _stretches(np.where(same.all(1), cols, same.argmin(1)))  # the first page that is not the next one's too
            both = upload([*start, *pages], self.device)
            self._groups = both[:len(start)], both[len(start):]
        return self._groups

    @property
    def _group_start(self) -> torch.Tensor:
        return self._group()[0]

    @property
    def _prefix_pages(self) -> torch.Tensor:
        return self._group()[1]

    def fork(self, parents: Sequence[int], children: Sequence[int]) -> None:
        """Let the empty sequences ``children[i]`` begin with the tokens of ``parents[i]``, on the same pages."""
        children, parents = self._numbers(children), [int(p) for p in parents]
        if len(parents) != len(children) or any(p < 0 or p >= len(self.lengths) or p in children for p in parents):
            raise ValueError("fork takes one parent for each child, and no child among the parents")
        if any(self.lengths[c] for c in children):
            raise ValueError("the children must be empty: free them first")
        self.table.fork(parents, children)
        self._note(dict.fromkeys(parents))
        for p, c in zip(parents, children):
            held = -(-self.lengths[p] // PAGE)
            self._contents[c, :held] = self._contents[p, :held]
            self.lengths[c] = self._known[c] = self.lengths[p]
        self._groups = None

    def truncate(self, seqs: Sequence[int], new_lens: Sequence[int]) -> None:
        """Drop the tokens past ``new_lens`` (rejected drafts)."""
        seqs, new_lens = self._numbers(seqs), [int(n) for n in new_lens]
        if len(new_lens) != len(seqs) or any(n < 0 for n in new_lens):
            raise ValueError("truncate takes one length for each sequence")
        self.table.truncate(seqs, new_lens)
        alone = []
        for s, n in zip(seqs, new_lens):
            if n < self._known[s]:
                # cut back into pages that others hold too it goes on by itself: kept with them, it would hold down what
                # all of them read once
                full = n // PAGE
                if 0 < n and full < self._known[s] // PAGE and np.count_nonzero(
                        (self._contents[:, full] == self._contents[s, full]) & (np.array(self._known) // PAGE > full)) > 1:
                    alone.append(s)
                self._known[s] = n
            self.lengths[s] = min(self.lengths[s], n)
        if alone:
            self._written(alone, np.zeros(len(alone), dtype=np.int64), np.array([-(-self.lengths[s] // PAGE) for s in alone]))
        self._new, self._groups = 0, None

    def free(self, seqs: Sequence[int]) -> None:
        """End the sequences and give their pages back."""
        seqs = list(seqs)
        self.truncate(seqs, [0] * len(seqs))

    def compact(self) -> None:
        """Move the pages in use to the front of the pools."""
        self.table.compact()
        self._new = 0

    def check(self) -> None:
        """Raise if a call since the last check ran out of pages (waits for the device).  Lengths, and which pages sequences
        share, are then taken from the device, and work goes on from there; what model calls returned since the one that
        ran out is not to be used.  Raises too if a bounded wait inside the attention gave up: outputs are NaN then."""
        try:
            self.table.check()
        except RuntimeError:
            self.lengths = self.table.seq_lens.tolist()
            # a page's number says what is in it; the numbers of pages that are written to from here on are others
            rows = self.table.block_table.cpu().numpy().astype(np.int64)
            held = np.arange(rows.shape[1]) < -(-np.array(self.lengths)[:, None] // PAGE)
            self._contents = np.where(held & (rows >= 0), rows + self._next_content, -1)
            self._next_content += self.table.n_pages
            self._known, self._new, self._groups = list(self.lengths), 0, None
            raise
        if self._workspace is not None:
            self._gave_up |= self._workspace.status_word
            self._workspace.status_word.zero_()
        if int(self._gave_up.item()):
            self._gave_up.zero_()
            raise RuntimeError("shared-prefix decode: a wait inside a kernel gave up, outputs since the last check may be NaN")

    def get_seq_length(self, layer_idx: int = 0) -> int:
        """Tokens of the longest active sequence."""
        return max((self.lengths[s] for s in self._seqs), default=0)

    # ---- a model call --------------------------------------------------------------------------------------
    def extend(self, n_new: int) -> None:
        """Room for ``n_new`` more tokens of every active sequence; once per model call, before its layers."""
        self._not_captured()
        if not self._seqs:
            raise RuntimeError("activate the sequences first")
        if n_new <= 0 or max(self.lengths[s] for s in self._seqs) + n_new > self.max_seq_len:
            raise ValueError(f"cache capacity {self.max_seq_len} exceeded ({self.get_seq_length()} + {n_new})")
        at = self._slice if self._slice is not None else self._rows
        self._positions = self.table.seq_lens[at].clone() if self._slice is not None else self.table.seq_lens[at]
        self.table.extend(self._rows, n_new)
        self._new = n_new
        for s in self._seqs:
            self.lengths[s] += n_new
        self._bt, self._lens = self.table.block_table[at], self.table.seq_lens[at]
        self._counts = self._lens - self._positions   # 0 where there were no pages: nothing is written then

    def _not_captured(self) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a SharedPrefixFP8Fp8Cache follows its sequences on the host: a graph would replay the lengths and table "
                               "of the step that was captured.  PageTable, append and decode can be captured")

    def _extended(self) -> None:
        self._not_captured()
        if self._new == 0:
            raise RuntimeError("extend first: the active sequences or their pages changed since")

    def positions(self) -> torch.Tensor:
        """Positions ``[B, n_new]`` of the tokens of this model call."""
        self._extended()
        return self._positions[:, None] + torch.arange(self._new, dtype=torch.int32, device=self.device)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int) -> None:
        """Write the new tokens' post-RoPE keys (quantised) and values ``[B, n_new, HKV, 128]``."""
        self._extended()
        if key_states.shape != (len(self._seqs), self._new, self.num_kv_heads, self.head_dim) or value_states.shape != key_states.shape:
            raise ValueError(f"expected [B={len(self._seqs)}, {self._new}, HKV={self.num_kv_heads}, {self.head_dim}] keys and values")
        append_ragged_fp8fp8(key_states.to(self.dtype), value_states.to(self.dtype), self.key_base[layer_idx],
                             self.key_residual[layer_idx], self.value[layer_idx], self._bt, self._positions, self._counts)

    def decode(self, q: torch.Tensor, layer_idx: int, scale: Optional[float] = None) -> torch.Tensor:
        """Attention of ``q [B, 1, HQ, 128]`` over all tokens of its sequence -> ``[B, HQ, 128]``, a buffer that the next
        call overwrites."""
        self._extended()
        ws = self._workspace
        if ws is None or not ws.matches(q.shape[0], q.shape[2], self.num_kv_heads, q.device, q.dtype):
            if ws is not None:
                self._gave_up |= ws.status_word
            ws = self._workspace = SharedPrefixWorkspace(q.shape[0], q.shape[2], self.num_kv_heads, q.device, q.dtype)
        return attn_forward_decode_shared_prefix_fp8fp8(
            q, self.key_base[layer_idx], self.value[layer_idx], k_residual=self.key_residual[layer_idx], block_table=self._bt,
            seq_lens=self._lens, group_start=self._group_start, prefix_pages=self._prefix_pages, scale=scale, workspace=ws)
