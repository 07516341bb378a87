"""fp8 K + fp8 residual decode attention for a batch whose sequences share leading pages.

Several samples of one prompt (``PageTable.fork``) hold the prompt's pages together.  ``attn_forward_decode_fp8fp8``
on such a batch would read the prompt once per sequence; here the shared pages are read once for all sequences of a
group and the own pages of each sequence follow, in one softmax.  Every token counts: pruning would save no bytes on a
page that some other sequence of the group keeps.  The reference has no counterpart."""
from __future__ import annotations

import math

import torch

from ... import _lib

PAGE = 64


class SharedPrefixWorkspace:
    """Output and scratch of the shared-prefix decode, for one batch size and head layout.  One call at a time may
    use it (two captured graphs that may run at the same time need one each)."""

    def __init__(self, B: int, HQ: int, HKV: int, device, dtype):
        self.B, self.HQ, self.HKV, self.device, self.dtype = int(B), int(HQ), int(HKV), torch.device(device), dtype
        nbytes = _lib.lib().ffa_shared_prefix_workspace_bytes(self.B, self.HQ, self.HKV)
        if nbytes == 0:
            raise ValueError(f"no workspace for B={B}, HQ={HQ}, HKV={HKV}: B must be 1 to 4096, HQ a multiple of HKV")
        self.scratch = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self.scratch[:512].zero_()
        self.o = torch.empty((self.B, self.HQ, 128), dtype=dtype, device=self.device)

    def matches(self, B: int, HQ: int, HKV: int, device, dtype) -> bool:
        return (self.B, self.HQ, self.HKV, self.o.device, self.dtype) == (B, HQ, HKV, device, dtype)

    def status(self) -> int:
        """Device status word (synchronises): 0 = ok, 1 = a bounded wait inside a kernel gave up (the affected
        outputs are NaN)."""
        return int(self.scratch[256:260].view(torch.int32).item())


def allocate_shared_prefix_workspace(q: torch.Tensor, v: torch.Tensor) -> SharedPrefixWorkspace:
    """Workspace for calls with ``q [B, 1, HQ, 128]`` and the pool ``v [n_pages, 64, HKV, 128]``."""
    return SharedPrefixWorkspace(q.shape[0], q.shape[2], v.shape[2], q.device, q.dtype)


def attn_forward_decode_shared_prefix_fp8fp8(
    q: torch.Tensor,              # [B, 1, HQ, 128]
    k_fp8: torch.Tensor,          # [n_pages, 64, HKV, 128] fp8
    v: torch.Tensor,              # [n_pages, 64, HKV, 128] float16 / bfloat16
    *,
    block_table: torch.Tensor,    # [B, pages] int32
    seq_lens: torch.Tensor,       # [B] int32
    group_start: torch.Tensor,    # [n_groups + 1] int32, ascending from 0 to B
    prefix_pages: torch.Tensor,   # [n_groups] int32
    k_residual: torch.Tensor | None = None,
    use_fp8_residual: bool = True,
    scale: float | None = None,
    workspace: SharedPrefixWorkspace | None = None,
    out: torch.Tensor | None = None,
    partial_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of one query token per sequence over all its cached tokens -> ``[B, HQ, 128]``.

    Sequences ``group_start[g] .. group_start[g+1] - 1`` share their first ``prefix_pages[g]`` pages: those are taken
    from the table row of the group's first sequence.  ``seq_lens`` counts all tokens of a sequence, shared ones
    included; a sequence of length 0 gives zeros.  Lengths and groups are read on the device when the kernels run.
    ``partial_out [B, HQ, 129]`` (fp32) also receives the normalised output and the base-2 log-sum-exp."""
    if not (q.is_cuda and k_fp8.is_cuda and v.is_cuda):
        raise ValueError("q, K and V must be CUDA tensors (this build has no CPU path)")
    if q.dim() != 4 or q.shape[1] != 1 or q.shape[3] != 128:
        raise ValueError(f"q must be [B, 1, HQ, 128], got {tuple(q.shape)}")
    B, _, HQ, _ = q.shape
    if k_fp8.dim() != 4 or k_fp8.shape[1] != PAGE or k_fp8.shape[3] != 128 or v.shape != k_fp8.shape:
        raise ValueError(f"K and V must be paged pools [n_pages, 64, HKV, 128], got {tuple(k_fp8.shape)} and {tuple(v.shape)}")
    n_pages, _, HKV, _ = k_fp8.shape
    if HKV == 0 or HQ % HKV != 0:
        raise ValueError(f"HQ ({HQ}) must be divisible by HKV ({HKV}) for GQA")
    if HQ // HKV > 8:
        raise ValueError(f"this build supports GQA group sizes up to 8, got {HQ // HKV}")
    fp8 = _lib.fp8_code(k_fp8.dtype)
    v_code = _lib.float_code(v.dtype)
    if v_code == _lib.F32:
        raise ValueError("v must be float16 or bfloat16")
    if use_fp8_residual:
        if k_residual is None:
            raise ValueError("use_fp8_residual=True requires k_residual")
        if k_residual.shape != k_fp8.shape or k_residual.dtype != k_fp8.dtype:
            raise ValueError("k_residual must have the shape and fp8 encoding of k_fp8")
    else:
        k_residual = None
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B or block_table.shape[1] == 0 \
            or block_table.stride(1) != 1 or (B > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError("block_table must be an int32 tensor [B, pages] with unit stride in its last dimension")
    NG = prefix_pages.shape[0] if prefix_pages.dim() == 1 else 0
    for name, t, n in (("seq_lens", seq_lens, B), ("group_start", group_start, NG + 1), ("prefix_pages", prefix_pages, NG)):
        if t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector of {n} entries")
    if not 1 <= NG <= B:
        raise ValueError(f"there must be 1 to B = {B} groups, got {NG}")
    for name, t in (("q", q), ("k_fp8", k_fp8), ("v", v), ("k_residual", k_residual)):
        if t is not None and not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    for t in (k_fp8, v, k_residual, block_table, seq_lens, group_start, prefix_pages, out, partial_out):
        if t is not None and t.device != q.device:
            raise ValueError(f"all tensors must be on {q.device}")
    if workspace is None:
        workspace = SharedPrefixWorkspace(B, HQ, HKV, q.device, q.dtype)
    elif not workspace.matches(B, HQ, HKV, q.device, q.dtype):
        raise ValueError("workspace shape/device/dtype mismatch")
    o = workspace.o if out is None else out
    if o.shape != (B, HQ, 128) or o.dtype != q.dtype or not o.is_contiguous():
        raise ValueError("out must be a contiguous [B, HQ, 128] tensor of q's dtype")
    if partial_out is not None and (partial_out.shape != (B, HQ, 129) or partial_out.dtype != torch.float32
                                    or not partial_out.is_contiguous()):
        raise ValueError("partial_out must be a contiguous fp32 [B, HQ, 129] tensor")
    a = _lib.FfaSharedPrefixArgs(
        B, HQ, HKV, 128, NG, n_pages, block_table.shape[1], block_table.stride(0) if B > 1 else block_table.shape[1],
        _lib.float_code(q.dtype), v_code, fp8, int(use_fp8_residual), 1.0 / math.sqrt(128) if scale is None else float(scale),
        q.data_ptr(), k_fp8.data_ptr(), _lib.ptr(k_residual), v.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
        group_start.data_ptr(), prefix_pages.data_ptr(), o.data_ptr(), _lib.ptr(partial_out), workspace.scratch.data_ptr(),
        workspace.scratch.numel())
    _lib.enqueue(q.device, _lib.lib().ffa_decode_shared_prefix, "ffa_decode_shared_prefix", a)
    return o
