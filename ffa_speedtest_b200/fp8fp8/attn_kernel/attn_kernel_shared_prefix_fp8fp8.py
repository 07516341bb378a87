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
_SCALE = 1.0 / math.sqrt(128)


class SharedPrefixWorkspace:
    """Output and scratch of the shared-prefix decode, for one batch size and head layout.  One call at a time may
    use it (two captured graphs that may run at the same time need one each).  It is zeroed on the stream that is current
    when it is made: calls on another stream have to come after that."""

    def __init__(self, B: int, HQ: int, HKV: int, device, dtype):
        self.B, self.HQ, self.HKV, self.device, self.dtype = int(B), int(HQ), int(HKV), torch.device(device), dtype
        self.nbytes = nbytes = _lib.lib().ffa_shared_prefix_workspace_bytes(self.B, self.HQ, self.HKV)
        if nbytes == 0:
            raise ValueError(f"no workspace for B={B}, HQ={HQ}, HKV={HKV}: B must be 1 to 4096, HQ a multiple of HKV")
        self.scratch = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self.scratch[:512].zero_()
        self.status_word = self.scratch[256:260].view(torch.int32)
        self.o = torch.empty((self.B, self.HQ, 128), dtype=dtype, device=self.device)

    def matches(self, B: int, HQ: int, HKV: int, device, dtype) -> bool:
        return (self.B, self.HQ, self.HKV, self.o.device, self.dtype) == (B, HQ, HKV, device, dtype)

    def status(self) -> int:
        """Device status word (synchronises): 0 = ok, 1 = a bounded wait inside a kernel gave up (the affected
        outputs are NaN)."""
        return int(self.status_word.item())


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
    included; a sequence of length 0 gives zeros, one that is shorter than its group's prefix sees its own tokens only (V
    of the others has to be finite there).  Lengths and groups are read on the device when the kernels run.
    ``partial_out [B, HQ, 129]`` (fp32) also receives the normalised output and the base-2 log-sum-exp.  Without ``out`` the
    result is the workspace's own buffer, which its next call overwrites."""
    if not (q.is_cuda and k_fp8.is_cuda and v.is_cuda):
        raise ValueError("q, K and V must be CUDA tensors (this build has no CPU path)")
    q_shape, k_shape = q.shape, k_fp8.shape
    if len(q_shape) != 4 or q_shape[1] != 1 or q_shape[3] != 128:
        raise ValueError(f"q must be [B, 1, HQ, 128], got {tuple(q_shape)}")
    if len(k_shape) != 4 or k_shape[1] != PAGE or k_shape[3] != 128 or v.shape != k_shape:
        raise ValueError(f"K and V must be paged pools [n_pages, 64, HKV, 128], got {tuple(k_shape)} and {tuple(v.shape)}")
    B, HQ, n_pages, HKV = q_shape[0], q_shape[2], k_shape[0], k_shape[2]
    if HKV == 0 or HQ % HKV != 0:
        raise ValueError(f"HQ ({HQ}) must be divisible by HKV ({HKV}) for GQA")
    if HQ // HKV > 8:
        raise ValueError(f"this build supports GQA group sizes up to 8, got {HQ // HKV}")
    device, q_dtype, k_dtype = q.device, q.dtype, k_fp8.dtype
    fp8, v_code = _lib.fp8_code(k_dtype), _lib.float_code(v.dtype)
    if v_code == _lib.F32:
        raise ValueError("v must be float16 or bfloat16")
    if use_fp8_residual:
        if k_residual is None:
            raise ValueError("use_fp8_residual=True requires k_residual")
        if k_residual.shape != k_shape or k_residual.dtype != k_dtype:
            raise ValueError("k_residual must have the shape and fp8 encoding of k_fp8")
    else:
        k_residual = None
    table_shape = block_table.shape
    if block_table.dtype != torch.int32 or len(table_shape) != 2 or table_shape[0] != B or table_shape[1] == 0:
        raise ValueError("block_table must be an int32 tensor [B, pages]")
    cols, table_stride = table_shape[1], block_table.stride(0) if B > 1 else table_shape[1]
    if block_table.stride(1) != 1 or table_stride < cols:
        raise ValueError("block_table must have unit stride in its last dimension and rows that do not overlap")
    NG = prefix_pages.numel()
    for name, t, n in (("seq_lens", seq_lens, B), ("group_start", group_start, NG + 1), ("prefix_pages", prefix_pages, NG)):
        if t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector of {n} entries")
    if not 1 <= NG <= B:
        raise ValueError(f"there must be 1 to B = {B} groups, got {NG}")
    for t in (q, k_fp8, v, k_residual):
        if t is not None and not t.is_contiguous():
            raise ValueError("q, K, residual and V must be contiguous")
    for t in (k_fp8, v, k_residual, block_table, seq_lens, group_start, prefix_pages, out, partial_out):
        if t is not None and t.device != device:
            raise ValueError(f"all tensors must be on {device}")
    if workspace is None:
        workspace = SharedPrefixWorkspace(B, HQ, HKV, device, q_dtype)
    elif not workspace.matches(B, HQ, HKV, device, q_dtype):
        raise ValueError("workspace shape/device/dtype mismatch")
    if out is None:
        out = workspace.o
    elif out.shape != (B, HQ, 128) or out.dtype != q_dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous [B, HQ, 128] tensor of q's dtype")
    if partial_out is not None and (partial_out.shape != (B, HQ, 129) or partial_out.dtype != torch.float32
                                    or not partial_out.is_contiguous()):
        raise ValueError("partial_out must be a contiguous fp32 [B, HQ, 129] tensor")
    a = _lib.FfaSharedPrefixArgs(
        B, HQ, HKV, 128, NG, n_pages, cols, table_stride, _lib.float_code(q_dtype), v_code, fp8, int(use_fp8_residual),
        _SCALE if scale is None else float(scale), q.data_ptr(), k_fp8.data_ptr(), _lib.ptr(k_residual), v.data_ptr(),
        block_table.data_ptr(), seq_lens.data_ptr(), group_start.data_ptr(), prefix_pages.data_ptr(), out.data_ptr(),
        _lib.ptr(partial_out), workspace.scratch.data_ptr(), workspace.nbytes)
    _lib.enqueue(device, _lib.lib().ffa_decode_shared_prefix, "ffa_decode_shared_prefix", a)
    return out
