"""What the page table and the ragged append refuse before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch


def table(L, **kw):
    from ffa_speedtest_b200 import _lib
    a = _lib.FfaPageTable()
    a.n_pages, a.max_seqs, a.cols, a.bt_stride = 10, 4, 6, 6
    a.block_table = a.seq_lens = a.refcount = a.status = a.scratch = 256
    a.scratch_bytes = L.ffa_pages_scratch_bytes(10, 4)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_c_entries_refuse(built_lib):
    from ffa_speedtest_b200 import _lib
    L = _lib.lib()
    pools = _lib.FfaPagePools()
    good = table(L)
    for bad, code in [(dict(block_table=None), -1), (dict(refcount=None), -1), (dict(scratch=None), -1), (dict(n_pages=0), -2),
                      (dict(max_seqs=0), -2), (dict(bt_stride=5), -2), (dict(cols=1 << 30, bt_stride=1 << 30), -2),
                      (dict(max_seqs=65537), -7), (dict(scratch_bytes=64), -4)]:
        t = table(L, **bad)
        assert L.ffa_pages_truncate(t, 256, 256, 1, None) == code, bad
        assert L.ffa_pages_fork(t, 256, 256, 1, None) == code, bad
        assert L.ffa_pages_extend(t, pools, 256, 256, 1, None) == code, bad
        assert L.ffa_pages_compact(t, pools, 256, 256, None) == code, bad
    assert L.ffa_pages_truncate(good, None, 256, 1, None) == -1
    assert L.ffa_pages_fork(good, 256, None, 1, None) == -1
    assert L.ffa_pages_extend(good, None, 256, 256, 1, None) == -1
    assert L.ffa_pages_compact(good, pools, None, 256, None) == -1
    for n in (0, -1, 5):
        assert L.ffa_pages_truncate(good, 256, 256, n, None) == -2
        assert L.ffa_pages_extend(good, pools, 256, 256, n, None) == -2
    pools.n_pools, pools.bases, pools.token_bytes, pools.max_token_bytes = 1, 256, 256, 24
    assert L.ffa_pages_extend(good, pools, 256, 256, 1, None) == -2
    pools.bases = None
    assert L.ffa_pages_compact(good, pools, 256, 256, None) == -1
    args = [256, 256, 1, 2, 3, 4, 1, 256, 256, 256, 9, 256, 6, 6, 256, None, None]
    for at, value, code in [(0, None, -1), (7, None, -1), (14, None, -1), (3, 0, -2), (4, 0, -2), (12, 5, -2), (10, 0, -2), (2, 2, -3),
                            (6, 2, -3), (0, 264, -8), (9, 260, -8)]:
        a = list(args)
        a[at] = value
        assert L.ffa_cache_append_ragged(*a) == code, (at, value)


def test_scratch_grows_with_the_table(built_lib):
    from ffa_speedtest_b200 import _lib
    size = _lib.lib().ffa_pages_scratch_bytes
    assert size(0, 4) == size(4, 0) == 0
    assert 4 * (16 + 4 * 100 + 7) <= size(100, 7) < size(101, 7) <= size(101, 102)


def test_python_refuses(built_lib):
    from ffa_speedtest_b200.pages import PageTable, append_ragged_fp8fp8
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU path"):
        PageTable.wrap(i32(3, 4), i32(3), i32(9))
    with pytest.raises(ValueError, match="int32"):
        PageTable.wrap(i32(3, 4).long(), i32(3), i32(9))
    with pytest.raises(ValueError, match="non-empty"):
        PageTable.wrap(i32(0, 4), i32(0), i32(9))
    with pytest.raises(ValueError, match="positive"):
        PageTable(0, 3, 4, device="cpu")
    k = torch.zeros(2, 1, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        append_ragged_fp8fp8(k, k, k, k, k, i32(2, 1), i32(2))
