"""How a batch is cut into groups that share pages, and what the cache refuses to be made for (no GPU needed)."""
import random

import numpy as np
import pytest
import torch

from ffa_speedtest_b200.fp8fp8.e2e.shared_cache import SharedPrefixFP8Fp8Cache, _stretches


def saved(common, start):
    return sum((b - a - 1) * min(common[a:b - 1]) for a, b in zip(start[:-1], start[1:]) if b - a > 1)


@pytest.mark.parametrize("common,start,pages", [
    ([], [0, 1], [0]),
    ([0], [0, 1, 2], [0, 0]),
    ([3, 3, 3], [0, 4], [3]),                               # samples of one prompt
    ([3, 0, 5], [0, 2, 4], [3, 5]),
    ([160, 160, 3, 3], [0, 3, 5], [160, 3]),                # forks of a grown sample, then samples of its prompt
    ([10, 11, 12], [0, 4], [10]),                           # forked at every other step: one group reads least
])
def test_cuts(common, start, pages):
    assert _stretches(np.array(common, dtype=np.int64)) == (start, pages)


def test_no_cut_saves_more():
    r = random.Random(0)
    for _ in range(600):
        n = r.randint(1, 8)
        common = [r.choice([0, 1, 2, 3, 5, 9]) for _ in range(n - 1)]
        start, pages = _stretches(np.array(common, dtype=np.int64))
        assert start[0] == 0 and start[-1] == n and start == sorted(set(start))
        assert pages == [min(common[a:b - 1]) if b - a > 1 else 0 for a, b in zip(start[:-1], start[1:])]
        assert saved(common, start) == max(saved(common, [0, *(i for i in range(1, n) if cut >> i & 1), n]) for cut in range(0, 1 << n, 2))


@pytest.mark.parametrize("bad", [dict(dtype=torch.float32), dict(fp8_dtype=torch.bfloat16), dict(num_kv_heads=0), dict(head_dim=64),
                                 dict(num_layers=0), dict(dtype=torch.float8_e5m2)])
def test_a_cache_that_no_step_could_fill_is_refused(bad):
    """Before a step has extended its sequences, and before anything is allocated."""
    args = dict(max_seqs=2, num_kv_heads=2, max_seq_len=128, num_layers=1, fp8_dtype=torch.float8_e5m2, device="cpu")
    with pytest.raises(ValueError, match=next(iter(bad)).replace("max_", "")):
        SharedPrefixFP8Fp8Cache(**{**args, **bad})
