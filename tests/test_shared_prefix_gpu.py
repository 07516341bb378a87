"""Shared-prefix decode attention against the definition in 64 bits.

Bound of an output element: half a step of the output's type on the value, plus A = sum_t w_t |v_t| times what a weight
may be off: half a step of V's type (the weights are rounded to it) and the error of the scores, which is that of q as
sums of fp8 pieces (2^-18 of the largest |q|, times sum |k|) and of fp32 sums of 1536 products (2^-24 each way)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE, D = 64, 128
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Batch:
    """Groups of sequences with shared leading pages on one pool, pages in seeded disorder."""

    def __init__(self, sizes, prefix, own, HQ, HKV, qd=torch.bfloat16, vd=torch.bfloat16, fp8=E4, seed=0, gain=2.0, spare=3,
                 n_pages=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        B = sum(sizes)
        self.B, self.HQ, self.HKV, self.sizes, self.prefix = B, HQ, HKV, sizes, prefix
        grp = [i for i, n in enumerate(sizes) for _ in range(n)]
        self.grp, self.first = grp, [sum(sizes[:i]) for i in range(len(sizes))]
        self.lens = [prefix[grp[b]] * PAGE + own[b % len(own)] for b in range(B)]
        cols = max(1, max(-(-n // PAGE) for n in self.lens), max(prefix))
        need = sum(prefix) + sum(max(0, -(-n // PAGE) - prefix[grp[b]]) for b, n in enumerate(self.lens))
        used = need + spare
        n_pages = n_pages or used
        place = (torch.randperm(used, generator=torch.Generator().manual_seed(seed)) + (n_pages - used)).tolist()
        at, rows, firsts = 0, [], []
        for n in prefix:
            firsts.append(place[at:at + n])
            at += n
        for b in range(B):
            n = max(0, -(-self.lens[b] // PAGE) - prefix[grp[b]])
            rows.append((firsts[grp[b]] + place[at:at + n] + [-1] * cols)[:cols])
            at += n
        dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.table, self.seq_lens, self.prefix_pages = dev(rows), dev(self.lens), dev(prefix)
        self.group_start = dev(self.first + [B])
        shape = (n_pages, PAGE, HKV, D)
        self.k, self.r = torch.empty(shape, dtype=fp8, device="cuda"), torch.empty(shape, dtype=fp8, device="cuda")
        self.v = torch.empty(shape, dtype=vd, device="cuda")
        lo = n_pages - used
        chan = torch.exp(0.5 * torch.randn(HKV, D, generator=g, device="cuda"))
        x = (torch.randn(used, PAGE, HKV, D, generator=g, device="cuda") * chan).to(torch.bfloat16).float()
        self.k[lo:] = x.to(fp8)
        self.r[lo:] = (x - self.k[lo:].float()).to(fp8)
        self.v[lo:] = torch.randn(used, PAGE, HKV, D, generator=g, device="cuda").to(vd)
        self.q = (gain * torch.randn(B, 1, HQ, D, generator=g, device="cuda")).to(qd)

    def call(self, **kw):
        from ffa_speedtest_b200.fp8fp8.attn_kernel.attn_kernel_shared_prefix_fp8fp8 import attn_forward_decode_shared_prefix_fp8fp8
        args = dict(k_residual=self.r, block_table=self.table, seq_lens=self.seq_lens, group_start=self.group_start,
                    prefix_pages=self.prefix_pages)
        args.update(kw)
        return attn_forward_decode_shared_prefix_fp8fp8(self.q, self.k, self.v, **args)

    def exact(self, scale=None, residual=True, lens=None):
        """(output, allowed error, log-sum-exp in base 2) in 64 bits."""
        G, scale = self.HQ // self.HKV, 1 / math.sqrt(D) if scale is None else scale
        o = torch.zeros(self.B, self.HQ, D, dtype=torch.float64, device="cuda")
        tol, lse = torch.zeros_like(o), torch.full((self.B, self.HQ), -math.inf, dtype=torch.float64, device="cuda")
        qd = self.q.dtype if self.q.dtype != torch.float32 else torch.float16
        for b, n in enumerate(lens or self.lens):
            if n == 0:
                continue
            shared = min(self.prefix[self.grp[b]], -(-n // PAGE))
            row = torch.cat([self.table[self.first[self.grp[b]], :shared], self.table[b, shared:-(-n // PAGE)]]).long()
            k, v = self.k[row].double(), self.v[row].double().flatten(0, 1)[:n]
            k = ((k + self.r[row].double()) if residual else k).flatten(0, 1)[:n]
            for h in range(self.HKV):
                s = slice(h * G, (h + 1) * G)
                q = self.q[b, 0, s].to(qd).double()
                d = q @ k[:, h].T * scale
                w = torch.softmax(d, -1)
                o[b, s] = w @ v[:, h]
                lse[b, s] = torch.logsumexp(d, -1) / math.log(2)
                # an error of the dot product grows with the size of the scale, whatever its sign
                score = abs(scale) * (2.0 ** -18 * q.abs().amax(-1) * k[:, h].abs().sum(-1).amax()
                                 + 1536 * 2.0 ** -24 * (q.abs() @ k[:, h].abs().T).amax(-1))
                weight = half_step(self.v.dtype) + 2 * score + 2.0 ** -20
                tol[b, s] = (w @ v[:, h].abs()) * weight[:, None] + half_step(self.q.dtype) * o[b, s].abs() + 1e-7
                self.lse_tol = max(getattr(self, "lse_tol", 0.0), float(2 * score.max()) / math.log(2) + 1e-5)
        return o, tol, lse

    def check(self, got, **kw):
        o, tol, _ = self.exact(**kw)
        off = (got.double() - o).abs()
        assert got.shape == o.shape and bool(torch.isfinite(got).all())
        assert bool((off <= tol).all()), f"largest error {float(off.max()):.3g}, {float((off / tol).max()):.3g} of what is allowed"


CASES = [
    # sizes, shared pages, own tokens, HQ, HKV
    ([1], [0], [1], 1, 1),
    ([2], [1], [1], 4, 2),
    ([3], [2], [0], 4, 1),
    ([1, 1], [0, 0], [64, 129], 8, 8),
    ([4, 1, 2], [3, 0, 5], [0, 1, 63, 64, 65, 127, 128], 6, 2),
    ([9], [37], [5, 300, 0, 77], 24, 8),
    ([16, 17], [8, 1], [10, 200], 32, 4),          # 128 query rows, and 8 more
    ([40], [11], [3], 40, 5),                      # 320 rows
    ([33, 1], [64, 3], [1, 2, 500], 8, 1),
    ([1], [1100], [17], 8, 1),
    ([1] * 20, [0] * 20, [0, 1, 700, 64, 900, 2000], 16, 8),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("qd,vd,fp8", [(torch.bfloat16, torch.bfloat16, E5), (torch.float16, torch.float16, E4)])
def test_against_the_definition(case, qd, vd, fp8):
    b = Batch(*CASES[case], qd=qd, vd=vd, fp8=fp8, seed=case)
    b.check(b.call())


@pytest.mark.parametrize("rows", [7, 8, 9, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129])
def test_numbers_of_query_rows(rows):
    """Around the numbers of rows where the way they lie in the tile changes, one head and many partials to a row."""
    b = Batch([rows], [301], [0, 1, 130], 1, 1, seed=rows)
    b.check(b.call())


@pytest.mark.parametrize("B", [1, 4, 5, 9, 10, 18, 19, 37, 74, 75])
def test_numbers_of_sequences(B):
    """Around the numbers where the merge is cut differently (37, 74 and 148 heads of sequences, and two and more to an SM)."""
    b = Batch([B - B // 2] + [B // 2] * (B > 1), [40, 25][:1 + (B > 1)], [70, 0, 260], 16, 8, seed=B)
    b.check(b.call())


@pytest.mark.parametrize("qd", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vd", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fp8", [E4, E5])
def test_types(qd, vd, fp8):
    b = Batch([5, 2], [3, 9], [1, 100], 16, 2, qd=qd, vd=vd, fp8=fp8, seed=3)
    b.check(b.call())
    b.check(b.call(use_fp8_residual=False, k_residual=None), residual=False)
    b.check(b.call(scale=0.3), scale=0.3)


def test_lengths_of_zero_one_and_inside_the_prefix():
    b = Batch([6, 3], [4, 2], [1, 70], 12, 4, seed=5)
    lens = [0, 1, 64, 200, 256, 257, 0, 0, 0]
    b.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    part = torch.full((9, 12, 129), 7.0, device="cuda")
    got = b.call(partial_out=part)
    b.check(got, lens=lens)
    _, _, lse = b.exact(lens=lens)
    assert bool((got[[0, 6, 7, 8]] == 0).all()) and bool((part[[0, 6, 7, 8], :, :128] == 0).all())
    assert bool((part[[0, 6, 7, 8], :, 128] == -math.inf).all())
    live = [1, 2, 3, 4, 5]
    assert float((part[live, :, 128].double() - lse[live]).abs().max()) <= b.lse_tol
    b.seq_lens.zero_()                                       # nobody holds anything
    assert bool((b.call() == 0).all())


@pytest.mark.parametrize("sizes,prefix", [([3, 1], [2, 0]), ([40, 2], [3, 1])])
def test_padding_that_holds_nothing_gives_zeros_whatever_its_q(sizes, prefix):
    b = Batch(sizes, prefix, [20], 8, 2, seed=18)
    empty = [0, 2, b.B - 1]
    lens = [0 if i in empty else n for i, n in enumerate(b.lens)]
    b.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    b.seq_lens[0] = -5                                       # below zero is as good as zero
    b.q[empty] = 0
    want = b.call().clone()
    b.check(want, lens=lens)
    for bad in (math.nan, math.inf):
        b.q[empty] = bad
        part = torch.full((b.B, 8, 129), 7.0, device="cuda")
        got = b.call(partial_out=part)
        assert torch.equal(got, want)
        assert bool((part[empty, :, :128] == 0).all()) and bool((part[empty, :, 128] == -math.inf).all())


def test_garbage_outside_the_sequences():
    """NaN and infinities in the unused rows of pages, in unused pages and in unused table entries."""
    b = Batch([3, 2], [2, 0], [1, 65, 100], 8, 2, seed=6, spare=9)
    used = torch.zeros(b.k.shape[0], PAGE, dtype=torch.bool, device="cuda")
    for i, n in enumerate(b.lens):
        for j in range(-(-n // PAGE)):
            used[int(b.table[i, j]), :min(PAGE, n - j * PAGE)] = True
    nan = torch.full_like(b.v, math.nan)
    nan[:, ::2] = math.inf
    b.v = torch.where(used[..., None, None], b.v, nan)
    for name in ("k", "r"):
        x = getattr(b, name).view(torch.uint8)
        setattr(b, name, torch.where(used[..., None, None], x, torch.full_like(x, 0x7f)).view(b.k.dtype))
    for i, n in enumerate(b.lens):
        b.table[i, -(-n // PAGE):] = 2 ** 31 - 1
    b.check(b.call())


def test_growing_scores_and_one_loud_token():
    """Maxima that rise from tile to tile by far more than exp2 can hold, then fall."""
    b = Batch([7], [21], [40, 400], 16, 2, seed=7)
    pages = b.table[0, :21].long()
    x = b.k[pages].float()
    x *= torch.linspace(0.05, 12.0, 21, device="cuda")[:, None, None, None]
    b.k[pages] = x.to(b.k.dtype)
    b.check(b.call())
    b.k[pages[3], 11] = (8 * b.q[0, 0].view(2, 8, D).float().mean(1)).to(b.k.dtype)
    b.check(b.call())
    b.v.fill_(1.0)                                           # weights add up to one
    assert float((b.call().float() - 1).abs().max()) <= half_step(torch.bfloat16)


@pytest.mark.parametrize("vd", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", [17, 25])
@pytest.mark.parametrize("sizes,prefix,own", [([1, 1], 0, 2048), ([12], 32, 10), ([40], 32, 10), ([100], 32, 10)])
def test_one_token_far_above_many(sizes, prefix, own, gap, vd):
    """A first token whose weight is 2^gap times that of the others and whose V is zero: what the others add up to is the
    output, whatever the type that weights are held in.  Ways of all layouts of the query rows."""
    b = Batch(sizes, [prefix] * len(sizes), [own], 1, 1, qd=torch.float32, vd=vd, seed=gap + sum(sizes))
    u = 2 * torch.randn(D, generator=torch.Generator(device="cuda").manual_seed(gap), device="cuda")
    b.q = (u * (1 + 0.01 * torch.randn(b.B, 1, 1, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")))
    b.k = (0.02 * b.k.float()).to(b.k.dtype)
    b.r.zero_()
    b.v = b.v.abs() + 0.5
    for i in set(b.first) if prefix else range(b.B):
        page = int(b.table[i, 0])
        b.k[page, 0, 0] = (gap * math.log(2) * math.sqrt(D) * u / u.square().sum()).to(b.k.dtype)
        b.v[page, 0] = 0
    b.check(b.call())


def test_infinite_values_stay_where_they_are():
    b = Batch([2], [2], [30], 8, 2, seed=8)
    page = int(b.table[1, 2])                                # a page of the second sequence alone
    b.v[page, 3, 1, 5] = math.inf
    b.v[page, 4, 0, 9] = math.nan
    got = b.call().double()
    assert bool(torch.isfinite(got[0]).all())
    bad = ~torch.isfinite(got[1])
    want = torch.zeros(8, D, dtype=torch.bool, device="cuda")
    want[4:, 5] = True
    want[:4, 9] = True
    assert torch.equal(bad, want)


def test_scales_of_any_sign_and_a_row_that_is_not_finite():
    for vd, sizes in ((torch.bfloat16, [3]), (torch.float16, [20])):
        b = Batch(sizes, [3], [70], 8, 2, seed=15, vd=vd)
        for scale in (-0.2, 0.0, 1e-6):
            b.check(b.call(scale=scale), scale=scale)
        want = b.call().clone()
        b.q[1, 0, 5, 17] = math.inf
        b.q[2, 0, 0, 3] = math.nan
        got = b.call()
        bad = torch.zeros(b.B, 8, dtype=torch.bool, device="cuda")
        bad[1, 5] = bad[2, 0] = True
        assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], want[~bad])


def test_a_scale_that_is_not_finite():
    b = Batch([3], [2], [40], 8, 2, seed=15)
    for scale in (math.nan, math.inf, -math.inf):
        assert bool(torch.isnan(b.call(scale=scale)).all())
    b.check(b.call())


def test_single_sequences_in_groups_of_their_own_and_empty_groups():
    b = Batch([1, 1, 1], [2, 0, 5], [33, 1, 200], 8, 2, seed=16)
    b.check(b.call())
    dev = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    b.check(b.call(group_start=dev(0, 0, 1, 3), prefix_pages=dev(7, 2, 0)))       # an empty group; two sequences that share nothing


def test_large_batch():
    """More sequences and groups than the kernel's threads and its near list of groups."""
    sizes = [1, 2, 3] * 170
    b = Batch(sizes, [i % 3 for i in range(510)], [0, 1, 5, 64, 70], 4, 1, seed=17)
    assert b.B == 1020
    b.check(b.call())


def test_largest_batch():
    from ffa_speedtest_b200.fp8fp8.attn_kernel.attn_kernel_shared_prefix_fp8fp8 import SharedPrefixWorkspace
    sizes = [1] * 900 + [2, 3] * 600 + [196]
    b = Batch(sizes, [(i % 3 + 1) // 2 for i in range(len(sizes))], [0, 1, 5, 64, 70], 2, 1, seed=19)
    assert b.B == 4096
    b.check(b.call())
    with pytest.raises(ValueError, match="1 to 4096"):
        SharedPrefixWorkspace(4097, 2, 1, b.q.device, b.q.dtype)


def test_same_as_the_pruned_decode_that_drops_nothing():
    from ffa_speedtest_b200.fp8fp8.attn_kernel.attn_kernel_v1210_fused_bsz_fp8fp8 import attn_forward_decode_fp8fp8
    b = Batch([4], [30], [100], 32, 8, seed=9)
    o = attn_forward_decode_fp8fp8(b.q, b.k, b.v, k_residual=b.r, BS=64, SBS=64, delta=1e4, block_table=b.table,
                                   seq_len=b.lens[0])
    got = b.call()
    b.check(got)
    assert float((o.float() - got.float()).abs().max()) <= 2e-2


def test_halves_merge_to_the_whole():
    from ffa_speedtest_b200 import _lib
    b = Batch([5], [6], [100], 8, 4, seed=10)
    parts = torch.empty(2, 5, 8, 129, device="cuda")
    b.call(seq_lens=torch.full((5,), 256, dtype=torch.int32, device="cuda"), prefix_pages=torch.tensor([4], dtype=torch.int32, device="cuda"),
           partial_out=parts[0])
    b.call(block_table=b.table[:, 4:], seq_lens=b.seq_lens - 256, prefix_pages=torch.tensor([2], dtype=torch.int32, device="cuda"),
           partial_out=parts[1])
    out = torch.empty(5, 8, 128, device="cuda", dtype=torch.bfloat16)
    _lib.check(_lib.lib().ffa_merge_partials(parts.data_ptr(), 2, 40, out.data_ptr(), _lib.BF16, _lib.current_stream(out.device)), "merge")
    b.check(out)


def test_streams_workspaces_and_capture():
    from ffa_speedtest_b200.fp8fp8.attn_kernel.attn_kernel_shared_prefix_fp8fp8 import allocate_shared_prefix_workspace
    a, b = Batch([3, 4], [5, 2], [70, 3], 8, 2, seed=11), Batch([7], [50], [9], 8, 2, seed=12)
    wa, wb = (allocate_shared_prefix_workspace(x.q, x.v) for x in (a, b))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):                                      # two calls at a time
        with torch.cuda.stream(s1):
            oa = a.call(workspace=wa)
        with torch.cuda.stream(s2):
            ob = b.call(workspace=wb)
    torch.cuda.synchronize()
    a.check(oa)
    b.check(ob)
    assert wa.status() == wb.status() == 0
    first = a.call(workspace=wa).clone()
    assert torch.equal(first, oa)                            # the same call gives the same bits
    out = torch.zeros_like(first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.call(workspace=wa, out=out)
    g.replay()
    assert torch.equal(out, first)
    lens = [x - 60 if i % 2 else x // 3 for i, x in enumerate(a.lens)]
    a.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))  # a replay follows the lengths
    a.q.mul_(0.5)
    g.replay()
    a.check(out, lens=lens)


def test_pool_past_32_bit_offsets():
    n_pages = 36000                                          # 4.7 GB of V, 2.4 GB each of base and residual
    b = Batch([3], [4], [70], 16, 8, seed=13, n_pages=n_pages)
    assert b.v.numel() * 2 > 2 ** 32 and int(b.table.max()) > 35000
    b.check(b.call())


def test_groups_that_are_not_what_they_should_be_stay_inside_the_tensors():
    """Bounds that do not ascend or leave sequences out: no particular result, no access outside, and sequences
    outside every group have no shared part."""
    b = Batch([2, 2], [3, 3], [10], 8, 2, seed=14)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for start, pages in (([0, 4, 0], [3, 3]), ([3, -5, 99], [3, 3]), ([0, 4, 4], [-2, 5000]), ([2, 2, 2], [3, 3])):
        assert b.call(group_start=dev(start), prefix_pages=dev(pages)).shape == (4, 8, 128)
    b.table[:, :3] = torch.stack([b.table[i, :3] for i in (0, 0, 2, 2)])
    b.check(b.call(group_start=dev([0, 2, 2])))
    b.seq_lens[1], b.seq_lens[2] = 2 ** 31 - 1, -7
    b.call()
    torch.cuda.synchronize()


def test_refusals():
    b = Batch([2], [1], [5], 4, 2)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for bad in (dict(k_residual=None), dict(k_residual=b.r.float().to(E5)), dict(block_table=b.table.long()), dict(block_table=b.table[:1]),
                dict(block_table=b.table[:, :0]), dict(block_table=b.table.t()), dict(seq_lens=b.seq_lens[:1]), dict(seq_lens=b.seq_lens.long()),
                dict(group_start=i32(0, 1, 2)), dict(prefix_pages=i32()), dict(prefix_pages=i32(0, 0, 0), group_start=i32(0, 1, 2, 2)),
                dict(seq_lens=b.seq_lens.cpu()), dict(out=torch.empty(2, 4, 128, device="cuda")), dict(partial_out=torch.empty(2, 4, 128, device="cuda"))):
        with pytest.raises(ValueError):
            b.call(**bad)
    q, k, v, r = b.q, b.k, b.v, b.r
    for name, x in (("q", q.cpu()), ("q", q[:, :, :3]), ("q", q[..., :64]), ("q", torch.cat([q, q], 1)), ("v", v.float()), ("k", k.float()),
                    ("v", v[:1]), ("k", k[:, :32]), ("q", torch.zeros(2, 1, 18, 128, device="cuda", dtype=torch.bfloat16))):
        setattr(b, name, x)
        with pytest.raises(ValueError):
            b.call()
        b.q, b.k, b.v, b.r = q, k, v, r
    from ffa_speedtest_b200.fp8fp8.attn_kernel.attn_kernel_shared_prefix_fp8fp8 import SharedPrefixWorkspace
    with pytest.raises(ValueError, match="mismatch"):
        b.call(workspace=SharedPrefixWorkspace(3, 4, 2, q.device, q.dtype))
    with pytest.raises(ValueError, match="workspace"):
        SharedPrefixWorkspace(20000, 4, 2, q.device, q.dtype)
