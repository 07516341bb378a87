"""Page table (fork, extend, truncate, compact) and the ragged append against plain models of them."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 64


class Model:
    """The page table in plain Python: same rules, one page at a time."""

    def __init__(self, n_pages, max_seqs, cols, pools):
        self.n, self.cols = n_pages, cols
        self.table = [[-1] * cols for _ in range(max_seqs)]
        self.lens, self.count, self.status = [0] * max_seqs, [0] * n_pages, 0
        self.pools = [p.clone() for p in pools]

    def refuse(self, bit):
        self.status |= bit

    def truncate(self, seqs, lens):
        if any(s < 0 or s >= len(self.lens) for s in seqs) or any(x < 0 for x in lens):
            return self.refuse(1)
        for s, n in zip(seqs, lens):
            if n < self.lens[s]:
                for j in range(-(-n // PAGE), -(-self.lens[s] // PAGE)):
                    self.count[self.table[s][j]] -= 1
                    self.table[s][j] = -1
                self.lens[s] = n

    def fork(self, parents, children):
        ok = all(0 <= s < len(self.lens) for s in parents + children) and len(set(children)) == len(children)
        if not ok or set(children) & set(parents) or any(self.lens[c] for c in children):
            return self.refuse(1)
        for p, c in zip(parents, children):
            self.table[c], self.lens[c] = list(self.table[p]), self.lens[p]
            for page in self.table[c]:
                if page >= 0:
                    self.count[page] += 1

    def extend(self, seqs, new):
        if any(s < 0 or s >= len(self.lens) for s in seqs) or len(set(seqs)) != len(seqs) or any(x < 0 for x in new) \
                or any(self.lens[s] + x > self.cols * PAGE for s, x in zip(seqs, new)):
            return self.refuse(1)
        free = [p for p in range(self.n) if self.count[p] == 0]
        plan, shared = [], list(self.count)
        for s, x in zip(seqs, new):
            n = self.lens[s]
            own = x > 0 and n % PAGE and shared[self.table[s][n // PAGE]] > 1
            need = (-(-(n + x) // PAGE) - -(-n // PAGE) if x else 0) + (1 if own else 0)
            plan.append((s, x, own, need))
        if sum(p[3] for p in plan) > len(free):
            return self.refuse(2)
        for s, x, own, need in plan:
            n, got = self.lens[s], free[:need]
            del free[:need]
            if own:
                old, page = self.table[s][n // PAGE], got.pop(0)
                for pool in self.pools:
                    pool[page, :n % PAGE] = pool[old, :n % PAGE]
                self.count[old] -= 1
                self.count[page] = 1
                self.table[s][n // PAGE] = page
            for j, page in enumerate(got):
                self.table[s][-(-n // PAGE) + j] = page
                self.count[page] = 1
            self.lens[s] = n + x

    def compact(self):
        live = sum(c > 0 for c in self.count)
        src = [p for p in range(live, self.n) if self.count[p]]
        dst = [p for p in range(live) if not self.count[p]]
        to = dict(zip(src, dst))
        for a, b in to.items():
            for pool in self.pools:
                pool[b] = pool[a]
            self.count[b], self.count[a] = self.count[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]

    def same_as(self, t):
        assert t.block_table.tolist() == self.table
        assert t.seq_lens.tolist() == self.lens
        assert t.refcount.tolist() == self.count
        assert t.status() == self.status
        for a, b in zip(t.pools, self.pools):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def make(n_pages, max_seqs, cols, shapes=((1, 128), (3, 16), (2, 256)), seed=0):
    from ffa_speedtest_b200.pages import PageTable
    g = torch.Generator(device="cuda").manual_seed(seed)
    pools = [torch.randint(0, 256, (n_pages, PAGE, *s), generator=g, device="cuda", dtype=torch.uint8) for s in shapes]
    return PageTable(n_pages, max_seqs, cols, pools=pools), Model(n_pages, max_seqs, cols, pools)


def both(t, m, what, *args):
    getattr(t, what)(*args)
    getattr(m, what)(*args)
    m.same_as(t)


def test_fork_write_end_and_compact():
    t, m = make(40, 8, 9)
    both(t, m, "extend", [0, 3], [130, 64])
    both(t, m, "fork", [0, 0, 3], [1, 2, 4])
    both(t, m, "extend", [1, 2, 4, 0], [1, 200, 1, 62])      # open page of 0 is shared by three, that of 3 is full
    both(t, m, "truncate", [0, 2], [0, 100])
    both(t, m, "fork", [2], [0])
    both(t, m, "extend", [0], [1])                            # 2 and 0 share an open page again
    both(t, m, "compact")
    both(t, m, "extend", [5], [300])
    assert t.status() == 0
    t.check()


@pytest.mark.parametrize("seed", range(6))
def test_random_walk(seed):
    r = random.Random(seed)
    n_pages, seqs, cols = r.choice([(1, 2, 2), (31, 5, 8), (32, 9, 6), (97, 16, 12), (1100, 40, 33)])
    t, m = make(n_pages, seqs, cols, seed=seed)
    for _ in range(40):
        some = r.sample(range(seqs), r.randint(1, seqs))
        what = r.choice(["extend", "extend", "truncate", "fork", "compact"])
        if what == "extend":
            both(t, m, what, some, [r.choice([0, 1, r.randint(0, cols * PAGE // 2)]) for _ in some])
        elif what == "truncate":
            some = [r.choice(some) for _ in some]             # numbers may come twice
            both(t, m, what, some, [r.randint(0, cols * PAGE) for _ in some])
        elif what == "fork":
            empty = [s for s in some if m.lens[s] == 0] or some[:1]
            full = [s for s in range(seqs) if s not in empty] or some[:1]
            both(t, m, what, [r.choice(full) for _ in empty], empty)
        else:
            both(t, m, what)


def test_refusals_change_nothing():
    t, m = make(10, 6, 4)
    both(t, m, "extend", [0, 1], [70, 10])
    for what, *args in [("extend", [0, 0], [1, 1]), ("extend", [6], [1]), ("extend", [-1], [1]), ("extend", [0], [-1]),
                        ("extend", [0], [256 - 70 + 1]), ("fork", [0, 0], [2, 2]), ("fork", [0], [1]), ("fork", [0], [0]),
                        ("fork", [0, 2], [2, 3]), ("fork", [9], [2]), ("fork", [0], [-3]), ("truncate", [0, 6], [0, 0]),
                        ("truncate", [0], [-1])]:
        both(t, m, what, *args)
        assert t.status() == 1
        with pytest.raises(RuntimeError, match="not allowed"):
            t.check()
        m.status = 0
    both(t, m, "extend", [2, 3, 4], [256, 200, 1])            # 9 pages, 7 are free
    with pytest.raises(RuntimeError, match="free pages"):
        t.check()
    m.status = 0
    both(t, m, "extend", [2, 3], [256, 192])
    assert t.free_pages() == 0
    both(t, m, "extend", [0, 1], [58, 54])                    # fits into the pages they hold
    both(t, m, "extend", [0], [1])
    assert t.status() == 2


def test_many_sequences_and_pages():
    t, m = make(70001, 3000, 40, shapes=())
    r = random.Random(1)
    lens = [r.randint(0, 1000) for _ in range(1400)]
    both(t, m, "extend", list(range(1400)), lens)
    both(t, m, "fork", [r.randrange(1400) for _ in range(1500)], list(range(1500, 3000)))
    both(t, m, "extend", list(range(1, 3000, 2)), [r.randint(0, 700) for _ in range(1500)])
    both(t, m, "truncate", list(range(0, 3000, 3)), [0] * 1000)
    both(t, m, "compact")
    both(t, m, "extend", list(range(0, 3000, 3)), [65] * 1000)
    assert t.status() == 0


def test_compact_beside_the_state():
    t, m = make(64, 4, 12)
    both(t, m, "extend", [0, 1, 2], [700, 650, 320])
    both(t, m, "fork", [2], [3])
    both(t, m, "truncate", [0], [0])
    old = [row[:] for row in m.table], list(m.count)
    out, count = torch.empty_like(t.block_table), torch.empty_like(t.refcount)
    pages = {p for row in m.table for p in row if p >= 0}
    before = {p: [x[p].clone() for x in t.pools] for p in pages}
    t.compact(block_table_out=out, refcount_out=count)
    assert (t.block_table.tolist(), t.refcount.tolist()) == old
    for p in pages:                                           # the old table's pages hold what they held
        assert all(torch.equal(a, x[p]) for a, x in zip(before[p], t.pools))
    m.compact()
    assert out.tolist() == m.table and count.tolist() == m.count
    assert all(torch.equal(a, b) for a, b in zip(t.pools, m.pools))
    with pytest.raises(ValueError, match="both"):
        t.compact(block_table_out=out)
    with pytest.raises(ValueError, match="strides"):
        t.compact(block_table_out=out[:, :5], refcount_out=count)


def test_empty_lists_do_nothing():
    t, m = make(10, 4, 4)
    both(t, m, "extend", [0], [70])
    for what, *args in (("extend", [], []), ("truncate", [], []), ("fork", [], [])):
        both(t, m, what, *args)
    t.free([])
    t.extend([], 3)
    m.same_as(t)


def test_lists_are_refused_while_a_graph_is_captured(monkeypatch):
    t, m = make(10, 4, 4)
    both(t, m, "extend", [0], [70])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: t.extend([0], 1), lambda: t.truncate([0], [1]), lambda: t.fork([0], [1]), lambda: t.free([0])):
        with pytest.raises(ValueError, match="device tensor"):
            call()
    monkeypatch.undo()
    m.same_as(t)


def test_wrapped_slice_and_other_stream():
    from ffa_speedtest_b200.pages import PageTable
    big = torch.full((7, 20), 99, dtype=torch.int32, device="cuda")
    view = big[1:6, 3:9]
    view.fill_(-1)
    pool = torch.randint(0, 256, (30, PAGE, 32), device="cuda", dtype=torch.uint8)
    t = PageTable.wrap(view, torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(30, dtype=torch.int32, device="cuda"), pools=[pool])
    m = Model(30, 5, 6, [pool])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        t.extend([0, 4], [100, 70])
        t.fork([0], [2])
        t.extend([2, 0], [1, 1])
        t.free([4])
        t.compact()
    s.synchronize()
    m.extend([0, 4], [100, 70])
    m.fork([0], [2])
    m.extend([2, 0], [1, 1])
    m.truncate([4], [0])
    m.compact()
    m.same_as(t)
    edge = big.clone()
    edge[1:6, 3:9] = 99
    assert bool((edge == 99).all())


def test_captured_step():
    """Free, fork and extend as one graph, replayed over lengths that change between the replays."""
    t, m = make(60, 6, 12)
    both(t, m, "extend", [0], [150])
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    child, parent, zero, new = dev([1, 2, 3]), dev([0, 0, 0]), dev([0, 0, 0]), dev([5, 5, 5])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t.truncate(child, zero)
        t.fork(parent, child)
        t.extend(child, new)
    m.same_as(t)                                              # capturing ran nothing
    for n in (5, 200, 64):
        new.fill_(n)
        g.replay()
        m.truncate([1, 2, 3], [0] * 3)
        m.fork([0] * 3, [1, 2, 3])
        m.extend([1, 2, 3], [n] * 3)
        m.same_as(t)
        both(t, m, "extend", [0], [1])


def test_more_pages_than_32_bits_count_are_refused():
    from ffa_speedtest_b200.pages import PageTable
    t = PageTable(50, 2500, 900000)                           # 2.25e9 pages asked for
    seqs = torch.arange(2500, dtype=torch.int32, device="cuda")
    t.extend(seqs, 900000 * PAGE)
    assert t.status() == 2 and int(t.seq_lens.max()) == 0 and int(t.refcount.max()) == 0


def test_a_length_below_zero_is_refused():
    from ffa_speedtest_b200.pages import PageTable
    lens = torch.tensor([0, -70], dtype=torch.int32, device="cuda")
    bt, rc = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    t = PageTable.wrap(bt, lens, rc)
    t.extend([0, 1], 1)
    assert t.status() == 1 and lens.tolist() == [0, -70] and int(bt.max()) == -1 and int(rc.max()) == 0


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 63, 2 ** 31 - 64, 200, 130])
def test_a_new_length_above_the_present_one_changes_nothing(length):
    from ffa_speedtest_b200.pages import PageTable
    t, m = make(12, 4, 6)
    both(t, m, "extend", [1, 2], [130, 64])
    both(t, m, "truncate", [1, 2, 0], [length, length, length])
    both(t, m, "truncate", [1, 1], [length, 70])              # the smaller of two
    t.check()
    # a wrapped length that the table cannot hold: shortened, and only the row's own columns are touched
    bt, rc = torch.tensor([[0, 1], [2, -1]], dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    lens = torch.tensor([2 ** 31 - 1, 64], dtype=torch.int32, device="cuda")
    PageTable.wrap(bt, lens, rc).truncate([0], [64])
    assert bt.tolist() == [[0, -1], [2, -1]] and lens.tolist() == [64, 64] and rc.tolist() == [1, 0, 1]


def test_capture_with_a_copy_between_the_calls():
    t, m = make(30, 4, 8)
    host = torch.tensor([70, 3], dtype=torch.int32).pin_memory()
    new, seqs = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t.truncate(seqs, zero)
        new.copy_(host, non_blocking=True)
        t.extend(seqs, new)
        new.add_(1)
        t.extend(seqs, new)
    for a, b in ((70, 3), (1, 130)):
        host.copy_(torch.tensor([a, b], dtype=torch.int32))
        g.replay()
        m.truncate([0, 3], [0, 0])
        m.extend([0, 3], [a, b])
        m.extend([0, 3], [a + 1, b + 1])
        m.same_as(t)


# ---- ragged append ------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fp8", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("B,T,HKV", [(1, 1, 1), (3, 70, 5), (17, 3, 8)])
def test_append_ragged(dtype, fp8, B, T, HKV):
    from ffa_speedtest_b200.pages import append_ragged_fp8fp8
    from ffa_speedtest_b200.quantize import quantize_k_fp8_fp8_residual
    g = torch.Generator(device="cuda").manual_seed(B)
    cols = 6
    k = torch.randn(B, T, HKV, 256, generator=g, device="cuda").to(dtype)[..., ::2]     # strided
    v = torch.randn(B, HKV, T, 128, generator=g, device="cuda").to(dtype).transpose(1, 2)
    wide = torch.randperm(B * (cols + 1), generator=g, device="cuda").to(torch.int32).view(B, cols + 1)
    table = wide[:, :cols]
    table[0, 2] = -1                                                                    # a page that is not there
    pos = torch.tensor([(i * 53) % (cols * PAGE) for i in range(B)], dtype=torch.int32, device="cuda")
    pos[-1] = cols * PAGE - 2 if B > 1 else 5                                           # runs past the table
    counts = torch.tensor([T - i % (T + 1) for i in range(B)], dtype=torch.int32, device="cuda")
    shape = (B * (cols + 1), PAGE, HKV, 128)
    base, res = torch.full(shape, 1.5, device="cuda").to(fp8), torch.full(shape, -2.0, device="cuda").to(fp8)
    vp = torch.full(shape, 7.0, device="cuda", dtype=dtype)
    want = [base.clone(), res.clone(), vp.clone()]
    kb, kr = quantize_k_fp8_fp8_residual(k.contiguous(), fp8)
    for b in range(B):
        for t in range(int(counts[b])):
            p = int(pos[b]) + t
            page = int(table[b, p // PAGE]) if p < cols * PAGE else -1
            if page >= 0:
                for w, x in zip(want, (kb, kr, v)):
                    w[page, p % PAGE] = x[b, t]
    append_ragged_fp8fp8(k, v, base, res, vp, table, pos, counts)
    for a, b in zip((base, res, vp), want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    append_ragged_fp8fp8(k[:, :0], v[:, :0], base, res, vp, table, pos)                 # nothing to do


def test_append_ragged_refusals():
    from ffa_speedtest_b200.pages import append_ragged_fp8fp8
    mk = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda").to(dt)
    f8 = torch.float8_e5m2
    pool, vp = mk(4, PAGE, 2, 128, dt=f8), mk(4, PAGE, 2, 128)
    k, v = mk(2, 1, 2, 128), mk(2, 1, 2, 128)
    bt, pos = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in [(k.float(), v.float(), pool, pool, vp, bt, pos), (k, v[:1], pool, pool, vp, bt, pos), (k, v, vp, pool, vp, bt, pos),
                (k, v, pool, pool.float().to(torch.float8_e4m3fn), vp, bt, pos), (k, v, pool, pool, vp.half(), bt, pos),
                (k, v, pool, pool, vp, bt.long(), pos), (k, v, pool, pool, vp, bt, pos.long()), (k, v, pool, pool, vp, bt[:1], pos),
                (k, v, pool, pool, vp, bt, pos[:1]), (k.cpu(), v.cpu(), pool, pool, vp, bt, pos),
                (k, v, pool, pool, vp, bt.cpu(), pos), (k, v, pool[:, :32], pool[:, :32], vp[:, :32], bt, pos)]:
        with pytest.raises(ValueError):
            append_ragged_fp8fp8(*bad)
