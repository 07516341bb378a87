"""Cases for serving many continuations of one prompt from the paged fp8 + fp8-residual cache.

Four operators of the package, each with a plain torch form beside it:

* ``attend``: one decode step of a batch whose sequences fall into groups that share leading pages (samples of
  one prompt); the shared pages are attended to once for the whole group, the rest of each sequence on its own;
* ``append``: K and V of new tokens, quantised and written at each sequence's own position;
* ``admit``: sequences that end give their pages back, new ones are forked from prompts and get room for new
  tokens, the shared open page copied on first write;
* ``compact``: live pages moved down into the free ones, block table and reference counts rewritten.

The cache is ``[pages, 64, kv-heads, 128]`` per tensor: fp8 base and fp8 residual of K (K = base + residual), V
in 16 bits.  Sizes are those of the package's decode benchmark (32 query heads, 8 kv-heads, head dimension 128,
4K to 128K tokens) and of its end-to-end tests (4 query heads, 2 kv-heads), with odd ones between.
"""
import math

import torch

own = False

PAGE, D = 64, 128
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
F16 = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases ------------------------------------------------------------------------------------------

def listed():
    return [
        # two samples of a one-page prompt on a small model: nothing but launch and latency
        attend("attend 2 samples, 128 tokens", "2", "2", 1, 5, 4, 2, "bf16", "e5m2"),
        # the usual serving step: eight samples of a 32K prompt, each some hundred tokens on
        attend("attend 8 samples of 32K", "8", "512", 1, 700, 32, 8, "bf16", "e5m2"),
        # 32 samples of a 16K prompt in float16: 128 query rows for each kv-head
        attend("attend 32 samples of 16K", "32", "256", 200, 1000, 32, 8, "fp16", "e4m3"),
        # a mixed batch: prompts of odd lengths with one to sixteen samples each, one without a shared part (and
        # sequences that hold nothing yet), a group of three query heads to a kv-head
        attend("attend ragged prompts", "1,5,16,2,9", "37,0,255,100,7", 0, 333, 24, 8, "bf16", "e4m3"),
        # sixteen unrelated sequences of different lengths: no page is shared
        attend("attend 16 private", ",".join(["1"] * 16), ",".join(["0"] * 16), 4000, 9000, 32, 8, "bf16", "e5m2"),
        # the largest: 64 samples of a 128K prompt, 256 query rows for each kv-head
        attend("attend 64 samples of 128K", "64", "2048", 1, 2000, 32, 8, "bf16", "e4m3"),
        # one decode step of 64 sequences: one token each, at 64 different positions
        append("append 64 x 1", 64, 1, 3000, 8, "bf16", "e5m2", 1),
        # prompts of odd lengths, padded to the longest, into the cache
        append("append 8 ragged prompts", 8, 8191, 100, 8, "fp16", "e4m3", 0),
        # four samples replaced in one layer of a small model
        admit("admit 4 of 1K, 1 layer", 1, 1000, 4, 1, 1, 2),
        # 64 samples replaced by new ones of two 32K prompts, eight layers
        admit("admit 64 of 32K, 8 layers", 2, 32700, 64, 4, 8, 8),
        # a small pool, a quarter of it free
        compact("compact 200 pages", 200, 150, 6, 1, 2),
        # half of a pool of four layers in use, and scattered
        compact("compact 2000 pages, 4 layers", 2000, 1100, 40, 4, 8),
    ]


def attend(name, groups, prefix, lo, hi, hq, hkv, dtype, fp8):
    return {"name": name, "kind": "attend", "groups": groups, "prefix_pages": prefix, "suffix_from": lo, "suffix_to": hi,
            "hq": hq, "hkv": hkv, "dtype": dtype, "fp8": fp8}


def append(name, batch, new, held, hkv, dtype, fp8, full):
    return {"name": name, "kind": "append", "batch": batch, "new": new, "held": held, "hkv": hkv, "dtype": dtype,
            "fp8": fp8, "full": full}


def admit(name, prompts, tokens, children, new, layers, hkv):
    return {"name": name, "kind": "admit", "prompts": prompts, "tokens": tokens, "children": children, "new": new,
            "layers": layers, "hkv": hkv}


def compact(name, pages, live, seqs, layers, hkv):
    return {"name": name, "kind": "compact", "pages": pages, "live": live, "seqs": seqs, "layers": layers, "hkv": hkv}


def draw(rng):
    def log(lo, hi):
        return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind = rng.choice(["attend", "attend", "attend", "append", "admit", "compact"])
    hkv = rng.choice([1, 2, 5, 8])
    if kind == "attend":
        n = rng.choice([1, 1, 2, 3, 7, 16])
        total = log(n, 64)
        cuts = sorted(rng.randint(0, total - n) for _ in range(n - 1))
        sizes = [b - a + 1 for a, b in zip([0] + cuts, cuts + [total - n])]
        pages = [rng.choice([0, 1]) * log(1, 2048 // n) if n > 1 else log(1, 2048) for _ in range(n)]
        lo = rng.choice([0, 1, 60])
        c = attend("", ",".join(map(str, sizes)), ",".join(map(str, pages)), lo, lo + log(1, 1900), hkv * rng.choice([1, 2, 3, 4, 8]) if hkv < 8
                   else rng.choice([8, 24, 32]), hkv, rng.choice(["bf16", "fp16"]), rng.choice(["e4m3", "e5m2"]))
    elif kind == "append":
        b = log(1, 64)
        c = append("", b, log(1, 65536 // b), log(1, 4096), hkv, rng.choice(["bf16", "fp16"]), rng.choice(["e4m3", "e5m2"]), rng.choice([0, 1]))
    elif kind == "admit":
        p = rng.choice([1, 2, 3])
        c = admit("", p, log(1, 32700), p * log(1, 21), log(1, 200), rng.choice([1, 2, 8]), hkv)
    else:
        pages = log(16, 2000)
        live = max(4, int(pages * rng.uniform(0.1, 0.95)))
        c = compact("", pages, live, rng.randint(1, min(40, live)), rng.choice([1, 3, 4]), hkv)
    del c["name"]
    return c


def ints(text):
    return [int(x) for x in text.split(",")]


def spread(lo, hi, n):
    """n numbers of lo..hi in no order, the same for the same arguments."""
    return [lo + (i * 7919 + i * i * 31) % (hi - lo + 1) for i in range(n)]


# ---- inputs -----------------------------------------------------------------------------------------

def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def tensor(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


def encode(k, fp8):
    """K of a 16-bit type as fp8 base and fp8 residual."""
    base = k.to(fp8)
    return base, (k.float() - base.float()).to(fp8)


def pools(g, layers, pages, hkv, dtype, fp8):
    """Base, residual and V of every layer, ``[layers, pages, 64, kv-heads, 128]``, channels of K of unequal size."""
    size = torch.exp(0.5 * randn(g, hkv, D)).to(dtype)
    k = [encode(randn(g, pages, PAGE, hkv, D, dtype=dtype) * size, fp8) for _ in range(layers)]
    v = torch.empty(layers, pages, PAGE, hkv, D, device="cuda", dtype=dtype).normal_(generator=g)
    return torch.stack([x[0] for x in k]), torch.stack([x[1] for x in k]), v


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "attend":
        sizes, shared = ints(case["groups"]), ints(case["prefix_pages"])
        B, hkv = sum(sizes), case["hkv"]
        more = spread(case["suffix_from"], case["suffix_to"], B)
        of = [i for i, n in enumerate(sizes) for _ in range(n)]
        lens = [shared[of[b]] * PAGE + more[b] for b in range(B)]
        cols = max(1, max(-(-n // PAGE) for n in lens))
        n_pages = sum(shared) + sum(-(-n // PAGE) for n in more) + 3
        place = torch.randperm(n_pages, generator=host).tolist()
        at, rows, first = 0, [], []
        for n in shared:
            first.append(place[at:at + n])
            at += n
        for b in range(B):
            n = -(-more[b] // PAGE)
            rows.append((first[of[b]] + place[at:at + n] + [-1] * cols)[:cols])
            at += n
        k, r, v = pools(g, 1, n_pages, hkv, F16[case["dtype"]], FP8[case["fp8"]])
        start = [0]
        for n in sizes:
            start.append(start[-1] + n)
        s |= {"k": k[0], "r": r[0], "v": v[0], "q": 2.0 * randn(g, B, 1, case["hq"], D, dtype=F16[case["dtype"]]), "block_table": tensor(rows),
              "seq_lens": tensor(lens), "group_start": tensor(start), "prefix_pages": tensor(shared)}
    elif case["kind"] == "append":
        B, T, hkv, dt = case["batch"], case["new"], case["hkv"], F16[case["dtype"]]
        at = spread(0, case["held"], B)
        cols = -(-(max(at) + T) // PAGE)
        place = torch.randperm(B * cols, generator=host).view(B, cols)
        shape = (B * cols, PAGE, hkv, D)
        s |= {"k_new": randn(g, B, T, hkv, D, dtype=dt) * torch.exp(0.5 * randn(g, hkv, D)).to(dt), "v_new": randn(g, B, T, hkv, D, dtype=dt),
              "k": torch.zeros(shape, device="cuda", dtype=FP8[case["fp8"]]), "r": torch.zeros(shape, device="cuda", dtype=FP8[case["fp8"]]),
              "v": torch.zeros(shape, device="cuda", dtype=dt), "block_table": place.to(torch.int32).cuda(), "positions": tensor(at),
              "counts": tensor([T] * B if case["full"] else spread(T - T // 2, T, B))}
    elif case["kind"] == "admit":
        P, n, L = case["prompts"], case["children"], case["layers"]
        lens = [case["tokens"] - min(case["tokens"] - 1, 37 * p) for p in range(P)]
        held = [-(-x // PAGE) for x in lens]
        cols = -(-(max(lens) + case["new"]) // PAGE)
        n_pages = sum(held) + n * (1 - (-case["new"] // PAGE) + 1)
        place = torch.randperm(n_pages, generator=host)[:sum(held)]
        table = torch.full((P + n, cols), -1, dtype=torch.int32)
        at = 0
        for p in range(P):
            table[p, :held[p]] = place[at:at + held[p]]
            at += held[p]
        count = torch.zeros(n_pages, dtype=torch.int32)
        count[place] = 1
        k, r, v = pools(g, L, n_pages, case["hkv"], torch.bfloat16, torch.float8_e5m2)
        s |= {"k": k, "r": r, "v": v, "block_table": table.cuda(), "refcount": count.cuda(), "seq_lens": tensor(lens + [0] * n),
              "children": torch.arange(P, P + n, dtype=torch.int32).cuda(), "parents": (torch.arange(n, dtype=torch.int32) * P // n).cuda(),
              "none": torch.zeros(n, dtype=torch.int32).cuda(), "new": torch.full((n,), case["new"], dtype=torch.int32).cuda()}
    else:
        live, n = case["live"], case["seqs"]
        place = torch.randperm(case["pages"], generator=host)[:live].to(torch.int32)
        held = [live // n + (i < live % n) for i in range(n)]
        table = torch.full((n + 2, max(held) + 1), -1, dtype=torch.int32)
        at = 0
        for i in range(n):
            table[i, :held[i]] = place[at:at + held[i]]
            at += held[i]
        table[n] = table[0]                                             # a forked sequence holds the first one's pages too
        count = torch.zeros(case["pages"], dtype=torch.int32)
        count[place.long()] = 1
        count[table[0, :held[0]].long()] = 2
        k, r, v = pools(g, case["layers"], case["pages"], case["hkv"], torch.bfloat16, torch.float8_e4m3fn)
        s |= {"k": k, "r": r, "v": v, "block_table": table.cuda(), "refcount": count.cuda(),
              "seq_lens": tensor([h * PAGE - 5 for h in held] + [held[0] * PAGE - 5, 0]),
              "table_out": table.cuda(), "count_out": count.cuda()}
    return s


# ---- the operators ----------------------------------------------------------------------------------

def run(s):
    return {"attend": run_attend, "append": run_append, "admit": run_admit, "compact": run_compact}[s["case"]["kind"]](s)


def run_attend(s):
    if own:
        from ffa_speedtest_b200.fp8fp8.attn_kernel import attn_kernel_shared_prefix_fp8fp8 as m
        if "workspace" not in s:
            s["workspace"] = m.allocate_shared_prefix_workspace(s["q"], s["v"])
        return m.attn_forward_decode_shared_prefix_fp8fp8(
            s["q"], s["k"], s["v"], k_residual=s["r"], block_table=s["block_table"], seq_lens=s["seq_lens"],
            group_start=s["group_start"], prefix_pages=s["prefix_pages"], workspace=s["workspace"])
    sizes, shared = ints(s["case"]["groups"]), ints(s["case"]["prefix_pages"])
    B, NG, big, hkv = sum(sizes), len(sizes), max(sizes), s["case"]["hkv"]
    G = s["case"]["hq"] // hkv
    start, bt, lens, pre = s["group_start"].long(), s["block_table"].long(), s["seq_lens"].long(), s["prefix_pages"].long()
    seq = torch.arange(B, device="cuda")
    grp = torch.searchsorted(start[1:], seq, right=True)                # the group of each sequence and its place in it
    member = seq - start[grp]
    q = s["q"].view(B, hkv, G, D).float() / math.sqrt(D)
    # shared part: every group's queries against the group's pages
    n_pre, n_own = max(shared), max(1, -(-s["case"]["suffix_to"] // PAGE))
    top = torch.zeros(B, hkv, G, 1, device="cuda") - math.inf
    if n_pre:
        pages = bt[start[:-1], :n_pre].clamp(min=0)
        k = (s["k"][pages].float() + s["r"][pages].float()).view(NG, n_pre * PAGE, hkv, D).permute(0, 2, 3, 1)
        qg = torch.zeros(NG, big, hkv, G, D, device="cuda")
        qg[grp, member] = q
        dots = torch.matmul(qg.permute(0, 2, 1, 3, 4).reshape(NG, hkv, big * G, D), k).view(NG, hkv, big, G, n_pre * PAGE)
        beyond = torch.arange(n_pre * PAGE, device="cuda") >= (pre * PAGE)[:, None]
        dots.masked_fill_(beyond[:, None, None, None], -math.inf)
        top = dots.amax(-1)[grp, :, member].unsqueeze(-1)
    # each sequence's own part
    col = pre[grp][:, None] + torch.arange(n_own, device="cuda")
    pages = bt.gather(1, col.clamp(max=bt.shape[1] - 1)).clamp(min=0)
    k = (s["k"][pages].float() + s["r"][pages].float()).view(B, n_own * PAGE, hkv, D).permute(0, 2, 3, 1)
    mine = torch.matmul(q, k)
    beyond = torch.arange(n_own * PAGE, device="cuda") >= (lens - pre[grp] * PAGE)[:, None]
    mine.masked_fill_(beyond[:, None, None], -math.inf)
    top = torch.maximum(top, mine.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)     # a sequence that holds nothing
    mine = (mine - top).exp_()
    v = s["v"][pages].float().view(B, n_own * PAGE, hkv, D).masked_fill_(beyond[:, :, None, None], 0).transpose(1, 2)
    total, o = mine.sum(-1, keepdim=True), torch.matmul(mine, v)
    if n_pre:
        tops = torch.zeros(NG, hkv, big, G, 1, device="cuda")
        tops[grp, :, member] = top
        dots = (dots - tops).exp_()
        pages = bt[start[:-1], :n_pre].clamp(min=0)
        v = s["v"][pages].float().view(NG, n_pre * PAGE, hkv, D).permute(0, 2, 1, 3)
        total = total + dots.sum(-1, keepdim=True)[grp, :, member]
        o = o + torch.matmul(dots.view(NG, hkv, big * G, -1), v).view(NG, hkv, big, G, D)[grp, :, member]
    return torch.where(total > 0, o / total, torch.zeros_like(o)).view(B, hkv * G, D).to(s["q"].dtype)


def run_append(s):
    if own:
        from ffa_speedtest_b200.pages import append_ragged_fp8fp8
        append_ragged_fp8fp8(s["k_new"], s["v_new"], s["k"], s["r"], s["v"], s["block_table"], s["positions"], s["counts"])
    else:
        B, T, hkv = s["k_new"].shape[:3]
        t = torch.arange(T, device="cuda")
        pos = s["positions"].long()[:, None] + t
        row = s["block_table"].long().gather(1, pos // PAGE) * PAGE + pos % PAGE
        row = row[t < s["counts"][:, None]]
        new = s["k_new"][t < s["counts"][:, None]]
        base, res = encode(new, s["k"].dtype)
        s["k"].view(torch.uint8).view(-1, hkv, D)[row] = base.view(torch.uint8)
        s["r"].view(torch.uint8).view(-1, hkv, D)[row] = res.view(torch.uint8)
        s["v"].view(-1, hkv, D)[row] = s["v_new"][t < s["counts"][:, None]]
    return {"base": s["k"], "residual": s["r"], "v": s["v"]}


def page_table(s):
    """The handle that a program keeps beside its pools."""
    from ffa_speedtest_b200.pages import PageTable
    if "handle" not in s:
        layers = [x for three in zip(s["k"], s["r"], s["v"]) for x in three]
        s["handle"] = PageTable.wrap(s["block_table"], s["seq_lens"], s["refcount"], pools=layers)
    return s["handle"]


def run_admit(s):
    if own:
        t = page_table(s)
        t.truncate(s["children"], s["none"])
        t.fork(s["parents"], s["children"])
        t.extend(s["children"], s["new"])
    else:
        table, lens, count = s["block_table"], s["seq_lens"], s["refcount"]
        child, parent, n = s["children"].long(), s["parents"].long(), s["children"].shape[0]
        rows = table[child]                                             # pages of the sequences that end
        count.index_add_(0, rows.clamp(min=0).flatten().long(), -(rows >= 0).flatten().int())
        rows = table[parent]                                            # and of the prompts that the new ones begin with
        count.index_add_(0, rows.clamp(min=0).flatten().long(), (rows >= 0).flatten().int())
        old = lens[parent]
        last = rows.gather(1, ((old - 1).clamp(min=0) // PAGE).long()[:, None])[:, 0].long()
        col = torch.arange(table.shape[1], device="cuda")
        opened = (old % PAGE != 0) & (count[last] > 1)
        fresh = (col >= ((old + 63) // PAGE)[:, None]) & (col < ((old + s["new"] + 63) // PAGE)[:, None])
        fresh |= opened[:, None] & (col == (old // PAGE)[:, None])
        free = torch.argsort((count != 0).int(), stable=True)           # free pages first, lowest first
        page = free[(fresh.flatten().cumsum(0) - 1).clamp(min=0)].view(n, -1)
        count.index_add_(0, last, -opened.int())
        count.index_add_(0, torch.where(fresh, page, 0).flatten(), fresh.flatten().int())
        rows = torch.where(fresh, page.int(), rows)
        table[child] = rows
        lens[child] = old + s["new"]
        to = rows.gather(1, ((old - 1).clamp(min=0) // PAGE).long()[:, None])[:, 0].long()
        token = torch.arange(PAGE, device="cuda")
        which = (token < (old % PAGE)[:, None]) & opened[:, None]
        src, dst = (last[:, None] * PAGE + token)[which], (to[:, None] * PAGE + token)[which]
        x = s["k"].view(torch.uint8).flatten(1, 2)
        x[:, dst] = x[:, src]
        x = s["r"].view(torch.uint8).flatten(1, 2)
        x[:, dst] = x[:, src]
        x = s["v"].flatten(1, 2)
        x[:, dst] = x[:, src]
    return {"table": s["block_table"], "lens": s["seq_lens"], "count": s["refcount"], "base": s["k"], "residual": s["r"], "v": s["v"]}


def run_compact(s):
    if own:
        page_table(s).compact(block_table_out=s["table_out"], refcount_out=s["count_out"])
    else:
        used = s["refcount"] != 0
        number = torch.arange(used.shape[0], device="cuda")
        live = used.sum()
        src, dst = number[used & (number >= live)], number[~used & (number < live)]
        to = number.int()
        to[src] = dst.int()
        table = s["block_table"]
        s["table_out"].copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
        s["count_out"].copy_(s["refcount"])
        s["count_out"][dst] = s["refcount"][src]
        s["count_out"][src] = 0
        x = s["k"].view(torch.uint8)
        x[:, dst] = x[:, src]
        x = s["r"].view(torch.uint8)
        x[:, dst] = x[:, src]
        x = s["v"]
        x[:, dst] = x[:, src]
    return {"table": s["table_out"], "count": s["count_out"], "base": s["k"], "residual": s["r"], "v": s["v"]}


# ---- what a pass cannot do without ------------------------------------------------------------------

def work(case):
    row = case["hkv"] * D * 4                                           # bytes of one token: base, residual, V
    if case["kind"] == "attend":
        sizes, shared = ints(case["groups"]), ints(case["prefix_pages"])
        more = spread(case["suffix_from"], case["suffix_to"], sum(sizes))
        tokens = sum(shared) * PAGE + sum(more)
        pairs = sum(n * p * PAGE for n, p in zip(sizes, shared)) + sum(more)
        return {"bytes": tokens * row + 4 * sum(sizes) * case["hq"] * D, "flops": 4.0 * pairs * case["hq"] * D}
    if case["kind"] == "append":
        T = case["new"]
        tokens = case["batch"] * T if case["full"] else sum(spread(T - T // 2, T, case["batch"]))
        return {"bytes": 2 * tokens * row, "flops": 3.0 * tokens * case["hkv"] * D}
    if case["kind"] == "admit":
        lens = [case["tokens"] - min(case["tokens"] - 1, 37 * p) for p in range(case["prompts"])]
        per = case["children"] // case["prompts"]
        rows = sum(per * (x % PAGE) for x in lens)
        entries = sum(per * -(-x // PAGE) for x in lens)
        return {"bytes": 2 * rows * row * case["layers"] + 8 * entries, "flops": 0}
    moved = case["live"] * (case["pages"] - case["live"]) // case["pages"]
    return {"bytes": 2 * moved * PAGE * row * case["layers"] + 16 * case["live"] + 8 * case["pages"], "flops": 0}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "attend":
        s = prepare(case, seed)
        hkv, B = case["hkv"], s["q"].shape[0]
        out = torch.zeros(B, case["hq"], D, device="cuda", dtype=torch.float64)
        for b in range(B):
            n = int(s["seq_lens"][b])
            if n:
                pages = s["block_table"][b, :-(-n // PAGE)].long()
                for h in range(hkv):
                    k = s["k"][:, :, h][pages].flatten(0, 1)[:n].double() + s["r"][:, :, h][pages].flatten(0, 1)[:n].double()
                    heads = slice(h * case["hq"] // hkv, (h + 1) * case["hq"] // hkv)
                    w = torch.softmax(s["q"][b, 0, heads].double() @ k.T / math.sqrt(D), -1)
                    out[b, heads] = w @ s["v"][:, :, h][pages].flatten(0, 1)[:n].double()
        return out
    if case["kind"] == "append":
        s = prepare(case, seed)
        mantissa, least, most = (3, -6, 448.0) if case["fp8"] == "e4m3" else (2, -14, 57344.0)

        def nearest(x):
            step = torch.exp2(torch.frexp(x)[1].double() - 1).clamp(min=2.0 ** least) * 2.0 ** -mantissa
            return (x / step).round().mul(step).clamp(-most, most)      # to even where two are as near

        out = {"base": torch.zeros(s["k"].shape, device="cuda", dtype=torch.float64), "v": None}
        out["residual"] = torch.zeros_like(out["base"])
        for b in range(case["batch"]):
            n, at = int(s["counts"][b]), int(s["positions"][b])
            pos = torch.arange(at, at + n, device="cuda")
            page, slot = s["block_table"][b].long()[pos // PAGE], pos % PAGE
            x = s["k_new"][b, :n].double()
            out["base"][page, slot] = nearest(x)
            out["residual"][page, slot] = nearest(x - nearest(x))
        return out
    return None                                                         # page numbers and copies: whole values
