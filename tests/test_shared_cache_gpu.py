"""Prompts, forks, decode steps and page management together, through the model and the cache that it uses."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from ffa_speedtest_b200.fp8fp8.e2e.modeling_llama import DenseCache, LlamaConfig, LlamaForCausalLM
from ffa_speedtest_b200.fp8fp8.e2e.shared_cache import SharedPrefixFP8Fp8Cache

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def build(layers=2, heads=4, kv=2, vocab=97, seed=0):
    torch.manual_seed(seed)
    cfg = LlamaConfig(hidden_size=128 * heads, num_attention_heads=heads, num_key_value_heads=kv, num_hidden_layers=layers,
                      max_position_embeddings=512, vocab_size=vocab)
    return cfg, LlamaForCausalLM(cfg).to(device="cuda", dtype=torch.bfloat16).eval()


def dense_logits(model, cfg, tokens):
    """Logits of the last token of each of the token lists, one dense run each."""
    out = []
    for t in tokens:
        cache = DenseCache(1, cfg.num_key_value_heads, 512, 128, torch.bfloat16, "cuda")
        out.append(model(torch.tensor([t], device="cuda"), past_key_values=cache, use_cache=True)[0, -1])
    return torch.stack(out).float()


def close(got, ref):
    # K is held as fp8 base + fp8 residual, as in the tests of the other cache: logits within 2 % of their largest
    assert bool(torch.isfinite(got).all())
    assert float((got.float() - ref).abs().max()) <= 2e-2 * max(1.0, float(ref.abs().max()))


def test_samples_of_two_prompts_track_the_dense_model():
    """Two prompts, three samples of the first and two of the second; one of each ends and is replaced by a fork of another
    sample, the pages are compacted, and everything goes on."""
    cfg, model = build()
    g = torch.Generator().manual_seed(1)
    draw = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()
    cache = SharedPrefixFP8Fp8Cache(9, 2, 512, num_layers=2, n_pages=40, fp8_dtype=torch.float8_e4m3fn)
    text = {0: draw(150), 1: draw(70)}
    for p in (0, 1):                                        # prompts of different lengths, one after the other
        cache.activate([p])
        logits = model(torch.tensor([text[p]], device="cuda"), past_key_values=cache, use_cache=True)[:, -1]
        close(logits, dense_logits(model, cfg, [text[p]]))
    cache.fork([0, 0, 0, 1, 1], [2, 3, 4, 5, 6])
    text.update({c: list(text[p]) for p, c in zip((0, 0, 0, 1, 1), (2, 3, 4, 5, 6))})

    def steps(seqs, n):
        cache.activate(seqs)
        for _ in range(n):
            new = draw(len(seqs))
            for s, x in zip(seqs, new):
                text[s].append(x)
            logits = model(torch.tensor(new, device="cuda")[:, None], past_key_values=cache, use_cache=True)[:, -1]
        close(logits, dense_logits(model, cfg, [text[s] for s in seqs]))
        assert [cache.lengths[s] for s in seqs] == cache.table.seq_lens[torch.tensor(seqs, device="cuda")].tolist()

    steps([2, 3, 4, 5, 6], 1)                               # open pages are shared: all write at once
    steps([2, 3, 4, 5, 6], 60)                              # past page boundaries
    steps([6, 5, 0, 3], 7)                                  # the prompt itself and its sample, out of order
    cache.free([2, 5])
    cache.fork([3, 6], [2, 5])                              # forks of forks
    text[2], text[5] = list(text[3]), list(text[6])
    before = cache.table.free_pages()
    cache.compact()
    assert cache.table.free_pages() == before
    live = 40 - before
    assert int((cache.table.refcount[:live] > 0).sum()) == live
    steps([2, 3, 4, 5, 6], 9)
    cache.truncate([3, 4], [100, 200])                      # drafts rejected, one inside the shared pages
    del text[3][100:], text[4][200:]
    steps([0, 2, 3, 4], 5)
    cache.truncate([2, 4], [64, 130])                       # while they are active: the next step must not use the old groups
    del text[2][64:], text[4][130:]
    for s in (0, 2, 3, 4):
        text[s].append(5)
    logits = model(torch.full((4, 1), 5, device="cuda"), past_key_values=cache, use_cache=True)[:, -1]
    close(logits, dense_logits(model, cfg, [text[s] for s in (0, 2, 3, 4)]))
    cache.check()


def test_runs_out_of_pages_and_says_so():
    cache = SharedPrefixFP8Fp8Cache(3, 2, 512, num_layers=1, n_pages=4)
    cache.activate([0, 1])
    cache.extend(128)
    cache.check()
    cache.extend(1)                                         # two pages more than there are
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()


def test_without_pages_nothing_is_written_and_work_goes_on():
    """A step that finds no page may not touch a token of any sequence; after the check the lengths are the device's."""
    cfg, model = build()
    g = torch.Generator().manual_seed(5)
    draw = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()
    for seqs in ([0, 1, 2], [2, 0, 1]):                     # side by side in the table, and not
        cache = SharedPrefixFP8Fp8Cache(4, 2, 512, num_layers=2, n_pages=4, fp8_dtype=torch.float8_e4m3fn)
        text = {0: draw(100)}
        cache.activate([0])
        model(torch.tensor([text[0]], device="cuda"), past_key_values=cache, use_cache=True)
        cache.fork([0, 0], [1, 2])                          # the open page is shared by three: two copies are needed, both there are
        cache.truncate([1], [90])                           # its next token falls into a token of the others
        text[1], text[2] = text[0][:90], list(text[0])
        cache.fork([0], [3])
        cache.activate(seqs)
        pools = [x.clone() for x in cache.table.pools]
        state = cache.table.seq_lens.clone()
        model(torch.full((3, 1), 3, device="cuda"), past_key_values=cache, use_cache=True)          # three copies: one too many
        with pytest.raises(RuntimeError, match="free pages"):
            cache.check()
        assert torch.equal(cache.table.seq_lens, state) and cache.lengths == state.tolist()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pools, cache.table.pools))
        cache.free([3])
        cache.activate([1, 2])
        for s, x in ((1, 7), (2, 9)):
            text[s].append(x)
        logits = model(torch.tensor([[7], [9]], device="cuda"), past_key_values=cache, use_cache=True)[:, -1]
        cache.check()
        close(logits, dense_logits(model, cfg, [text[1], text[2]]))


def test_sharing_goes_on_after_running_out_of_pages():
    cfg, model = build()
    g = torch.Generator().manual_seed(6)
    draw = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()
    cache = SharedPrefixFP8Fp8Cache(6, 2, 512, num_layers=2, n_pages=9, fp8_dtype=torch.float8_e4m3fn)
    pages = lambda: (cache._group_start.tolist(), cache._prefix_pages.tolist())
    text = {0: draw(150), 5: draw(60)}
    for s in (0, 5):
        cache.activate([s])
        model(torch.tensor([text[s]], device="cuda"), past_key_values=cache, use_cache=True)
    cache.fork([0] * 3, [1, 2, 3])                          # four pages are held
    for s in (1, 2, 3):
        text[s] = list(text[0])

    def step(seqs):
        new = draw(len(seqs))
        logits = model(torch.tensor(new, device="cuda")[:, None], past_key_values=cache, use_cache=True)[:, -1]
        for s, x in zip(seqs, new):
            text[s].append(x)
        return logits

    seqs = [1, 2, 3, 5]
    cache.activate(seqs)
    for _ in range(4):                                      # three open pages are copied: two are left
        logits = step(seqs)
    close(logits, dense_logits(model, cfg, [text[s] for s in seqs]))
    for _ in range(39):                                     # one goes to sequence 5, and at 192 tokens the others need three
        step(seqs)
    cache.fork([2], [4])                                    # forked before anyone has noticed
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()
    assert cache.lengths == cache.table.seq_lens.tolist()
    for s in (*seqs, 4):
        text[s] = text[2 if s == 4 else s][:cache.lengths[s]]
    assert [cache.lengths[s] for s in (1, 2, 3, 4, 5)] == [192] * 4 + [102]
    cache.activate([1, 2, 4, 3, 5])
    assert pages() == ([0, 4, 5], [2, 0])                   # the prompt is read once still
    cache.free([0])
    cache.activate([1, 2, 4])
    assert pages() == ([0, 3], [2])
    step([1, 2, 4])
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()                                       # three are needed, two are free
    for s in (1, 2, 4):
        del text[s][-1:]
    cache.activate([2, 4])
    assert pages() == ([0, 2], [3])
    cache.free([1, 5])
    logits = step([2, 4])
    cache.check()
    close(logits, dense_logits(model, cfg, [text[s] for s in (2, 4)]))


def test_check_reports_an_attention_that_gave_up():
    """The word is set here by hand: no wait in the kernel depends on anything that a caller could hold back."""
    cache = SharedPrefixFP8Fp8Cache(4, 2, 256, num_layers=1)
    zeros = lambda b, h: torch.zeros(b, 1, h, 128, dtype=torch.bfloat16, device="cuda")

    def step(seqs):
        cache.activate(seqs)
        cache.extend(1)
        cache.update(zeros(len(seqs), 2), zeros(len(seqs), 2), 0)
        cache.decode(zeros(len(seqs), 4), 0)

    step([0, 1])
    cache.check()
    cache._workspace.status_word.fill_(1)
    with pytest.raises(RuntimeError, match="gave up"):
        cache.check()
    cache.check()                                           # reported once
    cache._workspace.status_word.fill_(1)
    step([2])                                               # another workspace in the meantime
    assert cache._workspace.status() == 0
    with pytest.raises(RuntimeError, match="gave up"):
        cache.check()
    cache.check()


def test_groups_through_forks_and_rejected_drafts():
    cache = SharedPrefixFP8Fp8Cache(6, 2, 1024, num_layers=1)
    pages = lambda: (cache._group_start.tolist(), cache._prefix_pages.tolist())
    cache.activate([0])
    cache.extend(200)
    cache.activate([0, 1, 2])
    assert pages() == ([0, 1, 2, 3], [0, 0, 0])
    cache.fork([0, 0], [1, 2])                              # while they are active
    assert pages() == ([0, 3], [3])
    cache.extend(70)
    cache.truncate([0, 1, 2], [210, 201, 199])              # behind what was forked: still one prompt
    assert pages() == ([0, 3], [3])
    cache.truncate([0], [190])                              # into it: the other two have its third page, it will have another
    assert pages() == ([0, 1, 3], [0, 3])
    cache.free([1, 2])
    cache.activate([1])
    cache.extend(130)                                       # a prompt in the place of a sample
    cache.fork([1], [2])
    cache.activate([1, 2, 0])
    assert pages() == ([0, 2, 3], [2, 0])
    cache.activate([3])
    cache.extend(20)
    cache.fork([3], [4])                                    # no full page to share; both go on by themselves
    cache.activate([3, 4])
    cache.extend(300)
    cache.fork([4], [5])
    cache.activate([3, 4, 5])
    assert pages() == ([0, 1, 3], [0, 5])
    cache.check()


def test_forks_of_a_grown_sample_share_what_it_wrote():
    cache = SharedPrefixFP8Fp8Cache(8, 2, 768, num_layers=1)
    pages = lambda: (cache._group_start.tolist(), cache._prefix_pages.tolist())
    cache.activate([0])
    cache.extend(200)
    cache.fork([0, 0], [1, 2])
    cache.activate([1])
    cache.extend(500)                                       # the sample is 700 tokens long, 200 of them the prompt's
    cache.fork([1, 1], [3, 4])
    cache.activate([1, 3, 4])
    assert pages() == ([0, 3], [10])
    cache.activate([1, 3, 4, 0, 2])
    assert pages() == ([0, 3, 5], [10, 3])
    cache.activate([1, 0, 3])                               # not side by side: the prompt is what they have in common
    assert pages() == ([0, 3], [3])
    cache.free([0, 2])                                      # the prompt's end changes nothing for them
    cache.activate([1, 3, 4])
    cache.extend(60)
    cache.fork([3], [5])
    cache.activate([1, 3, 5, 4])
    assert pages() == ([0, 4], [10])
    cache.activate([3, 5, 4])
    cache.extend(8)                                         # to the last token that a sequence can hold
    assert pages() == ([0, 3], [10])
    cache.activate([3, 5])
    assert pages() == ([0, 2], [11])
    cache.check()


def test_forks_of_grown_samples_track_the_dense_model():
    cfg, model = build()
    g = torch.Generator().manual_seed(3)
    draw = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()
    cache = SharedPrefixFP8Fp8Cache(8, 2, 512, num_layers=2, fp8_dtype=torch.float8_e4m3fn)
    text = {0: draw(140)}
    cache.activate([0])
    model(torch.tensor([text[0]], device="cuda"), past_key_values=cache, use_cache=True)

    def steps(seqs, n):
        cache.activate(seqs)
        for _ in range(n):
            new = draw(len(seqs))
            for s, x in zip(seqs, new):
                text[s].append(x)
            logits = model(torch.tensor(new, device="cuda")[:, None], past_key_values=cache, use_cache=True)[:, -1]
        close(logits, dense_logits(model, cfg, [text[s] for s in seqs]))

    def fork(parents, children):
        cache.fork(parents, children)
        for p, c in zip(parents, children):
            text[c] = list(text[p])

    fork([0, 0], [1, 2])
    steps([1, 2], 70)
    fork([1, 2, 1], [3, 4, 5])
    steps([1, 3, 5, 0, 2, 4], 3)
    assert (cache._group_start.tolist(), cache._prefix_pages.tolist()) == ([0, 6], [2])
    steps([1, 3, 5, 2, 4], 2)
    assert (cache._group_start.tolist(), cache._prefix_pages.tolist()) == ([0, 3, 5], [3, 3])
    steps([2, 1, 4, 3, 5], 66)                              # out of order
    cache.truncate([3, 4], [205, 150])
    del text[3][205:], text[4][150:]
    fork([3], [6])
    steps([6, 3, 1, 5, 4, 2], 61)
    cache.check()


def test_decode_needs_an_extend_after_the_pages_changed():
    cache = SharedPrefixFP8Fp8Cache(4, 2, 256, num_layers=1)
    q, k = torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device="cuda")
    for change in (lambda: cache.activate([0]), lambda: cache.truncate([0], [1]), cache.compact):
        cache.activate([0])
        cache.extend(1)
        cache.update(k, k, 0)
        cache.decode(q, 0)
        change()
        for call in (lambda: cache.decode(q, 0), lambda: cache.update(k, k, 0), cache.positions):
            with pytest.raises(RuntimeError, match="extend first"):
                call()


def test_refusals():
    cache = SharedPrefixFP8Fp8Cache(4, 2, 128, num_layers=1)
    with pytest.raises(RuntimeError, match="activate"):
        cache.extend(1)
    for bad in ([], [0, 0], [4], [-1]):
        with pytest.raises(ValueError):
            cache.activate(bad)
    cache.activate([0])
    cache.extend(65)
    with pytest.raises(ValueError, match="capacity"):
        cache.extend(64)
    with pytest.raises(ValueError, match="expected"):
        cache.update(torch.zeros(1, 2, 2, 128, device="cuda"), torch.zeros(1, 2, 2, 128, device="cuda"), 0)
    for parents, children in (([0], [0]), ([0, 0], [1]), ([7], [1]), ([0, 0], [1, 1])):
        with pytest.raises(ValueError):
            cache.fork(parents, children)
    cache.fork([0], [1])
    with pytest.raises(ValueError, match="empty"):
        cache.fork([0], [1])
    with pytest.raises(ValueError):
        cache.truncate([0], [-1])
    with pytest.raises(ValueError, match="num_layers"):
        SharedPrefixFP8Fp8Cache(4, 2, 128, num_layers=0)
    cfg, model = build(layers=1)
    cache.activate([0])
    with pytest.raises(RuntimeError, match="prefill from empty"):
        model(torch.zeros(1, 2, dtype=torch.long, device="cuda"), past_key_values=cache, use_cache=True)


def test_a_refused_model_call_leaves_the_cache_as_it_was():
    cfg, model = build()
    make = lambda n=2, kv=2, layers=2: SharedPrefixFP8Fp8Cache(n, kv, 1024, num_layers=layers)
    ids = lambda b, t: torch.ones(b, t, dtype=torch.long, device="cuda")
    cache = make()
    cache.activate([0])
    model(ids(1, 511), past_key_values=cache, use_cache=True)              # one position is left of the model's 512
    model(ids(1, 1), past_key_values=cache, use_cache=True)
    other = make()
    other.activate([0, 1])

    def refused(c, tokens, error, match):
        before = [c.table.seq_lens.clone(), c.table.block_table.clone(), c.table.refcount.clone(), *(x.clone() for x in c.table.pools)]
        lengths = list(c.lengths)
        with pytest.raises(error, match=match):
            model(tokens, past_key_values=c, use_cache=True)
        after = [c.table.seq_lens, c.table.block_table, c.table.refcount, *c.table.pools]
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, after)) and c.lengths == lengths

    refused(cache, ids(1, 1), ValueError, "max_position")
    refused(cache, ids(1, 3), RuntimeError, "prefill from empty")
    refused(other, ids(2, 513), ValueError, "max_position")
    refused(other, ids(1, 4), ValueError, "2 sequences are active")
    refused(other, ids(3, 1), ValueError, "2 sequences are active")
    refused(make(), ids(1, 1), ValueError, "0 sequences are active")
    for wrong in (make(kv=1), make(layers=1)):
        wrong.activate([0])
        refused(wrong, ids(1, 1), ValueError, "the cache is for")
    model(ids(2, 5), past_key_values=other, use_cache=True)
    other.check()


def test_nothing_waits_for_the_device():
    """Sequences come and go and steps are taken without a copy or a question that waits for the stream."""
    cache = SharedPrefixFP8Fp8Cache(6, 2, 256, num_layers=1)
    kv, q = torch.zeros(3, 1, 2, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, 1, 4, 128, dtype=torch.bfloat16, device="cuda")
    prompt = torch.zeros(1, 100, 2, 128, dtype=torch.bfloat16, device="cuda")
    torch.cuda.set_sync_debug_mode("error")
    try:
        cache.activate([0])
        cache.extend(100)
        cache.update(prompt, prompt, 0)
        cache.fork([0, 0, 0], [1, 2, 4])
        for seqs in ([1, 2, 4], [0, 1, 2]):                 # side by side in the table, and not
            cache.activate(seqs)
            cache.extend(1)
            cache.positions()
            cache.update(kv, kv, 0)
            cache.decode(q, 0)
        cache.truncate([1, 2], [90, 70])
        cache.free([4])
        cache.compact()
        cache.table.extend([0], 1)
        cache.table.truncate([0], [5])
    finally:
        torch.cuda.set_sync_debug_mode("default")
    cache.check()


def test_capture_is_refused(monkeypatch):
    """A replay would use the host's lengths of the captured step."""
    cache = SharedPrefixFP8Fp8Cache(2, 2, 256, num_layers=1)
    kv, q = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16, device="cuda")
    cache.activate([0])
    cache.extend(1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: cache.extend(1), lambda: cache.update(kv, kv, 0), lambda: cache.decode(q, 0), cache.positions):
        with pytest.raises(RuntimeError, match="captured"):
            call()
    assert cache.lengths == [1, 0]
    monkeypatch.undo()
    cache.update(kv, kv, 0)
    cache.decode(q, 0)
    assert cache.table.seq_lens.tolist() == [1, 0]
    cache.check()


def test_driver_with_samples():
    r = subprocess.run([sys.executable, "-m", "ffa_speedtest_b200.fp8fp8.e2e.bench_llama_fp8fp8", "--context", "300", "--samples", "3",
                        "--decode-steps", "70", "--batch", "2", "--iters", "2", "--warmup", "1", "--json"], cwd=ROOT, capture_output=True,
                       text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "[FP8FP8-samples][Decode@300]" in r.stdout and "samples_decode_tok_s" in r.stdout
