"""The Qwen3 runner on the paged KV cache in 8 bits: against the fp16 pool, continued prompts, and a bounded cache.

Cached codes are off by at most half a step, 1/254 of a block's largest magnitude, so layer outputs of the 8-bit runner
stay within a few percent (relative 2-norm) of the fp16 runner's; what must be equal is compared exactly."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _runner(batch=2, max_seq=256, **kw):
    from test_qwen3_gpu import SMALL
    from torch2vk_b200.qwen3 import Qwen3Config, Qwen3Runner, random_weights

    cfg = Qwen3Config(**SMALL)
    if not hasattr(_runner, "weights"):
        _runner.weights = random_weights(cfg, seed=3, topology="q4_k_m")
    return cfg, Qwen3Runner(cfg, _runner.weights, batch=batch, max_seq=max_seq, max_new_tokens=120, page_size=16,
                            decode_splits=4, **kw)


def _ids(cfg, batch, tokens, seed):
    return torch.randint(0, cfg.vocab, (batch, tokens), generator=torch.Generator().manual_seed(seed)).cuda()


def _near(a, b, rel):
    return float((a.float() - b.float()).norm() / b.float().norm()) < rel


def _clean():
    from torch2vk_b200 import kernels

    torch.cuda.synchronize()
    assert kernels.device_status(clear=True) == 0


def _cache_follows(q8, fp, tokens, steps):
    """Layer 0 of the cache: the rotated keys and the values that the fp16 pool holds, to `steps` steps of their head's
    largest magnitude; 2e-3 of the value is the fp16 rounding of what is read back and of the scale."""
    from torch2vk_b200 import kernels

    n = torch.full((2,), tokens, dtype=torch.int32, device="cuda")
    k, v = kernels.kv_cache_read_q8(q8.paged.layer(0), torch.zeros_like(n), n, q8.paged.block_table, tokens=tokens)
    for got, pages in ((k, fp.paged.k[0]), (v, fp.paged.v[0])):
        for s in range(2):
            rows = torch.cat([pages[p] for p in fp.paged.pages(s)])[:tokens].float()
            step = rows.abs().amax(-1, keepdim=True).amax(0, keepdim=True) / 127
            assert bool(((got[s].float() - rows).abs() <= steps * step + 2e-3 * rows.abs()).all())


def test_runner_follows_the_fp16_pool():
    cfg, q8 = _runner(kv_bits=8)
    _, fp = _runner()
    ids = _ids(cfg, 2, 45, 1)
    a, b = [], []
    q8.prefill(ids, layer_outputs=a)
    fp.prefill(ids, layer_outputs=b)
    for x, y in zip(a, b):
        assert _near(x, y, 0.03)
    _cache_follows(q8, fp, 45, 0.51)
    a, b = [], []
    fp.next_token.copy_(q8.next_token)
    q8.decode_step(layer_outputs=a)
    fp.decode_step(layer_outputs=b)
    for x, y in zip(a, b):
        assert _near(x, y, 0.03)
    # the appended token can raise its block's scale: the codes before it round once more, half of a larger step
    _cache_follows(q8, fp, 46, 1.02)
    _clean()


def test_greedy_tokens_and_graph():
    """generate() through the captured graph equals eager decode steps bit for bit."""
    cfg, r = _runner(kv_bits=8)
    ids = _ids(cfg, 2, 30, 2)
    tokens = r.generate(ids, 40).clone()
    _, e = _runner(kv_bits=8)
    e.prefill(ids)
    for _ in range(39):
        e.decode_step()
    assert torch.equal(tokens, e.generated[:, :40])
    assert r.length == e.length == r.cached == 69
    assert int(r.positions[0]) == int(r.slots[0]) == 69
    _clean()


def test_prompt_in_two_pieces():
    """prefill(append=True) on a prefix gives what one prompt gives (the cut at a block's edge: the same codes)."""
    cfg, one = _runner(kv_bits=8)
    _, two = _runner(kv_bits=8)
    ids = _ids(cfg, 2, 83, 3)
    a, b = [], []
    one.prefill(ids, layer_outputs=a)
    two.prefill(ids[:, :48].contiguous())
    two.prefill(ids[:, 48:].contiguous(), layer_outputs=b, append=True)
    assert torch.equal(one.paged.k[0][one.paged.pages(0)[0]], two.paged.k[0][two.paged.pages(0)[0]])
    for x, y in zip(a, b):
        x = x.view(2, 83, -1)[:, 48:]
        assert _near(y.view(2, 35, -1), x, 0.01)
    assert two.length == one.length == 83 and int(two.slots[1]) == 83
    for _ in range(5):
        one.step()
        two.step()
    _clean()


def test_budget_bounds_the_cache():
    """A prompt longer than the budget and a long generation: rows and pages stay bounded, positions go on, sinks and the
    recent window survive each cut; a budget that is never reached changes no token."""
    cfg, free = _runner(kv_bits=8)
    _, wide = _runner(kv_bits=8, kv_budget=200)
    _, tight = _runner(kv_bits=8, kv_budget=64, kv_sinks=4, kv_recent=16)
    ids = _ids(cfg, 2, 100, 4)
    want = free.generate(ids, 60).clone()
    assert torch.equal(wide.generate(ids, 60), want)
    assert wide.cached == 159 and int(wide.slots[0]) == 159
    tight.prefill(ids)
    assert tight.cached == 64 and int(tight.positions[0]) == 100 and tight.slots.tolist() == [64, 64]
    assert len(tight.paged.pages(0)) == 5  # 64 + one page
    most = 0
    for _ in range(100):
        tight.step()
        most = max(most, tight.cached)
    assert most <= 80 and tight.length == 200 and int(tight.positions[1]) == 200
    assert int(tight.slots[0]) == tight.cached
    out = tight.generated
    assert bool(((out >= 0) & (out < cfg.vocab)).all())
    # the kept weights sum to about a group's worth for every token that attended since the window
    w = tight.paged.weights[0][:, :, : tight.cached]
    assert bool((w >= 0).all()) and bool(torch.isfinite(w).all())
    # and again from a new prompt: everything starts over
    tight.prefill(ids[:, :50].contiguous())
    assert tight.cached == 50 and tight.length == 50
    _clean()


def test_weights_are_the_attention_that_was_paid():
    """After a prompt, each KV head's weights sum to group * window; every decoded token adds the group."""
    cfg, r = _runner(kv_bits=8, kv_budget=200, kv_window=8)
    ids = _ids(cfg, 2, 60, 5)
    r.prefill(ids)
    group = cfg.heads // cfg.kv_heads
    for layer in range(cfg.layers):
        total = r.paged.weights[layer][:, :, :60].sum(-1)
        assert bool((total - 8 * group).abs().max() < 1e-3 * 8 * group)
    for i in range(3):
        r.step()
    for layer in range(cfg.layers):
        total = r.paged.weights[layer][:, :, :63].sum(-1)
        assert bool((total - 11 * group).abs().max() < 1e-3 * 11 * group)
    _clean()


def test_runner_refusals():
    from test_qwen3_gpu import SMALL
    from torch2vk_b200.qwen3 import Qwen3Config, Qwen3Runner

    cfg, r = _runner()
    w = _runner.weights
    with pytest.raises(ValueError, match="paged"):
        Qwen3Runner(Qwen3Config(**SMALL), w, batch=1, max_seq=64, kv_bits=8)
    with pytest.raises(ValueError, match="kv_budget"):
        _runner(kv_budget=64)
    with pytest.raises(ValueError, match="kv_budget"):
        _runner(kv_bits=8, kv_budget=20)
    with pytest.raises(ValueError, match="kv_budget"):
        _runner(kv_bits=8, kv_budget=256)
    with pytest.raises(ValueError, match="8-bit"):
        r.prefill(_ids(cfg, 2, 8, 6), append=True)


def test_appended_prompts_stage_their_own_rows():
    """The memory that a continued prompt takes goes by its tokens, not by how long the conversation has become."""
    cfg, r = _runner(kv_bits=8, kv_budget=64, kv_recent=16)
    ids = _ids(cfg, 2, 20, 7)
    r.prefill(ids)

    def peak():
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        r.prefill(ids, append=True)
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - before

    peak()  # buffers that stay
    first = peak()
    for _ in range(110):
        r.step()
    for _ in range(8):
        last = peak()
    assert r.length > 300 and r.cached <= 80
    # what is not bound to the tokens: lists of kept rows where an eviction follows, 4 bytes a row and KV head
    assert last <= first + 2 * cfg.kv_heads * 64 * 4 * cfg.layers + 4096
    _clean()


def test_pool_sized_for_the_budget():
    """With a budget a sequence takes the pages of its bound (or of a longer prompt), however many tokens may follow."""
    cfg, r = _runner(kv_bits=8, kv_budget=64, kv_recent=16, kv_pages=10)  # 80 rows for each of two sequences
    _, wide = _runner(kv_bits=8, kv_budget=64, kv_recent=16)
    ids = _ids(cfg, 2, 50, 8)
    tokens = r.generate(ids, 100)
    assert torch.equal(tokens, wide.generate(ids, 100))
    assert r.paged.free_pages == 0 and r.cached <= 80
    r.prefill(ids[:, :10].contiguous(), append=True)
    r.step()
    _clean()


def test_generation_past_max_seq_with_a_budget():
    """max_seq bounds the cached rows; with a budget a generation may be longer."""
    cfg, r = _runner(max_seq=96, kv_bits=8, kv_budget=64, kv_recent=16)
    _, wide = _runner(max_seq=256, kv_bits=8, kv_budget=64, kv_recent=16)
    ids = _ids(cfg, 2, 60, 9)
    tokens = r.generate(ids, 110).clone()
    assert r.length == 169 and int(r.positions[0]) == 169 and r.cached <= 80
    assert torch.equal(tokens, wide.generate(ids, 110))
    _, free = _runner(max_seq=96, kv_bits=8)
    with pytest.raises(ValueError, match="max_seq"):
        free.generate(ids, 110)
    _clean()


@pytest.mark.parametrize("bad", [dict(kv_window=0), dict(kv_window=-1), dict(kv_sinks=-1), dict(kv_recent=-2)])
def test_runner_refuses_bad_windows(bad):
    with pytest.raises(ValueError, match="kv_window|kv_sinks"):
        _runner(kv_bits=8, kv_budget=64, **bad)


def test_capture_of_a_full_cache():
    """capture() runs a step, so it makes room first: page 0, which is another sequence's, keeps what it has."""
    cfg, r = _runner(kv_bits=8, kv_budget=64, kv_recent=16)
    _, e = _runner(kv_bits=8, kv_budget=64, kv_recent=16)
    ids = _ids(cfg, 2, 60, 10)
    r.prefill(ids)
    e.prefill(ids)
    while r.cached < 80:
        r.decode_step()
        e.decode_step()
    r.capture()
    _clean()
    for _ in range(10):
        r.step()
        e.decode_step()
    assert torch.equal(r.generated, e.generated) and r.cached == e.cached
    for i in range(cfg.layers):
        assert torch.equal(r.paged.k[i], e.paged.k[i]) and torch.equal(r.paged.k_scale[i], e.paged.k_scale[i])
    _clean()


def _rows(r, tokens):
    from torch2vk_b200 import kernels

    n = torch.full((2,), tokens, dtype=torch.int32, device="cuda")
    return [x.float() for x in kernels.kv_cache_read_q8(r.paged.layer(0), torch.zeros_like(n), n, r.paged.block_table, tokens=tokens)]


def test_cut_keeps_sinks_and_the_recent_window():
    """After a cut the first rows of each head are the prompt's first, the last its last, to half a step of the block they
    moved to; 2e-3 of the value is the fp16 rounding of both reads and of the scale."""
    cfg, free = _runner(kv_bits=8)
    _, tight = _runner(kv_bits=8, kv_budget=64, kv_sinks=4, kv_recent=16)
    ids = _ids(cfg, 2, 100, 11)
    free.prefill(ids)
    tight.prefill(ids)
    assert tight.cached == 64
    for was, now in zip(_rows(free, 100), _rows(tight, 64)):
        step = was.abs().amax((1, 3), keepdim=True) / 127  # of a head
        for a, b in ((slice(0, 4), slice(0, 4)), (slice(84, 100), slice(48, 64))):
            assert bool(((now[:, b] - was[:, a]).abs() <= 0.51 * step + 2e-3 * was[:, a].abs()).all())
        assert not torch.equal(now[:, 4:48], was[:, 4:48])
    _clean()


def test_continued_prompt_after_a_cut():
    """prefill(append=True) on a cache that was cut, rows and positions apart: the weights grow by what the window's
    queries pay, and the layer outputs are those of the same tokens fed one by one."""
    def bounded():
        cfg, r = _runner(kv_bits=8, kv_budget=128, kv_sinks=4, kv_recent=32, kv_window=8)
        r.prefill(_ids(cfg, 2, 200, 12))
        for _ in range(3):
            r.decode_step()
        return cfg, r

    cfg, r = bounded()
    _, one = bounded()
    assert r.cached == 131 and r.length == 203 and r.slots.tolist() == [131, 131] and r.positions.tolist() == [203, 203]
    held = [w[:, :, :131].double().clone() for w in r.paged.weights]
    ids = _ids(cfg, 2, 10, 13)
    outs = []
    r.prefill(ids, append=True, layer_outputs=outs)
    assert r.cached == 141 and r.length == 213 and r.slots.tolist() == [141, 141] and r.positions.tolist() == [213, 213]
    group = cfg.heads // cfg.kv_heads
    for w, was in zip(r.paged.weights, held):
        now = w[:, :, :141].double()
        assert bool((now[:, :, :131] >= was - 1e-6).all()) and bool((now[:, :, 131:] >= 0).all())
        paid = now.sum(-1) - was.sum(-1)
        assert bool((paid - 8 * group).abs().max() < 1e-3 * 8 * group)
    for t in range(10):
        step = []
        one.next_token.copy_(ids[:, t])
        one.decode_step(layer_outputs=step)
        for x, y in zip(outs, step):
            assert _near(x.view(2, 10, -1)[:, t], y, 0.03)
    r.step()
    _clean()


def test_tensor_parallel_runner_on_the_8_bit_pool():
    """make_tp_runner takes the cache's settings; one rank gives the plain runner's tokens."""
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(__file__))
    code = f"""
import sys
sys.path[:0] = [{here!r}, {os.path.dirname(here)!r}]
from datetime import timedelta
import torch, torch.distributed as dist
from test_kv8_runner_gpu import _ids, _runner
from torch2vk_b200.tp import make_tp_runner
torch.cuda.set_device(0)
dist.init_process_group("nccl", init_method="tcp://127.0.0.1:29577", rank=0, world_size=1, timeout=timedelta(seconds=60))
kw = dict(kv_bits=8, kv_budget=64, kv_recent=16)
cfg, plain = _runner(**kw)
tp = make_tp_runner(cfg, _runner.weights, rank=0, tp=1, batch=2, max_seq=256, max_new_tokens=120, page_size=16, decode_splits=4, **kw)
ids = _ids(cfg, 2, 100, 14)
for r in (plain, tp):
    r.prefill(ids)
    for _ in range(40):
        r.decode_step()
assert torch.equal(plain.generated[:, :41], tp.generated[:, :41]) and plain.cached == tp.cached
torch.cuda.synchronize()
dist.destroy_process_group()
print("tp ok")
"""
    run = subprocess.run(["timeout", "-k", "30", "240", sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "tp ok" in run.stdout, (run.stdout + run.stderr)[-3000:]
