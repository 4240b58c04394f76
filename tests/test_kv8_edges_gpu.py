"""Edges of the paged KV cache in 8 bits.

Codes, scales, kept positions and moved weights are compared bit for bit with the 64-bit statement (tests/kv8_ref.py);
attention within the bounds that tests/test_kv8_gpu.py derives."""

from __future__ import annotations

import math

import kv8_ref as ref
import pytest
import torch
from test_kv8_gpu import attention_case, check_attention, check_weights, clean, device_pages, i32, same_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    from torch2vk_b200 import kernels

    kernels.device_status(clear=True)


def _weights(B, heads, positions, seed):
    """Weights with many ties and zeros."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 6, (B, heads, positions), generator=g).float() / 4
    return torch.where(torch.rand(w.shape, generator=g) < 0.5, w, torch.rand(w.shape, generator=g))


def _check_kept(kept, moved, chosen, w, keep):
    for b, heads in enumerate(chosen):
        for h, want in enumerate(heads):
            assert kept[b, h].cpu().tolist() == want + [-1] * (keep - len(want)), (b, h)
            assert torch.equal(moved[b, h, : len(want)].cpu(), w[b, h, want]), (b, h)


# ------------------------------------------------------------------ eviction
@pytest.mark.parametrize("lengths,keep", [([300, 100, 129, 0, 1, 128], 128), ([640, 500, 501, 3, 499, 640], 500), ([5, 60, 64, 0, 1, 2], 64)])
@pytest.mark.parametrize("dim,page,block", [(128, 64, 16), (64, 16, 16)])
def test_evict_in_place_own_weights_out(lengths, keep, dim, page, block):
    """Rows in place, their weights to another tensor: also those of the sequences that keep everything."""
    from torch2vk_b200 import kernels

    B, NK, width = len(lengths), 3, 640 // page
    cache = ref.pool(B * width + 1, NK, page, dim, block, seed=201)
    table = ref.tables(B, width, 1, seed=202)
    w = _weights(B, NK, width * page, 203)
    pages, bt, wd = device_pages(cache), table.cuda(), w.cuda()
    big = torch.full((B, NK + 1, keep + 3), -9.0, device="cuda")
    wo = big[:, 1:, :keep]  # strides of its own
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32(lengths), bt, keep=keep, sinks=4, recent=32, weights_out=wo)
    clean()
    chosen, want_left = ref.evict(cache, w, lengths, table, table, keep=keep, sinks=4, recent=32)
    assert left.cpu().tolist() == want_left
    _check_kept(kept, wo, chosen, w, keep)
    for b, n in enumerate(want_left):
        assert bool((wo[b, :, n:] == -9.0).all())
    assert torch.equal(wd.cpu(), w) and bool((big[:, 0] == -9.0).all()) and bool((big[:, :, keep:] == -9.0).all())
    same_cache(pages, cache)


def test_evict_refuses_one_tensor_with_two_strides():
    from torch2vk_b200 import kernels

    cache, table = ref.pool(9, 2, 16, 64, 16, seed=205), ref.tables(2, 4, 1, seed=206)
    buf = torch.zeros(2 * 2 * 64, device="cuda")
    with pytest.raises(RuntimeError, match="strides"):
        kernels.kv_cache_evict_q8(device_pages(cache), buf.view(2, 2, 64), i32([60, 60]), table.cuda(), keep=32,
                                  weights_out=buf[:128].view(2, 2, 32))


@pytest.mark.parametrize("bad", [dict(keep=0), dict(keep=10, sinks=-1), dict(keep=10, recent=-1), dict(keep=10, sinks=6, recent=5)])
def test_evict_says_what_it_needs(bad):
    """No sinks and no recent window are fine; what is refused is what the message says."""
    from torch2vk_b200 import kernels

    cache, table = ref.pool(9, 2, 16, 64, 16, seed=207), ref.tables(2, 4, 1, seed=208)
    w = torch.zeros(2, 2, 64, device="cuda")
    with pytest.raises(RuntimeError, match="keep > 0, sinks >= 0, recent >= 0 and sinks \\+ recent <= keep"):
        kernels.kv_cache_evict_q8(device_pages(cache), w, i32([60, 60]), table.cuda(), **bad)


def test_evict_in_place_through_a_view_of_the_table():
    """A view that begins where the block table does names the same pages: the move is in place, the weights too."""
    from torch2vk_b200 import kernels

    B, NK, page, dim, block, width, keep = 3, 2, 32, 64, 16, 6, 40
    lengths = [190, 40, 41]
    cache, table = ref.pool(B * width, NK, page, dim, block, seed=211), ref.tables(B, width, 0, seed=212)
    w = _weights(B, NK, width * page, 213)
    pages, bt, wd = device_pages(cache), table.cuda(), w.cuda()
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32(lengths), bt, keep=keep, sinks=2, recent=8, out_table=bt[:, :2])
    clean()
    chosen, want_left = ref.evict(cache, w, lengths, table, table, keep=keep, sinks=2, recent=8)
    assert left.cpu().tolist() == want_left
    _check_kept(kept, wd, chosen, w, keep)
    same_cache(pages, cache)


def test_evict_to_other_pages_needs_a_place_for_the_weights():
    from torch2vk_b200 import kernels

    cache, both = ref.pool(16, 2, 16, 64, 16, seed=215), ref.tables(2, 8, 0, seed=216).cuda()
    w = torch.zeros(2, 2, 64, device="cuda")
    with pytest.raises(ValueError, match="weights_out"):
        kernels.kv_cache_evict_q8(device_pages(cache), w, i32([60, 60]), both[:, :4].contiguous(), keep=32,
                                  out_table=both[:, 4:].contiguous())


# ------------------------------------------------------------------ blocks that read as NaN
def _seen_nan(out, lse, want, poisoned):
    """out is NaN where `poisoned` [B, T, NH] and nowhere else; the rest, and every log-sum-exp, as without the NaN."""
    mask = poisoned.unsqueeze(-1).expand(out.shape)
    assert torch.equal(torch.isnan(out).cpu(), mask)
    check_attention(torch.where(mask, want["out"].half(), out.cpu()), lse, want)


@pytest.mark.parametrize("NH,NK,dim", [(16, 8, 128), (6, 2, 64), (24, 2, 128)])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_nan_values_leave_scores_alone(NH, NK, dim, splits):
    """A V block of NaN makes the outputs that see it NaN and nothing else: log-sum-exps, the weights a decode step adds
    and the key weights come from the scores, so they stay what they are."""
    from torch2vk_b200 import kernels

    page, block, T, width = 64, 16, 37, 6
    positions = [20, 300, -3]
    cache, table, g, _ = attention_case(3, NH, NK, dim, page, block, width, 221)
    q = torch.randn(3, T, NH, dim, generator=g).half()
    want = ref.attention(cache, q, positions, table, dim ** -0.5)
    cache["vs"][table[0, 0], 0, 1] = math.nan  # keys 16 .. 31 of KV head 0: seen by all queries
    cache["vs"][table[1, 5], 1, 0] = math.nan  # keys 320 .. 335 of KV head 1: seen from query 20 on
    cache["v"][table[1, 5], 1, :16] = 0
    group = NH // NK
    poisoned = torch.zeros(3, T, NH, dtype=torch.bool)
    poisoned[0, :, :group] = True
    poisoned[1, 20:, group: 2 * group] = True
    pages, bt = device_pages(cache), table.cuda()
    out, lse = kernels.attn_prefill_q8(q.cuda(), pages, i32(positions), bt, splits=splits, return_lse=True)
    clean()
    _seen_nan(out, lse, want, poisoned)
    before = torch.rand(3, NK, width * page, generator=g)
    w = before.cuda()
    kernels.attn_key_weights_q8(q.cuda(), lse, pages, i32(positions), bt, weights=w, weights_out=w)
    clean()
    check_weights(w, before, want, positions, T, NK)

    last = [p + T - 1 for p in positions]
    w, lse1 = before.cuda(), torch.empty(3, NH, device="cuda")
    out1 = kernels.attn_decode_q8(q[:, -1].cuda(), pages, i32(last), bt, splits=splits, lse=lse1, weights=w, weights_out=w)
    clean()
    one = {n: (x[:, -1:] if n in ("out", "spread") else x[:, :, -1:]) for n, x in want.items() if n != "probs"}
    one["probs"] = [p[:, -1:] for p in want["probs"]]
    _seen_nan(out1.unsqueeze(1), lse1.unsqueeze(-1), one, poisoned[:, -1:])
    check_weights(w, before, one, last, 1, NK)


def test_nan_values_in_a_short_cache():
    """The same where one launch joins a cluster: 200 keys, the NaN block in one CTA's tile."""
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block = 8, 2, 128, 32, 32
    cache, table, g, _ = attention_case(2, NH, NK, dim, page, block, 7, 225)
    q = torch.randn(2, NH, dim, generator=g).half()
    positions = [199, 120]
    want = ref.attention(cache, q.unsqueeze(1), positions, table, dim ** -0.5)
    cache["vs"][table[0, 4], 1, 0] = math.nan  # keys 128 .. 159 of KV head 1
    cache["vs"][table[1, 4], :, 0] = math.nan  # past the keys of sequence 1
    poisoned = torch.zeros(2, 1, NH, dtype=torch.bool)
    poisoned[0, :, 4:] = True
    pages, bt = device_pages(cache), table.cuda()
    before = torch.rand(2, NK, 7 * page, generator=g)
    w, lse = before.cuda(), torch.empty(2, NH, device="cuda")
    out = kernels.attn_decode_q8(q.cuda(), pages, i32(positions), bt, lse=lse, weights=w, weights_out=w)
    clean()
    _seen_nan(out.unsqueeze(1), lse.unsqueeze(-1), want, poisoned)
    check_weights(w, before, want, positions, 1, NK)


# ------------------------------------------------------------------ views
def _loose(x, dims):
    """x on the GPU, with a stride of 5 along its dimensions of one entry, where no stride counts."""
    x = x.cuda()
    strides = [5 if d in dims else s for d, s in enumerate(x.stride())]
    y = torch.as_strided(x, x.shape, strides)
    assert y.shape == x.shape and all(x.shape[d] == 1 for d in dims)
    return y


def test_strides_of_dimensions_of_one_entry_do_not_count():
    """One sequence, one token, one head or one page: what their strides say is no reason to refuse a call."""
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block, T = 4, 1, 64, 64, 16, 5
    cache, table = ref.pool(1, NK, page, dim, block, seed=231), torch.zeros(1, 1, dtype=torch.int32)
    g = torch.Generator().manual_seed(232)
    pages = kernels.Q8Pages(_loose(cache["k"], (0, 1)), _loose(cache["v"], (0, 1)), cache["ks"].cuda(), cache["vs"].cuda())
    bt = _loose(table, (0,))
    k, v = (torch.randn(1, T, NK, dim, generator=g).half() for _ in range(2))
    q = torch.randn(1, T, NH, dim, generator=g).half()
    kernels.kv_cache_write_q8(pages, _loose(k, (0, 2)), _loose(v, (0, 2)), i32([20]), bt)
    ref.write(cache, k, v, [20], table)
    clean()
    same_cache(pages, cache)
    want = ref.attention(cache, q, [20], table, dim ** -0.5)
    out, lse = kernels.attn_prefill_q8(_loose(q, (0,)), pages, i32([20]), bt, return_lse=True,
                                       out=_loose(torch.zeros_like(q), (0,)))
    before = torch.rand(1, NK, page, generator=g)
    w = _loose(before, (0, 1))
    kernels.attn_key_weights_q8(_loose(q, (0,)), lse, pages, i32([20]), bt, weights=w, weights_out=w)
    clean()
    check_attention(out, lse, want)
    check_weights(w, before, want, [20], T, NK)
    for t in (0, 4):
        one = kernels.attn_decode_q8(_loose(q[:, t], (0,)), pages, i32([20 + t]), bt, out=_loose(torch.zeros(1, NH, dim).half(), (0,)))
        clean()
        check_attention(one.unsqueeze(1), None, {n: (x[:, t: t + 1] if n in ("out", "spread") else x[:, :, t: t + 1])
                                                 for n, x in want.items() if n != "probs"})
    w = _weights(1, NK, page, 233)
    wd = _loose(w, (0, 1))
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32([60]), bt, keep=21, sinks=2, recent=3)
    clean()
    chosen, want_left = ref.evict(cache, w, [60], table, table, keep=21, sinks=2, recent=3)
    assert left.cpu().tolist() == want_left
    _check_kept(kept, wd, chosen, w, 21)
    same_cache(pages, cache)
    k1, _ = kernels.kv_cache_read_q8(pages, i32([0]), left, bt, tokens=21)
    assert torch.equal(k1[0].cpu(), ref.rows(cache, table[0], 21)[0].transpose(0, 1).half())


def test_evict_one_sequence_through_a_view_of_the_table():
    """One row of the table: in place whatever the rows' strides."""
    from torch2vk_b200 import kernels

    NK, page, dim, block, keep = 2, 32, 64, 16, 40
    cache, table = ref.pool(6, NK, page, dim, block, seed=235), ref.tables(1, 6, 0, seed=236)
    w = _weights(1, NK, 6 * page, 237)
    pages, bt, wd = device_pages(cache), table.cuda(), w.cuda()
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32([190]), bt, keep=keep, sinks=2, recent=8, out_table=_loose(bt, (0,))[:, :2])
    clean()
    chosen, want_left = ref.evict(cache, w, [190], table, table, keep=keep, sinks=2, recent=8)
    assert left.cpu().tolist() == want_left
    _check_kept(kept, wd, chosen, w, keep)
    same_cache(pages, cache)


# ------------------------------------------------------------------ eviction: entries, lengths, layouts, NaN, and what follows it
def _evict_case(B, NK, page, dim, block, width, keep, seed):
    out = -(-keep // page)
    cache, both = ref.pool(B * (width + out) + 1, NK, page, dim, block, seed=seed), ref.tables(B, width + out, 0, seed=seed + 1) + 1  # page 0 is nobody's
    return cache, both[:, :width].contiguous(), both[:, width:].contiguous(), _weights(B, NK, width * page, seed + 2)


@pytest.mark.parametrize("layout", ["head_major", "token_major"])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_nan_blocks_and_layouts(in_place, layout):
    """Rows of a block that reads as NaN make the block they move to read as NaN; pages in either order in memory."""
    from torch2vk_b200 import kernels

    B, NK, page, dim, block, width, keep = 2, 3, 32, 128, 16, 10, 150
    cache, table, to, w = _evict_case(B, NK, page, dim, block, width, keep, 241)
    cache["ks"][table[0, 4], 1, 1], cache["vs"][table[1, 9], 2, 0] = math.nan, math.nan
    lengths = [320, 311]
    pages, bt, wd = device_pages(cache, layout), table.cuda(), w.cuda()
    wo = wd if in_place else torch.zeros(B, NK, keep, device="cuda")
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32(lengths), bt, keep=keep, sinks=4, recent=40,
                                           out_table=None if in_place else to.cuda(), weights_out=wo)
    clean()
    chosen, want_left = ref.evict(cache, w, lengths, table, table if in_place else to, keep=keep, sinks=4, recent=40)
    assert left.cpu().tolist() == want_left
    _check_kept(kept, wo, chosen, w, keep)
    same_cache(pages, cache)
    k, v = kernels.kv_cache_read_q8(pages, i32([0, 0]), left, bt if in_place else to.cuda(), tokens=keep)
    assert bool(torch.isnan(k[0, :, 1]).any()) and bool(torch.isnan(v[1, :, 2]).any()) and not torch.isnan(k[1]).any()


def test_evict_reports_bad_entries():
    """A source entry outside the pool is reported and read as page 0; rows of a destination entry outside it are skipped."""
    from torch2vk_b200 import kernels

    B, NK, page, dim, block, width, keep = 2, 2, 32, 64, 16, 5, 70
    cache, table, to, w = _evict_case(B, NK, page, dim, block, width, keep, 251)
    assert not (table == 0).any() and not (to == 0).any()
    lengths = [160, 133]
    bad, zero = table.clone(), table.clone()
    bad[0, 1], bad[1, 3], zero[0, 1], zero[1, 3] = 1 << 20, -7, 0, 0
    pages, wd, wo = device_pages(cache), w.cuda(), torch.zeros(B, NK, keep, device="cuda")
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32(lengths), bad.cuda(), keep=keep, sinks=4, recent=40, out_table=to.cuda(),
                                           weights_out=wo)
    assert kernels.device_status(clear=True) == 1 << 1
    chosen, _ = ref.evict(cache, w, lengths, zero, to, keep=keep, sinks=4, recent=40)
    _check_kept(kept, wo, chosen, w, keep)
    same_cache(pages, cache)
    was = {n: x.clone() for n, x in cache.items()}
    bad = to.clone()
    bad[0, 1] = cache["k"].shape[0]
    kept, _ = kernels.kv_cache_evict_q8(pages, wd, i32(lengths), table.cuda(), keep=keep, sinks=4, recent=40, out_table=bad.cuda(),
                                        weights_out=wo)
    assert kernels.device_status(clear=True) == 1 << 1
    chosen, _ = ref.evict(cache, w, lengths, table, to, keep=keep, sinks=4, recent=40)
    for n in cache:
        cache[n][to[0, 1]] = was[n][to[0, 1]]
    same_cache(pages, cache)
    assert kept[0, 0].cpu().tolist() == chosen[0][0]


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_reports_lengths_out_of_range(in_place):
    """A length past the table counts as the table's positions, a negative one as none; both are reported."""
    from torch2vk_b200 import kernels

    B, NK, page, dim, block, width, keep = 3, 2, 32, 64, 16, 4, 50
    cache, table, to, w = _evict_case(B, NK, page, dim, block, width, keep, 261)
    pages, bt, wd = device_pages(cache), table.cuda(), w.cuda()
    wo = wd if in_place else torch.zeros(B, NK, keep, device="cuda")
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32([width * page + 9, -4, 60]), bt, keep=keep, sinks=1, recent=9,
                                           out_table=None if in_place else to.cuda(), weights_out=wo)
    assert kernels.device_status(clear=True) == 1 << 1
    lengths = [width * page, 0, 60]
    chosen, want_left = ref.evict(cache, w, lengths, table, table if in_place else to, keep=keep, sinks=1, recent=9)
    assert left.cpu().tolist() == want_left
    _check_kept(kept, wo, chosen, w, keep)
    same_cache(pages, cache)


@pytest.mark.parametrize("page,block", [(64, 64), (32, 16)])
def test_append_after_an_eviction(page, block):
    """Rows appended to the block that an eviction left partly filled: its scale grows from the evicted rows' one."""
    from torch2vk_b200 import kernels

    B, NK, dim, width, keep = 3, 2, 128, 320 // page, 101
    cache = ref.pool(B * width, NK, page, dim, block, seed=271)
    table = ref.tables(B, width, 0, seed=272)
    w = _weights(B, NK, width * page, 273)
    pages, bt, wd = device_pages(cache), table.cuda(), w.cuda()
    g = torch.Generator().manual_seed(274)
    lengths = [300, 90, 102]
    for T, gain in ((1, 0.2), (1, 4.0), (30, 9.0)):
        _, left = kernels.kv_cache_evict_q8(pages, wd, i32(lengths), bt, keep=keep, sinks=4, recent=16)
        _, want = ref.evict(cache, w, lengths, table, table, keep=keep, sinks=4, recent=16)
        w = wd.cpu()
        assert left.cpu().tolist() == want
        k, v = (torch.randn(B, T, NK, dim, generator=g).half() * gain for _ in range(2))
        kernels.kv_cache_write_q8(pages, k.cuda(), v.cuda(), left, bt)
        clean()
        ref.write(cache, k, v, want, table)
        same_cache(pages, cache)
        lengths = [n + T for n in want]


@pytest.mark.parametrize("B,n,keep", [(1, 30000, 9000), (2, 9001, 2500), (1, 70000, 40000)])
def test_evict_long_moves_the_weights(B, n, keep):
    """In place, several rounds a head: a round's weights are read before an earlier round's stores reach them."""
    from torch2vk_b200 import kernels

    NK, page, dim, block = 2, 64, 64, 16
    width = -(-n // page)
    cache, table = ref.pool(B * width, NK, page, dim, block, seed=281), ref.tables(B, width, 0, seed=282)
    w = torch.exp(2 * torch.randn(B, NK, width * page, generator=torch.Generator().manual_seed(283)))
    pages, bt, wd = device_pages(cache), table.cuda(), w.cuda()
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32([n - 31 * b for b in range(B)]), bt, keep=keep, sinks=4, recent=100)
    clean()
    assert left.cpu().tolist() == [keep] * B
    assert torch.equal(wd[:, :, :keep].cpu(), torch.gather(w, 2, kept.long().cpu()))
    assert bool((kept[:, :, 1:] > kept[:, :, :-1]).all()) and bool((kept[:, :, :4].cpu() == torch.arange(4)).all())
