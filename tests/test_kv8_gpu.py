"""The paged KV cache in 8 bits against its 64-bit statement (tests/kv8_ref.py).

Codes and scales are compared bit for bit: scale and code are each one correctly rounded quotient of numbers of at
most 18 significant bits.  Attention tolerances, per output: the output is rounded to fp16 (2^-11 of itself), each
probability is rounded to fp16 once before the product with V (2^-11 of sum p |v|, allowed 1.5 times for the running
rescaling), and a score is an fp32 sum of head_dim exact products, so it is off by at most 2^-17 of sum |q k| * scale
(128 roundings), which moves numerator and denominator by that factor each.  A log-sum-exp moves by the score's error
plus a few fp32 roundings; a key weight by the score's and the log-sum-exp's errors."""

from __future__ import annotations

import math

import kv8_ref as ref
import pytest
import torch

pytestmark = pytest.mark.gpu


def device_pages(cache, layout="head_major"):
    """Q8Pages on the GPU; "token_major": memory [pages, page_size, heads, dim], passed as a strided view."""
    from torch2vk_b200 import kernels

    def codes(x):
        x = x.cuda()
        return x.transpose(1, 2).contiguous().transpose(1, 2) if layout == "token_major" else x

    return kernels.Q8Pages(codes(cache["k"]), codes(cache["v"]), cache["ks"].cuda(), cache["vs"].cuda())


def same_cache(pages, cache):
    for got, want in ((pages.k, cache["k"]), (pages.v, cache["v"])):
        assert torch.equal(got.cpu(), want)
    for got, want in ((pages.k_scale, cache["ks"]), (pages.v_scale, cache["vs"])):
        assert torch.equal(got.cpu().nan_to_num(-1.0), want.nan_to_num(-1.0))


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def clean():
    from torch2vk_b200 import kernels

    torch.cuda.synchronize()
    assert kernels.device_status(clear=True) == 0


@pytest.fixture(autouse=True)
def _status():
    from torch2vk_b200 import kernels

    kernels.device_status(clear=True)


# ------------------------------------------------------------------ write and read
@pytest.mark.parametrize("dim,page,block", [(128, 64, 16), (128, 32, 32), (64, 64, 64), (64, 16, 16), (128, 128, 64)])
@pytest.mark.parametrize("layout", ["head_major", "token_major"])
def test_write_matches_definition(dim, page, block, layout):
    """A prompt, then single rows of growing size (each append rescales a block's earlier rows), then a middle chunk."""
    from torch2vk_b200 import kernels

    B, NK, width = 3, 2, -(-320 // page)
    cache = ref.pool(B * width + 2, NK, page, dim, block, seed=1)
    table = ref.tables(B, width, 2, seed=2)
    pages, bt = device_pages(cache, layout), table.cuda()
    g = torch.Generator().manual_seed(3)
    starts = [0, 5, 63]
    for T, grow in ((70, 1.0), (1, 1.5), (1, 0.1), (1, 9.0), (1, 9.5), (33, 2.0), (129, 0.5)):
        x = (torch.randn(B, T, 2 * NK * dim + 8, generator=g) * grow).half()
        k, v = (x[..., o: o + NK * dim].view(B, T, NK, dim) for o in (0, NK * dim))
        xd = x.cuda()  # strided views of one buffer, as a fused projection leaves them
        kd, vd = (xd[..., o: o + NK * dim].view(B, T, NK, dim) for o in (0, NK * dim))
        kernels.kv_cache_write_q8(pages, kd, vd, i32(starts), bt)
        ref.write(cache, k, v, starts, table)
        clean()
        same_cache(pages, cache)
        starts = [s + T for s in starts]


def test_write_special_values():
    """All-zero blocks, subnormal and largest fp16 values, exact ties, infinities and NaN, and a block after one."""
    from torch2vk_b200 import kernels

    B, NK, page, dim, block = 1, 2, 32, 64, 16
    cache = ref.pool(6, NK, page, dim, block, seed=5)
    table = ref.tables(B, 4, 2, seed=6)
    pages, bt = device_pages(cache), table.cuda()
    x = torch.zeros(1, 96, NK, dim)
    x[0, 16:32] = torch.randn(16, NK, dim) * 2.0 ** -24
    x[0, 32:48] = torch.randn(16, NK, dim) * 30000
    x[0, 40, 0, 3], x[0, 41, 1, 4] = 65504.0, -65504.0
    x[0, 48:64] = torch.arange(-64, 64).view(2, 64)[:, None].repeat(8, NK, 1) / 2  # with top 127: codes on halves
    x[0, 50, :, 0] = 127.0
    x[0, 64:80] = torch.randn(16, NK, dim)
    x[0, 70, 0, 9] = math.inf
    x[0, 71, 1, 9] = math.nan
    x[0, 80:96] = torch.randn(16, NK, dim)
    x = x.half()
    ref.write(cache, x, x, [0], table)
    kernels.kv_cache_write_q8(pages, x.cuda(), x.cuda(), i32([0]), bt)
    clean()
    same_cache(pages, cache)
    k, v = kernels.kv_cache_read_q8(pages, i32([0]), i32([96]), bt, tokens=96)
    want = ref.rows(cache, table[0], 96)[0].transpose(0, 1).half()
    assert torch.equal(k[0].cpu().nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(k.nan_to_num(7.0), v.nan_to_num(7.0))
    # a block reads as NaN where (and only where) one of its values was not finite, for each head
    finite = torch.isfinite(x[0].view(6, 16, NK, dim)).all(3).all(1)
    assert not finite[4].any() and bool(finite[[0, 1, 3, 5]].all())
    assert torch.equal(torch.isfinite(k[0].cpu().view(6, 16, NK, dim)), finite[:, None, :, None].expand(6, 16, NK, dim))
    # a finite row appended to a poisoned block stays NaN; the block's first row clears it
    one = torch.ones(1, 1, NK, dim).half()
    for at in (72, 64):
        ref.write(cache, one, one, [at], table)
        kernels.kv_cache_write_q8(pages, one.cuda(), one.cuda(), i32([at]), bt)
        same_cache(pages, cache)
    assert bool(torch.isfinite(kernels.kv_cache_read_q8(pages, i32([64]), i32([65]), bt, tokens=1)[0]).all())


def test_write_largest_values():
    """The largest fp16 values keep code 127 of a scale whose products fp16 still holds."""
    from torch2vk_b200 import kernels

    cache, table = ref.pool(2, 1, 16, 64, 16, seed=5), ref.tables(1, 2, 0, seed=6)
    pages, bt = device_pages(cache), table.cuda()
    x = torch.linspace(-65504, 65504, 16 * 64).half().view(1, 16, 1, 64)
    kernels.kv_cache_write_q8(pages, x.cuda(), x.cuda(), i32([0]), bt)
    ref.write(cache, x, x, [0], table)
    clean()
    same_cache(pages, cache)
    k, _ = kernels.kv_cache_read_q8(pages, i32([0]), i32([16]), bt, tokens=16)
    assert float((k.cpu().float() - x.float()).abs().max()) <= 515.5 / 2 + 32  # half a step, half an fp16 step
    assert int(pages.k[bt[0, 0].long()].max()) == 127


def test_write_padding_and_out_of_range_rows():
    """Rows at negative positions are skipped silently; rows past the table and bad table entries are skipped and reported."""
    from torch2vk_b200 import kernels

    B, NK, page, dim, block = 3, 2, 16, 64, 16
    cache = ref.pool(B * 4 + 1, NK, page, dim, block, seed=7)
    table = ref.tables(B, 4, 1, seed=8)
    pages, bt = device_pages(cache), table.cuda()
    x = torch.randn(B, 40, NK, dim).half()
    starts = [-13, -40, 0]
    kernels.kv_cache_write_q8(pages, x.cuda(), x.cuda(), i32(starts), bt)
    ref.write(cache, x, x, starts, table)
    clean()
    same_cache(pages, cache)
    starts = [50, 64, 3]  # 14 rows fit, none fits, all fit
    kernels.kv_cache_write_q8(pages, x.cuda(), x.cuda(), i32(starts), bt)
    ref.write(cache, x, x, starts, table)
    assert kernels.device_status(clear=True) == 1 << 1
    same_cache(pages, cache)
    bad = table.clone()
    bad[0, 1], bad[1, 0] = 99, -1
    before = {n: t.clone() for n, t in cache.items()}
    kernels.kv_cache_write_q8(pages, x.cuda(), x.cuda(), i32([0, 0, 0]), bad.cuda())
    assert kernels.device_status(clear=True) == 1 << 1
    ref.write(cache, x, x, [0, 0, 0], table)
    for n in cache:  # the two pages that the bad entries stood for keep what they had
        for b, i in ((0, 1), (1, 0)):
            cache[n][table[b, i]] = before[n][table[b, i]]
    same_cache(pages, cache)
    k, _ = kernels.kv_cache_read_q8(pages, i32([0, 0, 0]), i32([40, 40, 40]), bad.cuda(), tokens=40)
    assert kernels.device_status(clear=True) == 1 << 1
    assert not k[0, 16:32].any() and not k[1, :16].any() and k[0, :16].any()


@pytest.mark.parametrize("dim,page,block", [(128, 64, 32), (64, 16, 16)])
def test_read_back(dim, page, block):
    from torch2vk_b200 import kernels

    B, NK, width = 2, 3, 6
    cache = ref.pool(B * width + 1, NK, page, dim, block, seed=9)
    table = ref.tables(B, width, 1, seed=10)
    pages, bt = device_pages(cache, "token_major"), table.cuda()
    first, lengths, T = [3, -2], [page + 7, 5], page + 20
    k, v = kernels.kv_cache_read_q8(pages, i32(first), i32(lengths), bt, tokens=T)
    clean()
    for b in range(B):
        for got, x in zip((k, v), ref.rows(cache, table[b], lengths[b])):
            want = torch.zeros(T, NK, dim, dtype=torch.float16)
            for t in range(T):
                if 0 <= first[b] + t < lengths[b]:
                    want[t] = x[:, first[b] + t].half()
            assert torch.equal(got[b].cpu(), want)


# ------------------------------------------------------------------ attention
def check_attention(got, lse, want):
    eps = want["reach"] * 2.0 ** -17  # of a row's scores
    e = eps.transpose(1, 2).unsqueeze(-1)
    tol = 2.0 ** -11 * want["out"].abs() + 1.5 * 2.0 ** -11 * want["spread"] + 2 * e * want["spread"] + 2.0 ** -24
    assert not bool(torch.isnan(got).any())
    err = (got.double().cpu() - want["out"]).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    if lse is not None:
        seen = want["lse"] > -math.inf
        assert torch.equal(lse.cpu() > -math.inf, seen)
        err = (lse.double().cpu() - want["lse"])[seen].abs()
        tol = eps[seen] + 4e-7 * want["lse"][seen].abs() + 2e-6
        assert bool((err <= tol).all()), float((err / tol).max())


def check_weights(got, before, want, positions, T, heads):
    """weights: before + the probabilities summed; nothing written past the last query's key."""
    for b, p0 in enumerate(positions):
        n = max(0, p0 + T)
        p = want["probs"][b]
        step = p.view(heads, -1, n).sum(1) if n else torch.zeros(heads, 0, dtype=torch.float64)
        old = torch.where(torch.arange(n) < p0, before[b, :, :n].double(), torch.zeros(()).double())
        eps = float(want["reach"][b].max()) * 2.0 ** -17 if n else 0.0
        tol = step * (2 * eps + 1e-5) + 1e-6 * old + 1e-12
        err = (got[b, :, :n].double().cpu() - (old + step)).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()))
        assert torch.equal(got[b, :, n:].cpu(), before[b, :, n:])


def attention_case(B, NH, NK, dim, page, block, width, seed, q_gain=1.0):
    cache = ref.pool(B * width + 2, NK, page, dim, block, seed=seed)
    table = ref.tables(B, width, 2, seed=seed + 1)
    return cache, table, torch.Generator().manual_seed(seed + 2), q_gain


@pytest.mark.parametrize("NH,NK,dim", [(32, 8, 128), (16, 8, 128), (16, 16, 64), (8, 1, 64), (6, 2, 128), (20, 4, 64), (16, 1, 128), (24, 2, 128)])
@pytest.mark.parametrize("page,block", [(64, 16), (16, 16), (64, 64)])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_decode_matches_definition(NH, NK, dim, page, block, splits):
    from torch2vk_b200 import kernels

    positions = [0, -1, 1, 15, 16, page - 1, page, 200, 6 * page + 5]
    width = max(7, -(-201 // page))
    cache, table, g, _ = attention_case(len(positions), NH, NK, dim, page, block, width, 11)
    pages, bt = device_pages(cache), table.cuda()
    q = torch.randn(len(positions), NH, dim, generator=g).half()
    want = ref.attention(cache, q.unsqueeze(1), positions, table, dim ** -0.5)
    before = torch.rand(len(positions), NK, width * page, generator=g)
    lse = torch.empty(len(positions), NH, device="cuda")
    weights = before.cuda()
    out = kernels.attn_decode_q8(q.cuda(), pages, i32(positions), bt, splits=splits, lse=lse, weights=weights, weights_out=weights)
    clean()
    check_attention(out.unsqueeze(1), lse.unsqueeze(-1), want)
    check_weights(weights, before, want, positions, 1, NK)
    assert not out[1].any()
    # without the weights, a bound on the lengths and a strided q: the same answer
    qs = torch.zeros(len(positions), NH + 3, dim, dtype=torch.float16, device="cuda")
    qs[:, 2: NH + 2] = q.cuda()
    again = kernels.attn_decode_q8(qs[:, 2: NH + 2], pages, i32(positions), bt, splits=splits, max_len=max(positions) + 1)
    clean()
    check_attention(again.unsqueeze(1), None, want)


@pytest.mark.parametrize("B,NH,NK,dim", [(22, 32, 8, 128), (110, 6, 2, 128), (28, 24, 2, 128), (12, 64, 4, 64), (40, 16, 16, 64)])
def test_decode_many_sequences(B, NH, NK, dim):
    """More heads than the SMs hold joining blocks: a block joins several heads; one sequence much longer than the others."""
    from torch2vk_b200 import kernels

    g = torch.Generator().manual_seed(B)
    positions = torch.randint(-1, 700, (B,), generator=g).tolist()
    positions[B // 2], positions[1], positions[2] = 2999, 0, -1
    cache, table, g, _ = attention_case(B, NH, NK, dim, 64, 16, 47, B + 1)
    pages, bt = device_pages(cache), table.cuda()
    q = torch.randn(B, NH, dim, generator=g).half()
    want = ref.attention(cache, q.unsqueeze(1), positions, table, dim ** -0.5)
    before = torch.rand(B, NK, 47 * 64, generator=g)
    lse = torch.empty(B, NH, device="cuda")
    weights = before.cuda()
    out = kernels.attn_decode_q8(q.cuda(), pages, i32(positions), bt, lse=lse, weights=weights, weights_out=weights)
    clean()
    check_attention(out.unsqueeze(1), lse.unsqueeze(-1), want)
    check_weights(weights, before, want, positions, 1, NK)


@pytest.mark.parametrize("length", [1000, 5003, 20011])
def test_decode_long(length):
    """Long caches, large scores (one key draws nearly all of the weight) and a token-major pool."""
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block = 8, 2, 128, 64, 16
    width = -(-length // page)
    cache, table, g, _ = attention_case(2, NH, NK, dim, page, block, width, 21)
    positions = [length - 1, length // 3]
    pages, bt = device_pages(cache, "token_major"), table.cuda()
    for gain in (0.3, 6.0):
        q = (torch.randn(2, NH, dim, generator=g) * gain).half()
        want = ref.attention(cache, q.unsqueeze(1), positions, table, dim ** -0.5)
        new = torch.full((2, NK, width * page), 7.0, device="cuda")
        out = kernels.attn_decode_q8(q.cuda(), pages, i32(positions), bt, weights_out=new)
        clean()
        check_attention(out.unsqueeze(1), None, want)
        for b, p in enumerate(positions):
            assert bool((new[b, :, p + 1:] == 7.0).all())
            total = new[b, :, : p + 1].double().sum(-1).cpu()
            assert bool((total - NH // NK).abs().max() < 1e-3)
        zero = torch.zeros(2, NK, width * page)
        check_weights(torch.where(new == 7.0, torch.zeros_like(new), new), zero, want, positions, 1, NK)


@pytest.mark.parametrize("NH,NK,dim", [(32, 8, 128), (16, 16, 64), (6, 2, 128), (8, 1, 64), (16, 1, 128)])
@pytest.mark.parametrize("T", [1, 2, 17, 64, 129, 300])
@pytest.mark.parametrize("page,block,splits", [(64, 16, 0), (16, 16, 1), (64, 32, 3), (128, 64, 2)])
def test_prefill_matches_definition(NH, NK, dim, T, page, block, splits):
    """Prompts from their first token, on prefixes that end inside a page, and left padding (rows that see nothing)."""
    from torch2vk_b200 import kernels

    positions = [0, 37, -min(T, 5), 257]
    width = -(-(257 + T) // page)
    cache, table, g, _ = attention_case(4, NH, NK, dim, page, block, width, 31)
    pages, bt = device_pages(cache), table.cuda()
    q = torch.randn(4, T, NH, dim, generator=g).half()
    want = ref.attention(cache, q, positions, table, dim ** -0.5)
    out, lse = kernels.attn_prefill_q8(q.cuda(), pages, i32(positions), bt, splits=splits, return_lse=True)
    clean()
    check_attention(out, lse, want)
    assert not out[2, : min(T, 5)].any()
    # heads before tokens in memory, out in place of a larger buffer
    qh = q.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    big = torch.full((4, T, NH + 1, dim), 3.0, dtype=torch.float16, device="cuda")
    again = kernels.attn_prefill_q8(qh, pages, i32(positions), bt, splits=splits, max_len=257 + T, out=big[:, :, :NH])
    clean()
    check_attention(again, None, want)
    assert bool((big[:, :, NH] == 3.0).all())


@pytest.mark.parametrize("T,length", [(5, 4000), (700, 2100), (1100, 1100)])
def test_prefill_long(T, length):
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block = 8, 2, 128, 32, 32
    width = -(-length // page)
    cache, table, g, _ = attention_case(1, NH, NK, dim, page, block, width, 41)
    pages, bt = device_pages(cache, "token_major"), table.cuda()
    for gain in (0.3, 5.0):
        q = (torch.randn(1, T, NH, dim, generator=g) * gain).half()
        want = ref.attention(cache, q, [length - T], table, dim ** -0.5)
        out, lse = kernels.attn_prefill_q8(q.cuda(), pages, i32([length - T]), bt, return_lse=True)
        clean()
        check_attention(out, lse, want)


@pytest.mark.parametrize("NH,NK,dim", [(4, 2, 64), (8, 2, 128), (3, 1, 64)])
@pytest.mark.parametrize("splits", [0, 1, 2])
def test_prefill_rising_scores(NH, NK, dim, splits):
    """Scores that rise by 45 to 70 (in log2 units) from each page of 128 keys to the next: the running reference moves in
    every tile, after sums of earlier tiles were taken."""
    from torch2vk_b200 import kernels

    length, T, page, block = 2500, 150, 128, 64
    width = -(-length // page)
    cache, table, g, _ = attention_case(1, NH, NK, dim, page, block, width, 61)
    u = torch.randn(dim, generator=g).sign()
    k = cache["k"]
    k.copy_((u * 100 + torch.randint(-20, 21, k.shape, generator=g)).to(torch.int8))
    for i, p in enumerate(table[0].tolist()):
        cache["ks"][p] = (i + 1) * 0.44 / dim ** 0.5
    pages, bt = device_pages(cache), table.cuda()
    q = (u * 8 / dim ** 0.5 + torch.randn(1, T, NH, dim, generator=g) * 0.1).half()
    want = ref.attention(cache, q, [length - T], table, dim ** -0.5)
    out, lse = kernels.attn_prefill_q8(q.cuda(), pages, i32([length - T]), bt, splits=splits, return_lse=True)
    clean()
    check_attention(out, lse, want)
    scores = want["lse"]
    assert float(scores.min()) > 200 and float(scores.max()) < 5000


def test_attention_scales_apart():
    """Blocks whose scales differ by many powers of two, zero blocks, and the largest values: no overflow, no loss."""
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block = 8, 2, 64, 64, 16
    cache, table, g, _ = attention_case(1, NH, NK, dim, page, block, 4, 51)
    for p in range(cache["vs"].shape[0]):
        cache["vs"][p] = (2.0 ** torch.randint(-24, 9, cache["vs"][p].shape, generator=g).float()).half()
        cache["ks"][p] = (2.0 ** torch.randint(-24, -4, cache["ks"][p].shape, generator=g).float()).half()
    for name in ("ks", "vs"):
        cache[name][table[0, 1], :, 1] = 0.0
    cache["vs"][table[0, 0], 0, 2] = 515.5
    pages, bt = device_pages(cache), table.cuda()
    q = torch.randn(1, 3, NH, dim, generator=g).half()
    for p0 in (0, 15, 80, 200):
        want = ref.attention(cache, q, [p0], table, dim ** -0.5)
        out, lse = kernels.attn_prefill_q8(q.cuda(), pages, i32([p0]), bt, return_lse=True)
        one = kernels.attn_decode_q8(q[:, 2].cuda(), pages, i32([p0 + 2]), bt)
        clean()
        check_attention(out, lse, want)
        last = {n: (x[:, 2:] if n in ("out", "spread") else x[:, :, 2:]) for n, x in want.items() if n != "probs"}
        check_attention(one.unsqueeze(1), None, last)


def test_attention_ignores_what_is_not_seen():
    """NaN scales and any codes past a query's last key change nothing; a NaN block that is seen makes its rows NaN."""
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block = 16, 8, 128, 64, 16
    cache, table, g, _ = attention_case(2, NH, NK, dim, page, block, 4, 61)
    pages, bt = device_pages(cache), table.cuda()
    T, positions = 21, [30, 100]
    q = torch.randn(2, T, NH, dim, generator=g).half().cuda()

    def everything():
        out, lse = kernels.attn_prefill_q8(q, pages, i32(positions), bt, return_lse=True)
        one = kernels.attn_decode_q8(q[:, -1], pages, i32([p + T - 1 for p in positions]), bt)
        w = kernels.attn_key_weights_q8(q, lse, pages, i32(positions), bt, weights_out=torch.zeros(2, NK, 4 * page, device="cuda"))
        clean()
        return out, lse, one, w

    was = everything()
    for b, p in enumerate(positions):
        first = -(-(p + T) // block) * block  # first block that no query sees
        for at in range(first, 4 * page, block):
            pages.k_scale[bt[b, at // page].long(), :, at % page // block] = math.nan
            pages.v_scale[bt[b, at // page].long(), :, at % page // block] = math.nan
    for x, y in zip(everything(), was):
        assert torch.equal(x, y)
    pages.v_scale[bt[1, 0].long(), 3, 0] = math.nan  # keys 0..15 of KV head 3 of sequence 1
    out, lse, one, w = everything()
    assert bool(torch.isnan(out[1, :, 6:8]).all()) and bool(torch.isnan(one[1, 6:8]).all())
    keep = [h for h in range(NH) if h not in (6, 7)]
    assert torch.equal(out[1][:, keep], was[0][1][:, keep]) and torch.equal(out[0], was[0][0])


def test_attention_rows_before_a_poisoned_block():
    """A NaN block makes the rows that see it NaN, and no row before it."""
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block = 8, 2, 64, 32, 16
    cache, table, g, _ = attention_case(1, NH, NK, dim, page, block, 10, 65)
    pages, bt = device_pages(cache), table.cuda()
    T = 200
    q = torch.randn(1, T, NH, dim, generator=g).half()
    want = ref.attention(cache, q, [40], table, dim ** -0.5)
    for scale in (pages.k_scale, pages.v_scale):
        keep = scale.clone()
        scale[bt[0, 144 // page].long(), :, 144 % page // block] = math.nan  # keys 144 .. 159, seen from query 104 on
        out, lse = kernels.attn_prefill_q8(q.cuda(), pages, i32([40]), bt, return_lse=True)
        clean()
        assert bool(torch.isnan(out[:, 104:]).all())
        part = {n: (x[:, :104] if n in ("out", "spread") else x[:, :, :104]) for n, x in want.items() if n != "probs"}
        check_attention(out[:, :104], lse[:, :, :104], part)
        scale.copy_(keep)


def test_attention_reports_bad_entries_and_lengths():
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block = 16, 8, 128, 16, 16
    cache, table, g, _ = attention_case(2, NH, NK, dim, page, block, 4, 71)
    pages = device_pages(cache)
    q = torch.randn(2, 3, NH, dim, generator=g).half().cuda()
    bad = table.clone()
    bad[1, 1] = 1 << 20
    lse = torch.zeros(2, NH, 3, device="cuda")
    w = torch.zeros(2, NK, 4 * page, device="cuda")
    for call in (lambda t, p: kernels.attn_decode_q8(q[:, 0], pages, p, t), lambda t, p: kernels.attn_prefill_q8(q, pages, p, t),
                 lambda t, p: kernels.attn_key_weights_q8(q, lse, pages, p, t, weights_out=w)):
        good = call(table.cuda(), i32([20, 20])).clone()
        clean()
        got = call(bad.cuda(), i32([20, 20]))
        assert kernels.device_status(clear=True) == 1 << 1
        assert torch.equal(got[0], good[0])
        call(table.cuda(), i32([4 * page + 9, 20]))  # more positions than the table has
        assert kernels.device_status(clear=True) == 1 << 1
    kernels.attn_decode_q8(q[:, 0], pages, i32([20, 40]), table.cuda(), max_len=32)
    assert kernels.device_status(clear=True) == 1 << 1


@pytest.mark.parametrize("NH,NK,dim", [(32, 8, 128), (16, 16, 64), (6, 2, 128), (16, 1, 64)])
@pytest.mark.parametrize("T", [1, 8, 33, 200])
@pytest.mark.parametrize("page,block", [(64, 16), (16, 16), (64, 64)])
def test_key_weights_match_definition(NH, NK, dim, T, page, block):
    from torch2vk_b200 import kernels

    positions = [0, 130, -min(T, 3), 257]
    width = -(-(257 + T) // page)
    cache, table, g, _ = attention_case(4, NH, NK, dim, page, block, width, 81)
    pages, bt = device_pages(cache), table.cuda()
    q = torch.randn(4, T, NH, dim, generator=g).half()
    want = ref.attention(cache, q, positions, table, dim ** -0.5)
    before = torch.rand(4, NK, width * page, generator=g)
    lse = want["lse"].float().cuda()
    w = before.cuda()
    kernels.attn_key_weights_q8(q.cuda(), lse, pages, i32(positions), bt, weights=w, weights_out=w)
    clean()
    check_weights(w, before, want, positions, T, NK)
    fresh = before.cuda()
    kernels.attn_key_weights_q8(q.cuda(), lse, pages, i32(positions), bt, max_len=257 + T, weights_out=fresh)
    clean()
    for b, p0 in enumerate(positions):
        n = max(0, p0 + T)
        step = want["probs"][b].view(NK, -1, n).sum(1) if n else torch.zeros(NK, 0)
        eps = float(want["reach"][b].max()) * 2.0 ** -17 if n else 0.0
        assert bool(((fresh[b, :, :n].double().cpu() - step).abs() <= step * (2 * eps + 1e-5) + 1e-12).all())


@pytest.mark.parametrize("NH,NK,dim,T,p0", [(16, 1, 64, 1100, 0), (24, 2, 128, 900, 70), (8, 2, 128, 3, 5000)])
def test_key_weights_long(NH, NK, dim, T, p0):
    """Many query tiles (their keys' sums shared out over a cluster) and many keys under few queries (several key tiles a CTA)."""
    from torch2vk_b200 import kernels

    page, block = 64, 32
    width = -(-(p0 + T) // page)
    cache, table, g, _ = attention_case(1, NH, NK, dim, page, block, width, 85)
    pages, bt = device_pages(cache, "token_major"), table.cuda()
    q = torch.randn(1, T, NH, dim, generator=g).half()
    want = ref.attention(cache, q, [p0], table, dim ** -0.5)
    before = torch.rand(1, NK, width * page, generator=g)
    w = torch.zeros(1, NK, width * page, device="cuda")
    b = before.cuda()
    qh = q.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    kernels.attn_key_weights_q8(qh, want["lse"].float().cuda(), pages, i32([p0]), bt, weights=b, weights_out=w)
    clean()
    n = p0 + T
    step = want["probs"][0].view(NK, -1, n).sum(1)
    old = torch.where(torch.arange(n) < p0, before[0, :, :n].double(), torch.zeros(()).double())
    eps = float(want["reach"].max()) * 2.0 ** -17
    assert bool(((w[0, :, :n].double().cpu() - (old + step)).abs() <= step * (2 * eps + 1e-5) + 1e-6 * old + 1e-12).all())
    assert torch.equal(b.cpu(), before)


# ------------------------------------------------------------------ eviction
@pytest.mark.parametrize("dim,page,block", [(128, 64, 16), (64, 16, 16), (64, 64, 64), (128, 64, 32)])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lengths,keep,sinks,recent", [
    ([300, 100, 129, 0, 1], 128, 4, 32), ([319, 320, 7, 50, 200], 50, 0, 0), ([320, 300, 299, 64, 33], 33, 33, 0),
    ([320, 311, 200, 199, 10], 199, 1, 198), ([64, 65, 66, 300, 17], 1, 0, 1),
])
def test_evict_matches_definition(dim, page, block, in_place, lengths, keep, sinks, recent):
    from torch2vk_b200 import kernels

    B, NK, width = len(lengths), 3, 320 // page
    cache = ref.pool(B * width * 2 + 1, NK, page, dim, block, seed=91)
    both = ref.tables(B, 2 * width, 1, seed=92)
    table, to = both[:, :width].contiguous(), both[:, width: width + -(-keep // page)].contiguous()
    g = torch.Generator().manual_seed(93)
    # few distinct weights: many ties, also at the threshold; some zeros of either sign
    w = torch.randint(0, 6, (B, NK, width * page), generator=g).float() / 4
    w = torch.where(torch.rand(w.shape, generator=g) < 0.5, w, torch.rand(w.shape, generator=g))
    w[torch.rand(w.shape, generator=g) < 0.1] = -0.0
    pages = device_pages(cache)
    wd = w.cuda()
    bt = table.cuda()
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32(lengths), bt, keep=keep, sinks=sinks, recent=recent,
                                           out_table=None if in_place else to.cuda(),
                                           weights_out=None if in_place else (wo := torch.full((B, NK, keep), -9.0, device="cuda")))
    clean()
    chosen, want_left = ref.evict(cache, w, lengths, table, table if in_place else to, keep=keep, sinks=sinks, recent=recent)
    assert left.cpu().tolist() == want_left
    moved = wd if in_place else wo
    for b in range(B):
        for h in range(NK):
            want = chosen[b][h]
            assert kept[b, h].cpu().tolist() == want + [-1] * (keep - len(want)), (b, h)
            assert torch.equal(moved[b, h, : len(want)].cpu(), w[b, h, want])
    same_cache(pages, cache)


@pytest.mark.parametrize("B,n,keep", [(1, 30000, 9000), (2, 9001, 2500), (1, 70000, 40000)])
def test_evict_long(B, n, keep):
    """Long sequences, in place: several rounds and several CTAs per head; infinite and NaN weights count as largest."""
    from torch2vk_b200 import kernels

    NK, page, dim, block = 2, 64, 64, 16
    width = -(-n // page)
    cache = ref.pool(B * width, NK, page, dim, block, seed=95)
    table = ref.tables(B, width, 0, seed=96)
    w = torch.exp(2 * torch.randn(B, NK, width * page, generator=torch.Generator().manual_seed(97)))
    w[:, :, 100:400:3] = 0.0
    w[:, :, 1000], w[:, :, 1001], w[:, 1, 7] = math.inf, math.nan, math.nan
    pages, bt, wd = device_pages(cache), table.cuda(), w.cuda()
    lengths = [n - 31 * b for b in range(B)]
    kept, left = kernels.kv_cache_evict_q8(pages, wd, i32(lengths), bt, keep=keep, sinks=4, recent=100)
    clean()
    chosen, want_left = ref.evict(cache, w, lengths, table, table, keep=keep, sinks=4, recent=100)
    assert left.cpu().tolist() == want_left
    for b in range(B):
        for h in range(NK):
            assert kept[b, h].cpu().tolist() == chosen[b][h]
    same_cache(pages, cache)


# ------------------------------------------------------------------ refusals, streams
def test_refusals():
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block = 16, 8, 128, 64, 16
    cache, table, _, _ = attention_case(1, NH, NK, dim, page, block, 2, 101)
    pages, bt = device_pages(cache), table.cuda()
    q = torch.zeros(1, 4, NH, dim, device="cuda").half()
    row = torch.zeros(1, 4, NK, dim, device="cuda").half()
    pos = i32([0])
    with pytest.raises(ValueError, match="int8"):
        kernels.Q8Pages(pages.k.float(), pages.v, pages.k_scale, pages.v_scale)
    with pytest.raises(ValueError, match="page_size / block"):
        kernels.Q8Pages(pages.k, pages.v, pages.k_scale[:, :4], pages.v_scale[:, :4])
    with pytest.raises(ValueError, match="unit last stride"):
        kernels.Q8Pages(pages.k.transpose(2, 3), pages.v.transpose(2, 3), pages.k_scale, pages.v_scale)
    with pytest.raises(ValueError, match="float16"):
        kernels.kv_cache_write_q8(pages, row.float(), row.float(), pos, bt)
    with pytest.raises(ValueError, match="int32"):
        kernels.kv_cache_write_q8(pages, row, row, pos.long(), bt)
    with pytest.raises(ValueError, match="int32"):
        kernels.attn_prefill_q8(q, pages, i32([0, 0]), bt)
    with pytest.raises(ValueError, match="block_table"):
        kernels.attn_prefill_q8(q, pages, pos, bt.long())
    with pytest.raises(ValueError, match="max_len"):
        kernels.attn_decode_q8(q[:, 0], pages, pos, bt, max_len=129)
    with pytest.raises(ValueError, match="weights_out"):
        kernels.attn_decode_q8(q[:, 0], pages, pos, bt, weights_out=torch.zeros(1, NK, 127, device="cuda"))
    with pytest.raises(ValueError, match="without weights_out"):
        kernels.attn_decode_q8(q[:, 0], pages, pos, bt, weights=torch.zeros(1, NK, 128, device="cuda"))
    with pytest.raises(ValueError, match="lse"):
        kernels.attn_prefill_q8(q, pages, pos, bt, lse=torch.zeros(1, 4, NH, device="cuda"))
    with pytest.raises(RuntimeError, match="bad shape"):
        kernels.attn_decode_q8(q[:, 0, :12].contiguous(), pages, pos, bt)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        kernels.attn_decode_q8(torch.zeros(1, NH * dim + 4, device="cuda").half()[:, 4:].view(1, NH, dim), pages, pos, bt)
    with pytest.raises(RuntimeError, match="splits"):
        kernels.attn_prefill_q8(q, pages, pos, bt, splits=-1)
    w = torch.zeros(1, NK, 128, device="cuda")
    with pytest.raises(RuntimeError, match="workspace"):
        kernels.attn_decode_q8(q[:, 0], pages, pos, bt, splits=2, weights_out=w, workspace=torch.empty(1, device="cuda"))
    with pytest.raises(RuntimeError, match="keep"):
        kernels.kv_cache_evict_q8(pages, w, i32([100]), bt, keep=10, sinks=6, recent=5)
    with pytest.raises(RuntimeError, match="exceeds"):
        kernels.kv_cache_evict_q8(pages, w, i32([100]), bt, keep=100, out_table=bt[:, :1].contiguous(),
                                  weights_out=torch.zeros(1, NK, 100, device="cuda"))
    with pytest.raises(RuntimeError, match="new_lengths"):
        n = i32([100])
        kernels.kv_cache_evict_q8(pages, w, n, bt, keep=10, new_lengths=n)
    for page, block in ((24, 8), (64, 8), (16, 16)):
        c = ref.pool(2, NK, page, dim, block, seed=1)
        p = device_pages(c)
        if block == 16:
            kernels.kv_cache_write_q8(p, row, row, pos, i32([[0, 1]]))
            continue
        with pytest.raises(RuntimeError, match="page_size|block"):
            kernels.kv_cache_write_q8(p, row, row, pos, i32([[0, 1]]))
    wide = ref.pool(2, NK, 64, 96, 16, seed=1)
    with pytest.raises(RuntimeError, match="head_dim"):
        kernels.kv_cache_write_q8(device_pages(wide), *[torch.zeros(1, 4, NK, 96, device="cuda").half()] * 2, pos, bt)
    clean()


def test_on_another_stream_and_in_a_graph():
    """A decode step (write, attention with weights) on a side stream, captured and replayed: the same numbers."""
    from torch2vk_b200 import kernels

    NH, NK, dim, page, block = 16, 8, 128, 64, 16
    cache, table, g, _ = attention_case(2, NH, NK, dim, page, block, 3, 111)
    positions = [70, 127]
    q = torch.randn(2, NH, dim, generator=g).half()
    kv = torch.randn(2, 1, NK, dim, generator=g).half()
    pages, bt = device_pages(cache), table.cuda()
    qd, kvd, pos = q.cuda(), kv.cuda(), i32(positions)
    w, out = torch.zeros(2, NK, 3 * page, device="cuda"), torch.zeros(2, NH, dim, device="cuda").half()
    ws = torch.empty(max(1, kernels.attn_decode_q8_workspace(pages, bt, batch=2, n_heads=NH, with_weights=True)), device="cuda")

    def step():
        kernels.kv_cache_write_q8(pages, kvd, kvd, pos, bt)
        kernels.attn_decode_q8(qd, pages, pos, bt, weights_out=w, workspace=ws, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    out.zero_()
    w.zero_()
    graph.replay()
    clean()
    ref.write(cache, kv, kv, positions, table)
    want = ref.attention(cache, q.unsqueeze(1), positions, table, dim ** -0.5)
    check_attention(out.unsqueeze(1), None, want)
    check_weights(w, torch.zeros(2, NK, 3 * page), want, positions, 1, NK)
