"""Cases of the operators on a paged KV cache held in 8 bits: the write with its quantizer and the read back, attention
of single tokens and of prompts over the cache, the attention weight each key has received, and the eviction by it.

The cache is a pool of pages k, v int8 [num_pages, kv_heads, page_size, head_dim] with one fp16 scale for each block of
`block` consecutive tokens of a KV head, k_scale, v_scale [num_pages, kv_heads, page_size / block]; a stored code stands
for code * scale.  A block table [sequences, pages] int32 maps logical to physical pages.  The plain forms below are
elementary torch operations in 32 bits on the same buffers; `exact` states the definitions in 64 bits.
"""

import math

import torch

own = False

# Head counts: 32 query / 8 KV heads of 128 and 16 / 8 of 128 are the decoders this framework runs (8B and 0.6B), 16 / 16
# heads of 64 the ungrouped form of its attention tests.
HEADS = {"32x8x128": (32, 8, 128), "16x8x128": (16, 8, 128), "16x16x64": (16, 16, 64)}


def listed():
    return [
        # one new token for each sequence of a served batch at its own position: blocks partly filled, codes rescaled
        dict(name="write 48 sequences", op="write", batch=48, tokens=1, length=4021, heads="16x8x128", page=32, block=32, ragged=True),
        # a long prompt's rows, from an odd position to an odd one
        dict(name="write prompt 8191", op="write", batch=1, tokens=8191, length=8200, heads="32x8x128", page=64, block=16, ragged=False),
        # the smallest decode step: one chat with a short history
        dict(name="decode 1 x 333", op="decode", batch=1, length=333, heads="16x8x128", page=32, block=16, ragged=False, weights=False),
        # one chat with a long history
        dict(name="decode 1 x 32.8k", op="decode", batch=1, length=32801, heads="32x8x128", page=64, block=16, ragged=False, weights=False),
        # a served batch with lengths from a quarter of the longest up; the attention weight of each key is kept for eviction
        dict(name="decode 32 x 6k weights", op="decode", batch=32, length=6007, heads="32x8x128", page=64, block=32, ragged=True, weights=True),
        # a follow-up question of 45 tokens on a conversation in the cache: few queries, many keys
        dict(name="prefill 45 on 9k", op="prefill", batch=1, tokens=45, length=9111, heads="32x8x128", page=64, block=16, ragged=False),
        # a chunk of several prompts at once, each on its own prefix
        dict(name="prefill 4 x 512 ragged", op="prefill", batch=4, tokens=512, length=3500, heads="16x16x64", page=32, block=32, ragged=True),
        # a long prompt from its first token: matrix products
        dict(name="prefill 8192", op="prefill", batch=1, tokens=8192, length=8192, heads="32x8x128", page=64, block=16, ragged=False),
        # the weights of a prompt's keys under its last queries (an observation window before an eviction) ...
        dict(name="key weights 32 of 16k", op="weights", batch=2, tokens=32, length=16007, heads="32x8x128", page=64, block=16, ragged=True),
        # ... and under all queries of a prompt
        dict(name="key weights 6000", op="weights", batch=1, tokens=6000, length=6000, heads="16x8x128", page=64, block=16, ragged=False),
        # one chat brought back to its budget after a few hundred tokens
        dict(name="evict 1 x 1k to 700", op="evict", batch=1, length=1003, heads="16x8x128", page=32, block=16, ragged=False, keep=700, sinks=4, recent=128),
        # a batch of long sequences cut to a quarter: first tokens and a recent window stay, the rest goes by weight
        dict(name="evict 4 x 16k to 4k", op="evict", batch=4, length=16007, heads="32x8x128", page=64, block=16, ragged=True, keep=4096, sinks=4, recent=256),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    heads = rng.choice(sorted(HEADS))
    page = rng.choice([16, 32, 64, 128])
    case = dict(op=rng.choice(["write", "decode", "decode", "prefill", "prefill", "weights", "evict"]), heads=heads, page=page,
                block=rng.choice([b for b in (16, 32, 64) if b <= page]), ragged=rng.random() < 0.5)
    if case["op"] == "write":
        batch = _log(rng, 1, 48)
        tokens = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 8191 // batch))
        return dict(case, batch=batch, tokens=tokens, length=tokens + _log(rng, 1, 4000))
    if case["op"] == "decode":
        batch = _log(rng, 1, 32)
        return dict(case, batch=batch, length=_log(rng, 1, min(32801, 190000 // batch)), weights=rng.random() < 0.5)
    if case["op"] == "prefill":
        batch = _log(rng, 1, 4)
        tokens = _log(rng, 2, 4096 // batch)
        return dict(case, batch=batch, tokens=tokens, length=tokens + _log(rng, 1, 8000))
    if case["op"] == "weights":
        batch = _log(rng, 1, 4)
        tokens = _log(rng, 8, 2048 // batch)
        return dict(case, batch=batch, tokens=tokens, length=tokens + _log(rng, 1, 12000))
    batch = _log(rng, 1, 4)
    length = _log(rng, 200, 16000)
    keep = max(64, int(length * rng.uniform(0.1, 0.9)))
    return dict(case, batch=batch, length=length, keep=keep, sinks=rng.randrange(0, 9), recent=rng.randrange(0, keep // 2))


def _lengths(case):
    """Positions in the cache for each sequence after the pass: equal, or spread from the longest down to about a quarter of it."""
    n, low = case["length"], case.get("tokens", 1)
    if not case["ragged"]:
        return [n] * case["batch"]
    return [max(low, n - (3 * n * b) // (4 * case["batch"]) - b % 7) for b in range(case["batch"])]


def work(case):
    nh, nk, d = HEADS[case["heads"]]
    lens, block, tokens = _lengths(case), case["block"], case.get("tokens", 1)
    row = nk * d
    scales = lambda n: 2 * 2 * nk * -(-n // block)  # noqa: E731
    seen = sum(sum(range(n - tokens + 1, n + 1)) for n in lens)  # (query, key) pairs
    cache = sum(n * row * 2 + scales(n) for n in lens)
    if case["op"] == "write":  # new rows in (fp16), codes and scales out, the blocks' values back (fp16)
        back = sum(n - (n - tokens) // block * block for n in lens)
        return {"bytes": 2 * row * (case["batch"] * tokens * (2 + 1) + back * 2) + sum(scales(tokens) for _ in lens), "flops": 0}
    if case["op"] == "decode":
        held = sum(8 * n * nk for n in lens) if case["weights"] else 0
        return {"bytes": cache + case["batch"] * nh * d * 4 + held, "flops": 4 * d * nh * seen}
    if case["op"] == "prefill":
        return {"bytes": cache + case["batch"] * tokens * nh * (d * 4 + 4), "flops": 4 * d * nh * seen}
    if case["op"] == "weights":
        return {"bytes": cache // 2 + case["batch"] * tokens * nh * (d * 2 + 4) + sum(8 * n * nk for n in lens), "flops": 2 * d * nh * seen}
    kept = sum(min(n, case["keep"]) for n in lens)  # weights in; kept rows in and out as codes, back as fp16; their index and weight
    return {"bytes": sum(4 * n * nk for n in lens) + kept * row * 2 * (1 + 1 + 2) + 2 * sum(scales(min(n, case["keep"])) for n in lens) + kept * nk * 8, "flops": 0}


# ------------------------------------------------------------------ inputs
def _half_up(x):
    """Smallest fp16 value that is at least x (x >= 0, within range)."""
    h = x.to(torch.float16)
    return torch.where(h.to(x.dtype) < x, (h.view(torch.int16) + 1).view(torch.float16), h)


def _quantize(x, block):
    """x fp16 [pages, heads, page, dim] -> codes int8, scales fp16."""
    n, h, p, d = x.shape
    g = x.view(n, h, p // block, block * d).float()
    s = _half_up(g.abs().amax(-1) / 127)
    q = torch.round(g / s.float().clamp_min(1e-30).unsqueeze(-1))
    return q.to(torch.int8).view(n, h, p, d), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    nh, nk, d = HEADS[case["heads"]]
    batch, page, block, tokens = case["batch"], case["page"], case["block"], case.get("tokens", 1)
    lens = _lengths(case)
    width = -(-(case["length"] + block) // page)
    spare = -(-case["keep"] // page) if case["op"] == "evict" else 0
    num = batch * (width + spare) + 3
    # pages are handed out as sequences grow, so a sequence's pages lie anywhere in the pool
    order = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    table = order[: batch * width].view(batch, width).contiguous()
    # keys after their norm and rotation: unit channels and a few large ones; values smaller, of unequal heads
    gain = torch.ones(d, device="cuda")
    gain[torch.randint(0, d, (4,), generator=g, device="cuda")] = 4.0
    k = (rnd(num, nk, page, d) * gain).half()
    v = (rnd(num, nk, page, d) * (0.2 + torch.rand(nk, 1, 1, generator=g, device="cuda"))).half()
    (kq, ks), (vq, vs) = _quantize(k, block), _quantize(v, block)
    state = {"case": case, "pages": (kq, vq, ks, vs), "table": table}
    total = torch.tensor(lens, dtype=torch.int32, device="cuda")
    start = total - tokens
    state["positions"] = start
    if case["op"] == "write":
        state["k"] = (rnd(batch, tokens, nk, d) * gain).half()
        state["v"] = (rnd(batch, tokens, nk, d) * 0.7).half()
        state["first"], state["lengths"] = start // block * block, total
        state["span"] = -(-(tokens + block - 1) // block) * block
    elif case["op"] == "decode":
        state["q"] = (rnd(batch, nh, d) * 1.4).half()
        if case["weights"]:
            state["seen"] = torch.rand(batch, nk, width * page, generator=g, device="cuda")
            state["seen_out"] = torch.zeros_like(state["seen"])
    elif case["op"] in ("prefill", "weights"):
        state["q"] = (rnd(batch, tokens, nh, d) * 1.4).half()
        if case["op"] == "weights":  # the softmax statistics that the prompt's attention left
            state["seen"] = torch.rand(batch, nk, width * page, generator=g, device="cuda")
            state["seen_out"] = torch.zeros_like(state["seen"])
            state["lse"] = torch.logsumexp(_scores(state), -1).view(batch, nh, tokens).contiguous()
    else:
        w = torch.exp(1.5 * rnd(batch, nk, width * page))  # a few keys draw most of the weight, some drew none
        state["seen"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.1, torch.zeros_like(w), w)
        state["seen_out"] = torch.zeros(batch, nk, spare * page, device="cuda")
        state["lengths"] = total
        state["to"] = order[batch * width: batch * (width + spare)].view(batch, spare).contiguous()
        state["first"] = torch.zeros(batch, dtype=torch.int32, device="cuda")
    return state


# ------------------------------------------------------------------ plain forms
def _values(codes, scales, table):
    """Rows of each sequence in order, fp32 [batch, kv_heads, positions, dim]."""
    table = table.long()
    b, w = table.shape
    n, h, p, d = codes.shape
    s = scales.float().repeat_interleave(p // scales.shape[2], 2)
    rows = codes[table].float() * s[table].unsqueeze(-1)
    return rows.transpose(1, 2).reshape(b, h, w * p, d)


def _scores(state):
    """Scaled scores fp32 [batch, kv_heads, group * tokens, positions], -inf where the query does not see the key."""
    case = state["case"]
    nh, nk, d = HEADS[case["heads"]]
    b, t = case["batch"], case.get("tokens", 1)
    k = _values(state["pages"][0], state["pages"][2], state["table"])
    q = state["q"].float().view(b, t, nk, nh // nk, d).permute(0, 2, 3, 1, 4).reshape(b, nk, nh // nk * t, d)
    s = (q @ k.transpose(-1, -2)).mul_(d ** -0.5)
    last = state["positions"][:, None] + torch.arange(t, device="cuda")
    hidden = torch.arange(k.shape[2], device="cuda") > last[:, :, None]
    return s.view(b, nk, nh // nk, t, -1).masked_fill_(hidden[:, None, None], -math.inf).view(b, nk, nh // nk * t, -1)


def _attend(state):
    case = state["case"]
    nh, nk, d = HEADS[case["heads"]]
    b, t = case["batch"], case.get("tokens", 1)
    p = _scores(state)
    m = p.amax(-1, keepdim=True)
    p = p.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    out = (p @ _values(state["pages"][1], state["pages"][3], state["table"])) / l
    out = out.view(b, nk, nh // nk, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, nh, d).half()
    return out, (m + l.log()).view(b, nh, t), p.div_(l)


def _held(state, step):
    """Weights after a pass: what the keys had, and the pass's sum over the heads of a group and the queries; keys of the pass's own
    tokens start from zero."""
    at = torch.arange(step.shape[-1], device="cuda")
    start, total = state["positions"][:, None, None], state["positions"][:, None, None] + state["case"].get("tokens", 1)
    return torch.where(at < total, step + torch.where(at < start, state["seen"], torch.zeros_like(step)), torch.zeros_like(step))


def _rows_back(codes, scales, table, first, lengths, span):
    """fp16 rows [batch, span, kv_heads, dim] from position first[b] on; zero from lengths[b] on."""
    b, p, block = table.shape[0], codes.shape[2], codes.shape[2] // scales.shape[2]
    at = first.long()[:, None] + torch.arange(span, device="cuda")
    there = at < lengths[:, None]
    at = torch.where(there, at, torch.zeros_like(at))
    page, row = table.long().gather(1, at // p), at % p
    x = codes[page, :, row].float() * scales[page, :, row // block].float().unsqueeze(-1)
    return torch.where(there[:, :, None, None], x, torch.zeros_like(x)).half()


def _write(state):
    case = state["case"]
    block, page, tokens, span = case["block"], case["page"], case["tokens"], state["span"]
    first, start, total = (state[x].long()[:, None] for x in ("first", "positions", "lengths"))
    at = first + torch.arange(span, device="cuda")
    b, table = at.shape[0], state["table"].long()
    pages, row = table.gather(1, (at // page).clamp_max(table.shape[1] - 1)), at % page
    old, new = (at < start)[:, :, None, None], ((at >= start) & (at < total))[:, :, None, None]
    grouped = lambda x: x.view(b, span // block, block, *x.shape[2:])  # noqa: E731
    for x, codes, scales in zip((state["k"], state["v"]), state["pages"][:2], state["pages"][2:]):
        q, s = codes[pages, :, row].float(), scales[pages, :, row // block].float()
        src = torch.gather(x, 1, (at - start).clamp(0, tokens - 1)[:, :, None, None].expand(-1, -1, *x.shape[2:])).float()
        src = torch.where(new, src, torch.zeros_like(src))
        top = grouped(src).abs().amax((2, 4))
        kept = torch.where((grouped(at) < start[:, :, None]).any(2)[..., None], grouped(s)[:, :, 0], torch.zeros_like(top))
        into = torch.maximum(kept, _half_up(top / 127).float())
        touched = (grouped(at) < total[:, :, None]).any(2)[..., None]
        into = torch.where(touched, into, grouped(s)[:, :, 0])
        each = into.repeat_interleave(block, 1)[..., None]
        safe = torch.where(each > 0, each, torch.ones_like(each))
        moved = torch.where(old, torch.round(q * s[..., None] / safe), q)
        codes[pages, :, row] = torch.where(new, torch.round(src / safe), moved).to(torch.int8)
        scales[pages, :, row // block] = each[..., 0].half()
    return [_rows_back(c, s, state["table"], state["first"], state["lengths"], span) for c, s in zip(state["pages"][:2], state["pages"][2:])]


def _evict(state):
    case = state["case"]
    nh, nk, d = HEADS[case["heads"]]
    b, keep, block, page = case["batch"], case["keep"], case["block"], case["page"]
    w, lens = state["seen"], state["lengths"].long()[:, None, None]
    at = torch.arange(w.shape[-1], device="cuda")
    rank = torch.where((at < case["sinks"]) | (at >= lens - case["recent"]), torch.full_like(w, math.inf), w)
    rank = torch.where(at < lens, rank, torch.full_like(w, -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.sort(torch.where(order < lens, order, torch.full_like(order, 1 << 30)), dim=-1).values
    here = kept < (1 << 30)
    kept = torch.where(here, kept, torch.full_like(kept, -1))
    src = kept.clamp_min(0)
    if src.shape[-1] < keep:
        src, here, kept = (torch.nn.functional.pad(x, (0, keep - x.shape[-1]), value=y) for x, y in ((src, 0), (here, False), (kept, -1)))
    table, to = state["table"].long(), state["to"].long()
    heads = torch.arange(nk, device="cuda")[None, :, None]
    span = -(-keep // block) * block
    pad = lambda x: torch.nn.functional.pad(x, (0, span - keep))  # noqa: E731
    src, there = pad(src), pad(here)
    page_in = torch.gather(table[:, None].expand(-1, nk, -1), 2, src // page)
    slot = torch.arange(span, device="cuda")
    page_out = to[:, slot // page][:, None].expand(-1, nk, -1)
    for codes, scales in zip(state["pages"][:2], state["pages"][2:]):
        x = codes[page_in, heads, src % page].float() * scales[page_in, heads, src % page // block].float()[..., None]
        x = torch.where(there[..., None], x, torch.zeros_like(x))
        s = _half_up(x.view(b, nk, span // block, block * d).abs().amax(-1) / 127)
        each = s.float().repeat_interleave(block, 2)[..., None]
        q = torch.round(x / torch.where(each > 0, each, torch.ones_like(each))).to(torch.int8)
        old = codes[page_out, heads, slot % page]
        codes[page_out, heads, slot % page] = torch.where(there[..., None], q, old)
        blocks = torch.arange(0, span, block, device="cuda")
        old = scales[page_out[..., ::block], heads, blocks % page // block]
        scales[page_out[..., ::block], heads, blocks % page // block] = torch.where(there[..., ::block], s, old)
    state["seen_out"][..., :keep] = torch.where(here, torch.gather(w, 2, src[..., :keep]), torch.zeros((), device="cuda"))
    left = state["lengths"].clamp_max(keep)
    rows = [_rows_back(c, s, state["to"], state["first"], left, keep) for c, s in zip(state["pages"][:2], state["pages"][2:])]
    return [kept.int(), left, state["seen_out"][..., :keep], *rows]


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return _own(state, op)
    if op == "write":
        return _write(state)
    if op == "decode":
        out, _, p = _attend(state)
        out = out[:, 0]
        nh, nk, _ = HEADS[case["heads"]]
        return [out, _held(state, p.view(case["batch"], nk, nh // nk, -1).sum(2))] if case["weights"] else out
    if op == "prefill":
        return _attend(state)[:2]
    if op == "weights":
        nk = HEADS[case["heads"]][1]
        p = _scores(state).sub_(state["lse"].view(case["batch"], nk, -1, 1)).exp_()
        return _held(state, p.sum(2))
    return _evict(state)


def _own(state, op):
    from torch2vk_b200 import kernels

    pages, table, case = kernels.Q8Pages(*state["pages"]), state["table"], state["case"]
    if op == "write":
        kernels.kv_cache_write_q8(pages, state["k"], state["v"], state["positions"], table)
        return kernels.kv_cache_read_q8(pages, state["first"], state["lengths"], table, tokens=state["span"])
    if op == "decode":
        if not case["weights"]:
            return kernels.attn_decode_q8(state["q"], pages, state["positions"], table, max_len=case["length"])
        out = kernels.attn_decode_q8(state["q"], pages, state["positions"], table, max_len=case["length"], weights=state["seen"],
                                     weights_out=state["seen_out"])
        return [out, state["seen_out"]]
    if op == "prefill":
        return kernels.attn_prefill_q8(state["q"], pages, state["positions"], table, max_len=case["length"], return_lse=True)
    if op == "weights":
        return kernels.attn_key_weights_q8(state["q"], state["lse"], pages, state["positions"], table, max_len=case["length"],
                                           weights=state["seen"], weights_out=state["seen_out"])
    kept, left = kernels.kv_cache_evict_q8(pages, state["seen"], state["lengths"], table, keep=case["keep"], sinks=case["sinks"],
                                           recent=case["recent"], out_table=state["to"], weights_out=state["seen_out"])
    rows = kernels.kv_cache_read_q8(pages, state["first"], left, state["to"], tokens=case["keep"])
    return [kept, left, state["seen_out"][..., :case["keep"]], *rows]


# ------------------------------------------------------------------ 64 bits
def _sequence(codes, scales, pages, length):
    """The first `length` rows of one sequence in 64 bits, [kv_heads, length, dim]."""
    got = [c.double() * s.double().repeat_interleave(c.shape[1] // s.shape[1], 1).unsqueeze(-1) for c, s in ((codes[p], scales[p]) for p in pages)]
    return torch.cat(got, 1)[:, :length]


def _block_scale(top):
    """Least fp16 value at or above top / 127, from the value itself in 64 bits."""
    want = top / 127
    near = want.to(torch.float16)
    up = (near.view(torch.int16).int() + 1).to(torch.int16).view(torch.float16)
    return torch.where(near.double() < want, up, near).double()


def exact(case, seed):
    state = prepare(case, seed)
    nh, nk, d = HEADS[case["heads"]]
    group, tokens, block = nh // nk, case.get("tokens", 1), case["block"]
    kq, vq, ks, vs = state["pages"]
    tables, lens = state["table"].tolist(), _lengths(case)
    if case["op"] == "write":
        outs = []
        for x, codes, scales in ((state["k"], kq, ks), (state["v"], vq, vs)):
            back = torch.zeros(case["batch"], state["span"], nk, d, dtype=torch.float64, device="cuda")
            for b, n in enumerate(lens):
                first, p0 = (n - tokens) // block * block, n - tokens
                rows = torch.zeros(nk, state["span"], d, dtype=torch.float64, device="cuda")
                floor = torch.zeros(nk, state["span"] // block, dtype=torch.float64, device="cuda")
                if p0 > first:
                    page, row = tables[b][first // case["page"]], first % case["page"]
                    floor[:, 0] = scales[page, :, row // block].double()
                    rows[:, : p0 - first] = codes[page, :, row: row + p0 - first].double() * floor[:, :1, None]
                rows[:, p0 - first: n - first] = x[b].double().transpose(0, 1)
                fresh = rows.clone()
                fresh[:, : p0 - first] = 0
                s = torch.maximum(floor, _block_scale(fresh.view(nk, -1, block * d).abs().amax(-1)))
                s = s.repeat_interleave(block, 1).unsqueeze(-1)
                back[b] = torch.where(s > 0, torch.round(rows / s.clamp_min(1e-300)) * s, s).transpose(0, 1)
                back[b, n - first:] = 0
            outs.append(back)
        return outs
    if case["op"] == "evict":
        width = -(-case["keep"] // case["page"]) * case["page"]
        keep, span = case["keep"], -(-case["keep"] // block) * block
        kept_all = torch.full((case["batch"], nk, keep), -1, dtype=torch.int32)
        seen = torch.zeros(case["batch"], nk, width, dtype=torch.float64, device="cuda")
        back = [torch.zeros(case["batch"], keep, nk, d, dtype=torch.float64, device="cuda") for _ in range(2)]
        for b, n in enumerate(lens):
            rows = [_sequence(c, s, tables[b][: -(-n // case["page"])], n) for c, s in ((kq, ks), (vq, vs))]
            for h in range(nk):
                w = state["seen"][b, h, :n].tolist()
                if n <= keep:
                    chosen = list(range(n))
                else:
                    fixed = set(range(case["sinks"])) | set(range(n - case["recent"], n))
                    rest = sorted((i for i in range(n) if i not in fixed), key=lambda i: (-w[i], i))
                    chosen = sorted(fixed | set(rest[: keep - len(fixed)]))
                kept_all[b, h, : len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
                at = torch.tensor(chosen, device="cuda")
                seen[b, h, : len(chosen)] = state["seen"][b, h, at].double()
                for out, x in zip(back, rows):
                    y = torch.zeros(span, d, dtype=torch.float64, device="cuda")
                    y[: len(chosen)] = x[h, at]
                    s = _block_scale(y.view(-1, block * d).abs().amax(-1)).repeat_interleave(block)[:, None]
                    out[b, :, h] = torch.where(s > 0, torch.round(y / s.clamp_min(1e-300)) * s, s)[:keep]
                    out[b, len(chosen):, h] = 0
        left = torch.tensor([min(n, keep) for n in lens], dtype=torch.int32)
        return [kept_all, left, seen[..., :keep], *back]
    if nh * tokens * max(lens) * case["batch"] * d > 3e11:  # pairs times width that 64 bits take long for
        return None
    width = state["table"].shape[1] * case["page"]
    out = torch.zeros(case["batch"], tokens, nh, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(case["batch"], nh, tokens, dtype=torch.float64, device="cuda")
    seen = torch.zeros(case["batch"], nk, width, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        k, v = (_sequence(c, s, tables[b][: -(-n // case["page"])], n) for c, s in ((kq, ks), (vq, vs)))
        if "seen" in state:
            seen[b, :, : n - tokens] = state["seen"][b, :, : n - tokens].double()
        sees = torch.ones(tokens, n, dtype=torch.bool, device="cuda").tril(n - tokens)
        for h in range(nh):
            q = state["q"].view(case["batch"], tokens, nh, d)[b, :, h].double()
            s = (q @ k[h // group].T) / math.sqrt(d)
            s[~sees] = -math.inf
            if case["op"] == "weights":
                seen[b, h // group, :n] += torch.exp(s - state["lse"][b, h].double()[:, None]).sum(0)
                continue
            p = torch.softmax(s, -1)
            out[b, :, h] = p @ v[h // group]
            lse[b, h] = torch.logsumexp(s, -1)
            seen[b, h // group, :n] += p.sum(0)
    if case["op"] == "weights":
        return seen
    if case["op"] == "prefill":
        return [out, lse]
    return [out[:, 0], seen] if case["weights"] else out[:, 0]
