"""Plain 64-bit statement of the paged 8-bit KV cache (write, read, attention, key weights, eviction), on CPU tensors.

A cache is a dict: k, v int8 [pages, heads, page_size, dim], ks, vs float16 [pages, heads, page_size / block]."""

from __future__ import annotations

import math

import numpy as np
import torch


def half_up(x: float) -> np.float16:
    """Least fp16 number >= x (x >= 0)."""
    h = np.float16(x)
    return np.nextafter(h, np.float16(np.inf)) if float(h) < x else h


def scale_for(top: float) -> np.float16:
    if not math.isfinite(top):
        return np.float16(np.nan)
    return half_up(min(top / 127, 515.5))


def codes_for(x: np.ndarray, s: np.float16) -> np.ndarray:
    s = float(s)
    if not s > 0:
        return np.zeros(x.shape, np.int8)
    return np.rint(x / s).astype(np.int8)  # numpy rounds half to even


def pool(pages: int, heads: int, page: int, dim: int, block: int, seed: int) -> dict[str, torch.Tensor]:
    g = torch.Generator().manual_seed(seed)
    codes = lambda: torch.randint(-127, 128, (pages, heads, page, dim), generator=g, dtype=torch.int8)  # noqa: E731
    scales = lambda: (0.002 + 0.03 * torch.rand(pages, heads, page // block, generator=g)).half()  # noqa: E731
    return {"k": codes(), "v": codes(), "ks": scales(), "vs": scales()}


def tables(batch: int, width: int, spare: int, seed: int) -> torch.Tensor:
    """Block table with every sequence's pages scattered over batch * width + spare pages."""
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(batch * width + spare, generator=g)[: batch * width].view(batch, width).to(torch.int32)


def write(cache: dict, k: torch.Tensor, v: torch.Tensor, positions: list[int], table: torch.Tensor) -> None:
    """k / v float16 [B, T, heads, dim], appended in place."""
    heads, page, dim = cache["k"].shape[1:]
    block = page // cache["ks"].shape[2]
    capacity = table.shape[1] * page
    for x, codes, scales in ((k, cache["k"].numpy(), cache["ks"].numpy()), (v, cache["v"].numpy(), cache["vs"].numpy())):
        x = x.double().numpy()
        for b, p0 in enumerate(positions):
            p1 = min(p0 + x.shape[1], capacity)
            for start in range(max(p0, 0) // block * block, p1, block):
                lo, hi = max(p0, start), min(p1, start + block)
                at, row = int(table[b, start // page]), start % page
                for h in range(heads):
                    new = x[b, lo - p0: hi - p0, h]
                    s = scale_for(np.abs(new).max() if np.isfinite(new).all() else math.inf)
                    old = codes[at, h, row: row + lo - start].astype(np.float64)
                    if lo > start:
                        was = scales[at, h, row // block]
                        s = np.float16(np.nan) if np.isnan(s) or np.isnan(was) else max(s, was)
                        if s != was:
                            codes[at, h, row: row + lo - start] = codes_for(old * float(was), s)
                    codes[at, h, row + lo - start: row + hi - start] = codes_for(new, s)
                    scales[at, h, row // block] = s


def rows(cache: dict, table_row: torch.Tensor, length: int) -> tuple[torch.Tensor, torch.Tensor]:
    """float64 k, v [heads, length, dim] of one sequence."""
    page = cache["k"].shape[2]
    used = table_row[: -(-length // page)].long()
    out = []
    for c, s in ((cache["k"], cache["ks"]), (cache["v"], cache["vs"])):
        block = page // s.shape[2]
        x = c[used].double() * s[used].double().repeat_interleave(block, 2).unsqueeze(-1)
        out.append(x.transpose(0, 1).reshape(c.shape[1], -1, c.shape[3])[:, :length])
    return out[0], out[1]


def attention(cache: dict, q: torch.Tensor, positions: list[int], table: torch.Tensor, scale: float) -> dict:
    """q float16 [B, T, NH, dim].  out and lse; `spread` = sum p |v| and `reach` = the largest sum |q k| * scale a row
    sees (what the rounding bounds are in); probs[b] float64 [NH, T, n]."""
    B, T, NH, D = q.shape
    NK = cache["k"].shape[1]
    out = torch.zeros(B, T, NH, D, dtype=torch.float64)
    spread, reach = torch.zeros_like(out), torch.zeros(B, NH, T, dtype=torch.float64)
    lse = torch.full((B, NH, T), -math.inf, dtype=torch.float64)
    probs = []
    for b, p0 in enumerate(positions):
        n = max(0, p0 + T)
        if n == 0:
            probs.append(torch.zeros(NH, T, 0, dtype=torch.float64))
            continue
        k, v = (x.repeat_interleave(NH // NK, 0) for x in rows(cache, table[b], n))
        qd = q[b].double().transpose(0, 1)
        s = qd @ k.transpose(1, 2) * scale
        sees = torch.arange(n)[None] <= (p0 + torch.arange(T))[:, None]
        s = s.masked_fill(~sees, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m)).masked_fill(~sees, 0)
        l = p.sum(-1, keepdim=True)
        some = (l > 0).squeeze(-1) | torch.isnan(l.squeeze(-1))
        p = p / torch.where(l == 0, torch.ones_like(l), l)
        out[b] = (p @ v).transpose(0, 1)
        spread[b] = (p @ v.abs()).transpose(0, 1)
        reach[b] = (qd.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~sees, 0).amax(-1)
        lse[b] = torch.where(some, (m.squeeze(-1) + l.squeeze(-1).log()), lse[b])
        probs.append(p)
    return {"out": out, "lse": lse, "spread": spread, "reach": reach, "probs": probs}


def evict(cache: dict, weights: torch.Tensor, lengths: list[int], table: torch.Tensor, out_table: torch.Tensor, *,
          keep: int, sinks: int, recent: int) -> tuple[list[list[list[int]]], list[int]]:
    """Kept positions per sequence and head; moves the rows in `cache` (out_table is table: in place)."""
    heads, page, dim = cache["k"].shape[1:]
    block = page // cache["ks"].shape[2]
    chosen_all = []
    for b, n in enumerate(lengths):
        chosen_all.append([])
        src = rows(cache, table[b], n) if n else None
        for h in range(heads):
            if n <= keep:
                chosen = list(range(n))
            else:
                fixed = set(range(sinks)) | set(range(n - recent, n))
                w = weights[b, h, :n].tolist()
                rest = sorted((i for i in range(n) if i not in fixed), key=lambda i: (-math.inf if math.isnan(w[i]) else -w[i],
                                                                                       not math.isnan(w[i]), i))
                chosen = sorted(fixed | set(rest[: keep - len(fixed)]))
            chosen_all[-1].append(chosen)
            if not chosen or (n <= keep and out_table is table):
                continue
            for x, codes, scales in ((src[0], cache["k"], cache["ks"]), (src[1], cache["v"], cache["vs"])):
                y = x[h, chosen].numpy()
                for start in range(0, len(chosen), block):
                    part = y[start: start + block]
                    s = scale_for(np.abs(part).max() if np.isfinite(part).all() else math.inf)
                    at, row = int(out_table[b, start // page]), start % page
                    codes.numpy()[at, h, row: row + len(part)] = codes_for(part, s)
                    scales.numpy()[at, h, row // block] = s
    return chosen_all, [min(n, keep) for n in lengths]
