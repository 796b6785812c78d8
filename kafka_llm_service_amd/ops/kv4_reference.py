"""Plain fp32 forms of the 4-bit cache's operators (``kv4.py``; pages: csrc/kv4.h). CPU tensors run them, and the kernels are tested
against the same formulas in 64 bits."""
from __future__ import annotations

import math

import torch

PAGE = 16
EXP_MIN, EXP_MAX = -124, 125
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
#: borders between neighbouring levels, and whether the border itself goes up (to the even code)
BORDERS = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))


def head_dim(cache: torch.Tensor) -> int:
    return cache.shape[-1] * 32 // 17


def quant(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[..., D] -> (codes uint8 [..., D], exponents int32 [..., D / 32]): groups of 32 divided by the least 2^e that brings them to at
    most 6, each to the nearest level, ties to the even code. Not a number counts as zero, an infinity as the largest."""
    g = torch.nan_to_num(x.bfloat16().float(), nan=0.0, posinf=3.3895313892515355e38, neginf=-3.3895313892515355e38)
    g = g.unflatten(-1, (x.shape[-1] // 32, 32))
    m, e = torch.frexp(g.abs().amax(-1))
    e = torch.where(m > 0, e - 3 + (m > 0.75).int(), torch.full_like(e, EXP_MIN)).clamp(EXP_MIN, EXP_MAX)
    y = torch.ldexp(g, -e[..., None])
    a = y.abs()
    c = torch.zeros_like(a, dtype=torch.int32)
    for t, up in BORDERS:
        c += (a >= t) if up else (a > t)
    return (c + 8 * (g < 0)).flatten(-2).to(torch.uint8), e.int()


def values(codes: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """What codes [..., D] with exponents [..., D / 32] stand for, in fp32."""
    lut = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    return torch.ldexp(lut[codes.long()].unflatten(-1, (e.shape[-1], 32)), e[..., None]).flatten(-2)


def pack(codes: torch.Tensor, e: torch.Tensor, value: bool) -> torch.Tensor:
    """Codes [pages, heads, 16, D] and exponents [pages, heads, 16, D / 32] -> pages (of values where ``value``)."""
    n, h, _, D = codes.shape
    b, s = codes[..., 0::2] | (codes[..., 1::2] << 4), (e + 127).to(torch.uint8)
    if value:
        b, s = b.view(n, h, 4, 4, D // 8, 4).transpose(3, 4), s.transpose(2, 3)
    return torch.cat([b.reshape(n, h, -1), s.reshape(n, h, -1)], -1).view(n, h, PAGE, D // 2 + D // 32)


def unpack(pages: torch.Tensor, value: bool) -> tuple[torch.Tensor, torch.Tensor]:
    n, h = pages.shape[:2]
    D = head_dim(pages)
    flat = pages.flatten(2)
    b, s = flat[..., :PAGE * D // 2], flat[..., PAGE * D // 2:]
    if value:
        b = b.reshape(n, h, 4, D // 8, 4, 4).transpose(3, 4).reshape(n, h, PAGE, D // 2)
        s = s.reshape(n, h, D // 32, PAGE).transpose(2, 3)
    else:
        b, s = b.reshape(n, h, PAGE, D // 2), s.reshape(n, h, PAGE, D // 32)
    return torch.stack([b & 15, b >> 4], -1).flatten(-2), s.int() - 127


def pack_pages(k: torch.Tensor, v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Natural-order K, V [pages, heads, 16, D] -> their pages."""
    return pack(*quant(k), False), pack(*quant(v), True)


def store(x: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, value: bool) -> None:
    """Rows [T, heads, D] into their slots (those outside of the cache are left out)."""
    ok = (slots >= 0) & (slots < cache.shape[0] * PAGE)
    slots = slots[ok]
    if not slots.numel():
        return
    pages, at = torch.unique(slots // PAGE, return_inverse=True)
    codes, e = unpack(cache[pages], value)
    nc, ne = quant(x[ok])
    codes[at, :, slots % PAGE], e[at, :, slots % PAGE] = nc, ne
    cache[pages] = pack(codes, e, value)


def read(k_cache, v_cache, slots):
    out = []
    there = (slots >= 0) & (slots < k_cache.shape[0] * PAGE)
    at = torch.where(there, slots, torch.zeros_like(slots))
    for cache, value in ((k_cache, False), (v_cache, True)):
        codes, e = unpack(cache[at // PAGE], value) if cache.shape[0] else (None, None)
        i = torch.arange(len(at), device=cache.device)
        x = values(codes[i, :, at % PAGE], e[i, :, at % PAGE])
        x[~there] = math.nan
        x[slots < 0] = 0.0
        out.append(x.bfloat16())
    return tuple(out)


def gather(k_cache, v_cache, table, n: int, seen=None):
    """fp32 K, V [n, heads, D] of a sequence's first n keys (where the table names a page outside of the cache K is no numbers and V zeros,
    so that rows in front of it, whose weights there are zero, stay numbers); of pages without a key that is ``seen``, bool [n], anything."""
    ids = table[:(n + PAGE - 1) // PAGE].long()
    if seen is not None:
        pages = torch.nn.functional.pad(seen, (0, -n % PAGE)).view(-1, PAGE).any(1)
        ids = torch.where(pages, ids, torch.zeros_like(ids))
    there = (ids >= 0) & (ids < k_cache.shape[0])
    out = []
    for c, value in ((k_cache, False), (v_cache, True)):
        x = values(*unpack(c[torch.where(there, ids, torch.zeros_like(ids))], value))
        x[~there] = 0.0 if value else math.nan
        if seen is not None:
            x[~pages] = 0.0
        out.append(x.transpose(1, 2).flatten(0, 1)[:n])
    return tuple(out)


def visible(pos: torch.Tensor, n: int, window: int, first: int) -> torch.Tensor:
    """bool [rows, n]: the keys that rows at ``pos`` see."""
    j, p = torch.arange(n, device=pos.device), pos[:, None]
    see = j <= p
    return see & ((j > p - window) | (j < first)) if window else see


def _seen(seg, window, first, device):
    """bool [keys]: those that a row of the segment sees."""
    _, rows, p0, _ = seg
    return visible(p0 + torch.arange(rows, device=device), p0 + rows, window, first).any(0)


def _scores(q, k, seg, window, first, scale):
    t0, rows, p0, _ = seg
    H, G = k.shape[1], q.shape[1] // k.shape[1]
    x = q[t0:t0 + rows].float().unflatten(1, (H, G))
    s = torch.matmul(x.permute(1, 2, 0, 3), k.permute(1, 2, 0).contiguous()[:, None]) * scale     # [H, G, rows, n]
    see = visible(p0 + torch.arange(rows, device=q.device), k.shape[0], window, first)
    return torch.where(see, s, torch.full_like(s, -math.inf))


def attn(q, k_cache, v_cache, tables, segs, window, first, scale, out, lse):
    for seg in segs:
        t0, rows, p0, tr = seg
        if not rows:
            continue
        k, v = gather(k_cache, v_cache, tables[tr], p0 + rows, _seen(seg, window, first, q.device))
        s = _scores(q, k, seg, window, first, scale)
        ls = torch.logsumexp(s, -1)
        o = torch.matmul(torch.exp(s - ls[..., None]), v.transpose(0, 1)[:, None])
        out[t0:t0 + rows] = o.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
        if lse is not None:
            lse[t0:t0 + rows] = ls.permute(2, 0, 1).flatten(1, 2) * math.log2(math.e)


def attn_mass(q, lse, k_cache, tables, segs, window, first, scale, out):
    """out[segment] += the segment's weights."""
    for i, seg in enumerate(segs):
        t0, rows, p0, tr = seg
        if not rows:
            continue
        k, _ = gather(k_cache, k_cache, tables[tr], p0 + rows, _seen(seg, window, first, q.device))
        s = _scores(q, k, seg, window, first, scale)
        ls = (lse[t0:t0 + rows] / math.log2(math.e)).unflatten(1, (k.shape[1], -1)).permute(1, 2, 0)[..., None]
        w = torch.where(torch.isinf(ls) & (ls < 0), torch.zeros_like(s), torch.exp(s - ls))
        out[i, :, :p0 + rows] += w.sum((1, 2))


def evict_keep(mass, lens, budget, first, recent):
    N, j = mass.shape[2], torch.arange(mass.shape[2], device=mass.device)
    n = lens.long().clamp(0, N)[:, None, None]
    low = -math.inf
    rank = torch.where(torch.isnan(mass), torch.full_like(mass, low), mass).double()
    # not a number goes below -inf, what is always kept above +inf, what is not there below everything: in whole steps around them
    order = torch.argsort(rank, dim=-1, descending=True, stable=True)
    place = torch.empty_like(order).scatter_(-1, order, torch.arange(N, device=mass.device).expand_as(order).contiguous())
    place = torch.where(torch.isnan(mass), place + N, place)
    place = torch.where((j < first) | (j >= n - recent), torch.full_like(place, -1), place)
    place = torch.where(j < n, place, torch.full_like(place, 4 * N + 1))
    order = torch.argsort(place, dim=-1, stable=True)
    if N < budget:
        order = torch.nn.functional.pad(order, (0, budget - N), value=N)
    kept = order[..., :budget]
    kept = torch.where(kept < n, kept, torch.full_like(kept, N + 1)).sort(dim=-1).values
    return torch.where(kept < n, kept, torch.full_like(kept, -1)).int()


def evict_copy(k_cache, v_cache, tables, kept, new_tables, mass, new_mass):
    R, H, budget = kept.shape
    if mass is not None:
        ok = (kept >= 0) & (kept < mass.shape[2])
        new_mass.copy_(torch.where(ok, torch.gather(mass, 2, torch.where(ok, kept, 0).long()) if mass.shape[2] else torch.zeros(()),
                                   torch.zeros(())))
    nb = k_cache.shape[0]
    for r in range(R):
        for h in range(H):
            for i, s in enumerate(kept[r, h].tolist()):
                if s < 0 or s // PAGE >= tables.shape[1] or i // PAGE >= new_tables.shape[1]:
                    continue
                a, b = int(tables[r, s // PAGE]), int(new_tables[r, i // PAGE])
                if not (0 <= a < nb and 0 <= b < nb):
                    continue
                for cache, value in ((k_cache, False), (v_cache, True)):
                    src, dst = unpack(cache[a:a + 1, h:h + 1], value), unpack(cache[b:b + 1, h:h + 1], value)
                    dst[0][0, 0, i % PAGE], dst[1][0, 0, i % PAGE] = src[0][0, 0, s % PAGE], src[1][0, 0, s % PAGE]
                    cache[b, h] = pack(*dst, value)[0, 0]
