"""The 4-bit cache (kv_dtype "mx4"): writer, reader, attention, weights of the keys and eviction against plain forms in 64 bits.

Tolerances. Stored numbers, kept keys and moved pages are compared bit for bit: rounding to a code is decided by comparisons of
numbers that 32 bits hold exactly (the rotation's products are rounded one by one in both). Attention, for weights w (their sum 1), with
A the largest sum_d |scale q_d k_d| of a row: a score is a sum of D exact products in fp32 and a product by the scale, off by at
most (D + 4) 2^-24 A, and where Q goes in two parts of e4m3 by 2^-21 B, B the largest scale max |q| sum_d |k_d| (a part's
step is 2^-9, its factor 2^-4, and the largest element comes to at least 128: an element is off by half of 2^-13 / 128 of that), and by C, what
the instruction cuts: it adds products of eight neighbouring d, each cut to whole multiples of 2^(E - 13), E the largest sum of two factors'
exponents among them, where 1/2 has the exponent of 1, so 2^E <= 2 max |product|. A product has four bits behind its first and is whole from the
exponent E - 9 on; one that is not is below 4 * 2^(E - 10) <= 2^-7 of the largest. With a part's own step (2^-4) the first part loses less than
(1 + 2^-4) 2^-12 of the largest for each product below 2^-6 of it, the second, a 2^-4 of the first at most, 7 * 2^-16 a group. (Where
elements are so small that e4m3 has no leading bit for them the cut is 2^-19 of their unit: 2^-20 B holds that too.) The
exponential and its argument add 2^-22 (1 + A): EW = 2 ((D + 4) 2^-24 A + 2^-20 B + C + 2^-22 (1 + A)) bounds a weight's relative error with its
sum's. P is rounded to bf16 (2^-8), the output too: |do| <= (2^-8 + EW + n 2^-24) sum w |v| + 2^-8 |o|.
The logarithm is off by (EW + n 2^-24) / ln 2 and its own rounding; a key's weight, from R rows, by the weights' errors, that of
the logarithm and R additions: (2 EW + (n + R + 2) 2^-24 + 2^-23 |lse|) of itself."""
import math

import pytest
import torch

from kafka_llm_service_amd import ops
from kafka_llm_service_amd.ops import kv4
from kafka_llm_service_amd.ops import kv4_reference as kref
from kafka_llm_service_amd.ops import reference as ref

LEV = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


# ---- oracles in 64 bits ---------------------------------------------------------------------------------------------------
def nearest(x):
    """float64 numbers that groups of 32 along the last dim stand for, by distance to the levels."""
    x = x.unflatten(-1, (-1, 32))
    big = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(big, -124)
    for k in range(-123, 126):
        e = torch.where(big > 6 * 2.0 ** (k - 1), torch.full_like(e, k), e)
    y = (x / torch.exp2(e)).abs().clamp(max=6)
    dist = (y[..., None] - LEV.to(x.device)).abs()
    best = dist.min(-1, keepdim=True).values
    code = torch.arange(8, device=x.device)
    pick = torch.where(dist == best, code % 2 * 8 + code, torch.full_like(code, 99).expand_as(dist)).argmin(-1)   # of two: the even
    return (LEV.to(x.device)[pick] * torch.sign(x) * torch.exp2(e)).flatten(-2)


def numbers(cache, value):
    """float64 [pages, heads, 16, D] of pages, byte by byte from the layout."""
    n, h, _, w = cache.shape
    D = w * 32 // 17
    flat = cache.reshape(n, h, -1).long()
    o, d = torch.arange(16)[:, None], torch.arange(D)[None]
    byte = ((o // 4) * (D // 8) + d // 8) * 16 + o % 4 * 4 + d % 8 // 2 if value else o * (D // 2) + d // 2
    sc = 8 * D + (d // 32 * 16 + o if value else o * (D // 32) + d // 32)
    nib = flat[..., byte.to(cache.device)] >> (4 * (d % 2)).to(cache.device) & 15
    val = LEV.to(cache.device)[nib % 8] * torch.where(nib >= 8, -1.0, 1.0).double()
    return val * torch.exp2(flat[..., sc.to(cache.device)].double() - 127)


def _cut(x, k):
    """C of rows x [rows, D] and keys k [n, D]: [rows, n]."""
    out = torch.empty(len(x), len(k))
    step = max(1, 20_000_000 // k.numel())
    for i in range(0, len(x), step):
        p = (x[i:i + step, None].abs().float() * k.abs().float()).unflatten(-1, (-1, 8))
        big = p.amax(-1)
        small = ((p > 0) & (p < big[..., None] * 2.0 ** -6)).sum(-1)
        out[i:i + step] = ((small * (1 + 2.0 ** -4) * 2.0 ** -12 + 7 * 2.0 ** -16) * big).sum(-1)
    return out.double()


def oracle(q, kc, vc, tables, segs, window, first, scale):
    """(out, lse base 2, mass [segments, heads, keys], bounds of out, of lse, of mass) in 64 bits."""
    T, Hq, D = q.shape
    H = kc.shape[1]
    G = Hq // H
    N = max(s[2] + s[1] for s in segs)
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse, blse = torch.zeros(T, Hq, dtype=torch.float64), torch.zeros(T, Hq, dtype=torch.float64)
    bout, mass, bmass = torch.zeros_like(out), torch.zeros(len(segs), H, N, dtype=torch.float64), torch.zeros(len(segs), H, N, dtype=torch.float64)
    for i, (t0, rows, p0, tr) in enumerate(segs):
        n = p0 + rows
        if not rows:
            continue
        ids = tables[tr, :(n + 15) // 16].long()
        k, v = (numbers(c[ids], val).transpose(1, 2).flatten(0, 1)[:n] for c, val in ((kc, False), (vc, True)))
        j, p = torch.arange(n)[None], p0 + torch.arange(rows)[:, None]
        see = (j <= p) & ((p - j < window) | (j < first)) if window else j <= p
        for h in range(Hq):
            x, kh, vh = q[t0:t0 + rows, h].double(), k[:, h // G], v[:, h // G]
            s = (x @ kh.T * scale).masked_fill(~see, -math.inf)
            A = (x.abs() @ kh.abs().T * scale).masked_fill(~see, 0).amax(-1, keepdim=True)
            B = x.abs().amax(-1, keepdim=True) * kh.abs().sum(-1).max() * scale
            C = (_cut(x, kh) * scale).masked_fill(~see, 0).amax(-1, keepdim=True)
            EW = 2 * ((D + 4) * 2.0 ** -24 * A + 2.0 ** -20 * B + C + 2.0 ** -22 * (1 + A))
            ls = torch.logsumexp(s, -1, keepdim=True)
            w = torch.exp(s - ls)
            o = w @ vh
            out[t0:t0 + rows, h] = o
            bout[t0:t0 + rows, h] = (2.0 ** -8 + EW + n * 2.0 ** -24) * (w @ vh.abs()) + 2.0 ** -8 * o.abs()
            lse[t0:t0 + rows, h] = ls[:, 0] / math.log(2)
            blse[t0:t0 + rows, h] = ((EW + n * 2.0 ** -24) / math.log(2) + 2.0 ** -23 * (1 + ls.abs()))[:, 0]
            mass[i, h // G, :n] += w.sum(0)
            bmass[i, h // G, :n] += (w * (2 * EW + (n + rows * G + 2) * 2.0 ** -24 + 2.0 ** -22 * (1 + ls.abs()))).sum(0) + 2.0 ** -120
    return out, lse, mass, bout, blse, bmass


def within(got, want, bound, what):
    bad = ~((got.double().cpu() - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}, most " \
                          f"{float(((got.double().cpu() - want).abs() / bound.clamp(min=1e-300)).nan_to_num(9e9).max()):.3g} of the bound"


def world(segs, H, D, seed=0, device="cpu", spare=2, garbage=True):
    """Pages for the segments' table rows, shuffled; every place that holds no key is filled with bytes of 255."""
    g = torch.Generator().manual_seed(seed)
    lens = {}
    for _, rows, p0, tr in segs:
        lens[tr] = max(lens.get(tr, 0), p0 + rows)
    R = max(lens) + 1
    need = [(lens.get(r, 0) + 15) // 16 for r in range(R)]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g)
    tables = torch.full((R, max(need) + 1), -7, dtype=torch.int32)       # (what no key needs is no page)
    k = torch.randn(total, H, 16, D, generator=g) * torch.exp(0.5 * torch.randn(total, H, 16, 1, generator=g))
    v = torch.randn(total, H, 16, D, generator=g) * torch.exp2(torch.randint(-3, 4, (total, H, 16, 1), generator=g).float())
    kc, vc = kref.pack_pages(k, v)
    at = 0
    for r in range(R):
        tables[r, :need[r]] = order[at:at + need[r]].int()
        at += need[r]
        left = lens.get(r, 0) % 16
        if garbage and left:
            page = int(tables[r, need[r] - 1])
            for c, val in ((kc, False), (vc, True)):
                codes, e = kref.unpack(c[page:page + 1], val)
                codes[:, :, left:], e[:, :, left:] = 15, 128
                c[page] = kref.pack(codes, e, val)[0]
    return kc.to(device), vc.to(device), tables.to(device)


def queries(T, Hq, D, seed=1, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return (1.5 * torch.randn(T, Hq, D, generator=g)).bfloat16().to(device)


#: (query heads, kv heads, dim, segments, window, first)
CASES = [
    (8, 2, 128, [(0, 1, 0, 0)], 0, 0),                                            # one token, one key
    (8, 2, 128, [(0, 1, 14, 0), (1, 1, 15, 1), (2, 1, 16, 2), (3, 1, 62, 3), (4, 1, 63, 4), (5, 1, 64, 5)], 0, 0),
    (4, 4, 64, [(0, 1, 200, 2), (1, 1, 999, 0)], 0, 0),                           # a key/value head for each query head
    (16, 1, 128, [(0, 1, 700, 0)], 0, 0),                                         # one for sixteen
    (10, 2, 128, [(0, 3, 300, 0), (3, 1, 77, 1)], 0, 0),                          # three tokens of five heads
    (12, 4, 64, [(0, 5, 40, 0), (5, 16, 0, 1)], 0, 0),
    (8, 2, 128, [(0, 37, 0, 0)], 0, 0),
    (8, 2, 128, [(2, 50, 333, 1), (60, 1, 500, 0), (61, 0, 9, 0)], 0, 0),         # rows of no segment, one of none
    (32, 8, 128, [(0, 1, 4000, 0), (1, 1, 31, 1), (2, 1, 2047, 2)], 0, 0),        # ranges in pieces
    (8, 2, 128, [(0, 1, 1000, 0), (1, 1, 5, 1)], 128, 0),
    (8, 2, 128, [(0, 1, 1000, 0), (1, 1, 5, 1), (2, 1, 130, 2)], 100, 4),
    (6, 2, 64, [(0, 90, 700, 0), (90, 1, 900, 1)], 65, 70),
    (8, 2, 128, [(0, 200, 0, 0)], 33, 1),
    (8, 8, 128, [(0, 70, 150, 0)], 1, 0),                                         # a window of the row itself
    (14, 2, 128, [(0, 130, 65, 0)], 64, 129),
    (8, 2, 64, [(0, 300, 500, 0), (300, 1, 2000, 1), (301, 2, 100, 2)], 5000, 4), # a window that hides nothing
    (32, 2, 128, [(0, 130, 1, 0), (130, 9, 700, 1)], 0, 0),                       # 16 heads a group, keys widened first
    (10, 2, 64, [(0, 333, 61, 0)], 200, 65),
    (8, 2, 128, [(0, 64, 0, 0), (64, 40, 3000, 1), (110, 33, 130, 2)], 0, 0),     # ranges in pieces
    (4, 4, 128, [(0, 600, 0, 0)], 64, 3),
    (8, 2, 128, [(0, 40, 2000, 0), (40, 40, 2000, 1)], 300, 100),
]


def _id(c):
    return f"{c[0]}x{c[1]}x{c[2]}-{'_'.join(f'{s[1]}at{s[2]}' for s in c[3])}-w{c[4]}f{c[5]}"


def _check_attention(case, device, seed=0):
    Hq, H, D, segs, window, first = case
    kc, vc, tables = world(segs, H, D, seed, device)
    T = max(s[0] + s[1] for s in segs) + 2
    q = queries(T, Hq, D, seed + 1, device)
    plan = kv4.attn_plan(segs, Hq, H, D, window, first, device)
    lse = torch.full((T, Hq), 77.0, device=device)
    scale = 1 / math.sqrt(D)
    out = torch.full_like(q, 5.0)
    assert kv4.attn(q, kc, vc, tables, plan, scale, out=out, lse=lse) is out
    o, l, m, bo, bl, bm = oracle(q.cpu(), kc.cpu(), vc.cpu(), tables.cpu(), segs, window, first, scale)
    mine = torch.zeros(T, dtype=torch.bool)
    for t0, rows, _, _ in segs:
        mine[t0:t0 + rows] = True
    within(out[mine.to(device)], o[mine], bo[mine], "out")
    within(lse[mine.to(device)], l[mine], bl[mine], "lse")
    assert (out[~mine.to(device)] == 5).all() and (lse[~mine.to(device)] == 77).all()
    new = kv4.attn(q, kc, vc, tables, plan, scale)
    assert torch.equal(new[mine.to(device)], out[mine.to(device)]) and (new[~mine.to(device)] == 0).all()
    mass = kv4.attn_mass(q, lse, kc, tables, plan, scale)
    assert mass.shape == m.shape
    within(mass, m, bm, "mass")
    g = torch.Generator().manual_seed(9)
    base = torch.rand(m.shape[0], m.shape[1], m.shape[2] + 100, generator=g).to(device)
    wide = kv4.attn_mass(q, lse, kc, tables, plan, scale, base=base)
    N = m.shape[2]
    within(wide[..., :N], base[..., :N].double().cpu() + m, bm + 2.0 ** -24 * (base[..., :N].double().cpu() + m), "mass on a base")
    assert torch.equal(wide[..., N:], base[..., N:])
    acc = base.clone()
    assert kv4.attn_mass(q, lse, kc, tables, plan, scale, base=acc, out=acc) is acc
    assert torch.equal(acc, wide)


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_attention_reference(case):
    _check_attention(case, "cpu")


def _all_bf16():
    """Rows of groups of 32 that hold every bf16 number, beside larger and smaller ones."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    near = x[torch.argsort(x.float().abs().nan_to_num(0), stable=True)]           # neighbours in a group
    return torch.cat([x, near, near[torch.randperm(65536, generator=g)]]).view(-1, 128)


def _oracle_rows(x):
    y = torch.nan_to_num(x.double(), nan=0.0, posinf=3.3895313892515355e38, neginf=-3.3895313892515355e38)
    return nearest(y)


def test_rounding_to_four_bits():
    x = _all_bf16()
    codes, e = kref.quant(x)
    assert torch.equal(kref.values(codes, e).double(), _oracle_rows(x))
    assert int(e.min()) >= -124 and int(e.max()) <= 125
    k, v = x[:512].view(32, 1, 16, 128).repeat(1, 3, 1, 1), x[512:1024].view(32, 1, 16, 128).repeat(1, 3, 1, 1)
    kc, vc = kref.pack_pages(k, v)
    assert torch.equal(numbers(kc, False), _oracle_rows(k)) and torch.equal(numbers(vc, True), _oracle_rows(v))


def _write(T, Hq, H, D, device, slab=0, seed=0, special=False):
    g = torch.Generator().manual_seed(seed)
    W = (Hq + 2 * H) * D
    if slab:
        qkv = torch.randn(slab, T, W, generator=g)
    else:
        qkv = (torch.randn(T, W + 8, generator=g) * torch.exp2(torch.randint(-9, 5, (T, 1), generator=g).float())).bfloat16()[:, :W]
        if special:
            x = qkv.reshape(-1)
            x[::97], x[5::301], x[9::307], x[3::11] = math.inf, -math.inf, math.nan, 0.0
            qkv = x.view(T, W)
    nb = T // 16 + 4
    slots = torch.randperm(nb * 16, generator=g)[:T]
    slots[1::7] = -1
    slots[4::29] = nb * 16 + 3 if T > 4 else -1
    pos = torch.randint(0, 3000, (T,), generator=g)
    cs = ref.rope_cos_sin(4096, D, 500000.0)
    shape, _, dt = ops.kv_cache_shapes(nb, H, D, "mx4")
    kc, vc = torch.full(shape, 201, dtype=dt, device=device), torch.full(shape, 202, dtype=dt, device=device)
    q = torch.zeros(T, Hq, D, dtype=torch.bfloat16, device=device)
    ops.rope_kv_write(qkv.to(device), pos.to(device), cs.to(device), q, kc, vc, slots.to(device), Hq, H)
    return qkv, pos, cs, slots, q.cpu(), kc.cpu(), vc.cpu()


WRITES = [(1, 8, 2, 128, 0), (40, 8, 2, 128, 0), (40, 8, 2, 64, 0), (33, 4, 4, 64, 2), (5, 32, 8, 128, 4), (300, 10, 2, 128, 0), (3, 3, 1, 128, 1)]


@pytest.mark.parametrize("T,Hq,H,D,slab", WRITES)
def test_writer_reference(T, Hq, H, D, slab):
    """Keys are those of the bf16 cache, rounded; places of no row stay as they were."""
    qkv, pos, cs, slots, q, kc, vc = _write(T, Hq, H, D, "cpu", slab)
    nb = kc.shape[0]
    kb, vb = torch.zeros(nb, H, 16, D, dtype=torch.bfloat16), torch.zeros(nb, H, D, 16, dtype=torch.bfloat16)
    q2 = torch.empty_like(q)
    inside = torch.where(slots < nb * 16, slots, torch.full_like(slots, -1))
    x = qkv.sum(0) if slab else qkv
    ref.rope_kv_write(x, pos, cs, q2, kb, vb, inside, Hq, H)
    assert torch.equal(q, q2)
    at = inside[inside >= 0]
    want_k = _oracle_rows(ref.k_natural(kb)[at // 16, :, at % 16].bfloat16() if not slab else
                          _rot(x, pos, cs, Hq, H, D)[inside >= 0][:, Hq:].bfloat16())
    want_v = _oracle_rows(x.view(T, -1, D)[inside >= 0][:, Hq + H:].bfloat16())
    assert torch.equal(numbers(kc, False)[at // 16, :, at % 16], want_k)
    assert torch.equal(numbers(vc, True)[at // 16, :, at % 16], want_v)
    k, v = kv4.read(kc, vc, torch.cat([at, torch.tensor([-1, nb * 16])]))
    assert torch.equal(k[:-2].double(), want_k) and torch.equal(v[:-2].double(), want_v)
    assert (k[-2] == 0).all() and (v[-2] == 0).all() and k[-1].isnan().all() and v[-1].isnan().all()
    free = torch.ones(nb * 16, dtype=torch.bool)
    free[at] = False
    before = numbers(torch.full_like(kc, 201), False).view(-1)[0], numbers(torch.full_like(vc, 202), True).view(-1)[0]
    assert (numbers(kc, False).transpose(1, 2).flatten(0, 1)[free][..., 0] == before[0]).all()
    assert (numbers(vc, True).transpose(1, 2).flatten(0, 1)[free][..., 0] == before[1]).all()


def _rot(x, pos, cs, Hq, H, D):
    x = x.float().view(x.shape[0], -1, D)[:, :Hq + H]
    c, s = cs[pos][:, None, :D // 2], cs[pos][:, None, D // 2:]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _keep_oracle(mass, lens, budget, first, recent):
    R, H, N = mass.shape
    out = torch.full((R, H, budget), -1, dtype=torch.int32)
    for r in range(R):
        n = min(max(int(lens[r]), 0), N)
        for h in range(H):
            m = mass[r, h].tolist()
            if n <= budget:
                keep = list(range(n))
            else:
                mid = sorted(range(first, n - recent), key=lambda i: (m[i] != m[i], -m[i] if m[i] == m[i] else 0.0, i))
                keep = sorted(list(range(first)) + mid[:budget - first - recent] + list(range(n - recent, n)))
            out[r, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
    return out


def _masses(R, H, N, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    m = torch.exp(3 * torch.randn(R, H, N, generator=g))
    if kind == "ties":
        m = torch.randint(0, 4, (R, H, N), generator=g).float()
    elif kind == "same":
        m = torch.full((R, H, N), 0.25)
    elif kind == "special":
        m = torch.randn(R, H, N, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1e-42, 3.4e38)):
            m[..., i::11] = x
    return m


KEEPS = [(3, 2, 200, 64, 4, 16, "plain"), (2, 2, 3000, 1024, 4, 256, "ties"), (1, 3, 1500, 1000, 0, 0, "same"), (2, 1, 1025, 64, 32, 32, "plain"),
         (2, 2, 2500, 1500, 1, 100, "special"), (1, 1, 5, 1, 0, 0, "plain"), (2, 2, 30, 64, 4, 16, "plain"), (1, 2, 9000, 4097, 16, 1, "plain"),
         (2, 1, 700, 1, 1, 0, "ties"), (1, 1, 2000, 300, 0, 300, "special"),
         (2, 2, 40000, 9000, 4, 1000, "plain"), (1, 1, 40000, 20000, 0, 7, "ties"), (1, 2, 16385, 500, 3, 0, "special"), (1, 1, 16384, 16383, 0, 0, "same"),
         (2, 1, 4097, 1000, 4, 100, "plain"), (1, 2, 8193, 3000, 0, 9, "ties"), (2, 2, 12288, 5000, 5, 0, "special"), (1, 1, 12289, 700, 1, 1, "plain")]


def _lens(R, N):
    return torch.tensor([max(0, N - 37 * i) for i in range(R)], dtype=torch.int32)


@pytest.mark.parametrize("R,H,N,budget,first,recent,kind", KEEPS)
def test_evict_keep_reference(R, H, N, budget, first, recent, kind):
    m, lens = _masses(R, H, N, kind), _lens(R, N)
    assert torch.equal(kv4.evict_keep(m, lens, budget, first, recent), _keep_oracle(m, lens, budget, first, recent))


def _move(device, H=2, D=128, lens=(100, 37, 3), budget=40):
    segs = [(i, 1, n - 1, i) for i, n in enumerate(lens)]
    kc, vc, tables = world(segs, H, D, 3, device, spare=48)
    nb = kc.shape[0]
    free = [p for p in range(nb) if p not in set(tables.flatten().tolist())]
    need = [(min(n, budget) + 15) // 16 for n in lens]
    new = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for r, n in enumerate(need):
        new[r, :n] = torch.tensor([free.pop() for _ in range(n)], dtype=torch.int32)
    m = _masses(len(lens), H, max(lens), "plain").to(device)
    ln = torch.tensor(lens, dtype=torch.int32, device=device)
    kept = kv4.evict_keep(m, ln, budget, 2, 5)
    old = kc.clone(), vc.clone()
    nm = kv4.evict(kc, vc, tables, kept, new.to(device), m)
    kept, m, nm, tables, kc, vc = kept.cpu(), m.cpu(), nm.cpu(), tables.cpu(), kc.cpu(), vc.cpu()
    touched = torch.zeros(nb, H, 16, dtype=torch.bool)
    for c, o, val in ((kc, old[0].cpu(), False), (vc, old[1].cpu(), True)):
        a, b = numbers(c, val), numbers(o, val)
        for r in range(len(lens)):
            for h in range(H):
                for i, s in enumerate(kept[r, h].tolist()):
                    assert nm[r, h, i] == (m[r, h, s] if s >= 0 else 0)
                    if s >= 0:
                        p = int(new[r, i // 16])
                        touched[p, h, i % 16] = True
                        assert torch.equal(a[p, h, i % 16], b[int(tables[r, s // 16]), h, s % 16])
        same = (a == b) | (a.isnan() & b.isnan())
        assert same.all(-1)[~touched].all()
    return kc, vc, kept, new


def test_evict_reference():
    _move("cpu")
    _move("cpu", H=3, D=64)


# ---- refusals -------------------------------------------------------------------------------------------------------------
def test_refusals():
    ks, vs, dt = ops.kv_cache_shapes(4, 2, 128, "mx4")
    assert ks == vs == (4, 2, 16, 68) and dt == torch.uint8 and ops.kv_page_bytes(2, 128, "mx4") == 2 * 2 * 1088
    kc, vc = torch.zeros(ks, dtype=dt), torch.zeros(vs, dtype=dt)
    assert ops.is_mx4_cache(kc) and not ops.is_fp8_cache(kc)
    for bad in (96, 32, 256):
        with pytest.raises(ValueError):
            ops.kv_cache_shapes(4, 2, bad, "mx4")
    plan = lambda *a, **k: kv4.attn_plan(*a, device="cpu", **k)
    for segs in ([(-1, 1, 0, 0)], [(0, 1, -1, 0)], [(0, -1, 0, 0)], [(0, 1, 0, -1)], [(0, 4, 0, 0), (3, 1, 0, 1)], [(0, 1, 1 << 26, 0)],
                 [(1, 1, 0, 0), (1, 1, 0, 0)], [(1 << 26, 1, 0, 0)], [(0, 1, 0)] * 4, [0, 1, 0, 0], [(0, 1, 0, 0), (1, 1)]):
        with pytest.raises(ValueError):
            plan(segs, 8, 2, 128)
    for heads in ((9, 2, 128), (34, 2, 128), (8, 2, 96), (8, 0, 128), (0, 2, 128)):
        with pytest.raises(ValueError):
            plan([(0, 1, 0, 0)], *heads)
    for kw in (dict(window=-1), dict(window=4, first=-1), dict(first=4)):
        with pytest.raises(ValueError):
            plan([(0, 1, 0, 0)], 8, 2, 128, **kw)
    p = plan([(0, 2, 30, 1)], 8, 2, 128)
    q, bt = queries(2, 8, 128), torch.zeros(2, 2, dtype=torch.int32)
    kv4.attn(q, kc, vc, bt, p, 0.1)
    lse = torch.zeros(2, 8)
    for args in ((q[:1], kc, vc, bt), (q.float(), kc, vc, bt), (q[:, :6], kc, vc, bt), (q, kc.float(), vc, bt), (q, kc, vc[:3], bt),
                 (q, kc, vc, bt[:1]), (q, kc, vc, bt[:, :1]), (q, kc, vc, bt.long())):
        with pytest.raises(ValueError):
            kv4.attn(*args, p, 0.1)
    for scale in (0.0, -0.1, math.inf, math.nan):
        with pytest.raises(ValueError):
            kv4.attn(q, kc, vc, bt, p, scale)
        with pytest.raises(ValueError):
            kv4.attn_mass(q, lse, kc, bt, p, scale)
    with pytest.raises(ValueError):
        kv4.attn(q, kc[:0], vc[:0], bt, p, 0.1)
    for kw in (dict(out=torch.zeros(2, 8, 64)), dict(lse=torch.zeros(2, 7)), dict(lse=lse.double())):
        with pytest.raises(ValueError):
            kv4.attn(q, kc, vc, bt, p, 0.1, **kw)
    for kw in (dict(base=torch.zeros(1, 2, 31)), dict(base=torch.zeros(2, 2, 32)), dict(base=torch.zeros(1, 2, 32), out=torch.zeros(1, 2, 40)),
               dict(out=torch.zeros(1, 2, 64)[:, :, ::2])):
        with pytest.raises(ValueError):
            kv4.attn_mass(q, lse, kc, bt, p, 0.1, **kw)
    m, ln = torch.zeros(2, 2, 50), torch.tensor([50, 40], dtype=torch.int32)
    for args in ((m, ln, 0, 0, 0), (m, ln, 10, 6, 5), (m, ln, 10, -1, 0), (m, ln, 10, 0, -1), (m.double(), ln, 10, 0, 0), (m, ln.long(), 10, 0, 0),
                 (m, ln[:1], 10, 0, 0), (m[0], ln, 10, 0, 0)):
        with pytest.raises(ValueError):
            kv4.evict_keep(*args)
    kept = torch.zeros(2, 2, 10, dtype=torch.int32)
    for args in ((kc, vc, bt[:1], kept, bt), (kc, vc, bt, kept, bt[:1]), (kc, vc, bt, kept[:, :1], bt), (kc, vc, bt.long(), kept, bt),
                 (kc, vc, bt, kept, bt, m[:1])):
        with pytest.raises(ValueError):
            kv4.evict(*args)
    with pytest.raises(ValueError):
        kv4.read(kc, vc, torch.zeros(3))


def _bad_pages(device):
    """Pages that are none: the rows that see them are no numbers, the others as without."""
    segs = [(0, 1, 99, 0), (1, 1, 99, 1), (2, 1, 99, 2)]
    kc, vc, tables = world(segs, 2, 128, 0, device)
    q = queries(3, 8, 128, 1, device)
    plan = kv4.attn_plan(segs, 8, 2, 128, device=device)
    lse = torch.zeros(3, 8, device=device)
    good = kv4.attn(q, kc, vc, tables, plan, 0.1)
    bad = tables.clone()
    bad[0, 3], bad[2, 6] = -1, kc.shape[0]
    out = kv4.attn(q, kc, vc, bad, plan, 0.1, lse=lse)
    assert out[0].isnan().all() and out[2].isnan().all() and lse[0].isnan().all() and torch.equal(out[1], good[1])
    kept = torch.arange(100, dtype=torch.int32, device=device).expand(3, 2, 100).contiguous()
    kept[0, 0, 4], kept[1, 1, 5] = 1 << 30, -5
    before = kc.clone(), vc.clone()
    none = torch.full((3, 7), -1, dtype=torch.int32, device=device)
    none[1] = kc.shape[0]
    kv4.evict(kc, vc, bad, kept, none)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


def test_bad_pages_reference():
    _bad_pages("cpu")


def _pages_left_behind(device, D, segs):
    """Pages that the window has passed, and the first keys do not reach, may be anything: no page, or one that nobody ever wrote."""
    window, first = 100, 20
    kc, vc, tables = world(segs, 2, D, 3, device, spare=3)
    T = max(s[0] + s[1] for s in segs)
    q = queries(T, 8, D, 1, device)
    plan = kv4.attn_plan(segs, 8, 2, D, window, first, device=device)
    lse, again = torch.zeros(T, 8, device=device), torch.zeros(T, 8, device=device)
    out = kv4.attn(q, kc, vc, tables, plan, 0.1, lse=lse)
    mass = kv4.attn_mass(q, lse, kc, tables, plan, 0.1)
    assert not out.isnan().any()
    used = set(tables.flatten().tolist())
    free = [p for p in range(kc.shape[0]) if p not in used][0]
    if 0 in used:                                            # page 0 too is one that nobody wrote
        tables[tables == 0] = free
        kc[free], vc[free] = kc[0], vc[0]
        free = 0
    kc[free], vc[free] = 255, 255
    for what in (-1, kc.shape[0], free):
        left = tables.clone()
        for _, rows, p0, tr in segs:
            for page in range(left.shape[1]):
                if page * 16 >= first and (page * 16 + 15 <= p0 - window or page * 16 >= p0 + rows):
                    left[tr, page] = what
        assert (left != tables).sum() > 10
        assert torch.equal(kv4.attn(q, kc, vc, left, plan, 0.1, lse=again), out) and torch.equal(lse, again)
        assert torch.equal(kv4.attn_mass(q, lse, kc, left, plan, 0.1), mass)


LEFT = [[(0, 1, 300, 0), (1, 1, 555, 1), (2, 1, 37, 2)], [(0, 9, 411, 0), (9, 1, 800, 1)], [(0, 300, 333, 0), (300, 140, 900, 1)]]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("segs", LEFT, ids=["tokens", "short", "long"])
def test_pages_left_behind_reference(D, segs):
    _pages_left_behind("cpu", D, segs)


def _nothing(device):
    """Plans without a segment, or without rows: nothing is written, masses stay what they were."""
    kc, vc = (torch.zeros(2, 2, 16, 68, dtype=torch.uint8, device=device) for _ in range(2))
    bt = torch.full((1, 1), -1, dtype=torch.int32, device=device)
    q, lse = queries(3, 8, 128, device=device), torch.full((3, 8), 7.0, device=device)
    for segs in ([], [(0, 0, 0, 0)], [(2, 0, 500, 9), (1, 0, 0, 0)]):
        for kw in ({}, dict(window=5, first=2)):
            plan = kv4.attn_plan(segs, 8, 2, 128, device=device, **kw)
            out = torch.full_like(q, 3.0)
            kv4.attn(q, kc, vc, bt, plan, 0.1, out=out, lse=lse)
            assert (out == 3).all() and (lse == 7).all() and (kv4.attn(q, kc, vc, bt, plan, 0.1) == 0).all()
            assert kv4.attn_mass(q, lse, kc, bt, plan, 0.1).shape == (len(segs), 2, 0)
            base = torch.rand(len(segs), 2, 130, device=device)
            assert torch.equal(kv4.attn_mass(q, lse, kc, bt, plan, 0.1, base=base), base)
    none = torch.zeros(0, dtype=torch.int64, device=device)
    assert kv4.read(kc, vc, none)[0].shape == (0, 2, 128)
    ops.rope_kv_write(torch.zeros(0, 12 * 128, dtype=torch.bfloat16, device=device), none, torch.zeros(1, 128, device=device), q[:0], kc, vc, none, 8, 2)
    kept = kv4.evict_keep(torch.zeros(2, 2, 0, device=device), torch.zeros(2, dtype=torch.int32, device=device), 5)
    assert (kept == -1).all() and kept.shape == (2, 2, 5)
    two = bt.expand(2, 1).contiguous()
    assert (kv4.evict(kc, vc, two, kept, two, torch.zeros(2, 2, 0, device=device)) == 0).all()
    assert kv4.evict_keep(torch.zeros(0, 2, 9, device=device), torch.zeros(0, dtype=torch.int32, device=device), 5).shape == (0, 2, 5)
    assert (kc == 0).all() and (vc == 0).all()


def test_nothing_reference():
    _nothing("cpu")


def test_plan_covers_every_block_once():
    """Pieces of tiles of any length and window cover the blocks that the tile sees, each once."""
    import numpy as np

    g = torch.Generator().manual_seed(0)
    for _ in range(200):
        r = lambda hi: int(torch.randint(0, hi, (1,), generator=g))
        segs = np.array([(100 * i, 1 + r(90), r(5000), i) for i in range(1 + r(6))])
        window, first = (0, 0) if r(3) == 0 else (1 + r(700), r(200))
        tok = 1 + r(16)
        tiles = kv4._tiles(segs, tok)
        assert sum(t[1] for t in tiles) == segs[:, 1].sum() and max(t[1] for t in tiles) <= tok
        _, count = kv4._blocks(tiles[:, 2], tiles[:, 1], window, first)
        n = (kv4._narrow_split(count, 2, 16 + 16 * r(2))[1], kv4._wide_split(count, 2, 256), np.array([1 + r(9) for _ in tiles]))[r(3)]
        pieces, merges, slots = kv4._pieces(tiles, count, n)
        seen = {}
        for t, lo, hi, slot, i, of in pieces.tolist():
            assert lo < hi and 0 <= i < of and (slot >= 0) == (of > 1)
            seen.setdefault(int(tiles[t, 0]), []).append((lo, hi, slot + i))
        for row, n, pos, tab, _ in tiles.tolist():
            parts = sorted(seen[row])
            need = {j // 64 for p in range(pos, pos + n) for j in range(p + 1) if not window or j > p - window or j < first}
            head, count = (int(x) for x in kv4._blocks(np.array(pos), np.array(n), window, first))
            tail = max(0, pos - window + 1) // 64 if window else 0
            listed = [b if b < head else b - head + tail for b in range(count)]
            assert need <= set(listed) and len(set(listed)) == len(listed) and max(listed) == (pos + n - 1) // 64
            assert parts[0][0] == 0 and parts[-1][1] == count and all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
            m = [x for x in merges.tolist() if x[0] == row]
            if len(parts) == 1:
                assert parts[0][2] < 0 and not m
            else:
                assert m == [[row, n, parts[0][2], len(parts)]] and [x[2] for x in parts] == list(range(parts[0][2], parts[0][2] + len(parts)))
        used = sorted(x for m in merges.tolist() for x in range(m[2], m[2] + m[3]))
        assert used == list(range(slots))


# ---- GPU ------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_rounding_on_the_gpu(cuda):
    """Every bf16 number through the writer's value path and back."""
    x = _all_bf16()
    T = x.shape[0] // 2
    qkv = torch.cat([torch.zeros(T, 3 * 128, dtype=torch.bfloat16), x.view(T, 256)], 1).to(cuda)
    shape, _, dt = ops.kv_cache_shapes(T // 16 + 1, 2, 128, "mx4")
    kc, vc = torch.zeros(shape, dtype=dt, device=cuda), torch.zeros(shape, dtype=dt, device=cuda)
    q = torch.empty(T, 1, 128, dtype=torch.bfloat16, device=cuda)
    slots = torch.arange(T, device=cuda)
    ops.rope_kv_write(qkv, slots, ref.rope_cos_sin(T, 128, 500000.0, device=cuda), q, kc, vc, slots, 1, 2)
    codes, e = kref.quant(x.view(T, 2, 128))
    k, v = kv4.read(kc, vc, slots)
    assert torch.equal(v.double().cpu(), _oracle_rows(x.view(T, 2, 128)))
    got = kref.unpack(vc.cpu(), True)
    at = slots.cpu()
    neg = (codes >= 8) & (codes % 8 != 0)                                                    # (the sign of a zero is free)
    c = got[0][at // 16, :, at % 16]
    assert torch.equal(c % 8, codes % 8) and ((c >= 8) == (codes >= 8))[neg | (codes % 8 != 0)].all()
    assert torch.equal(got[1][at // 16, :, at % 16], e) and (k == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,Hq,H,D,slab", WRITES)
@pytest.mark.parametrize("special", [False, True])
def test_writer_on_the_gpu(cuda, T, Hq, H, D, slab, special):
    if slab and special:
        pytest.skip("slabs hold sums of products")
    a, b = (_write(T, Hq, H, D, dev, slab, special=special) for dev in ("cpu", cuda))
    nan = a[4].isnan()
    assert torch.equal(nan, b[4].isnan()) and torch.equal(a[4][~nan], b[4][~nan])
    for i, val in ((5, False), (6, True)):
        x, y = numbers(a[i], val), numbers(b[i], val)
        assert torch.equal(x, y), int((x != y).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_attention_on_the_gpu(cuda, monkeypatch, case, wide):
    """Every kind of tile, whatever the sizes from which on a plan takes it."""
    if wide:
        monkeypatch.setattr(kv4, "MANY_COST", -1e9)
        monkeypatch.setattr(kv4, "LEAST_SHARE", 0)
        monkeypatch.setattr(kv4, "SOME_PIECE", 2)
        monkeypatch.setattr(kv4, "MASS_TILES", 1)
    else:
        monkeypatch.setattr(kv4, "MANY_COST", 1e9)
    _check_attention(case, cuda)


@pytest.mark.gpu
def test_attention_again_is_the_same(cuda, monkeypatch):
    """Bit for bit, whatever ran in between; on another stream; as rows of a wider tensor."""
    monkeypatch.setattr(kv4, "MANY_COST", -1e9)
    segs = [(0, 1, 3000, 0), (1, 40, 500, 1), (41, 1, 70, 2)]
    kc, vc, tables = world(segs, 2, 128, 0, cuda)
    q = queries(42, 8, 128, 1, cuda)
    plan = kv4.attn_plan(segs, 8, 2, 128, 300, 4, cuda)
    lse = torch.empty(42, 8, device=cuda)
    a = kv4.attn(q, kc, vc, tables, plan, 0.1, lse=lse)
    m = kv4.attn_mass(q, lse, kc, tables, plan, 0.1)
    wide = torch.zeros(42, 8 * 128 + 256, dtype=torch.bfloat16, device=cuda)
    wide[:, :1024] = q.view(42, 1024)
    view = wide[:, :1024].unflatten(1, (8, 128))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lse2 = torch.empty(42, 8, device=cuda)
        b = kv4.attn(view, kc, vc, tables, plan, 0.1, lse=lse2)
        m2 = kv4.attn_mass(view, lse2, kc, tables, plan, 0.1)
    s.synchronize()
    assert torch.equal(a, b) and torch.equal(lse, lse2) and torch.equal(m, m2)


@pytest.mark.gpu
def test_together_and_captured(cuda):
    """A step as it is used, eager and replayed: write, attend, weigh, evict, attend to what is left."""
    Hq, H, D, lens, budget = 8, 2, 128, (90, 200, 33), 64
    g = torch.Generator().manual_seed(2)
    segs = [(i, 1, n - 1, i) for i, n in enumerate(lens)]
    kc0, vc0, tables = world(segs, H, D, 4, cuda, spare=14)
    free = [p for p in range(kc0.shape[0]) if p not in set(tables.flatten().tolist())]
    new = torch.tensor([[free.pop() for _ in range(4)] for _ in lens], dtype=torch.int32, device=cuda)
    qkv = torch.randn(3, (Hq + 2 * H) * D, generator=g).bfloat16().to(cuda)
    pos = torch.tensor([n - 1 for n in lens], device=cuda)
    slots = tables.long()[torch.arange(3), pos // 16] * 16 + pos % 16
    cs = ref.rope_cos_sin(1024, D, 500000.0, device=cuda)
    ln = torch.tensor(lens, dtype=torch.int32, device=cuda)
    kc, vc = kc0.clone(), vc0.clone()
    q, lse = torch.empty(3, Hq, D, dtype=torch.bfloat16, device=cuda), torch.empty(3, Hq, device=cuda)
    base = torch.rand(3, H, max(lens), generator=g).to(cuda)
    plan = kv4.attn_plan(segs, Hq, H, D, device=cuda)
    after = kv4.attn_plan([(i, 1, min(n, budget) - 1, i) for i, n in enumerate(lens)], Hq, H, D, device=cuda)

    def step():
        ops.rope_kv_write(qkv, pos, cs, q, kc, vc, slots, Hq, H)
        out = kv4.attn(q, kc, vc, tables, plan, 0.09, lse=lse)
        mass = kv4.attn_mass(q, lse, kc, tables, plan, 0.09, base=base)
        kept = kv4.evict_keep(mass, ln, budget, 4, 16)
        nm = kv4.evict(kc, vc, tables, kept, new, mass)
        return out, mass, kept, nm, kv4.attn(q, kc, vc, new, after, 0.09)

    eager = [t.clone() for t in step()]
    assert torch.equal(eager[2].cpu(), _keep_oracle(eager[1].cpu(), ln.cpu(), budget, 4, 16))
    o, _, _, bo, _, _ = oracle(q.cpu(), kc.cpu(), vc.cpu(), tables.cpu(), segs, 0, 0, 0.09)
    within(eager[0], o, bo, "out")
    o, _, _, bo, _, _ = oracle(q.cpu(), kc.cpu(), vc.cpu(), new.cpu(), [(i, 1, min(n, budget) - 1, i) for i, n in enumerate(lens)], 0, 0, 0.09)
    within(eager[4], o, bo, "out of the kept")
    graphs = []
    for _ in range(2):                                   # two graphs that live together
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(6):
        graph, outs = graphs[i % 2]
        kc.copy_(kc0)
        vc.copy_(vc0)
        for t in outs:
            t.zero_()
        torch.randn(1000, 1000, device=cuda).sum()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i


@pytest.mark.gpu
@pytest.mark.parametrize("R,H,N,budget,first,recent,kind", KEEPS)
def test_evict_keep_on_the_gpu(cuda, R, H, N, budget, first, recent, kind):
    m, lens = _masses(R, H, N, kind), _lens(R, N)
    want = _keep_oracle(m, lens, budget, first, recent)
    wide = torch.full((R, H, N + 3), 1e30, device=cuda)
    wide[..., :N] = m.to(cuda)
    assert torch.equal(kv4.evict_keep(wide[..., :N], lens.to(cuda), budget, first, recent).cpu(), want)


@pytest.mark.gpu
def test_evict_on_the_gpu(cuda):
    for kw in (dict(), dict(H=3, D=64), dict(lens=(1000, 17, 1, 640), budget=300)):
        a, b = _move("cpu", **kw), _move(cuda, **kw)
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_nothing_on_the_gpu(cuda):
    _nothing(cuda)


@pytest.mark.gpu
def test_bad_pages_on_the_gpu(cuda):
    _bad_pages(cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("segs", LEFT, ids=["tokens", "short", "long"])
def test_pages_left_behind_on_the_gpu(cuda, monkeypatch, D, segs, wide):
    monkeypatch.setattr(kv4, "MANY_COST", -1e9 if wide else 1e9)
    _pages_left_behind(cuda, D, segs)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_rows_without_angles(cuda, D):
    """A position that cos_sin does not have: the row's queries are no numbers, the cache stays as it is."""
    n = 7
    qkv = torch.randn(n, 4 * D + 4 * D, device=cuda).bfloat16()
    pos = torch.tensor([0, 5, -1, 6, 2 ** 40, 1, -2 ** 50], device=cuda)
    cs = torch.rand(6, D, device=cuda)
    slots = torch.arange(3, 3 + n, device=cuda)
    q = torch.zeros(n, 4, D, dtype=torch.bfloat16, device=cuda)
    kc, vc = (torch.full((1, 2, 16, D // 2 + D // 32), 255, dtype=torch.uint8, device=cuda) for _ in range(2))
    want = [t.clone() for t in (q, kc, vc)]
    ok = (pos >= 0) & (pos < 6)
    ops.rope_kv_write(qkv, pos, cs, q, kc, vc, slots, 4, 2)
    ops.rope_kv_write(qkv[ok], pos[ok], cs, (some := want[0][ok].clone()), *want[1:], slots[ok], 4, 2)
    assert torch.equal(q[ok], some) and q[~ok].isnan().all()
    assert torch.equal(kc, want[1]) and torch.equal(vc, want[2])


@pytest.mark.gpu
def test_pages_far_behind(cuda):
    """Pages whose bytes lie beyond 4 GiB."""
    H, D = 8, 128
    segs = [(0, 1, 200, 0), (1, 20, 60, 1)]
    kc, vc, tables = world(segs, H, D, 0, cuda)
    n = kc.shape[0]
    far = 600_000 - n
    big = [torch.zeros(600_000, H, 16, 68, dtype=torch.uint8, device=cuda) for _ in range(2)]
    big[0][far:], big[1][far:] = kc, vc
    q = queries(21, 32, D, 1, cuda)
    plan = kv4.attn_plan(segs, 32, H, D, device=cuda)
    lse, lse2 = torch.empty(21, 32, device=cuda), torch.empty(21, 32, device=cuda)
    a = kv4.attn(q, kc, vc, tables, plan, 0.1, lse=lse)
    b = kv4.attn(q, *big, tables + far, plan, 0.1, lse=lse2)
    assert torch.equal(a, b) and torch.equal(lse, lse2)
    assert torch.equal(kv4.attn_mass(q, lse, kc, tables, plan, 0.1), kv4.attn_mass(q, lse2, big[0], tables + far, plan, 0.1))
    slots = tables[0, :13].long().repeat_interleave(16) * 16 + torch.arange(16, device=cuda).repeat(13)
    for x, y in zip(kv4.read(kc, vc, slots), kv4.read(*big, slots + far * 16)):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    qkv = torch.randn(13 * 16, (32 + 16) * D, device=cuda).bfloat16()
    cs = ref.rope_cos_sin(400, D, 500000.0, device=cuda)
    pos = torch.arange(13 * 16, device=cuda)
    for c, s in (((kc, vc), slots), (big, slots + far * 16)):
        ops.rope_kv_write(qkv, pos, cs, torch.empty(13 * 16, 32, D, dtype=torch.bfloat16, device=cuda), *c, s, 32, H)
    assert torch.equal(big[0][far:], kc) and torch.equal(big[1][far:], vc)
    kept = torch.arange(1, 101, dtype=torch.int32, device=cuda).expand(1, H, 100).contiguous()
    to = torch.arange(7, dtype=torch.int32, device=cuda)[None]
    kv4.evict(*big, tables[:1] + far, kept, to + 100)
    ks = torch.arange(100 * 16, 100 * 16 + 100, device=cuda)
    for x, y in zip(kv4.read(*big, ks), kv4.read(*big, slots[1:101] + far * 16)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_refusals_on_the_gpu(cuda):
    ks, vs, dt = ops.kv_cache_shapes(4, 2, 128, "mx4")
    kc, vc = torch.zeros(ks, dtype=dt, device=cuda), torch.zeros(vs, dtype=dt, device=cuda)
    q, bt = queries(2, 8, 128, device=cuda), torch.zeros(2, 2, dtype=torch.int32, device=cuda)
    plan = kv4.attn_plan([(0, 2, 30, 1)], 8, 2, 128, device=cuda)
    with pytest.raises(ValueError):
        kv4.attn(q, kc, vc, bt, kv4.attn_plan([(0, 2, 30, 1)], 8, 2, 128, device="cpu"), 0.1)
    odd = torch.zeros(2 * 8 * 128 + 4, dtype=torch.bfloat16, device=cuda)[4:].view(2, 8, 128)
    for args in ((odd, kc, vc, bt), (q, kc, vc, bt.cpu()), (q, kc, vc.cpu(), bt), (q, kc[:0], vc[:0], bt)):
        with pytest.raises(ValueError):
            kv4.attn(*args, plan, 0.1)
    for scale in (0.0, -0.1, math.inf, math.nan):
        with pytest.raises(ValueError):
            kv4.attn(q, kc, vc, bt, plan, scale)
        with pytest.raises(ValueError):
            kv4.attn_mass(q, torch.zeros(2, 8, device=cuda), kc, bt, plan, scale)
    with pytest.raises(ValueError):
        kv4.read(kc, vc, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.rope_kv_write(torch.zeros(2, 100, dtype=torch.bfloat16, device=cuda), torch.zeros(2, dtype=torch.long, device=cuda),
                          torch.zeros(9, 128, device=cuda), q, kc, vc, None, 8, 2)
    kv4.attn(q, kc, vc, bt, plan, 0.1)


# ---- engine ---------------------------------------------------------------------------------------------------------------
def _dense(model, tokens):
    """Logits of the dense model in fp32 whose keys and values stand for what the cache holds of them."""
    from kafka_llm_service_amd.models import oracle as orc

    cfg, D, hq, hkv = model.cfg, model.D, model.hq, model.hkv
    t = torch.tensor(tokens, device=model.device)
    T = t.shape[0]
    cs = model.cos_sin[:T].float()
    h = model.embed[t].float()
    see = torch.ones(T, T, dtype=torch.bool, device=h.device).tril()
    four = lambda x: kref.values(*kref.quant(x))
    for lw in model.layers:
        qkv = orc._lin(orc._rms(h, lw.input_norm, cfg.rms_norm_eps), lw.qkv).view(T, hq + 2 * hkv, D)
        q, k, v = orc._rope(qkv[:, :hq], cs), four(orc._rope(qkv[:, hq:hq + hkv], cs)), four(qkv[:, hq + hkv:])
        o = torch.empty(T, hq, D, device=h.device)
        for x in range(hq):
            s = (q[:, x] @ k[:, x * hkv // hq].T.contiguous() * model.scale).masked_fill(~see, -math.inf)
            o[:, x] = torch.softmax(s, -1) @ v[:, x * hkv // hq].contiguous()
        h = h + orc._lin(o.view(T, -1), lw.o)
        gu = orc._lin(orc._rms(h, lw.post_norm, cfg.rms_norm_eps), lw.gate_up)
        f = gu.shape[-1] // 2
        h = h + orc._lin(torch.nn.functional.silu(gu[:, :f]) * gu[:, f:], lw.down)
    return orc._lin(orc._rms(h, model.final_norm, cfg.rms_norm_eps), model.lm_head)[:, :cfg.vocab_size]


def _engine(model, device, gap):
    """Every greedy token is the oracle's best within ``gap`` of its logits, as with the other caches; prefixes are shared."""
    from kafka_llm_service_amd.engine.engine import EngineConfig, LLMEngine
    from kafka_llm_service_amd.engine.sequence import SamplingParams

    eng = LLMEngine(EngineConfig(model=model, device=device, num_kv_blocks=1024, max_model_len=4096, kv_dtype="mx4"))
    assert ops.is_mx4_cache(eng.runner.k_caches[0])
    g = torch.Generator().manual_seed(11)
    pre = torch.randint(0, 5000, (130,), generator=g).tolist()
    prompts = [pre + torch.randint(0, 5000, (n,), generator=g).tolist() for n in (3, 60, 150, 7)]
    sp = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True)
    for _ in range(2):                                      # (the second time behind cached prefixes)
        for p, o in zip(prompts, eng.generate(prompts, sp)):
            assert len(o) == 6
            lg = _dense(eng.model, p + o).cpu()
            for i, tok in enumerate(o):
                row = lg[len(p) - 1 + i]
                assert (row.max() - row[tok]).item() < gap, f"token {i}: gap {(row.max() - row[tok]).item():.3f}"


def test_engine_cpu():
    _engine("tiny-llama", "cpu", 0.15)


@pytest.mark.gpu
def test_engine_on_the_gpu(cuda):
    _engine("small-llama", str(cuda), 0.25)


@pytest.mark.gpu
def test_step_plan_is_the_plan(cuda, monkeypatch):
    """An engine step's tables, as uploaded, give what attn_plan's give."""
    monkeypatch.setattr(kv4, "MANY_COST", -1e9)
    segs = [(0, 1, 500, 0), (1, 1, 33, 1), (2, 177, 900, 2), (179, 3, 4000, 3), (182, 10, 70, 4)]
    flat = kv4.step_tables(segs, 32, 2, 128)
    p = kv4.step_plan(flat, torch.from_numpy(flat).to(cuda), 32, 2, 128)
    assert (p.rows, p.covered, p.keys, p.tables) == (192, 192, 4003, 5)
    assert [s[0] for s in kv4._tables(kv4._plan(segs, 32, 2, 128, 0, 0)[1], 32, 2, 128, 0, 0)[0]] == [16, 32, 256]
    kc, vc, tables = world(segs, 2, 128, 0, cuda)
    q = queries(192, 32, 128, 1, cuda)
    want = kv4.attn(q, kc, vc, tables, kv4.attn_plan(segs, 32, 2, 128, device=cuda), 0.1)
    assert torch.equal(kv4.attn(q, kc, vc, tables, p, 0.1), want)
    with pytest.raises(ValueError):
        kv4.attn_mass(q, torch.zeros(192, 32, device=cuda), kc, tables, p, 0.1)


def test_widened_keys_are_those_that_a_tile_sees(monkeypatch):
    """Every block of a wide tile's list is at its place among its segment's in the workspace."""
    import numpy as np

    g = torch.Generator().manual_seed(1)
    r = lambda hi: int(torch.randint(0, hi, (1,), generator=g))
    monkeypatch.setattr(kv4, "MANY_COST", -1e9)
    for _ in range(100):
        segs = np.array([(1000 * i, 33 + r(400), r(6000), 10 + i) for i in range(1 + r(4))])
        window, first = (0, 0) if r(3) == 0 else (1 + r(1500), r(300))
        shapes, (items, merges, keys) = kv4._tables(segs, 8, 2, 128, window, first)
        assert [s[0] for s in shapes] == [256]
        for row, n, pos, base, head, tail, lo, hi, _, *_ in items.tolist():
            t, f = max(0, pos - window + 1) // 64 if window else 0, 0
            f = min(-(-first // 64), t)
            for v in range(lo, hi):
                b = v if v < f else v - f + t
                k = keys[base + (b if b < head else b - tail + head)].tolist()
                seg = segs[row // 1000]
                assert k[:3] == [seg[3], b, seg[1] + seg[2] - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
def test_split_tiles_side_by_side(cuda, monkeypatch, wide):
    """Work in several parts whose last one joins them: the same plan eager on two streams and in two graphs, all at once and again."""
    monkeypatch.setattr(kv4, "MANY_COST", -1e9 if wide else 1e9)
    monkeypatch.setattr(kv4, "SOME_PIECE", 2)
    monkeypatch.setattr(kv4, "MASS_TILES", 1)
    segs = [(0, 1, 4000, 0), (1, 1, 9000, 1), (2, 2, 2500, 2), (4, 90, 1500, 3)]
    kc, vc, tables = world(segs, 2, 128, 0, cuda)
    q = queries(94, 8, 128, 1, cuda)
    plan = kv4.attn_plan(segs, 8, 2, 128, device=cuda)
    p, a = kv4._plan(segs, 8, 2, 128, 0, 0)
    shapes = kv4._tables(a, 8, 2, 128, 0, 0)[0]
    assert [x[0] for x in shapes] == ([16, 256] if wide else [16, 32]) and all(x[2] > 3 for x in shapes)   # (slots of partial results)
    assert kv4._mass_tables(a, 4, 2, p.keys, 0, 0)[2] > 3

    def step():
        l = torch.zeros(94, 8, device=cuda)
        o = kv4.attn(q, kc, vc, tables, plan, 0.1, lse=l)
        return o, l, kv4.attn_mass(q, l, kc, tables, plan, 0.1)

    want = step()
    streams, runs = [torch.cuda.Stream() for _ in range(4)], []
    for s in streams[:2]:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                outs = step()
            runs.append((graph, outs))
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    eager = []
    for _ in range(10):
        for s, (graph, _) in zip(streams, runs):
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams[2:]:
            with torch.cuda.stream(s):
                eager.append(step())
    torch.cuda.synchronize()
    for outs in eager + [r[1] for r in runs]:
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


# ---- segments without rows beside others ----------------------------------------------------------------------------------
def _empty_beside(device):
    """A segment without rows, wherever its first row would be, gives its keys nothing: they keep what they had."""
    for segs, T in (([(0, 1, 0, 0), (5, 0, 0, 1)], 1), ([(900, 0, 77, 1), (0, 40, 100, 0), (40, 0, 3, 0), ((1 << 26) - 1, 0, 0, 2)], 40)):
        kc, vc, tables = world(segs, 2, 128, 0, device)
        q, lse = queries(T, 8, 128, 1, device), torch.zeros(T, 8, device=device)
        full = [s for s in segs if s[1]]
        plan, alone = (kv4.attn_plan(x, 8, 2, 128, device=device) for x in (segs, full))
        out = kv4.attn(q, kc, vc, tables, plan, 0.1, lse=lse)
        assert torch.equal(out, kv4.attn(q, kc, vc, tables, alone, 0.1))
        want = torch.zeros(len(segs), 2, plan.keys, device=device)
        want[[i for i, s in enumerate(segs) if s[1]]] = kv4.attn_mass(q, lse, kc, tables, alone, 0.1)
        got = torch.full_like(want, 5.0)
        assert kv4.attn_mass(q, lse, kc, tables, plan, 0.1, out=got) is got and torch.equal(got, want)
        base = torch.rand(want.shape, generator=torch.Generator().manual_seed(3)).to(device)
        got = torch.full_like(want, 5.0)
        kv4.attn_mass(q, lse, kc, tables, plan, 0.1, base=base, out=got)
        assert torch.equal(got, base + want)


def test_empty_segments_beside_others_reference():
    _empty_beside("cpu")


@pytest.mark.gpu
def test_empty_segments_beside_others_on_the_gpu(cuda):
    _empty_beside(cuda)
