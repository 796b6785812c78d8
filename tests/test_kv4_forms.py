"""The 4-bit cache's kernels form by form: loops as deep as long sequences make them, scores without the 4-bit product's cut, pages
that are none in every kind of tile.

Tolerances of ``_sharp``: each query has one element in every eight neighbours, of at most two bits of mantissa and within a factor of
four of each other, so that every form of the kernels takes it exactly (in e4m3 as well), a group of eight products is one exact
number, and nothing of it is cut. A score is then a sum of D / 8 exact numbers in fp32 and a product by the scale; with an addition that cuts
instead of rounding, 2^-23 of A = the largest sum_d |scale q_d k_d| of a row for each, S = 2 (D / 8 + 4) 2^-24 A bounds its error. The
exponential and its argument add 2^-22 (1 + A): EW = 2 (S + 2^-22 (1 + A)) bounds a weight's relative error with its sum's. lse is off by
(EW + n 2^-24) / ln 2 and its own rounding, a key's weight from R rows by 2 EW + (n + R + 2) 2^-24 + 2^-22 (1 + |lse|) of itself; keys that no
row sees have received exactly nothing. The output has P in bf16 and its own rounding: (2^-8 + EW + n 2^-24) sum w |v| + 2^-8 |o|.
``_fine``: queries whose elements have all eight bits of bf16, one of every eight neighbours between 1 and 2, the others between 2^-8 and 2^-5, so that
in 20 bits of fixed point below the largest of 32 each is whole; every product is a multiple of a unit of which a row's sum of sizes has less than 2^24 (asserted), so a score is exact in fp32 in
whatever order it is summed, and S = 2^-23 max |scale q k|."""
import math

import numpy as np
import pytest
import torch

from kafka_llm_service_amd import ops
from kafka_llm_service_amd.ops import kv4
from kafka_llm_service_amd.ops import kv4_reference as kref
from kafka_llm_service_amd.ops import reference as ref
from test_kv4 import CASES, _check_attention, _id, numbers, oracle, queries, within, world


# ---- deep loops -----------------------------------------------------------------------------------------------------------
def _one_piece(monkeypatch, waves=0):
    """Plans whose tiles are taken in one piece each, those of single tokens by 4 or 8 waves."""
    monkeypatch.setattr(kv4, "CUS", 1)
    monkeypatch.setattr(kv4, "LEAST_SHARE", 0)
    monkeypatch.setattr(kv4, "SHORT_TILE", 1 << 40 if waves == 4 else 0)
    monkeypatch.setattr(kv4, "SOME_PIECE", 1 << 40)
    monkeypatch.setattr(kv4, "MANY_BLOCKS", 1 << 40)
    monkeypatch.setattr(kv4, "MASS_WGS", 1)
    monkeypatch.setattr(kv4, "MASS_MANY_WGS", 1)


def _items(case):
    Hq, H, D, segs, window, first = case
    p, a = kv4._plan(segs, Hq, H, D, window, first)
    shapes, arrays = kv4._tables(a[a[:, 1] > 0], Hq, H, D, window, first)
    return shapes, arrays, kv4._mass_tables(a, Hq // H, H, p.keys, window, first)


#: single tokens: (waves, case); of 4 and 8 waves, more than 16 and more than 32 blocks a wave
TOKENS = [(4, (4, 2, 128, [(0, 1, 8700, 0), (1, 1, 4500, 1), (2, 1, 100, 2)], 0, 0)),
          (4, (8, 1, 64, [(0, 1, 8500, 0), (1, 1, 4300, 1)], 0, 0)),
          (4, (4, 1, 128, [(0, 1, 9000, 0), (1, 2, 4444, 1)], 4300, 130)),
          (8, (4, 1, 128, [(0, 1, 17000, 0), (1, 1, 9000, 1)], 0, 0)),
          (8, (2, 1, 64, [(0, 1, 16999, 0), (1, 1, 700, 1)], 0, 0)),
          (8, (3, 1, 64, [(0, 3, 12000, 0)], 9000, 20))]


@pytest.mark.gpu
@pytest.mark.parametrize("waves,case", TOKENS, ids=lambda x: _id(x) if isinstance(x, tuple) else f"{x}waves")
def test_single_tokens_of_long_sequences(cuda, monkeypatch, waves, case):
    _one_piece(monkeypatch, waves)
    shapes, (items, *_), (few, many, _) = _items(case)
    assert [s[:3] for s in shapes] == [(16, waves, 0)]
    assert max(hi - lo for *_, lo, hi, _, _ in items.tolist()) > 16 * waves
    if not case[4]:
        assert max(hi - lo for *_, lo, hi, _, _ in items.tolist()) > 32 * waves
    sizes = sorted({it[6] - it[5] for it in few.tolist()})
    assert sizes[-1] == 32 and not len(many)                  # (eight blocks a wave, and the rest)
    _check_attention(case, cuda)


#: short portions: tiles of 32 rows, four waves
SHORT = [(4, 1, 128, [(0, 9, 8300, 0), (9, 5, 4500, 1)], 0, 0), (4, 2, 64, [(0, 17, 8260, 0)], 0, 0), (5, 1, 64, [(0, 13, 9000, 0)], 4600, 130),
         (4, 1, 128, [(0, 20, 7000, 0)], 5000, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", SHORT, ids=_id)
def test_short_portions_behind_long_histories(cuda, monkeypatch, case):
    monkeypatch.setattr(kv4, "MANY_COST", 1e9)
    _one_piece(monkeypatch)
    shapes, (items, *_), _ = _items(case)
    assert [s[:3] for s in shapes] == [(32, 4, 0)]
    assert max(hi - lo for *_, lo, hi, _, _ in items.tolist()) > (16 if case[4] else 32) * 4
    _check_attention(case, cuda)


#: long portions: tiles of keys an item sees, odd and even numbers of them
LONG = [(4, 1, 128, [(0, 200, 1000, 0)], 0, 0), (4, 1, 128, [(0, 150, 1100, 0)], 0, 0), (4, 1, 64, [(0, 100, 1000, 0), (100, 70, 1500, 1)], 0, 0),
        (8, 2, 64, [(0, 70, 1230, 0)], 900, 70), (3, 1, 128, [(0, 190, 1300, 0)], 1000, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LONG, ids=_id)
def test_long_portions_in_one_piece(cuda, monkeypatch, case):
    monkeypatch.setattr(kv4, "MANY_COST", -1e9)
    _one_piece(monkeypatch)
    shapes, (items, *_), (_, many, slots) = _items(case)
    assert [s[0] for s in shapes] == [kv4.MANY_ROWS[case[2]]] and shapes[0][2] == 0
    sizes = {it[7] - it[6] for it in items.tolist()}
    assert min(sizes) > 8 and {n % 2 for n in sizes} == {0, 1}
    assert slots == 0 and len(many)
    _check_attention(case, cuda)


# ---- scores without a cut -------------------------------------------------------------------------------------------------
def _sparse(T, Hq, D, seed=2):
    g = torch.Generator().manual_seed(seed)
    size = torch.tensor([1.0, 1.5, 2.0, 3.0])[torch.randint(0, 4, (T, Hq, D // 8), generator=g)]
    size *= torch.randint(0, 2, size.shape, generator=g) * 2 - 1
    q = torch.zeros(T, Hq, D // 8, 8)
    return q.scatter_(-1, torch.randint(0, 8, size.shape, generator=g)[..., None], size[..., None]).flatten(-2).bfloat16()


def _fine(T, Hq, D, seed=6):
    g = torch.Generator().manual_seed(seed)
    size = torch.randint(6, 9, (T, Hq, D // 8, 8), generator=g)
    size.scatter_(-1, torch.randint(0, 8, (T, Hq, D // 8, 1), generator=g), 0)      # (of every eight one of the largest)
    q = (1 + torch.randint(0, 128, (T, Hq, D), generator=g) / 128) * torch.exp2(-size.flatten(-2).float())
    return (q * (torch.randint(0, 2, q.shape, generator=g) * 2 - 1)).bfloat16()


def _sharp(case, device, fine=False):
    Hq, H, D, segs, window, first = case
    G = Hq // H
    kc, vc, tables = world(segs, H, D, 5, device)
    T = max(s[0] + s[1] for s in segs)
    q, scale = (_fine if fine else _sparse)(T, Hq, D), 0.25
    plan = kv4.attn_plan(segs, Hq, H, D, window, first, device)
    lse = torch.empty(T, Hq, device=device)
    out = kv4.attn(q.to(device), kc, vc, tables, plan, scale, lse=lse).cpu()
    mass = kv4.attn_mass(q.to(device), lse, kc, tables, plan, scale).cpu().double()
    lse, kc, vc, tables = lse.cpu(), kc.cpu(), vc.cpu(), tables.cpu()
    for i, (t0, rows, p0, tr) in enumerate(segs):
        if not rows:
            assert (mass[i] == 0).all()
            continue
        n = p0 + rows
        ids = tables[tr, :(n + 15) // 16].long()
        k, v = (numbers(c[ids], val).transpose(1, 2).flatten(0, 1)[:n] for c, val in ((kc, False), (vc, True)))
        back = p0 + torch.arange(rows)[:, None] - torch.arange(n)[None]
        see = (back >= 0) & ((back < window) | (torch.arange(n) < first)[None]) if window else back >= 0
        for h in range(H):
            want, bound = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
            for g in range(h * G, (h + 1) * G):
                x = q[t0:t0 + rows, g].double()
                s = (x @ k[:, h].T * scale).masked_fill(~see, -math.inf)
                A = (x.abs() @ k[:, h].abs().T * scale).masked_fill(~see, 0).amax(-1, keepdim=True)
                if fine:
                    e = kref.unpack(kc[ids], False)[1].transpose(1, 2).flatten(0, 1)[:n, h].amin(-1)       # 2^-15 times 1/2 times the key's least scale
                    assert (x.abs() @ k[:, h].abs().T / torch.exp2(e - 16.0) < 2.0 ** 24).all()
                    A = s.masked_fill(~see, 0).abs().amax(-1, keepdim=True)
                    S = 2.0 ** -23 * A
                else:
                    S = 2 * (D // 8 + 4) * 2.0 ** -24 * A
                EW = 2 * (S + 2.0 ** -22 * (1 + A))
                ls = torch.logsumexp(s, -1, keepdim=True)
                w = torch.exp(s - ls)
                o = w @ v[:, h]
                within(out[t0:t0 + rows, g], o, (2.0 ** -8 + EW + n * 2.0 ** -24) * (w @ v[:, h].abs()) + 2.0 ** -8 * o.abs(), "out")
                within(lse[t0:t0 + rows, g], ls[:, 0] / math.log(2), ((EW + n * 2.0 ** -24) / math.log(2) + 2.0 ** -23 * (1 + ls.abs()))[:, 0], "lse")
                want += w.sum(0)
                bound += (w * (2 * EW + (n + rows * G + 2) * 2.0 ** -24 + 2.0 ** -22 * (1 + ls.abs()))).sum(0)
            within(mass[i, h, :n], want, bound + 2.0 ** -120, "mass")
            unseen = ~see.any(0)
            assert (mass[i, h, :n][unseen] == 0).all() and (mass[i, h, n:] == 0).all()
            # (no bound hides a bias: it is below a thousandth of every weight of an ordinary size)
            assert (bound <= 1e-3 * want)[~unseen & (want > 1e-30)].all()


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_sharp_scores_reference(case):
    _sharp(case, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_sharp_scores_on_the_gpu(cuda, monkeypatch, case, wide):
    monkeypatch.setattr(kv4, "MANY_COST", -1e9 if wide else 1e9)
    _sharp(case, cuda)


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_fine_scores_reference(case):
    _sharp(case, "cpu", True)


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_fine_scores_on_the_gpu(cuda, monkeypatch, case, wide):
    """Nothing of a score is lost in any form: as exact as 32 bits are."""
    monkeypatch.setattr(kv4, "MANY_COST", -1e9 if wide else 1e9)
    _sharp(case, cuda, True)


# ---- queries of all sizes -------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,cost", [(1, 1e9), (9, 1e9), (150, -1e9)])
@pytest.mark.parametrize("D", [64, 128])
def test_small_elements_beside_a_large_one(cuda, monkeypatch, D, rows, cost):
    """An element 2^-t of its neighbour, which meets only zeros, under a scale 2^t as large: the same scores, whole down to 2^-11."""
    monkeypatch.setattr(kv4, "MANY_COST", cost)
    n = 400
    segs = [(0, rows, n - rows, 0)]
    kc, vc, tables = world(segs, 1, D, 0, cuda, garbage=False)
    g = torch.Generator().manual_seed(2)
    k = torch.zeros(n // 16, 1, 16, D)
    k[..., 1] = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])[torch.randint(0, 8, (n // 16, 1, 16), generator=g)]
    k[..., 2] = 6.0                                           # (the scale is one; no query looks here)
    kc[tables[0, :n // 16].long()] = kref.pack_pages(k, k)[0].to(cuda)
    plan = kv4.attn_plan(segs, 4, 1, D, device=cuda)
    x = k[:, 0, :, 1].flatten().double()
    see = torch.arange(n)[None] <= n - rows + torch.arange(rows)[:, None]
    first = None
    for t in range(12):
        q = torch.zeros(rows, 4, D, dtype=torch.bfloat16, device=cuda)
        q[..., 0], q[..., 1] = 1.9921875, 1.9921875 * 2.0 ** -t
        lse = torch.zeros(rows, 4, device=cuda)
        out = kv4.attn(q, kc, vc, tables, plan, 0.5 * 2.0 ** t, lse=lse)
        mass = kv4.attn_mass(q, lse, kc, tables, plan, 0.5 * 2.0 ** t)
        if first is None:
            first = out, lse, mass
            want = torch.logsumexp((x * 1.9921875 * 0.5).expand(rows, n).masked_fill(~see, -math.inf), -1) / math.log(2)
            # scores below 6, a sum of 400 numbers: (400 2^-24 + 2 * 7 * 2^-22) / ln 2
            assert ((lse.double().cpu() - want[:, None]).abs() <= 4e-5).all()
        assert all(torch.equal(a, b) for a, b in zip((out, lse, mass), first)), t


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cost", [(1, 1e9), (9, 1e9), (150, -1e9)])
@pytest.mark.parametrize("D", [64, 128])
def test_queries_that_are_no_numbers(cuda, monkeypatch, D, rows, cost):
    """A row with an infinity or no number in it is no numbers, those beside it and rows of zeros and of the smallest numbers are right. (Not
    bit for bit as without it: a tile's rows raise their maxima together, and by what P is divided before it is rounded decides its last bit.)"""
    monkeypatch.setattr(kv4, "MANY_COST", cost)
    segs = [(0, rows, 300, 0)]
    kc, vc, tables = world(segs, 2, D, 0, cuda)
    q = queries(rows, 8, D, 1, cuda)
    plan = kv4.attn_plan(segs, 8, 2, D, device=cuda)
    lse2 = torch.zeros(rows, 8, device=cuda)
    o, l, _, bo, bl, _ = oracle(q.cpu(), kc.cpu(), vc.cpu(), tables.cpu(), segs, 0, 0, 0.1)
    bad = q.clone()
    bad[-1, 3, 5], bad[-1, 6, D - 1], bad[0, 0, D // 2] = math.nan, math.inf, -math.inf
    bad[0, 5], bad[0, 1], bad[0, 2] = 0.0, 1e-38, 0.0
    bad[0, 1, 1::2] = -9e-41
    out = kv4.attn(bad, kc, vc, tables, plan, 0.1, lse=lse2)
    none = torch.zeros(rows, 8, dtype=torch.bool, device=cuda)
    none[-1, 3] = none[-1, 6] = none[0, 0] = True
    other = ~none
    other[0, 5] = other[0, 1] = other[0, 2] = False
    assert out[none].isnan().all() and lse2[none].isnan().all()
    other = other.cpu()
    within(out.cpu()[other], o[other], bo[other], "out")
    within(lse2.cpu()[other], l[other], bl[other], "lse")
    even = math.log2(301)                                     # of 301 equal weights
    assert out[0, (1, 2, 5),].isfinite().all() and ((lse2[0, (1, 2, 5),] - even).abs() < 1e-5).all()


# ---- pages that are none, in every kind of tile ---------------------------------------------------------------------------
def _bad_portions(device, D, rows):
    """Rows in front of a page that is none are what they are without it, those that see it no numbers."""
    segs = [(0, rows, 0, 0), (rows, rows, 200, 1), (2 * rows, rows, 200, 2)]
    kc, vc, tables = world(segs, 2, D, 1, device)
    q = queries(3 * rows, 8, D, 1, device)
    plan = kv4.attn_plan(segs, 8, 2, D, device=device)
    lse, lse2 = torch.zeros(3 * rows, 8, device=device), torch.zeros(3 * rows, 8, device=device)
    good = kv4.attn(q, kc, vc, tables, plan, 0.1, lse=lse)
    for what in (-1, kc.shape[0], -(1 << 31), (1 << 31) - 1):
        bad = tables.clone()
        bad[0, (rows - 1) // 16], bad[2, 5] = what, what       # the last page of the first, a page of the history of the last
        out = kv4.attn(q, kc, vc, bad, plan, 0.1, lse=lse2)
        sees = torch.arange(rows, device=device) >= (rows - 1) // 16 * 16
        assert out[:rows][sees].isnan().all() and lse2[:rows][sees].isnan().all()
        far = max(0, (rows - 1) // 16 * 16 - 32)              # (rows next to them, in a tile of up to 32, may be)
        if kv4.MANY_COST < 0:
            far = (rows - 1) // 16 * 16
        assert torch.equal(out[:far], good[:far]) and torch.equal(lse2[:far], lse[:far])
        assert torch.equal(out[rows:2 * rows], good[rows:2 * rows]) and out[2 * rows:].isnan().all() and lse2[2 * rows:].isnan().all()
        mass = kv4.attn_mass(q, lse, kc, bad, plan, 0.1)
        good_mass = kv4.attn_mass(q, lse, kc, tables, plan, 0.1)
        assert torch.equal(mass[1], good_mass[1]) and mass[2, :, 80:96].isnan().all()


@pytest.mark.parametrize("rows", [40, 150])
@pytest.mark.parametrize("D", [64, 128])
def test_bad_pages_of_portions_reference(D, rows):
    _bad_portions("cpu", D, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cost", [(40, 1e9), (150, 1e9), (150, -1e9)])
@pytest.mark.parametrize("D", [64, 128])
def test_bad_pages_of_portions_on_the_gpu(cuda, monkeypatch, D, rows, cost):
    monkeypatch.setattr(kv4, "MANY_COST", cost)
    _bad_portions(cuda, D, rows)


# ---- outputs over inputs ---------------------------------------------------------------------------------------------------
def _overlaps(device):
    """An output may take its input's place; one that covers a part of it is refused."""
    segs = [(0, 1, 300, 0), (1, 9, 500, 1), (10, 140, 700, 2)]
    kc, vc, tables = world(segs, 2, 128, 0, device)
    q = queries(151, 8, 128, 1, device)
    plan = kv4.attn_plan(segs, 8, 2, 128, device=device)
    lse = torch.zeros(150, 8, device=device)
    want = kv4.attn(q[:150], kc, vc, tables, plan, 0.1, lse=lse)
    mass = kv4.attn_mass(q[:150], lse, kc, tables, plan, 0.1)
    for first in (0, 1):
        both = q.clone()
        mine, other = both[first:150 + first], both[1 - first:151 - first]
        mine.copy_(q[:150])
        with pytest.raises(ValueError):
            kv4.attn(mine, kc, vc, tables, plan, 0.1, out=other)
        assert torch.equal(mine, q[:150])
        assert kv4.attn(mine, kc, vc, tables, plan, 0.1, out=mine) is mine and torch.equal(mine, want)
        buf = torch.zeros(mass.numel() + 4, device=device)
        base, out = buf[4 * first:][:mass.numel()].view(mass.shape), buf[4 * (1 - first):][:mass.numel()].view(mass.shape)
        with pytest.raises(ValueError):
            kv4.attn_mass(q[:150], lse, kc, tables, plan, 0.1, base=base, out=out)
        assert (buf == 0).all()
        kv4.attn_mass(q[:150], lse, kc, tables, plan, 0.1, base=base, out=base.view(mass.shape))
        assert torch.equal(base, mass)


def test_overlaps_reference():
    _overlaps("cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
def test_overlaps_on_the_gpu(cuda, monkeypatch, wide):
    monkeypatch.setattr(kv4, "MANY_COST", -1e9 if wide else 1e9)
    monkeypatch.setattr(kv4, "SOME_PIECE", 2)
    _overlaps(cuda)


# ---- the room that widened keys take --------------------------------------------------------------------------------------
def _widened_bytes(case):
    shapes, arrays, _ = _items(case)
    return sum(s[5] for s in shapes) * case[1] * 256 * case[2], [s[0] for s in shapes]


def test_room_of_widened_keys(monkeypatch):
    """However many portions a step has, and however long their histories are, what is widened for them stays within its bound."""
    segs = [(128 * i, 128, 131000, i) for i in range(64)]
    size, shapes = _widened_bytes((32, 8, 128, segs, 0, 0))
    assert 0 < size <= kv4.MANY_BYTES < 64 * 131128 * 8 * 512 and shapes == [32, 256]
    g = torch.Generator().manual_seed(0)
    r = lambda hi: int(torch.randint(0, hi, (1,), generator=g))
    monkeypatch.setattr(kv4, "MANY_COST", -1e9)
    for _ in range(50):
        case = (8, 2, (64, 128)[r(2)], [(100 * i, 32 + r(68), r(9000), i) for i in range(1 + r(9))], *((0, 0) if r(2) else (1 + r(900), r(100))))
        monkeypatch.setattr(kv4, "MANY_BYTES", 1 << (20 + r(8)))
        assert _widened_bytes(case)[0] <= kv4.MANY_BYTES
        monkeypatch.setattr(kv4, "MANY_BYTES", 1 << 40)
        assert _widened_bytes(case)[1] == [kv4.MANY_ROWS[case[2]]]


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_portions_beyond_the_room_for_widened_keys(cuda, monkeypatch, D):
    """Portions that fit and portions that do not, beside single tokens, in one call."""
    case = (8, 2, D, [(0, 1, 300, 0), (1, 90, 400, 1), (91, 60, 1000, 2), (151, 40, 100, 3)], 0, 0)
    monkeypatch.setattr(kv4, "MANY_COST", -1e9)
    monkeypatch.setattr(kv4, "MANY_BYTES", 10 * 2 * 256 * D)
    assert _widened_bytes(case) == (8 * 2 * 256 * D, [16, 32, kv4.MANY_ROWS[D]])
    _check_attention(case, cuda)


# ---- large values ---------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,cost", [(1, 1e9), (9, 1e9), (150, -1e9)])
@pytest.mark.parametrize("D", [64, 128])
def test_large_values(cuda, monkeypatch, D, rows, cost):
    """Values just below 2^104 / n, whose weights reach 2^23 times the first keys': right; other rows do not notice larger ones."""
    monkeypatch.setattr(kv4, "MANY_COST", cost)
    H, Hq, n = 1, 4, 2000
    segs = [(0, rows, n - rows, 0), (rows, rows, n - rows, 1)]
    kc, vc, tables = world(segs, H, D, 0, cuda, garbage=False)
    order = tables[:, :n // 16].long()
    j = torch.arange(n, device=cuda).view(-1, 16)
    k = torch.zeros(n // 16, H, 16, D, device=cuda)
    k[..., 0] = torch.where(j < 64, 0.0, 6.0)[:, None]
    v = torch.full((n // 16, H, 16, D), 6 * 2.0 ** 90, device=cuda)                 # 6 * 2^90 < 2^104 / 2000
    for s, x in ((0, v), (1, torch.full_like(v, math.inf))):
        a, b = kref.pack_pages(k.cpu(), x.cpu())
        kc[order[s]], vc[order[s]] = a.to(cuda), b.to(cuda)
    q = torch.zeros(2 * rows, Hq, D, dtype=torch.bfloat16, device=cuda)
    q[..., 0] = 1
    scale = 23 * math.log(2) / 6                                                   # base 2: the later keys' scores are 23, the first ones' 0
    lse = torch.zeros(2 * rows, Hq, device=cuda)
    out = kv4.attn(q, kc, vc, tables, kv4.attn_plan(segs, Hq, H, D, device=cuda), scale, lse=lse)
    assert torch.equal(out[:rows].float(), torch.full((rows, Hq, D), 6 * 2.0 ** 90, device=cuda))
    want = torch.log2((n - rows + 1 + torch.arange(2 * rows, device=cuda) % rows - 64).double() * 2.0 ** 23 + 64)
    assert ((lse.double() - want[:, None]).abs() <= 2.0 ** -12).all()              # (sums of n numbers: n 2^-24 / ln 2, a score of 23: 2^-18)


# ---- writer: sums of slabs that are no numbers ----------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("T,Hq,H,D,slab", [(33, 4, 4, 64, 2), (5, 32, 8, 128, 4), (3, 3, 1, 128, 1)])
def test_writer_of_slabs_with_infinities(cuda, T, Hq, H, D, slab):
    """As the plain form: not a number (also the sum of two infinities) is stored as zero, an infinity as the largest."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(slab, T, (Hq + 2 * H) * D, generator=g)
    flat = x.view(-1)
    flat[::97], flat[5::301], flat[9::307], flat[3::11] = math.inf, -math.inf, math.nan, 3e38
    pos, slots = torch.arange(T) * 7, torch.randperm(T + 20, generator=g)[:T]
    cs = ref.rope_cos_sin(1024, D, 500000.0)
    shape, _, dt = ops.kv_cache_shapes((T + 35) // 16, H, D, "mx4")
    got = []
    for dev in ("cpu", cuda):
        q = torch.zeros(T, Hq, D, dtype=torch.bfloat16, device=dev)
        kc, vc = torch.zeros(shape, dtype=dt, device=dev), torch.zeros(shape, dtype=dt, device=dev)
        ops.rope_kv_write(x.to(dev), pos.to(dev), cs.to(dev), q, kc, vc, slots.to(dev), Hq, H)
        got.append((q.cpu(), numbers(kc.cpu(), False), numbers(vc.cpu(), True)))
    (qa, ka, va), (qb, kb, vb) = got
    nan = qa.isnan()
    assert nan.any() and torch.equal(nan, qb.isnan()) and torch.equal(qa[~nan], qb[~nan])
    assert torch.equal(ka, kb) and torch.equal(va, vb) and ka.isfinite().all() and va.isfinite().all() and float(va.abs().max()) > 1e38


# ---- engine ---------------------------------------------------------------------------------------------------------------
def _dense4(model, tokens):
    """Logits of the dense model in its own type whose keys and values stand for what the cache holds of them, experts one by one."""
    from kafka_llm_service_amd.models import oracle as orc
    from kafka_llm_service_amd.models.moe import route

    cfg, D, hq, hkv = model.cfg, model.D, model.hq, model.hkv
    t = torch.tensor(tokens, device=model.device)
    T = t.shape[0]
    cs = model.cos_sin[:T].float()
    h = model.embed[t]
    see = torch.ones(T, T, dtype=torch.bool, device=h.device).tril()
    four = lambda x: kref.values(*kref.quant(x))
    glu = lambda x, w13, w2: orc._lin((torch.nn.functional.silu((gu := orc._lin(x, w13).float())[:, :gu.shape[1] // 2]) * gu[:, gu.shape[1] // 2:]).to(x.dtype), w2)
    for lw in model.layers:
        qkv = orc._lin(orc._rms(h, lw.input_norm, cfg.rms_norm_eps), lw.qkv).view(T, hq + 2 * hkv, D)
        q, k, v = orc._rope(qkv[:, :hq], cs).float(), four(orc._rope(qkv[:, hq:hq + hkv], cs)), four(qkv[:, hq + hkv:])
        o = torch.empty(T, hq, D, device=h.device)
        for x in range(hq):
            s = (q[:, x] @ k[:, x * hkv // hq].T.contiguous() * model.scale).masked_fill(~see, -math.inf)
            o[:, x] = torch.softmax(s, -1) @ v[:, x * hkv // hq].contiguous()
        h = (h.float() + orc._lin(o.view(T, -1).to(h.dtype), lw.o).float()).to(h.dtype)
        x = orc._rms(h, lw.post_norm, cfg.rms_norm_eps)
        if lw.router is None:
            delta = glu(x, lw.gate_up, lw.down).float()
        else:
            w, e = route(orc._lin(x, lw.router), cfg.num_experts_per_tok)
            delta = torch.zeros(T, x.shape[1], device=h.device)
            for j in range(cfg.num_experts):
                rows = (e == j).any(-1).nonzero().flatten()
                if rows.numel():
                    delta[rows] += glu(x[rows], lw.w13[j], lw.w2[j]).float() * (w * (e == j))[rows].sum(-1, keepdim=True)
        h = (h.float() + delta.to(h.dtype).float()).to(h.dtype)
    return orc._lin(orc._rms(h, model.final_norm, cfg.rms_norm_eps), model.lm_head).float()[:, :cfg.vocab_size]


def _served(model, device, gap, **kw):
    """Threads that decode while long new prompts come in: every greedy token within ``gap`` of the dense form's best."""
    from kafka_llm_service_amd.engine.engine import EngineConfig, LLMEngine
    from kafka_llm_service_amd.engine.sequence import SamplingParams

    if torch.device(device).type == "cuda":                   # (rows that nobody writes are no numbers)
        junk = [torch.full((1 << 26,), math.nan, device=device) for _ in range(4)]
        del junk
    eng = LLMEngine(EngineConfig(model=model, device=device, num_kv_blocks=1024, max_model_len=4096, kv_dtype="mx4", **kw))
    g = torch.Generator().manual_seed(13)
    draw = lambda n: torch.randint(0, 5000, (n,), generator=g).tolist()
    sp = SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True)
    prompts = [draw(n) for n in (40, 9, 77, 130, 150, 181)]
    seqs = [eng.add_request(f"a{i}", p, sp) for i, p in enumerate(prompts[:3])]
    rows = set()
    for i, p in enumerate(prompts[3:]):
        for _ in range(2):
            eng.step()
            rows |= {(st["T"], st["B"]) for st in eng.runner.recent_stats}
        seqs.append(eng.add_request(f"b{i}", p, sp))
    while any(not s.finished for s in seqs):
        eng.step()
        rows |= {(st["T"], st["B"]) for st in eng.runner.recent_stats}
    for p, s in zip(prompts, seqs):
        lg = _dense4(eng.model, p + s.output_ids).cpu()
        assert len(s.output_ids) == 8
        for i, tok in enumerate(s.output_ids):
            row = lg[len(p) - 1 + i]
            assert (row.max() - row[tok]).item() < gap, f"token {i}: gap {(row.max() - row[tok]).item():.3f}"
    return rows


def test_engine_with_experts_cpu():
    _served("tiny-mixtral", "cpu", 0.15)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["auto", "blas"])
@pytest.mark.parametrize("model", ["tiny-mixtral", "small-llama"])
def test_engine_with_new_turns_on_the_gpu(cuda, model, mode):
    rows = _served(model, str(cuda), 0.25, decode_gemm=mode)
    if mode == "blas":                                        # (steps of 129 to 256 rows are padded to 16 k + 8)
        assert any(B > 0 and T in (168, 184, 200) for T, B in rows), rows


def test_engine_refusals():
    """What the cache cannot hold or attend to is refused when the engine is made, not by its first step."""
    from dataclasses import replace

    from kafka_llm_service_amd.engine.engine import EngineConfig, LLMEngine
    from kafka_llm_service_amd.models.config import get_config

    make = lambda mc, kv: LLMEngine(EngineConfig(device="cpu", num_kv_blocks=64, max_model_len=256, kv_dtype=kv), model_cfg=mc)
    tiny = replace(get_config("tiny-llama"), vocab_size=512)
    for mc in (replace(tiny, num_heads=17, num_kv_heads=1), replace(tiny, head_dim=32), get_config("budurax-tiny")):
        with pytest.raises(ValueError, match="4.bit|mx4"):
            make(mc, "mx4")
        make(mc, "bf16")
    make(replace(tiny, num_heads=16, num_kv_heads=1), "mx4")


def test_step_of_the_cache_as_its_followers_get_it():
    """A step's tables, planned on the host, come whole out of what a leader sends its followers."""
    from kafka_llm_service_amd.engine import model_runner as mr
    from kafka_llm_service_amd.engine.engine import EngineConfig, LLMEngine
    from kafka_llm_service_amd.engine.sequence import SamplingParams

    eng = LLMEngine(EngineConfig(model="tiny-llama", device="cpu", num_kv_blocks=256, max_model_len=2048, kv_dtype="mx4"))
    g = torch.Generator().manual_seed(1)
    draw = lambda n: torch.randint(0, 5000, (n,), generator=g).tolist()
    eng.add_request("a", draw(100), SamplingParams(temperature=0.0, max_tokens=9, ignore_eos=True))
    eng.step()
    eng.step()
    eng.add_request("b", draw(200), SamplingParams(temperature=0.0, max_tokens=9, ignore_eos=True))
    steps, build = [], type(eng.runner).build_host

    def both(batch, want=None):
        eng.runner.mx4 = True
        steps.append((build(eng.runner, batch, want)[0], [s.total_len for s in batch.decode], [(a, b) for _, a, b in batch.prefill]))
        eng.runner.mx4 = False
        return build(eng.runner, batch, want)

    eng.runner.build_host = both
    for _ in range(3):
        eng.step()
    assert any(d and p for _, d, p in steps)
    z = np.zeros(0, np.float32)
    for h, dec, pre in steps:
        segs = [(i, 1, n - 1, i) for i, n in enumerate(dec)]
        r = len(dec)
        for j, (a, b) in enumerate(pre):
            segs.append((r, b - a, a, len(dec) + j))
            r += b - a
        model = eng.model
        want = kv4.step_tables(segs, model.hq, model.hkv, model.D)
        o = h.nbt * h.bt_w + h.T
        assert h.bt_need <= h.bt_w and h.bt_w * 16 >= want[2]
        got, _ = mr.unpack_plan(*mr.pack_plan(h, mr.SampleParams(z, z, z.astype(np.int32), z.astype(np.int64), None, True)))
        for x in (h, got):
            assert np.array_equal(x.i32[o:], want) and np.array_equal(x.i32, h.i32) and np.array_equal(x.i64, h.i64)
            assert (x.B, x.T, x.nbt, x.bt_w, x.n_rows) == (h.B, h.T, h.nbt, h.bt_w, h.n_rows)


@pytest.mark.timeout(300)
def test_two_ranks_on_the_cache():
    """Tensor parallel on the 4-bit cache: both ranks' heads together give the dense form's tokens."""
    import torch.multiprocessing as mp

    import test_tp_equivalence as tp
    from kafka_llm_service_amd.engine.engine import EngineConfig, LLMEngine

    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), tp._port()
    procs = [ctx.Process(target=tp._group_main, args=(r, 2, port, q, {"kv_dtype": "mx4"})) for r in range(2)]
    for p in procs:
        p.start()
    res = dict((m[0], m[1:]) for m in (q.get(timeout=240) for _ in range(2)))
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    model = LLMEngine(EngineConfig(**dict(tp.CFG, kv_dtype="mx4"))).model
    for p, o in zip(tp._prompts(), res["outs"][0]):
        lg = _dense4(model, p + o)
        for i, tok in enumerate(o):
            row = lg[len(p) - 1 + i]
            assert (row.max() - row[tok]).item() < 0.15
