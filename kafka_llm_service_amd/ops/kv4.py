"""Operators of the 4-bit KV cache (``kv_cache_shapes(..., "mx4")``): elements e2m1, one power of two for every 32 elements of a key's or
value's head vector, 4.25 bits each in all, a little over a quarter of the bf16 cache; head dims 64 and 128, pages of 16 keys (csrc/kv4.h).

  ops.rope_kv_write   writes a step's rows (a cache of this kind given)            csrc/kv4.hip
  read                keys and values of slots as numbers                          csrc/kv4.hip
  attn_plan / attn    attention of single tokens and prompt portions over pages,   csrc/kv4_attn.hip
                      causal, or a window and the first tokens
  attn_mass           the weight that every cached key has received                csrc/kv4_attn.hip
  evict_keep / evict  the keys that stay, by their weight; their move to new pages csrc/kv4.hip

Rows of a call are described by segments (first row, rows, position of the first, row of the block table): consecutive tokens of
one sequence, whose keys lie in the cache at their positions. GPU tensors run the HIP kernels on the caches' device and its current
stream, CPU tensors the references of ``kv4_reference.py``. Workspaces are made per call, so calls on several streams and captured
graphs do not meet. A plan holds the tables that the kernels read and, for each stream that it is used on, counters that every
call leaves at zero (a captured call has its own, in its graph); like a call's tensors it has to live until the stream, or the graph, is
done with it.
"""
from __future__ import annotations

import numpy as np
import torch

from . import kv4_reference as ref
from ._ext import ext

PAGE = ref.PAGE
BLOCK = 64                 # keys that a wave takes at a time
MAX_POS = 1 << 26
MAX_GROUP = 16             # query heads for a key/value head


def _gpu(t: torch.Tensor) -> bool:
    return t.is_cuda


def _check_cache(k_cache, v_cache, who: str) -> None:
    for c in (k_cache, v_cache):
        if c.dtype != torch.uint8 or c.dim() != 4 or c.shape[0] == 0 or c.shape[2] != PAGE or c.shape[3] not in (34, 68) or c.shape != k_cache.shape:
            raise ValueError(f"{who}: caches of kv_cache_shapes(..., \"mx4\") with head dim 64 or 128 expected")


def read(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(K, V) [T, heads, D] bf16 of ``slots`` int64 [T] (page * 16 + key), exactly what the cache holds. Negative slots give zeros,
    slots behind the cache no numbers."""
    if _gpu(k_cache):
        return ext().kv4_read(k_cache, v_cache, slots)
    _check_cache(k_cache, v_cache, "kv4.read")
    if slots.dim() != 1 or slots.dtype != torch.int64:
        raise ValueError("kv4.read: slots int64 [T]")
    return ref.read(k_cache, v_cache, slots)


def _check_apart(out, other, who: str) -> None:
    """``out`` is ``other``, or they have no byte in common (as far as contiguous tensors tell)."""
    a, b = ((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (out, other))
    if out.is_contiguous() and other.is_contiguous() and a != b and a[0] < b[1] and b[0] < a[1]:
        raise ValueError(f"{who} overlap in part")


# ---- plans --------------------------------------------------------------------------------------------------------------
FEW_ROWS = 16              # rows (tokens x query heads of a group) of a tile for single tokens
SOME_ROWS = 32             # of a tile for short portions
MANY_ROWS = {128: 256, 64: 128}   # of a tile for portions whose keys are widened first, by head dim (csrc/kv4_tile.hip)
MANY_WGS = {128: 256, 64: 768}    # workgroups of these that the CUs hold
MANY_MIN = 128             # rows of a segment from which on its keys may be widened first (_wide)
MANY_BLOCKS = 4            # least blocks of a piece of a wide tile (300 rows behind 1000 keys 25 us; of 8 blocks 30, of 16 40)
CUS = 256
MANY_BYTES = 8 << 30       # most that the keys widened for a call may take (2 million keys of 8 heads of 128); what is beyond goes in tiles of 32 rows
LEAST_SHARE = 2            # blocks a CU up to which every four of them are a workgroup, one for each wave
SHORT_TILE = 48            # blocks of a tile on average below which four waves take it, where there is more than a tile a CU (_narrow_split)
SOME_WGS, SOME_PIECE = 256, 8     # workgroups that a launch of short portions is split towards, least blocks of a piece
MANY_COST = 14.            # what two more launches and a workspace cost (_wide)
MASS_FEW = 16              # rows of a segment up to which a wave takes them all for its block of keys
MASS_WGS = 1024            # workgroups that a launch of few rows is split towards (64 threads of 2000 23.5 us, 256 28, 4096 37)
MASS_MANY_WGS = 2048       # ... of portions (twice as many as the CUs hold: parts of rows are unequal; 1900 rows 45 us, with 1024 49, 512 62)
MASS_TILES = 8             # least tiles of 16 rows of a part (200 rows behind 1000 keys 12.2 us, of 16 tiles 16.9; 1900 rows 50.5 and 48.8)


class AttnPlan:
    """Work of ``attn`` and ``attn_mass`` for a step's segments (``attn_plan``); every layer of the step uses the same."""

    def __init__(self):
        self.segs: list[tuple[int, int, int, int]] = []
        self.heads = self.kv_heads = self.dim = self.window = self.first = 0
        self.rows = self.covered = self.keys = self.tables = 0
        self.native = None          # what the kernels' callers read (csrc/kv4_bindings.cpp Plan), on a GPU


def _blocks(pos, tokens, window: int, first: int):
    """(blocks below the window, blocks in all) that tiles of ``tokens`` rows from ``pos`` on see: csrc/kv4_attn.hip Blocks."""
    tail = np.maximum(0, pos - window + 1) // BLOCK if window else np.zeros_like(pos)
    head = np.minimum((first + BLOCK - 1) // BLOCK, tail)
    return head, head + (pos + tokens - 1) // BLOCK + 1 - tail


def _tiles(segs: np.ndarray, tokens: int):
    """Tiles of at most ``tokens`` rows: int64 [n, 5] (first row, rows, position, table row, segment)."""
    n = (segs[:, 1] + tokens - 1) // tokens
    s = np.repeat(np.arange(len(segs)), n)
    i = (np.arange(len(s)) - np.repeat(np.cumsum(n) - n, n)) * tokens
    return np.stack([segs[s, 0] + i, np.minimum(segs[s, 1] - i, tokens), segs[s, 2] + i, segs[s, 3], s], 1)


def _pieces(tiles: np.ndarray, count: np.ndarray, n: np.ndarray):
    """(tile, first block, last + 1, first slot of the tile's partial results, number among them, how many) int64 [n, 6], merges int64 [m, 4],
    slots: tiles of ``count`` blocks in ``n`` pieces each (or fewer), the longest first. The slot of a tile in one piece is -1."""
    each = (count + n - 1) // n
    n = np.maximum(1, (count + each - 1) // each)
    t = np.repeat(np.arange(len(tiles)), n)
    at = np.cumsum(n) - n
    i = np.arange(len(t)) - at[t]
    split = n > 1
    base = np.cumsum(np.where(split, n, 0)) - np.where(split, n, 0)
    lo = i * each[t]
    pieces = np.stack([t, lo, np.minimum(lo + each[t], count[t]), np.where(split[t], base[t], -1), i, n[t]], 1)
    merges = np.stack([tiles[split, 0], tiles[split, 1], base[split], n[split]], 1)
    return pieces[np.argsort(pieces[:, 1] - pieces[:, 2], kind="stable")], merges, int(n[split].sum())


def _narrow_split(count: np.ndarray, kv_heads: int, rows: int) -> tuple[int, np.ndarray]:
    """(waves of a workgroup, pieces of every tile) for tiles of ``rows`` rows that see ``count`` blocks."""
    total = int(count.sum()) * kv_heads
    share = -(-total // CUS)
    if rows == FEW_ROWS and share > LEAST_SHARE:
        # 48 / 64 / 100 threads of 500 keys on four waves 10.4 / 11.4 / 18.1 us, on eight 13.8 / 15.7 / 27.5; of 3000 keys 32 / 39 / 62 and
        # 33 / 38 / 70; 20 / 32 threads (a tile a CU or less) of 2000 keys 17 / 20 and 15 / 19 (32/8 heads of 128, 64/8 heads alike)
        waves = 4 if len(count) * kv_heads > CUS and int(count.sum()) < SHORT_TILE * len(count) else 8
        return waves, np.maximum(1, count // max(8, share))
    if rows == FEW_ROWS:   # (one thread of 1500 keys 7.5 us, by its share on eight waves 9.2; of 8000 11.4 and 10.5)
        return 4, np.maximum(1, (count + 3) // 4)
    # 90 sizes of 1 to 16 portions of 33 to 512 tokens behind 0 to 8000: 3% off the best split of each on average, in pieces of at least 4
    # blocks and for 512 workgroups 7%, at most 47% (the last piece's join costs as much as 4 blocks)
    return 4, np.maximum(1, count // max(SOME_PIECE, -(-total // SOME_WGS)))


def _wide(full: np.ndarray, heads: int, kv_heads: int, dim: int, window: int, first: int) -> np.ndarray:
    """Which segments are taken in wide tiles whose keys are widened first: none or all of MANY_MIN rows or more (in their order as many as
    MANY_BYTES hold), by the microseconds that both ways take. Measured (32/8 heads of 128 / 64/8 heads of 128 / 24/8 heads of 64): 512 rows cold 21 against 14 with tiles of 32 rows / 25
    against 25 / 17 against 10, 300 rows behind 1000 keys 24 against 23 / 31 against 33 / 18 against 14, 8 portions of 200 cold 20 against
    35 / - / -, three of 1100 behind 900 in a window of 512 75 against 99 / - / 38 against 61."""
    G = heads // kv_heads
    wide = full[:, 1] * G >= MANY_MIN
    part = full[wide]
    if len(part):
        def work(rows):
            t = _tiles(part, rows // G)
            return len(t) * kv_heads, int(_blocks(t[:, 2], t[:, 1], window, first)[1].sum()) * kv_heads

        wgs, blocks = work(SOME_ROWS)
        few = 7. * max(1., wgs / 512) + blocks * (0.9 if dim == 128 else 0.8) / 512     # rounds of workgroups, and blocks
        wgs, blocks = work(MANY_ROWS[dim])
        keys = int(_blocks(part[:, 2], part[:, 1], window, first)[1].sum()) * BLOCK * kv_heads
        many = MANY_COST + blocks * (2.1 if dim == 128 else 0.8) / 256 + keys * dim * 5 / 4.5e6
        if few <= many:
            wide[:] = False
    size = np.where(wide, _blocks(full[:, 2], full[:, 1], window, first)[1] * kv_heads * 256 * dim, 0)
    return wide & (np.cumsum(size) <= MANY_BYTES)


def _wide_split(count: np.ndarray, kv_heads: int, wgs: int) -> np.ndarray:
    """Pieces of every wide tile: the nearest whole number to its share of the CUs' work."""
    size = max(MANY_BLOCKS, -(-int(count.sum()) * kv_heads // wgs))
    return np.maximum(1, (count + size // 2) // size)


def _tables(full: np.ndarray, heads: int, kv_heads: int, dim: int, window: int, first: int):
    """(shapes, arrays) of ``attn``: of each kind of tiles (rows of one, waves, slots, items, merges, tiles of keys) and its items, merges, tiles of
    keys."""
    G = heads // kv_heads
    rows = full[:, 1] * G
    wide = _wide(full, heads, kv_heads, dim, window, first)
    shapes, arrays = [], []
    for size, part in ((FEW_ROWS, full[(rows <= FEW_ROWS) & ~wide]), (SOME_ROWS, full[(rows > FEW_ROWS) & ~wide]), (MANY_ROWS[dim], full[wide])):
        if not len(part):
            continue
        tiles = _tiles(part, size // G)
        _, count = _blocks(tiles[:, 2], tiles[:, 1], window, first)
        if size > SOME_ROWS:  # a segment's blocks lie one after the other in the workspace, those below the window first
            waves = 0
            pieces, merges, slots = _pieces(tiles, count, _wide_split(count, kv_heads, MANY_WGS[dim]))
            t = tiles[pieces[:, 0]]
            head, count = _blocks(part[:, 2], part[:, 1], window, first)
            tail = head + (part[:, 2] + part[:, 1] - 1) // BLOCK + 1 - count
            base = np.cumsum(count) - count
            s = np.repeat(np.arange(len(part)), count)
            i = np.arange(len(s)) - base[s]
            keys = np.stack([part[s, 3], np.where(i < head[s], i, i - head[s] + tail[s]), (part[:, 2] + part[:, 1] - 1)[s], part[s, 2]], 1)
            s = t[:, 4]
            cols = [t[:, 0], t[:, 1], t[:, 2], base[s], head[s], tail[s], pieces[:, 1], pieces[:, 2],
                    np.where(pieces[:, 3] < 0, -1, pieces[:, 3] + pieces[:, 4])]
        else:
            waves, n = _narrow_split(count, kv_heads, size)
            pieces, merges, slots = _pieces(tiles, count, n)
            t = tiles[pieces[:, 0]]
            keys = np.zeros((0, 4))
            cols = [t[:, 0], t[:, 1], t[:, 2], t[:, 3], pieces[:, 1], pieces[:, 2], pieces[:, 3], pieces[:, 5] << 16 | pieces[:, 4]]
            merges = merges[:0]                                            # (the last piece to end joins them)
        items = np.stack(cols + [np.zeros_like(t[:, 0])] * ((12 if len(keys) else 8) - len(cols)), 1)
        shapes.append((size, waves, slots, len(items), len(merges), len(keys)))
        arrays += [x.astype(np.int32) for x in (items, merges, keys)]
    return shapes, arrays


def _mass_tables(a: np.ndarray, G: int, kv_heads: int, keys: int, window: int, first: int):
    """Items of ``attn_mass`` for single tokens, for portions, and their partial results: every block of 64 of the plan's ``keys`` of every
    segment once, or in parts of the rows that see it where the blocks by themselves are too few workgroups."""
    nb = (keys + BLOCK - 1) // BLOCK
    few = a[:, 1] * G <= MASS_FEW
    idx = np.nonzero(few)[0]
    step = min(32, max(4, -(-nb * len(idx) * kv_heads // MASS_WGS // 4) * 4))
    b = np.arange(0, nb, step)
    s, b = np.repeat(idx, len(b)), np.tile(b, len(idx))
    single = np.concatenate([a[s], np.stack([s, b, np.minimum(b + step, nb), np.zeros_like(s)], 1)], 1).astype(np.int32)
    if few.all():
        return single, np.zeros((0, 12), np.int32), 0
    idx = np.nonzero(~few)[0]
    nq = (nb + 3) // 4
    s, b = np.repeat(idx, nq), np.tile(4 * np.arange(nq), len(idx))
    # columns (row, query head) that may see one of four blocks: rows from its first key's position on, to the last whose window has its last
    lo = np.minimum(np.maximum(0, (b * BLOCK - a[s, 2]) * G) // 16 * 16, a[s, 1] * G)
    hi = a[s, 1] * G
    if window:
        end = np.clip((b * BLOCK + 4 * BLOCK - 1 + window - a[s, 2]) * G, 0, hi)
        hi = np.where(b * BLOCK < first, hi, end)
    tiles = np.maximum(0, hi - lo + 15) // 16
    size = max(MASS_TILES, -(-int(tiles.sum()) * kv_heads // MASS_MANY_WGS))
    n = np.maximum(1, (tiles + size // 2) // size)
    each = np.maximum(1, (tiles + n - 1) // n)
    n = np.maximum(1, (tiles + each - 1) // each)
    t = np.repeat(np.arange(len(s)), n)
    i = np.arange(len(t)) - np.repeat(np.cumsum(n) - n, n)
    split = np.where(n > 1, n, 0)
    slot = np.where(n > 1, np.cumsum(split) - split, -1)
    s, b, at = s[t], b[t], lo[t] + 16 * each[t] * i
    z = np.zeros_like(s)
    many = np.stack([a[s, 0], a[s, 1], a[s, 2], a[s, 3], s, b, at, np.minimum(at + 16 * each[t], hi[t]), slot[t], n[t] << 16 | i, z, z], 1)
    return single, many[np.argsort(many[:, 6] - many[:, 7], kind="stable")].astype(np.int32), int(split.sum())


class _Take:
    """Tables one behind the other in a flat int32 tensor."""

    def __init__(self, flat: torch.Tensor):
        self.flat, self.at = flat, 0

    def __call__(self, n: int, cols: int) -> torch.Tensor:
        self.at += n * cols
        return self.flat[self.at - n * cols:self.at].view(n, cols)


def _native(p: AttnPlan, take: _Take, shapes) -> None:
    p.native = ext().Kv4Plan(p.heads, p.kv_heads, p.dim, p.window, p.first, p.rows, p.covered, p.keys, p.tables)
    for rows, waves, slots, items, merges, keys in shapes:
        p.native.add(rows, waves, slots, take(items, 12 if keys else 8), take(merges, 4), take(keys, 4))


def check_heads(heads: int, kv_heads: int, dim: int) -> None:
    """Refuses heads that the cache's attention does not take."""
    if dim not in (64, 128) or kv_heads < 1 or heads % kv_heads or not 1 <= heads // kv_heads <= MAX_GROUP:
        raise ValueError(f"the 4-bit cache takes head dims of 64 and 128 and 1 to {MAX_GROUP} query heads for each key/value head, not {heads} / "
                         f"{kv_heads} heads of {dim}")


def _plan(segs, heads: int, kv_heads: int, dim: int, window: int, first: int) -> tuple[AttnPlan, np.ndarray]:
    check_heads(heads, kv_heads, dim)
    if window < 0 or first < 0 or window >= 1 << 30 or first >= MAX_POS:
        raise ValueError("kv4.attn_plan: window and first may not be negative (window 0: every earlier position)")
    if first and not window:
        raise ValueError("kv4.attn_plan: first tokens stay visible beside a window")
    p = AttnPlan()
    a = np.array(list(segs), dtype=np.int64)
    if a.size and (a.ndim != 2 or a.shape[1] != 4):
        raise ValueError("kv4.attn_plan: segments of (first row, rows, position, table row)")
    a = a.reshape(-1, 4)
    p.segs = [tuple(s) for s in a.tolist()]
    if (a < 0).any() or (a[:, 0] + a[:, 1] >= MAX_POS).any() or (a[:, 2] + a[:, 1] >= MAX_POS).any() or (a[:, 3] >= 1 << 30).any():
        raise ValueError("kv4.attn_plan: segments of (first row, rows, position, table row), none negative, positions below 2^26")
    full = a[a[:, 1] > 0]
    byrow = full[np.argsort(full[:, 0], kind="stable")]
    if (byrow[1:, 0] < byrow[:-1, 0] + byrow[:-1, 1]).any():
        raise ValueError("kv4.attn_plan: a row in two segments")
    p.heads, p.kv_heads, p.dim, p.window, p.first = heads, kv_heads, dim, int(window), int(first)
    if len(full):
        p.rows, p.covered = int((full[:, 0] + full[:, 1]).max()), int(full[:, 1].sum())
        p.keys, p.tables = int((full[:, 2] + full[:, 1]).max()), int(full[:, 3].max()) + 1
    return p, a


def attn_plan(segs, heads: int, kv_heads: int, dim: int, window: int = 0, first: int = 0, device="cuda") -> AttnPlan:
    """Plan for ``segs``, host integers (first row, rows, position of the first, row of the block table) each: the row at position p sees
    the keys j <= p, with ``window`` > 0 only those with j > p - window or j < ``first``. Rows of different segments are different."""
    p, a = _plan(segs, heads, kv_heads, dim, window, first)
    dev = torch.device(device)
    if dev.type != "cuda":
        return p
    shapes, arrays = _tables(a[a[:, 1] > 0], heads, kv_heads, dim, p.window, p.first)
    few, many, slots = _mass_tables(a, heads // kv_heads, kv_heads, p.keys, p.window, p.first)
    take = _Take(torch.from_numpy(np.concatenate([t.reshape(-1) for t in arrays + [few, many]])).to(dev))
    _native(p, take, shapes)
    p.native.weigh(take(len(few), 8), take(len(many), 12), slots, len(a))
    return p


STEP_PARTS, STEP_SHAPE = 3, 6   # kinds of tiles that a step may have; numbers that describe one


def step_tables(segs, heads: int, kv_heads: int, dim: int) -> np.ndarray:
    """The plan of an engine step as one int32 array, for its upload: what ``step_plan`` reads on the host, then the tables."""
    p, a = _plan(segs, heads, kv_heads, dim, 0, 0)
    shapes, arrays = _tables(a[a[:, 1] > 0], heads, kv_heads, dim, 0, 0)
    head = np.zeros(4 + STEP_SHAPE * STEP_PARTS, dtype=np.int32)
    head[:4] = p.rows, p.covered, p.keys, p.tables
    for i, s in enumerate(shapes):
        head[4 + STEP_SHAPE * i:4 + STEP_SHAPE * (i + 1)] = s
    return np.concatenate([head] + [t.reshape(-1) for t in arrays])


def step_plan(host: np.ndarray, device: torch.Tensor, heads: int, kv_heads: int, dim: int) -> AttnPlan:
    """The ``attn`` plan in ``step_tables``' array and its copy on the device (no segments are kept: ``attn_mass`` has a plan of its own)."""
    p = AttnPlan()
    p.heads, p.kv_heads, p.dim = heads, kv_heads, dim
    p.rows, p.covered, p.keys, p.tables = (int(x) for x in host[:4])
    n = 4 + STEP_SHAPE * STEP_PARTS
    _native(p, _Take(device[n:]), [shape for shape in host[4:n].reshape(-1, STEP_SHAPE).tolist() if shape[0]])
    return p


def _check_call(q, k_cache, block_tables, plan: AttnPlan, scale: float, who: str) -> None:
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"{who}: a positive scale expected")
    if q.dim() != 3 or q.dtype != torch.bfloat16 or q.shape[1] != plan.heads or q.shape[2] != plan.dim or \
            k_cache.shape[1] != plan.kv_heads or ref.head_dim(k_cache) != plan.dim:
        raise ValueError(f"{who}: q bf16 [T, heads, dim] and a cache of the plan's heads expected")
    if q.shape[0] < plan.rows:
        raise ValueError(f"{who}: the plan has {plan.rows} rows, q {q.shape[0]}")
    if block_tables.dim() != 2 or block_tables.dtype != torch.int32 or block_tables.shape[0] < plan.tables or \
            block_tables.shape[1] * PAGE < plan.keys:
        raise ValueError(f"{who}: int32 block tables of {plan.tables} rows for {plan.keys} keys expected")


def attn(q, k_cache, v_cache, block_tables, plan: AttnPlan, scale: float, out=None, lse=None) -> torch.Tensor:
    """softmax(scale q k^T) v of the plan's rows: q [T, heads, dim] bf16 -> out (a new tensor unless given; q itself may be), the same shape.
    ``lse`` fp32 [T, heads] gets the base-2 logarithm of each row's sum of 2^(scores in base 2). Rows of no segment are left as they
    were (zeros in a new ``out``). Sums are formed before they are divided: with n keys values below 2^104 / n (2^78 for any n) are right, larger
    ones, as infinities are stored, may come out as infinities or no numbers in the rows that see them. Of a page that no row of the segment sees a key of (behind the last one, or between the first ones
    and the window) the table may name anything; where it names none of the cache's for one that is seen, the rows that see it come out
    as no numbers, and rows of the segment next to them may."""
    if _gpu(q):
        if plan.native is None:
            raise ValueError("kv4.attn: the plan was made for another device")
        return ext().kv4_attn(q, k_cache, v_cache, block_tables, plan.native, scale, out, lse)
    _check_cache(k_cache, v_cache, "kv4.attn")
    _check_call(q, k_cache, block_tables, plan, scale, "kv4.attn")
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("kv4.attn: out like q expected")
    else:
        _check_apart(out, q, "kv4.attn: out and q")
    if lse is not None and (lse.shape != q.shape[:2] or lse.dtype != torch.float32):
        raise ValueError("kv4.attn: lse fp32 [T, heads] expected")
    ref.attn(q, k_cache, v_cache, block_tables, plan.segs, plan.window, plan.first, float(scale), out, lse)
    return out


def attn_mass(q, lse, k_cache, block_tables, plan: AttnPlan, scale: float, base=None, out=None) -> torch.Tensor:
    """Weight of every key: out[s, h, j] = base[s, h, j] + the sum over segment s's rows and the query heads of h of
    2^(score - lse), fp32 [segments, kv heads, keys], with ``lse`` from ``attn`` over the same rows. ``out`` may be ``base``: weights that
    accumulate from step to step. Without either, a new tensor as wide as the plan's longest sequence. A key's sum is always formed in
    the same order."""
    if _gpu(q):
        if plan.native is None:
            raise ValueError("kv4.attn_mass: the plan was made for another device")
        return ext().kv4_mass(q, lse, k_cache, block_tables, plan.native, scale, base, out)
    _check_cache(k_cache, k_cache, "kv4.attn_mass")
    _check_call(q, k_cache, block_tables, plan, scale, "kv4.attn_mass")
    if lse.shape != q.shape[:2] or lse.dtype != torch.float32:
        raise ValueError("kv4.attn_mass: lse fp32 [T, heads] expected")
    like = base if base is not None else out
    shape = (len(plan.segs), plan.kv_heads, like.shape[2] if like is not None and like.dim() == 3 else plan.keys)
    for t in (base, out):
        if t is not None and (t.shape != shape or t.dtype != torch.float32 or not t.is_contiguous() or t.shape[2] < plan.keys):
            raise ValueError(f"kv4.attn_mass: base and out contiguous fp32 [segments, kv heads, at least {plan.keys}], alike, expected")
    if base is not None and out is not None:
        _check_apart(out, base, "kv4.attn_mass: base and out")
    if out is None:
        out = torch.empty(shape, dtype=torch.float32)
    if base is None:
        out.zero_()
    elif base is not out:
        out.copy_(base)
    ref.attn_mass(q, lse, k_cache, block_tables, plan.segs, plan.window, plan.first, float(scale), out)
    return out


# ---- eviction -----------------------------------------------------------------------------------------------------------
def evict_keep(mass: torch.Tensor, lens: torch.Tensor, budget: int, first: int = 0, recent: int = 0) -> torch.Tensor:
    """The keys that stay, int32 [sequences, kv heads, budget], ascending, per head: of a sequence of ``lens`` keys the ``first`` ones,
    the ``recent`` last ones, and of the rest those of the largest ``mass`` [sequences, kv heads, keys] fp32 (equal masses: the
    lowest index; not a number: after all others). Sequences within the budget keep everything, -1 behind their last."""
    if _gpu(mass):
        return ext().kv4_evict_keep(mass, lens, budget, first, recent)
    if mass.dim() != 3 or mass.dtype != torch.float32 or lens.shape != (mass.shape[0],) or lens.dtype != torch.int32 or \
            lens.device != mass.device:
        raise ValueError("kv4.evict_keep: mass fp32 [sequences, kv heads, keys] and lens int32 [sequences] on its device expected")
    if budget < 1 or first < 0 or recent < 0 or first + recent > budget or budget >= MAX_POS:
        raise ValueError("kv4.evict_keep: first and recent keys within a budget of at least one")
    return ref.evict_keep(mass, lens, int(budget), int(first), int(recent))


def evict(k_cache, v_cache, block_tables, kept, new_tables, mass=None):
    """Copies the ``kept`` keys and values (``evict_keep``) of every sequence and head from the pages of ``block_tables`` to those of
    ``new_tables``, int32 [sequences, pages] both, in order: key i of a head becomes kept[.., i]. The new pages are none of the old ones
    (which other sequences may share, and which their owner may free afterwards), and each is one sequence's alone; places behind a
    sequence's last key are left as they were, as are keys whose index, or whose page, is outside. Returns the kept keys' ``mass`` [sequences, kv heads, budget]
    (zero behind the last) if it is given, else None."""
    if _gpu(k_cache):
        return ext().kv4_evict_copy(k_cache, v_cache, block_tables, kept, new_tables, mass)
    _check_cache(k_cache, v_cache, "kv4.evict")
    if kept.dim() != 3 or kept.dtype != torch.int32 or kept.shape[1] != k_cache.shape[1]:
        raise ValueError("kv4.evict: kept int32 [sequences, kv heads, budget] expected")
    for t in (block_tables, new_tables):
        if t.dim() != 2 or t.dtype != torch.int32 or t.shape[0] != kept.shape[0]:
            raise ValueError("kv4.evict: int32 tables [sequences, pages] expected")
    if mass is not None and (mass.dim() != 3 or mass.shape[:2] != kept.shape[:2] or mass.dtype != torch.float32):
        raise ValueError("kv4.evict: mass fp32 [sequences, kv heads, keys] expected")
    new_mass = torch.empty(kept.shape, dtype=torch.float32) if mass is not None else None
    ref.evict_copy(k_cache, v_cache, block_tables, kept, new_tables, mass, new_mass)
    return new_mass
