"""The 4-bit cache's kernels form by form: pages that are none in every kind of tile."""
import pytest
import torch

from kafka_llm_service_amd.ops import kv4
from test_kv4 import queries, world


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
