"""One new token against the longest sequences that a table may name: 2^31 - 256 positions, most of them the same page."""
import math

import pytest
import torch

import dwarf_b200
from tests.serving_util import HALF, attention64, quantize64
from tests.test_gpu_paged import held_as

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, E4 = torch.bfloat16, torch.float8_e4m3fn
PAGE, COLUMNS = 12032, 178481                                     # their product is 2^31 - 256


# The form on tensor cores, and the one on CUDA cores at its narrowest row.
@pytest.mark.parametrize("D", [32, 8])
@pytest.mark.parametrize("back", [0, 5000])
def test_last_positions_of_the_longest_table(D, back):
    """Keys of the page that all columns but the last name score 200 below those of the last: what comes out is attention to the last page."""
    assert PAGE * COLUMNS == 2 ** 31 - 256
    g = torch.Generator().manual_seed(D)
    q = torch.randn(1, 1, D, generator=g).to(BF)
    rows = torch.randn(2, PAGE, 2, D, generator=g) * 0.5
    away = q[0, 0].float() * 100 * math.sqrt(D) / q[0, 0].float().square().sum()
    rows[0, :, 0], rows[1, :, 0] = -away, rows[1, :, 0] + away
    kn, vn = (rows[1, PAGE - 1 - back, i][None, None].to(BF) for i in (0, 1))
    rows[1, PAGE - 1 - back] = 0                                  # the new token's slot: written by the call
    v, s = quantize64(rows[:, None])
    kv, ks = v.float().to(E4).to(DEV), (torch.log2(s) + 127).to(torch.uint8).view(torch.float8_e8m0fnu).to(DEV)
    table = torch.zeros(1, COLUMNS, dtype=torch.int32, device=DEV)
    table[0, -1] = 1
    n = torch.tensor([PAGE * COLUMNS - back], dtype=torch.int32, device=DEV)
    out = dwarf_b200.paged_attention_step(q.to(DEV), kn.to(DEV), vn.to(DEV), kv, table, n, kv_scale=ks).double().cpu()
    rows[1, PAGE - 1 - back, 0], rows[1, PAGE - 1 - back, 1] = kn[0, 0].float(), vn[0, 0].float()
    r = held_as(rows[1, :PAGE - back], E4)
    assert torch.equal(kv[1, 0, PAGE - 1 - back].float().cpu().double() * torch.exp2(ks[1, 0, PAGE - 1 - back].view(torch.uint8).cpu().double() - 127)[:, None], r[-1])
    o, spread, ds = attention64(q[0].double(), r[:, 0], r[:, 1], 1 / math.sqrt(D))
    assert ((out[0] - o).abs() <= HALF[BF] * o.abs() + (2 * ds + 2.0 ** -11 + PAGE * 2.0 ** -24) * spread * 1.01).all()
