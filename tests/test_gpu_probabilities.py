"""How exactly the steps on tensor cores weigh value rows: in bf16 and in 8 bits a probability is two 16-bit numbers, whose sum is off by no more than the
products of their rounding."""
import math

import pytest
import torch

import dwarf_b200
from tests.serving_util import HALF, attention64
from tests.test_gpu_paged import held_as, make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def paged_bound(qs, r, sc, o, spread, ds, p_half):
    """What a step may be off: the scores' error, p_half of every term, the fp32 sums over n positions (and 64 more roundings), and its own rounding to bf16."""
    more = (2 * ds[:, None] + p_half + (r.shape[0] + 64) * 2.0 ** -24) * spread
    return HALF[BF] * o.abs() + more * (1 + HALF[BF])


@pytest.mark.parametrize("H,G,D,page", [(2, 1, 32, 16), (1, 4, 128, 64), (2, 3, 96, 48), (1, 12, 64, 32), (1, 17, 128, 16), (2, 8, 80, 32), (1, 2, 48, 16)])
def test_bf16_pages(H, G, D, page):
    """bf16 keeps 2^-8 of a number and 2^-8 of what is left of it: 2^-16.  Scores near one another, so that their own error is far below, and values that
    cancel, so that the result's rounding is too."""
    g = torch.Generator().manual_seed(D + G)
    lengths, sc = [1, 2, 20, 45, 300, 1000], 0.02
    S = len(lengths)
    kv, _, table, rows = make_cache(lengths, H, page, D, BF, g)
    q = torch.randn(S, H * G, D, generator=g).to(BF)
    out = dwarf_b200.paged_attention_step(q.to(DEV), None, None, kv, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=sc).double().cpu()
    for s in range(S):
        for h in range(H):
            qs, r = q[s, h * G:(h + 1) * G].double(), rows[s][:, h]
            o, spread, ds = attention64(qs, r[:, 0], r[:, 1], sc)
            off, bound = (out[s, h * G:(h + 1) * G] - o).abs(), paged_bound(qs, r, sc, o, spread, ds, 2.0 ** -16)
            assert (off <= bound).all(), (lengths[s], h, (off / bound).max())
