"""How a paged step is cut into parts follows from the sizes and types; what comes out does not."""
import math
import random

import pytest
import torch

import dwarf_b200
from tests.serving_util import HALF, attention64
from tests.test_gpu_paged import make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.mark.parametrize("seed", range(40))
def test_any_room(seed):
    """Tables with room for 1 to 1,000,000 positions over the same sequences: scratch is enough for every plan, and parts of any length give the result."""
    r = random.Random(seed)
    dtype, q_dt = r.choice([(BF, BF), (E4, BF), (BF, BF), (E4, BF), (F, F), (E4, F), (BF, F)])
    S, H, G, D, page = r.choice([1, 2, 5, 15, 16, 17]), r.choice([1, 2, 3]), r.choice([1, 2, 4, 8, 9, 17]), r.choice([32, 48, 64, 80, 96, 128, 40]), r.choice([16, 48, 64, 24])
    lengths = [r.choice([0, 1, 63, 64, 65, 128, 129, r.randint(1, 300)]) for _ in range(S)]
    g = torch.Generator().manual_seed(seed)
    kv, ks, table, rows = make_cache(lengths, H, page, D, dtype, g)
    q = torch.randn(S, H * G, D, generator=g).to(q_dt)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    sc = 0.3 / math.sqrt(D)
    for room in (1, 400, 3000, 30000, 200000, 1000000):
        wide = torch.nn.functional.pad(table, (0, max(0, -(-room // page) - table.shape[1])), value=-1)
        out = dwarf_b200.paged_attention_step(q.to(DEV), None, None, kv, wide, n, kv_scale=ks, scale=sc).double().cpu()
        for s in range(S):
            for h in range(H):
                qs, x = q[s, h * G:(h + 1) * G].double(), rows[s][:, h]
                o, spread, ds = attention64(qs, x[:, 0], x[:, 1], sc)
                # operands in two 16-bit numbers: 2^-16, and what f16 leaves of the smallest
                more = (2 * ds[:, None] + 2.0 ** -15 + (len(x) + 64) * 2.0 ** -24) * spread
                assert ((out[s, h * G:(h + 1) * G] - o).abs() <= HALF[q_dt] * o.abs() + 1.01 * more).all(), (room, s, h)


def test_advance_does_not_wait_for_the_gpu():
    """A token within the pages at hand, with and without an empty slot of the batch: nothing is copied from the host."""
    for counts in ([5, 0, 40], [5, 1, 40]):
        c = dwarf_b200.PagedKVCache(1, 3, 1, 32, max_length=200, page_size=64, device=DEV)
        c.extend(counts)
        torch.cuda.set_sync_debug_mode("error")
        try:
            for _ in range(10):
                c.advance()
        finally:
            torch.cuda.set_sync_debug_mode("default")
        assert c.lengths.tolist() == [n + 10 if n else 0 for n in counts] == c._length


def test_scales_at_the_ends_of_fp32():
    """A scale that fp32 rounds to 0 is refused and not taken for the default; the smallest that it holds weighs all positions alike."""
    g = torch.Generator().manual_seed(0)
    for dtype, q_dt in ((BF, BF), (E4, BF), (F, F)):
        kv, ks, table, rows = make_cache([40], 1, 16, 64, dtype, g)
        q, n = torch.randn(1, 1, 64, generator=g).to(q_dt).to(DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
        for bad in (1e-60, 1e-46, 3.5e38):
            with pytest.raises(ValueError):
                dwarf_b200.paged_attention_step(q, None, None, kv, table, n, kv_scale=ks, scale=bad)
        for small in (1e-30, 1e-44):
            out = dwarf_b200.paged_attention_step(1e-3 * q, None, None, kv, table, n, kv_scale=ks, scale=small).double().cpu()
            v = rows[0][:, 0, 1]
            assert ((out[0, 0] - v.mean(0)).abs() <= HALF[q_dt] * v.mean(0).abs() + 1.01 * (2.0 ** -15 + 104 * 2.0 ** -24) * v.abs().mean(0)).all()
