"""How exactly the steps on tensor cores weigh value rows: in bf16 and in 8 bits a probability is two 16-bit numbers, whose sum is off by no more than the
products of their rounding."""
import math

import pytest
import torch

import dwarf_b200
from tests.serving_util import HALF, attention64, quantize64
from tests.test_gpu_paged import held_as, make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def paged_bound(qs, r, sc, o, spread, ds, p_half):
    """What a step may be off: the scores' error, p_half of every term, the fp32 sums over n positions (and 64 more roundings), and its own rounding to bf16."""
    more = (2 * ds[:, None] + p_half + (r.shape[0] + 64) * 2.0 ** -24) * spread
    return HALF[BF] * o.abs() + more * (1 + HALF[BF])


@pytest.mark.parametrize("H,G,D,page", [(2, 1, 32, 16), (1, 4, 128, 64), (2, 3, 96, 48), (1, 12, 64, 32), (1, 17, 128, 16), (2, 8, 80, 32), (1, 2, 48, 16)])
@pytest.mark.parametrize("room", [0, 1 << 20], ids=["short_parts", "one_part"])
def test_bf16_pages(H, G, D, page, room):
    """bf16 cut off leaves up to 2^-7 of a number, and rounding that is off by 2^-8 of it: 2^-15.  Scores near one another, so that their own error is far below, and values that
    cancel, so that the result's rounding is too."""
    g = torch.Generator().manual_seed(D + G)
    lengths, sc = [1, 2, 20, 45, 300, 1000], 0.02
    S = len(lengths)
    kv, _, table, rows = make_cache(lengths, H, page, D, BF, g)
    table = torch.nn.functional.pad(table, (0, max(0, room // page - table.shape[1])), value=-1)
    q = torch.randn(S, H * G, D, generator=g).to(BF)
    out = dwarf_b200.paged_attention_step(q.to(DEV), None, None, kv, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=sc).double().cpu()
    for s in range(S):
        for h in range(H):
            qs, r = q[s, h * G:(h + 1) * G].double(), rows[s][:, h]
            o, spread, ds = attention64(qs, r[:, 0], r[:, 1], sc)
            off, bound = (out[s, h * G:(h + 1) * G] - o).abs(), paged_bound(qs, r, sc, o, spread, ds, 2.0 ** -15)
            assert (off <= bound).all(), (lengths[s], h, (off / bound).max())


@pytest.mark.parametrize("H,G,D,page", [(2, 1, 32, 16), (1, 4, 128, 64), (1, 12, 64, 32), (1, 2, 48, 16), (1, 2, 64, 10)])
@pytest.mark.parametrize("room", [0, 1 << 20], ids=["short_parts", "one_part"])
def test_an_infinity_in_a_value_row_is_one_in_the_result(H, G, D, page, room):
    """softmax v is infinite with the sign of v in the columns where one row is, whatever its probability is rounded to (1 and 1/2 leave nothing to round)."""
    g = torch.Generator().manual_seed(D)
    lengths = [1, 2, 40, 150]
    kv, _, table, rows = make_cache(lengths, H, page, D, BF, g)
    q = torch.randn(4, H * G, D, generator=g).to(BF)
    for s, n in enumerate(lengths):
        p, i = int(table[s, (n - 1) // page]), (n - 1) % page
        kv[p, :, i, 1, 3], kv[p, :, i, 1, 5] = float("inf"), -float("inf")
        if n == 2:
            kv[p, :, :2, 0] = 0                                   # both scores are 0
    table = torch.nn.functional.pad(table, (0, max(0, room // page - table.shape[1])), value=-1)
    out = dwarf_b200.paged_attention_step(q.to(DEV), None, None, kv, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=0.02)
    assert (out[:, :, 3] == float("inf")).all() and (out[:, :, 5] == -float("inf")).all()
    rest = [d for d in range(D) if d not in (3, 5)]
    assert torch.isfinite(out[:, :, rest]).all()


def cache8(rows, page):
    """Pages in 8 bits that hold rows [n,H,2,D] of every sequence: (kv, scale, table, the values they stand for)."""
    S, per = len(rows), [-(-r.shape[0] // page) for r in rows]
    _, H, _, D = rows[0].shape
    x = torch.zeros(sum(per), H, page, 2, D)
    table, at = torch.full((S, max(per)), -1, dtype=torch.int32), 0
    for s, r in enumerate(rows):
        for c in range(per[s]):
            part = r[c * page:(c + 1) * page]
            x[at, :, :part.shape[0]] = part.transpose(0, 1)
            table[s, c] = at
            at += 1
    v, sc = quantize64(x)
    byte = (torch.log2(sc) + 127).to(torch.uint8)
    return v.float().to(E4).to(DEV), byte.view(torch.float8_e8m0fnu).to(DEV), table.to(DEV), [held_as(r, E4) for r in rows]


def e4m3_bound(qs, r, sc, o, spread, ds, p):
    """As paged_bound: f16 keeps 2^-11 of a number and 2^-11 of what is left of it; exponents up to 64 are rounded three times (2^-18 each, times ln 2); below its
    normal range f16 is off by 2^-25, where the largest term of the result is at 2^9.5 (and values of a row are within 2 of its largest); queries are off by 2^-24 of
    their largest element, at keys that carry weight."""
    far = r.shape[0] * 2.0 ** -33.5 * (p * r[:, 1].abs().max(1).values).max(1).values[:, None]
    live = p.max(0).values > 1e-12
    dq = 2 * sc * 2.0 ** -24 * qs.abs().max() * r[live, 0].abs().sum(1).max()
    return paged_bound(qs, r, sc, o, spread, ds, 2.0 ** -22 + 3 * 2.0 ** -18 + dq) + 1.01 * far


def check8(rows, q, page, sc, room=0):
    """room: positions that the table has columns for, which decide how long a part is."""
    S, H = len(rows), rows[0].shape[1]
    G = q.shape[1] // H
    kv, ks, table, held = cache8(rows, page)
    table = torch.nn.functional.pad(table, (0, max(0, room // page - table.shape[1])), value=-1)
    n = torch.tensor([r.shape[0] for r in rows], dtype=torch.int32, device=DEV)
    out = dwarf_b200.paged_attention_step(q.to(DEV), None, None, kv, table, n, kv_scale=ks, scale=sc).double().cpu()
    for s in range(S):
        for h in range(H):
            qs, r = q[s, h * G:(h + 1) * G].double(), held[s][:, h]
            o, spread, ds = attention64(qs, r[:, 0], r[:, 1], sc)
            off, bound = (out[s, h * G:(h + 1) * G] - o).abs(), e4m3_bound(qs, r, sc, o, spread, ds, torch.softmax(sc * qs @ r[:, 0].T, 1))
            assert (off <= bound).all(), (s, h, (off / bound).max())


SHAPES = [(2, 1, 32, 16), (1, 4, 128, 64), (2, 3, 96, 48), (1, 12, 64, 32), (1, 17, 128, 16), (2, 8, 80, 32), (1, 2, 48, 16), (1, 9, 32, 10)]


@pytest.mark.parametrize("H,G,D,page", SHAPES)
@pytest.mark.parametrize("room", [0, 1 << 20], ids=["short_parts", "one_part"])
def test_e4m3_pages(H, G, D, page, room):
    g = torch.Generator().manual_seed(D + G)
    rows = [torch.randn(n, H, 2, D, generator=g) * torch.exp(0.7 * torch.randn(n, H, 2, 1, generator=g)) for n in (1, 2, 20, 45, 300)]
    check8(rows, torch.randn(len(rows), H * G, D, generator=g).to(BF), page, 0.02, room)


@pytest.mark.parametrize("H,G,D,page", SHAPES)
@pytest.mark.parametrize("room", [0, 1 << 20], ids=["short_parts", "one_part"])
@pytest.mark.parametrize("above", [12, 20, 26, 60])
def test_e4m3_value_rows_that_carry_no_weight_take_no_bits(H, G, D, page, above, room):
    """One value row 2^above the others, first, in the middle and last, whose key's score is 100 or more below: e^-100 2^60 of it is below 2^-84."""
    g = torch.Generator().manual_seed(D + G + above)
    n, sc = 150, 1 / math.sqrt(D)
    far = [0, 75, 149]
    q0 = torch.randn(1, H, 1, D, generator=g)
    q = (q0 + 0.05 * torch.randn(len(far), H, G, D, generator=g)).reshape(len(far), H * G, D).to(BF)
    rows = [0.3 * torch.randn(n, H, 2, D, generator=g) for _ in far]
    for r, at in zip(rows, far):
        r[at, :, 0] = -120 / sc * q0[0, :, 0] / q0[0, :, 0].square().sum(-1, keepdim=True)
        r[at, :, 1] = 2.0 ** above
    check8(rows, q, page, sc, room)


@pytest.mark.parametrize("H,G,D,page", SHAPES)
@pytest.mark.parametrize("room", [0, 1 << 20], ids=["short_parts", "one_part"])
def test_e4m3_value_rows_of_zeros_take_no_bits(H, G, D, page, room):
    """A row of zeros is held with a scale of 1, which says nothing of its size: values of 2^-30 beside it, first, last and in a tile of its own."""
    g = torch.Generator().manual_seed(D + G)
    rows = [torch.randn(150, H, 2, D, generator=g) * torch.tensor([1.0, 2.0 ** -30])[None, None, :, None] for _ in range(3)]
    rows[0][0, :, 1], rows[1][149, :, 1], rows[2][16:40, :, 1] = 0, 0, 0
    rows[2][16:40, :, 1, 0] = -0.0
    check8(rows, torch.randn(3, H * G, D, generator=g).to(BF), page, 0.02, room)


@pytest.mark.parametrize("H,G,D,page", SHAPES)
@pytest.mark.parametrize("room", [0, 1 << 20], ids=["short_parts", "one_part"])
def test_e4m3_growing_values_and_scores(H, G, D, page, room):
    """Scores and scales that grow along the sequence, and that shrink: both bases move at every tile, in parts of few tiles and in one part of all."""
    g = torch.Generator().manual_seed(5)
    n = 600
    q0 = torch.randn(1, H, 1, D, generator=g)
    q = (q0 + 0.02 * torch.randn(4, H, G, D, generator=g)).reshape(4, H * G, D).to(BF)
    rows = [torch.randn(n, H, 2, D, generator=g) for _ in range(4)]
    step = torch.arange(n)[:, None, None] / n
    for r, score, value in zip(rows, (40, 40, -40, 0), (60, -40, 60, 60)):
        r[:, :, 0] = 0.1 * r[:, :, 0] + score * step * math.sqrt(D) * q0[0, :, 0] / q0[0, :, 0].square().sum(-1, keepdim=True)
        r[:, :, 1] *= torch.exp2(value * step)
    check8(rows, q, page, 1 / math.sqrt(D), room)


# ---- rings
MANY, FEW = tuple(range(100)) + (128,), (0, 1, 2, 3, 4, 5, 6, 8, 16, 32, 40)


def check_ring8(rows, q, offsets):
    """rows [S,H,R,2,D]: what the rings hold; the new token of a sequence is what stands at slot 0."""
    S, H, R, _, D = rows.shape
    v, sc = quantize64(rows)
    kv, ks = v.float().to(E4).to(DEV), (torch.log2(sc) + 127).to(torch.uint8).view(torch.float8_e8m0fnu).to(DEV)
    held, head, sc = held_as(rows, E4), torch.zeros(S, dtype=torch.int32, device=DEV), 1 / math.sqrt(D)
    new = rows[:, :, 0].to(BF)
    assert torch.equal(held_as(new, E4), held[:, :, 0])               # the new token's rows in bf16 are held as those in fp32
    pb = torch.zeros(len(offsets), H, device=DEV)
    for overlap in (False, True):
        out = dwarf_b200.dsqg_decode_step_kv(q.to(DEV), *(new[:, :, i].contiguous().to(DEV) for i in (0, 1)), kv, head, pb, None, None, offsets, None, overlap=overlap,
                                             kv_scale=ks).double().cpu()
        at = [(0 - o) % R for o in offsets]
        for s in range(S):
            for h in range(H):
                qs, r = q[s, h][None].double(), held[s, h, at]
                o, spread, ds = attention64(qs, r[:, 0], r[:, 1], sc)
                off, bound = (out[s, h] - o[0]).abs(), e4m3_bound(qs, r, sc, o, spread, ds, torch.softmax(sc * qs @ r[:, 0].T, 1))[0]
                assert (off <= bound).all(), (s, h, (off / bound).max())


def ring_rows(S, H, D, offsets, g):
    return torch.randn(S, H, max(offsets) + 1, 2, D, generator=g).to(BF).float()


@pytest.mark.parametrize("H,D", [(2, 32), (3, 64), (1, 128)])
@pytest.mark.parametrize("offsets", [FEW, MANY], ids=["one_pass", "passes"])
def test_ring8(H, D, offsets):
    g = torch.Generator().manual_seed(D)
    rows, q = ring_rows(3, H, D, offsets, g), torch.randn(3, H, D, generator=g).to(BF)
    check_ring8(rows, 0.05 * q, offsets)


@pytest.mark.parametrize("H,D", [(2, 32), (3, 64), (1, 128), (2, 48)])
@pytest.mark.parametrize("offsets", [FEW, MANY], ids=["one_pass", "passes"])
@pytest.mark.parametrize("above", [12, 20, 26, 60])
def test_ring8_value_rows_that_carry_no_weight_take_no_bits(H, D, offsets, above):
    g = torch.Generator().manual_seed(D + above)
    S = 3
    rows, q0 = 0.25 * ring_rows(S, H, D, offsets, g), torch.randn(S, H, D, generator=g)
    R = rows.shape[2]
    for s, o in enumerate((0, offsets[5], offsets[-1])):
        rows[s, :, (0 - o) % R, 0] = (-120 * math.sqrt(D) * q0[s] / q0[s].square().sum(-1, keepdim=True)).to(BF).float()
        rows[s, :, (0 - o) % R, 1] = 2.0 ** above
    check_ring8(rows, q0.to(BF), offsets)


@pytest.mark.parametrize("H,D", [(2, 32), (3, 64), (1, 128)])
@pytest.mark.parametrize("offsets", [FEW, MANY], ids=["one_pass", "passes"])
def test_ring8_value_rows_of_zeros_take_no_bits(H, D, offsets):
    g = torch.Generator().manual_seed(D)
    rows = ring_rows(3, H, D, offsets, g) * torch.tensor([1.0, 2.0 ** -30])[:, None]
    R = rows.shape[2]
    for s, o in enumerate((0, offsets[5], offsets[-1])):
        rows[s, :, (0 - o) % R, 1] = -0.0
    check_ring8(rows, 0.05 * torch.randn(3, H, D, generator=g).to(BF), offsets)
