"""The paged cache: written, read back and attended to, against plain forms in 64 bits."""
import math

import pytest
import torch

import dwarf_b200
from tests.serving_util import HALF, attention64, quantize64, scale_values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def make_cache(lengths, H, page, D, dtype, g, spare=3, nan=True):
    """Pages in shuffled order; rows no sequence owns are NaN.  Returns (kv, scale, table, rows [S] of [n,H,2,D] float64)."""
    per = [-(-n // page) for n in lengths]
    P, cols = sum(per) + spare, max(1, max(per))
    order = torch.randperm(P, generator=g).tolist()
    kv = torch.full((P, H, page, 2, D), float("nan") if nan else 0.0)
    table = torch.full((len(lengths), cols), -1, dtype=torch.int32)
    rows = []
    for s, n in enumerate(lengths):
        x = torch.randn(n, H, 2, D, generator=g) * torch.exp(0.7 * torch.randn(n, H, 2, 1, generator=g))
        if dtype is not E4:
            x = x.to(dtype).float()
        for c in range(per[s]):
            p = order.pop()
            table[s, c] = p
            part = x[c * page:(c + 1) * page]
            kv[p, :, :part.shape[0]] = part.transpose(0, 1)
        rows.append(x.double())
    if dtype is not E4:
        return kv.to(dtype).to(DEV), None, table.to(DEV), rows
    v, s = quantize64(kv)
    byte = torch.where(torch.isnan(s), torch.full_like(s, 255), torch.log2(s) + 127).to(torch.uint8)
    v8 = torch.nan_to_num(v, 0.0).float().to(E4)
    v8.view(torch.uint8)[torch.isnan(v)] = 0x7f
    held = []
    for x in rows:
        a, b = quantize64(x)
        held.append(a * b[..., None])
    return v8.to(DEV), byte.view(torch.float8_e8m0fnu).to(DEV), table.to(DEV), held


def held_as(x, dtype):
    """Rows as a cache of this type holds them, float64."""
    if dtype is E4:
        a, b = quantize64(x)
        return a * b[..., None]
    return x.to(dtype).double()


def check_step(lengths, H, G, D, page, dtype, q_dt, new=True, max_length=None, scale=None, seed=0):
    g = torch.Generator().manual_seed(seed + D + page + G)
    S = len(lengths)
    kv, ks, table, rows = make_cache(lengths, H, page, D, dtype, g)
    q, kn, vn = torch.randn(S, H * G, D, generator=g).to(q_dt), torch.randn(S, H, D, generator=g).to(q_dt), torch.randn(S, H, D, generator=g).to(q_dt)
    if S > 1:
        vn[0] *= 1000.0                                           # the last value row far above the others: the running scale moves
    ln = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    before = kv.clone()
    args = (kn.to(DEV), vn.to(DEV)) if new else (None, None)
    out = dwarf_b200.paged_attention_step(q.to(DEV), *args, kv, table, ln, kv_scale=ks, scale=scale, max_length=max_length)
    assert out.shape == q.shape and out.dtype is q_dt
    sc = 1 / math.sqrt(D) if scale is None else scale
    # the form on tensor cores: widths that are multiples of 32, and 48 and 80, pages of a multiple of 16 positions
    p_half = 0.0 if (q_dt is F or dtype is F or (D % 32 and D not in (48, 80)) or page % 16) else 2.0 ** -8 if dtype is BF else 2.0 ** -11      # probabilities as an operand in 16 bits
    for s, n in enumerate(lengths):
        for h in range(H):
            r = rows[s][:, h].clone()
            if new and n:
                r[n - 1, 0], r[n - 1, 1] = held_as(kn[s, h][None], dtype)[0], held_as(vn[s, h][None], dtype)[0]
            qs = q[s, h * G:(h + 1) * G].double()
            o, spread, ds = attention64(qs, r[:, 0], r[:, 1], sc)
            got = out[s, h * G:(h + 1) * G].double().cpu()
            more = (2 * ds[:, None] + p_half + (n + 64) * 2.0 ** -24) * spread
            if p_half == 2.0 ** -11:
                # f16 below its normal range: probabilities times scales to 2^-25 of the largest value, queries to 2^-25 of their largest element
                more = more + n * 2.0 ** -25 * (r[:, 1].abs().max() if n else 0) / 1.0
                more = more + 2 * sc * 2.0 ** -24 * qs.abs().max() * (r[:, 0].abs().sum(1).max() if n else 0) * spread
            bound = HALF[q_dt] * o.abs() + more * (1 + HALF[q_dt])
            assert ((got - o).abs() <= bound).all(), (s, h, n, ((got - o).abs() - bound).max())
    # the new rows are stored, and nothing else is touched
    after, had = kv.view(torch.uint8).cpu(), before.view(torch.uint8).cpu()
    same = torch.ones(kv.shape[:3], dtype=torch.bool)
    for s, n in enumerate(lengths):
        if new and n:
            p, i = int(table[s, (n - 1) // page]), (n - 1) % page
            same[p, :, i] = False
            want = held_as(torch.stack([kn[s], vn[s]], 1), dtype)
            got = kv[p, :, i].float().double().cpu()
            assert torch.equal(got if ks is None else got * scale_values(ks[p, :, i])[..., None], want)
    assert torch.equal(after[same], had[same])


TYPES = [(BF, BF), (E4, BF), (F, F), (E4, F), (BF, F), (F, BF)]


@pytest.mark.parametrize("dtype,q_dt", TYPES, ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("H,G,D,page", [(1, 1, 32, 16), (2, 1, 64, 48), (1, 4, 128, 64), (2, 3, 96, 16), (1, 12, 64, 32), (1, 20, 32, 16), (2, 2, 80, 16), (1, 1, 8, 16),
                                        (1, 5, 64, 10), (2, 1, 40, 1), (1, 17, 128, 16), (3, 8, 128, 32), (2, 3, 48, 16), (1, 9, 80, 48), (1, 17, 48, 64), (3, 8, 80, 32)])
def test_step(dtype, q_dt, H, G, D, page):
    check_step([0, 1, 2, 15, 16, 17, 63, 64, 65, 130], H, G, D, page, dtype, q_dt)
    check_step([33, 16], H, G, D, page, dtype, q_dt, new=False, scale=0.3)


@pytest.mark.parametrize("dtype,q_dt", TYPES, ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("lengths,most", [([2000, 0, 1, 777], None), ([1025], None), ([64 * 30, 64 * 30 + 1], 2048), ([5000], 5000)])
def test_step_split_over_the_length(dtype, q_dt, lengths, most):
    check_step(lengths, 2, 2, 64, 64, dtype, q_dt, max_length=most)
    check_step(lengths, 1, 1, 40, 20, dtype, q_dt, max_length=most)
    check_step(lengths, 1, 3, 80, 32, dtype, q_dt, max_length=most)


def test_bad_tables_and_lengths_give_nan_and_touch_nothing():
    g = torch.Generator().manual_seed(0)
    for dtype, D, page in ((BF, 64, 16), (E4, 64, 16), (F, 64, 16), (E4, 40, 16), (BF, 64, 10)):
        lengths = [40, 40, 40, 40, 40, 40]
        kv, ks, table, rows = make_cache(lengths, 1, page, D, dtype, g, nan=False)
        t = table.clone()
        good = dwarf_b200.paged_attention_step(*[torch.ones(6, 1, D, device=DEV, dtype=BF)] * 3, kv.clone(), t, torch.tensor(lengths, dtype=torch.int32, device=DEV),
                                               kv_scale=None if ks is None else ks.clone())
        t[1, 0], t[2, 1], t[3, (40 - 1) // page] = -1, kv.shape[0], 2 ** 30
        n = torch.tensor([40, 40, 40, 40, -3, t.shape[1] * page + 1], dtype=torch.int32, device=DEV)
        before = kv.clone()
        out = dwarf_b200.paged_attention_step(*[torch.ones(6, 1, D, device=DEV, dtype=BF)] * 3, kv, t, n, kv_scale=ks)
        assert torch.equal(out[0], good[0]) and torch.isnan(out[1:]).all()
        changed = (kv.view(torch.uint8) != before.view(torch.uint8)).view(kv.shape[0], -1).any(1).cpu()
        owned = {int(table[s, (40 - 1) // page]) for s in (0, 1, 2)}
        assert {i for i, c in enumerate(changed.tolist()) if c} <= owned
        short = dwarf_b200.paged_attention_step(*[torch.ones(6, 1, D, device=DEV, dtype=BF)] * 3, kv, table, torch.tensor([5, 6, 7, 17, 0, 16], dtype=torch.int32, device=DEV),
                                                kv_scale=ks, max_length=16)
        assert torch.isnan(short[3]).all() and (short[4] == 0).all() and torch.isfinite(short[[0, 1, 2, 5]]).all()


def test_values_that_are_not_finite_stay_with_their_sequence_and_head():
    g = torch.Generator().manual_seed(0)
    for dtype, q_dt in TYPES:
        kv, ks, table, _ = make_cache([40, 40], 2, 16, 64, dtype, g)
        q = torch.randn(2, 4, 64, generator=g).to(q_dt).to(DEV)
        kn = torch.randn(2, 2, 64, generator=g).to(q_dt).to(DEV)
        vn = kn.clone()
        vn[0, 1, 5] = float("inf")
        out = dwarf_b200.paged_attention_step(q, kn, vn, kv, table, torch.tensor([40, 40], dtype=torch.int32, device=DEV), kv_scale=ks)
        assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, :2]).all() and not torch.isfinite(out[0, 2:, 5]).any()


@pytest.mark.parametrize("dtype", [BF, F, E4], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("src", [BF, F], ids=["from_bf16", "from_fp32"])
@pytest.mark.parametrize("H,D,page", [(1, 8, 16), (2, 64, 16), (3, 40, 7), (2, 128, 64), (12, 80, 32)])
def test_write_and_read(dtype, src, H, D, page):
    g = torch.Generator().manual_seed(D)
    lengths, start = [5, 0, 33, 1, 64], [3, 7, 0, 31, 16]
    S, cols = 5, -(-80 // page)
    P = S * cols + 2
    table = torch.randperm(P, generator=g)[:S * cols].view(S, cols).to(torch.int32)
    table[2, cols - 1] = P                                        # no page there; sequence 2 ends in front of it
    shape = (P, H, page, 2, D)
    kv = torch.full(shape, 0x55, dtype=torch.uint8).view(E4) if dtype is E4 else torch.full(shape, 3.25, dtype=dtype)
    ks = torch.full(shape[:4], 130, dtype=torch.uint8).view(torch.float8_e8m0fnu) if dtype is E4 else None
    kv, ks, table = kv.to(DEV), None if ks is None else ks.to(DEV), table.to(DEV)
    cu = [2]                                                      # two rows in front of the first sequence, three behind the last
    for n in lengths:
        cu.append(cu[-1] + n)
    T = cu[-1] + 3
    fused = torch.randn(T, 3, H, D, generator=g).to(src).to(DEV)
    k, v = fused[:, 1], fused[:, 2]
    to = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    before = kv.clone()
    dwarf_b200.paged_kv_write(k, v, kv, table, to(cu), to(start), kv_scale=ks)
    want = before.float().double().cpu() * (1 if ks is None else 8.0)
    for s, n in enumerate(lengths):
        for i in range(n):
            p = start[s] + i
            t = cu[s] + i
            want[int(table[s, p // page]), :, p % page] = held_as(torch.stack([k[t], v[t]], 1).cpu(), dtype)
    got = kv.float().double().cpu() * (1 if ks is None else scale_values(ks)[..., None])
    assert torch.equal(got, want)
    for dt in (BF, F):
        rk, rv = dwarf_b200.paged_kv_read(kv, table, to(cu), T, to(start), kv_scale=ks, dtype=dt)
        assert rk.shape == (T, H, D) and rk.dtype is dt
        for r, x in ((rk, k), (rv, v)):
            w = held_as(x.cpu(), dtype).to(dt).double()           # 8-bit values are exact in both types
            w[:2], w[cu[-1]:] = 0, 0
            assert torch.equal(r.double().cpu(), w)
    # positions beyond the table, or in front of 0, or without a page: dropped, and NaN when read
    dwarf_b200.paged_kv_write(k[:6], v[:6], kv, table, to([0, 1, 2, 3, 4, 6]), to([cols * page, -1, 2 ** 31 - 1, -2 ** 31, cols * page - 1]), kv_scale=ks)
    last = (int(table[4, cols - 1]), page - 1)
    got2 = kv.float().double().cpu() * (1 if ks is None else scale_values(ks)[..., None])
    want[last[0], :, last[1]] = held_as(torch.stack([k[4], v[4]], 1).cpu(), dtype)
    assert torch.equal(got2, want)
    rk, _ = dwarf_b200.paged_kv_read(kv, table, to([0, 1, 2, 3, 4, 6]), 6, to([cols * page, -1, 2 ** 31 - 1, -2 ** 31, cols * page - 1]), kv_scale=ks)
    assert torch.isnan(rk[[0, 1, 2, 3, 5]]).all() and torch.isfinite(rk[4]).all()


@pytest.mark.parametrize("dtype", [BF, E4], ids=["bf16", "e4m3"])
def test_cache_object(dtype):
    """A prompt in two chunks, tokens one by one over page ends, a sequence that leaves and one that takes its place."""
    g = torch.Generator().manual_seed(4)
    L, S, H, G, D, page = 2, 3, 2, 2, 32, 16
    c = dwarf_b200.PagedKVCache(L, S, H, D, max_length=100, pages=12, page_size=page, dtype=dtype, device=DEV)
    text = [[[] for _ in range(S)] for _ in range(L)]

    def chunk(counts):
        ch = c.extend(counts)
        for layer in range(L):
            kv = torch.randn(ch[2], 2, H, D, generator=g).to(BF)
            c.write(layer, kv[:, 0].to(DEV), kv[:, 1].to(DEV), ch)
            at = 0
            for s, n in enumerate(counts):
                text[layer][s] += list(held_as(kv[at:at + n], dtype))
                at += n
    chunk([20, 0, 15])
    chunk([10, 0, 1])
    for step in range(20):
        if step == 7:
            c.release(0)
            for layer in range(L):
                text[layer][0] = []
        if step == 9:
            chunk([0, 33, 0])
        c.advance()
        for layer in range(L):
            q, kn, vn = torch.randn(S, H * G, D, generator=g).to(BF), torch.randn(S, H, D, generator=g).to(BF), torch.randn(S, H, D, generator=g).to(BF)
            out = c.step(layer, q.to(DEV), kn.to(DEV), vn.to(DEV)).double().cpu()
            for s in range(S):
                if not text[layer][s]:
                    assert (out[s] == 0).all()
                    continue
                text[layer][s].append(held_as(torch.stack([kn[s], vn[s]], 1)[None], dtype)[0].transpose(0, 1))
                r = torch.stack(text[layer][s])                                                  # [n,2,H,D]
                for h in range(H):
                    qs = q[s, h * G:(h + 1) * G].double()
                    o, spread, ds = attention64(qs, r[:, 0, h], r[:, 1, h], 1 / math.sqrt(D))
                    bound = 2.0 ** -8 * o.abs() + (2 * ds[:, None] + 2.0 ** -8 + len(r) * 2.0 ** -20) * spread * 1.01
                    assert ((out[s, h * G:(h + 1) * G] - o).abs() <= bound).all()
    k, v, cu = c.read(0)
    assert cu.tolist()[-1] == sum(len(t) for t in text[0]) == k.shape[0]
    want = torch.cat([torch.stack(t) for t in text[0] if t])
    assert torch.equal(k.double().cpu(), want[:, 0].to(BF).double()) and torch.equal(v.double().cpu(), want[:, 1].to(BF).double())


@pytest.mark.parametrize("dtype", [BF, E4], ids=["bf16", "e4m3"])
def test_captured_steps_follow_lengths_and_tables(dtype):
    g = torch.Generator().manual_seed(2)
    c = dwarf_b200.PagedKVCache(1, 2, 1, 64, max_length=1500, page_size=64, dtype=dtype, device=DEV)
    for s in range(2):
        c.reserve(s, 1500)
    ch = c.extend([700, 3])
    c.write(0, *(torch.randn(703, 1, 64, generator=g).to(BF).to(DEV) for _ in range(2)), ch)
    c.advance()
    q, kn, vn = (torch.randn(2, 1, 64, generator=g).to(BF).to(DEV) for _ in range(3))
    call = lambda: c.step(0, q, kn, vn, max_length=1500)  # noqa: E731
    call()
    graphs, outs = [], []
    for _ in range(2):                                            # two graphs, each with scratch of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for _ in range(3):
        c.advance()
        kn.normal_(), q.normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        assert torch.equal(outs[0], call())


def test_two_streams_at_once():
    g = torch.Generator().manual_seed(2)
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for i in range(2):
        kv, ks, table, _ = make_cache([3000, 100], 2, 64, 64, E4, g)
        q = torch.randn(2, 4, 64, generator=g).to(BF).to(DEV)
        k = torch.randn(2, 2, 64, generator=g).to(BF).to(DEV)
        work.append((q, k, k, kv, table, torch.tensor([3000, 100], dtype=torch.int32, device=DEV), ks))
    want = [dwarf_b200.paged_attention_step(*w) for w in work]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(dwarf_b200.paged_attention_step(*work[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_offsets_beyond_32_bits():
    """Pages whose elements lie beyond 2^31 (and bytes beyond 2^32) of the start of the cache."""
    P, H, page, D = 70000, 4, 64, 128                             # 4.6e9 elements
    kv = torch.zeros(P, H, page, 2, D, dtype=torch.uint8, device=DEV).view(E4)
    ks = torch.full((P, H, page, 2), 127, dtype=torch.uint8, device=DEV)
    table = torch.tensor([[P - 1, 3], [1, P - 2]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(200, H, D, generator=g).to(BF).to(DEV) for _ in range(2))
    cu = torch.tensor([0, 100, 200], dtype=torch.int32, device=DEV)
    dwarf_b200.paged_kv_write(k, v, kv, table, cu, kv_scale=ks)
    rk, rv = dwarf_b200.paged_kv_read(kv, table, cu, 200, kv_scale=ks)
    assert torch.equal(rk.double().cpu(), held_as(k.cpu(), E4)) and torch.equal(rv.double().cpu(), held_as(v.cpu(), E4))
    q = torch.randn(2, H, D, generator=g).to(BF).to(DEV)
    n = torch.tensor([100, 100], dtype=torch.int32, device=DEV)
    out = dwarf_b200.paged_attention_step(q, None, None, kv, table, n, kv_scale=ks).double().cpu()
    for s in range(2):
        for h in range(H):
            o, spread, ds = attention64(q[s, h][None].double().cpu(), rk[s * 100:(s + 1) * 100, h].double().cpu(), rv[s * 100:(s + 1) * 100, h].double().cpu(), 1 / math.sqrt(D))
            assert ((out[s, h] - o[0]).abs() <= 2.0 ** -8 * o[0].abs() + (2 * ds + 2.0 ** -10) * spread[0]).all()


def test_refusals():
    kv = torch.zeros(4, 2, 16, 2, 64, device=DEV, dtype=BF)
    kv8, ks = torch.zeros(4, 2, 16, 2, 64, device=DEV, dtype=torch.uint8).view(E4), torch.zeros(4, 2, 16, 2, device=DEV, dtype=torch.uint8)
    table, n = torch.zeros(3, 2, dtype=torch.int32, device=DEV), torch.ones(3, dtype=torch.int32, device=DEV)
    q, k = torch.zeros(3, 4, 64, device=DEV, dtype=BF), torch.zeros(3, 2, 64, device=DEV, dtype=BF)
    step = lambda q=q, k=k, v=k, kv=kv, table=table, n=n, **kw: dwarf_b200.paged_attention_step(q, k, v, kv, table, n, **kw)  # noqa: E731
    step()
    for bad in (lambda: step(q=q[:, :3]), lambda: step(q=q[:2]), lambda: step(k=None), lambda: step(k=k.float()), lambda: step(k=k[:, :1]), lambda: step(kv=kv8),
                lambda: step(kv_scale=ks), lambda: step(kv=kv8, kv_scale=ks[:3]), lambda: step(kv=kv.transpose(1, 2)), lambda: step(table=table.long()), lambda: step(n=n.long()),
                lambda: step(n=n[:2]), lambda: step(n=n.cpu()), lambda: step(table=table.cpu()), lambda: step(q=q.cpu()), lambda: step(scale=0.0), lambda: step(scale=float("nan")),
                lambda: step(max_length=-1), lambda: step(out=q[:2]), lambda: step(table=table.t().contiguous().t())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: step(q=q.half()), lambda: step(kv=kv.half())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(dwarf_b200.DSQGError):
        wide = torch.zeros(1, 1, 16, 2, 256, device=DEV, dtype=BF)
        x = torch.zeros(3, 1, 256, device=DEV, dtype=BF)
        step(q=x, k=x, v=x, kv=wide)
    with pytest.raises(RuntimeError):
        step(q=q.requires_grad_(True))
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV)
    for bad in (lambda: dwarf_b200.paged_kv_write(k, k[:2], kv, table, cu), lambda: dwarf_b200.paged_kv_write(k, k, kv, table, cu[:3]), lambda: dwarf_b200.paged_kv_write(k, k, kv8, table, cu),
                lambda: dwarf_b200.paged_kv_read(kv, table, cu, -1), lambda: dwarf_b200.paged_kv_read(kv, table, cu.long(), 3)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        dwarf_b200.paged_kv_read(kv, table, cu, 3, dtype=torch.float16)
    dwarf_b200.paged_kv_write(k[:0], k[:0], kv, table, torch.zeros(4, dtype=torch.int32, device=DEV))
    assert dwarf_b200.paged_kv_read(kv, table, cu, 0)[0].shape == (0, 2, 64)
