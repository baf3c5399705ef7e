"""Rings in 8 bits: quantised as they are written, read by the decode step and read back."""
import math

import pytest
import torch

import dwarf_b200
from tests.serving_util import HALF, attention64, dequantize64, quantize64, scale_values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4 = torch.float8_e4m3fn
SETS = {"43": dwarf_b200.OFFSETS_43, "late": (1, 2, 5, 9), "one": (0,), "many": tuple(range(100)) + (128,)}


def rings(S, H, R, D, g):
    raw = torch.randn(S, H, R, 2, D, generator=g) * torch.exp(torch.randn(S, H, R, 2, 1, generator=g))
    v, s = quantize64(raw)
    byte = (torch.log2(s) + 127).to(torch.uint8)
    return v.float().to(E4).to(DEV), byte.view(torch.float8_e8m0fnu).to(DEV)


def oracle(q, kn, vn, kv, ks, head, fill, pb, gain, se, offsets, f16):
    """(out, bound): the step in 64 bits on what the ring holds after it, and what may be off before the result is rounded.  f16: probabilities
    are operands in f16 (relative 2^-11 each, and values below its normal range are off by at most 2^-25 of the largest value a tap), and the query is after
    a power of two that brings its largest element to [1, 2) (elements off by at most 2^-25 of that)."""
    S, H, R, _, D = kv.shape
    rows = dequantize64(kv, ks)
    out, bound = torch.zeros(S, H, D, dtype=torch.float64), torch.zeros(S, H, D, dtype=torch.float64)
    for s in range(S):
        taps = [(j, o) for j, o in enumerate(offsets) if o < fill[s]]
        if not taps:
            continue
        at = [(head[s] - o) % R for _, o in taps]
        for h in range(H):
            k, v = rows[s, h, at, 0], rows[s, h, at, 1]
            if se is not None:
                k = k + se[[j for j, _ in taps]]
            o, spread, ds = attention64(q[s, h][None], k, v, 1 / math.sqrt(D), pb[[j for j, _ in taps], h])
            out[s, h] = o[0] * gain[h]
            bound[s, h] = (2 * ds[0] + 64 * 2.0 ** -24) * spread[0]
            if f16:
                bound[s, h] += 2.0 ** -11 * spread[0] + len(at) * 2.0 ** -25 * v.abs().max()
                bound[s, h] += 2 * (2.0 ** -24 * q[s, h].abs().max() * k.abs().sum(1).max() / math.sqrt(D)) * spread[0]
            bound[s, h] *= gain[h].abs()
    return out, bound


@pytest.mark.parametrize("S,H,D", [(1, 1, 64), (3, 2, 32), (2, 3, 128), (5, 1, 48), (2, 2, 8), (2, 1, 40), (3, 2, 80), (2, 1, 120), (1, 2, 16)])
@pytest.mark.parametrize("name", list(SETS))
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("overlap", [False, True])
def test_step(S, H, D, name, dt, overlap):
    offsets = SETS[name]
    if name == "43" and D not in (64, 32, 40):
        offsets = tuple(range(32)) + (48, 64)
    R = max(offsets) + 1 + (name == "one")
    g = torch.Generator().manual_seed(S * 100 + D)
    kv, ks = rings(S, H, R, D, g)
    q, kn, vn = (torch.randn(S, H, D, generator=g).to(dt) for _ in range(3))
    kn[0, 0] = 0                                                  # a row of zeros
    head = torch.randint(0, R, (S,), generator=g, dtype=torch.int32)
    fill = torch.randint(1, R + 1, (S,), generator=g, dtype=torch.int32)
    fill[0] = R
    if S > 1:
        fill[1] = 1
    pb, gain = torch.randn(len(offsets), H, generator=g), 0.8 + 0.4 * torch.rand(H, generator=g)
    for se in (None, torch.randn(len(offsets), D, generator=g) * 0.1):
        kv1, ks1 = kv.clone(), ks.clone()
        # slots that are no tap of the step, or older than the sequence, hold NaN: they must not count
        out = dwarf_b200.dsqg_decode_step_kv(q.to(DEV), kn.to(DEV), vn.to(DEV), kv1, head.to(DEV), pb.to(DEV), gain.to(DEV), None if se is None else se.to(DEV), offsets,
                                             fill.to(DEV), overlap=overlap, kv_scale=ks1)
        new, new_s = quantize64(torch.stack([kn, vn], 2))
        got, got_s = kv1.cpu().float().double(), scale_values(ks1)
        want, want_s = kv.cpu().float().double(), scale_values(ks)
        for s in range(S):
            want[s, :, head[s]], want_s[s, :, head[s]] = new[s], new_s[s]
        assert torch.equal(got, want) and torch.equal(got_s, want_s)              # the new slot, bit for bit, and no other
        o, b = oracle(q.double(), kn, vn, kv1, ks1, head.tolist(), fill.tolist(), pb.double(), gain.double(), None if se is None else se.double(), offsets,
                      dt is torch.bfloat16 and se is None and D in (32, 64, 128))
        err = (out.double().cpu() - o).abs()
        assert out.dtype is dt and (err <= HALF[dt] * o.abs() + b * (1 + HALF[dt])).all(), (err - HALF[dt] * o.abs() - b).max()


def test_slots_that_are_no_tap_do_not_count():
    offsets, S, H, D, R = (0, 1, 5), 2, 2, 64, 6
    g = torch.Generator().manual_seed(1)
    kv, ks = rings(S, H, R, D, g)
    q, kn, vn = (torch.randn(S, H, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(3))
    head, fill = torch.tensor([2, 0], dtype=torch.int32, device=DEV), torch.tensor([6, 3], dtype=torch.int32, device=DEV)
    pb = torch.zeros(3, H, device=DEV)
    want = dwarf_b200.dsqg_decode_step_kv(q, kn, vn, kv.clone(), head, pb, None, None, offsets, fill, kv_scale=ks.clone())
    bytes_ = ks.clone().view(torch.uint8)
    taps = {0: {2, 1, 3}, 1: {0, 5}}                              # sequence 1: three tokens, offset 5 is older than that
    for s in range(S):
        for r in range(R):
            if r not in taps[s]:
                bytes_[s, :, r] = 255
    got = dwarf_b200.dsqg_decode_step_kv(q, kn, vn, kv.clone(), head, pb, None, None, offsets, fill, kv_scale=bytes_.view(torch.float8_e8m0fnu))
    assert torch.isfinite(got).all() and torch.equal(got, want)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N", [1, 5, 49, 50, 130])
@pytest.mark.parametrize("D", [8, 40, 64, 128])
def test_cache_prefill_steps_and_read(dt, N, D):
    offsets, S, H = (0, 1, 2, 3, 8, 48), 2, 3
    g = torch.Generator().manual_seed(N + D)
    c = dwarf_b200.DSQGRingCache(2, S, H, D, offsets, dtype=E4, device=DEV)
    k, v = (torch.randn(S, H, N, D, generator=g).to(dt) for _ in range(2))
    k[0, 0, N - 1, 0] = float("nan")
    c.prefill(1, k.to(DEV), v.to(DEV))
    assert c.head.tolist() == [(N - 1) % 49] * S and c.fill.tolist() == [min(N, 49)] * S
    keep = list(range(max(0, N - 49), N))
    for name, src in ((0, k), (1, v)):
        vals, s = quantize64(src[:, :, keep])
        got = c.kv[1][:, :, [p % 49 for p in keep], name].cpu().float().double()
        gs = scale_values(c.kv_scale[1][:, :, [p % 49 for p in keep], name])
        assert torch.equal(torch.nan_to_num(got, 1234.0), torch.nan_to_num(vals, 1234.0)) and torch.equal(torch.nan_to_num(gs, 1234.0), torch.nan_to_num(s, 1234.0))
        assert torch.isnan(got[0, 0, -1]).all() == (name == 0)
        back = c.read(1, torch.float32)[name][:, :, [p % 49 for p in keep]].cpu().double()
        assert torch.equal(torch.nan_to_num(back, 1234.0), torch.nan_to_num(vals * s[..., None], 1234.0))      # exact in fp32
        b16 = c.read(1)[name][:, :, [p % 49 for p in keep]].cpu().double()
        assert torch.equal(torch.nan_to_num(b16, 1234.0), torch.nan_to_num(vals * s[..., None], 1234.0))       # and in bf16
    assert (c.kv[0].view(torch.uint8) == 0).all()
    # a step behind the prompt equals the step over a ring in full precision that holds the same values
    full = dwarf_b200.DSQGRingCache(1, S, H, D, offsets, dtype=torch.float32, device=DEV)
    c.prefill(0, v.to(DEV), v.to(DEV))
    full.prefill(0, *(t[:, :, [p % 49 for p in range(N)]].contiguous() if N <= 49 else None for t in c.read(0, torch.float32))) if N <= 49 else None
    if N <= 49:
        c.advance(), full.advance()
        q, kn, vn = (torch.randn(S, H, D, generator=g).to(DEV) for _ in range(3))
        hold = lambda t: (lambda a, b: (a * b[..., None]).float().to(DEV))(*quantize64(t))  # noqa: E731
        pb = torch.zeros(6, H, device=DEV)
        a = c.step(0, q, kn, vn, pb)
        b = full.step(0, q, hold(kn), hold(vn), pb)
        assert (a - b).abs().max() <= 2.0 ** -16 * b.abs().max() + 1e-6           # both fp32 evaluations of the same sums


def test_refusals():
    S, H, D, R = 2, 2, 32, 4
    offsets = (0, 1, 3)
    kv = torch.zeros(S, H, R, 2, D, dtype=torch.uint8, device=DEV).view(E4)
    ks = torch.zeros(S, H, R, 2, dtype=torch.uint8, device=DEV)
    q = torch.zeros(S, H, D, dtype=torch.bfloat16, device=DEV)
    head = torch.zeros(S, dtype=torch.int32, device=DEV)
    pb = torch.zeros(3, H, device=DEV)
    step = lambda q=q, kv=kv, **kw: dwarf_b200.dsqg_decode_step_kv(q, q, q, kv, head, pb, None, None, offsets, **kw)  # noqa: E731
    assert step(kv_scale=ks).shape == q.shape
    for bad in (lambda: step(), lambda: step(kv_scale=ks[:1]), lambda: step(kv_scale=ks.float()), lambda: step(kv_scale=ks.cpu()), lambda: step(kv=kv.float(), kv_scale=ks)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        step(q=q.half(), kv_scale=ks)
    c = dwarf_b200.DSQGRingCache(1, S, H, D, offsets, dtype=E4, device=DEV)
    x = torch.zeros(S, H, 3, D, device=DEV)
    with pytest.raises(TypeError):
        c.prefill(0, x.half(), x.half())
    with pytest.raises(ValueError):
        c.prefill(0, x, x.bfloat16())
    with pytest.raises(ValueError):
        c.prefill(0, x.cpu(), x.cpu())


@pytest.mark.parametrize("S,H,D", [(3, 2, 32), (2, 3, 64), (2, 1, 128), (3, 1, 48), (2, 2, 8), (2, 1, 40), (2, 1, 120)])
@pytest.mark.parametrize("name", list(SETS))
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("overlap", [False, True])
def test_slots_that_are_no_tap_hold_nan(S, H, D, name, dt, overlap):
    """Every width, type, form and number of passes: rows of NaN in all slots but the live taps change nothing, and stay where they are."""
    offsets = SETS[name]
    R = max(offsets) + 1 + (name == "one")
    g = torch.Generator().manual_seed(S * 100 + D)
    kv, ks = rings(S, H, R, D, g)
    q, kn, vn = (torch.randn(S, H, D, generator=g).to(dt).to(DEV) for _ in range(3))
    head = torch.randint(0, R, (S,), generator=g, dtype=torch.int32)
    fill = torch.randint(1, R + 1, (S,), generator=g, dtype=torch.int32)
    fill[0], fill[1] = R, 1
    pb = torch.randn(len(offsets), H, generator=g).to(DEV)
    dead = torch.ones(S, R, dtype=torch.bool)
    for s in range(S):
        for o in offsets:
            if o < fill[s]:
                dead[s, (head[s] - o) % R] = False
    dead = dead.to(DEV)[:, None].expand(S, H, R)
    for se in (None, 0.1 * torch.randn(len(offsets), D, generator=g).to(DEV)):
        runs = []
        for poison in (False, True):
            kv1, ks1 = kv.clone(), ks.clone()
            if poison:
                kv1.view(torch.uint8)[dead], ks1.view(torch.uint8)[dead] = 0x7f, 255
            before, before_s = kv1.view(torch.uint8).clone(), ks1.view(torch.uint8).clone()
            out = dwarf_b200.dsqg_decode_step_kv(q, kn, vn, kv1, head.to(DEV), pb, None, se, offsets, fill.to(DEV), overlap=overlap, kv_scale=ks1)
            at = (torch.arange(S), slice(None), head.long())
            new, new_s = quantize64(torch.stack([kn, vn], 2))
            assert torch.equal(kv1[at].float().double().cpu(), new) and torch.equal(scale_values(ks1[at]), new_s)
            kv1.view(torch.uint8)[at], ks1.view(torch.uint8)[at] = before[at], before_s[at]
            assert torch.equal(kv1.view(torch.uint8), before) and torch.equal(ks1.view(torch.uint8), before_s)
            runs.append(out)
        assert torch.isfinite(runs[1]).all() and torch.equal(runs[0], runs[1])
