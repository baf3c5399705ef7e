"""int4_linear against the product in 64 bits."""
import pytest
import torch

import dwarf_b200
from tests.serving_util import quantize64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(M, K, N, group, e4m3, seed=0):
    g = torch.Generator().manual_seed(seed + M + K + N)
    w = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    s = (torch.randn(N, K // group, generator=g) * 0.01).to(torch.bfloat16)
    b = torch.randn(N, generator=g)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
    if not e4m3:
        x = x.to(torch.bfloat16)
        return x, None, w, s, b, x.double()
    v, sc = quantize64(x)
    return v.float().to(torch.float8_e4m3fn), (torch.log2(sc) + 127).to(torch.uint8).view(torch.float8_e8m0fnu), w, s, b, v * sc[:, None]


def oracle(x64, w, s, b):
    W = torch.stack([w & 15, w >> 4], -1).flatten(1).double() - 8
    W = W * s.double().repeat_interleave(W.shape[1] // s.shape[1], 1)
    y = x64 @ W.T
    size = x64.abs() @ W.abs().T
    return (y, size) if b is None else (y + b.double(), size + b.double().abs())


def run(x, xs, w, s, b):
    to = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    return dwarf_b200.int4_linear(to(x), to(w), to(s), to(b), x_scale=to(xs))


@pytest.mark.parametrize("M,K,N", [(1, 128, 16), (1, 256, 768), (3, 384, 17), (8, 1152, 100), (9, 128, 33), (16, 4096, 40), (17, 256, 48), (1, 16384, 5), (65, 640, 70), (2, 1024, 1), (24, 2048, 64)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16", "e4m3"])
def test_products(M, K, N, group, e4m3):
    if K % 128 == 0 and group == 32 and K > 128:
        K += 32                                                   # the last tile of columns is not whole
    if group == 64 and K > 128:
        K += 64
    x, xs, w, s, b, x64 = make(M, K, N, group, e4m3)
    for bias in (None, b):
        y = run(x, xs, w, s, bias)
        want, size = oracle(x64, w, s, bias)
        # products are exact in fp32; sums in fp32 (whatever their order, K 2^-24 of the sum of magnitudes; tensor cores may truncate: twice that), one rounding to bf16
        bound = 2.0 ** -8 * want.abs() + 2 * (K + 16) * 2.0 ** -24 * size * 1.01
        assert y.dtype is torch.bfloat16 and y.shape == (M, N)
        err = (y.double().cpu() - want).abs()
        assert (err <= bound).all(), (err - bound).max()


def test_every_nibble_and_column_is_where_it_belongs():
    """x picks one column: y is that column of W, exactly."""
    K, N, group = 224, 37, 32
    _, _, w, s, _, _ = make(1, K, N, group, False)
    s = torch.exp2(torch.randint(-3, 3, s.shape, generator=torch.Generator().manual_seed(0)).float()).to(torch.bfloat16)
    x = torch.eye(K).to(torch.bfloat16)
    want, _ = oracle(x.double(), w, s, None)
    assert torch.equal(run(x, None, w, s, None).double().cpu(), want)
    one = torch.full((K,), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    assert torch.equal(run(torch.eye(K).to(torch.float8_e4m3fn), one, w, s, None).double().cpu(), want)


def test_rows_do_not_mix():
    x, _, w, s, b, x64 = make(20, 256, 64, 64, False)
    want = run(x, None, w, s, b)
    bad = x.clone()
    bad[3, 7], bad[18, 0] = float("nan"), float("inf")
    got = run(bad, None, w, s, b)
    keep = [i for i in range(20) if i not in (3, 18)]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[3]).all() and not torch.isfinite(got[18]).any()
    one = torch.cat([run(x[i:i + 1], None, w, s, b) for i in range(20)])
    assert (one.double() - want.double()).abs().max() <= 2.0 ** -7 * want.double().abs().max()
    v, xs, w, s, b, _ = make(5, 256, 64, 64, True)
    xs.view(torch.uint8)[2] = 255
    got = run(v, xs, w, s, b)
    assert torch.isnan(got[2]).all() and torch.isfinite(got[[0, 1, 3, 4]]).all()


def test_module_and_norm_in_front():
    """Norm in 8 bits -> 4-bit projection, as a decode step runs them; the module on bf16, fp32 and 8-bit rows."""
    g = torch.Generator().manual_seed(0)
    lin = torch.nn.Linear(256, 96).to(DEV)
    m = dwarf_b200.Int4Linear.from_linear(lin, 64)
    x, r = torch.randn(4, 256, generator=g).to(torch.bfloat16).to(DEV), torch.randn(4, 256, generator=g).to(DEV)
    w = (1 + 0.1 * torch.randn(256, generator=g)).to(DEV)
    with torch.no_grad():
        y8, s8, h = dwarf_b200.rms_norm_e4m3(x, w, r)
        got = m(dwarf_b200.Rows8(y8, s8))
        x64 = y8.float().double().cpu() * torch.exp2(s8.view(torch.uint8).double().cpu() - 127)[:, None]
        want, size = oracle(x64, m.weight.cpu(), m.scales.cpu(), m.bias.cpu())
        assert ((got.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 600 * 2.0 ** -24 * size).all()
        a, b = m(h), m(h.to(torch.bfloat16))
        assert a.dtype is torch.float32 and torch.equal(a, b.float())
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert m(h).dtype is torch.bfloat16
        assert m(h.view(2, 2, 256)).shape == (2, 2, 96) and m(h[:0]).shape == (0, 96)
        # 4 bits instead of 32: within half a step of every weight
        full = torch.nn.functional.linear(h.double(), lin.weight.double(), lin.bias.double())
        step = m.scales.double().repeat_interleave(64, 1)
        lim = h.double().abs() @ (0.54 * step).T
        assert ((a.double() - full).abs() <= lim + 2.0 ** -7 * (full.abs() + h.double().abs() @ lin.weight.double().abs().T)).all()


def test_repeatable_and_captured():
    x, _, w, s, b, _ = make(4, 4096, 512, 128, False)
    x, w, s, b = (t.to(DEV) for t in (x, w, s, b))
    want = dwarf_b200.int4_linear(x, w, s, b)
    for _ in range(5):
        assert torch.equal(dwarf_b200.int4_linear(x, w, s, b), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = dwarf_b200.int4_linear(x, w, s, b)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, dwarf_b200.int4_linear(x, w, s, b))


def test_refusals():
    x, w = torch.zeros(2, 128, device=DEV, dtype=torch.bfloat16), torch.zeros(8, 64, device=DEV, dtype=torch.uint8)
    s, b = torch.zeros(8, 2, device=DEV, dtype=torch.bfloat16), torch.zeros(8, device=DEV)
    f = dwarf_b200.int4_linear
    f(x, w, s, b)
    x8 = x.to(torch.float8_e4m3fn)
    xs = torch.zeros(2, device=DEV, dtype=torch.uint8)
    for bad in (lambda: f(x[:, :64], w, s), lambda: f(x, w.t(), s), lambda: f(x, w.int(), s), lambda: f(x, w, s.float()), lambda: f(x, w, s[:4]), lambda: f(x, w, s[:, :1].expand(8, 8).contiguous()),
                lambda: f(x, w, s, b[:4]), lambda: f(x, w, s, b.cpu()), lambda: f(x8, w, s), lambda: f(x, w, s, x_scale=xs), lambda: f(x8, w, s, x_scale=xs[:1]), lambda: f(x, w.cpu(), s)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(x.float(), w, s), lambda: f(x.half(), w, s)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        f(x.requires_grad_(True), w, s)


@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("M", [524_288, 524_289, 1_048_560, 1_048_563])
def test_a_prompt_of_many_sequences(M, e4m3):
    """As many rows as 256 prompts of 2048 tokens have, and more than one launch takes (65,535 blocks of 16)."""
    x, xs, w, s, b, x64 = make(16, 32, 5, 32, e4m3)
    y, size = oracle(x64, w, s, b)
    at = torch.arange(M, device=DEV) * 7 % 16
    out = dwarf_b200.int4_linear(x.to(DEV).view(torch.uint8)[at].view(x.dtype), w.to(DEV), s.to(DEV), b.to(DEV), x_scale=None if xs is None else xs.to(DEV).view(torch.uint8)[at].view(xs.dtype))
    assert out.shape == (M, 5)
    assert ((out.double() - y.to(DEV)[at]).abs() <= 2.0 ** -8 * y.abs().to(DEV)[at] + 40 * 2.0 ** -24 * size.to(DEV)[at]).all()      # 32 products, their scale, the bias
