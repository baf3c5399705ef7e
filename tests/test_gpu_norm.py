"""rms_norm and rms_norm_e4m3 against the formulas in 64 bits."""
import pytest
import torch

import dwarf_b200
from tests.serving_util import HALF, quantize64, scale_values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F = torch.bfloat16, torch.float32
EPS = 1e-6
# Sums of D squares or products in fp32: a thread adds at most 32 of them one after the other, at most 10 steps join threads; rsqrt, division
# and the products behind them round a handful of times more.
SUM = 64 * 2.0 ** -24


def make(shape, x_dt, s_dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    x = (torch.randn(*shape, generator=g) * 0.5).to(x_dt).to(DEV)
    r = None if s_dt is None else torch.randn(*shape, generator=g).to(s_dt).to(DEV)
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(DEV)
    return x, r, w, g


def forward64(x, r, w):
    h = x.double() if r is None else (x.double() + r.double()).to(r.dtype).double()
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    return h, h * rstd * w.double(), rstd


def near(got, want, more):
    """got is want rounded once, and off by `more` before."""
    err = (got.double() - want).abs()
    bound = HALF[got.dtype] * want.abs() + more * (1 + HALF[got.dtype])
    assert (err <= bound).all(), f"largest excess {(err - bound).max().item()}, error {err.max().item()}"


SHAPES = [(1, 1), (3, 7), (2, 5, 8), (33, 64), (17, 72), (5, 128), (9, 248), (300, 256), (7, 512), (4, 1000), (2, 1024), (3, 1111), (5, 2048), (3, 2056), (2, 4096), (2, 4097),
          (3, 8192), (2, 8200), (1, 40000), (1, 33001)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("x_dt,s_dt,y_dt", [(BF, F, BF), (BF, BF, BF), (F, F, F), (F, None, BF), (BF, None, F), (F, BF, F)])
def test_forward_and_gradients(shape, x_dt, s_dt, y_dt):
    x, r, w, g = make(shape, x_dt, s_dt)
    for t in (x, w) + (() if r is None else (r,)):
        t.requires_grad_(True)
    got = dwarf_b200.rms_norm(x, w, r, eps=EPS, out_dtype=y_dt)
    y, h = got if r is not None else (got, None)
    h64, y64, rstd = forward64(x.detach(), None if r is None else r.detach(), w.detach())
    assert y.dtype is y_dt and y.shape == x.shape
    near(y.detach(), y64, SUM * y64.abs())
    if r is not None:
        assert h.dtype is s_dt and torch.equal(h.detach().double(), h64)          # one rounding of an exact sum, or of fp32's
    dy = torch.randn(*shape, generator=g).to(y_dt).to(DEV)
    dh = None if r is None else torch.randn(*shape, generator=g).to(s_dt).to(DEV)
    outs, ups = ([y], [dy]) if r is None else ([y, h], [dy, dh])
    grads = torch.autograd.grad(outs, [x, w] + ([] if r is None else [r]), ups)
    xh, gw = h64 * rstd, dy.double() * w.detach().double()
    mean = (gw * xh).mean(-1, keepdim=True)
    d = rstd * (gw - xh * mean) + (0 if dh is None else dh.double())
    size = rstd * (gw.abs() + xh.abs() * (gw * xh).abs().mean(-1, keepdim=True)) + (0 if dh is None else dh.double().abs())
    near(grads[0], d, SUM * size)
    if r is not None:
        near(grads[2], d, SUM * size)
    terms = (dy.double() * xh).reshape(-1, shape[-1])
    # at most 592 partial sums, of rows / 592 and a block's 32 row groups each, every addition one rounding; a term has the error of x^ as well
    adds = 700 + terms.shape[0] / 592
    assert ((grads[1].double() - terms.sum(0)).abs() <= (adds * 2.0 ** -24 + SUM) * terms.abs().sum(0)).all()
    assert grads[1].dtype is w.dtype and grads[0].dtype is x_dt


# More rows than a block for each takes, of widths that are and are not a multiple of eight: a block's sums of columns go over rows a grid apart.
@pytest.mark.parametrize("shape", [(25000, 7), (12001, 40), (7000, 65), (6001, 201), (1999, 1111), (1601, 2048), (700, 4097), (601, 8192), (301, 16383), (300, 30001)], ids=str)
@pytest.mark.parametrize("x_dt,s_dt,y_dt", [(BF, BF, BF), (BF, F, BF), (F, F, F)])
def test_many_rows(shape, x_dt, s_dt, y_dt):
    test_forward_and_gradients(shape, x_dt, s_dt, y_dt)


def test_gradients_are_the_differences_of_the_formula():
    x, r, w, g = make((3, 24), F, F, seed=3)
    dy, dh = torch.randn(3, 24, generator=g).double(), torch.randn(3, 24, generator=g).double()
    for t in (x, r, w):
        t.requires_grad_(True)
    y, h = dwarf_b200.rms_norm(x, w, r, eps=EPS)
    grads = torch.autograd.grad([y, h], [x, r, w], [dy.float().to(DEV), dh.float().to(DEV)])

    def value(a, b, c):
        s = a + b
        return float((s / torch.sqrt((s * s).mean(-1, keepdim=True) + EPS) * c * dy.float().double()).sum() + (s * dh.float().double()).sum())
    base = [t.detach().double().cpu() for t in (x, r, w)]
    for i, t in enumerate(base):
        for at in ((0, 0), (1, 7), (2, 23)) if t.dim() == 2 else ((0,), (11,), (23,)):
            e = 1e-5
            hi, lo = [b.clone() for b in base], [b.clone() for b in base]
            hi[i][at] += e
            lo[i][at] -= e
            diff = (value(*hi) - value(*lo)) / (2 * e)
            # a central difference of step 1e-5: e^2 times a third derivative of order 1..100, and 2^-53 |value| / e
            assert abs(float(grads[i][at]) - diff) <= 1e-5 * (1 + abs(diff))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("x_dt,s_dt", [(BF, F), (BF, BF), (F, None)])
def test_e4m3_output(shape, x_dt, s_dt):
    x, r, w, _ = make(shape, x_dt, s_dt, seed=5)
    with torch.no_grad():
        if x[..., :].numel() > 40:
            (x if r is None else r).view(-1, shape[-1])[0] = 0                    # a row of zeros (or of x alone)
        got = dwarf_b200.rms_norm_e4m3(x, w, r, eps=EPS)
    y8, s8 = got[0], got[1]
    assert y8.dtype is torch.float8_e4m3fn and s8.dtype is torch.float8_e8m0fnu and s8.shape == x.shape[:-1] and y8.shape == x.shape
    h64, y64, _ = forward64(x, r, w)
    if r is not None:
        assert torch.equal(got[2].double(), h64)
    s = scale_values(s8).to(DEV)[..., None]
    top = y64.abs().amax(-1, keepdim=True)
    zero = top == 0
    assert (s[zero] == 1).all()
    assert ((top <= 448 * s * (1 + SUM)) & ((top > 224 * s * (1 - SUM)) | zero | (s == 2.0 ** -126))).all()
    # half a step relative, half of e4m3's smallest step 2^-9 s near zero
    err = (y8.float().double() * s - y64).abs()
    assert (err <= HALF[torch.float8_e4m3fn] * y64.abs() + 2.0 ** -10 * s + 2 * SUM * y64.abs()).all()


@pytest.mark.parametrize("D", [40, 41, 8200, 2048])
def test_rows_with_values_that_are_not_finite_stay_by_themselves(D):
    x, _, w, _ = make((5, D), F, None)
    x[1, 3], x[2, D - 1], x[3] = float("nan"), float("inf"), 0
    with torch.no_grad():
        y = dwarf_b200.rms_norm(x, w)
        y8, s8 = dwarf_b200.rms_norm_e4m3(x, w)
    assert torch.isfinite(y[[0, 3, 4]]).all() and torch.isnan(y[1]).all() and (y[3] == 0).all()
    b = s8.view(torch.uint8).cpu().tolist()
    assert b[1] == 255 and b[2] == 255 and b[3] == 127 and b[0] < 255 and b[4] < 255
    assert torch.isnan(y8[1].float()).all() and torch.isfinite(y8[[0, 3, 4]].float()).all()


def test_scales_are_powers_of_two_chosen_by_the_largest_value():
    # eps = 0 and one column: y = sign(x) w, so w is the row's largest value
    for v in (448.0, 449.0, 447.9, 1.0, 1.75, 1.7500001, 3.4e38, 2.0 ** -100, 2.0 ** -126, 1e-45):
        x = torch.tensor([[4.0]], device=DEV)
        with torch.no_grad():
            y8, s8 = dwarf_b200.rms_norm_e4m3(x, torch.tensor([v], device=DEV), eps=0.0)
        val, s = quantize64(torch.tensor([[v]], dtype=torch.float32))
        assert float(scale_values(s8)) == float(s) and float(y8.float()) == float(val)


def test_odd_calls():
    x, r, w, _ = make((6, 256), BF, F)
    with torch.no_grad():
        want = dwarf_b200.rms_norm(x, w, r)
        strided = torch.stack([x, x], 1).view(6, 512)[:, :256]                    # rows 512 apart
        assert all(torch.equal(a, b) for a, b in zip(dwarf_b200.rms_norm(strided, w, r), want))
        odd = torch.empty(6 * 256 + 1, dtype=BF, device=DEV)[1:].view(6, 256).copy_(x)       # starts on 2 bytes
        assert all(torch.equal(a, b) for a, b in zip(dwarf_b200.rms_norm(odd, w, r), want))
        e = dwarf_b200.rms_norm(x[:0], w, r[:0])
        assert e[0].shape == (0, 256) and e[1].shape == (0, 256) and dwarf_b200.rms_norm_e4m3(x[:0], w)[1].shape == (0,)
        wb = w.to(BF)
        near(dwarf_b200.rms_norm(x, wb, r)[0], forward64(x, r, wb)[1], SUM * forward64(x, r, wb)[1].abs())
    assert dwarf_b200.rms_norm(x, w).dtype is BF and dwarf_b200.rms_norm(x, w, r)[0].dtype is F
    z = x[:0].detach().requires_grad_(True)
    wz = w.detach().clone().requires_grad_(True)
    dz, dwz = torch.autograd.grad(dwarf_b200.rms_norm(z, wz).float().sum(), [z, wz])
    assert dz.shape == (0, 256) and (dwz == 0).all()


def test_parts_of_the_gradient():
    x, r, w, g = make((37, 256), BF, F)
    dy, dh = torch.randn(37, 256, generator=g).to(DEV), torch.randn(37, 256, generator=g).to(DEV)
    full = [t.detach().clone().requires_grad_(True) for t in (x, r, w)]
    y, h = dwarf_b200.rms_norm(full[0], full[2], full[1])
    want = torch.autograd.grad([y, h], full, [dy, dh])
    for keep in ((0,), (1,), (2,), (0, 2), (1, 2)):
        ts = [t.detach().clone().requires_grad_(i in keep) for i, t in enumerate((x, r, w))]
        y, h = dwarf_b200.rms_norm(ts[0], ts[2], ts[1])
        got = torch.autograd.grad([y, h], [ts[i] for i in keep], [dy, dh])
        assert all(torch.equal(a, want[i]) for a, i in zip(got, keep))
    # only h, only y
    ts = [t.detach().clone().requires_grad_(True) for t in (x, r, w)]
    y, h = dwarf_b200.rms_norm(ts[0], ts[2], ts[1])
    dx, dr, dw = torch.autograd.grad(h, ts, dh, allow_unused=True, retain_graph=True)
    assert torch.equal(dr, dh) and torch.equal(dx, dh.to(BF)) and dw is None
    a = torch.autograd.grad(y, ts, dy, retain_graph=True)
    b = torch.autograd.grad([y, h], ts, [dy, torch.zeros_like(dh)])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # gradients are the caller's to change
    y, h = dwarf_b200.rms_norm(full[1], full[2], full[1].detach())
    y, h = dwarf_b200.rms_norm(full[1], full[2], full[1] * 1)
    g1 = torch.autograd.grad([y, h], [full[1]], [dy, dh])[0]
    assert torch.isfinite(g1.mul_(2)).all()


def test_large_offsets_and_repeatability():
    x, r, w, g = make((70001, 256), BF, BF, seed=11)
    dy = torch.randn(70001, 256, generator=g).to(BF).to(DEV)
    outs = []
    for _ in range(2):
        ts = [t.detach().clone().requires_grad_(True) for t in (x, r, w)]
        y, h = dwarf_b200.rms_norm(ts[0], ts[2], ts[1])
        outs.append([y, h, *torch.autograd.grad([y, h], ts, [dy, dy])])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    _, y64, _ = forward64(x[-3:], r[-3:], w)
    near(outs[0][0][-3:].detach(), y64, SUM * y64.abs())


def test_refusals():
    x, r, w, _ = make((6, 256), BF, F)
    for bad in (lambda: dwarf_b200.rms_norm(x, w[:8]), lambda: dwarf_b200.rms_norm(x, w, r[:3]), lambda: dwarf_b200.rms_norm(x, w.cpu()), lambda: dwarf_b200.rms_norm(x, w, r.cpu())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: dwarf_b200.rms_norm(x.half(), w), lambda: dwarf_b200.rms_norm(x, w, r.half()), lambda: dwarf_b200.rms_norm(x, w, out_dtype=torch.float16),
                lambda: dwarf_b200.rms_norm(x, w.to(torch.int32))):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        dwarf_b200.rms_norm_e4m3(x.detach().requires_grad_(True), w)
    t = x.detach().requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(dwarf_b200.rms_norm(t, w).float().sum(), t, create_graph=True)


def test_captured_and_replayed_on_another_stream():
    x, r, w, g = make((64, 256), BF, F)
    ts = [t.detach().clone().requires_grad_(True) for t in (x, r, w)]
    dy = torch.randn(64, 256, generator=g).to(DEV)

    def step():
        y, h = dwarf_b200.rms_norm(ts[0], ts[2], ts[1])
        return [y.detach(), *torch.autograd.grad([y, h], ts, [dy, dy])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        ts[0].mul_(-0.5)
    graph.replay()
    torch.cuda.synchronize()
    got = [o.clone() for o in out]
    del graph, out
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
