"""CPU tests of the operators around a decode step: what the C ABI refuses, the paged cache's bookkeeping, the packing of 4-bit weights."""
import ctypes

import pytest
import torch

import dwarf_b200
from dwarf_b200 import _lib
from dwarf_b200.build import build_library


@pytest.fixture(scope="module")
def lib():
    build_library()
    return _lib.load()


A = 4096           # a non-null, 16-byte aligned fake device address (never dereferenced)


def test_norm_refusals(lib):
    def fwd(**kw):
        f = dict(x=A, residual=2 * A, weight=3 * A, h=4 * A, y=5 * A, y_scale=6 * A, rstd=7 * A, rows=4, D=256, eps=1e-6, x_dtype=0, stream_dtype=1, y_dtype=2)
        p = _lib.RmsNorm(**{**f, **kw})
        return lib.dsqg_rms_norm_fwd(ctypes.byref(p), None)
    assert lib.dsqg_rms_norm_fwd(None, None) == -1
    for name in ("x", "weight", "y", "h", "y_scale"):
        assert fwd(**{name: None}) == -1, name
    assert fwd(rows=0) == -2 and fwd(D=0) == -2 and fwd(rows=1 << 40) == -2 and fwd(rows=1 << 30, D=1 << 20) == -2
    assert fwd(x_dtype=2) == -4 and fwd(stream_dtype=2) == -4 and fwd(y_dtype=3) == -4
    for name in ("x", "residual", "weight", "h", "y"):
        assert fwd(**{name: A + 8}) == -5, name

    def bwd(dy=8 * A, dh=9 * A, dx=10 * A, dr=11 * A, dw=12 * A, scratch=13 * A, nbytes=1 << 30, **kw):
        f = dict(x=A, residual=2 * A, weight=3 * A, h=4 * A, rstd=7 * A, rows=4, D=256, x_dtype=0, stream_dtype=1, y_dtype=0)
        p = _lib.RmsNorm(**{**f, **kw})
        return lib.dsqg_rms_norm_bwd(ctypes.byref(p), dy, dh, dx, dr, dw, scratch, nbytes, None)
    assert bwd(dy=None) == -1 and bwd(weight=None) == -1 and bwd(rstd=None) == -1 and bwd(h=None) == -1 and bwd(scratch=None) == -1
    assert bwd(dx=None, dr=None, dw=None) == -1 and bwd(residual=None, x=None) == -1
    assert bwd(y_dtype=2) == -4 and bwd(rows=0) == -2 and bwd(dy=A + 2) == -5 and bwd(dr=A + 4) == -5
    need = lib.dsqg_rms_norm_bwd_scratch_bytes(4, 256)
    assert need >= 256 * 4 and bwd(nbytes=need - 1) == -6
    assert lib.dsqg_rms_norm_bwd_scratch_bytes(0, 256) == 0


def _pages(**kw):
    f = dict(kv=A, scale=2 * A, table=3 * A, dtype=2, sequences=2, columns=4, pages=8, page_size=16, heads=2, D=64)
    return ctypes.byref(_lib.Pages(**{**f, **kw}))


def test_paged_refusals(lib):
    def write(k=4 * A, v=5 * A, strides=(128, 64, 128, 64), cu=6 * A, tokens=7, dtype=0, **kw):
        return lib.dsqg_paged_write(_pages(**kw), k, v, *strides, cu, None, tokens, dtype, None)
    assert lib.dsqg_paged_write(None, A, A, 8, 8, 8, 8, A, None, 1, 0, None) == -1
    for name in ("kv", "table", "scale"):
        assert write(**{name: None}) == -1, name
    assert write(k=None) == -1 and write(v=None) == -1 and write(cu=None) == -1
    for kw in (dict(D=12), dict(D=136), dict(D=0), dict(heads=0), dict(pages=0), dict(page_size=0), dict(columns=0), dict(sequences=0), dict(sequences=70000), dict(tokens=0),
               dict(columns=1 << 20, page_size=1 << 12), dict(pages=1 << 30, heads=60000, page_size=1 << 10, columns=1)):
        assert write(**kw) == -2, kw
    assert write(dtype=2) == -4
    assert lib.dsqg_paged_write(_pages(dtype=5), A, A, 8, 8, 8, 8, A, None, 1, 0, None) == -4
    assert write(k=A + 8) == -5 and write(strides=(4, 64, 128, 64)) == -5 and write(kv=A + 8) == -5 and write(scale=A + 1) == -5

    def read(k=4 * A, v=5 * A, cu=6 * A, tokens=7, dtype=0, **kw):
        return lib.dsqg_paged_read(_pages(**kw), k, v, cu, None, tokens, dtype, None)
    assert lib.dsqg_paged_read(None, A, A, A, None, 1, 0, None) == -1
    assert read(k=None) == -1 and read(cu=None) == -1 and read(tokens=0) == -2 and read(dtype=2) == -4 and read(v=A + 4) == -5 and read(D=20) == -2

    def step(q=4 * A, k=5 * A, v=6 * A, lengths=7 * A, heads=4, most=64, scale=0.0, out=8 * A, scratch=9 * A, nbytes=1 << 30, dtype=0, **kw):
        return lib.dsqg_paged_step(_pages(**kw), q, k, v, lengths, heads, most, scale, out, scratch, nbytes, dtype, None)
    for name in ("q", "lengths", "out", "k", "v"):
        assert step(**{name: None}) == -1, name                                  # k and v come together
    assert step(heads=3) == -2 and step(heads=1) == -2 and step(heads=0) == -2 and step(most=-1) == -2 and step(most=65) == -2       # 4 columns of 16
    assert step(scale=float("inf")) == -8 and step(scale=float("nan")) == -8 and step(dtype=2) == -4
    assert step(q=A + 8) == -5 and step(out=A + 2) == -5 and step(scratch=A + 4) == -5
    need = lib.dsqg_paged_step_scratch_bytes(2, 2, 4, 64, 4096)
    assert need > 0 and step(columns=256, most=4096, nbytes=need - 1) == -6 and step(columns=256, most=4096, scratch=None) == -1
    assert lib.dsqg_paged_step_scratch_bytes(2, 2, 4, 64, 16) == 0               # one part: nothing to join
    assert lib.dsqg_paged_step_scratch_bytes(0, 2, 4, 64, 16) == 0 and lib.dsqg_paged_step_scratch_bytes(2, 2, 3, 64, 1 << 20) == 0


def test_ring8_and_int4_refusals(lib):
    off = (ctypes.c_int32 * 3)(0, 1, 9)

    def dec(q=A, kv=4 * A, scale=5 * A, head=6 * A, R=10, S=2, H=2, D=32, dtype=0):
        return lib.dsqg_decode_kv_e4m3(q, 2 * A, 3 * A, kv, scale, head, None, 7 * A, None, None, off, 3, R, 8 * A, S, H, D, dtype, None, 0)
    assert dec(q=None) == -1 and dec(kv=None) == -1 and dec(scale=None) == -1 and dec(head=None) == -1
    assert dec(R=9) == -3 and dec(D=12) == -2 and dec(S=0) == -2 and dec(dtype=2) == -4 and dec(kv=A + 8) == -5 and dec(scale=A + 1) == -5

    def pre(k=A, scale=4 * A, N=5, D=32, R=10, dtype=0, S=2):
        return lib.dsqg_ring_prefill_e4m3(k, 2 * A, 3 * A, scale, 5 * A, 6 * A, S, 2, N, D, R, dtype, None)
    assert pre(k=None) == -1 and pre(scale=None) == -1 and pre(N=0) == -2 and pre(D=12) == -2 and pre(R=0) == -2 and pre(dtype=2) == -4 and pre(k=A + 8) == -5
    deq = lambda x=A, out=3 * A, rows=4, D=32, dtype=0: lib.dsqg_dequantize_rows(x, 2 * A, out, rows, D, dtype, None)  # noqa: E731
    assert deq(x=None) == -1 and deq(rows=0) == -2 and deq(D=12) == -2 and deq(dtype=2) == -4 and deq(out=A + 8) == -5

    def lin(x=A, xs=None, w=2 * A, s=3 * A, y=4 * A, M=1, N=16, K=256, group=32, dtype=0):
        return lib.dsqg_int4_linear(x, xs, w, s, None, y, M, N, K, group, dtype, None)
    assert lin(x=None) == -1 and lin(w=None) == -1 and lin(s=None) == -1 and lin(y=None) == -1 and lin(dtype=2) == -1
    assert lin(dtype=1) == -4 and lin(group=16) == -8 and lin(group=256) == -8 and lin(K=48) == -2 and lin(K=96, group=64) == -2
    assert lin(M=0) == -2 and lin(N=0) == -2 and lin(x=A + 8) == -5 and lin(w=A + 4) == -5


def test_python_refusals_without_a_gpu():
    t = torch.zeros
    with pytest.raises(RuntimeError):
        dwarf_b200.rms_norm(t(2, 8), t(8))
    with pytest.raises(RuntimeError):
        dwarf_b200.rms_norm_e4m3(t(2, 8), t(8))
    with pytest.raises(RuntimeError):
        dwarf_b200.int4_linear(t(2, 32, dtype=torch.bfloat16), t(4, 16, dtype=torch.uint8), t(4, 1, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        dwarf_b200.paged_kv_write(t(2, 1, 8), t(2, 1, 8), t(1, 1, 16, 2, 8), t(1, 1, dtype=torch.int32), t(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        dwarf_b200.DSQGRingCache(1, 1, 1, 32, dtype=torch.float8_e4m3fn, device="cpu", interleaved=False)
    with pytest.raises(ValueError):
        dwarf_b200.quantize_int4(t(4, 48), 32)
    with pytest.raises(ValueError):
        dwarf_b200.Int4Linear(100, 8)
    with pytest.raises(ValueError):
        dwarf_b200.PagedKVCache(1, 0, 1, 32, 10, device="cpu")
    with pytest.raises(TypeError):
        dwarf_b200.PagedKVCache(1, 1, 1, 32, 10, dtype=torch.float16, device="cpu")


def test_paged_cache_bookkeeping():
    c = dwarf_b200.PagedKVCache(1, 3, 1, 8, max_length=40, pages=7, page_size=16, device="cpu")
    assert tuple(c.block_table.shape) == (3, 3) and c.step_dtype is torch.bfloat16
    cu, start, tokens = c.extend([20, 0, 16])
    assert cu.tolist() == [0, 20, 20, 36] and start.tolist() == [0, 0, 0] and tokens == 36 and c.lengths.tolist() == [20, 0, 16]
    used = [p for row in c.block_table.tolist() for p in row if p >= 0]
    assert len(used) == 3 == len(set(used)) and c.block_table[1].tolist() == [-1, -1, -1]
    c.advance()                                                  # the empty slot stays empty; sequence 2 crosses into a new page
    assert c.lengths.tolist() == [21, 0, 17] and (c.block_table[2] >= 0).sum() == 2
    cu, start, tokens = c.extend([0, 33, 0])
    assert start.tolist() == [21, 0, 17] and c.lengths.tolist() == [21, 33, 17]
    before = c.block_table.clone()
    with pytest.raises(RuntimeError):                            # 7 pages: none left
        c.reserve(0, 40)
    with pytest.raises(ValueError):
        c.reserve(0, 41)
    with pytest.raises(ValueError):
        c.extend([1, 2])
    assert torch.equal(before, c.block_table) and c.lengths.tolist() == [21, 33, 17]
    c.release(1)
    assert c.lengths.tolist() == [21, 0, 17] and c.block_table[1].tolist() == [-1, -1, -1]
    c.reserve(0, 40)
    used = [p for row in c.block_table.tolist() for p in row if p >= 0]
    assert len(used) == len(set(used)) == 5 and all(0 <= p < 7 for p in used)
    e = dwarf_b200.PagedKVCache(2, 1, 1, 8, max_length=5, dtype=torch.float8_e4m3fn, device="cpu")
    assert e.kv.dtype is torch.float8_e4m3fn and e.kv_scale.shape == e.kv.shape[:-1] and e.kv_scale.dtype is torch.float8_e8m0fnu


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_int4_packs_the_nearest_of_sixteen_values(group):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(5, 256, generator=g)
    w[0, :group] = 0.0
    w[1, 0] = -9.0
    packed, scales = dwarf_b200.quantize_int4(w, group)
    assert packed.shape == (5, 128) and scales.shape == (5, 256 // group) and scales.dtype is torch.bfloat16
    nib = torch.stack([packed & 15, packed >> 4], -1).flatten(1).double() - 8
    s = scales.double().repeat_interleave(group, 1)
    back = nib * s
    # half a step; at the ends the scale's own rounding to bf16 (2^-8) may leave up to 8 * 2^-8 steps more
    assert ((back - w.double()).abs() <= s * (0.5 + 8 * 2.0 ** -8)).all()
    assert (back[0, :group] == 0).all() and (nib[0, :group] == 0).all()
    m = dwarf_b200.Int4Linear.from_linear(torch.nn.Linear(256, 5), group)
    assert m.half().scales.dtype is torch.bfloat16 and m.weight.dtype is torch.uint8 and m.bias.dtype is torch.float32
    n = dwarf_b200.Int4Linear(256, 5, group=group)
    n.load_state_dict(m.state_dict())
    assert torch.equal(n.weight, m.weight)


def test_int4_linear_keeps_its_values_through_casts():
    g = torch.Generator().manual_seed(0)
    lin = torch.nn.Linear(64, 5)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(5, 64, generator=g) * 1e6)
        lin.bias.copy_(torch.randn(5, generator=g))
    m = dwarf_b200.Int4Linear.from_linear(lin, 32)
    before = {n: b.clone() for n, b in m.named_buffers()}
    m.to(torch.bfloat16).half().float().double()
    for n, b in m.named_buffers():
        assert b.dtype == before[n].dtype and torch.equal(b, before[n])


def test_sizes_next_to_the_last_int_are_refused(lib):
    """A row's index arithmetic goes a little beyond its sizes: what would leave an int is not launched."""
    f = dict(x=A, residual=None, weight=3 * A, y=5 * A, rstd=7 * A, rows=1, eps=1e-6, x_dtype=0, stream_dtype=0, y_dtype=0)
    for D in (2 ** 31 - 1, 2 ** 31 - 8, 0x7ffff001):
        p = _lib.RmsNorm(**f, D=D)
        assert lib.dsqg_rms_norm_fwd(ctypes.byref(p), None) == -2
        assert lib.dsqg_rms_norm_bwd(ctypes.byref(p), 8 * A, None, 9 * A, None, None, None, 0, None) == -2
        assert lib.dsqg_rms_norm_bwd_scratch_bytes(1, D) == 0
    assert lib.dsqg_rms_norm_bwd_scratch_bytes(1, 0x7ffff000) > 0
    for N, K in ((2 ** 31 - 1, 32), (0x7fffff01, 32), (16, 2 ** 31 - 32), (16, 0x7fffc020)):
        assert lib.dsqg_int4_linear(A, None, 2 * A, 3 * A, None, 4 * A, 1, N, K, 32, 0, None) == -2


def test_quantize_weights_changes_nothing_when_a_width_does_not_fit():
    from dwarf_b200.model import CondMLM
    m = CondMLM(vocab=11, dim=128, heads=2, layers=2, ffn=192, seq_len=32, full_attention_layer=1, offsets=(0, 1, 2))
    before = dict(m.named_modules())
    with pytest.raises(ValueError):
        m.quantize_weights(128)                                   # fc2 has 192 columns
    after = dict(m.named_modules())
    assert before.keys() == after.keys() and all(after[n] is before[n] for n in before)
    m.quantize_weights(64)
    assert sum(type(x) is dwarf_b200.Int4Linear for x in m.modules()) == 2 * 2 + 3 + 2
