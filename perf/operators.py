"""The operators of a quantised decode step (and of the norms of a training step): what is measured, and what each computes.

A case is a dict of plain values with a "kind":

  norm        `rms_norm` with the residual's addition, forward and backward (training)
  norm8       `rms_norm_e4m3`: the same norm with its output in 8 bits and a scale per row (serving)
  ring8       `dsqg_decode_step_kv` over a ring in 8 bits: one token of one DSQG layer
  write       `paged_kv_write`: the keys and values of a batch of prompts into a paged cache
  read        `paged_kv_read`: the rows of a paged cache back in token order
  step        `paged_attention_step`: one new token per sequence against a paged cache
  int4        `int4_linear`: a projection with 4-bit weights and group scales

8-bit rows are e4m3 with one scale per row, the smallest power of two 2^e with max|row| <= 448 * 2^e (-126 <= e; 1 for a row of zeros), held as
float8_e8m0fnu.  4-bit weights are w[n, k] = (nibble - 8) * scales[n, k // group], the nibble of an even k in the low half of its byte.

Lengths of sequences come from the case alone (`_lengths`), everything else from the seed.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
# dense 0..31 and eleven sparse taps: the 43-offset set of the decode benchmark; a ring of 1537 slots
_OFFSETS = tuple(range(32)) + (48, 64, 96, 128, 192, 256, 384, 512, 768, 1024, 1536)
_EPS = 1e-6


def listed():
    return [
        # norm of one token of four sequences in front of 4-bit projections: nothing but latency
        dict(kind="norm8", rows=4, D=256, x="bf16", stream="fp32", name="norm8 4x256"),
        # a training step of the 13M model (32 x 2048 tokens, width 256): bf16 branch onto an fp32 residual stream, under autocast
        dict(kind="norm", rows=65536, D=256, x="bf16", stream="fp32", y="bf16", name="norm train 65536x256"),
        # a bf16 stream, an odd number of rows, a width that fills no power of two
        dict(kind="norm", rows=4099, D=1000, x="bf16", stream="bf16", y="bf16", name="norm train 4099x1000"),
        # one DSQG layer of the decode benchmark (256 sequences, 12 heads of 64, full rings), rings in 8 bits
        dict(kind="ring8", S=256, H=12, D=64, prompt=0, name="ring8 256x12x64"),
        # eight ragged prompts of up to 2048 tokens into 8-bit pages
        dict(kind="write", S=8, most=2048, H=12, D=64, page=64, pages="e4m3", dtype="bf16", len_seed=1, name="write8 8x2048x12x64"),
        # and back in bf16 (a chunked prompt, a cache handed to another server)
        dict(kind="read", S=8, most=2048, H=12, D=64, page=64, pages="e4m3", dtype="bf16", len_seed=1, name="read8 8x2048x12x64"),
        # a few sequences just after short prompts: the full-attention layer of the 13M model
        dict(kind="step", S=3, most=45, H=8, G=1, D=32, page=16, pages="bf16", len_seed=2, name="step 3x45 8x32"),
        # a serving batch of ragged sequences, grouped heads
        dict(kind="step", S=64, most=4096, H=8, G=4, D=128, page=64, pages="bf16", len_seed=3, name="step 64x4096 8x4x128"),
        # few long sequences in 8 bits
        dict(kind="step", S=4, most=100001, H=4, G=8, D=128, page=128, pages="e4m3", len_seed=4, name="step8 4x100001 4x8x128"),
        # the qkv projection of the 13M model for one token
        dict(kind="int4", M=1, K=256, N=768, group=32, x="bf16", bias=True, name="int4 1x256x768"),
        # one token through a large projection: weights only
        dict(kind="int4", M=1, K=4096, N=16384, group=128, x="bf16", bias=False, name="int4 1x4096x16384"),
        # sixteen sequences, activations in 8 bits from the norm
        dict(kind="int4", M=16, K=8192, N=8192, group=64, x="e4m3", bias=True, name="int4 16x8192x8192"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm8", "ring8", "write", "read", "step", "step", "step", "int4", "int4", "int4"])
    seed = rng.randrange(1 << 20)
    if kind in ("norm", "norm8"):
        D = 8 * _log_uniform(rng, 8, 1024) if rng.random() < 0.85 else _log_uniform(rng, 1, 2000)
        rows = _log_uniform(rng, 1, max(1, min(65536, 16_000_000 // D)))
        c = dict(kind=kind, rows=rows, D=D, x=rng.choice(["bf16", "bf16", "fp32"]), stream=rng.choice(["bf16", "fp32"]))
        return {**c, "y": rng.choice(["bf16", "bf16", "fp32"])} if kind == "norm" else c
    if kind == "ring8":
        return dict(kind=kind, S=_log_uniform(rng, 1, 256), H=rng.choice([1, 8, 12]), D=rng.choice([32, 48, 64, 128]) if rng.random() < 0.5 else 64,
                    prompt=rng.choice([0, 0, rng.randint(1, 2000)]))
    if kind in ("write", "read"):
        return dict(kind=kind, S=_log_uniform(rng, 1, 16), most=_log_uniform(rng, 1, 1500), H=rng.choice([1, 2, 8, 12]), D=rng.choice([32, 40, 64, 64, 80, 128]),
                    page=rng.choice([16, 48, 64, 128, 256]), pages=rng.choice(["e4m3", "e4m3", "bf16", "fp32"]), dtype=rng.choice(["bf16", "bf16", "fp32"]), len_seed=seed)
    if kind == "step":
        pages = rng.choice(["bf16", "bf16", "e4m3", "e4m3", "fp32"])
        H, G, D = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 3, 4, 8, 12]), rng.choice([32, 64, 64, 80, 96, 128, 128])
        size = {"bf16": 2, "e4m3": 1, "fp32": 4}[pages]
        room = (300_000_000 if pages != "fp32" and D % 32 == 0 else 20_000_000) // (H * 2 * D * size)
        S = _log_uniform(rng, 1, 64)
        return dict(kind=kind, S=S, most=_log_uniform(rng, 1, min(100_000, max(2, room // S))), H=H, G=G, D=D, page=rng.choice([16, 32, 48, 64, 256]),
                    pages=pages, len_seed=seed)
    group = rng.choice([32, 64, 128])
    K = group * _log_uniform(rng, 1, 8192 // group)
    return dict(kind=kind, M=_log_uniform(rng, 1, 16), K=K, N=_log_uniform(rng, 17, max(17, min(16384, 60_000_000 // K))), group=group,
                x=rng.choice(["bf16", "e4m3"]), bias=rng.random() < 0.5)


def _lengths(c):
    """The lengths of the sequences: one of the longest, the others spread from nothing (a slot of the batch that waits) up to it."""
    r = np.random.RandomState(c["len_seed"])
    n = r.randint(0, c["most"] + 1, c["S"])
    n[r.randint(c["S"])] = c["most"]
    return [int(v) for v in n]


# ---- 8 and 4 bits, in elementary operations

def _row_scale(x):
    """[..., D] fp32 -> [..., 1] fp32: the smallest power of two s >= 2^-126 with max|row| <= 448 s, 1 for a row of zeros."""
    top = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)                                     # top = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-126, 127)
    return torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), torch.ones_like(top))


def _quantize(x):
    """Rows of x as (e4m3, float8_e8m0fnu scale)."""
    x = x.float()
    s = _row_scale(x)
    return (x / s).to(torch.float8_e4m3fn), _e8m0(s.squeeze(-1))


def _e8m0(s):
    # a power of two from 2^-126 on: its exponent field
    return (s.contiguous().view(torch.int32) >> 23).to(torch.uint8).view(torch.float8_e8m0fnu)


def _scale_of(s8):
    return torch.ldexp(torch.ones(s8.shape, device=s8.device), s8.view(torch.uint8).to(torch.int32) - 127)


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float() - 8.0


# ---- inputs

def _pages(c, g, lengths, filled):
    """A cache whose sequences own pages in shuffled order.  filled: rows as a model leaves them; else uninitialised memory (zeros here)."""
    S, H, D, page = c["S"], c["H"], c["D"], c["page"]
    per = [-(-n // page) for n in lengths]
    most, total = max(1, max(per)), max(1, sum(per))
    P = total + 1 + total // 16
    order = torch.randperm(P, generator=g, device="cuda")[:total].to(torch.int32)
    table = torch.zeros(S, most, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = order[at:at + n]
        at += n
    st = {"table": table, "kv_scale": None}
    dt = _DTYPES[c["pages"]]
    if not filled:
        st["kv"] = torch.zeros(P, H, page, 2, D, dtype=torch.uint8 if dt.itemsize == 1 else dt, device="cuda").view(dt)
        if dt.itemsize == 1:
            st["kv_scale"] = torch.zeros(P, H, page, 2, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    elif dt.itemsize == 1:
        st["kv"], st["kv_scale"] = _quantize(torch.randn(P, H, page, 2, D, generator=g, device="cuda", dtype=torch.bfloat16))
    else:
        st["kv"] = torch.randn(P, H, page, 2, D, generator=g, device="cuda", dtype=dt)
    return st


def prepare(case, seed):
    c, kind = case, case["kind"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape, std=1.0, dt=torch.float32: torch.randn(*shape, generator=g, device="cuda", dtype=dt) * std  # noqa: E731
    st = {"case": c}
    if kind in ("norm", "norm8"):
        grad = kind == "norm"
        rows, D = c["rows"], c["D"]
        st["x"] = rand(rows, D, std=0.5, dt=_DTYPES[c["x"]]).requires_grad_(grad)
        st["residual"] = rand(rows, D, dt=_DTYPES[c["stream"]]).requires_grad_(grad)
        st["weight"] = (1.0 + rand(D, std=0.1)).requires_grad_(grad)
        if grad:
            st["dy"], st["dh"] = rand(rows, D, dt=_DTYPES[c["y"]]), rand(rows, D, dt=_DTYPES[c["stream"]])
        return st
    if kind == "ring8":
        S, H, D, R = c["S"], c["H"], c["D"], _OFFSETS[-1] + 1
        kv, kv_scale = _quantize(rand(S, H, R, 2, D, dt=torch.bfloat16))
        n = c["prompt"]
        head = torch.randint(0, R, (S,), generator=g, device="cuda", dtype=torch.int32) if not n else torch.full((S,), n % R, dtype=torch.int32, device="cuda")
        fill = torch.full((S,), min(n + 1, R) if n else R, dtype=torch.int32, device="cuda")
        slope = torch.linspace(0.2, 2.0, H, device="cuda")
        bias = -torch.log1p(torch.tensor(_OFFSETS, device="cuda", dtype=torch.float32))[:, None] * slope + rand(len(_OFFSETS), H, std=0.05)
        return {**st, "kv": kv, "kv_scale": kv_scale, "head": head, "fill": fill, "bias": bias, "gain": torch.rand(H, generator=g, device="cuda") * 0.4 + 0.8,
                "qkv": [rand(S, H, D, dt=torch.bfloat16) for _ in range(3)]}
    if kind in ("write", "read", "step"):
        lengths = _lengths(c)
        st.update(_pages(c, g, lengths, kind != "write"))
        if kind == "step":
            dt = torch.float32 if c["pages"] == "fp32" else torch.bfloat16
            S, H, G, D = c["S"], c["H"], c["G"], c["D"]
            st.update(lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), q=rand(S, H * G, D, dt=dt), k=rand(S, H, D, dt=dt), v=rand(S, H, D, dt=dt))
            return st
        st.update(cu=torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda"), tokens=sum(lengths))
        if kind == "write":
            dt = _DTYPES[c["dtype"]]
            # a fused projection's key and value columns: token rows 2 H D apart
            kv = rand(max(1, st["tokens"]), 2, c["H"], c["D"], dt=dt)[:st["tokens"]]
            st.update(k=kv[:, 0], v=kv[:, 1])
        return st
    M, K, N, G = c["M"], c["K"], c["N"], c["group"]
    st["weight"] = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    st["scales"] = (0.002 + 0.01 * torch.rand(N, K // G, generator=g, device="cuda")).to(torch.bfloat16)
    st["bias"] = rand(N, std=0.02) if c["bias"] else None
    x = rand(M, K, dt=torch.bfloat16)
    st["x"], st["x_scale"] = _quantize(x) if c["x"] == "e4m3" else (x, None)
    return st


# ---- one pass

def run(st):
    c = st["case"]
    kind = c["kind"]
    if own:
        import dwarf_b200 as d
        if kind == "norm":
            y, h = d.rms_norm(st["x"], st["weight"], st["residual"], eps=_EPS, out_dtype=_DTYPES[c["y"]])
            dx, dr, dw = torch.autograd.grad([y, h], [st["x"], st["residual"], st["weight"]], [st["dy"], st["dh"]])
            return {"y": y.detach(), "h": h.detach(), "dx": dx, "dr": dr, "dw": dw}
        if kind == "norm8":
            y, s, h = d.rms_norm_e4m3(st["x"], st["weight"], st["residual"], eps=_EPS)
            return {"y": y, "scale": s, "h": h}
        if kind == "ring8":
            out = d.dsqg_decode_step_kv(*st["qkv"], st["kv"], st["head"], st["bias"], st["gain"], None, _OFFSETS, st["fill"], kv_scale=st["kv_scale"])
            return {"out": out, "kv": st["kv"], "kv_scale": st["kv_scale"]}
        if kind == "write":
            d.paged_kv_write(st["k"], st["v"], st["kv"], st["table"], st["cu"], kv_scale=st["kv_scale"])
            return {"kv": st["kv"], "kv_scale": st["kv_scale"]}
        if kind == "read":
            k, v = d.paged_kv_read(st["kv"], st["table"], st["cu"], st["tokens"], kv_scale=st["kv_scale"], dtype=_DTYPES[c["dtype"]])
            return {"k": k, "v": v}
        if kind == "step":
            out = d.paged_attention_step(st["q"], st["k"], st["v"], st["kv"], st["table"], st["lengths"], kv_scale=st["kv_scale"], max_length=c["most"])
            return {"out": out, "kv": st["kv"], "kv_scale": st["kv_scale"]}
        return d.int4_linear(st["x"], st["weight"], st["scales"], st["bias"], x_scale=st["x_scale"])
    with torch.no_grad():
        return {"norm": _norm, "norm8": _norm8, "ring8": _ring8, "write": _write, "read": _read, "step": _step, "int4": _int4}[kind](st)


def _normed(st):
    h = (st["x"].float() + st["residual"].float()).to(st["residual"].dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.square().mean(-1, keepdim=True) + _EPS)
    return h, hf * rstd, rstd


def _norm(st):
    h, xh, rstd = _normed(st)
    w, dy = st["weight"], st["dy"].float()
    g = dy * w
    dh = st["dh"].float() + rstd * (g - xh * (g * xh).mean(-1, keepdim=True))
    return {"y": (xh * w).to(st["dy"].dtype), "h": h, "dx": dh.to(st["x"].dtype), "dr": dh.to(st["residual"].dtype), "dw": (dy * xh).sum(0)}


def _norm8(st):
    h, xh, _ = _normed(st)
    y, s = _quantize(xh * st["weight"])
    return {"y": y, "scale": s, "h": h}


def _bytes(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _ring8(st):
    q, k, v = st["qkv"]
    kv, ks = st["kv"], st["kv_scale"]
    S, H, R, _, D = kv.shape
    s_at, h_at = torch.arange(S, device="cuda")[:, None], torch.arange(H, device="cuda")[None]
    head = st["head"].long()
    new, new_s = _quantize(torch.stack([k, v], 2))                                    # the step attends to what the ring holds
    _bytes(kv)[s_at, h_at, head[:, None]] = _bytes(new)
    _bytes(ks)[s_at, h_at, head[:, None]] = _bytes(new_s)
    off = torch.tensor(_OFFSETS, device="cuda")
    slots = (head[:, None] - off) % R                                                 # [S, J]
    at = (s_at[..., None], h_at[..., None], slots[:, None])
    rows = _bytes(kv)[at].view(kv.dtype).float() * _scale_of(_bytes(ks)[at])[..., None]   # [S, H, J, 2, D]
    score = (q.float()[:, :, None] * rows[..., 0, :]).sum(-1) / math.sqrt(D) + st["bias"].t()
    score = score.masked_fill((off >= st["fill"].long()[:, None])[:, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p[..., None] * rows[..., 1, :]).sum(2) / p.sum(-1, keepdim=True) * st["gain"][:, None]
    return {"out": out.to(q.dtype), "kv": kv, "kv_scale": ks}


def _places(st, tokens):
    """(page, row in it) of every token of a ragged batch."""
    page = st["case"]["page"]
    t = torch.arange(tokens, device="cuda")
    cu = st["cu"].long()
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos = t - cu[seq]
    return st["table"].long()[seq, pos // page], pos % page


def _write(st):
    kv, ks = st["kv"], st["kv_scale"]
    pages, rows = _places(st, st["tokens"])
    new = torch.stack([st["k"], st["v"]], 2)                                          # [T, H, 2, D]
    if ks is None:
        kv[pages, :, rows] = new.to(kv.dtype)
    else:
        new, s = _quantize(new)
        _bytes(kv)[pages, :, rows] = _bytes(new)
        _bytes(ks)[pages, :, rows] = _bytes(s)
    return {"kv": kv, "kv_scale": ks}


def _read(st):
    pages, rows = _places(st, st["tokens"])
    got = _bytes(st["kv"])[pages, :, rows].view(st["kv"].dtype).float()
    if st["kv_scale"] is not None:
        got = got * _scale_of(_bytes(st["kv_scale"])[pages, :, rows])[..., None]
    dt = _DTYPES[st["case"]["dtype"]]
    return {"k": got[:, :, 0].to(dt), "v": got[:, :, 1].to(dt)}


def _step(st):
    c = st["case"]
    S, H, G, D, page = c["S"], c["H"], c["G"], c["D"], c["page"]
    kv, ks, n = st["kv"], st["kv_scale"], st["lengths"].long()
    new, new_s = _quantize(torch.stack([st["k"], st["v"]], 2)) if ks is not None else (torch.stack([st["k"], st["v"]], 2).to(kv.dtype), None)
    live = torch.nonzero(n > 0).squeeze(-1)
    last = n[live] - 1
    at = (st["table"].long()[live, last // page], slice(None), last % page)
    _bytes(kv)[at] = _bytes(new)[live]
    if ks is not None:
        _bytes(ks)[at] = _bytes(new_s)[live]
    table = st["table"].long()
    rows = _bytes(kv)[table].view(kv.dtype).float()                                   # [S, pages, H, page, 2, D]
    if ks is not None:
        rows = rows * _scale_of(_bytes(ks)[table])[..., None]
    rows = rows.transpose(1, 2).reshape(S, H, table.shape[1] * page, 2, D)
    q = st["q"].float().view(S, H, G, D)
    score = torch.matmul(q, rows[..., 0, :].transpose(-1, -2)) / math.sqrt(D)
    gone = torch.arange(rows.shape[2], device="cuda") >= n[:, None]
    score = score.masked_fill(gone[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    out = torch.matmul(p, rows[..., 1, :]) / p.sum(-1, keepdim=True).clamp_min(1e-30)   # nothing to attend to: zeros
    return {"out": out.view(S, H * G, D).to(st["q"].dtype), "kv": kv, "kv_scale": ks}


def _int4(st):
    N, K = st["weight"].shape[0], st["weight"].shape[1] * 2
    G = K // st["scales"].shape[1]
    w = (_unpack(st["weight"]).view(N, K // G, G) * st["scales"].float()[..., None]).view(N, K)
    x = st["x"].float() if st["x_scale"] is None else st["x"].float() * _scale_of(st["x_scale"])[:, None]
    y = torch.matmul(x, w.t())
    return (y if st["bias"] is None else y + st["bias"]).to(torch.bfloat16)


# ---- the definition in 64 bits, row by row

def _held(row):
    """What an e4m3 row with a power-of-two scale holds of `row` (float64 [..., D]): (the e4m3 values, the scales)."""
    top = row.abs().amax(-1)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 448.0))
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e)).clamp(min=-126)
    s = torch.where(top > 0, torch.exp2(e), torch.ones_like(top))
    v = row / s[..., None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)      # three bits behind the leading one, 2^-9 below 2^-6
    return torch.round(v / step) * step, s


def _softmax_rows(q, k, v, scale, bias=0.0):
    s = k @ q * scale + bias
    p = torch.exp(s - s.max())
    return (p @ v) / p.sum()


def exact(case, seed):
    c, kind = case, case["kind"]
    st = prepare(case, seed)
    f = lambda t: t.detach().double()  # noqa: E731
    power = lambda s8: torch.exp2(s8.view(torch.uint8).double() - 127.0)  # noqa: E731
    if kind in ("norm", "norm8"):
        h = (f(st["x"]) + f(st["residual"])).to(st["residual"].dtype)
        n = torch.linalg.vector_norm(f(h), dim=1, keepdim=True)
        r = 1.0 / torch.sqrt(n * n / c["D"] + _EPS)
        w = f(st["weight"])
        y = f(h) * r * w
        if kind == "norm8":
            y8, s = _held(y)
            return {"y": y8, "scale": s, "h": f(h)}
        dy = f(st["dy"])
        # d/dh of sum(dy y): y = w h r(h), dr/dh = -r^3 h / D
        dh = f(st["dh"]) + w * dy * r - f(h) * r ** 3 * (w * dy * f(h)).sum(1, keepdim=True) / c["D"]
        return {"y": y, "h": f(h), "dx": dh, "dr": dh, "dw": torch.einsum("nd,nd,n->d", dy, f(h), r[:, 0])}
    if kind == "ring8":
        S, H, D = c["S"], c["H"], c["D"]
        q, k, v = (f(t) for t in st["qkv"])
        head, fill, R = st["head"].tolist(), st["fill"].tolist(), _OFFSETS[-1] + 1
        out = torch.zeros(S, H, D, dtype=torch.float64, device="cuda")
        off = torch.tensor(_OFFSETS, device="cuda")
        (k8, ks), (v8, vs) = _held(k), _held(v)
        bias, scale = f(st["bias"]), power(st["kv_scale"])
        for s in range(S):
            taps = off[off < fill[s]]
            at = (head[s] - taps) % R
            rows = f(st["kv"][s].view(torch.uint8)[:, at].view(torch.float8_e4m3fn)) * scale[s][:, at][..., None]     # [H, taps, 2, D]
            rows[:, 0] = torch.stack([k8[s] * ks[s][:, None], v8[s] * vs[s][:, None]], 1)                             # offset 0: the new token
            sc = torch.einsum("hd,hjd->hj", q[s], rows[:, :, 0]) / math.sqrt(D) + bias[:len(taps)].t()
            out[s] = torch.einsum("hj,hjd->hd", torch.softmax(sc, 1), rows[:, :, 1]) * f(st["gain"])[:, None]
        return {"out": out, "kv": None, "kv_scale": None}
    if kind == "write":
        table, page, k, v = st["table"].tolist(), c["page"], f(st["k"]), f(st["v"])
        kv = torch.zeros(st["kv"].shape, dtype=torch.float64, device="cuda")
        scale = power(st["kv_scale"]) if st["kv_scale"] is not None else None
        first = 0
        for s, n in enumerate(_lengths(c)):
            for p in range(-(-n // page)):
                i, m = table[s][p], min(page, n - p * page)
                rows = torch.stack([k[first:first + m], v[first:first + m]], 2).transpose(0, 1)
                if scale is None:
                    kv[i, :, :m] = rows
                else:
                    kv[i, :, :m], scale[i, :, :m] = _held(rows)
                first += m
        return {"kv": kv, "kv_scale": scale}
    if kind == "read":
        table, page = st["table"].tolist(), c["page"]
        ks, vs = [], []
        for s, n in enumerate(_lengths(c)):
            for p in range(-(-n // page)):
                i, m = table[s][p], min(page, n - p * page)
                rows = f(st["kv"][i, :, :m])
                rows = rows if st["kv_scale"] is None else rows * power(st["kv_scale"][i, :, :m])[..., None]
                ks.append(rows[:, :, 0].transpose(0, 1)), vs.append(rows[:, :, 1].transpose(0, 1))
        return {"k": torch.cat(ks), "v": torch.cat(vs)} if ks else None
    if kind == "step":
        S, H, G, D, page = c["S"], c["H"], c["G"], c["D"], c["page"]
        out = torch.zeros(S, H * G, D, dtype=torch.float64, device="cuda")
        table, q = st["table"].long(), f(st["q"])
        hold = lambda t: (lambda a, b: a * b[..., None])(*_held(f(t))) if st["kv_scale"] is not None else f(t)  # noqa: E731
        kn, vn = hold(st["k"]), hold(st["v"])
        for s, n in enumerate(_lengths(c)):
            for h in range(H if n else 0):
                old = table[s, :-(-n // page)]
                rows = f(st["kv"].view(torch.uint8)[old, h].view(torch.float8_e4m3fn) if c["pages"] == "e4m3" else st["kv"][old, h])
                if st["kv_scale"] is not None:
                    rows = rows * power(st["kv_scale"].view(torch.uint8)[old, h])[..., None]
                rows = rows.reshape(-1, 2, D)[:n]
                rows[n - 1, 0], rows[n - 1, 1] = kn[s, h], vn[s, h]
                for g in range(G):
                    out[s, h * G + g] = _softmax_rows(q[s, h * G + g], rows[:, 0], rows[:, 1], 1.0 / math.sqrt(D))
        return {"out": out, "kv": None, "kv_scale": None}
    x = f(st["x"]) if st["x_scale"] is None else f(st["x"]) * power(st["x_scale"])[:, None]
    b, K = st["weight"].to(torch.int16), c["K"]
    w = torch.empty(c["N"], K, dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = (b % 16 - 8).double(), (b // 16 - 8).double()
    y = x @ (w * f(st["scales"]).repeat_interleave(c["group"], 1)).t()
    return y if st["bias"] is None else y + f(st["bias"])


def work(case):
    """Inputs once, outputs once; a cache counts for the rows that the pass reads or writes."""
    c, kind = case, case["kind"]
    size = {"bf16": 2, "fp32": 4, "e4m3": 1}
    if kind in ("norm", "norm8"):
        n = c["rows"] * c["D"]
        if kind == "norm8":
            return {"bytes": n * (size[c["x"]] + 2 * size[c["stream"]] + 1) + c["rows"] + 4 * c["D"], "flops": 6 * n}
        # x, residual, dy, dh in; y, h, dx and the residual's gradient out
        return {"bytes": n * (2 * size[c["x"]] + 4 * size[c["stream"]] + 2 * size[c["y"]]) + 8 * c["D"], "flops": 16 * n}
    if kind == "ring8":
        pairs, D = c["S"] * c["H"], c["D"]
        fill = min(c["prompt"] + 1, _OFFSETS[-1] + 1) if c["prompt"] else _OFFSETS[-1] + 1
        taps = sum(o < fill for o in _OFFSETS)
        # key and value rows of the older taps and the new slot with their scales; q, k, v in and the result out in bf16
        return {"bytes": pairs * (taps * 2 * (D + 1) + 4 * 2 * D) + (len(_OFFSETS) + 1) * c["H"] * 4 + c["S"] * 8, "flops": pairs * taps * 4 * D}
    H, D = c.get("H"), c.get("D")
    if kind in ("write", "read", "step"):
        n, row = sum(_lengths(c)), 2 * H * (D * size[c["pages"]] + (c["pages"] == "e4m3"))
        if kind == "step":
            s = size["fp32" if c["pages"] == "fp32" else "bf16"]
            return {"bytes": n * row + c["S"] * (2 * H * c["G"] + 2 * H) * D * s + sum(-(-v // c["page"]) for v in _lengths(c)) * 4, "flops": n * H * c["G"] * 4 * D}
        return {"bytes": max(1, n * (row + 2 * H * D * size[c["dtype"]])), "flops": n * 2 * H * D}
    M, K, N = c["M"], c["K"], c["N"]
    return {"bytes": N * K // 2 + N * (K // c["group"]) * 2 + M * K * size[c["x"]] + M * N * 2 + (4 * N if c["bias"] else 0), "flops": 2 * M * N * K}
