"""Plain forms in 64 bits for the operators around a decode step, on the CPU."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}   # half a rounding step, relative
E8M0 = torch.float8_e8m0fnu


def scale_values(s8):
    """float8_e8m0fnu -> float64 (any device), 255 as NaN."""
    b = s8.cpu().view(torch.uint8).double()
    return torch.where(b == 255, torch.full_like(b, float("nan")), torch.exp2(b - 127))


def quantize64(x):
    """(e4m3 values as float64, scale float64) of rows x: the definition, row by row."""
    x = x.double().cpu()
    flat = x.reshape(-1, x.shape[-1])
    vals, scales = torch.empty_like(flat), torch.empty(flat.shape[0], dtype=torch.float64)
    for i, row in enumerate(flat):
        if not torch.isfinite(row).all():
            vals[i], scales[i] = float("nan"), float("nan")
            continue
        top = float(row.abs().max()) if row.numel() else 0.0
        e = 0
        if top > 0:
            e = -126
            if top > 448.0 * 2.0 ** -126:
                e = math.ceil(math.log2(top / 448.0)) - 1
                while top > 448.0 * 2.0 ** e:
                    e += 1
        scales[i] = 2.0 ** e
        vals[i] = (row / 2.0 ** e).float().to(torch.float8_e4m3fn).double()      # a power of two: the division rounds nothing in fp32 either
    return vals.view(x.shape), scales.view(x.shape[:-1])


def dequantize64(v8, s8):
    return v8.cpu().float().double() * scale_values(s8)[..., None]


def attention64(q, k, v, scale, bias=None):
    """softmax(scale q.k + bias) v in 64 bits and what the error of an evaluation may be.

    q [G,D], k, v [n,D] float64 (bias [n]).  Returns (out [G,D], spread [G,D], ds [G]): spread = sum_j p_j |v_j|, and ds bounds the error of a
    score whose products are summed in fp32 (any order, D terms: relative D 2^-24 of sum |q k|, and the few roundings behind it) together with
    that of the exponential (2^-22, CUDA's bound for exp2f and __expf at arguments of this size).  An error ds of the scores moves the
    result by at most 2 ds spread."""
    if k.shape[0] == 0:
        z = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
        return z, z, torch.zeros(q.shape[0], dtype=torch.float64)
    s = scale * q @ k.T
    mag = scale * q.abs() @ k.abs().T
    if bias is not None:
        s, mag = s + bias, mag + bias.abs()
    p = torch.softmax(s, 1)
    # only scores that carry weight move the result: the largest magnitude among them
    ds = (q.shape[1] + 8) * 2.0 ** -24 * mag.max(1).values + 2.0 ** -21
    return p @ v, p @ v.abs(), ds
