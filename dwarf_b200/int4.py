"""Projections with 4-bit weights and a scale per group of input columns, for the few rows of a decode step.

What a decode step spends its time on is reading the weights once: four bits an element are a quarter of bf16's.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

from . import _lib


class Rows8(NamedTuple):
    """Rows in 8 bits: values float8_e4m3fn [..., D] and scale float8_e8m0fnu [...], as rms_norm_e4m3 returns them."""
    values: torch.Tensor
    scale: torch.Tensor


def quantize_int4(weight, group=128):
    """weight [N,K] -> (packed uint8 [N,K/2], scales bf16 [N,K/group]): weight[n,k] ~ (nibble - 8) * scales[n, k // group], the nibble of an even k
    in the low half of its byte.  A group's scale is the smallest that holds both its ends (-8 and 7 steps)."""
    N, K = weight.shape
    if group not in (32, 64, 128) or K % group:
        raise ValueError(f"quantize_int4: a group must be of 32, 64 or 128 columns and divide K = {K}, got {group}")
    w = weight.detach().float().view(N, K // group, group)
    scales = torch.maximum(w.amax(-1) / 7, -w.amin(-1) / 8).clamp_min(0).to(torch.bfloat16)
    s = scales.float()[..., None]
    q = torch.where(s > 0, torch.round(w / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(w)).clamp(-8, 7).add(8).to(torch.uint8).view(N, K)
    return (q[:, 0::2] | q[:, 1::2] << 4).contiguous(), scales.contiguous()


def int4_linear(x, weight, scales, bias=None, x_scale=None):
    """x [..., K] bf16, or float8_e4m3fn with x_scale [...] float8_e8m0fnu -> [..., N] bf16 = x W^T + bias, W as quantize_int4 packs it.  fp32 sums, no
    backward pass.  Made for a few rows: up to 16 of them read the weights once."""
    return _lib.native().int4_linear(x, weight, scales, bias, x_scale)


class Int4Linear(nn.Module):
    """nn.Linear for inference with 4-bit weights.  Takes bf16 (or fp32, rounded to bf16, the result in fp32 again outside autocast) rows, or
    Rows8."""

    def __init__(self, in_features, out_features, bias=True, group=128, device=None):
        super().__init__()
        if group not in (32, 64, 128) or in_features % group:
            raise ValueError(f"Int4Linear: a group must be of 32, 64 or 128 columns and divide in_features = {in_features}, got {group}")
        self.in_features, self.out_features, self.group = in_features, out_features, group
        self.register_buffer("weight", torch.full((out_features, in_features // 2), 0x88, dtype=torch.uint8, device=device))
        self.register_buffer("scales", torch.zeros(out_features, in_features // group, dtype=torch.bfloat16, device=device))
        self.register_buffer("bias", torch.zeros(out_features, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear, group=128):
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, group, linear.weight.device)
        m.weight, m.scales = quantize_int4(linear.weight, group)
        if linear.bias is not None:
            m.bias = linear.bias.detach().float().clone()
        return m

    def _apply(self, fn, recurse=True):
        # .to(dtype), .half(), ... move this module but leave its types and values alone: they are the format
        before = dict(self._buffers)
        super()._apply(fn, recurse)
        for n, b in before.items():
            if b is not None and self._buffers[n].dtype != b.dtype:
                self._buffers[n] = b.to(self._buffers[n].device)
        return self

    def forward(self, x):
        if isinstance(x, Rows8):
            return int4_linear(x.values, self.weight, self.scales, self.bias, x.scale)
        if x.dtype is torch.bfloat16:
            return int4_linear(x, self.weight, self.scales, self.bias)
        y = int4_linear(x.to(torch.bfloat16), self.weight, self.scales, self.bias)
        return y if torch.is_autocast_enabled("cuda") else y.to(x.dtype)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, group={self.group}"
