"""Single-token DSQG decode over per-layer circular K/V ring buffers.

The DWARF reference has no decode path (README.md:175-179 describes the O(1) cache in
prose; its generate() re-runs the whole prefix, train/train_2048_condU.py:463-487).
This module provides that cache: a ring of R = max(offsets)+1 slots per (sequence, head),
a write head per sequence, and one kernel launch per layer per token.
"""
from __future__ import annotations

from typing import Sequence

import torch

from . import _lib
from .ops import OFFSETS_43, _dtype_code


def dsqg_decode_step(q, k_new, v_new, k_ring, v_ring, head, pos_bias, head_gain=None,
                     scale_embed=None, offsets: Sequence[int] = OFFSETS_43, fill=None, out=None, overlap=False):
    """One decode step for one layer.

    q, k_new, v_new [S,H,D]; k_ring, v_ring [S,H,R,D] (updated in place at slot head[s]);
    head int32 [S] on the device; fill int32 [S] (valid tokens incl. the new one) or None
    for a full ring.  Returns out [S,H,D].

    overlap=True launches the kernel so that its ring gather runs while the kernel ahead of it
    in the stream is still finishing (`dsqg_decode_overlapped`): allowed only when that kernel
    writes none of this call's head, fill, k_ring, v_ring.
    """
    return _lib.native().decode_step(q, k_new, v_new, k_ring, v_ring, head, pos_bias, head_gain, scale_embed,
                                     _lib.offsets_handle(offsets), fill, out, overlap)


def dsqg_decode_step_kv(q, k_new, v_new, kv_ring, head, pos_bias, head_gain=None, scale_embed=None,
                        offsets: Sequence[int] = OFFSETS_43, fill=None, out=None, overlap=False, kv_scale=None):
    """dsqg_decode_step over one ring that holds key and value of a slot side by side:
    kv_ring [S,H,R,2,D] (updated in place).  A tap is one contiguous read of 2*D elements.

    kv_ring may be in 8 bits: float8_e4m3fn with kv_scale [S,H,R,2] float8_e8m0fnu, a power of two per row (both updated in place); q, k_new, v_new are
    then bf16 or fp32, and the step attends to what the ring holds, the new token's quantised rows included."""
    return _lib.native().decode_step_kv(q, k_new, v_new, kv_ring, None, head, pos_bias, head_gain, scale_embed,
                                        _lib.offsets_handle(offsets), fill, out, overlap, kv_scale)


class DSQGRingCache:
    """K/V rings for L layers, one shared write head per sequence.  interleaved=True (default) keeps
    key and value of a slot side by side in one tensor kv [L,S,H,R,2,D] (a tap is one contiguous
    read; `k` and `v` are strided views of it); interleaved=False keeps two tensors k, v [L,S,H,R,D].
    dtype=torch.float8_e4m3fn keeps the rows in 8 bits with a power-of-two scale each, kv_scale [L,S,H,R,2] float8_e8m0fnu: they are
    quantised as they are written, and `step` takes and returns bf16 (or fp32)."""

    kv_scale = None

    def __init__(self, layers, sequences, heads, head_dim, offsets: Sequence[int] = OFFSETS_43,
                 dtype=torch.bfloat16, device="cuda", interleaved=True):
        self.offsets = offsets
        self.R = max(self.offsets) + 1
        self.interleaved = interleaved
        if dtype is torch.float8_e4m3fn:
            if not interleaved:
                raise ValueError("dsqg ring cache: 8-bit rings keep key and value side by side (interleaved=True)")
            shape = (layers, sequences, heads, self.R, 2)
            self.kv = torch.zeros(*shape, head_dim, dtype=torch.uint8, device=device).view(dtype)
            self.kv_scale = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
            self.k, self.v = self.kv[..., 0, :], self.kv[..., 1, :]
        elif interleaved:
            self.kv = torch.zeros(layers, sequences, heads, self.R, 2, head_dim, dtype=dtype, device=device)
            self.k, self.v = self.kv[..., 0, :], self.kv[..., 1, :]
        else:
            self.kv = None
            self.k = torch.zeros(layers, sequences, heads, self.R, head_dim, dtype=dtype, device=device)
            self.v = torch.zeros_like(self.k)
        self.head = torch.full((sequences,), -1, dtype=torch.int32, device=device)
        self.fill = torch.zeros(sequences, dtype=torch.int32, device=device)

    # The native form of the offsets is kept beside them: looking it up hashes all of them, 0.3 us of a step of 5.5 us on the host.
    # It belongs to this process and is left out of copies and pickles.
    @property
    def offsets(self):
        return self._offsets

    @offsets.setter
    def offsets(self, offsets):
        self._offsets, self._handle = tuple(int(o) for o in offsets), None

    def __getstate__(self):
        state = dict(self.__dict__)
        state["offsets"] = state.pop("_offsets")
        del state["_handle"]
        return state

    def __setstate__(self, state):
        for name, value in state.items():
            setattr(self, name, value)

    @property
    def step_dtype(self):
        """The type of q, k and v that `step` takes (8-bit rings: bf16; fp32 works too)."""
        return self.k.dtype if self.kv_scale is None else torch.bfloat16

    def read(self, layer, dtype=torch.bfloat16):
        """(k, v) [S,H,R,D]: what the rings of `layer` hold, slot by slot; slots that no token has reached yet are not defined."""
        if self.kv_scale is None:
            return self.k[layer].to(dtype), self.v[layer].to(dtype)
        kv = self.kv[layer]
        out = torch.empty(kv.shape, dtype=dtype, device=kv.device)
        with torch.cuda.device(kv.device):
            _lib.check(_lib.load().dsqg_dequantize_rows(kv.data_ptr(), self.kv_scale[layer].data_ptr(), out.data_ptr(), kv.numel() // kv.shape[-1],
                                                        kv.shape[-1], _dtype_code(out), torch.cuda.current_stream(kv.device).cuda_stream), "dsqg_dequantize_rows")
        return out[..., 0, :], out[..., 1, :]

    def prefill(self, layer, k, v):
        """Load the rings of `layer` from a prefix in training layout: k, v [S,H,N,D].  Sets head
        and fill for the whole cache (call it with the same N for every layer)."""
        lib = _lib.load()
        S, H, N, D = k.shape
        if tuple(self.k[layer].shape) != (S, H, self.R, D) or (k.dtype != self.k.dtype and self.kv_scale is None) or v.shape != k.shape:
            raise ValueError("dsqg ring prefill: k, v must be [S,H,N,D] matching the cache")
        if self.kv_scale is not None and (v.dtype != k.dtype or k.device != self.kv.device or v.device != k.device):
            raise ValueError("dsqg ring prefill: k, v must be of one type on the device of the cache")
        k, v = k.contiguous(), v.contiguous()
        with torch.cuda.device(k.device):
            stream = torch.cuda.current_stream(k.device).cuda_stream
            if self.kv_scale is not None:
                _lib.check(lib.dsqg_ring_prefill_e4m3(k.data_ptr(), v.data_ptr(), self.kv[layer].data_ptr(), self.kv_scale[layer].data_ptr(),
                                                      self.head.data_ptr(), self.fill.data_ptr(), S, H, N, D, self.R, _dtype_code(k), stream),
                           "dsqg_ring_prefill_e4m3")
                return
            if self.interleaved:
                _lib.check(lib.dsqg_ring_prefill_kv(k.data_ptr(), v.data_ptr(), self.kv[layer].data_ptr(),
                                                    self.head.data_ptr(), self.fill.data_ptr(),
                                                    S, H, N, D, self.R, _dtype_code(k), stream), "dsqg_ring_prefill_kv")
                return
            _lib.check(lib.dsqg_ring_prefill(k.data_ptr(), v.data_ptr(), self.k[layer].data_ptr(),
                                             self.v[layer].data_ptr(), self.head.data_ptr(), self.fill.data_ptr(),
                                             S, H, N, D, self.R, _dtype_code(k), stream), "dsqg_ring_prefill")

    def advance(self):
        """Move every write head to the next slot; call once per token before the layers run."""
        self.head, self.fill = _lib.native().ring_advance(self.head, self.fill, self.R)

    def step(self, layer, q, k_new, v_new, pos_bias, head_gain=None, scale_embed=None, out=None, overlap=False):
        """Decode step of `layer`.  overlap=True is safe from the second layer of a token on (the
        kernel ahead is then another layer's step or a projection, never `advance`/`prefill`)."""
        if self.interleaved:
            handle = self._handle
            if handle is None:
                handle = self._handle = _lib.offsets_handle(self._offsets)
            return _lib.native().decode_step_kv(q, k_new, v_new, self.kv, layer, self.head, pos_bias, head_gain, scale_embed,
                                                handle, self.fill, out, overlap, self.kv_scale)
        return dsqg_decode_step(q, k_new, v_new, self.k[layer], self.v[layer], self.head, pos_bias,
                                head_gain, scale_embed, self.offsets, self.fill, out, overlap)
