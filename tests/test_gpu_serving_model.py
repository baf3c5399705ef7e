"""The model's training path with fused norms, and its decode path over paged and 8-bit caches, with 4-bit projections: the operators as they are used
together."""
import pytest
import torch
import torch.nn as nn

import dwarf_b200
from dwarf_b200.int4 import Int4Linear
from dwarf_b200.model import CondMLM

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OFFSETS = (0, 1, 2, 3, 4, 8, 16, 48)


def model(attention="condU", dim=64, seq_len=160, full=1, **kw):
    torch.manual_seed(7)
    m = CondMLM(vocab=211, dim=dim, heads=2, layers=3, ffn=128, seq_len=seq_len, full_attention_layer=full, offsets=OFFSETS, attention=attention, **kw).to(DEV)
    with torch.no_grad():
        for blk in m.blocks:
            if hasattr(blk.attn, "scale_embed"):
                blk.attn.scale_embed.normal_(0.0, 0.05)
                blk.attn.if_gain.uniform_(0.8, 1.2)
        for p in m.parameters():
            if p.dim() == 2:
                p.mul_(8.0)
            elif p.dim() == 1:
                p.add_(torch.randn_like(p) * 0.1)
    return m


def off(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def ids_of(S, n, seed=1):
    return torch.randint(0, 211, (S, n), device=DEV, generator=torch.Generator(DEV).manual_seed(seed))


@pytest.mark.parametrize("attention", ["condU", "condM"])
def test_fused_norms_are_the_model(attention):
    """fp32: the same sums in another order, so 1e-5 apart but for the attention's bf16 inputs, which a last bit may round the other way (2^-8 of
    single elements): 1e-3.  Under autocast the norm is rounded to bf16 once in both."""
    plain, fused = model(attention), model(attention, fused_norms=True)
    assert all(torch.equal(a, b) for a, b in zip(plain.parameters(), fused.parameters()))
    ids = ids_of(2, 60)
    for autocast, tol in ((False, 1e-3), (True, 2e-2)):
        got = []
        for m in (plain, fused):
            m.zero_grad()
            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
                y = m(ids)
            y.float().square().mean().backward()
            got.append([y.detach()] + [p.grad.clone() for p in m.parameters()])
        assert off(got[1][0], got[0][0]) < tol
        for a, b, (name, _) in zip(got[1][1:], got[0][1:], plain.named_parameters()):
            # gradients that nearly cancel (a key bias moves no softmax) say nothing
            if b.norm() > 1e-4 * max(g.norm() for g in got[0][1:]):
                assert off(a, b) < 5 * tol, name
    # calling it again and again, eager, gives the same bits
    with torch.no_grad():
        assert torch.equal(fused(ids), fused(ids))


@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 2e-2), (torch.float8_e4m3fn, 0.15)], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("attention,full", [("condU", 1), ("condM", 0), ("condU", 5)])
def test_decode_over_paged_caches_follows_the_whole_prefix(dtype, tol, attention, full):
    """bf16 caches: as the contiguous ones.  8 bits: every element of a cached row is off by up to 2^-4, 3.6 % in the mean square, and three layers add up."""
    m = model(attention, full=full).eval()
    S, prompt, new = 3, 70, 12
    ids = ids_of(S, prompt + new)
    with torch.no_grad():
        full_logits = m(ids).float()
        logits, state = m.prefill(ids[:, :prompt], max_len=prompt + new, cache_dtype=dtype, page_size=16)
        assert off(logits, full_logits[:, prompt - 1]) < 2e-2
        for t in range(prompt, prompt + new):
            logits = m.decode_token(ids[:, t], state)
            assert off(logits, full_logits[:, t]) < tol, f"position {t}"
    assert state["t"] == prompt + new
    if full < 3:
        assert state["paged"].lengths.tolist() == [prompt + new] * S
    a, b = m.generate(ids[:, :prompt], 6, cache_dtype=dtype), m.generate(ids[:, :prompt], 6, cache_dtype=dtype)
    assert a.shape == (S, prompt + 6) and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn], ids=["bf16", "e4m3"])
def test_four_bit_projections_eight_bit_norms_and_caches_together(dtype):
    """Against the same model with the 4-bit weights written out, in its plain decode path.  Norms in 8 bits: 3.6 % in the mean square on the inputs of two
    thirds of the projections; caches as above."""
    m = model("condU").eval()
    q = model("condU").eval().quantize_weights()
    for blk, qb in zip(m.blocks, q.blocks):
        for a, b in ((blk.attn, qb.attn), (blk.ffn, qb.ffn)):
            for name, child in a.named_children():
                if isinstance(child, nn.Linear):
                    c = getattr(b, name)
                    assert type(c) is Int4Linear and c.group == (128 if child.in_features % 128 == 0 else 64)
                    nib = torch.stack([c.weight & 15, c.weight >> 4], -1).flatten(1).float() - 8
                    with torch.no_grad():
                        child.weight.copy_(nib * c.scales.float().repeat_interleave(c.group, 1))
    S, prompt, new = 2, 60, 10
    ids = ids_of(S, prompt + new, 3)
    with torch.no_grad():
        want, plain = m.prefill(ids[:, :prompt], max_len=prompt + new)
        got, state = q.prefill(ids[:, :prompt], max_len=prompt + new, cache_dtype=dtype)
        assert off(got, want) < 2e-2                                  # the prompt's projections read bf16
        for t in range(prompt, prompt + new):
            want, got = m.decode_token(ids[:, t], plain), q.decode_token(ids[:, t], state)
            assert off(got, want) < 0.2, f"position {t}"
    assert q.generate(ids[:, :prompt], 5, cache_dtype=dtype).shape == (S, prompt + 5)
    sd = q.state_dict()
    again = model("condU").eval().quantize_weights()
    again.load_state_dict(sd)
    with torch.no_grad():
        assert torch.equal(again(ids[:, :20]), q(ids[:, :20]))


def test_refusals():
    with pytest.raises(ValueError):
        model("condM", dim=48).quantize_weights()
    with pytest.raises(ValueError):
        model("condM").quantize_weights(128)                          # inputs of 64 columns
    m = model("condU").eval().quantize_weights()
    with pytest.raises(RuntimeError):
        m(ids_of(1, 8))                                               # no backward pass through 4-bit projections
    with pytest.raises(TypeError):
        with torch.no_grad():
            m.prefill(ids_of(1, 8), cache_dtype=torch.float16)


@pytest.mark.parametrize("attention,full", [("condU", 1), ("condM", 0)])
@pytest.mark.parametrize("dtype,bits4", [(torch.bfloat16, False), (torch.float8_e4m3fn, False), (torch.float8_e4m3fn, True)], ids=["bf16", "e4m3", "e4m3_int4"])
def test_a_bf16_model_serves(attention, full, dtype, bits4):
    """The documented serving model: bf16 parameters throughout, fused norms.  Its decode path against its whole prefix: both round every activation to bf16 (2^-8, some 20 in a row
    and in three layers, 2e-2 as above and as much again for what differs in order), with 8-bit caches and norms as above."""
    m = model(attention, full=full, fused_norms=True).to(torch.bfloat16).eval()
    if bits4:
        m.quantize_weights()
    S, prompt, new = 3, 70, 12
    ids = ids_of(S, prompt + new)
    with torch.no_grad():
        whole = m(ids)
        assert whole.dtype is torch.bfloat16
        logits, state = m.prefill(ids[:, :prompt], max_len=prompt + new, cache_dtype=dtype, page_size=16)
        assert off(logits, whole[:, prompt - 1]) < 4e-2
        for t in range(prompt, prompt + new):
            logits = m.decode_token(ids[:, t], state)
            assert logits.dtype is torch.bfloat16 and off(logits, whole[:, t]) < (0.2 if bits4 else 0.15 if dtype is torch.float8_e4m3fn else 4e-2), f"position {t}"
    a, b = m.generate(ids[:, :prompt], 6, cache_dtype=dtype), m.generate(ids[:, :prompt], 6, cache_dtype=dtype)
    assert a.shape == (S, prompt + 6) and torch.equal(a, b)


def test_a_bf16_model_trains_with_fused_norms():
    """bf16 parameters: the same roundings of every activation in both, but for the sums of a norm.  Where bf16 rounds one the other way the two part by 2^-8 of it: 4e-2 as above for
    the result, five times that for gradients."""
    plain, fused = model("condU").to(torch.bfloat16), model("condU", fused_norms=True).to(torch.bfloat16)
    ids, got = ids_of(2, 60), []
    for m in (plain, fused):
        y = m(ids)
        y.float().square().mean().backward()
        got.append([y.detach()] + [p.grad.clone() for p in m.parameters()])
    assert off(got[1][0], got[0][0]) < 4e-2
    for a, b, (name, p) in zip(got[1][1:], got[0][1:], plain.named_parameters()):
        assert a.dtype is p.dtype
        if b.norm() > 1e-2 * max(g.norm() for g in got[0][1:]):
            assert off(a, b) < 0.2, name
