"""Blocks and norms that a program has replaced, wrapped or listens in on are called by the fused paths of the model too."""
import pytest
import torch
import torch.nn as nn

from dwarf_b200.model import Block, RMSNorm
from tests.test_gpu_serving_model import ids_of, model, off

pytestmark = pytest.mark.gpu


class Doubled(RMSNorm):
    def forward(self, x):
        return 2 * super().forward(x)


class Wrapped(nn.Module):
    def __init__(self, block):
        super().__init__()
        self.block, self.calls = block, 0

    def forward(self, x):
        self.calls += 1
        return self.block(x)


def doubled(m, where):
    for name in where:
        owner, _, attr = name.rpartition(".")
        owner = m.get_submodule(owner)
        new = Doubled(getattr(owner, attr).weight.numel()).to(getattr(owner, attr).weight)
        new.weight = getattr(owner, attr).weight
        setattr(owner, attr, new)
    return m


@pytest.mark.parametrize("where", [["blocks.0.norm1"], ["blocks.2.norm2"], ["norm"], ["blocks.1.norm1", "norm"]])
def test_a_replaced_norm_counts_in_training(where):
    ids = ids_of(2, 60)
    with torch.no_grad():
        plain, fused = doubled(model("condU"), where)(ids), doubled(model("condU", fused_norms=True), where)(ids)
        assert off(fused, plain) < 1e-3 and off(model("condU")(ids), plain) > 1e-2


def test_hooks_and_wrapped_blocks_are_called_in_training():
    m, ids, seen = model("condU", fused_norms=True), ids_of(2, 60), []
    want = m(ids).detach()
    for name in ("blocks.0", "blocks.1.norm2", "norm"):
        m.get_submodule(name).register_forward_hook(lambda mod, args, out, name=name: seen.append((name, tuple(out.shape))))
    grads = []
    m.blocks[0].norm1.register_full_backward_hook(lambda mod, gi, go: grads.append(go[0].shape))
    m.blocks[2] = Wrapped(m.blocks[2])
    out = m(ids)
    out.square().mean().backward()
    assert [s[0] for s in seen] == ["blocks.0", "blocks.1.norm2", "norm"] and all(s[1] == (2, 60, 64) for s in seen) and len(grads) == 1 and m.blocks[2].calls == 1
    assert type(m.blocks[2].block) is Block and off(out.detach(), want) < 1e-3


@pytest.mark.parametrize("bits4", [False, True])
@pytest.mark.parametrize("where", [["blocks.0.norm1"], ["blocks.1.norm1"], ["blocks.2.norm2"], ["norm"]])
def test_a_replaced_norm_counts_in_decode(where, bits4):
    """Against the plain decode path; 8-bit norms in front of the other projections, and bf16 caches against bf16 caches."""
    ids = ids_of(2, 50)

    def logits(m, **kw):
        m = m.eval()
        if bits4:
            m.quantize_weights()
        with torch.no_grad():
            _, state = m.prefill(ids[:, :49], max_len=60, **kw)
            return m.decode_token(ids[:, 49], state).float()
    got, want, without = logits(doubled(model("condU"), where), cache_dtype=torch.bfloat16), logits(doubled(model("condU"), where)), logits(model("condU"))
    # a path that passes the replaced norm by gives `without`, up to its own error e: off(without, want) - e from `want`, which is more than half of that for any e
    # below the other half
    assert off(got, want) < (0.2 if bits4 else 2e-2) and off(got, want) < 0.5 * off(without, want)


@pytest.mark.parametrize("bits4", [False, True])
def test_hooks_see_tensors_in_decode(bits4):
    m, ids, seen = model("condU").eval(), ids_of(2, 50), []
    if bits4:
        m.quantize_weights()
    for name in ("blocks.0.norm1", "blocks.1.attn.qkv_proj", "blocks.2.ffn", "blocks.0.ffn.fc1", "norm"):
        m.get_submodule(name).register_forward_hook(lambda mod, args, out, name=name: seen.append((name, type(args[0]), out.shape[0])))
    with torch.no_grad():
        _, state = m.prefill(ids[:, :49], max_len=60, cache_dtype=torch.float8_e4m3fn)
        seen.clear()
        m.decode_token(ids[:, 49], state)
    assert sorted(seen, key=str) == sorted(((n, torch.Tensor, 2) for n in ("blocks.0.norm1", "blocks.1.attn.qkv_proj", "blocks.2.ffn", "blocks.0.ffn.fc1", "norm")), key=str)
