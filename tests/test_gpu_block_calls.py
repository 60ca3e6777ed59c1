"""Calls of the block's operators that their own files do not make."""
import pytest
import torch

import ulm_infer
import ulm_ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') * std).to(dtype)


# ---------------------------------------------------------------------------
# activations in 8 bits
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F16, BF16, F32])
def test_a_traced_packing_packs_other_inputs(dtype):
    """What a tracer does not see made is a constant of its trace."""
    def through(x):
        packed = ulm_ops.pack_8bit(x)
        return packed.codes, packed.exponents, ulm_ops.unpack_8bit(packed), ulm_ops.unpack_8bit(packed, F32)
    traced = torch.jit.trace(through, randn((5, 40), dtype, 1))
    x = randn((5, 40), dtype, 2, 3.0)
    for a, b in zip(traced(x), through(x)):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_packing_has_no_gradient_and_needs_none():
    x = randn((3, 40), F32, 1).requires_grad_()
    packed = ulm_ops.pack_8bit(x)
    assert not ulm_ops.unpack_8bit(packed).requires_grad
    with torch.autograd.forward_ad.dual_level():
        dual = ulm_ops.pack_8bit(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)))
    assert torch.equal(dual.codes, packed.codes) and torch.equal(dual.exponents, packed.exponents)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('autocast', [False, True])
def test_prefill_builds_no_graph(autocast):
    qkv = randn((2, 7, 384), BF16, 1).requires_grad_()
    with torch.autocast('cuda', dtype=BF16, enabled=autocast):
        out = ulm_infer.causal_attention(qkv, 2, rotary=ulm_ops.Rotary(64).cuda())
    assert not any(t.requires_grad for t in out)           # the keys and values go into a cache
