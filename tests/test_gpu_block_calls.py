"""Calls of the block's operators that their own files do not make."""
import pytest
import torch

import ulm_infer
import ulm_ops
from oracle import rotary as ro

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


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('at', [1, -1, 2, 3, 100, -4097, 1 << 20])
def test_slow_pairs_turn_by_their_own_small_angle(at, interleaved):
    """The sine alone (a pair of 0 and 1), relative to itself, in units of 2^-24: the angle's lower part, the factor and their product one
    each, what is cut off behind 2^-58 of a turn two at 2^-35 of a turn, the slowest here, or instead the sum's rounding where an upper part is there too;
    the polynomial's last step one.  Times 1 and plus 0 the result is the sine."""
    turns = torch.cat([ulm_ops.rotary_turns(d, base, dict(kind='linear', factor=f))[0] for d, base, f in ((64, 1e4, 1.0), (128, 1e6, 8.0), (256, 1e8, 64.0))])
    n = len(turns)
    x = torch.zeros(1, 1, 1, 2 * n, device='cuda')
    (x[..., 1::2] if interleaved else x[..., n:]).fill_(1)
    y = ulm_ops.rotary(x, None, turns.cuda(), torch.tensor([at], device='cuda'), interleaved)[0].double().cpu()
    y, want = (t[..., 0::2] if interleaved else t[..., :n] for t in (y, ro.rotary(x, [at], turns, interleaved)))
    assert bool(((y - want).abs() <= 6 * 2.0 ** -24 * want.abs()).all()), float(((y - want) / want).abs().max())
