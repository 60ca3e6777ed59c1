"""Calls of the block's operators that their own files do not make."""
import pytest
import torch

import ulm_infer
import ulm_ops
import ulm_train
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


LAYERS = {
    'linear': lambda x, w, packed: ulm_ops.linear_8bit(x, w[0], packed),
    'feed-forward': lambda x, w, packed: ulm_ops.feed_forward_8bit(x, w[0], w[1], w[2], 0.2, 5, packed),
}


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('layer', list(LAYERS))
@pytest.mark.parametrize('shape', [(5, 72), (2, 33, 40), (64,), (0, 64)])
def test_an_input_packed_once_gives_the_same_bits(layer, dtype, shape):
    d = shape[-1]
    x = randn(shape, F32, 1).requires_grad_()
    w = [randn(s, F32, 2 + i, 0.2).requires_grad_() for i, s in enumerate([(48, d), (48, d), (24, 48)])]
    with torch.autocast('cuda', dtype=dtype, enabled=dtype != F32):
        want, got = (LAYERS[layer](x, w, packed) for packed in (None, ulm_ops.pack_8bit(x.to(dtype))))
    assert torch.equal(got, want)
    leaves = [x, *w[:1 if layer == 'linear' else 3]]
    for a, b in zip(torch.autograd.grad(got.sum(), leaves), torch.autograd.grad(want.sum(), leaves)):
        assert torch.equal(a, b)


@pytest.mark.parametrize('layer', list(LAYERS))
@pytest.mark.parametrize('bad', ['shape', 'type of the codes', 'exponents', 'type of the product', 'devices', 'no exponents'])
def test_another_packing_is_refused(layer, bad):
    x, w = randn((4, 64), BF16, 1).requires_grad_(), [randn((64, 64), BF16, 2 + i) for i in range(3)]
    packed = ulm_ops.pack_8bit(x)
    packed = {'shape': lambda: ulm_ops.pack_8bit(x.view(2, 2, 64)), 'type of the codes': lambda: packed._replace(codes=packed.codes.byte()),
              'exponents': lambda: packed._replace(exponents=packed.exponents[1:]), 'type of the product': lambda: ulm_ops.pack_8bit(x.float()),
              'devices': lambda: packed._replace(codes=packed.codes.cpu()), 'no exponents': lambda: packed._replace(exponents=None)}[bad]()
    for graph in (True, False):
        with pytest.raises(ValueError), torch.set_grad_enabled(graph):
            LAYERS[layer](x, w, packed)


def test_changed_codes_are_noticed_and_frozen_weights_keep_none():
    x, w = randn((4, 64), BF16, 1).requires_grad_(), [randn((64, 64), BF16, 2 + i).requires_grad_() for i in range(3)]
    packed = ulm_ops.pack_8bit(x)
    for f in LAYERS.values():
        y = f(x, w, packed)
        packed.codes.zero_()
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            torch.autograd.grad(y.sum(), w[0])
        y = f(x, [t.detach() for t in w], packed)
        packed.codes.zero_()
        assert torch.autograd.grad(y.sum(), x)[0].any()
    with torch.autograd.graph.save_on_cpu():
        parked = ulm_ops.linear_8bit(x, w[0], ulm_ops.pack_8bit(x))
    assert torch.equal(torch.autograd.grad(parked.sum(), w[0])[0], torch.autograd.grad(ulm_ops.linear_8bit(x, w[0]).sum(), w[0])[0])


def test_a_traced_projection_of_a_packed_input():
    w = torch.nn.ParameterList([randn((64, 64), F32, 2 + i) for i in range(3)])

    class Both(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = w

        def forward(self, x):
            packed = ulm_ops.pack_8bit(x)
            return LAYERS['linear'](x, self.w, packed) + LAYERS['feed-forward'](x, self.w, packed)
    m, x = Both(), randn((4, 64), F32, 7)
    got, want = torch.jit.trace(m, randn((4, 64), F32, 1))(x), m(x)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got.sum(), list(w)), torch.autograd.grad(want.sum(), list(w))):
        assert float((a - b).norm()) <= 2.0 ** -20 * float(b.norm())       # the sums of two gradients may be taken in another order


@pytest.mark.parametrize('dropout', [0.0, 0.2])
def test_a_branch_gate_shares_the_packed_input(dropout):
    """With a gate behind the branches a layer keeps no more of its two normalised inputs than without one."""
    kept = {}
    for gate in (False, True):
        for bits in (False, True):
            model, _ = ulm_train.build('tiny64', 'cuda', dropout=dropout, counter_dropout=True, branch_norm=True, branch_gate=gate, activations_8bit=bits)
            for layer in model.layers:
                layer.self_attn.dropout = 0.0
            own, seen = {p.untyped_storage().data_ptr() for p in model.parameters()}, {}

            def count(t):
                if t.untyped_storage().data_ptr() not in own:          # noqa: B023
                    seen[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()      # noqa: B023
                return t
            ids = torch.randint(4, 4096, (16, 256), generator=torch.Generator().manual_seed(3)).cuda()
            with torch.autograd.graph.saved_tensors_hooks(count, lambda t: t), torch.autocast('cuda', dtype=BF16), ulm_ops.weight_cast_scope():
                h = model.forward_hidden(ids)
            kept[gate, bits] = sum(seen.values())
            del h
    tokens, ff, d = 16 * 256, 344, 128
    for gate in (False, True):
        assert kept[gate, False] - kept[gate, True] == 2 * tokens * ((6 - 2.0625) * ff + (4 - 2.0625) * d)
    assert kept[True, True] - kept[False, True] == 2 * tokens * 2 * 2 * d      # the gates themselves


def test_a_watched_branch_shares_nothing():
    """A hook may change what a branch projects: what it is handed is then packed by itself, and the gate has the input as it was."""
    grads = []
    for watched in (False, True):
        model, _ = ulm_train.build('tiny64', 'cuda', seed=0, branch_norm=True, branch_gate=True, activations_8bit=True)
        if watched:
            for layer in model.layers:
                layer.self_attn.register_forward_pre_hook(lambda m, a: (a[0] * 2,))
                layer.ff.register_forward_pre_hook(lambda m, a: (a[0] * 2,))
        else:
            with torch.no_grad():
                for layer in model.layers:
                    for m in (layer.self_attn.wqkv, layer.ff.w1, layer.ff.w3):
                        m.weight.mul_(2)
        with torch.autocast('cuda', dtype=BF16):
            loss = model.compute_loss(torch.randint(4, 4096, (4, 120), generator=torch.Generator().manual_seed(3)).cuda())
        grads.append((loss.detach(), *torch.autograd.grad(loss, [model.layers[0].self_attn.wqkv.weight, model.layers[1].ff.w1.weight])))
    assert torch.equal(grads[0][0], grads[1][0])           # powers of two
    for a, b in zip(grads[0][1:], grads[1][1:]):
        assert torch.equal(2 * a, b)


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
