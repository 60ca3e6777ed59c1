"""Calls at the edge of what the gate, dropout, norm and loss ops take: operands elsewhere, gradients of any alignment and
rows of any stride, hooked modules, second derivatives, captured steps."""
import pytest
import torch

import _native as N
import ulm_ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') * std).to(dtype)


@pytest.mark.parametrize('op', [ulm_ops.swiglu, lambda a, b: ulm_ops.swiglu_dropout(a, b, 0.5, 1)])
@pytest.mark.parametrize('elsewhere', ['cpu', 'meta'])
def test_gate_refuses_operands_of_two_devices(op, elsewhere):
    a = torch.ones(4, 64, device='cuda')
    with pytest.raises(ValueError, match='one CUDA device'):
        op(a, torch.ones(4, 64, device=elsewhere))
    with pytest.raises(ValueError, match='one CUDA device'):
        op(torch.ones(4, 64, device=elsewhere), a)


@pytest.mark.parametrize('bad', ['weight on the host', 'short weight', 'long weight', 'branch on the host'])
def test_norms_refuse_what_they_cannot_read(bad):
    x, b = torch.ones(4, 64, device='cuda'), torch.ones(4, 64, dtype=F16, device='cpu' if bad == 'branch on the host' else 'cuda')
    w = torch.ones({'short weight': 32, 'long weight': 65}.get(bad, 64), device='cpu' if bad == 'weight on the host' else 'cuda')
    with pytest.raises(ValueError):
        ulm_ops.add_rms_norm(x, b, w)
    if bad != 'branch on the host':
        for dtype in (F16, BF16, F32):
            with pytest.raises(ValueError, match='one weight per column'):
                ulm_ops.rms_norm(x.to(dtype), w)


def shifted(t):
    """The same values, contiguous, one element past an aligned address."""
    v = torch.empty(t.numel() + 1, device='cuda', dtype=t.dtype)[1:].view_as(t)
    return v.copy_(t)


OPS = {
    'swiglu': lambda dt: (ulm_ops.swiglu, [randn((5, 64), dt, 1), randn((5, 64), dt, 2)]),
    'swiglu_dropout': lambda dt: (lambda a, b: ulm_ops.swiglu_dropout(a, b, 0.5, 1), [randn((5, 64), dt, 1), randn((5, 64), dt, 2)]),
    'dropout': lambda dt: (lambda a: ulm_ops.dropout(a, 0.5, 1), [randn((5, 64), dt, 1)]),
    'rms_norm': lambda dt: (ulm_ops.rms_norm, [randn((5, 64), dt, 1), randn(64, F32, 2)]),
    'rms_norm, wide rows': lambda dt: (ulm_ops.rms_norm, [randn((5, 1000), dt, 1), randn(1000, F32, 2)]),
    'add_rms_norm': lambda dt: (ulm_ops.add_rms_norm, [randn((5, 64), F32, 1), randn((5, 64), BF16 if dt is F32 else dt, 2), randn(64, F32, 3)]),
    'dropout_add_rms_norm': lambda dt: (lambda x, b, w: ulm_ops.dropout_add_rms_norm(x, b, w, 0.5, 1),
                                        [randn((5, 64), F32, 1), randn((5, 64), BF16 if dt is F32 else dt, 2), randn(64, F32, 3)]),
}
# the operands of these go to library products, which may take another kernel for another alignment
PROJECTED = {
    'gated_linear': lambda dt: (ulm_ops.gated_linear, [randn((5, 64), dt, 1), randn((32, 64), dt, 2), randn((32, 64), dt, 3)]),
    'gated_linear with dropout': lambda dt: (lambda x, w, v: ulm_ops.gated_linear(x, w, v, 0.5, 1), [randn((5, 64), dt, 1), randn((32, 64), dt, 2), randn((32, 64), dt, 3)]),
}


def outputs_and_gradients(op, ins, of_input=lambda t: t, of_grad=lambda t: t):
    ins = [of_input(t).detach().requires_grad_() for t in ins]
    out = op(*ins)
    out = list(out) if isinstance(out, tuple) else [out]
    grads = torch.autograd.grad(out, ins, [of_grad(randn(o.shape, o.dtype, 9 + i)) for i, o in enumerate(out)])
    return [*out, *grads]


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('name', [*OPS, *PROJECTED])
def test_gradients_of_any_alignment(name, dtype):
    op, ins = {**OPS, **PROJECTED}[name](dtype)
    for got, want in zip(outputs_and_gradients(op, ins, of_grad=shifted), outputs_and_gradients(op, ins)):
        assert torch.equal(got, want)


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('name', list(OPS))
def test_operands_of_any_alignment(name, dtype):
    op, ins = OPS[name](dtype)
    for got, want in zip(outputs_and_gradients(op, ins, of_input=shifted), outputs_and_gradients(op, ins)):
        assert torch.equal(got, want)


def odd_row(t):
    """The same values; where there is one row, its stride is no multiple of anything (torch calls it contiguous all the same)."""
    if t.dim() < 2:
        return t
    n = t.shape[-1]
    v = torch.empty(n + 3, device='cuda', dtype=t.dtype).as_strided(t.shape, [n + 3] * (t.dim() - 1) + [1])
    return v.copy_(t)


@pytest.mark.parametrize('name', ['rms_norm', 'add_rms_norm', 'dropout_add_rms_norm'])
def test_one_row_of_any_stride(name):
    op, ins = OPS[name](F32)
    ins = [t[:1] if t.dim() > 1 else t for t in ins]
    assert odd_row(ins[0]).is_contiguous()
    want = outputs_and_gradients(op, ins)
    for got in (outputs_and_gradients(op, ins, of_input=odd_row), outputs_and_gradients(op, ins, of_grad=odd_row)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('shape', [(2, 3, 64), (1, 1, 64), (64,), (2, 2, 2, 64)])
@pytest.mark.parametrize('name', ['rms_norm', 'add_rms_norm', 'dropout_add_rms_norm'])
def test_norms_of_any_number_of_dimensions(name, shape):
    op, ins = OPS[name](F32)
    rows = torch.Size(shape).numel() // 64
    wide = [randn((rows, 64), t.dtype, 4 + i) if t.dim() > 1 else t for i, t in enumerate(ins)]
    flat = outputs_and_gradients(op, wide)
    shaped = outputs_and_gradients(lambda *a: op(*a), [t.view(shape) if t.dim() > 1 else t for t in wide])
    for got, want in zip(shaped, flat):
        assert torch.equal(got.reshape(want.shape), want)
        assert got.shape == (shape if want.dim() > 1 else want.shape)


ONCE = {
    'swiglu_dropout': OPS['swiglu_dropout'],
    'gated_linear with dropout': PROJECTED['gated_linear with dropout'],
    'dropout_add_rms_norm': OPS['dropout_add_rms_norm'],
    'streamed_cross_entropy': lambda dt: (lambda h, w: ulm_ops.streamed_cross_entropy(h, w, torch.tensor([3, 0, 8, 1, 8], device='cuda'), compute_dtype=BF16),
                                          [randn((5, 64), dt, 1), randn((9, 64), dt, 2)]),
}


@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('name', list(ONCE))
def test_second_derivatives_are_refused_and_not_left_out(name, dtype):
    op, ins = ONCE[name](dtype)
    ins = [t.requires_grad_() for t in ins]
    out = op(*ins)
    out = list(out) if isinstance(out, tuple) else [out]
    ups = [torch.ones_like(o, requires_grad=True) for o in out]
    want = torch.autograd.grad(out, ins, ups, retain_graph=True)
    got = torch.autograd.grad(out, ins, ups, create_graph=True)
    for g, w in zip(got, want):
        assert g.requires_grad and torch.equal(g.detach(), w)
    for i, x in enumerate(ins):
        total = got[i].float().square().sum() + sum((t.float() ** 3).sum() for t in ins)
        for wrt in (x, ups[0]):
            with pytest.raises(RuntimeError, match='has no second derivative'):
                torch.autograd.grad(total, wrt, retain_graph=True, allow_unused=True)
        with pytest.raises(RuntimeError, match='has no second derivative'):
            total.backward(retain_graph=True)
    # what does not go through the gradients is not in the way
    assert torch.autograd.grad(sum((t.float() ** 3).sum() for t in ins), ins[0])[0] is not None


@pytest.mark.parametrize('rows,d,piece_bytes', [(4096, 1024, 16 << 20), (16384, 256, 1 << 20), (300, 64, 1 << 16)])
def test_memory_of_the_streamed_backward(rows, d, piece_bytes, monkeypatch):
    """The softmax of a piece, hidden's fp32 sum, the parts of cut tiles; and the gradients."""
    V = 32768
    monkeypatch.setattr(ulm_ops, 'PIECE_BYTES', piece_bytes)
    h, w = (randn(s, BF16, i).requires_grad_() for i, s in enumerate([(rows, d), (V, d)]))
    loss = ulm_ops.streamed_cross_entropy(h, w, torch.randint(1, V, (rows,), device='cuda'))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    torch.autograd.grad(loss, [h, w])
    peak = torch.cuda.max_memory_allocated() - before - 2 * (rows + V) * d
    piece = max(256, piece_bytes // (2 * rows) // 256 * 256)
    parts = N.lib().ulm_streamed_ce_slots(rows, V, d, piece, 1, 1) * 4
    assert parts % (256 * 256 * 4) == 0
    # what the allocator rounds each of four tensors up to: 2 MB at most
    assert peak <= max(piece_bytes, 512 * rows) + 4 * rows * d + parts + (8 << 20)
    assert peak >= 4 * rows * d


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('rows,V,d', [(300, 32000, 1024), (64, 4096, 768), (200, 1000, 128)])
@pytest.mark.parametrize('logit', [10.0, 14.0, 17.0, 22.0])
def test_gradient_of_rows_that_are_almost_certain(rows, V, d, dtype, logit):
    """The target's probability p is close to 1; what is left of the gradient is as small as 1 - p."""
    w = randn((V, d), F32, 1, d ** -0.5).to(dtype)
    t = torch.randint(1, V, (rows,), generator=torch.Generator(device='cuda').manual_seed(2), device='cuda')
    h, wt = randn((rows, d), F32, 3, 0.5), w[t].float()
    h = (h + wt * ((logit - (h * wt).sum(1)) / wt.square().sum(1))[:, None]).to(dtype).requires_grad_()
    up = 2.0 ** 12
    dh, = torch.autograd.grad(ulm_ops.streamed_cross_entropy(h, w, t, denominator=1.0), [h], torch.tensor(up, device='cuda'))
    z = h.detach().double() @ w.double().T
    lse, at = torch.logsumexp(z, 1), torch.arange(rows, device='cuda')
    g = torch.exp(z - lse[:, None])
    rest = 1 - g[at, t]                                    # exact to 1e-16
    g[at, t] = 0
    others = g @ w.double()
    want = up * (others - rest[:, None] * w[t].double())
    unit = {F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype]
    norm = w.double().norm(dim=1)
    # the log-sum-exp's rounding to fp32, and 2^-22 for the sum behind it and its parts; one rounding of each probability and of
    # p - 1; logits short by 2^-16 at most (1e-6 of 22); one rounding of the result
    bound = up * ((2.0 ** -24 * lse.abs() + 2.0 ** -21) * norm[t] + (unit + 2.0 ** -16) * ((g * norm).sum(1) + rest * norm[t])) + unit * want.norm(dim=1)
    assert bool(((dh.double() - want).norm(dim=1) <= bound).all())


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('V,d', [(32000, 1024), (4096, 128), (1, 64)])
def test_no_loss_is_negative(V, d, dtype):
    w, h = randn((V, d), F32, 1, d ** -0.5).to(dtype), randn((256, d), F32, 2, 40.0).to(dtype)
    t = (h.float() @ w.float().T).argmax(1)                # the most likely column of rows that are sharp: p = 1 for many
    losses = torch.stack([ulm_ops.streamed_cross_entropy(h[i:i + 1], w, t[i:i + 1], ignore_index=-1) for i in range(256)])
    assert bool((losses >= 0).all()) and bool((losses < 1e-6).any())
    h[0, 0] = float('nan')
    assert ulm_ops.streamed_cross_entropy(h[:1], w, t[:1], ignore_index=-1).isnan()
