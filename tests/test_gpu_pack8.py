"""Activations in 8 bits between forward and backward: the form itself bit for bit, the gate, a linear layer and the feed-forward on it."""
import math

import numpy as np
import pytest
import torch

import ulm_ops
from oracle import dropout as od
from oracle import pack8 as op

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}          # largest relative error of one rounding
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}       # and absolute, among subnormals


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') * std).to(dtype)


def within(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0)) and torch.equal(a.isnan(), b.isnan())


# ---------------------------------------------------------------------------
# the form
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('n', [1, 7, 31, 32, 33, 63, 64, 255, 256, 4095, 4096, 8191, 8192, 8193, 70003])
def test_codes_and_values_to_the_bit(dtype, n):
    x = randn(n, F32, n) * torch.exp2(torch.randint(-20, 12, (n,), generator=torch.Generator(device='cuda').manual_seed(n), device='cuda').float())
    x = x.to(dtype)
    p = ulm_ops.pack_8bit(x)
    codes, exps = op.pack(x)
    assert p.codes.dtype == torch.int8 and p.exponents.dtype == torch.uint8 and p.dtype == dtype and p.codes.shape == x.shape
    assert np.array_equal(p.codes.cpu().numpy(), codes) and np.array_equal(p.exponents.cpu().numpy(), exps)
    back = ulm_ops.unpack_8bit(p)
    assert back.dtype == dtype and torch.equal(back.double(), op.through(x))


@pytest.mark.parametrize('dtype', [F16, BF16])
def test_every_number_of_the_type(dtype):
    """Each bit pattern once as its block's largest, among neighbours of every smaller size, and once among larger ones."""
    all16 = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(dtype).cuda()
    x = torch.zeros(1 << 16, 32, device='cuda', dtype=dtype)
    x[:, 5] = all16
    x[:, 6] = all16 / 2
    x[:, 30] = -all16 / 512
    x[:, 31] = torch.where(torch.isfinite(all16), all16.float() * 0.9921875, 0.0).to(dtype)
    p = ulm_ops.pack_8bit(x)
    codes, exps = op.pack(x)
    finite = exps != 255
    assert np.array_equal(p.exponents.cpu().numpy(), exps) and np.array_equal(p.codes.cpu().numpy()[finite], codes.reshape(-1, 32)[finite])
    assert same(ulm_ops.unpack_8bit(p).double(), op.through(x))
    y = all16.view(-1, 32).clone()
    y[:, 0] = 1.0
    assert same(ulm_ops.unpack_8bit(ulm_ops.pack_8bit(y)).double(), op.through(y))


def test_ties_go_to_even():
    x = (torch.arange(-256, 257, device='cuda').float() / 128)[:512].view(-1, 32).clone()      # halves of a step for blocks of 1 to 2
    x[:, 0] = 1.5
    for dtype in (F32, F16, BF16):
        assert torch.equal(ulm_ops.unpack_8bit(ulm_ops.pack_8bit(x.to(dtype))).double(), op.through(x.to(dtype)))


def test_infinities_and_nans_spoil_their_block_alone():
    for bad in (float('inf'), float('-inf'), float('nan')):
        for dtype in (F16, BF16, F32):
            for at in (0, 37, 100):                       # 100: in the short block at the end
                x = randn(104, dtype, 1)
                want = ulm_ops.unpack_8bit(ulm_ops.pack_8bit(x))
                x[at] = bad
                back = ulm_ops.unpack_8bit(ulm_ops.pack_8bit(x))
                block = torch.arange(104, device='cuda') // 32 == at // 32
                assert back[block].isnan().all() and torch.equal(back[~block], want[~block])


def test_smallest_and_largest_numbers():
    for dtype in (F16, BF16, F32):
        f = torch.finfo(dtype)
        x = torch.tensor([f.max, -f.max, f.tiny, -f.tiny, f.tiny / 4, 0.0, -0.0, f.max / 3] * 8, dtype=dtype, device='cuda').view(8, 8)
        for t in (x, x[:, 2:7].contiguous(), torch.zeros(64, dtype=dtype, device='cuda')):
            assert torch.equal(ulm_ops.unpack_8bit(ulm_ops.pack_8bit(t)).double(), op.through(t))


@pytest.mark.parametrize('form', ['transposed', 'off its alignment', 'columns', 'empty', 'scalar', 'broadcast'])
def test_layouts(form):
    base = randn((37, 64), BF16, 3)
    x = {'transposed': base.t(), 'off its alignment': base.reshape(-1)[3:], 'columns': base[:, 5:18], 'empty': base[:0], 'scalar': base[0, 0], 'broadcast': base[:1].expand(5, 64)}[form]
    back = ulm_ops.unpack_8bit(ulm_ops.pack_8bit(x))
    assert back.shape == x.shape and torch.equal(back.double(), op.through(x))


def test_another_type_and_codes_of_any_layout():
    x = randn((33, 40), F32, 1)
    p = ulm_ops.pack_8bit(x)
    assert torch.equal(ulm_ops.unpack_8bit(p, BF16), op.through(x).to(BF16)) and torch.equal(ulm_ops.unpack_8bit(p, F16), op.through(x).to(F16))
    odd = ulm_ops.Packed8(torch.cat([p.codes.reshape(-1)[:1], p.codes.reshape(-1)])[1:].view(33, 40), p.exponents, F32)
    assert torch.equal(ulm_ops.unpack_8bit(odd), ulm_ops.unpack_8bit(p))
    for bad in (p._replace(exponents=p.exponents[:-1]), p._replace(codes=p.codes.int()), p._replace(exponents=p.exponents.cpu()), p._replace(dtype=torch.int8), p._replace(codes=p.codes.cpu())):
        with pytest.raises(ValueError):
            ulm_ops.unpack_8bit(bad)


def test_every_exponent_and_code():
    """Also those that no tensor packed here has."""
    codes = torch.arange(-128, 128, dtype=torch.int16).to(torch.int8).repeat(256).cuda()
    exps = torch.arange(256, dtype=torch.int16).to(torch.uint8).repeat_interleave(8).cuda()
    back = ulm_ops.unpack_8bit(ulm_ops.Packed8(codes, exps, F32))
    want = torch.from_numpy(op.unpack(codes.cpu().numpy(), exps.cpu().numpy())).float().cuda()
    assert same(back, want)


def test_past_32_bit_offsets():
    n = (1 << 32) + 77
    x = torch.empty(n, dtype=F16, device='cuda')
    row = randn(4096, F16, 9)
    x[:1 << 32].view(-1, 4096).copy_(row.expand(1 << 20, 4096))
    x[1 << 32:] = row[:77]
    back = ulm_ops.unpack_8bit(ulm_ops.pack_8bit(x))
    want = op.through(row).to(F16)
    for at in (0, 1 << 31, (1 << 32) - 4096):
        assert torch.equal(back[at:at + 4096], want)
    assert torch.equal(back[1 << 32:], op.through(row[:77]).to(F16))


# ---------------------------------------------------------------------------
# the gate
# ---------------------------------------------------------------------------
def mask(shape, p, seed):
    return torch.from_numpy(od.keep_mask(math.prod(shape), p, seed).reshape(shape)).cuda()


def gate64(a, b, gy, p=0.0, seed=0):
    """y of the operands, the gradients and y~ of their 8-bit forms, and what the errors of each are relative to."""
    keep, c = (mask(a.shape, p, seed), od.scale(p)) if p else (torch.ones(a.shape, dtype=torch.bool, device='cuda'), 1.0)
    drop = lambda v: torch.where(keep, v * c, 0.0)                 # noqa: E731
    A, B = a.double(), b.double()
    y = drop(A * torch.sigmoid(A) * B)
    A, B, G = op.through(a), op.through(b), drop(gy.double())
    s = torch.sigmoid(A)
    return dict(y=y, da=G * B * s * (1 + A * (1 - s)), db=G * A * s, again=drop(A * s * B), s=s, A=A, B=B, G=G)


def check_gate(a, b, gy, y, da, db, p=0.0, seed=0):
    dtype, t = a.dtype, gate64(a.detach(), b.detach(), gy, p, seed)
    # one rounding of the result; before it the sigmoid of 16-bit tensors is within 2^-18 (1 - s of its complement: within 2^-18 of s, which
    # silu' = s (1 + a (1 - s)) takes at most 1 + |a| fold), fp32 within a few ulps
    slack = 2.0 ** -17 if dtype != F32 else 2.0 ** -21
    assert y.dtype == da.dtype == db.dtype == dtype
    within(y, t['y'], (UNIT[dtype] + slack) * t['y'].abs() + TINY[dtype])
    within(db, t['db'], (UNIT[dtype] + slack) * t['db'].abs() + TINY[dtype])
    within(da, t['da'], UNIT[dtype] * t['da'].abs() + slack * (t['G'] * t['B'] * t['s']).abs() * (1 + t['A'].abs()) + TINY[dtype])


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('shape', [(1, 1), (1, 8), (3, 11), (2, 32), (3, 344), (5, 771), (129, 2048), (4097,)])
@pytest.mark.parametrize('p', [0.0, 0.3, 1.0])
def test_gate(dtype, shape, p):
    a, b, gy = (randn(shape, dtype, 10 + i, 1.5) for i in range(3))
    a.requires_grad_(), b.requires_grad_()
    y = ulm_ops.swiglu_8bit(a, b, p, 1 << 40)
    da, db = torch.autograd.grad(y, [a, b], gy)
    check_gate(a, b, gy, y, da, db, p, 1 << 40)
    if p == 1.0:
        assert not y.any() and not da.any() and not db.any()
    if p == 0.3:
        assert torch.equal(y, ulm_ops.swiglu_dropout(a, b, p, 1 << 40))


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('form', ['halves', 'halves of three dimensions', 'columns apart', 'off its alignment', 'odd width', 'every other row', 'rows unequally apart', 'one transposed', 'broadcast', 'one row'])
@pytest.mark.parametrize('graph', [True, False])
def test_gate_of_operands_of_any_layout(dtype, form, graph):
    base = randn((6, 10, 160), dtype, 1)
    flat = base.view(60, 160)
    a, b = {'halves': lambda: (flat[:, :80], flat[:, 80:]), 'halves of three dimensions': lambda: (base[..., :80], base[..., 80:]), 'columns apart': lambda: (flat[:, :80:2], flat[:, 80::2]),
            'off its alignment': lambda: (flat[:, 1:73], flat[:, 81:153]), 'odd width': lambda: (flat[:, :75], flat[:, 80:155]), 'every other row': lambda: (flat[::2, :80], flat[::2, 80:]),
            'rows unequally apart': lambda: (base[:, ::3, :80], base[:, ::3, 80:]), 'one transposed': lambda: (flat[:, :60], flat[:, :60].t()),
            'broadcast': lambda: (flat[:1, :80].expand(60, 80), flat[1:2, 80:].expand(60, 80)), 'one row': lambda: (flat[3:4, :80], flat[3:4, 80:])}[form]()
    gy = randn(a.shape, dtype, 2)

    def call(p, q):
        p, q = p.detach().requires_grad_(graph), q.detach().requires_grad_(graph)
        y = ulm_ops.swiglu_8bit(p, q, 0.2, 3)
        return (y.detach(), *torch.autograd.grad(y, [p, q], gy)) if graph else (y,)
    for got, want in zip(call(a, b), call(a.contiguous(), b.contiguous())):
        assert torch.equal(got, want)


def test_gate_keeps_little():
    a, b = randn((4096, 2048), BF16, 1).requires_grad_(), randn((4096, 2048), BF16, 2).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = ulm_ops.swiglu_8bit(a, b)
    n = a.numel()
    assert torch.cuda.memory_allocated() - before - 2 * n <= 2 * n * 33 // 32 + (4 << 20)
    del y
    assert torch.cuda.memory_allocated() == before


def test_gate_gradient_against_differences():
    """In fp32 around numbers that the 8-bit form holds exactly, where the gradient is that of the gate itself."""
    a, b = (op.through(randn(64, F32, i)).float().requires_grad_() for i in (1, 2))
    y = ulm_ops.swiglu_8bit(a, b)
    da, db = torch.autograd.grad(y.sum(), [a, b])
    h = 2.0 ** -6
    for x, g, other, first in ((a.detach(), da, b.detach(), True), (b.detach(), db, a.detach(), False)):
        f = lambda t: ulm_ops.swiglu_8bit(*((t, other) if first else (other, t)))      # noqa: E731
        diff = (f(x + h) - f(x - h)).double() / (2 * h)
        # third derivative of silu below 0.6, times |b| < 4 and h^2 / 6; roundings of two values below 16 over 2 h
        within(g, diff, torch.full_like(diff, 0.6 * 4 * h * h / 6 + 16 * 2.0 ** -22 / h))


def test_gate_of_bad_numbers():
    a, b = randn(96, F16, 1), randn(96, F16, 2)
    a[40] = float('inf')
    a.requires_grad_(), b.requires_grad_()
    y = ulm_ops.swiglu_8bit(a, b)
    assert bool((torch.isfinite(y) == (torch.arange(96, device='cuda') != 40)).all())
    da, db = torch.autograd.grad(y, [a, b], torch.ones_like(y))
    block = torch.arange(96, device='cuda') // 32 == 1
    assert da[block].isnan().all() and db[block].isnan().all() and torch.isfinite(da[~block]).all() and torch.isfinite(db[~block]).all()


# ---------------------------------------------------------------------------
# linear layers and the feed-forward
# ---------------------------------------------------------------------------
def close(got, want, unit, k):
    """A product of k terms each, in the 2-norm: a rounding of the result, fp32 sums, and the operands' roundings that `want` has too."""
    assert got.shape == want.shape and float((got.double() - want).norm()) <= (unit + 2.0 ** -22 * math.sqrt(k) + 2.0 ** -24) * float(want.norm())


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('shape,out', [((65, 64), 96), ((2, 33, 40), 24), ((7,), 5), ((1, 72), 8)])
def test_linear(dtype, shape, out):
    x, w = randn(shape, dtype, 1).requires_grad_(), randn((out, shape[-1]), F32, 2, shape[-1] ** -0.5).requires_grad_()
    gy = randn((*shape[:-1], out), dtype, 3)
    with torch.autocast('cuda', dtype=dtype, enabled=dtype != F32):
        y = ulm_ops.linear_8bit(x, w)
        z = ulm_ops.linear(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], gy)
    dx0, _ = torch.autograd.grad(z, [x, w], gy)
    assert torch.equal(y, z) and torch.equal(dx, dx0) and dw.dtype == F32
    close(dw, gy.double().reshape(-1, out).T @ op.through(x.detach()).reshape(-1, shape[-1]), 2.0 ** -24, x.numel() // shape[-1])


@pytest.mark.parametrize('frozen', ['weight', 'x'])
def test_linear_of_a_frozen_side(frozen):
    x, w = randn((64, 256), BF16, 1), randn((128, 256), BF16, 2)
    (x if frozen == 'weight' else w).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = ulm_ops.linear_8bit(x, w)
    assert torch.cuda.memory_allocated() - before - y.numel() * 2 <= (512 if frozen == 'weight' else 64 * 256 * 33 // 32 + 512)
    y.sum().backward()
    assert (w.grad is None) == (frozen == 'weight') and (x.grad is None) == (frozen == 'x')


def ff_case(dtype, shape, ff, p=0.0, seed=7):
    d = shape[-1]
    x, w1, w3, w2 = randn(shape, dtype, 1), randn((ff, d), F32, 2, 1.5 * d ** -0.5), randn((ff, d), F32, 3, 1.5 * d ** -0.5), randn((d + 8, ff), F32, 4, ff ** -0.5)
    return [t.requires_grad_() for t in (x, w1, w3, w2)], randn((*shape[:-1], d + 8), dtype, 5), p, seed


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('shape,ff', [((2, 65, 64), 344), ((130, 128), 352), ((9, 24), 42), ((1, 32), 5)])
@pytest.mark.parametrize('p', [0.0, 0.25])
def test_feed_forward(dtype, shape, ff, p):
    ins, g, p, seed = ff_case(dtype, shape, ff, p)
    with torch.autocast('cuda', dtype=dtype, enabled=dtype != F32):
        out = ulm_ops.feed_forward_8bit(*ins, p, seed)
        grads = torch.autograd.grad(out, ins, g)
        # the same projections by the same library, and what follows from them in 64 bits
        x, w1, w3, w2 = (t.detach() for t in ins)
        a, b = ulm_ops.linear(x, w1), ulm_ops.linear(x, w3)
    rows, d = x.numel() // shape[-1], shape[-1]
    c1, c3, c2 = (w.to(dtype).double() for w in (w1, w3, w2))
    G = g.double().reshape(rows, -1)
    dy = G @ c2
    t = gate64(a.reshape(rows, ff), b.reshape(rows, ff), dy, p, seed)
    u = max(UNIT[dtype], 2.0 ** -20)
    norm = lambda got, want, k: float((got.detach().double().reshape(want.shape) - want).norm()) <= k * u * float(want.norm())      # noqa: E731
    # projections of two widths may be summed in two orders and differ in single roundings, which move codes by one: an eighth of a step's
    # size for bf16, of which a code's step is a sixty-fourth to a thirty-second: three roundings' worth in the 2-norm
    codes = 1.0 if dtype == F32 else 3.0
    assert norm(out, t['y'] @ c2.T, 2.5)
    X = op.through(x.to(dtype)).reshape(rows, d)
    da, db = t['da'], t['db']
    assert norm(grads[0], da @ c1 + db @ c3, 3 * codes) and norm(grads[1], da.T @ X, 3 * codes) and norm(grads[2], db.T @ X, 3 * codes)
    assert norm(grads[3], G.T @ t['again'], 2 * codes)
    for t0, t1 in zip(ins, grads):
        assert t0.shape == t1.shape and t0.dtype == t1.dtype


def test_gradients_near_those_of_the_kept_form():
    ins, g, _, _ = ff_case(BF16, (512, 256), 688)
    with torch.autocast('cuda', dtype=BF16):
        got = torch.autograd.grad(ulm_ops.feed_forward_8bit(*ins), ins, g)
        want = torch.autograd.grad(ulm_ops.linear(ulm_ops.gated_linear(*ins[:3]), ins[3]), ins, g)
    for a, b in zip(got, want):
        # two operands with 0.7 to 0.9 % of noise each in a product, as `pack_8bit` says of normal values, and the gate's slopes
        assert float((a.float() - b.float()).norm()) <= 0.02 * float(b.float().norm())


@pytest.mark.parametrize('asked', [(0,), (1,), (3,), (0, 3), (1, 2), (2,)])
def test_gradients_that_nobody_asked_for_are_not_formed(asked):
    ins, g, _, _ = ff_case(F16, (33, 64), 96)
    with torch.autocast('cuda', dtype=F16):
        whole = torch.autograd.grad(ulm_ops.feed_forward_8bit(*ins), ins, g)
        frozen = [t.detach().requires_grad_(i in asked) for i, t in enumerate(ins)]
        part = torch.autograd.grad(ulm_ops.feed_forward_8bit(*frozen), [frozen[i] for i in asked], g)
    for i, t in zip(asked, part):
        assert float((t - whole[i]).float().norm()) <= 2.0 ** -10 * float(whole[i].float().norm())


def test_weight_gradients_in_place():
    ins, g, _, _ = ff_case(F16, (64, 64), 96)
    ins = [torch.nn.Parameter(t.detach()) for t in ins]
    with torch.autocast('cuda', dtype=F16):
        want = torch.autograd.grad(ulm_ops.feed_forward_8bit(*ins), ins, g)
        flat = torch.zeros(sum(t.numel() for t in ins[1:]), device='cuda')
        at = 0
        for t in ins[1:]:
            t.grad = flat[at:at + t.numel()].view_as(t)
            at += t.numel()
        copies = ulm_ops.weight_copies(ins[1:], F16)
        for k in (1, 2):
            with ulm_ops.wgrad_in_place(), ulm_ops.weight_cast_scope(copies):
                ulm_ops.feed_forward_8bit(*ins).backward(g)
            for t, w in zip(ins[1:], want[1:]):
                assert float((t.grad - k * w).norm()) <= 2.0 ** -9 * k * float(w.norm())


def test_of_no_rows():
    ins, _, _, _ = ff_case(F16, (0, 64), 96)
    with torch.autocast('cuda', dtype=F16):
        out = ulm_ops.feed_forward_8bit(*ins)
        y = ulm_ops.linear_8bit(ins[0], ins[1])
    grads = torch.autograd.grad(out.sum() + y.sum(), ins)
    assert out.shape == (0, 72) and all(g.shape == t.shape and not g.any() for g, t in zip(grads, ins))
    a = torch.zeros(0, 8, device='cuda', requires_grad=True)
    assert torch.autograd.grad(ulm_ops.swiglu_8bit(a, a).sum(), a)[0].shape == (0, 8)


@pytest.mark.parametrize('name', ['swiglu_8bit', 'linear_8bit', 'feed_forward_8bit'])
def test_second_derivatives_are_refused(name):
    x, w = randn((8, 64), F32, 1).requires_grad_(), randn((64, 64), F32, 2).requires_grad_()
    y = {'swiglu_8bit': lambda: ulm_ops.swiglu_8bit(x, x * 2), 'linear_8bit': lambda: ulm_ops.linear_8bit(x, w), 'feed_forward_8bit': lambda: ulm_ops.feed_forward_8bit(x, w, w, w)}[name]()
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='has no second derivative'):
        torch.autograd.grad(g.square().sum(), x)


def test_changed_weights_are_noticed_and_changed_operands_do_not_matter():
    x, w = randn((8, 64), BF16, 1).requires_grad_(), randn((64, 64), BF16, 2).requires_grad_()
    want = torch.autograd.grad(ulm_ops.linear_8bit(x, w).sum(), w)[0]
    y = ulm_ops.linear_8bit(x, w)
    with torch.no_grad():
        x.zero_()                                         # its 8 bits are kept, not it
    assert torch.equal(torch.autograd.grad(y.sum(), w)[0], want)
    y = ulm_ops.linear_8bit(x, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(y.sum(), x)


def test_checkpointed_and_traced():
    from torch.utils.checkpoint import checkpoint
    ins, g, _, _ = ff_case(BF16, (40, 64), 96)
    with torch.autocast('cuda', dtype=BF16):
        want = torch.autograd.grad(ulm_ops.feed_forward_8bit(*ins), ins, g)
        got = torch.autograd.grad(checkpoint(ulm_ops.feed_forward_8bit, *ins, use_reentrant=False), ins, g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    a, b = randn((4, 64), F32, 1), randn((4, 64), F32, 2)
    traced = torch.jit.trace(lambda p, q: ulm_ops.swiglu_8bit(p, q), (a, b))
    assert torch.equal(traced(b, a), ulm_ops.swiglu_8bit(b, a))


def test_another_stream_and_a_graph():
    a, b, gy = (randn((513, 768), BF16, i) for i in (1, 2, 3))
    a.requires_grad_(), b.requires_grad_()

    def step():
        y = ulm_ops.swiglu_8bit(a, b, 0.1, 9)
        return (y.detach(), *torch.autograd.grad(y, [a, b], gy), ulm_ops.unpack_8bit(ulm_ops.pack_8bit(a.detach())))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        again = step()
    with torch.no_grad():
        a.mul_(2), gy.mul_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(again, step()))


@pytest.mark.parametrize('bad', ['types', 'shapes', 'devices', 'integers', 'p', 'seed'])
def test_gate_refusals(bad):
    a, b, p, seed = torch.ones(2, 8, device='cuda'), torch.ones(2, 8, device='cuda'), 0.0, 0
    if bad == 'types': b = b.half()
    if bad == 'shapes': b = b[:1]
    if bad == 'devices': b = b.cpu()
    if bad == 'integers': a, b = a.int(), b.int()
    if bad == 'p': p = 1.5
    if bad == 'seed': seed = 1 << 64
    with pytest.raises(ValueError):
        ulm_ops.swiglu_8bit(a, b, p, seed)


@pytest.mark.parametrize('bad', ['width', 'w3', 'w2', 'w2 on the host', 'double', 'integer weight', 'p', 'vector weight'])
def test_feed_forward_refusals(bad):
    x, w1, w3, w2, p = torch.ones(2, 8, device='cuda'), torch.ones(16, 8, device='cuda'), torch.ones(16, 8, device='cuda'), torch.ones(8, 16, device='cuda'), 0.0
    if bad == 'width': x = x[:, :4]
    if bad == 'w3': w3 = w3[:8]
    if bad == 'w2': w2 = w2[:, :8]
    if bad == 'w2 on the host': w2 = w2.cpu()
    if bad == 'double': x, w1, w3, w2 = x.double(), w1.double(), w3.double(), w2.double()
    if bad == 'integer weight': w1 = w1.int()
    if bad == 'p': p = -0.1
    if bad == 'vector weight': w1 = w1[0]
    with pytest.raises(ValueError):
        ulm_ops.feed_forward_8bit(x, w1, w3, w2, p)
