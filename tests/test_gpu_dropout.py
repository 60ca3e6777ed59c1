"""Dropout with an unstored mask against plain forms in 64 bits: alone, in the gate, and in residual add + norm."""
import math

import numpy as np
import pytest
import torch

import ulm_ops
from oracle import dropout as od

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}          # largest relative error of one rounding
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}       # and absolute, among subnormals


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=gen(seed), device='cuda') * std).to(dtype)


def mask(shape, p, seed):
    return torch.from_numpy(od.keep_mask(math.prod(shape), p, seed).reshape(shape)).cuda()


def drop64(v, keep, p):
    return torch.where(keep, v * od.scale(p), 0.0)


def within(got, want, bound):
    """Every element within its own bound."""
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


# ---------------------------------------------------------------------------
# alone
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('n', [1, 3, 4, 7, 8, 9, 4095, 4096, 4101, 70003])
@pytest.mark.parametrize('p', [0.0, 1e-9, 0.1, 0.5, 1 - 1e-9, 1.0])
def test_dropout_drops_what_the_definition_drops(dtype, n, p):
    seed = n * 0x9E3779B97F4A7C15 % (1 << 64)
    x = randn(n, dtype, n).requires_grad_()
    gy = randn(n, dtype, n + 1)
    keep = mask((n,), p, seed)
    y = ulm_ops.dropout(x, p, seed)
    dx, = torch.autograd.grad(y, x, gy)
    # one fp32 product by the rounded factor and one rounding: to the bit
    s = torch.tensor(od.scale(p), dtype=F32, device='cuda')
    for got, v in ((y, x.detach()), (dx, gy)):
        assert got.dtype == dtype and torch.equal(got, torch.where(keep, v.float() * s, 0.0).to(dtype))


@pytest.mark.parametrize('form', ['transposed', 'off its alignment', 'columns', 'empty', 'scalar'])
def test_dropout_of_any_layout(form):
    base = randn((37, 64), BF16, 3)
    x = {'transposed': base.t(), 'off its alignment': base.reshape(-1)[3:], 'columns': base[:, 5:18], 'empty': base[:0], 'scalar': base[0, 0]}[form]
    x = x.detach().requires_grad_()
    y = ulm_ops.dropout(x, 0.3, 17)
    assert y.shape == x.shape
    s = torch.tensor(od.scale(0.3), dtype=F32, device='cuda')
    assert torch.equal(y, torch.where(mask(tuple(x.shape), 0.3, 17), x.detach().float() * s, 0.0).to(BF16))
    assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape


def test_dropout_past_32_bit_offsets():
    n = (1 << 32) + 13
    x = torch.ones(n, dtype=F16, device='cuda')
    y = ulm_ops.dropout(x, 0.5, 77)
    for at in (0, (1 << 31) - 8, (1 << 32) - 64):
        m = min(128, n - at)
        assert np.array_equal(y[at:at + m].cpu().numpy() == 2, od.keep_mask(m, 0.5, 77, at))


def test_what_is_dropped_is_zero_whatever_it_held():
    for bad in (float('inf'), float('-inf'), float('nan')):
        x = torch.full((4096,), bad, device='cuda', dtype=F16)
        keep = mask((4096,), 0.5, 5)
        y = ulm_ops.dropout(x, 0.5, 5)
        assert not y[~keep].any() and not torch.isfinite(y[keep]).any()
        ones = torch.ones_like(x)
        z = ulm_ops.swiglu_dropout(ones, x, 0.5, 5)
        assert not z[~keep].any() and not torch.isfinite(z[keep]).any()
        x_new, _ = ulm_ops.dropout_add_rms_norm(torch.ones(4, 1024, device='cuda'), x.view(4, 1024), torch.ones(1024, device='cuda'), 0.5, 5)
        assert bool((x_new.view(-1)[~keep] == 1).all()) and not torch.isfinite(x_new.view(-1)[keep]).any()


def test_dropout_on_another_stream_and_in_a_graph():
    x = randn((513, 768), BF16, 1)
    want = ulm_ops.dropout(x, 0.1, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ulm_ops.dropout(x, 0.1, 9)
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    assert torch.equal(got, want)
    with torch.cuda.graph(graph, stream=side):
        again = ulm_ops.dropout(x, 0.1, 9)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, ulm_ops.dropout(x, 0.1, 9))


def test_dropout_can_be_differentiated_twice():
    x = randn(100, F32, 4).requires_grad_()
    y = ulm_ops.dropout(x, 0.25, 3)
    g, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
    h, = torch.autograd.grad(g.sum(), x)
    s, k = od.scale(0.25), mask((100,), 0.25, 3)
    want = torch.where(k, 6 * s ** 3 * x.detach().double(), 0.0)
    within(h, want, 2.0 ** -20 * want.abs())               # some ten fp32 roundings


# ---------------------------------------------------------------------------
# the gate
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('shape', [(1, 1), (1, 8), (3, 344), (5, 771), (129, 2048)])
@pytest.mark.parametrize('p', [0.1, 0.7])
def test_gate(dtype, shape, p):
    a, b, gy = (randn(shape, dtype, 10 + i) for i in range(3))
    a.requires_grad_(), b.requires_grad_()
    y = ulm_ops.swiglu_dropout(a, b, p, 1 << 40)
    da, db = torch.autograd.grad(y, [a, b], gy)
    keep = mask(shape, p, 1 << 40)
    A, B, G = a.detach().double(), b.detach().double(), drop64(gy.double(), keep, p)
    s = torch.sigmoid(A)
    # one rounding of the result; before it the sigmoid of 16-bit tensors is within 2^-18 (1 - s of its complement: within
    # 2^-18 of s, which silu' = s (1 + a (1 - s)) takes at most 1 + |a| fold), fp32 within a few ulps
    slack = 2.0 ** -17 if dtype != F32 else 2.0 ** -21
    for got, want, size in ((y, drop64(A * s * B, keep, p), (A * s * B).abs() * od.scale(p)), (db, G * A * s, (G * A * s).abs()),
                            (da, G * B * s * (1 + A * (1 - s)), (G * B * s).abs() * (1 + A.abs()))):
        assert got.dtype == dtype
        within(got, want, UNIT[dtype] * want.abs() + slack * size + TINY[dtype])
    assert not y[~keep].any() and not da[~keep].any() and not db[~keep].any()


def test_gate_without_dropout_is_the_gate():
    a, b = randn((33, 96), BF16, 1), randn((33, 96), BF16, 2)
    assert torch.equal(ulm_ops.swiglu_dropout(a, b, 0.0, 5), ulm_ops.swiglu(a, b))


def test_gate_gradient_against_differences():
    a, b = randn(64, F32, 1).requires_grad_(), randn(64, F32, 2).requires_grad_()
    y = ulm_ops.swiglu_dropout(a, b, 0.25, 8)
    da, db = torch.autograd.grad(y.sum(), [a, b])
    h = 2.0 ** -6
    for x, g, other, first in ((a.detach(), da, b.detach(), True), (b.detach(), db, a.detach(), False)):
        f = lambda t: ulm_ops.swiglu_dropout(*((t, other) if first else (other, t)), 0.25, 8)      # noqa: E731
        diff = (f(x + h) - f(x - h)).double() / (2 * h)    # elementwise: every element its own difference
        # third derivative of silu below 0.6, times |b| < 4 and h^2 / 6; roundings of two values below 16 over 2 h
        within(g, diff, torch.full_like(diff, 0.6 * 4 * od.scale(0.25) * h * h / 6 + 16 * 2.0 ** -22 / h))


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('ff', [344, 352, 42])
def test_gated_linear_with_dropout(dtype, ff):
    x, w1, w3 = randn((2, 65, 64), dtype, 1), randn((ff, 64), F32, 2, 0.125), randn((ff, 64), F32, 3, 0.125)
    gy = randn((2, 65, ff), dtype, 4)
    ins = [x.requires_grad_(), w1.requires_grad_(), w3.requires_grad_()]
    with torch.autocast('cuda', dtype=dtype, enabled=dtype != F32):
        y = ulm_ops.gated_linear(x, w1, w3, 0.2, 31)
        z = ulm_ops.swiglu_dropout(ulm_ops.linear(x, w1), ulm_ops.linear(x, w3), 0.2, 31)
    assert torch.equal(y == 0, z == 0)
    # both round the same projections, which library GEMMs of two widths may sum in two orders
    for got, want in zip((y, *torch.autograd.grad(y, ins, gy)), (z, *torch.autograd.grad(z, ins, gy))):
        assert float((got.double() - want.double()).norm()) <= 3 * max(UNIT[dtype], 2.0 ** -20) * float(want.double().norm())


# ---------------------------------------------------------------------------
# residual add + norm
# ---------------------------------------------------------------------------
def norm64(x, b, w, keep, p, gx, gy, eps):
    X, W, GY = x.double() + drop64(b.double(), keep, p), w.double(), gy.double()
    r = torch.rsqrt(X.square().mean(-1, keepdim=True) + eps)
    U, G = X * r, GY * W
    dz = r * (G - U * (G * U).mean(-1, keepdim=True))
    return dict(x_new=X, y=U * W, dx=dz + gx.double(), dw=(GY * U).reshape(-1, U.shape[-1]).sum(0), r=r, U=U, G=G, GY=GY)


def norm_case(x, b, w, p, seed, gx, gy, eps=1e-6):
    dtype, d = b.dtype, x.shape[-1]
    ins = [t.detach().requires_grad_() for t in (x, b, w)]
    x_new, y = ulm_ops.dropout_add_rms_norm(*ins, p, seed, eps=eps)
    dx, db, dw = torch.autograd.grad([x_new, y], ins, [gx, gy])
    keep = mask(tuple(x.shape), p, seed)
    t = norm64(x, b, w, keep, p, gx, gy, eps)
    assert (x_new.dtype, y.dtype, dx.dtype, db.dtype, dw.dtype) == (F32, dtype, F32, dtype, w.dtype)
    u = UNIT[F32]
    ax = x.double().abs() + drop64(b.double().abs(), keep, p)
    within(x_new, t['x_new'], 4 * u * ax)
    # the statistic is a sum of d squares in chains of at most 32 + log2 steps, a reciprocal root and two products; each
    # term of x_new carries its own rounding
    stat = 64 * u
    big = ax.max(-1, keepdim=True).values * t['r']         # 1 where the residual does not cancel
    within(y, t['y'], (UNIT[dtype] + stat) * t['y'].abs() + 8 * u * big * w.double().abs() + TINY[dtype])
    row = t['r'] * (t['G'].abs() + t['U'].abs() * (t['G'] * t['U']).abs().mean(-1, keepdim=True)) * (1 + big)
    within(dx, t['dx'], stat * row + 2 * u * gx.double().abs())
    want = drop64(t['dx'], keep, p)
    within(db, want, UNIT[dtype] * want.abs() + od.scale(p) * (stat * row + 2 * u * gx.double().abs()) + TINY[dtype])
    assert not db[~keep].any()
    n = t['GY'].reshape(-1, d).shape[0]
    size = (t['GY'].abs() * (t['U'].abs() + big)).reshape(-1, d).sum(0)
    within(dw, t['dw'], (UNIT[w.dtype] * t['dw'].abs() if w.dtype != F32 else 0) + (stat + u * (math.isqrt(n) + 64)) * size)


@pytest.mark.parametrize('d', [4, 8, 12, 128, 260, 768, 772, 1020, 1024, 1028, 2048, 3076, 4100, 6152, 8188, 8192])
@pytest.mark.parametrize('rows', [1, 2, 150])
def test_norm(d, rows):
    dtype = F16 if (d + rows) % 3 else BF16
    x, b, gx, gy = randn((rows, d), F32, 1, 2.0), randn((rows, d), dtype, 2), randn((rows, d), F32, 3), randn((rows, d), dtype, 4)
    norm_case(x, b, 1 + randn(d, F32, 5, 0.1), 0.1, d * rows + (1 << 33), gx, gy)


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('p', [0.0, 0.5, 1.0])
def test_norm_of_many_rows(dtype, p):
    x, b, gx, gy = randn((3, 1201, 768), F32, 1, 2.0), randn((3, 1201, 768), dtype, 2), randn((3, 1201, 768), F32, 3), randn((3, 1201, 768), dtype, 4)
    norm_case(x, b, 1 + randn(768, F32, 5, 0.1), p, 12, gx, gy)


@pytest.mark.parametrize('form', ['strided', 'eight bytes', 'two bytes', 'weight 16 bits'])
def test_norm_of_any_layout(form):
    rows, d = 9, 768
    x, b, gx, gy = randn((rows, d + 8), F32, 1)[:, :d], randn((rows, d + 8), BF16, 2), randn((rows, d), F32, 3), randn((rows, d), BF16, 4)
    b = b[:, 4:d + 4] if form == 'eight bytes' else b[:, 1:d + 1] if form == 'two bytes' else b[:, 8:]
    norm_case(x, b, (1 + randn(d, F32, 5, 0.1)).to(BF16 if form == 'weight 16 bits' else F32), 0.3, 4, gx, gy)


def test_norm_of_rows_of_zeros_and_of_no_rows():
    z = torch.zeros(3, 64, device='cuda')
    x_new, y = ulm_ops.dropout_add_rms_norm(z, z.half(), torch.ones(64, device='cuda'), 0.5, 1)
    assert not x_new.any() and not y.any()
    x, b, w = torch.zeros(0, 64, device='cuda', requires_grad=True), torch.zeros(0, 64, device='cuda', dtype=F16, requires_grad=True), torch.ones(64, device='cuda', requires_grad=True)
    x_new, y = ulm_ops.dropout_add_rms_norm(x, b, w, 0.5, 1)
    dx, db, dw = torch.autograd.grad([x_new.sum() + y.float().sum()], [x, b, w])
    assert x_new.shape == y.shape == dx.shape == db.shape == (0, 64) and dw.shape == (64,) and not dw.any()


@pytest.mark.parametrize('used', ['x_new', 'y'])
def test_norm_with_one_output_used(used):
    x, b, w = randn((5, 96), F32, 1).requires_grad_(), randn((5, 96), F16, 2).requires_grad_(), (1 + randn(96, F32, 3, 0.1)).requires_grad_()
    keep = mask((5, 96), 0.4, 6)
    x_new, y = ulm_ops.dropout_add_rms_norm(x, b, w, 0.4, 6)
    zero = torch.zeros(5, 96, device='cuda')
    gx, gy = (randn((5, 96), F32, 4), zero.half()) if used == 'x_new' else (zero, randn((5, 96), F16, 4))
    dx, db, dw = torch.autograd.grad(x_new if used == 'x_new' else y, [x, b, w], gx if used == 'x_new' else gy)
    t = norm64(x.detach(), b.detach(), w.detach(), keep, 0.4, gx, gy, 1e-6)
    scale = float(t['dx'].abs().max())
    within(dx, t['dx'], torch.full_like(t['dx'], 2.0 ** -17 * scale))
    within(db, drop64(t['dx'], keep, 0.4), torch.full_like(t['dx'], 2 * UNIT[F16] * scale))
    within(dw, t['dw'], torch.full_like(t['dw'], 2.0 ** -17 * (1 + float(t['dw'].abs().max()))))


def test_norm_gradient_against_differences():
    rows, d, h = 2, 32, 2.0 ** -5
    x, b, w = randn((rows, d), F32, 1, 2.0), randn((rows, d), F16, 2), 1 + randn(d, F32, 3, 0.1)
    gx, gy = randn((rows, d), F32, 4), randn((rows, d), F16, 5)
    ins = [x.requires_grad_(), b, w]
    x_new, y = ulm_ops.dropout_add_rms_norm(*ins, 0.25, 2)
    dx, = torch.autograd.grad([x_new, y], [x], [gx, gy])
    # the fp32 output is exact to 2^-23; y is rounded to fp16, so its differences are taken of a float64 restatement whose
    # forward the tests above hold the kernel to
    keep = mask((rows, d), 0.25, 2)

    def f(v):
        t = norm64(v, b, w, keep, 0.25, gx, gy, 1e-6)
        return float((t['x_new'] * gx.double()).sum() + (t['y'] * gy.double()).sum())
    for i in range(0, rows * d, 7):
        e = torch.zeros(rows * d, device='cuda', dtype=torch.float64)
        e[i] = h
        e = e.view(rows, d)
        diff = (f(x.detach().double() + e) - f(x.detach().double() - e)) / (2 * h)
        # third derivatives of x / rms over rows of deviation 2: below 1 a unit of gradient, |gradient| summed below 2 d
        assert abs(float(dx.view(-1)[i]) - diff) <= 2 * d * h * h / 6 + 2.0 ** -17 * 8


@pytest.mark.parametrize('bad', ['p', 'x dtype', 'branch dtype', 'shapes', 'width', 'too wide', 'weight', 'no width'])
def test_norm_refusals(bad):
    d = {'width': 66, 'too wide': 8196, 'no width': 0}.get(bad, 64)
    x, b, w = torch.ones(2, d, device='cuda'), torch.ones(2, d, device='cuda', dtype=F16), torch.ones(d, device='cuda')
    if bad == 'x dtype': x = x.half()
    if bad == 'branch dtype': b = b.float()
    if bad == 'shapes': b = b[:1]
    if bad == 'weight': w = w[:-4]
    with pytest.raises(ValueError):
        ulm_ops.dropout_add_rms_norm(x, b, w, 2.0 if bad == 'p' else 0.1, 0)


def test_dropout_refusals():
    x = torch.ones(8, device='cuda')
    for call in (lambda: ulm_ops.dropout(x, -0.1, 0), lambda: ulm_ops.dropout(x, float('nan'), 0), lambda: ulm_ops.dropout(x.long(), 0.1, 0),
                 lambda: ulm_ops.dropout(x.double(), 0.1, 0), lambda: ulm_ops.swiglu_dropout(x, x[:4], 0.1, 0),
                 lambda: ulm_ops.swiglu_dropout(x, x.half(), 0.1, 0), lambda: ulm_ops.swiglu_dropout(x, x, 1.1, 0)):
        with pytest.raises(ValueError):
            call()
