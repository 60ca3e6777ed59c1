"""Rotary positions against the definition in 64 bits: widths, pairings, layouts, positions near and far, gradients, refusals."""
import pytest
import torch

import ulm_ops
from oracle import rotary as ro

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}          # largest relative error of one rounding
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}       # and absolute, among subnormals
LAYOUTS = ['B,S,H,D', 'B,H,S,D', 'S,B,H,D', 'part of a projection', 'off its alignment', 'columns apart']


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda').to(dtype)


def laid_out(B, H, S, D, dtype, seed, layout):
    if layout == 'B,H,S,D':
        return randn((B, H, S, D), dtype, seed)
    if layout == 'B,S,H,D':
        return randn((B, S, H, D), dtype, seed).transpose(1, 2)
    if layout == 'S,B,H,D':
        return randn((S, B, H, D), dtype, seed).permute(1, 2, 0, 3)
    if layout == 'part of a projection':
        return randn((B, S, H + 3, D), dtype, seed)[:, :, 1:H + 1].transpose(1, 2)
    if layout == 'off its alignment':
        return randn(B * H * S * D + 1, dtype, seed)[1:].view(B, H, S, D)
    return randn((B, H, S, 2 * D), dtype, seed)[..., ::2]


def within(got, x, turns, positions, interleaved=False, factor=1.0, inverse=False):
    want = ro.rotary(x, positions, turns, interleaved, factor, inverse)
    # sine and cosine: the angle's one rounding below pi / 4, the polynomial's, the factor's; two products and a sum: eight units of
    # the pair at most; the angle's last 32 bits, 2^-32 of a turn, are a fortieth of a unit; one rounding of the result
    bound = UNIT[x.dtype] * want.abs() + 9 * 2.0 ** -24 * ro.reach(x, len(turns), interleaved, factor) + TINY[x.dtype]
    assert got.dtype == x.dtype and got.shape == x.shape
    off = (got.detach().double().cpu() - want).abs() - bound
    assert bool((off <= 0).all()), float(off.max())
    n = 2 * len(turns)
    assert torch.equal(got.detach()[..., n:], x.detach()[..., n:])


def case(q, k, turns, positions=None, at=None, interleaved=False, factor=1.0):
    """Forward and backward of both; `at`: the positions on the host."""
    at = list(range(q.shape[2])) if at is None else at
    ins = [t.detach().requires_grad_() for t in (q, k)]
    out = ulm_ops.rotary(*ins, turns.cuda(), positions, interleaved, factor)
    ups = [randn(t.shape, t.dtype, 90 + i) for i, t in enumerate(out)]
    grads = torch.autograd.grad(out, ins, ups)
    for x, y, u, g in zip(ins, out, ups, grads):
        within(y, x, turns, at, interleaved, factor)
        within(g, u, turns, at, interleaved, factor, inverse=True)


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('D,R', [(2, 2), (6, 2), (6, 6), (10, 4), (20, 20), (64, 64), (64, 32), (64, 2), (65, 64), (80, 20), (80, 80), (96, 48), (128, 64), (128, 128), (256, 256), (256, 6), (96, 2), (96, 50), (128, 66), (64, 34),
                                 (256, 210), (512, 130), (4096, 2), (24, 10)])
def test_widths(D, R, dtype, interleaved):
    q, k = laid_out(2, 5, 7, D, dtype, D, 'B,S,H,D'), laid_out(2, 3, 7, D, dtype, R + 1, 'B,S,H,D')
    case(q, k, ulm_ops.rotary_turns(R)[0], interleaved=interleaved)


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('B,Hq,Hk,S', [(1, 1, 1, 1), (1, 1, 7, 1), (3, 12, 12, 201), (1, 9, 2, 1363), (130, 16, 4, 1), (2, 32, 8, 33), (1, 3, 3, 4099)])
def test_head_counts_and_lengths(B, Hq, Hk, S, interleaved):
    dtype = BF16 if S % 2 else F16
    case(laid_out(B, Hq, S, 64, dtype, S, 'part of a projection'), laid_out(B, Hk, S, 64, dtype, S + 1, 'part of a projection'), ulm_ops.rotary_turns(64)[0], interleaved=interleaved)


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('D,R', [(96, 50), (256, 2), (16, 6), (512, 66)])
@pytest.mark.parametrize('B,Hq,Hk,S', [(1, 1, 1, 1), (2, 7, 2, 17), (5, 4, 3, 16), (3, 2, 1, 129), (1, 6, 5, 700)])
def test_rows_of_columns_that_turn_in_no_whole_vectors(D, R, B, Hq, Hk, S, interleaved):
    dtype = (F16, BF16, F32)[(S + Hq) % 3]
    at = torch.randint(-9999, 9999, (B, S), generator=torch.Generator().manual_seed(S))
    case(laid_out(B, Hq, S, D, dtype, S, 'part of a projection'), laid_out(B, Hk, S, D, dtype, S + 1, 'B,H,S,D'), ulm_ops.rotary_turns(R)[0], at.cuda(), at.numpy(), interleaved, 1.25)


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('D', [24, 64])
def test_layouts(layout, dtype, interleaved, D):
    case(laid_out(3, 5, 9, D, dtype, 1, layout), laid_out(3, 2, 9, D, dtype, 2, layout), ulm_ops.rotary_turns(16)[0], interleaved=interleaved)


@pytest.mark.parametrize('form', ['[S]', '[1, S]', '[B, S]', '[B, S] strided', 'one number for all'])
@pytest.mark.parametrize('kind', [torch.int32, torch.int64])
def test_positions(form, kind):
    B, S = 3, 11
    host = torch.randint(0, 1 << 20, (B, S), generator=torch.Generator().manual_seed(5), dtype=kind)
    if form == '[S]':
        host = host[0]
    elif form == '[1, S]':
        host = host[:1]
    dev = host.cuda()
    if form == '[B, S] strided':
        dev = torch.stack([dev, -dev], dim=2).transpose(0, 1)[..., 0].t()
        assert not dev.is_contiguous()
    elif form == 'one number for all':
        host, dev = torch.full((B, S), 77, dtype=kind), torch.tensor(77, dtype=kind, device='cuda').expand(B, S)
    case(laid_out(B, 4, S, 64, BF16, 1, 'B,S,H,D'), laid_out(B, 2, S, 64, BF16, 2, 'B,S,H,D'), ulm_ops.rotary_turns(64)[0], dev, host.numpy())


@pytest.mark.parametrize('at', [0, 1, -1, -4097, (1 << 24) + 1, (1 << 31) - 1, 1 << 31, -(1 << 31), (1 << 40) + 12345, -(1 << 62), (1 << 63) - 1])
def test_positions_near_and_far(at):
    x = laid_out(2, 3, 1, 64, F32, 3, 'B,S,H,D')
    case(x, x, ulm_ops.rotary_turns(64)[0], torch.full((2, 1), at, dtype=torch.int64, device='cuda'), [[at], [at]])


def test_every_eighth_of_a_turn_and_its_neighbours():
    """Angles at the borders of the reduction: position 1 and turns of k / 16, one more and one less."""
    turns = torch.tensor([(k << 60) + d for k in range(-8, 8) for d in (-1, 0, 1, -(1 << 31), 1 << 31, (1 << 32) - 1) if -(1 << 63) <= (k << 60) + d < 1 << 63], dtype=torch.int64)
    x = laid_out(1, 1, 2, 2 * len(turns), F32, 4, 'B,H,S,D')
    case(x, x, turns)


@pytest.mark.parametrize('scaling', [dict(kind='linear', factor=8.0), dict(kind='yarn', factor=8.0, original_length=4096)])
def test_module(scaling):
    m = ulm_ops.Rotary(32, interleaved=True, scaling=scaling).cuda()
    q, k = randn((2, 4, 9, 64), BF16, 1), randn((2, 1, 9, 64), BF16, 2)
    for x, y in zip((q, k), m(q, k)):
        within(y, x, m.turns.cpu(), list(range(9)), True, m.factor)
    y, none = m(q, None)
    assert none is None and torch.equal(y, m(q, k)[0])


def test_the_formula_at_a_million_positions():
    """Against angles formed in float64 from the formula itself, not from the fixed-point turns."""
    turns, _ = ulm_ops.rotary_turns(128)
    x, at = randn((1, 2, 5, 128), F32, 1), torch.tensor([3, 70001, 999983, 1 << 20, 777777])
    y = ulm_ops.rotary(x, None, turns.cuda(), at.cuda())[0].double().cpu()
    a = at.double()[:, None] * 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    p, m = x.double().cpu()[..., :64], x.double().cpu()[..., 64:]
    want = torch.cat([p * a.cos() - m * a.sin(), m * a.cos() + p * a.sin()], dim=-1)
    bound = 2.0 ** -24 * want.abs() + 9 * 2.0 ** -24 * ro.reach(x, 64) + 2.0 ** -30       # float64 angles of 2^20: 2^-33 and their cosines
    assert bool(((y - want).abs() <= bound).all())


def test_turning_back_and_norms():
    q, k = randn((2, 3, 50, 64), F32, 1), randn((2, 3, 50, 64), F32, 2)
    turns = ulm_ops.rotary_turns(64)[0].cuda()
    a, b = ulm_ops.rotary(*ulm_ops.rotary(q, k, turns), turns, inverse=True)
    for x, y in ((q, a), (k, b)):
        assert float((x - y).abs().max()) <= 32 * 2.0 ** -24 * float(x.abs().max()) * 2
    # scores depend on the distance alone
    at = torch.arange(50, device='cuda')
    score = lambda shift: torch.einsum('bhid,bhjd->bhij', *(t.double() for t in ulm_ops.rotary(q, k, turns, at + shift)))    # noqa: E731
    assert float((score(0) - score(123456)).abs().max()) <= 64 * 16 * 40 * 2.0 ** -24


def test_gradient_against_differences():
    x, up = randn((1, 2, 3, 8), F32, 1).requires_grad_(), randn((1, 2, 3, 8), F32, 2)
    turns = ulm_ops.rotary_turns(6)[0].cuda()
    f = lambda t: ulm_ops.rotary(t, None, turns, factor=1.5)[0]            # noqa: E731
    g, = torch.autograd.grad(f(x), x, up)
    for i in range(x.numel()):
        e = torch.zeros(x.numel(), device='cuda')
        e[i] = 0.5
        e = e.view_as(x)
        diff = float(((f(x.detach() + e) - f(x.detach() - e)).double() * up.double()).sum())       # linear: any step will do
        assert abs(diff - float(g.view(-1)[i])) <= 64 * 2.0 ** -24 * 4 * 1.5 * float(up.abs().max()) * 4


def test_second_derivatives_and_unused_outputs():
    turns = ulm_ops.rotary_turns(8)[0].cuda()
    q, k = randn((1, 2, 5, 8), F32, 1).requires_grad_(), randn((1, 1, 5, 8), F32, 2).requires_grad_()
    a, b = ulm_ops.rotary(q, k, turns)
    dq, dk = torch.autograd.grad(a.sum(), [q, k], retain_graph=True)
    assert not dk.any() and dq.any()
    dq, dk = torch.autograd.grad(b.sum(), [q, k], retain_graph=True)
    assert not dq.any() and dk.any()
    g, = torch.autograd.grad((a ** 3).sum(), q, create_graph=True)
    h, = torch.autograd.grad((g * q.detach()).sum(), q)
    want = 6 * a.detach() * ulm_ops.rotary(q.detach(), k.detach(), turns)[0]        # R^T diag(6 a) R x
    want = ulm_ops.rotary(want, None, turns, inverse=True)[0]
    assert float((h - want).abs().max()) <= 2.0 ** -18 * float(want.abs().max())


def test_broadcast_inputs_and_their_gradients():
    base = randn((1, 1, 6, 64), BF16, 1).requires_grad_()
    x = base.expand(3, 4, 6, 64)
    turns = ulm_ops.rotary_turns(64)[0]
    y, _ = ulm_ops.rotary(x, None, turns.cuda())
    within(y, x, turns, list(range(6)))
    up = randn((3, 4, 6, 64), BF16, 2)
    g, = torch.autograd.grad(y, base, up)
    want = ro.rotary(up, list(range(6)), turns, inverse=True).sum((0, 1), keepdim=True)
    assert float((g.double().cpu() - want).abs().max()) <= 13 * 2.0 ** -8 * float(up.abs().max()) * 1.5      # twelve rounded terms and their sum


def test_infinities_stay_in_their_pairs():
    x = torch.ones(1, 1, 2, 8, device='cuda')
    x[0, 0, 1, 1], x[0, 0, 1, 6] = float('inf'), float('nan')
    y, _ = ulm_ops.rotary(x, None, ulm_ops.rotary_turns(6)[0].cuda())
    assert torch.isfinite(y[0, 0, 0]).all()
    assert [bool(v) for v in torch.isfinite(y[0, 0, 1])] == [True, False, True, True, False, True, False, True]


@pytest.mark.parametrize('shape', [(0, 2, 3, 64), (2, 0, 3, 64), (2, 2, 0, 64)])
def test_of_nothing(shape):
    q = torch.zeros(shape, device='cuda', requires_grad=True)
    k = torch.zeros(shape[0], 1, shape[2], 64, device='cuda', requires_grad=True)
    a, b = ulm_ops.rotary(q, k, ulm_ops.rotary_turns(64)[0].cuda())
    assert a.shape == q.shape and b.shape == k.shape and not b.any()
    dq, dk = torch.autograd.grad(a.sum() + b.sum(), [q, k])
    assert dq.shape == q.shape and dk.shape == k.shape


def test_past_32_bit_offsets():
    B, S, D = 3, 1 << 18, 4096                             # 3 x 2^30 elements: 6 GB
    turns = ulm_ops.rotary_turns(64)[0]
    x = torch.empty(B, 1, S, D, device='cuda', dtype=BF16)
    x.copy_((torch.arange(D, device='cuda') % 251 / 64).to(BF16).expand_as(x))
    y, _ = ulm_ops.rotary(x, None, turns.cuda())
    for b, s in ((0, 0), (2, S - 1), (2, 5), (1, 77777)):
        within(y[b:b + 1, :, s:s + 1], x[b:b + 1, :, s:s + 1], turns, [s])


def test_another_stream_and_a_graph():
    q, k = randn((2, 4, 33, 64), BF16, 1), randn((2, 4, 33, 64), BF16, 2)
    m, at = ulm_ops.Rotary(64).cuda(), torch.arange(33, device='cuda')
    want = m(q, k, at)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m(q, k, at)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        again = m(q, k, at)
    q.mul_(2)
    at.add_(1000)                                          # the next step's positions
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, m(q, k, at)))


@pytest.mark.parametrize('bad', ['types', 'integers', 'dimensions', 'batch', 'length', 'width', 'too many turns', 'no turns', 'turns as floats', 'turns on the host',
                                 'positions of another length', 'positions of another batch', 'positions as floats', 'positions on the host', 'positions of three dimensions', 'k on the host'])
def test_refusals(bad):
    q, k = torch.zeros(2, 3, 5, 64, device='cuda', dtype=F16), torch.zeros(2, 1, 5, 64, device='cuda', dtype=F16)
    turns, at = ulm_ops.rotary_turns(64)[0].cuda(), None
    if bad == 'types': k = k.float()
    if bad == 'integers': q, k = q.int(), k.int()
    if bad == 'dimensions': q, k = q[0], k[0]
    if bad == 'batch': k = k[:1]
    if bad == 'length': k = k[:, :, :4]
    if bad == 'width': k = k[..., :32]
    if bad == 'too many turns': turns = ulm_ops.rotary_turns(66)[0].cuda()
    if bad == 'no turns': turns = turns[:0]
    if bad == 'turns as floats': turns = turns.double()
    if bad == 'turns on the host': turns = turns.cpu()
    if bad == 'positions of another length': at = torch.arange(4, device='cuda')
    if bad == 'positions of another batch': at = torch.zeros(3, 5, dtype=torch.int64, device='cuda')
    if bad == 'positions as floats': at = torch.arange(5.0, device='cuda')
    if bad == 'positions on the host': at = torch.arange(5)
    if bad == 'positions of three dimensions': at = torch.zeros(1, 2, 5, dtype=torch.int64, device='cuda')
    if bad == 'k on the host': k = k.cpu()
    with pytest.raises(ValueError):
        ulm_ops.rotary(q, k, turns, at)


def test_negative_positions_of_32_bits_and_both_forms_agree():
    x = laid_out(2, 3, 5, 64, F32, 3, 'B,S,H,D')
    at = torch.tensor([[-3, -1, 0, 1, -(1 << 31)], [(1 << 31) - 1, 7, -7, 5, 2]], dtype=torch.int32)
    case(x, x, ulm_ops.rotary_turns(64)[0], at.cuda(), at.numpy())
    turns = ulm_ops.rotary_turns(64)[0].cuda()
    assert torch.equal(ulm_ops.rotary(x, None, turns, at.cuda())[0], ulm_ops.rotary(x, None, turns, at.long().cuda())[0])


@pytest.mark.parametrize('D,R', [(64, 64), (80, 20), (65, 62), (9, 4), (96, 50), (64, 2)])
@pytest.mark.parametrize('interleaved', [False, True])
def test_in_place_through_the_library(D, R, interleaved):
    """Outputs may be the inputs; what passes through is then left alone."""
    import ctypes as C

    import _native as N
    x = randn((2, 7, 3, D), BF16, 1)
    turns = ulm_ops.rotary_turns(R)[0].cuda()
    want, _ = ulm_ops.rotary(x.transpose(1, 2), None, turns, None, interleaved)
    a = N.RotaryArgs()
    a.q = a.qo = x.data_ptr()
    a.turns = turns.data_ptr()
    a.q_sb = a.qo_sb = 21 * D
    a.q_ss = a.qo_ss = 3 * D
    a.q_sh = a.qo_sh = D
    a.B, a.Hq, a.Hk, a.S, a.D, a.R, a.dtype, a.interleaved, a.factor = 2, 3, 0, 7, D, R, N.ULM_BF16, int(interleaved), 1.0
    a.stream = torch.cuda.current_stream().cuda_stream
    N.check(N.lib().ulm_rotary(C.byref(a)), 'rotary')
    assert torch.equal(x.transpose(1, 2), want)
