"""The loss without logits against its definition in 64 bits: values, gradients, masks, sizes that end inside tiles, pieces."""
import contextlib
import math

import pytest
import torch

import flash_attn_v100_cuda as fa
import ulm_ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
G_TINY = {F16: 2.0 ** -39, BF16: 2.0 ** -130}                       # spacing of the 16-bit softmax near zero
OUT_TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -130, F32: 2.0 ** -145}


def case(rows, V, d, dtype, seed=1, ignored=0.1, ignore_index=0, std=1.4):
    g = torch.Generator(device='cuda').manual_seed(seed)
    h = torch.randn((rows, d), generator=g, device='cuda').to(dtype)
    w = (torch.randn((V, d), generator=g, device='cuda') * (std / math.sqrt(d))).to(dtype)
    t = torch.randint(0, V, (rows,), generator=g, device='cuda')
    t[torch.rand(rows, generator=g, device='cuda') < ignored] = ignore_index
    return h, w, t


def counted(t, V, ignore_index):
    return (t != ignore_index) & (t >= 0) & (t < V)


def definition(h, w, t, ignore_index, denominator=None):
    """The loss's value, gradient factors and the bounds on what the kernels' roundings may do to them, in 64 bits."""
    rows, d = h.shape
    V = w.shape[0]
    H, W, ok = h.double(), w.double(), counted(t, V, ignore_index)
    n = max(1, int((t != ignore_index).sum())) if denominator is None else denominator
    z = H @ W.t()
    logp = torch.log_softmax(z, 1)
    at, tt = torch.arange(rows, device='cuda'), t.clamp(0, V - 1)
    row_loss = torch.where(ok, -logp[at, tt], 0.0)
    prob = logp.exp()
    g = prob.clone()
    g[at, tt] -= 1.0
    g = torch.where(ok[:, None], g, 0.0)
    # a logit: exact products summed in fp32, sixteen a step; the softmax of it: two such errors, the row sum's and 2^x's
    e_z = (d / 16 + 4) * 2.0 ** -23 * (H.abs() @ W.abs().t())
    e_p = 2 * (e_z.amax(1, keepdim=True) + 2.0 ** -19)
    e_loss = (e_p[:, 0] + 2.0 ** -22 * (1 + row_loss.abs())) * ok
    e_g = UNIT[h.dtype] * g.abs() + prob * e_p * ok[:, None] + G_TINY[h.dtype]
    return dict(loss=float(row_loss.sum() / n), e_loss=float(e_loss.sum() / n) + 2.0 ** -23 * float(row_loss.sum() / n), n=n,
                g=g, e_g=e_g, H=H, W=W, prob=prob, e_p=e_p)


def check(loss, dh, dw, h, w, t, ignore_index, up=1.0, denominator=None, w_out=None):
    """``w_out``: the type the weight's gradient is rounded to (default: the operands')."""
    D = definition(h, w, t, ignore_index, denominator)
    assert abs(float(loss) - D['loss']) <= D['e_loss']
    f, u = up / D['n'], UNIT[h.dtype]
    for got, left, right, e_left, out in ((dh, D['g'], D['W'], D['e_g'], h.dtype), (dw, D['g'].t(), D['H'], D['e_g'].t(), w_out or h.dtype)):
        if got is None:
            continue
        want = f * (left @ right)
        k = left.shape[1]
        # every element: the 16-bit softmax's errors all one way, the fp32 sum's, and the result's one rounding
        size = abs(f) * (left.abs() @ right.abs())
        bound = abs(f) * (e_left @ right.abs()) + (k / 16 + 80) * 2.0 ** -23 * size + UNIT[out] * want.abs() + OUT_TINY[out]
        off = (got.double() - want).abs()
        assert got.dtype == out and bool((off <= bound).all()), float((off - bound).max())
        # all of them together: roundings are independent and uniform, a third of their bound squared; twice that
        var = (u * u / 3) * f * f * (left.square() @ right.square()) + (UNIT[out] ** 2 / 3) * want.square()
        systematic = (k / 16 + 80) * 2.0 ** -23 * size + abs(f) * ((e_left - u * left.abs()).clamp(min=0) @ right.abs())
        assert float(off.norm()) <= 2 * float(var.sum().sqrt()) + float(systematic.norm()) + OUT_TINY[out] * off.numel() ** 0.5


@contextlib.contextmanager
def piece_bytes(n):
    before, ulm_ops.PIECE_BYTES = ulm_ops.PIECE_BYTES, n
    try:
        yield
    finally:
        ulm_ops.PIECE_BYTES = before


def run(h, w, t, up=1.0, **kw):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ulm_ops.streamed_cross_entropy(h, w, t, **kw)
    dh, dw = torch.autograd.grad(loss, [h, w], torch.tensor(up, device='cuda'))
    fa.check_status()
    return loss.detach(), dh, dw


@pytest.mark.parametrize('rows', [1, 2, 127, 128, 129, 700])
@pytest.mark.parametrize('V', [1, 2, 7, 63, 255, 256, 257, 1000, 5003])
def test_sizes_that_end_inside_tiles(rows, V):
    dtype = F16 if (rows + V) % 2 else BF16
    h, w, t = case(rows, V, 200, dtype, ignore_index=-100)
    check(*run(h, w, t, up=float(rows), ignore_index=-100), h, w, t, -100, up=float(rows))


@pytest.mark.parametrize('d', [8, 16, 64, 72, 128, 256, 264, 768, 1024, 1288])
@pytest.mark.parametrize('dtype', [F16, BF16])
def test_widths(d, dtype):
    h, w, t = case(333, 1500, d, dtype)
    check(*run(h, w, t, up=333.0), h, w, t, 0, up=333.0)


@pytest.mark.parametrize('rows,V', [(5, 32000), (300, 32000), (3000, 4096), (9001, 600), (40, 50021)])
@pytest.mark.parametrize('dtype', [F16, BF16])
def test_shapes_of_training(rows, V, dtype):
    h, w, t = case(rows, V, 768, dtype)
    check(*run(h, w, t, up=float(rows)), h, w, t, 0, up=float(rows))


@pytest.mark.parametrize('rows,V,columns', [(300, 1000, 256), (1000, 1025, 256), (129, 5003, 1024), (2000, 4096, 1536), (4000, 2900, 768), (10000, 1100, 512)])
def test_pieces_of_the_vocabulary(rows, V, columns):
    h, w, t = case(rows, V, 328, BF16)
    with piece_bytes(2 * rows * columns):
        loss, dh, dw = run(h, w, t)
    check(loss, dh, dw, h, w, t, 0)
    whole = run(h, w, t)
    assert torch.equal(loss, whole[0])
    with piece_bytes(0):                                   # the least: 256 columns
        check(*run(h, w, t), h, w, t, 0)


def test_the_workspace_does_not_grow_with_the_vocabulary():
    def peak(V):
        h, w, t = case(4096, V, 64, BF16)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        run(h, w, t)
        return torch.cuda.max_memory_allocated() - before - 2 * w.numel()          # without the weight's gradient
    with piece_bytes(16 << 20):
        a, b = peak(8192), peak(32768)
    # row statistics: 16 bytes per row and group of column tiles; one 4096 x 32768 matrix of 16 bits would be 256 MB
    assert b <= a + 16 * 4096 * 128 and b < 64 << 20


def test_sharp_and_flat_rows():
    for std in (1e-3, 30.0):
        for dtype in (F16, BF16):
            h, w, t = case(257, 3000, 256, dtype, std=std)
            check(*run(h, w, t, up=257.0), h, w, t, 0, up=257.0)


@pytest.mark.parametrize('what', ['all ignored', 'none', 'negative', 'past the end'])
def test_masks(what):
    h, w, t = case(150, 300, 64, BF16, ignored=0.0)
    if what == 'all ignored':
        t[:] = 0
    elif what == 'negative':
        t[::3] = -5
    elif what == 'past the end':
        t[::3] = 300
    loss, dh, dw = run(h, w, t)
    check(loss, dh, dw, h, w, t, 0)
    if what == 'all ignored':
        assert float(loss) == 0 and not dh.any() and not dw.any()
    assert not dh[~counted(t, 300, 0)].any()


def test_ignored_rows_may_hold_anything_finite():
    h, w, t = case(150, 300, 64, BF16, ignored=0.0)
    t[::4] = 0
    other = h.clone()
    other[::4] = 3e38
    a, b = run(h, w, t), run(other, w, t)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])


def test_nan_and_infinite_rows_stay_in_their_rows():
    h, w, t = case(150, 300, 64, F16, ignored=0.0, ignore_index=-100)
    for bad in (float('nan'), float('inf'), float('-inf')):
        x = h.clone()
        x[70, 3] = bad
        hl = x.requires_grad_()
        loss = ulm_ops.streamed_cross_entropy(hl, w, t, ignore_index=-100)
        dh, = torch.autograd.grad(loss, hl)
        assert math.isnan(float(loss))
        rows = torch.arange(150, device='cuda') != 70
        assert torch.isfinite(dh[rows]).all() and not torch.isfinite(dh[70]).all()


def test_minus_infinity_logits_have_no_probability():
    # column 5's logit is -inf in every row: as if it were not there
    h, w, t = case(40, 300, 64, F32, ignored=0.0, ignore_index=-100)
    h[:, 0] = 1.0
    w[:, 0] = 0.0
    w[5, 0] = float('-inf')
    t[t == 5] = 6
    h, w = h.to(BF16), w.to(BF16)
    loss, _, _ = run(h, w, t, ignore_index=-100)
    keep = torch.arange(300, device='cuda') != 5
    want = definition(h, w[keep], torch.where(t > 5, t - 1, t), -100)
    assert abs(float(loss) - want['loss']) <= want['e_loss']


def test_strided_operands_and_other_streams():
    h, w, t = case(130, 520, 128, BF16)
    wide_h, wide_w = torch.zeros(130, 256, device='cuda', dtype=BF16), torch.zeros(520, 136, device='cuda', dtype=BF16)
    wide_h[:, 64:192], wide_w[:, 8:] = h, w
    odd = torch.zeros(130 * 128 + 1, device='cuda', dtype=BF16)[1:].view(130, 128)
    odd.copy_(h)
    want = run(h, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run(wide_h[:, 64:192], wide_w[:, 8:], t), run(odd, w, t), run(h.t().contiguous().t(), w, t)]
    torch.cuda.current_stream().wait_stream(side)
    for g in got:
        for a, b in zip(g, want):
            assert torch.equal(a, b)


def test_broadcast_rows():
    h, w, t = case(1, 520, 128, BF16)
    t = torch.arange(1, 6, device='cuda')
    for a, b in zip(run(h.expand(5, 128), w, t), run(h.expand(5, 128).contiguous(), w, t)):
        assert torch.equal(a, b)


def test_in_a_graph():
    h, w, t = case(700, 3000, 128, BF16)
    h.requires_grad_(), w.requires_grad_()
    up = torch.ones((), device='cuda')

    def step():
        loss = ulm_ops.streamed_cross_entropy(h, w, t)
        return [loss.detach(), *torch.autograd.grad(loss, [h, w], up)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        h.mul_(1.5)
        t[::7] = 0
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_the_same_bits_every_time():
    h, w, t = case(1111, 3001, 776, F16)
    first = run(h, w, t)
    for _ in range(3):
        for a, b in zip(run(h, w, t), first):
            assert torch.equal(a, b)


def test_backward_twice():
    h, w, t = case(77, 500, 64, BF16)
    h.requires_grad_(), w.requires_grad_()
    loss = ulm_ops.streamed_cross_entropy(h, w, t)
    a = torch.autograd.grad(loss, [h, w], retain_graph=True)
    b = torch.autograd.grad(loss, [h, w])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize('which', ['hidden', 'weight'])
def test_one_gradient_alone(which):
    h, w, t = case(77, 500, 64, BF16)
    _, dh, dw = run(h, w, t)
    (h if which == 'hidden' else w).requires_grad_()
    loss = ulm_ops.streamed_cross_entropy(h, w, t)
    loss.backward()
    assert torch.equal(h.grad, dh) if which == 'hidden' else torch.equal(w.grad, dw)
    assert (w if which == 'hidden' else h).grad is None


@pytest.mark.parametrize('denominator', [7, 123.5, -2.0, 'scalar', 'vector'])
def test_denominators(denominator):
    h, w, t = case(60, 300, 64, BF16)
    n = {'scalar': torch.tensor(50.0, device='cuda'), 'vector': torch.tensor([50.0], device='cuda')}.get(denominator, denominator)
    h.requires_grad_(), w.requires_grad_()
    loss = ulm_ops.streamed_cross_entropy(h, w, t, denominator=n)
    assert loss.shape == ((1,) if denominator == 'vector' else ())
    dh, dw = torch.autograd.grad(loss.sum(), [h, w])
    m = float(n)
    D = definition(h.detach(), w.detach(), t, 0, m)
    assert abs(float(loss) - D['loss']) <= abs(D['e_loss'])
    want = D['g'] @ D['W'] / m
    assert float((dh.double() - want).norm()) <= 2 * UNIT[BF16] * float(want.norm())


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('rows,V,d', [(200, 700, 128), (5000, 700, 128), (300, 40000, 264)])       # whole tiles, cut ones, both
def test_fp32_parameters_under_autocast(dtype, rows, V, d):
    h, w, t = case(rows, V, d, dtype)
    wp = w.float().requires_grad_()
    hp = h.float().requires_grad_()
    with torch.autocast('cuda', dtype=dtype):
        loss = ulm_ops.streamed_cross_entropy(hp, wp, t)
    dh, dw = torch.autograd.grad(loss, [hp, wp], torch.tensor(float(rows), device='cuda'))
    assert dh.dtype == F32 and dw.dtype == F32
    check(loss.detach(), dh.to(dtype), dw, h, w, t, 0, up=float(rows), w_out=F32)
    # into existing gradients, as the data-parallel step has it
    wp.grad = torch.full_like(wp, 0.5)
    with torch.autocast('cuda', dtype=dtype), ulm_ops.wgrad_in_place():
        (ulm_ops.streamed_cross_entropy(hp, wp, t) * rows).backward()
    assert float((wp.grad - 0.5 - dw).abs().max()) <= 2.0 ** -23 * (0.5 + float(dw.abs().max()))


def test_gradient_against_differences():
    h, w, t = case(6, 40, 16, BF16, ignored=0.0, ignore_index=-100)
    loss, dh, dw = run(h, w, t, up=6.0, ignore_index=-100)
    H, W = h.double(), w.double()
    f = lambda a, b: torch.nn.functional.cross_entropy(a @ b.t(), t, reduction='sum')          # noqa: E731
    step = 2.0 ** -10
    for X, got, other in ((H, dh, 0), (W, dw, 1)):
        for i in range(0, X.numel(), 5):
            e = torch.zeros(X.numel(), device='cuda', dtype=torch.float64)
            e[i] = step
            e = e.view_as(X)
            diff = float(f(H + e, W) - f(H - e, W) if other == 0 else f(H, W + e) - f(H, W - e)) / (2 * step)
            # the softmax's and the result's rounding, over 40 columns or 6 rows of |values| below 4; differences to h^2
            assert abs(float(got.view(-1)[i]) - diff) <= UNIT[BF16] * (abs(diff) + 2 * 4) + 64 * step * step


def test_weights_past_32_bit_offsets():
    V, d, rows = 2_900_000, 768, 64                        # 2.2e9 elements
    g = torch.Generator(device='cuda').manual_seed(3)
    w = torch.empty((V, d), dtype=BF16, device='cuda')
    for part in w.split(100_000):
        part.copy_(torch.randn(part.shape, generator=g, device='cuda') * 0.05)
    h = torch.randn((rows, d), generator=g, device='cuda').to(BF16)
    t = torch.randint(V - 1000, V, (rows,), generator=g, device='cuda')
    loss, dh, dw = run(h, w, t, up=float(rows), ignore_index=-100)
    lse = torch.full((rows,), -float('inf'), device='cuda', dtype=torch.float64)
    want = torch.zeros((rows, d), device='cuda', dtype=torch.float64)
    for part in w.split(100_000):
        lse = torch.logaddexp(lse, torch.logsumexp(h.double() @ part.double().t(), 1))
    for part in w.split(100_000):
        want += (h.double() @ part.double().t() - lse[:, None]).exp() @ part.double()
    want -= w[t].double()
    assert abs(float(loss) - float((lse - (h.double() * w[t].double()).sum(1)).mean())) <= 1e-4          # e_z: 52 steps of 2^-23 of |h||w| below 40
    assert float((dh.double() - want).norm()) <= 2 * UNIT[BF16] * float(want.norm())
    tail = w[-1000:].double()
    G = (h.double() @ tail.t() - lse[:, None]).exp()
    G[torch.arange(rows, device='cuda'), t - (V - 1000)] -= 1
    want = G.t() @ h.double()
    assert float((dw[-1000:].double() - want).norm()) <= 2 * UNIT[BF16] * float(want.norm())


def test_no_rows():
    loss = ulm_ops.streamed_cross_entropy(torch.zeros(0, 64, device='cuda', dtype=BF16), torch.zeros(10, 64, device='cuda', dtype=BF16),
                                          torch.zeros(0, device='cuda', dtype=torch.long))
    assert float(loss) == 0


@pytest.mark.parametrize('bad', ['width', 'target type', 'target size', 'target device', 'weight width', 'cpu', 'compute type', 'vocabulary', 'integers'])
def test_refusals(bad):
    d = 12 if bad == 'width' else 64
    h, w = torch.ones(4, d, device='cuda', dtype=BF16), torch.ones(0 if bad == 'vocabulary' else 10, d, device='cuda', dtype=BF16)
    t = torch.zeros(4, device='cuda', dtype=torch.int32 if bad == 'target type' else torch.long)
    if bad == 'target size': t = t[:3]
    if bad == 'target device': t = t.cpu()
    if bad == 'weight width': w = w[:, :56]
    if bad == 'cpu': h, w, t = h.cpu(), w.cpu(), t.cpu()
    if bad == 'integers': w = w.long()
    with pytest.raises(ValueError):
        ulm_ops.streamed_cross_entropy(h, w, t, compute_dtype=F32 if bad == 'compute type' else None)
