"""The norms behind and in front of a block with the residual add between them, against plain forms in 64 bits."""
import math

import pytest
import torch

import ulm_ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}          # largest relative error of one rounding
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}       # and absolute, among subnormals
SCALES = ['none', 'number', 'scalar', 'one element', 'channels']


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') * std).to(dtype)


def within(got, want, bound):
    assert got.shape == want.shape
    # what surely lies beyond the type's largest number (plus half a step) rounds to an infinity of its sign
    most = torch.finfo(got.dtype).max * (1 + UNIT[got.dtype] / 2)
    beyond = want.abs() - bound > most
    assert torch.equal(got.double()[beyond], want[beyond].sign() * float('inf'))
    off = ((got.double() - want).abs() - bound)[~beyond]
    assert bool((off <= 0).all()), float(off.max())


def inputs(rows, d, dtype, gate=False, scale='none', seed=1):
    shape = (rows, d) if isinstance(rows, int) else (*rows, d)
    s = dict(x=randn(shape, F32, seed, 2.0), b=randn(shape, dtype, seed + 1, 0.5), v=1 + randn(d, F32, seed + 2, 0.1), w=1 + randn(d, F32, seed + 3, 0.1),
             gx=randn(shape, F32, seed + 4), gy=randn(shape, dtype, seed + 5))
    if gate:
        s['gate'] = randn(shape, dtype, seed + 6, 2.0)
    if scale != 'none':
        s['scale'] = -0.75 if scale == 'number' else 0.5 + randn({'scalar': (), 'one element': 1, 'channels': d}[scale], F32, seed + 7, 0.3)
    return s


def call(s, eps=1e-6):
    """-> x_new, y and the gradients of all tensors, by name."""
    leaves = {n: s[n].detach().requires_grad_() for n in ('x', 'b', 'v', 'w', 'gate', 'scale') if isinstance(s.get(n), torch.Tensor)}
    t = {**s, **leaves}
    x_new, y = ulm_ops.norm_add_norm(t['x'], t['b'], t['v'], t['w'], gate=t.get('gate'), scale=t.get('scale'), eps=eps)
    grads = torch.autograd.grad([x_new, y], list(leaves.values()), [s['gx'], s['gy']])
    return dict(x_new=x_new, y=y, **{'d' + n: g for n, g in zip(leaves, grads)})


def forward64(s, eps):
    t = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    r1 = torch.rsqrt(t['b'].square().mean(-1, keepdim=True) + eps)
    sig = torch.sigmoid(t['gate']) if 'gate' in t else torch.ones_like(t['b'])
    term = t.get('scale', 1.0) * sig * t['b'] * r1 * t['v']
    x_new = t['x'] + term
    r2 = torch.rsqrt(x_new.square().mean(-1, keepdim=True) + eps)
    return dict(t=t, r1=r1, sig=sig, term=term, x_new=x_new, r2=r2, y=x_new * r2 * t['w'])


def check(s, got, eps=1e-6):
    dtype, d = s['b'].dtype, s['x'].shape[-1]
    f = forward64(s, eps)
    t, u = f['t'], UNIT[F32]
    rows = s['x'].numel() // d
    # a statistic is a sum of d squares in chains of at most 32 + log2 steps, a reciprocal root and a product or two
    stat = 64 * u
    big = t['x'].abs() + f['term'].abs()
    within(got['x_new'], f['x_new'], (stat + 8 * u) * f['term'].abs() + 2 * u * big)
    top = (big * f['r2']).amax(-1, keepdim=True)
    # x_new's own error, relative to its parts, and the statistic's
    within(got['y'], f['y'], (UNIT[dtype] + stat) * f['y'].abs() + 2 * stat * top * t['w'].abs() + TINY[dtype])
    h, G, U = f['x_new'] * f['r2'], t['gy'] * t['w'], t['b'] * f['r1']
    m = (G * h).mean(-1, keepdim=True)
    dx = f['r2'] * (G - h * m) + t['gx']
    am = (G * h).abs().mean(-1, keepdim=True)
    adx = f['r2'] * (G.abs() + h.abs() * am) * (1 + top) + t['gx'].abs()         # the sizes of what dx is a sum of
    within(got['dx'], dx, 2 * stat * adx)
    tv = t.get('scale', 1.0) * f['sig'] * t['v']
    n = dx * tv
    db = f['r1'] * (n - U * (n * U).mean(-1, keepdim=True))
    an = adx * tv.abs()
    adb = f['r1'] * (an + U.abs() * (an * U.abs()).mean(-1, keepdim=True))
    within(got['db'], db, UNIT[dtype] * db.abs() + 4 * stat * adb + TINY[dtype])
    chain = 4 * stat + u * (math.isqrt(rows) + 64)
    flat = lambda v: v.reshape(-1, d).sum(0)                       # noqa: E731
    weight = lambda name, want, size: within(got[name], want, (UNIT[s[name[1:]].dtype] if s[name[1:]].dtype != F32 else 0) * want.abs() + chain * size)     # noqa: E731
    weight('dw', flat(t['gy'] * h), flat(t['gy'].abs() * (h.abs() + top)))
    c = dx * f['sig'] * U
    ac = adx * f['sig'] * U.abs()
    weight('dv', flat(c * t.get('scale', 1.0)), flat(ac * abs(t.get('scale', 1.0))))
    if 'gate' in s:
        slope = f['sig'] * torch.sigmoid(-t['gate'])
        dg = dx * t.get('scale', 1.0) * t['v'] * U * slope
        within(got['dgate'], dg, UNIT[dtype] * dg.abs() + 4 * stat * adx * (t.get('scale', 1.0) * t['v'] * U).abs() * slope + TINY[dtype])
    if isinstance(s.get('scale'), torch.Tensor):
        one = s['scale'].numel() == 1
        ds, size = flat(c * t['v']), flat(ac * t['v'].abs())
        if one:
            ds, size = ds.sum().view(s['scale'].shape), size.sum()
        weight('dscale', ds, size)
    assert got['x_new'].dtype == got['dx'].dtype == F32 and got['y'].dtype == got['db'].dtype == dtype
    for n, g in got.items():
        if n.startswith('d'):
            assert g.dtype == s[n[1:]].dtype and g.shape == s[n[1:]].shape


@pytest.mark.parametrize('d', [4, 8, 12, 128, 260, 768, 772, 1020, 1024, 1028, 2048, 2052, 4100, 6152, 8188, 8192])
@pytest.mark.parametrize('rows', [1, 2, 150])
@pytest.mark.parametrize('gate', [False, True])
def test_widths(d, rows, gate):
    s = inputs(rows, d, F16 if (d + rows) % 3 else BF16, gate, SCALES[(d // 4 + rows) % 5], seed=d + rows)
    check(s, call(s))


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('scale', SCALES)
def test_many_rows(dtype, gate, scale):
    s = inputs((3, 1201), 768, dtype, gate, scale)
    check(s, call(s))


@pytest.mark.parametrize('scale', ['scalar', 'channels', 'number'])
@pytest.mark.parametrize('gate', [False, True])
def test_a_scale_of_zero_learns(scale, gate):
    """A branch that is switched off at the start: x passes, and the scale's gradient does not vanish."""
    s = inputs(40, 96, BF16, gate, scale)
    s['scale'] = 0.0 if scale == 'number' else torch.zeros_like(s['scale'])
    got = call(s)
    assert torch.equal(got['x_new'], s['x']) and not got['db'].any() and not got['dv'].any()
    assert scale == 'number' or bool(got['dscale'].abs().min() > 0)
    check(s, got)


@pytest.mark.parametrize('eps', [1e-6, 1e-2])
def test_rows_of_zeros_and_tiny_rows(eps):
    s = inputs(6, 64, F16, True, 'scalar')
    s['b'][0], s['b'][1], s['x'][2] = 0, s['b'][1] * 2.0 ** -14, 0
    s['b'][3], s['x'][3] = 0, 0
    got = call(s, eps)
    assert not got['y'][3].any() and torch.equal(got['x_new'][0], s['x'][0])
    check(s, got, eps)


def test_gates_open_and_closed():
    s = inputs(8, 64, F16, True, 'none')
    s['gate'][0], s['gate'][1], s['gate'][2], s['gate'][3] = float('inf'), float('-inf'), 60000.0, -60000.0
    got = call(s)
    plain = {k: v for k, v in s.items() if k != 'gate'}
    assert torch.equal(got['x_new'][0], call(plain)['x_new'][0]) and torch.equal(got['x_new'][2], got['x_new'][2])
    assert torch.equal(got['x_new'][1], s['x'][1]) and torch.equal(got['x_new'][3], s['x'][3])
    assert not got['dgate'][:4].any() and not got['db'][1].any()
    for t in got.values():
        assert torch.isfinite(t).all()


def test_open_gates_are_no_gates():
    """A gate that is open to the last bit leaves the very bits of the call without one, gradients included; a closed one passes x alone."""
    s = inputs(12, 64, F16, True, 'channels')
    s['gate'][:6], s['gate'][6:] = torch.tensor([float('inf'), 60000.0, 88.0, 17.5, 200.0, 1000.0], device='cuda')[:, None], float('inf')
    plain = {k: v for k, v in s.items() if k != 'gate'}
    got, want = call(s), call(plain)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    assert not got['dgate'][[0, 1, 4, 5]].any()
    check(s, got)
    s['gate'][1::2] *= -1
    got = call(s)
    assert torch.equal(got['x_new'][[0, 2, 4]], want['x_new'][[0, 2, 4]]) and torch.equal(got['x_new'][[1, 5]], s['x'][[1, 5]])
    check(s, got)


@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('d,rows', [(100, 10007), (300, 4001), (772, 2003), (1020, 2003), (1028, 2003), (2052, 1001), (3076, 701), (4100, 401), (5124, 401), (8188, 401),
                                    (128, 9001), (2048, 1501), (2560, 1001), (4096, 701), (5120, 401), (6144, 401), (8192, 401)])
def test_groups_that_take_a_third_row(d, rows, gate):
    """The backward's groups take row after row; their sums alternate between two sets of slots, and the row after next is asked for ahead."""
    s = inputs(rows, d, F16 if d % 3 else BF16, gate, SCALES[d // 4 % 5], seed=d)
    check(s, call(s))


@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('d,rows', [(4100, 19001), (8192, 19001), (2560, 60001)])
def test_forward_groups_that_take_a_third_row(d, rows, gate):
    """The same of the forward, whose grid is far larger."""
    s = inputs(rows, d, BF16, gate, 'scalar', seed=d)
    x_new, y = ulm_ops.norm_add_norm(s['x'], s['b'], s['v'], s['w'], gate=s.get('gate'), scale=s['scale'])
    stat = 64 * UNIT[F32]
    for at in range(0, rows, 2048):
        part = {k: v[at:at + 2048] if v.dim() == 2 else v for k, v in s.items()}
        f = forward64(part, 1e-6)
        big = f['t']['x'].abs() + f['term'].abs()
        within(x_new[at:at + 2048], f['x_new'], (stat + 8 * UNIT[F32]) * f['term'].abs() + 2 * UNIT[F32] * big)
        within(y[at:at + 2048], f['y'], (UNIT[BF16] + stat) * f['y'].abs() + 2 * stat * (big * f['r2']).amax(-1, keepdim=True) * f['t']['w'].abs() + TINY[BF16])


def test_a_bad_row_spoils_no_other():
    s = inputs(9, 128, BF16, True, 'channels')
    good = call(s)
    s['b'][4, 7], s['x'][6, 3], s['gate'][2, 1] = float('nan'), float('inf'), float('nan')
    got = call(s)
    for n in ('x_new', 'y', 'dx', 'db', 'dgate'):
        for row in (0, 1, 3, 5, 7, 8):
            assert torch.equal(got[n][row], good[n][row])
    assert got['y'][4].isnan().all() and not torch.isfinite(got['y'][6]).all() and got['y'][2].isnan().all()


@pytest.mark.parametrize('form', ['strided', 'eight bytes', 'two bytes', 'weights of 16 bits', 'broadcast branch', 'one dimension', 'transposed'])
def test_layouts(form):
    rows, d = 9, 768
    s = inputs(rows, d, BF16, True, 'channels')
    wide = lambda t, off, pad=8: torch.cat([t.new_zeros(rows, off), t, t.new_zeros(rows, pad - off)], 1)[:, off:off + d]     # noqa: E731
    if form == 'strided':
        s.update(x=wide(s['x'], 4), b=wide(s['b'], 0), gate=wide(s['gate'], 8), gy=wide(s['gy'], 8), gx=wide(s['gx'], 4))
    elif form == 'eight bytes':
        s.update(b=wide(s['b'], 4), gate=wide(s['gate'], 4), gy=wide(s['gy'], 4))
    elif form == 'two bytes':
        s.update(x=wide(s['x'], 1), b=wide(s['b'], 1), gate=wide(s['gate'], 1), gy=wide(s['gy'], 1), gx=wide(s['gx'], 1))
    elif form == 'weights of 16 bits':
        s.update(v=s['v'].bfloat16(), w=s['w'].bfloat16(), scale=s['scale'].bfloat16())
    elif form == 'broadcast branch':
        s.update(b=s['b'][:1].expand(rows, d), gate=s['gate'][:, :1].expand(rows, d))
    elif form == 'one dimension':
        s = {k: v[0] if v.dim() == 2 else v for k, v in s.items()}
    else:
        s.update(b=s['b'].t().contiguous().t(), x=s['x'].t().contiguous().t())
    check(s, call(s))


def test_gradients_of_broadcast_inputs_are_summed():
    rows, d = 12, 64
    s = inputs(rows, d, F16, True, 'scalar')
    s['b'], s['gate'] = s['b'][:1].expand(rows, d), s['gate'][:1].expand(rows, d)
    whole = call(s)
    b, gate = s['b'][:1].detach().requires_grad_(), s['gate'][:1].detach().requires_grad_()
    x_new, y = ulm_ops.norm_add_norm(s['x'], b.expand(rows, d), s['v'], s['w'], gate=gate.expand(rows, d), scale=s['scale'])
    db, dg = torch.autograd.grad([x_new, y], [b, gate], [s['gx'], s['gy']])
    for got, each in ((db, whole['db']), (dg, whole['dgate'])):
        within(got, each.double().sum(0, keepdim=True), (rows + 1) * UNIT[F16] * each.double().abs().sum(0, keepdim=True))


def test_of_no_rows():
    s = inputs(0, 64, F16, True, 'channels')
    got = call(s)
    assert got['x_new'].shape == got['y'].shape == got['db'].shape == got['dgate'].shape == (0, 64)
    for n in ('dv', 'dw', 'dscale'):
        assert got[n].shape == (64,) and not got[n].any()


@pytest.mark.parametrize('used', ['x_new', 'y'])
def test_one_output_used(used):
    s = inputs(5, 96, F16, True, 'scalar')
    leaves = [s[n].detach().requires_grad_() for n in ('x', 'b', 'v', 'w', 'gate', 'scale')]
    out = ulm_ops.norm_add_norm(*leaves[:4], gate=leaves[4], scale=leaves[5])
    i = 0 if used == 'x_new' else 1
    grads = torch.autograd.grad(out[i], leaves, s['gx'] if i == 0 else s['gy'])
    zero = {**s, 'gy' if i == 0 else 'gx': torch.zeros_like(s['gy' if i == 0 else 'gx'])}
    check(zero, dict(x_new=out[0], y=out[1], **{'d' + n: g for n, g in zip(('x', 'b', 'v', 'w', 'gate', 'scale'), grads)}))


@pytest.mark.parametrize('gate', [False, True])
def test_gradient_against_differences(gate):
    """The formulas of `check`, which the kernel is held to, against differences of the definition in 64 bits."""
    s = inputs(2, 8, F16, gate, 'channels')
    got, h = call(s), 2.0 ** -12

    def f(**change):
        o = forward64({**s, **change}, 1e-6)
        return float((o['x_new'] * s['gx'].double()).sum() + (o['y'] * s['gy'].double()).sum())
    for n in ('x', 'b', 'v', 'w', 'scale', *(['gate'] if gate else [])):
        base, g = s[n].double(), got['d' + n].double().view(-1)
        for i in range(base.numel()):
            e = torch.zeros(base.numel(), dtype=torch.float64, device='cuda')
            e[i] = h
            diff = (f(**{n: base + e.view_as(base)}) - f(**{n: base - e.view_as(base)})) / (2 * h)
            # third derivatives through both norms: rows of b have an rms of about half, so below (1 / 0.2)^3 times 40 terms; one rounding
            assert abs(float(g[i]) - diff) <= 40 * 125 * h * h + UNIT[F16] * abs(diff) + 2.0 ** -16 * float(g.abs().max())


def test_agrees_with_the_ops_it_is_made_of():
    s = inputs(130, 768, BF16)
    x_new, y = ulm_ops.norm_add_norm(s['x'], s['b'], s['v'], s['w'])
    sep = s['x'] + ulm_ops.rms_norm(s['b'].float(), s['v'])
    assert float((x_new - sep).abs().max()) <= 2.0 ** -19 and float((y - ulm_ops.rms_norm(sep, s['w']).bfloat16()).abs().max()) <= 2.0 ** -6


def test_changes_in_place_are_noticed():
    for n in ('b', 'gate', 'v', 'scale', 'x_new'):
        s = inputs((2, 3), 64, F16, True, 'channels')
        t = {k: v.clone().requires_grad_() for k, v in s.items() if k not in ('gx', 'gy')}
        x_new, y = ulm_ops.norm_add_norm(t['x'], t['b'], t['v'], t['w'], gate=t['gate'], scale=t['scale'])
        with torch.no_grad():
            (x_new if n == 'x_new' else t[n]).mul_(2)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            torch.autograd.grad(y.float().sum(), t['x'])


def test_second_derivatives_are_refused():
    s = inputs(3, 64, F16, True, 'scalar')
    x = s['x'].requires_grad_()
    x_new, y = ulm_ops.norm_add_norm(x, s['b'], s['v'], s['w'], gate=s['gate'], scale=s['scale'])
    g, = torch.autograd.grad(y.float().sum() + x_new.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='has no second derivative'):
        torch.autograd.grad(g.square().sum(), x)


def test_the_same_bits_every_time_and_on_another_stream():
    s = inputs(1500, 1024, BF16, True, 'scalar')
    a = call(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = call(s)
    side.synchronize()
    for n in a:
        assert torch.equal(a[n], b[n])


def test_two_captured_graphs():
    s = inputs(700, 768, F16, True, 'channels')
    t = inputs(300, 768, F16, True, 'channels', seed=50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(s), call(t)
    graphs, outs = [], []
    for case in (s, t):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(call(case))
    for case in (s, t):
        case['b'].mul_(-2), case['gx'].mul_(3)
    for g in (*graphs, *graphs[::-1]):
        g.replay()
    torch.cuda.synchronize()
    for case, out in zip((s, t), outs):
        want = call(case)
        for n in want:
            assert torch.equal(out[n], want[n])


@pytest.mark.parametrize('bad', ['x dtype', 'branch dtype', 'shapes', 'width', 'too wide', 'no width', 'short weight', 'post weight on the host', 'integer weight', 'gate dtype', 'gate shape',
                                 'gate on the host', 'scale shape', 'scale of two dimensions', 'scale on the host', 'integer scale', 'branch on the host', 'x on the host'])
def test_refusals(bad):
    d = {'width': 66, 'too wide': 8196, 'no width': 0}.get(bad, 64)
    x, b, v, w = torch.ones(2, d, device='cuda'), torch.ones(2, d, device='cuda', dtype=F16), torch.ones(d, device='cuda'), torch.ones(d, device='cuda')
    gate = scale = None
    if bad == 'x dtype': x = x.half()
    if bad == 'branch dtype': b = b.float()
    if bad == 'shapes': b = b[:1]
    if bad == 'short weight': w = w[:-4]
    if bad == 'post weight on the host': v = v.cpu()
    if bad == 'integer weight': v = v.int()
    if bad == 'gate dtype': gate = b.float()
    if bad == 'gate shape': gate = b[:1]
    if bad == 'gate on the host': gate = b.cpu()
    if bad == 'scale shape': scale = v[:4]
    if bad == 'scale of two dimensions': scale = v[None]
    if bad == 'scale on the host': scale = torch.ones(())
    if bad == 'integer scale': scale = torch.ones((), dtype=torch.int32, device='cuda')
    if bad == 'branch on the host': b = b.cpu()
    if bad == 'x on the host': x = x.cpu()
    with pytest.raises(ValueError):
        ulm_ops.norm_add_norm(x, b, v, w, gate=gate, scale=scale)


@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('scale', [None, 0.5])
@pytest.mark.parametrize('autocast', [False, True])
def test_the_module_in_and_out_of_the_training_layout(gated, scale, autocast):
    """`FusedRMSNorm.add_forward` behind a `BranchNorm`: the fused op under autocast, its separate ops for fp32 branches."""
    norm, post = ulm_ops.FusedRMSNorm(64).cuda(), ulm_ops.BranchNorm(64, gated, scale).cuda()
    for p in (*norm.parameters(), *post.parameters()):
        p.data.add_(randn(p.shape, F32, p.numel(), 0.1))
    x, h = randn((2, 5, 64), F32, 1, 2.0), randn((2, 5, 64), F32, 2)
    with torch.autocast('cuda', dtype=BF16, enabled=autocast):
        b = randn((2, 5, 64), BF16 if autocast else F32, 3).requires_grad_()
        gate = post.gate_of(h)
        x_new, y = norm.add_forward(x, b, post=post, gate=gate)
    s = dict(x=x, b=b.detach(), v=post.weight.detach(), w=norm.weight.detach())
    if gated:
        s['gate'] = gate.detach()
    if scale is not None:
        s['scale'] = post.scale.detach()
    f = forward64(s, 1e-6)
    within(x_new, f['x_new'], 2.0 ** -18 * (x.double().abs() + f['term'].abs()))
    within(y, f['y'], (UNIT[b.dtype] if autocast else 0) * f['y'].abs() + 2.0 ** -16 * (1 + f['y'].abs()))
    params = [*norm.parameters(), *post.parameters(), b]
    assert all(torch.isfinite(g).all() and g.any() for g in torch.autograd.grad(x_new.sum() + (y.float() ** 2).sum(), params))
