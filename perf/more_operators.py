"""Three more operators of a model's blocks, as cases that can be timed and compared.

  rotary   ulm_ops.rotary: queries [B, Hq, S, D] and keys [B, Hk, S, D], the first R of D columns turned by an angle that grows
           with the position; pairs of columns R/2 apart or next to one another, frequencies stretched for long contexts;
           forward and backward, and forward alone for one new token of each of many sequences
  norms    ulm_ops.norm_add_norm: x_new = x + scale * sigmoid(gate) * rms_norm(branch) and y = rms_norm(x_new): the norms behind
           and in front of a block with the residual add between them; forward and backward
  gate8    ulm_ops.swiglu_8bit: silu(a) * b, whose backward has a and b in 8 bits alone; forward and backward
  pack     ulm_ops.pack_8bit and unpack_8bit: what an activation kept in 8 bits between forward and backward comes back as

The 8 bits: blocks of 32 consecutive elements share the exponent e of their largest magnitude (at least -120) and keep x / 2^(e-6),
rounded to the nearest integer, ties to even, and held to +-127.  Every such value is a number of the tensor's own type.

`own` chooses between the plain form of each operator, in elementary torch operations and 32 bits (angles in 64), and the package's.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
_DTYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
_BYTES = {'fp16': 2, 'bf16': 2, 'fp32': 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # queries and keys of a training step's attention at the headline sizes
        dict(name='rotary_micro_batch', kind='rotary', B=8, S=4096, Hq=12, Hk=12, D=64, R=64, interleaved=False, scaling='none', dtype='bf16', train=True),
        # one long document of a model whose context is stretched eight times: half of each head turned, few key heads
        dict(name='rotary_long', kind='rotary', B=1, S=32001, Hq=16, Hk=4, D=128, R=64, interleaved=True, scaling='yarn', dtype='fp16', train=True),
        # heads of no power of two, in fp32, on a ragged batch
        dict(name='rotary_odd', kind='rotary', B=3, S=1363, Hq=6, Hk=1, D=80, R=20, interleaved=False, scaling='linear', dtype='fp32', train=True),
        # serving: the next token of each of 96 sequences, far into their contexts; launches count
        dict(name='rotary_token', kind='rotary', B=96, S=1, Hq=16, Hk=4, D=128, R=128, interleaved=False, scaling='parts', dtype='bf16', train=False),
        # norms behind the attention and in front of the feed-forward over a full micro-batch of the 100M preset
        dict(name='norms_micro_batch', kind='norms', rows=32768, d=768, gate=False, scale='none', dtype='fp16'),
        # the scaled preset's width on a ragged batch, with a gate and a learned residual scale
        dict(name='norms_gated', kind='norms', rows=12011, d=1024, gate=True, scale='scalar', dtype='bf16'),
        # wide rows, a scale for each channel
        dict(name='norms_wide', kind='norms', rows=4099, d=4096, gate=True, scale='channels', dtype='bf16'),
        # a handful of tokens: launches count
        dict(name='norms_few', kind='norms', rows=7, d=768, gate=False, scale='number', dtype='fp16'),
        # the feed-forward gate of a full micro-batch of the 100M preset
        dict(name='gate8_micro_batch', kind='gate8', rows=32768, d=2048, dtype='bf16'),
        # rows that are no whole vectors, ragged
        dict(name='gate8_odd', kind='gate8', rows=4099, d=2731, dtype='fp16'),
        # a projection's input over a full micro-batch
        dict(name='pack_micro_batch', kind='pack', rows=32768, d=768, dtype='bf16'),
        # one short sequence of the smallest preset's feed-forward: launches count
        dict(name='pack_few', kind='pack', rows=201, d=344, dtype='fp16'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['rotary', 'rotary', 'norms', 'norms', 'gate8', 'pack'])
    if kind == 'rotary':
        D = rng.choice([64, 80, 96, 128, 256])
        R = rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)])
        Hk = rng.choice([1, 2, 4, 8, 12, 16])
        Hq = Hk * rng.choice([1, 1, 2, 4, 7])
        most = 80_000_000 // ((Hq + Hk) * D)                      # the largest listed case's elements
        train = rng.random() < 0.7
        B = _log_int(rng, 1, 64 if train else 512)
        S = _log_int(rng, 1, max(1, min(32768, most // B))) if train else rng.choice([1, 1, 1, 3, 8])
        return dict(kind='rotary', B=B, S=S, Hq=Hq, Hk=Hk, D=D, R=R, interleaved=rng.random() < 0.5, scaling=rng.choice(['none', 'linear', 'ntk', 'parts', 'yarn']),
                    dtype=rng.choice(['fp16', 'bf16', 'bf16', 'fp32'] if (Hq + Hk) * D * B * S < 40_000_000 else ['fp16', 'bf16']), train=train)
    if kind == 'norms':
        d = rng.choice([128, 768, 1024, 4 * _log_int(rng, 16, 2048)])
        return dict(kind='norms', rows=_log_int(rng, 1, min(32768, 25_000_000 // d)), d=d, gate=rng.random() < 0.5, scale=rng.choice(['none', 'number', 'scalar', 'channels']),
                    dtype=rng.choice(['fp16', 'bf16']))
    dtype = rng.choice(['fp16', 'bf16', 'bf16', 'fp32'])
    if kind == 'gate8':
        d = rng.choice([344, 2048, 2816, _log_int(rng, 64, 2816)])
        return dict(kind='gate8', rows=_log_int(rng, 1, 23000 if dtype != 'fp32' else 11500), d=d, dtype=dtype)
    return dict(kind='pack', rows=_log_int(rng, 1, 32768), d=rng.choice([128, 768, 1024, _log_int(rng, 64, 2048)]), dtype=dtype)


# the stretched contexts: an original length of 4096 and eight times that (serving: up to a million positions)
_SCALING = {
    'none': None,
    'linear': dict(kind='linear', factor=8.0),
    'ntk': dict(kind='ntk', factor=8.0),
    'parts': dict(kind='parts', factor=8.0, original_length=4096, slow=1.0, fast=4.0),
    'yarn': dict(kind='yarn', factor=8.0, original_length=4096, slow=1.0, fast=32.0),
}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device='cuda').manual_seed(int(seed))
    dtype = _DTYPES[case['dtype']]

    def randn(*shape, std=1.0, to=dtype):
        return (torch.randn(shape, generator=g, device='cuda') * std).to(to)

    if case['kind'] == 'rotary':
        B, S, Hq, Hk, D = (case[n] for n in ('B', 'S', 'Hq', 'Hk', 'D'))
        # views of one projection's output, [B, S, queries | keys | values]; gradients as an attention's backward leaves them
        qkv = randn(B, S, Hq + 2 * Hk, D)
        q, k = (t.transpose(1, 2) for t in (qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]))
        s = dict(q=q, k=k)
        if case['train']:
            s.update(gq=randn(B, S, Hq, D).transpose(1, 2), gk=randn(B, S, Hk, D).transpose(1, 2))
        else:
            # how far each sequence has come, at the far end of long contexts
            start = torch.randint(0, 1 << 20, (B, 1), generator=g, device='cuda')
            s['positions'] = start + torch.arange(S, device='cuda')
        return s
    rows, d = case['rows'], case['d']
    if case['kind'] == 'norms':
        s = dict(x=randn(rows, d, std=2.0, to=torch.float32), b=randn(rows, d, std=0.5), v=1.0 + randn(d, std=0.1, to=torch.float32),
                 w=1.0 + randn(d, std=0.1, to=torch.float32), gx=randn(rows, d, to=torch.float32), gy=randn(rows, d))
        if case['gate']:
            s['gate'] = randn(rows, d)
        if case['scale'] == 'number':
            s['scale'] = 0.22
        elif case['scale'] != 'none':
            s['scale'] = 0.5 + randn(*([] if case['scale'] == 'scalar' else [d]), std=0.1, to=torch.float32)
        return s
    # activations: channels of different sizes, a few of them far larger than the rest
    size = torch.exp(torch.randn(d, generator=g, device='cuda') * 0.5)
    size[torch.rand(d, generator=g, device='cuda') < 0.01] *= 8.0
    if case['kind'] == 'gate8':
        return dict(a=(randn(rows, d, to=torch.float32) * size).to(dtype), b=(randn(rows, d, to=torch.float32) * size).to(dtype), gy=randn(rows, d))
    return dict(x=(randn(rows, d, to=torch.float32) * size).to(dtype))


_LEAVES = {'rotary': ('q', 'k'), 'norms': ('x', 'b', 'v', 'w', 'gate', 'scale'), 'gate8': ('a', 'b'), 'pack': ()}


def prepare(case, seed):
    s = dict(_inputs(case, seed), kind=case['kind'])
    if case.get('train', True):
        for name in _LEAVES[case['kind']]:
            if isinstance(s.get(name), torch.Tensor):
                s[name] = s[name].detach().requires_grad_()
    if case['kind'] == 'rotary':
        s.update(R=case['R'], interleaved=case['interleaved'], scaling=_SCALING[case['scaling']], train=case['train'])
        if own:
            s['rotary'] = _package().Rotary(case['R'], interleaved=case['interleaved'], scaling=_SCALING[case['scaling']]).cuda()
    return s


# ---------------------------------------------------------------------------
# one pass: the package's operators
# ---------------------------------------------------------------------------
def _package():
    path = os.path.abspath('universal-lm-trainer_b200')
    if path not in sys.path:
        sys.path.insert(0, path)
    import ulm_ops
    return ulm_ops


def _run_own(s):
    ops = _package()
    if s['kind'] == 'rotary':
        q, k = s['rotary'](s['q'], s['k'], s.get('positions'))
        if not s['train']:
            return dict(q=q, k=k)
        dq, dk = torch.autograd.grad([q, k], [s['q'], s['k']], [s['gq'], s['gk']])
        return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk)
    if s['kind'] == 'norms':
        x_new, y = ops.norm_add_norm(s['x'], s['b'], s['v'], s['w'], gate=s.get('gate'), scale=s.get('scale'), eps=EPS)
        names = [n for n in _LEAVES['norms'] if isinstance(s.get(n), torch.Tensor)]
        grads = torch.autograd.grad([x_new, y], [s[n] for n in names], [s['gx'], s['gy']])
        return dict(x_new=x_new.detach(), y=y.detach(), **{'d' + n: t for n, t in zip(names, grads)})
    if s['kind'] == 'gate8':
        y = ops.swiglu_8bit(s['a'], s['b'])
        da, db = torch.autograd.grad(y, [s['a'], s['b']], s['gy'])
        return dict(y=y.detach(), da=da, db=db)
    return ops.unpack_8bit(ops.pack_8bit(s['x']))


# ---------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------
def _frequencies(R, scaling):
    """Radians a position of each pair, in 64 bits, and what the turned vectors are multiplied by."""
    i = torch.arange(0, R, 2, device='cuda', dtype=torch.float64)
    if scaling is None:
        return 10000.0 ** (-i / R), 1.0
    f = scaling['factor']
    if scaling['kind'] == 'linear':
        return 10000.0 ** (-i / R) / f, 1.0
    if scaling['kind'] == 'ntk':
        return (10000.0 * f ** (R / (R - 2)) if R > 2 else 10000.0) ** (-i / R), 1.0
    # pairs that turn often within the original length stay, those that hardly turn are slowed down by the whole factor
    w = 10000.0 ** (-i / R)
    turns = scaling['original_length'] * w / (2 * math.pi)
    keep = ((turns - scaling['slow']) / (scaling['fast'] - scaling['slow'])).clamp(0.0, 1.0)
    return w * keep + w / f * (1.0 - keep), 0.1 * math.log(f) + 1.0 if scaling['kind'] == 'yarn' else 1.0


def _turned(x, cos, sin, R, interleaved, dtype):
    x = x.detach().float()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    p, m = a * cos - b * sin, b * cos + a * sin
    head = torch.stack([p, m], dim=-1).flatten(-2) if interleaved else torch.cat([p, m], dim=-1)
    return torch.cat([head, x[..., R:]], dim=-1).to(dtype)


def _two_to(e):
    """2^e in fp32, from its bits: -126 <= e <= 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _through_8bit(x):
    """What the 8-bit form of ``x`` stands for, in fp32."""
    flat = x.detach().float().reshape(-1)
    n = flat.numel()
    blocks = torch.cat([flat, flat.new_zeros(-n % 32)]).view(-1, 32)
    e = torch.frexp(blocks.abs().amax(1, keepdim=True))[1] - 1          # 2^e at most the largest magnitude, which is below 2^(e + 1)
    e = e.clamp(min=-120)
    codes = torch.round(blocks * _two_to(6 - e)).clamp(-127, 127)
    return (codes * _two_to(e - 6)).view(-1)[:n].view(x.shape)


def _run_plain(s):
    if s['kind'] == 'rotary':
        q, R, dtype = s['q'], s['R'], s['q'].dtype
        freq, factor = _frequencies(R, s['scaling'])
        positions = s.get('positions')
        if positions is None:
            positions = torch.arange(q.shape[2], device='cuda')[None]
        angle = (positions.double()[..., None] * freq)[:, None]                 # [B or 1, 1, S, R / 2]
        cos, sin = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()
        out = {n: _turned(s[n], cos, sin, R, s['interleaved'], dtype) for n in ('q', 'k')}
        if s['train']:
            # turned back; the columns beyond R pass through both ways
            out.update({'d' + n: _turned(s['g' + n], cos, -sin, R, s['interleaved'], dtype) for n in ('q', 'k')})
        return out
    if s['kind'] == 'norms':
        f = {k: v.detach().float() for k, v in s.items() if isinstance(v, torch.Tensor)}
        dtype, scale = s['b'].dtype, f.get('scale', s.get('scale', 1.0))
        r = torch.rsqrt((f['b'] * f['b']).mean(1, keepdim=True) + EPS)
        unit = f['b'] * r
        sig = 1.0 / (1.0 + torch.exp(-f['gate'])) if 'gate' in f else 1.0
        normed = unit * f['v']
        x_new = f['x'] + scale * sig * normed
        r2 = torch.rsqrt((x_new * x_new).mean(1, keepdim=True) + EPS)
        unit2, g2 = x_new * r2, f['gy'] * f['w']
        dx = r2 * (g2 - unit2 * (g2 * unit2).mean(1, keepdim=True)) + f['gx']
        g = dx * scale * sig * f['v']
        out = dict(x_new=x_new, y=(unit2 * f['w']).to(dtype), dx=dx, db=(r * (g - unit * (g * unit).mean(1, keepdim=True))).to(dtype),
                   dv=(dx * scale * sig * unit).sum(0), dw=(f['gy'] * unit2).sum(0))
        if 'gate' in f:
            out['dgate'] = (dx * scale * normed * sig * (1.0 - sig)).to(dtype)
        if 'scale' in f:
            per_channel = (dx * sig * normed).sum(0)
            out['dscale'] = per_channel if f['scale'].dim() else per_channel.sum()
        return out
    if s['kind'] == 'gate8':
        dtype = s['a'].dtype
        a, b = s['a'].detach().float(), s['b'].detach().float()
        y = (a * (1.0 / (1.0 + torch.exp(-a))) * b).to(dtype)
        a, b, g = _through_8bit(s['a']), _through_8bit(s['b']), s['gy'].float()
        sig = 1.0 / (1.0 + torch.exp(-a))
        return dict(y=y, da=(g * b * sig * (1.0 + a * (1.0 - sig))).to(dtype), db=(g * a * sig).to(dtype))
    return _through_8bit(s['x']).to(s['x'].dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _kept64(x):
    """The 8-bit form of ``x`` by its definition: a common power of two for 32 neighbours, integers beside it."""
    shape, n = x.shape, x.numel()
    v = torch.nn.functional.pad(x.double().reshape(-1), (0, -n % 32)).reshape(-1, 32)
    top = v.abs().max(dim=1).values
    power = lambda e: (e.long() + 1023 << 52).view(torch.float64)       # noqa: E731 - 2^e from its bits
    e = torch.floor(torch.log2(top)).clamp(min=-1000)
    e = torch.where(power(e) > top, e - 1, e)                       # log2 may round up to the next power
    e = torch.where(power(e + 1) <= top, e + 1, e).clamp(min=-120)
    step = power(e - 6)[:, None]
    whole = torch.floor(v / step)
    rest = v / step - whole                                          # exact: a quotient by a power of two
    up = (rest > 0.5) | ((rest == 0.5) & (whole % 2 != 0))
    return ((whole + up).clamp(-127, 127) * step).reshape(-1)[:n].reshape(shape)


def _rotation64(case, s, x, back):
    scaling, R = _SCALING[case['scaling']], case['R']
    k = torch.arange(R // 2, dtype=torch.float64, device='cuda')
    base, factor, grow = 10000.0, 1.0, torch.ones_like(k)
    if scaling is not None:
        f = scaling['factor']
        if scaling['kind'] == 'linear':
            grow = torch.full_like(k, f)
        elif scaling['kind'] == 'ntk':
            base = base * f ** (R / (R - 2)) if R > 2 else base
        else:
            per_turn = 2 * math.pi * base ** (2 * k / R)             # positions that a pair takes for a turn
            share = (scaling['original_length'] / per_turn - scaling['slow']) / (scaling['fast'] - scaling['slow'])
            share = share.clamp(0, 1)
            grow = 1.0 / ((1.0 - share) / f + share)
            if scaling['kind'] == 'yarn':
                factor = 0.1 * math.log(f) + 1.0
    at = s['positions'] if 'positions' in s else torch.arange(case['S'], device='cuda')[None]
    angle = at.double()[..., None] / (base ** (2 * k / R) * grow)
    z = torch.polar(torch.full_like(angle, factor), -angle if back else angle)[:, None]
    x, out = x.double(), x.double().clone()
    even, odd = (slice(0, R, 2), slice(1, R, 2)) if case['interleaved'] else (slice(0, R // 2), slice(R // 2, R))
    w = torch.complex(x[..., even], x[..., odd]) * z
    out[..., even], out[..., odd] = w.real, w.imag
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case['kind'] == 'rotary':
        out = {n: _rotation64(case, s, s[n], False) for n in ('q', 'k')}
        if case['train']:
            out.update({'d' + n: _rotation64(case, s, s['g' + n], True) for n in ('q', 'k')})
        return out
    if case['kind'] == 'pack':
        return _kept64(s['x'])
    if case['kind'] == 'gate8':
        a, b, g = s['a'].double(), s['b'].double(), s['gy'].double()
        y = torch.sigmoid(a) * a * b
        a, b = _kept64(s['a']), _kept64(s['b'])
        sig = torch.sigmoid(a)
        return dict(y=y, da=g * b * (sig + a * sig * torch.sigmoid(-a)), db=g * a * sig)
    t = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    scale = t.get('scale', 1.0)
    rms = torch.sqrt(t['b'].square().mean(1, keepdim=True) + EPS)
    u = t['b'] / rms
    opened = torch.sigmoid(t['gate']) if case['gate'] else torch.ones_like(u)
    x_new = t['x'] + scale * opened * u * t['v']
    rms2 = torch.sqrt(x_new.square().mean(1, keepdim=True) + EPS)
    u2, gw = x_new / rms2, t['gy'] * t['w']
    dx = t['gx'] + (gw - u2 * (gw * u2).mean(1, keepdim=True)) / rms2
    du = dx * scale * opened * t['v']
    out = dict(x_new=x_new, y=u2 * t['w'], dx=dx, db=(du - u * (du * u).mean(1, keepdim=True)) / rms, dv=(dx * scale * opened * u).sum(0), dw=(t['gy'] * u2).sum(0))
    if case['gate']:
        out['dgate'] = dx * scale * u * t['v'] * opened * torch.sigmoid(-t['gate'])
    if case['scale'] in ('scalar', 'channels'):
        moved = dx * opened * u * t['v']
        out['dscale'] = moved.sum(0) if case['scale'] == 'channels' else moved.sum()
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = _BYTES[case['dtype']]
    if case['kind'] == 'rotary':
        n = case['B'] * case['S'] * (case['Hq'] + case['Hk']) * case['D']
        return dict(bytes=(4 if case['train'] else 2) * e * n, flops=0)           # q, k and their gradients, in and out
    n = case['rows'] * case['d']
    if case['kind'] == 'norms':
        # x, g_x read, x_new, dx written in fp32; branch, g_y read, y, d_branch written in 16 bits; the gate and its gradient.
        # That the backward reads x_new, branch and gate again is not counted
        return dict(bytes=(16 + 4 * e + (2 * e if case['gate'] else 0)) * n + 16 * case['d'], flops=0)
    if case['kind'] == 'gate8':
        return dict(bytes=6 * e * n, flops=0)             # a, b, g_y; y, da, db; not what is kept in between
    return dict(bytes=2 * e * n, flops=0)                 # in and out; not the 8 bits in between
