"""Four operators of the training step, as cases that can be timed and compared: the loss over a large vocabulary
without its logits, and the dropout whose mask is never stored, alone and inside the two places a block has for it.

  loss     ulm_ops.streamed_cross_entropy: hidden [rows, d], lm-head weight [vocab, d], one target a row -> the mean loss
           over the targets that count, and the gradients of hidden and weight for a given gradient of the loss
  norm     ulm_ops.dropout_add_rms_norm: fp32 residual stream + dropout(16-bit branch), and the RMS norm that follows it;
           forward and backward
  gate     ulm_ops.swiglu_dropout: dropout(silu(a) * b), forward and backward
  drop     ulm_ops.dropout, forward and backward

The mask is a function of a 64-bit seed and of the element's place alone: Philox4x32 with ten rounds (Salmon, Moraes, Dror
and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011), key = the seed, counter = the number of the group of
eight consecutive elements; element j of a group has the j-th 16 bits of the 128 that come out.  It is dropped where
they are below 65536 p, the others are multiplied by the inverse of the share that is kept.

`own` chooses between the plain form of each operator, in elementary torch operations and 32 bits, and the package's.
"""
import math
import os
import sys

import numpy as np
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
        # lm head + loss of a full token-budget micro-batch of the 100M preset
        dict(name='loss_micro_batch', kind='loss', rows=32768, d=768, vocab=32000, dtype='bf16'),
        # the scaled preset's width on a ragged batch, fp16 with the loss scale that fp16 training uses
        dict(name='loss_wide', kind='loss', rows=12011, d=1024, vocab=32000, dtype='fp16'),
        # one long sequence against a vocabulary that is no multiple of anything
        dict(name='loss_odd_vocab', kind='loss', rows=1363, d=768, vocab=50021, dtype='bf16'),
        # a handful of tokens (a short answer scored with its gradient): the weights' bytes and launches count
        dict(name='loss_few_tokens', kind='loss', rows=7, d=768, vocab=32000, dtype='fp16'),
        # residual add + dropout + norm over a full micro-batch, what every block of a training step runs
        dict(name='norm_micro_batch', kind='norm', rows=32768, d=768, p=0.1, dtype='fp16'),
        # the scaled preset's width, ragged
        dict(name='norm_wide', kind='norm', rows=8191, d=1024, p=0.1, dtype='bf16'),
        # one short sequence: launches count
        dict(name='norm_short', kind='norm', rows=201, d=768, p=0.25, dtype='bf16'),
        # the feed-forward gate with its dropout over a full micro-batch
        dict(name='gate_micro_batch', kind='gate', rows=32768, d=2048, p=0.1, dtype='bf16'),
        # the scaled preset's feed-forward width, ragged
        dict(name='gate_wide', kind='gate', rows=4099, d=2816, p=0.3, dtype='fp16'),
        # dropout by itself (embeddings, an attention's output) over a full micro-batch
        dict(name='drop_micro_batch', kind='drop', rows=32768, d=768, p=0.1, dtype='bf16'),
        # fp32, with rows that are no whole vectors
        dict(name='drop_odd', kind='drop', rows=5003, d=771, p=0.5, dtype='fp32'),
        # a few rows of the smallest preset: launches count
        dict(name='drop_few', kind='drop', rows=67, d=128, p=0.1, dtype='fp16'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['loss', 'loss', 'loss', 'norm', 'norm', 'gate', 'drop'])
    if kind == 'loss':
        # the presets' widths and vocabularies, and others: any number of columns, a width of whole 16-byte vectors
        d = rng.choice([128, 768, 1024, 8 * _log_int(rng, 8, 160)])
        vocab = rng.choice([4096, 32000, _log_int(rng, 500, 64000), _log_int(rng, 500, 64000)])
        most = int(min(32768, 32768 * 768 * 32000 / (d * vocab)))
        return dict(kind='loss', rows=_log_int(rng, 1, most), d=d, vocab=vocab, dtype=rng.choice(['fp16', 'bf16']))
    p = rng.choice([0.05, 0.1, 0.25, 0.5])
    if kind == 'norm':
        d = rng.choice([128, 768, 1024, 4 * _log_int(rng, 16, 512)])
        return dict(kind='norm', rows=_log_int(rng, 1, 32768), d=d, p=p, dtype=rng.choice(['fp16', 'bf16']))
    dtype = rng.choice(['fp16', 'bf16', 'bf16', 'fp32'])
    if kind == 'gate':
        return dict(kind='gate', rows=_log_int(rng, 1, 32768), d=rng.choice([344, 2048, 2816, _log_int(rng, 64, 2816)]), p=p, dtype=dtype)
    return dict(kind='drop', rows=_log_int(rng, 1, 32768), d=rng.choice([128, 768, 1024, _log_int(rng, 64, 2048)]), p=p, dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device='cuda').manual_seed(int(seed))
    dtype = _DTYPES[case['dtype']]
    rows, d = case['rows'], case['d']

    def randn(*shape, std=1.0, to=dtype):
        return (torch.randn(shape, generator=g, device='cuda') * std).to(to)

    if case['kind'] == 'loss':
        vocab = case['vocab']
        w = randn(vocab, d, std=1.4 / math.sqrt(d), to=torch.float32)
        # tokens as frequent as in text (the k-th most frequent about 1/k of the first); 5 % of the targets are padding
        u = torch.rand(rows, generator=g, device='cuda', dtype=torch.float64)
        t = (torch.exp(u * math.log(vocab)).long() - 1).clamp_(1, vocab - 1)
        t[torch.rand(rows, generator=g, device='cuda') < 0.05] = 0
        # hidden states of a model that has learned something: the target's logit stands out by about four deviations
        h = torch.randn((rows, d), generator=g, device='cuda') + 4.0 * torch.nn.functional.normalize(w[t], dim=1)
        # d(total loss)/d(this loss): the fp16 loss scale, lower where few tokens would overflow with it; bf16: one of
        # several micro-batches
        up = torch.full((), min(65536.0, 32.0 * rows) if case['dtype'] == 'fp16' else 0.25, device='cuda')
        return dict(h=h.to(dtype), w=w.to(dtype), t=t, up=up)
    s = dict(p=case['p'], seed=int(seed) * 0x9E3779B97F4A7C15 % (1 << 63))
    if case['kind'] == 'norm':
        return dict(s, x=randn(rows, d, std=2.0, to=torch.float32), b=randn(rows, d), w=1.0 + randn(d, std=0.1, to=torch.float32),
                    gx=randn(rows, d, to=torch.float32), gy=randn(rows, d))
    if case['kind'] == 'gate':
        return dict(s, a=randn(rows, d), b=randn(rows, d), gy=randn(rows, d))
    return dict(s, x=randn(rows, d), gy=randn(rows, d))


_LEAVES = {'loss': ('h', 'w'), 'norm': ('x', 'b', 'w'), 'gate': ('a', 'b'), 'drop': ('x',)}


def prepare(case, seed):
    s = dict(_inputs(case, seed), kind=case['kind'])
    for name in _LEAVES[case['kind']]:
        s[name].requires_grad_()
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
    if s['kind'] == 'loss':
        loss = ops.streamed_cross_entropy(s['h'], s['w'], s['t'], ignore_index=0)
        dh, dw = torch.autograd.grad(loss, [s['h'], s['w']], s['up'])
        return dict(loss=loss.detach(), dh=dh, dw=dw)
    if s['kind'] == 'norm':
        x_new, y = ops.dropout_add_rms_norm(s['x'], s['b'], s['w'], s['p'], s['seed'], eps=EPS)
        dx, db, dw = torch.autograd.grad([x_new, y], [s['x'], s['b'], s['w']], [s['gx'], s['gy']])
        return dict(x_new=x_new.detach(), y=y.detach(), dx=dx, db=db, dw=dw)
    if s['kind'] == 'gate':
        y = ops.swiglu_dropout(s['a'], s['b'], s['p'], s['seed'])
        da, db = torch.autograd.grad(y, [s['a'], s['b']], s['gy'])
        return dict(y=y.detach(), da=da, db=db)
    y = ops.dropout(s['x'], s['p'], s['seed'])
    return dict(y=y.detach(), dx=torch.autograd.grad(y, s['x'], s['gy'])[0])


# ---------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------
def _threshold(p):
    """The 16-bit numbers below this drop their element, and what the others are multiplied by."""
    t = min(65535, max(1, round(p * 65536)))
    return t, 65536.0 / (65536 - t)


def _mul_hi_lo(a, m):
    # a * m of two numbers below 2^32 held in int64, in halves that do not overflow it
    low = a * (m & 0xFFFF)
    t = a * (m >> 16) + (low >> 16)
    return t >> 16, ((t & 0xFFFF) << 16) | (low & 0xFFFF)


def _keep(shape, p, seed):
    """Truth values of the elements that stay."""
    n = math.prod(shape)
    group = torch.arange((n + 7) // 8, device='cuda')
    c0, c1, c2, c3 = group & 0xFFFFFFFF, group >> 32, torch.zeros_like(group), torch.zeros_like(group)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for r in range(10):                                   # the generator's ten rounds
        h0, l0 = _mul_hi_lo(c0, 0xD2511F53)
        h1, l1 = _mul_hi_lo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ ((k0 + r * 0x9E3779B9) & 0xFFFFFFFF), l1, h0 ^ c3 ^ ((k1 + r * 0xBB67AE85) & 0xFFFFFFFF), l0
    words = torch.stack([c0, c1, c2, c3], dim=1)
    u = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)
    return (u >= _threshold(p)[0])[:n].view(shape)


def _dropped(v, keep, p):
    return torch.where(keep, v * _threshold(p)[1], torch.zeros((), device='cuda'))


def _run_plain(s):
    f = {k: v.detach().float() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if s['kind'] == 'loss':
        t, counts = s['t'], s['t'] != 0
        z = f['h'] @ f['w'].t()
        m = z.amax(1, keepdim=True)
        e = torch.exp(z - m)
        total = e.sum(1, keepdim=True)
        n = counts.sum().clamp(min=1)
        z_t = z.gather(1, t[:, None])
        row_loss = (m + torch.log(total) - z_t)[:, 0]
        loss = torch.where(counts, row_loss, torch.zeros((), device='cuda')).sum() / n
        g = (e / total).scatter_add_(1, t[:, None], torch.full_like(z_t, -1.0))
        g *= (counts * (f['up'] / n))[:, None]
        return dict(loss=loss, dh=(g @ f['w']).to(s['h'].dtype), dw=(g.t() @ f['h']).to(s['w'].dtype))
    if s['kind'] == 'norm':
        keep, w, dy = _keep(s['b'].shape, s['p'], s['seed']), f['w'], f['gy']
        x_new = f['x'] + _dropped(f['b'], keep, s['p'])
        rstd = torch.rsqrt((x_new * x_new).mean(1, keepdim=True) + EPS)
        xhat, g = x_new * rstd, dy * w
        dx = rstd * (g - xhat * (g * xhat).mean(1, keepdim=True)) + f['gx']
        return dict(x_new=x_new, y=(xhat * w).to(s['b'].dtype), dx=dx, db=_dropped(dx, keep, s['p']).to(s['b'].dtype), dw=(dy * xhat).sum(0))
    if s['kind'] == 'gate':
        keep, a, b, dtype = _keep(s['a'].shape, s['p'], s['seed']), f['a'], f['b'], s['a'].dtype
        sig, g = 1.0 / (1.0 + torch.exp(-a)), _dropped(f['gy'], keep, s['p'])
        return dict(y=_dropped(a * sig * b, keep, s['p']).to(dtype), da=(g * b * sig * (1.0 + a * (1.0 - sig))).to(dtype), db=(g * a * sig).to(dtype))
    keep = _keep(s['x'].shape, s['p'], s['seed'])
    return dict(y=_dropped(f['x'], keep, s['p']).to(s['x'].dtype), dx=_dropped(f['gy'], keep, s['p']).to(s['x'].dtype))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _mask64(shape, p, seed):
    """What each element is multiplied by, from unsigned 64-bit arithmetic on the host."""
    n, u64 = int(np.prod(shape)), np.uint64
    low = u64(0xFFFFFFFF)
    c = [np.arange((n + 7) // 8, dtype=np.uint64)] + [np.zeros((n + 7) // 8, dtype=np.uint64) for _ in range(3)]
    c[1] = c[0] >> u64(32)
    c[0] = c[0] & low
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
        c = [(b >> u64(32)) ^ c[1] ^ u64(key[0]), b & low, (a >> u64(32)) ^ c[3] ^ u64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    u = np.stack(c, axis=1).astype('<u4').view('<u2').reshape(-1)[:n]
    t = min(65535, max(1, round(p * 65536)))
    return torch.from_numpy(np.where(u >= t, 65536.0 / (65536 - t), 0.0).reshape(shape)).cuda()


def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
    if case['kind'] == 'loss':
        h, w, t = s['h'], s['w'], s['t']
        n, total = max(1, int((t != 0).sum())), 0.0
        dh, dw = torch.empty_like(h), torch.zeros_like(w)
        for i in range(0, len(h), 4096):                 # rows in portions that fit
            hi, ti = h[i:i + 4096], t[i:i + 4096]
            logp = torch.log_softmax(hi @ w.T, dim=1)
            at = torch.arange(len(ti), device='cuda')
            total -= float(logp[at, ti][ti != 0].sum())
            g = logp.exp_()
            g[at, ti] -= 1.0
            g[ti == 0] = 0.0
            g *= s['up'] / n
            dh[i:i + 4096] = g @ w
            dw += g.T @ hi
        return dict(loss=np.float64(total / n), dh=dh, dw=dw)
    shape = (case['rows'], case['d'])
    k = _mask64(shape, case['p'], s['seed'])
    # a dropped element is zero whatever it held
    drop = lambda v: torch.where(k > 0, v * k, 0.0)       # noqa: E731
    if case['kind'] == 'norm':
        x_new = s['x'] + drop(s['b'])
        norm = torch.sqrt(x_new.square().mean(1, keepdim=True) + EPS)
        unit, gw = x_new / norm, s['gy'] * s['w']
        dx = s['gx'] + (gw - unit * (gw * unit).mean(1, keepdim=True)) / norm
        return dict(x_new=x_new, y=unit * s['w'], dx=dx, db=drop(dx), dw=(s['gy'] * unit).sum(0))
    if case['kind'] == 'gate':
        a, b, g = s['a'], s['b'], drop(s['gy'])
        sig = torch.sigmoid(a)
        return dict(y=drop(a * sig * b), da=g * b * (sig + a * sig * torch.sigmoid(-a)), db=g * a * sig)
    return dict(y=drop(s['x']), dx=drop(s['gy']))


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    n, e = case['rows'] * case['d'], _BYTES[case['dtype']]
    if case['kind'] == 'loss':
        # hidden, weight and their gradients, targets; three products.  (Without the logits at hand one of them has to be
        # formed a second time; that is the price of not keeping them and not counted.)
        return dict(bytes=2 * e * (n + case['vocab'] * case['d']) + 8 * case['rows'], flops=6.0 * n * case['vocab'])
    if case['kind'] == 'norm':
        # x, g_x read, x_new, dx written in fp32; branch, g_y read, y, d_branch written in 16 bits.  The backward cannot
        # do without x_new either: it reads it again where it does not fit the chip's memory, which is not counted
        return dict(bytes=(16 + 4 * e) * n + 8 * case['d'], flops=0)
    if case['kind'] == 'gate':
        return dict(bytes=6 * e * n, flops=0)             # a, b, g_y; y, da, db
    return dict(bytes=4 * e * n, flops=0)                 # x, g_y; y, dx
