"""The model with rotary positions of another form, norms around its branches and activations in 8 bits: alone, together, as a step runs them."""
import pytest
import torch

import flash_attn_v100_cuda as fa
import ulm_dp
import ulm_infer
import ulm_model
import ulm_ops
import ulm_train
from oracle import rotary as ro

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
YARN = dict(kind='yarn', factor=4.0, original_length=64)
OPTIONS = {
    'plain': {},
    'rotary': dict(rotary=dict(base=5000.0)),
    'rotary, part of a head': dict(rotary=dict(rotary_dim=32, interleaved=True, scaling=YARN)),
    'norms': dict(branch_norm=True),
    'norms, gate and scale': dict(branch_norm=True, branch_gate=True, branch_scale=0.5),
    '8 bits': dict(activations_8bit=True),
    'all': dict(rotary=dict(rotary_dim=48, scaling=YARN), branch_norm=True, branch_gate=True, branch_scale=0.25, activations_8bit=True, streamed_loss=True),
}


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') * std).to(dtype)


def tiny(seed=0, **config):
    model, _ = ulm_train.build('tiny64', 'cuda', seed=seed, **config)
    with torch.no_grad():                                  # weights that give the branches something to do
        for n, p in model.named_parameters():
            if p.dim() == 2 and 'embedding' not in n and 'fc_out' not in n:
                p.mul_(4)
    return model


def ids_of(n=4, length=120, seed=3):
    return torch.randint(4, 4096, (n, length), generator=torch.Generator().manual_seed(seed)).cuda()


# ---------------------------------------------------------------------------
# the model against its definition in 64 bits
# ---------------------------------------------------------------------------
def rms64(x, w, eps=1e-6):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def turned64(x, rotary):
    angle = ro.angles(range(x.shape[2]), rotary.turns.cpu().numpy()).to(x.device)
    c, s, n = angle.cos() * rotary.factor, angle.sin() * rotary.factor, angle.shape[-1]
    i = torch.arange(n, device=x.device) * (2 if rotary.interleaved else 1)
    j = i + (1 if rotary.interleaved else n)
    a, b = x[..., i], x[..., j]
    out = x.clone()
    out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    return out


def loss64(model, p, ids):
    """The shifted mean cross-entropy in float64, of the parameters ``p`` by name."""
    cfg, (n, L) = model.config, ids.shape
    x = p['embedding.weight'][ids]
    H = cfg.n_heads
    bias = torch.full((L, L), float('-inf'), dtype=torch.float64, device='cuda').triu(1)
    for i in range(cfg.n_layers):
        w = lambda name: p[f'layers.{i}.{name}.weight']            # noqa: E731, B023

        def add(x, branch, post, h):
            if f'layers.{i}.{post}.weight' not in p:               # noqa: B023
                return x + branch
            branch = rms64(branch, w(post))
            if cfg.branch_gate:
                branch = branch * torch.sigmoid(h @ w(post + '.gate').T)
            return x + (branch if cfg.branch_scale is None else branch * p[f'layers.{i}.{post}.scale'])      # noqa: B023
        h = rms64(x, w('norm1'))
        q, k, v = (h @ w('self_attn.wqkv').T).view(n, L, 3, H, 64).unbind(2)
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        if model.rotary is not None:
            q, k = turned64(q, model.rotary), turned64(k, model.rotary)
        else:
            cos, sin = (t[0, :L, :64].double() for t in (model.rope.cos_cached, model.rope.sin_cached))
            half = lambda t: torch.cat([-t[..., 32:], t[..., :32]], -1)      # noqa: E731
            q, k = q * cos + half(q) * sin, k * cos + half(k) * sin
        a = torch.softmax(q @ k.transpose(-1, -2) / 8 + bias, -1) @ v
        x = add(x, a.transpose(1, 2).reshape(n, L, -1) @ w('self_attn.wo').T, 'attn_post', h)
        h = rms64(x, w('norm2'))
        x = add(x, (torch.nn.functional.silu(h @ w('ff.w1').T) * (h @ w('ff.w3').T)) @ w('ff.w2').T, 'ff_post', h)
    z = rms64(x, p['norm.weight']) @ p['embedding.weight'].T
    return torch.nn.functional.cross_entropy(z[:, :-1].reshape(-1, z.shape[-1]), ids[:, 1:].reshape(-1), ignore_index=0)


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('name', list(OPTIONS))
def test_loss_and_gradients_against_64_bits(name, dtype):
    model, ids = tiny(**OPTIONS[name]), ids_of()
    with torch.autocast('cuda', dtype=dtype):
        loss = model.compute_loss(ids)
    (loss * 1024).backward()
    p = {n: t.detach().double().requires_grad_() for n, t in model.named_parameters()}
    want = loss64(model, p, ids)
    grads = torch.autograd.grad(want * 1024, list(p.values()))
    unit = {F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype]
    # about forty roundings to 16 bits lie between a weight and the loss (ten a branch, four branches), growing as their root when they
    # are independent; the kept 8 bits put 0.7 to 0.9 % of noise on one or two factors of a weight's gradient
    assert abs(float(loss) - float(want)) <= 8 * unit * 2
    noise = 0.02 if model.config.activations_8bit else 0.0
    got = dict(model.named_parameters())
    for (n, q), g in zip(p.items(), grads):
        assert got[n].grad is not None and got[n].grad.shape == got[n].shape
        scale = g.norm() if g.numel() > 1 else sum(t.norm() for t, m in zip(grads, p) if m.endswith('scale'))
        assert float((got[n].grad.double() - g).norm()) <= (12 * unit + noise) * float(scale), n


@pytest.mark.parametrize('name', list(OPTIONS))
def test_checkpointed_steps_have_the_same_gradients(name):
    ids, grads = ids_of(), []
    for checkpointing in (False, True):
        model = tiny(use_gradient_checkpointing=checkpointing, **OPTIONS[name])
        with torch.autocast('cuda', dtype=BF16):
            loss = model.compute_loss(ids)
        loss.backward()
        grads.append([p.grad for p in model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_state_dicts_go_round_and_the_options_add_what_they_say():
    keys = {name: set(ulm_model.DecoderOnlyTransformer(ulm_model.ModelConfig(vocab_size=96, d_model=64, n_heads=1, n_layers=1, d_ff=128, max_seq_len=32, **o)).state_dict())
            for name, o in OPTIONS.items()}
    assert keys['8 bits'] == keys['plain']
    assert keys['plain'] - keys['rotary'] == {'rope.inv_freq', 'rope.cos_cached', 'rope.sin_cached'} and not keys['rotary'] - keys['plain']
    assert keys['norms'] - keys['plain'] == {f'layers.0.{n}.weight' for n in ('attn_post', 'ff_post')}
    assert keys['norms, gate and scale'] - keys['norms'] == {f'layers.0.{n}.{k}' for n in ('attn_post', 'ff_post') for k in ('gate.weight', 'scale')}
    assert ulm_train.build('tiny64', 'cpu', rotary={})[0].rotary.rotary_dim == 64 and ulm_train.build('tiny64', 'cpu')[0].rotary is None
    a, b = tiny(1, **OPTIONS['all']), tiny(2, **OPTIONS['all'])
    b.load_state_dict(a.state_dict(), strict=True)
    with torch.autocast('cuda', dtype=BF16):
        assert torch.equal(a.compute_loss(ids_of()).detach(), b.compute_loss(ids_of()).detach())


def test_a_model_built_on_the_device():
    with torch.device('cuda'):
        model, _ = ulm_train.build('tiny64', 'cuda', **OPTIONS['all'])
    with torch.autocast('cuda', dtype=BF16):
        model.compute_loss(ids_of()).backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())


@pytest.mark.parametrize('bad', [dict(branch_gate=True), dict(branch_scale=1.0), dict(rotary=dict(rotary_dim=66)), dict(rotary=dict(rotary_dim=31)), dict(rotary=dict(width=64))])
def test_options_that_do_not_fit_are_refused(bad):
    with pytest.raises((ValueError, TypeError)):
        ulm_train.build('tiny64', 'cpu', **bad)


@pytest.mark.parametrize('dropout', [0.0, 0.2])
def test_what_a_forward_keeps(dropout):
    kept = {}
    for bits in (False, True):
        model = tiny(dropout=dropout, counter_dropout=True, activations_8bit=bits)
        for layer in model.layers:
            layer.self_attn.dropout = 0.0
        own, seen = {p.untyped_storage().data_ptr() for p in model.parameters()}, {}

        def count(t):
            if t.untyped_storage().data_ptr() not in own:          # noqa: B023
                seen[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()      # noqa: B023
            return t
        with torch.autograd.graph.saved_tensors_hooks(count, lambda t: t), torch.autocast('cuda', dtype=BF16), ulm_ops.weight_cast_scope():
            h = model.forward_hidden(ids_of(16, 256))
        kept[bits] = sum(seen.values())
        del h
    tokens, ff, d = 16 * 256, 344, 128
    # a token and layer: 6 ff bytes become 2 1/16 ff, the two normalised inputs' 4 d 2 1/16 d
    assert kept[False] - kept[True] == 2 * tokens * ((6 - 2.0625) * ff + (4 - 2.0625) * d)


def test_dropout_that_is_not_counted_takes_the_kept_path(monkeypatch):
    model = tiny(dropout=0.5, activations_8bit=True)
    monkeypatch.setattr(ulm_model, 'feed_forward_8bit', None)      # not called
    with torch.autocast('cuda', dtype=BF16):
        model.compute_loss(ids_of()).backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    model.eval()
    with pytest.raises(TypeError), torch.autocast('cuda', dtype=BF16):
        model.compute_loss(ids_of())                       # idle: nothing to drop


@pytest.mark.parametrize('name', ['all', 'norms, gate and scale'])
def test_dropout_with_the_options(name):
    model, ids = tiny(dropout=0.2, counter_dropout=True, **OPTIONS[name]), ids_of()
    for layer in model.layers:
        layer.self_attn.dropout = 0.0
    losses = []
    for seed in (5, 5, 6):
        torch.manual_seed(seed)
        with torch.autocast('cuda', dtype=BF16):
            loss = model.compute_loss(ids)
        losses.append((float(loss.detach()), torch.autograd.grad(loss, list(model.parameters()))))
    assert losses[0][0] == losses[1][0] != losses[2][0]
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(losses[0][1], losses[1][1]))


@pytest.mark.parametrize('name', ['norms, gate and scale', 'all'])
def test_training_steps(name):
    model = tiny(**OPTIONS[name])
    step = ulm_dp.DataParallelStep(model, ulm_train.make_optimizer(model), samples_per_step=7, autocast_dtype=BF16)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    batches = [[ids_of(4, 100, s).cpu(), ids_of(3, 77, s + 10).cpu()] for s in range(3)]
    for b in batches:
        assert float(step.step(b)[0]) > 0
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n


def test_evaluation_and_scoring():
    model = tiny(**OPTIONS['all']).eval()
    windows = [torch.randint(4, 4096, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (2, 30, 77, 120)]
    losses, tokens, correct = ulm_infer.score_windows(model, windows, 0, torch.device('cuda'), 2, 64, amp_dtype=BF16)
    p = {n: t.detach().double() for n, t in model.named_parameters()}
    for w, got, n in zip(windows, losses, tokens):
        want = float(loss64(model, p, torch.tensor([w]).cuda())) * (len(w) - 1)
        assert n == len(w) - 1 and abs(got - want) <= 16 * 2.0 ** -8 * n
    ids = ids_of(2, 40)
    with torch.no_grad(), torch.autocast('cuda', dtype=BF16):
        one = model.forward_hidden(ids)
    with torch.autocast('cuda', dtype=BF16):
        two = model.forward_hidden(ids)
    assert torch.equal(one, two.detach())                  # with and without a graph


# ---------------------------------------------------------------------------
# the attention block on rotary positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('kw', [dict(rotary_dim=64), dict(rotary_dim=20, interleaved=True, scaling=YARN), dict(rotary_dim=64, interleaved=True)])
@pytest.mark.parametrize('n,L,H', [(1, 1, 1), (3, 67, 2), (2, 300, 5)])
@pytest.mark.parametrize('flat', [False, True])
def test_attention_block_is_rotation_and_attention(dtype, kw, n, L, H, flat):
    rotary = ulm_ops.Rotary(**kw).cuda()
    pad = 5 if flat else 0
    base = randn((n * L + pad, 3 * H * 64), dtype, 1)
    qkv = (base if flat else base.view(n, L, -1)).detach().requires_grad_()
    at = torch.randint(0, 5000, (n, L), generator=torch.Generator().manual_seed(2)).cuda()
    out = fa.qkv_rope_flash_attn(qkv, H, rotary=rotary, positions=at, flat_shape=(n, L) if flat else None)
    up = randn(out.shape, dtype, 3)
    g, = torch.autograd.grad(out, qkv, up)
    ref = base[:n * L].detach().requires_grad_()
    q, k, v = (t.transpose(1, 2) for t in ref.view(n, L, 3, H, 64).unbind(2))
    o = fa.flash_attn_v100(*rotary(q, k, at), v)
    want = o.transpose(1, 2).reshape(n * L, H * 64)
    gw, = torch.autograd.grad(want, ref, up.reshape(-1, H * 64)[:n * L])
    assert torch.equal(out.reshape(-1, H * 64)[:n * L], want) and torch.equal(g.reshape(-1, 3 * H * 64)[:n * L], gw)
    if flat:
        assert not out[n * L:].any() and not g[n * L:].any()
    else:
        a, ka, va = ulm_infer.causal_attention(qkv.detach(), H, rotary=rotary, positions=at)
        assert torch.equal(a, out) and torch.equal(ka, rotary(q, k, at)[1]) and torch.equal(va, v)


def test_rotary_with_the_tables_angles_is_the_tables_rope():
    """Half layout, all 64 columns, frequencies of a 64-wide table: the two paths agree to 16-bit rounding."""
    qkv = randn((2, 90, 3 * 128), BF16, 1)
    cos, sin = (t.cuda() for t in ulm_model.rope_tables(64, 90))
    a = fa.qkv_rope_flash_attn(qkv, 2, cos, sin)
    b = fa.qkv_rope_flash_attn(qkv, 2, rotary=ulm_ops.Rotary(64).cuda())
    assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -6


def test_attention_block_refusals_and_empty_inputs():
    qkv, rotary = torch.zeros(2, 5, 192, dtype=F16, device='cuda'), ulm_ops.Rotary(64).cuda()
    cos = torch.zeros(5, 64, device='cuda')
    for kw in (dict(cos2d=cos, sin2d=cos), dict(fuse='none'), dict(positions=torch.zeros(4, dtype=torch.int64, device='cuda')), dict(positions=torch.zeros(5, dtype=torch.int64))):
        with pytest.raises(ValueError):
            fa.qkv_rope_flash_attn(qkv, 1, rotary=rotary, **kw)
    with pytest.raises(ValueError):
        fa.qkv_rope_flash_attn(qkv, 1, positions=torch.arange(5, device='cuda'))
    with pytest.raises(ValueError):
        fa.qkv_rope_flash_attn(qkv, 1, rotary=ulm_ops.Rotary(66).cuda())
    with pytest.raises(ValueError):
        fa.qkv_rope_flash_attn(qkv, 1, rotary=ulm_ops.Rotary(64))              # on the host
    with pytest.raises(ValueError):
        ulm_infer.causal_attention(qkv, 1, cos, cos, rotary=rotary)
    with pytest.raises(ValueError):
        ulm_infer.causal_attention(qkv.float(), 1, rotary=rotary)
    e = torch.ones(0, 5, 192, dtype=F16, device='cuda', requires_grad=True)
    out = fa.qkv_rope_flash_attn(e, 1, rotary=rotary)
    assert out.shape == (0, 5, 64) and torch.autograd.grad(out.sum(), e)[0].shape == e.shape


def test_a_cached_context_is_continued():
    """Serving: keys turned at their own positions once, a new token turned at its; the scores are those of the whole sequence."""
    rotary = ulm_ops.Rotary(64, scaling=YARN).cuda()
    n, L, H = 3, 41, 2
    q, k = randn((n, L, H, 64), torch.float32, 1).transpose(1, 2), randn((n, L, H, 64), torch.float32, 2).transpose(1, 2)
    whole_q, whole_k = rotary(q, k)
    cache = torch.cat([rotary(q[:, :, s:e], k[:, :, s:e], torch.arange(s, e, device='cuda'))[1] for s, e in ((0, 20), (20, 40))], 2)
    new_q, new_k = rotary(q[:, :, 40:], k[:, :, 40:], torch.full((n, 1), 40, device='cuda'))
    assert torch.equal(torch.cat([cache, new_k], 2), whole_k) and torch.equal(new_q, whole_q[:, :, 40:])


# ---------------------------------------------------------------------------
# what a differentiable op owes its callers
# ---------------------------------------------------------------------------
class Traced(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.w, self.s = torch.nn.Parameter(torch.ones(64, device='cuda')), torch.nn.Parameter(torch.tensor(0.5, device='cuda'))
        self.rotary = ulm_ops.Rotary(16, interleaved=True).cuda()

    def forward(self, x):
        q, k = self.rotary(x.view(1, -1, 2, 32).transpose(1, 2), x.view(1, -1, 2, 32).transpose(1, 2))
        b = (q + k).transpose(1, 2).reshape(x.shape).half()
        x_new, y = ulm_ops.norm_add_norm(x, b, self.w, self.w, gate=b, scale=self.s)
        return x_new + ulm_ops.swiglu_8bit(y.float(), x_new)


def test_traced_ops_run_again_on_other_inputs():
    m, x = Traced(), randn((24, 64), torch.float32, 1)
    got, want = torch.jit.trace(m, randn((24, 64), torch.float32, 2))(x), m(x)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got.sum(), list(m.parameters())), torch.autograd.grad(want.sum(), list(m.parameters()))):
        assert float((a - b).norm()) <= 2.0 ** -10 * float(b.norm())       # 16-bit gradients rounded once more by the trace's casts


OPS = {
    'rotary': lambda x: ulm_ops.rotary(x.view(1, 1, 4, 64), None, ulm_ops.rotary_turns(64)[0].cuda())[0],
    'norm_add_norm': lambda x: ulm_ops.norm_add_norm(x, torch.ones(4, 64, device='cuda').half(), torch.ones(64, device='cuda'), torch.ones(64, device='cuda'))[0],
    'swiglu_8bit': lambda x: ulm_ops.swiglu_8bit(x, x),
    'linear_8bit': lambda x: ulm_ops.linear_8bit(x, torch.ones(8, 64, device='cuda')),
    'feed_forward_8bit': lambda x: ulm_ops.feed_forward_8bit(x, *(torch.ones(64, 64, device='cuda') for _ in range(3))),
}


@pytest.mark.parametrize('name', list(OPS))
def test_transforms_without_a_rule_are_refused(name):
    with pytest.raises((RuntimeError, NotImplementedError), match='autograd.Function'):
        torch.func.grad(lambda x: OPS[name](x).sum())(torch.ones(4, 64, device='cuda'))


@pytest.mark.parametrize('name', list(OPS))
def test_without_a_graph_and_through_saved_tensor_hooks(name):
    x = randn((4, 64), torch.float32, 1)
    want = OPS[name](x)
    with torch.inference_mode():
        assert torch.equal(OPS[name](x), want)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        parked = OPS[name](a)
    y = OPS[name](b)
    assert torch.equal(y.detach(), want) and torch.equal(*(torch.autograd.grad(t.sum(), u)[0] for t, u in ((parked, a), (y, b))))
    first, again = (torch.autograd.grad(OPS[name](b).sum(), b, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(first, again)


def test_a_graph_runs_backward_twice():
    x = randn((4, 64), torch.float32, 1).requires_grad_()
    for f in OPS.values():
        y = f(x)
        assert torch.equal(*(torch.autograd.grad(y.sum(), x, retain_graph=True)[0] for _ in range(2)))


def test_two_threads_at_once():
    import threading
    model, ids, out = tiny(**OPTIONS['all']), ids_of(), {}

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()), torch.autocast('cuda', dtype=BF16):
            for _ in range(3):
                loss = model.compute_loss(ids)
                out[i] = (loss.detach(), torch.autograd.grad(loss, list(model.parameters())))
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert torch.equal(out[0][0], out[1][0]) and all(torch.equal(a, b) for a, b in zip(out[0][1], out[1][1]))


def test_a_whole_step_replays():
    """Forward and backward of a block's ops captured once, replayed on other values."""
    rotary, w = ulm_ops.Rotary(64).cuda(), torch.ones(128, device='cuda')
    qkv, x, up = randn((2, 33, 384), BF16, 1), randn((2, 33, 128), torch.float32, 2), randn((2, 33, 128), BF16, 3)
    w1, w3, w2 = randn((96, 128), BF16, 4, 0.1), randn((96, 128), BF16, 5, 0.1), randn((128, 96), BF16, 6, 0.1)
    leaves = [t.requires_grad_() for t in (qkv, x, w1, w3, w2)]

    def step():
        a = fa.qkv_rope_flash_attn(qkv, 2, rotary=rotary)
        x_new, h = ulm_ops.norm_add_norm(x, a, w, w, gate=a, scale=0.5)
        y = ulm_ops.feed_forward_8bit(h, w1, w3, w2)
        return (x_new.detach(), y.detach(), *torch.autograd.grad([x_new, y], leaves, [x_new.detach(), up]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    with torch.no_grad():
        qkv.mul_(-1.5), x.add_(1), w1.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, step()):
        assert float((a - b).float().norm()) <= 2.0 ** -7 * float(b.float().norm())       # library products may be summed in another order
