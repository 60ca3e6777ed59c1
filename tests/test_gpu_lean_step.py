"""The model with dropout masks that are not stored and a loss without logits, run as a training step runs it."""
import pytest
import torch

import flash_attn_v100_cuda as fa
import ulm_dp
import ulm_model
import ulm_ops
import ulm_train
from oracle import dropout as od

pytestmark = pytest.mark.gpu

P = 0.2


class Explicit(torch.nn.Module):
    """Dropout by a mask that the oracle made: the plain form of `ulm_ops.Dropout`."""

    def forward(self, x):
        keep = torch.from_numpy(od.keep_mask(x.numel(), P, ulm_ops.next_dropout_seed()).reshape(x.shape)).cuda()
        return torch.where(keep, x * od.scale(P), 0.0).to(x.dtype)


def tiny(seed=0, **config):
    model, preset = ulm_train.build('tiny64', 'cuda', seed=seed, **config)
    for layer in model.layers:
        layer.self_attn.dropout = 0.0                      # the attention's own mask comes from another generator
    return model, preset


def ids_of(n=6, length=200, seed=3):
    ids = torch.randint(4, 4096, (n, length), generator=torch.Generator().manual_seed(seed))
    ids[:, length - 20:] = torch.where(torch.arange(n)[:, None] % 2 == 0, 0, ids[:, length - 20:])      # padding, as the collate makes it
    return ids.cuda()


def counted_seeds(monkeypatch):
    drawn = []

    def draw():
        drawn.append(1000 + len(drawn))
        return drawn[-1]
    monkeypatch.setattr(ulm_ops, 'next_dropout_seed', draw)
    return drawn


@pytest.mark.parametrize('dtype,loss_tol,grad_tol', [(torch.float16, 1e-3, 2e-2), (torch.bfloat16, 8e-3, 6e-2)])
def test_step_equals_its_plain_composition(monkeypatch, dtype, loss_tol, grad_tol):
    lean, _ = tiny(dropout=P, counter_dropout=True, streamed_loss=True)
    plain, _ = tiny(dropout=P)
    for layer in plain.layers:
        layer.dropout, layer.ff.dropout = Explicit(), Explicit()
    ids, got = ids_of(), []
    for model in (lean, plain):
        drawn = counted_seeds(monkeypatch)
        with torch.autocast('cuda', dtype=dtype):
            loss = model.compute_loss(ids)
        loss.backward()
        assert drawn == [1000, 1001, 1002, 1003]           # the gate's and the residual's mask of both blocks
        got.append((float(loss.detach()), {n: p.grad for n, p in model.named_parameters()}))
    fa.check_status()
    # 16-bit activations through two blocks, rounded at other places: the bounds of the model's own comparison with its oracle
    assert abs(got[0][0] - got[1][0]) <= loss_tol
    for name, g in got[1][1].items():
        assert float((got[0][1][name] - g).norm()) <= grad_tol * float(g.norm()), name


def test_evaluation_is_that_of_the_plain_model():
    a, _ = tiny(dropout=P, counter_dropout=True, streamed_loss=True)
    b, _ = tiny(dropout=P)
    ids = ids_of()
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        x, y = a.eval().forward_hidden(ids), b.eval().forward_hidden(ids)
        la, lb = a.compute_loss(ids), b.compute_loss(ids)
    assert torch.equal(x, y)
    assert abs(float(la) - float(lb)) <= 2.0 ** -8 * float(lb)        # one rounds its logits to bf16


def test_checkpointed_blocks_drop_the_same_elements_again():
    out = []
    for checkpointing in (False, True):
        model, _ = tiny(dropout=P, counter_dropout=True, streamed_loss=True, use_gradient_checkpointing=checkpointing)
        torch.manual_seed(11)
        with torch.autocast('cuda', dtype=torch.bfloat16):
            loss = model.compute_loss(ids_of())
        loss.backward()
        out.append((loss.detach(), [p.grad for p in model.parameters()]))
    assert torch.equal(out[0][0], out[1][0])
    for a, b in zip(out[0][1], out[1][1]):
        assert float((a - b).norm()) <= 1e-5 * float(a.norm())        # library GEMMs may sum in another order


def test_masks_differ_from_call_to_call_and_follow_the_seed():
    model, _ = tiny(dropout=P, counter_dropout=True, streamed_loss=True)
    losses = []
    for seed in (5, None, 5):
        if seed is not None:
            torch.manual_seed(seed)
        with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
            losses.append(float(model.compute_loss(ids_of())))
    assert losses[0] == losses[2] != losses[1]


def test_a_hooked_or_replaced_module_is_called():
    model, _ = tiny(dropout=P, counter_dropout=True)
    seen = []
    model.layers[0].dropout.register_forward_hook(lambda m, a, y: seen.append(y.shape))
    model.layers[1].ff.dropout = torch.nn.Identity()
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        model.compute_loss(ids_of())
    assert len(seen) == 1


def test_data_parallel_step_learns_with_both():
    model, preset = ulm_train.build('tiny64', 'cuda', dropout=0.1, counter_dropout=True, streamed_loss=True)
    step = ulm_dp.DataParallelStep(model, ulm_train.make_optimizer(model, lr=1e-3), samples_per_step=6, autocast_dtype=preset['dtype'])
    batch = [ids_of().cpu()]
    losses = [float(step.step(batch)[0]) for _ in range(30)]
    assert all(l == l for l in losses) and losses[-1] < losses[0] - 0.5


def test_no_logits_are_alive_between_forward_and_backward():
    rows, V = 16384, 32000

    def held(streamed):
        h = torch.randn(rows, 64, device='cuda', dtype=torch.bfloat16).requires_grad_()
        w = torch.randn(V, 64, device='cuda', dtype=torch.bfloat16).requires_grad_()
        t = torch.randint(0, V, (rows,), device='cuda')
        before = torch.cuda.memory_allocated()
        loss = (ulm_ops.streamed_cross_entropy if streamed else ulm_ops.chunked_cross_entropy)(h, w, t)
        alive = torch.cuda.memory_allocated() - before
        loss.backward()
        return alive
    assert held(True) <= 1 << 20 and held(False) >= 2 * rows * V


class Traced(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.w = torch.nn.Parameter(torch.ones(64, device='cuda'))

    def forward(self, x):
        b = ulm_ops.swiglu_dropout(x, ulm_ops.dropout(x, 0.3, 1), 0.3, 2)
        x_new, y = ulm_ops.dropout_add_rms_norm(x, b.half(), self.w, 0.3, 3)
        return x_new + y


def test_traced_ops_run_again_on_other_inputs():
    m, x = Traced(), torch.randn(24, 64, device='cuda')
    got, want = torch.jit.trace(m, torch.randn(8, 64, device='cuda'))(x), m(x)
    assert torch.equal(got, want)
    a, b = torch.autograd.grad(got.sum(), m.w)[0], torch.autograd.grad(want.sum(), m.w)[0]
    assert float((a - b).norm()) <= 2.0 ** -11 * float(b.norm())


@pytest.mark.parametrize('op', [
    lambda x: ulm_ops.dropout(x, 0.5, 1),
    lambda x: ulm_ops.swiglu_dropout(x, x, 0.5, 1),
    lambda x: ulm_ops.dropout_add_rms_norm(x, torch.ones(4, 64, device='cuda').half(), torch.ones(64, device='cuda'), 0.5, 1)[0],
    lambda x: ulm_ops.streamed_cross_entropy(x, torch.ones(9, 64, device='cuda'), torch.ones(4, device='cuda', dtype=torch.long), compute_dtype=torch.bfloat16),
])
def test_transforms_without_a_rule_are_refused(op):
    with pytest.raises((RuntimeError, NotImplementedError), match='autograd.Function'):
        torch.func.grad(lambda x: op(x).sum())(torch.ones(4, 64, device='cuda'))


def test_checkpointed_loss_and_saved_tensor_hooks():
    g = torch.Generator(device='cuda').manual_seed(1)
    h, w = torch.randn(300, 128, generator=g, device='cuda').half(), torch.randn(500, 128, generator=g, device='cuda').half()
    t = torch.randint(0, 500, (300,), generator=g, device='cuda')

    def grads(call):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.autograd.grad(call(a, b), [a, b])
    plain = grads(lambda a, b: ulm_ops.streamed_cross_entropy(a, b, t))
    again = grads(lambda a, b: torch.utils.checkpoint.checkpoint(ulm_ops.streamed_cross_entropy, a, b, t, use_reentrant=False))
    with torch.autograd.graph.save_on_cpu():
        parked = grads(lambda a, b: ulm_ops.streamed_cross_entropy(a, b, t))
    for other in (again, parked):
        assert all(torch.equal(x, y) for x, y in zip(other, plain))


def test_an_operand_changed_in_place_is_noticed():
    x, b, w = torch.randn(4, 64, device='cuda', requires_grad=True), torch.randn(4, 64, device='cuda').half(), torch.ones(64, device='cuda', requires_grad=True)
    x_new, y = ulm_ops.dropout_add_rms_norm(x, b, w, 0.5, 1)
    with torch.no_grad():
        x_new.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.float().sum().backward()
