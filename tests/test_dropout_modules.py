"""A dropout module that somebody watches or has changed is called; only one that nobody can tell apart is left to a kernel."""
import pytest
import torch
import torch.nn.modules.module as base

import ulm_model
import ulm_ops

WATCHED = {
    'forward hook': lambda m, seen: m.register_forward_hook(lambda *a: seen.append(1)),
    'forward pre-hook': lambda m, seen: m.register_forward_pre_hook(lambda *a: seen.append(1)),
    'backward hook': lambda m, seen: m.register_full_backward_hook(lambda *a: seen.append(1)),
    'backward pre-hook': lambda m, seen: m.register_full_backward_pre_hook(lambda *a: seen.append(1)),
    'global forward hook': lambda m, seen: base.register_module_forward_hook(lambda *a: seen.append(1)),
    'global backward hook': lambda m, seen: base.register_module_full_backward_hook(lambda *a: seen.append(1)),
}


def patch_forward(module, seen):
    def forward(x):
        seen.append(1)
        return x * 1.0
    module.forward = forward


@pytest.mark.parametrize('how', [*WATCHED, 'forward of its own'])
def test_a_watched_module_is_called(how):
    for module, use in ((torch.nn.Dropout(0.0), lambda m, x: ulm_model._drop(m, x)),
                        (ulm_ops.Dropout(0.5), lambda m, x: None if ulm_model._mask_of(m) is not None else m.eval()(x * 1.0))):
        seen, handle, x = [], None, torch.ones(3, requires_grad=True)
        assert ulm_model._mask_of(module) is not None or type(module) is torch.nn.Dropout
        try:
            handle = WATCHED[how](module, seen) if how in WATCHED else patch_forward(module, seen)
            y = use(module, x)
            assert y is not None, 'its work was handed to a kernel'
            y.sum().backward()
        finally:
            if handle is not None:
                handle.remove()
        assert seen == [1]


@pytest.mark.gpu
@pytest.mark.parametrize('how', ['backward hook', 'forward of its own'])
def test_the_model_calls_a_watched_module(how):
    import ulm_train
    model, _ = ulm_train.build('tiny64', 'cuda', dropout=0.2, counter_dropout=True, streamed_loss=True)
    seen = []
    for module in (model.layers[0].dropout, model.layers[1].ff.dropout):
        WATCHED[how](module, seen) if how in WATCHED else patch_forward(module, seen)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        loss = model.compute_loss(torch.randint(4, 4096, (3, 40), generator=torch.Generator().manual_seed(3)).cuda())
    loss.backward()
    assert len(seen) == 2
