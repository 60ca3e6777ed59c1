"""Modules put in the place of the model's own, on the host: they are called as they always were."""
import pytest
import torch

import ulm_model

CONFIG = dict(vocab_size=96, d_model=64, n_heads=1, n_layers=2, d_ff=128, max_seq_len=32, use_rope=True)


class Norm(torch.nn.Module):
    """The norms' interface without their kernels."""

    def forward(self, x):
        return x * 0.5

    def add_forward(self, x, branch, dropout_p=0.0, seed=0):
        return x + branch, (x + branch) * 0.5


class Attention(torch.nn.Module):
    head_dim = 64

    def __init__(self):
        super().__init__()
        self.w = torch.nn.Linear(64, 64, bias=False)

    def forward(self, x, cos=None, sin=None, shape=None):
        assert cos is not None and shape == (3, 5)
        return self.w(x)


class FeedForward(torch.nn.Module):
    def forward(self, x):
        return x.tanh()


class Layer(torch.nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x, pending=None, cos=None, sin=None, shape=None):
        return self.inner(x, pending, cos=cos, sin=sin, shape=shape)


def model_of(wrapped, **config):
    torch.manual_seed(1)
    model = ulm_model.DecoderOnlyTransformer(ulm_model.ModelConfig(**CONFIG, **config))
    model.norm = Norm()
    for i, layer in enumerate(model.layers):
        layer.norm1, layer.norm2, layer.self_attn, layer.ff = Norm(), Norm(), Attention(), FeedForward()
        if wrapped:
            model.layers[i] = Layer(layer)
            model.layers[i].self_attn = layer.self_attn    # the model asks the first layer for its heads' width
    return model


@pytest.mark.parametrize('wrapped', [False, True])
@pytest.mark.parametrize('checkpointing', [False, True])
@pytest.mark.parametrize('options', [{}, dict(activations_8bit=True)])
def test_modules_that_know_of_no_options(wrapped, checkpointing, options):
    model = model_of(wrapped, use_gradient_checkpointing=checkpointing, dropout=0.0, **options)
    ids = torch.arange(15).view(3, 5)
    out = model.forward_hidden(ids)
    x = model.embedding(ids.reshape(-1))
    for layer in model.layers:
        x = x + layer.self_attn(x * 0.5, cos=1, shape=(3, 5))
        x = x + (x * 0.5).tanh()
    assert torch.allclose(out.reshape(15, 64), x * 0.5, rtol=0, atol=2.0 ** -20)      # eight roundings of numbers below 2
    out.sum().backward()
    assert model.layers[0].self_attn.w.weight.grad.any()


def test_a_model_pickled_whole_before_the_options():
    model, ids = model_of(False, dropout=0.0), torch.arange(15).view(3, 5)
    want = model.forward_hidden(ids)
    del model.rotary
    for layer in model.layers:
        del layer.attn_post, layer.ff_post
    assert torch.equal(model.forward_hidden(ids), want)
    for module in (ulm_model.MultiHeadAttention(model.config), ulm_model.FeedForward(64, 128, 0.0)):
        del module.activations_8bit
        assert module.activations_8bit is False
