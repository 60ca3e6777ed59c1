"""The model takes the reference's own configuration object, which has the reference's fields and no others."""
import types

import pytest
import torch

import ulm_model
import ulm_ops

REFERENCE_FIELDS = dict(vocab_size=96, d_model=64, n_heads=1, n_layers=2, d_ff=128, max_seq_len=32, dropout=0.1, use_rope=True, tie_weights=True,
                        use_gradient_checkpointing=False)          # train.py:725-737


def test_a_configuration_of_the_reference_builds_the_reference_model():
    model = ulm_model.DecoderOnlyTransformer(types.SimpleNamespace(**REFERENCE_FIELDS))
    ours = ulm_model.DecoderOnlyTransformer(ulm_model.ModelConfig(**REFERENCE_FIELDS))
    assert {n: p.shape for n, p in model.state_dict().items()} == {n: p.shape for n, p in ours.state_dict().items()}
    for layer in model.layers:
        assert type(layer.dropout) is torch.nn.Dropout and type(layer.ff.dropout) is torch.nn.Dropout


@pytest.mark.gpu
def test_its_loss_is_the_chunked_one(monkeypatch):
    monkeypatch.setattr(ulm_ops, 'streamed_cross_entropy', None)
    losses = []
    for config in (types.SimpleNamespace(**REFERENCE_FIELDS), ulm_model.ModelConfig(**REFERENCE_FIELDS)):
        torch.manual_seed(1)
        model = ulm_model.DecoderOnlyTransformer(config).cuda().eval()
        with torch.autocast('cuda', dtype=torch.bfloat16):
            losses.append(model.compute_loss(torch.randint(1, 96, (3, 20), generator=torch.Generator().manual_seed(2)).cuda()))
        losses[-1].backward()
    assert torch.equal(losses[0].detach(), losses[1].detach())
