"""Calls at the edge of what the gate, dropout, norm and loss ops take: operands elsewhere, gradients of any alignment and
rows of any stride, hooked modules, second derivatives, captured steps."""
import pytest
import torch

import ulm_ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') * std).to(dtype)


@pytest.mark.parametrize('op', [ulm_ops.swiglu, lambda a, b: ulm_ops.swiglu_dropout(a, b, 0.5, 1)])
@pytest.mark.parametrize('elsewhere', ['cpu', 'meta'])
def test_gate_refuses_operands_of_two_devices(op, elsewhere):
    a = torch.ones(4, 64, device='cuda')
    with pytest.raises(ValueError, match='one CUDA device'):
        op(a, torch.ones(4, 64, device=elsewhere))
    with pytest.raises(ValueError, match='one CUDA device'):
        op(torch.ones(4, 64, device=elsewhere), a)


@pytest.mark.parametrize('bad', ['weight on the host', 'short weight', 'long weight', 'branch on the host'])
def test_norms_refuse_what_they_cannot_read(bad):
    x, b = torch.ones(4, 64, device='cuda'), torch.ones(4, 64, dtype=F16, device='cpu' if bad == 'branch on the host' else 'cuda')
    w = torch.ones({'short weight': 32, 'long weight': 65}.get(bad, 64), device='cpu' if bad == 'weight on the host' else 'cuda')
    with pytest.raises(ValueError):
        ulm_ops.add_rms_norm(x, b, w)
    if bad != 'branch on the host':
        for dtype in (F16, BF16, F32):
            with pytest.raises(ValueError, match='one weight per column'):
                ulm_ops.rms_norm(x.to(dtype), w)
