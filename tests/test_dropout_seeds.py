"""Where the seeds of unstored dropout masks come from."""
import pytest
import torch

import ulm_ops


def seeds():
    torch.manual_seed(5)
    return [ulm_ops.next_dropout_seed() for _ in range(3)]


@pytest.mark.parametrize('device', ['meta', pytest.param('cuda', marks=pytest.mark.gpu)])
def test_seeds_are_the_cpu_generators_under_any_default_device(device):
    want = seeds()
    with torch.device(device):
        assert seeds() == want
    torch.set_default_device(device)
    try:
        assert seeds() == want
    finally:
        torch.set_default_device(None)


def test_a_traced_module_would_drop_the_same_elements_every_time():
    m, x = ulm_ops.Dropout(0.5), torch.ones(4, 64)
    with pytest.raises(RuntimeError, match='every run'):
        torch.jit.trace(m, x)
    assert torch.equal(torch.jit.trace(m.eval(), x)(x), x)                     # idle: nothing to draw


@pytest.mark.gpu
def test_a_captured_module_would_drop_the_same_elements_every_time():
    m, x = ulm_ops.Dropout(0.5), torch.ones(4, 64, device='cuda')
    want = ulm_ops.dropout(x, 0.5, 7)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match='every run'):
            m(x)
        got = ulm_ops.dropout(x, 0.5, 7)                  # a seed that the caller chose is the caller's word
        idle = m.eval()(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and idle is x
    assert m.train()(x).shape == x.shape
