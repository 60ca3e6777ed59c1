"""Frequencies of the rotary positions, and which calls are refused on the host."""
import math
from fractions import Fraction

import pytest
import torch

import ulm_ops


def radians(turns):
    return [Fraction(int(t), 1 << 64) * 2 * Fraction(math.pi) for t in turns]


@pytest.mark.parametrize('dim', [2, 6, 20, 64, 128, 256])
@pytest.mark.parametrize('base', [10000.0, 500000.0, 2.0])
def test_frequencies_are_powers_of_the_base(dim, base):
    turns, factor = ulm_ops.rotary_turns(dim, base)
    assert turns.dtype == torch.int64 and turns.shape == (dim // 2,) and factor == 1.0
    for i, w in enumerate(radians(turns)):
        # a power, a quotient by 2 pi and its rounding to 64 bits
        assert abs(float(w) - base ** (-2 * i / dim)) <= 2.0 ** -50 * base ** (-2 * i / dim) + 2.0 ** -61


@pytest.mark.parametrize('dim', [2, 64, 96])
def test_stretched_frequencies(dim):
    plain = [float(w) for w in radians(ulm_ops.rotary_turns(dim)[0])]
    get = lambda **kw: ulm_ops.rotary_turns(dim, scaling=kw)       # noqa: E731
    close = lambda a, b: abs(a - b) <= 2.0 ** -48 * abs(b)         # noqa: E731
    lin, f = get(kind='linear', factor=4.0)
    assert f == 1.0 and all(close(float(w), p / 4) for w, p in zip(radians(lin), plain))
    ntk, f = get(kind='ntk', factor=4.0)
    ntk = [float(w) for w in radians(ntk)]
    assert f == 1.0 and close(ntk[0], 1.0) and (dim == 2 or close(ntk[-1], plain[-1] / 4))
    for kind, fast in (('parts', 4.0), ('yarn', 32.0)):
        got, f = get(kind=kind, factor=4.0, original_length=4096, slow=1.0, fast=fast)
        assert close(f, 0.1 * math.log(4.0) + 1.0) if kind == 'yarn' else f == 1.0
        for w, p in zip(radians(got), plain):
            turned = 4096 * p / (2 * math.pi)
            keep = min(1.0, max(0.0, (turned - 1.0) / (fast - 1.0)))
            assert close(float(w), p * keep + p / 4 * (1 - keep))
            assert (turned < fast or close(float(w), p)) and (turned > 1 or close(float(w), p / 4))
    assert torch.equal(get(kind='yarn', factor=4.0, original_length=4096)[0], get(kind='yarn', factor=4.0, original_length=4096, slow=1.0, fast=32.0)[0])
    assert get(kind='yarn', factor=4.0, original_length=4096, attention_factor=1.25)[1] == 1.25
    assert get(kind='linear', factor=1.0)[0].equal(ulm_ops.rotary_turns(dim)[0])


@pytest.mark.parametrize('kind', ['parts', 'yarn'])
@pytest.mark.parametrize('dim,base,length,slow,fast', [(64, 10000.0, 4096, 1.0, 32.0), (128, 1e6, 32768, 1.0, 4.0), (64, 10000.0, 64, 1.0, 32.0), (8, 10000.0, 4096, 15.0, 16.0), (2, 2.0, 4096, 1.0, 32.0)])
def test_the_ramp_over_the_pairs(kind, dim, base, length, slow, fast):
    """Against borders found by counting the pairs: the last that turns at least `fast` times, the first that turns at most `slow` times."""
    f, n = 8.0, dim // 2
    got, factor = ulm_ops.rotary_turns(dim, base, dict(kind=kind, factor=f, original_length=length, slow=slow, fast=fast, ramp='pairs'))
    assert factor == (1.0 if kind == 'parts' else pytest.approx(0.1 * math.log(f) + 1.0))
    turned = [length * base ** (-2 * i / dim) / (2 * math.pi) for i in range(4 * n + 16)]      # and of pairs that a wider head would have
    first = max([i for i, t in enumerate(turned) if t >= fast], default=0)
    last = min([i for i, t in enumerate(turned) if t <= slow])
    for i, w in enumerate(radians(got)):
        stays = 1.0 if i <= first else 0.0 if i >= last else 1.0 - (i - first) / (last - first)
        plain = base ** (-2 * i / dim)
        assert abs(float(w) - (plain * stays + plain / f * (1 - stays))) <= 2.0 ** -45 * plain + 2.0 ** -62      # half of 2^-64 turns


def test_the_two_ramps_are_told_apart():
    get = lambda **kw: [float(w) for w in radians(ulm_ops.rotary_turns(64, scaling=dict(kind='yarn', factor=8.0, original_length=4096, **kw))[0])]      # noqa: E731
    turns, pairs = get(), get(ramp='pairs')
    assert get(ramp='turns') == turns
    off = [b / a for a, b in zip(turns, pairs)]
    # 652 10000^(-i/32) turns in 4096 positions: 36.7 of pair 10, 27.5 of pair 11, 1.16 of pair 22, 0.87 of pair 23; 3.67 of pair 18, of which
    # 2.67 / 31 = 0.086 and 5 / 13 = 0.385 stay: (0.385 + 0.615 / 8) / (0.086 + 0.914 / 8) = 2.3
    assert [i for i, r in enumerate(off) if abs(r - 1) > 1e-9] == list(range(11, 23)) and 2.25 < off[18] == max(off) < 2.35


def test_frequencies_of_the_callers_own():
    w = [1.0, 0.25, -0.03, 0.0]
    got, factor = ulm_ops.rotary_turns(8, scaling=dict(kind='list', radians=torch.tensor(w, dtype=torch.float64), attention_factor=1.5))
    assert factor == 1.5 and all(abs(float(a) - b) <= 2.0 ** -50 * abs(b) + 2.0 ** -61 for a, b in zip([r if r < math.pi else r - 2 * Fraction(math.pi) for r in radians(got)], w))
    m = ulm_ops.Rotary(8, scaling=dict(kind='list', radians=[10000.0 ** (-i / 4) for i in range(4)]))
    assert torch.equal(m.turns, ulm_ops.rotary_turns(8)[0])


@pytest.mark.parametrize('scaling', [
    dict(kind='list'), dict(kind='list', radians=[1.0, 0.5, 0.1]), dict(kind='list', radians=[1.0, 0.5, 0.1, float('nan')]), dict(kind='list', radians=[1.0, 0.5, 0.1, 0.1], factor=2.0),
    dict(kind='yarn', factor=2.0, original_length=64, ramp='columns'), dict(kind='parts', factor=2.0, original_length=64, slow=0.0, ramp='pairs'), dict(kind='linear', factor=2.0, ramp='pairs')])
def test_refused_lists_and_ramps(scaling):
    with pytest.raises(ValueError):
        ulm_ops.rotary_turns(8, scaling=scaling)


@pytest.mark.parametrize('args', [
    dict(rotary_dim=0), dict(rotary_dim=-2), dict(rotary_dim=7), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, base=float('nan')),
    dict(rotary_dim=8, base=float('inf')), dict(rotary_dim=8, scaling=dict(factor=2.0)), dict(rotary_dim=8, scaling=dict(kind='longer', factor=2.0)),
    dict(rotary_dim=8, scaling=dict(kind='linear')), dict(rotary_dim=8, scaling=dict(kind='linear', factor=-1.0)), dict(rotary_dim=8, scaling=dict(kind='linear', factor=2.0, slow=1.0)),
    dict(rotary_dim=8, scaling=dict(kind='parts', factor=2.0)), dict(rotary_dim=8, scaling=dict(kind='parts', factor=2.0, original_length=64, slow=4.0, fast=4.0)),
    dict(rotary_dim=8, scaling=dict(kind='linear', factor=2.0, attention_factor=-1.0)), dict(rotary_dim=8, scaling=dict(kind='yarn', factor=2.0, original_length=8, attention_factor=0.0)),
    dict(rotary_dim=8, scaling={}), dict(rotary_dim=8, scaling=dict(kind='yarn', factor=1e-9, original_length=8)),
])
def test_refused_frequencies(args):
    with pytest.raises(ValueError):
        ulm_ops.rotary_turns(**args)


def test_the_module_keeps_nothing_in_a_state_dict_and_survives_casts():
    m = ulm_ops.Rotary(64, scaling=dict(kind='linear', factor=2.0))
    assert not m.state_dict() and m.half().turns.dtype == torch.int64
    assert torch.equal(m.turns, ulm_ops.rotary_turns(64, scaling=dict(kind='linear', factor=2.0))[0])


def test_a_module_without_memory_gets_its_frequencies_with_it():
    kw = dict(base=5000.0, scaling=dict(kind='linear', factor=2.0))
    want = ulm_ops.rotary_turns(32, **kw)[0]
    with torch.device('meta'):
        whole = torch.nn.ModuleDict({'inner': ulm_ops.Rotary(32, **kw)})
    assert whole['inner'].to('meta').turns.is_meta
    assert torch.equal(whole.to_empty(device='cpu')['inner'].turns, want)      # as a model around it does
    m = ulm_ops.Rotary(32, **kw)
    assert torch.equal(m.to_empty(device='cpu').turns, want) and torch.equal(m.double().turns, want) and m.turns.dtype == torch.int64
    m.turns = torch.arange(16)                             # frequencies that somebody else has put there move as they are
    assert torch.equal(m.to_empty(device='cpu').turns, torch.arange(16)) and 'turns' not in m.state_dict()


@pytest.mark.parametrize('where', ['cpu', 'meta'])
def test_tensors_elsewhere_are_refused(where):
    x = torch.zeros(1, 2, 3, 8, device=where)
    with pytest.raises(ValueError, match='CUDA'):
        ulm_ops.rotary(x, x, ulm_ops.rotary_turns(8)[0])
    with pytest.raises(ValueError, match='CUDA'):
        ulm_ops.rotary(x, None, ulm_ops.rotary_turns(8)[0])
