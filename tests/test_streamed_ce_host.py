"""The loss without logits, as far as it goes on the CPU: sizes of its buffers, refusals before any launch."""
import ctypes as C

import pytest
import torch

import _native as N
import ulm_ops


def args(**kw):
    a = N.StreamedCeArgs()
    a.h = a.w = a.target = a.lse = a.loss = a.scratch = a.mean = a.inv = 256
    a.rows, a.V, a.d, a.h_stride, a.w_stride, a.dtype = 128, 1000, 64, 64, 64, N.ULM_BF16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def grads(**kw):
    g = N.StreamedCeGrads()
    g.factor_dev = g.dh = g.dw = g.workspace = g.slots = g.dh_sum = 256
    g.dw_stride, g.piece = 64, 256
    for k, v in kw.items():
        setattr(g, k, v)
    return g


@pytest.mark.parametrize('bad,word', [(dict(dtype=N.ULM_F32), b'dtype'), (dict(d=12), b'multiple of 8'), (dict(d=0), b'multiple of 8'), (dict(V=0), b'V > 0'),
                                      (dict(rows=-1), b'rows'), (dict(h=None), b'null'), (dict(target=None), b'null'), (dict(rows=1 << 31), b'too many')])
def test_bad_operands(bad, word):
    lib = N.lib()
    assert lib.ulm_streamed_ce_fwd(C.byref(args(**bad))) < 0 and word in lib.ulm_last_error()
    assert lib.ulm_streamed_ce_bwd(C.byref(args(**bad)), C.byref(grads())) < 0 and word in lib.ulm_last_error()


@pytest.mark.parametrize('bad,word', [(dict(piece=0), b'piece'), (dict(piece=300), b'piece'), (dict(factor_dev=None), b'null'), (dict(workspace=None), b'null'),
                                      (dict(dh_sum=None), b'null'), (dict(slots=None), b'slots'), (dict(dw_stride=56), b'aligned'), (dict(dw_stride=68), b'aligned'),
                                      (dict(dh=264), b'aligned'), (dict(dw_add=1), b'fp32')])
def test_bad_gradients(bad, word):
    lib = N.lib()
    assert lib.ulm_streamed_ce_bwd(C.byref(args(rows=4096)), C.byref(grads(**bad))) == -1 and word in lib.ulm_last_error()


def test_nothing_to_do():
    lib = N.lib()
    assert lib.ulm_streamed_ce_fwd(C.byref(args(rows=0, h=None))) == 0
    assert lib.ulm_streamed_ce_bwd(C.byref(args(rows=0)), C.byref(grads())) == 0
    assert lib.ulm_streamed_ce_bwd(C.byref(args()), C.byref(grads(dh=None, dw=None))) == 0
    assert lib.ulm_streamed_ce_fwd(None) == -1 and lib.ulm_streamed_ce_bwd(None, None) == -1 and lib.ulm_streamed_ce_bwd(C.byref(args()), None) == -1
    loss = ulm_ops.streamed_cross_entropy(torch.zeros(0, 64), torch.zeros(10, 64), torch.zeros(0, dtype=torch.long))
    assert float(loss) == 0


def test_buffer_sizes():
    lib = N.lib()
    assert lib.ulm_streamed_ce_scratch(0, 10, 8) == 0 and lib.ulm_streamed_ce_slots(0, 10, 8, 256, 1, 1) == 0
    # whole 64-column blocks of a piece, and of a vocabulary below one
    assert lib.ulm_streamed_ce_workspace(10, 1000, 256) == 10 * 256 and lib.ulm_streamed_ce_workspace(10, 100, 256) == 10 * 128
    # one pair of statistics per column half, at least one group and at most one per 256 columns; a counter
    for rows, V in ((1, 1), (128, 32000), (32768, 32000), (3, 50021)):
        n = lib.ulm_streamed_ce_scratch(rows, V, 768)
        assert 4 * rows < n <= 4 * rows * -(-V // 256) + 1
    # a single row: dh's few tiles are cut along the vocabulary; slots hold 128 x 256 fp32 tiles
    n = lib.ulm_streamed_ce_slots(1, 32000, 768, 32000, 1, 0)
    assert n > 0 and n % (128 * 256) == 0 and n // (128 * 256) <= 148 * 3


@pytest.mark.parametrize('bad', ['cpu tensors', 'one dimension'])
def test_python_refusals(bad):
    h = torch.zeros(4, 64) if bad == 'cpu tensors' else torch.zeros(64)
    with pytest.raises(ValueError):
        ulm_ops.streamed_cross_entropy(h, torch.zeros(10, 64), torch.zeros(h.shape[0], dtype=torch.long))


def test_struct_sizes():
    assert C.sizeof(N.StreamedCeArgs) == 9 * 8 + 8 + 2 * 8 + 8 + 4 * 4 + 8 + 2 * 8
    assert C.sizeof(N.StreamedCeGrads) == 4 * 8 + 8 + 2 * 4 + 3 * 8 + 8
