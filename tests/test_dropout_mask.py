"""The dropout mask on the CPU: the generator's published answers, the mask's statistics, and the arguments that the ops refuse."""
import ctypes as C

import numpy as np
import pytest
import torch

import _native as N
import ulm_ops
from oracle import dropout as od


@pytest.mark.parametrize('counter,key,want', [
    ([0, 0, 0, 0], (0, 0), [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
    ([0xffffffff] * 4, (0xffffffff, 0xffffffff), [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
    ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], (0xa4093822, 0x299f31d0), [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]),
])
def test_generator_gives_its_published_answers(counter, key, want):
    assert od.philox4x32(np.array([counter], dtype=np.uint64), key).tolist() == [want]


@pytest.mark.parametrize('p', [0.0, 0.1, 0.5, 0.9, 1.0])
def test_share_of_kept_elements(p):
    n = 1 << 20
    keep = od.keep_mask(n, p, 1234567)
    # a binomial's mean, within five deviations (none at 0 and 1)
    assert abs(keep.mean() - (1 - od.threshold(p) / 65536)) <= 5 * (p * (1 - p) / n) ** 0.5
    # neighbours, and masks of neighbouring seeds, agree as often as independent ones do
    other = od.keep_mask(n, p, 1234568)
    same = p * p + (1 - p) * (1 - p)
    for a, b in ((keep[1:], keep[:-1]), (keep, other), (keep[8:], keep[:-8])):
        assert abs((a == b).mean() - same) <= 5 * (0.25 / n) ** 0.5 + 2 ** -15


def test_a_mask_is_a_function_of_place_and_seed():
    whole = od.keep_mask(1000, 0.3, 99)
    for start, n in ((0, 1), (7, 9), (8, 8), (500, 123)):
        assert np.array_equal(od.keep_mask(n, 0.3, 99, start), whole[start:start + n])
    far = 1 << 36                                          # the counter's second word
    assert np.array_equal(od.keep_mask(8, 0.5, 3, far), od.keep_mask(16, 0.5, 3, far - 8)[8:])
    assert not np.array_equal(od.keep_mask(64, 0.5, 3, far), od.keep_mask(64, 0.5, 3))


@pytest.mark.parametrize('p,t', [(0, 0), (1e-9, 1), (0.1, 6554), (0.5, 32768), (1 - 1e-9, 65535), (1, 65536)])
def test_threshold(p, t):
    assert od.threshold(p) == t


def test_seeds():
    assert ulm_ops._as_i64(0) == 0 and ulm_ops._as_i64((1 << 64) - 1) == -1 and ulm_ops._as_i64(-5) == -5
    for bad in (1 << 64, -(1 << 63) - 1):
        with pytest.raises(ValueError):
            ulm_ops._as_i64(bad)
    torch.manual_seed(5)
    a = [ulm_ops.next_dropout_seed() for _ in range(3)]
    torch.manual_seed(5)
    assert a == [ulm_ops.next_dropout_seed() for _ in range(3)] and len(set(a)) == 3


def test_module():
    m = ulm_ops.Dropout(0.3)
    x = torch.ones(3)
    assert m.eval()(x) is x and ulm_ops.Dropout(0.0).train()(x) is x and m.train().active()
    assert 'p=0.3' in repr(m)
    for p in (-0.1, 1.1, float('nan')):
        with pytest.raises(ValueError):
            ulm_ops.Dropout(p)


def test_refusals_come_before_any_launch():
    x = torch.ones(8, 64)
    for call in (lambda: ulm_ops.dropout(x, 0.1, 0), lambda: ulm_ops.swiglu_dropout(x, x, 0.1, 0),
                 lambda: ulm_ops.dropout_add_rms_norm(x, x.half(), torch.ones(64), 0.1, 0)):
        with pytest.raises(ValueError):                    # CPU tensors
            call()
    lib = N.lib()
    for p in (-0.1, 1.5, float('nan')):
        assert lib.ulm_dropout(256, 256, 8, N.ULM_F16, p, 0, None) == -1 and b'between 0 and 1' in lib.ulm_last_error()
    assert lib.ulm_dropout(256, 256, -1, N.ULM_F16, 0.1, 0, None) == -1
    assert lib.ulm_dropout(256, 256, 8, 9, 0.1, 0, None) == -1
    assert lib.ulm_dropout(None, 256, 8, N.ULM_F16, 0.1, 0, None) == -1
    assert lib.ulm_dropout(258, 256, 8, N.ULM_F16, 0.1, 0, None) == -1
    assert lib.ulm_dropout(None, None, 0, N.ULM_F16, 0.1, 0, None) == 0          # nothing to do
    a = N.SwigluArgs()
    a.n, a.dtype = 24, N.ULM_F16
    assert lib.ulm_swiglu_dropout(C.byref(a), 0, 12, 24, 0.1, 0) == -1 and b'vectors' in lib.ulm_last_error()
    assert lib.ulm_swiglu_dropout(C.byref(a), 0, 0, 0, 0.1, 0) == -1
    assert lib.ulm_swiglu_dropout(None, 0, 0, 0, 0.1, 0) == -1
    f = N.RmsFwdArgs()
    f.rows, f.d, f.x_dtype, f.w_dtype, f.y_kind = 4, 64, N.ULM_F32, N.ULM_F32, N.ULM_Y_SAME
    assert lib.ulm_add_dropout_norm_fwd(C.byref(f), 0.1, 0) == -1                # a 16-bit y is needed
    f.y_kind = N.ULM_Y_F16
    assert lib.ulm_add_dropout_norm_fwd(C.byref(f), 0.1, 0) == -1 and b'null' in lib.ulm_last_error()
    f.d = 66
    assert lib.ulm_add_dropout_norm_fwd(C.byref(f), 0.1, 0) == -1
    f.d = 8196
    assert lib.ulm_add_dropout_norm_fwd(C.byref(f), 0.1, 0) < 0 and b'8192' in lib.ulm_last_error()
    f.d, f.rows = 64, 0
    assert lib.ulm_add_dropout_norm_fwd(C.byref(f), 0.1, 0) == 0
    assert lib.ulm_add_dropout_norm_bwd(None, 0.1, 0) == -1
    assert lib.ulm_add_dropout_norm_partial_rows(0) == 1 and lib.ulm_add_dropout_norm_partial_rows(10 ** 9) == 444
