"""The 8-bit form's definition: what it promises of every tensor, and which calls are refused on the host."""
import ctypes as C

import numpy as np
import pytest
import torch

import _native as N
import ulm_ops
from oracle import pack8 as op


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('n', [1, 31, 32, 33, 1000])
def test_what_comes_back_is_near_and_a_number_of_the_type(dtype, n):
    x = (torch.randn(n, generator=torch.Generator().manual_seed(n)) * torch.logspace(-6, 4, n)).to(dtype)
    back = op.through(x)
    assert torch.equal(back.to(dtype).double(), back)
    top = torch.from_numpy(np.repeat(np.abs(np.pad(x.double().numpy(), (0, -n % 32)).reshape(-1, 32)).max(1), 32)[:n])
    off = (back - x.double()).abs()
    assert bool((off <= top / 64).all())
    held = np.abs(op.pack(x)[0]) == 127
    assert bool((off <= top / 128)[~torch.from_numpy(held)].all())


def test_rounding_error_of_normal_values():
    x = torch.randn(1 << 18, generator=torch.Generator().manual_seed(1))
    rms = float((op.through(x) - x.double()).square().mean().sqrt())
    # steps of 2^(e - 6) with 2^e mostly 1 or 2 at 32 values: between 1 / 64 and 1 / 32, an error of a step over sqrt(12)
    assert 1 / 64 / 12 ** 0.5 < rms < 1 / 32 / 12 ** 0.5


def test_ties_and_the_largest_code():
    x = torch.zeros(32)
    x[0], x[1], x[2], x[3], x[4], x[5] = 1.0, 0.5 / 64, 1.5 / 64, 2.5 / 64, -0.5 / 64, -1.5 / 64
    assert list(op.pack(x)[0][:6]) == [64, 0, 2, 2, 0, -2]
    x[0], x[1], x[2] = 1.999, 1.9921875 - 2 ** -9, -1.999
    assert list(op.pack(x)[0][:3]) == [127, 127, -127]


def test_the_same_tensor_again():
    x = torch.randn(5000, generator=torch.Generator().manual_seed(2))
    back = op.through(x)
    again = op.through(back.float())
    assert torch.equal(back, again)                        # no drift: a value that came back stays


@pytest.mark.parametrize('x', [torch.ones(32), torch.ones(32, device='meta'), torch.ones(32, dtype=torch.float64), torch.ones(32, dtype=torch.int32)])
def test_packing_refuses(x):
    with pytest.raises(ValueError):
        ulm_ops.pack_8bit(x)
    with pytest.raises(ValueError):
        ulm_ops.swiglu_8bit(x, x)


def test_projections_refuse_tensors_of_the_host():
    x, w = torch.ones(3, 8), torch.ones(4, 8)
    with pytest.raises(ValueError, match='CUDA'):
        ulm_ops.linear_8bit(x, w)
    with pytest.raises(ValueError, match='CUDA'):
        ulm_ops.feed_forward_8bit(x, w, w, torch.ones(8, 4))


def test_the_library_refuses_before_any_launch():
    lib = N.lib()
    assert lib.ulm_pack8_blocks(0) == 0 and lib.ulm_pack8_blocks(1) == 1 and lib.ulm_pack8_blocks(32) == 1 and lib.ulm_pack8_blocks(33) == 2
    assert lib.ulm_pack8(None, None, None, 8, 7, None) == -1 and b'dtype' in lib.ulm_last_error()
    assert lib.ulm_pack8(None, None, None, -1, 0, None) == -1 and lib.ulm_pack8(None, None, None, 0, 0, None) == 0
    assert lib.ulm_pack8(16, 8, 16, 8, 0, None) == -1 and b'16-byte' in lib.ulm_last_error()
    assert lib.ulm_unpack8(16, None, 16, 8, 0, None) == -1
    assert lib.ulm_pack8(16, 16, 16, 1 << 45, 0, None) == -4
    a = N.Swiglu8Args()
    a.n, a.dtype, a.p = 64, N.ULM_BF16, 2.0
    assert lib.ulm_swiglu8_fwd(C.byref(a)) == -1 and b'between 0 and 1' in lib.ulm_last_error()
    a.p, a.d, a.row_stride = 0.0, 12, 24
    assert lib.ulm_swiglu8_bwd(C.byref(a)) == -1 and b'whole 16-byte vectors' in lib.ulm_last_error()
    a.d = 0
    assert lib.ulm_swiglu8_fwd(C.byref(a)) == -1 and b'codes' in lib.ulm_last_error()
    assert lib.ulm_swiglu8_fwd(None) == -1 and lib.ulm_swiglu8_bwd(None) == -1


def test_struct_sizes_match_the_header():
    assert C.sizeof(N.Swiglu8Args) == 10 * 8 + 3 * 8 + 8 + 8 + 2 * 4 + 8
    assert C.sizeof(N.RotaryArgs) == 6 * 8 + 14 * 8 + 10 * 4 + 2 * 4 + 8
    assert C.sizeof(N.NormAddNormFwdArgs) == 10 * 8 + 6 * 8 + 6 * 4 + 8
    assert C.sizeof(N.NormAddNormBwdArgs) == 17 * 8 + 9 * 8 + 4 * 4 + 8


def test_rotary_and_norms_refuse_before_any_launch():
    lib = N.lib()
    r = N.RotaryArgs()
    r.B, r.Hq, r.Hk, r.S, r.D, r.R, r.dtype = 1, 1, 0, 4, 8, 8, 9
    assert lib.ulm_rotary(C.byref(r)) == -1 and b'dtype' in lib.ulm_last_error()
    r.dtype = N.ULM_F16
    for bad in (0, 3, 10, -2):
        r.R = bad
        assert lib.ulm_rotary(C.byref(r)) == -1 and b'even number' in lib.ulm_last_error()
    r.R = 8
    assert lib.ulm_rotary(C.byref(r)) == -1 and b'null' in lib.ulm_last_error()
    r.q = r.qo = 33                                       # not on a whole element
    r.turns = 64
    assert lib.ulm_rotary(C.byref(r)) == -1 and b'whole elements' in lib.ulm_last_error()
    r.q = r.qo = 64
    r.turns = 68
    assert lib.ulm_rotary(C.byref(r)) == -1 and b'whole elements' in lib.ulm_last_error()
    r.turns, r.pos_kind = 64, 3
    assert lib.ulm_rotary(C.byref(r)) == -1 and b'pos_kind' in lib.ulm_last_error()
    r.pos_kind, r.B, r.S = 0, 1 << 20, 1 << 20
    assert lib.ulm_rotary(C.byref(r)) == -4
    r.S = 0
    assert lib.ulm_rotary(C.byref(r)) == 0 and lib.ulm_rotary(None) == -1
    f = N.NormAddNormFwdArgs()
    f.rows, f.d, f.dtype = 4, 64, N.ULM_F32
    assert lib.ulm_norm_add_norm_fwd(C.byref(f)) == -1 and b'fp16 or bf16' in lib.ulm_last_error()
    f.dtype = N.ULM_F16
    for d, rc in ((0, -1), (6, -1), (8196, -4)):
        f.d = d
        assert lib.ulm_norm_add_norm_fwd(C.byref(f)) == rc
    f.d, f.scale_channels = 64, 1
    assert lib.ulm_norm_add_norm_fwd(C.byref(f)) == -1 and b'a scale a column' in lib.ulm_last_error()
    f.scale_channels = 0
    assert lib.ulm_norm_add_norm_fwd(C.byref(f)) == -1 and b'null' in lib.ulm_last_error()
    f.rows = 0
    assert lib.ulm_norm_add_norm_fwd(C.byref(f)) == 0 and lib.ulm_norm_add_norm_fwd(None) == -1 and lib.ulm_norm_add_norm_bwd(None) == -1
    b = N.NormAddNormBwdArgs()
    b.rows, b.d, b.dtype = 4, 64, N.ULM_F16
    assert lib.ulm_norm_add_norm_bwd(C.byref(b)) == -1 and b'null' in lib.ulm_last_error()
    assert lib.ulm_norm_add_norm_partial(1, 64) == 129 and lib.ulm_norm_add_norm_partial(10 ** 9, 64) == 296 * 129
