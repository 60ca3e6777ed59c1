"""Rotary positions in 64 bits (numpy integers and float64, on the CPU): what include/ulm_b200.h defines."""
import numpy as np
import torch


def angles(positions, turns):
    """Radians of each position and pair: the product modulo 2^64 is a share of a turn.  int64 arrays of any shape and [n]."""
    share = np.asarray(positions, dtype=np.int64).astype(np.uint64)[..., None] * np.asarray(turns, dtype=np.int64).astype(np.uint64)
    return torch.from_numpy(share.astype(np.int64).astype(np.float64) * (2 * np.pi / 2.0 ** 64))     # the same angle between -pi and pi


def rotary(x, positions, turns, interleaved=False, factor=1.0, inverse=False):
    """x [B, H, S, D] of any type, positions [S] or [B, S] -> float64."""
    x = x.detach().double().cpu()
    at = angles(positions, turns)
    at = (at if at.dim() == 3 else at[None])[:, None]
    c, s = at.cos() * factor, at.sin() * (-factor if inverse else factor)
    n = at.shape[-1]
    i = torch.arange(n) * 2 if interleaved else torch.arange(n)
    j = i + 1 if interleaved else i + n
    out = x.clone()
    out[..., i] = x[..., i] * c - x[..., j] * s
    out[..., j] = x[..., j] * c + x[..., i] * s
    return out


def reach(x, n, interleaved=False, factor=1.0):
    """|x_i| + |x_j| of each element's pair times the factor, 0 where an element passes through: what errors of angles are relative to."""
    x = x.detach().double().cpu().abs()
    i = torch.arange(n) * 2 if interleaved else torch.arange(n)
    j = i + 1 if interleaved else i + n
    out = torch.zeros_like(x)
    out[..., i] = out[..., j] = (x[..., i] + x[..., j]) * factor
    return out
