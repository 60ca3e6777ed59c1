"""RMSNorm, the SwiGLU gate, dropout, rotary positions and the cross-entropy on the sm_100a library, as autograd ops.

The reference has no custom kernels for these: ``FusedRMSNorm`` calls
F.rms_norm (train.py:1862-1875), dropout is nn.Dropout and ``compute_loss`` loops fc_out +
F.cross_entropy over row chunks (train.py:2059-2082).  The classes and functions
below keep those names and argument meanings.
"""
import contextlib
import ctypes as C
import math
import typing

import torch
import torch.nn as nn

import _native as N

_DT = {torch.float16: N.ULM_F16, torch.bfloat16: N.ULM_BF16, torch.float32: N.ULM_F32}
_16BIT = (torch.float16, torch.bfloat16)


def _stream(t=None):
    """torch's current stream on the tensor's device (or the current device)."""
    return N.current_stream(t.device.index if t is not None and t.device.index is not None else torch.cuda.current_device())


def rms_norm(x, weight, eps: float = 1e-6, out_dtype=None):
    """``weight * x * rsqrt(mean(x^2, -1) + eps)``; fp32 reduction.  The output has x's dtype,
    except that an fp32 x under CUDA autocast gives the autocast dtype directly: F.rms_norm
    (train.py:1872) would return fp32 there and the Linear that follows would round it to 16 bits,
    so rounding the fp32 result once in the kernel yields the same values and saves the cast pass
    (and, in the backward, the cast of the 16-bit gradient back to fp32).  ``out_dtype`` overrides."""
    return N.ext().rms_norm(x, weight, eps, out_dtype)


def add_rms_norm(x, branch, weight, eps: float = 1e-6):
    """The residual add in front of a norm fused with that norm: ``x_new = x + branch`` (train.py:1989,
    1993) and ``y = rms_norm(x_new)`` (the next norm: train.py:1991, 1988 of the following block, or 2054)
    in one pass over memory; returns ``(x_new, y)``.  x is the fp32 residual stream, branch the 16-bit
    output of the attention or feed-forward projection under autocast; x_new is fp32 and y has branch's
    dtype -- the values the unfused sequence (add in fp32, F.rms_norm in fp32, autocast's cast in front
    of the next Linear) produces.  The backward adds the gradient arriving at x_new to rms_norm's and
    writes the sum once, as the fp32 gradient of x and, rounded, as the 16-bit gradient of branch."""
    return N.ext().add_rms_norm(x, branch, weight, eps)


class FusedRMSNorm(nn.Module):
    """train.py:1862-1875."""

    def __init__(self, d_model: int, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d_model))
        self.eps = eps

    def forward(self, x):
        return rms_norm(x, self.weight, self.eps)

    def add_forward(self, x, branch, dropout_p=0.0, seed=0, post=None, gate=None):
        """(x + branch, norm(x + branch)); the fused kernel when the tensors have the training layout
        (fp32 residual stream, 16-bit branch, d <= 1024), the two separate ops otherwise.  With ``dropout_p`` the branch
        is dropped first, in the fused kernel (d <= 8192) or by `dropout`.  With ``post`` (`BranchNorm`) it is then normalised, multiplied by the
        sigmoid of ``gate`` and by post's scale before it is added: `norm_add_norm` in the training layout (d <= 8192), its separate ops otherwise."""
        if post is not None:
            return self._post_add(x, dropout(branch, dropout_p, seed) if dropout_p else branch, post, gate)
        d = x.shape[-1]
        if (x.is_cuda and x.dtype == torch.float32 and branch.dtype in _16BIT and d <= (8192 if dropout_p else 1024)
                and d % 4 == 0 and torch.is_autocast_enabled('cuda')
                and torch.get_autocast_dtype('cuda') == branch.dtype):
            if dropout_p:
                return dropout_add_rms_norm(x, branch, self.weight, dropout_p, seed, self.eps)
            return add_rms_norm(x, branch, self.weight, self.eps)
        x = x + (dropout(branch, dropout_p, seed) if dropout_p else branch)
        return x, rms_norm(x, self.weight, self.eps)

    def _post_add(self, x, branch, post, gate):
        d = x.shape[-1]
        if (x.is_cuda and x.dtype == torch.float32 and branch.dtype in _16BIT and d <= 8192 and d % 4 == 0 and self.eps == post.eps
                and torch.is_autocast_enabled('cuda') and torch.get_autocast_dtype('cuda') == branch.dtype and (gate is None or gate.dtype == branch.dtype)):
            return norm_add_norm(x, branch, post.weight, self.weight, gate=gate, scale=post.scale, eps=self.eps)
        branch = rms_norm(branch, post.weight, post.eps, branch.dtype).to(x.dtype)
        if gate is not None:
            branch = branch * torch.sigmoid(gate.to(x.dtype))
        x = x + (branch if post.scale is None else branch * post.scale.to(x.dtype))
        return x, rms_norm(x, self.weight, self.eps)


class BranchNorm(nn.Module):
    """What stands behind a block's branch before it is added: a norm's ``weight``, with ``gated`` the projection ``gate`` of the branch's input whose sigmoid
    multiplies it, and a learned ``scale`` that starts at the number given (None: there is none; 0: the branch is off at the start)."""

    def __init__(self, d_model: int, gated=False, scale=None, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d_model))
        self.gate = nn.Linear(d_model, d_model, bias=False) if gated else None
        self.scale = None if scale is None else nn.Parameter(torch.tensor(float(scale)))
        self.eps = eps

    def gate_of(self, x, packed=None):
        """The gate before its sigmoid, of the branch's input; ``packed``: as for `linear_8bit`, which then is the projection."""
        if self.gate is None:
            return None
        return linear(x, self.gate.weight) if packed is None else linear_8bit(x, self.gate.weight, packed)


def swiglu(a, b):
    """``F.silu(a) * b`` (the gate of train.py:1966-1975's feed-forward) in one kernel each way."""
    return N.ext().swiglu(a, b)


# ---------------------------------------------------------------------------
# Dropout with a mask that is never stored
# ---------------------------------------------------------------------------
def dropout(x, p, seed):
    """Inverted dropout of a CUDA fp16/bf16/fp32 tensor: each element is zero with probability ``p`` (in steps of 2^-16) and
    otherwise divided by the share that stays.  Which ones are dropped is a function of ``seed`` (any 64-bit integer) and of the
    element's row-major index alone (`Philox4x32`, include/ulm_b200.h says how), so nothing is kept for the backward: it forms
    the mask again.  The same seed drops the same elements of another tensor of that size; a captured graph replays the masks
    of the seeds it was captured with."""
    return N.ext().dropout(x, float(p), _as_i64(seed))


def swiglu_dropout(a, b, p, seed):
    """``dropout(silu(a) * b)`` in one kernel each way (the reference's feed-forward, train.py:1975); p = 0 is `swiglu`.
    Values stay in fp32 up to the one rounding of the result."""
    return N.ext().swiglu_dropout(a, b, float(p), _as_i64(seed))


def dropout_add_rms_norm(x, branch, weight, p, seed, eps: float = 1e-6):
    """`add_rms_norm` with dropout on the branch: ``x_new = x + dropout(branch)`` and ``y = rms_norm(x_new)`` in one pass
    (train.py:1993 with the norm behind it), returns ``(x_new, y)``.  x and x_new fp32, branch and y 16-bit, rows of at most 8192
    elements, a multiple of 4.  The backward gives the gradients of x, branch and weight in one pass and a column sum."""
    return N.ext().dropout_add_rms_norm(x, branch, weight, float(p), _as_i64(seed), float(eps))


def norm_add_norm(x, branch, post_weight, weight, gate=None, scale=None, eps: float = 1e-6):
    """The norms behind and in front of a block, with the residual add between them, in one pass each way:
    ``x_new = x + scale * sigmoid(gate) * rms_norm(branch, post_weight)`` and ``y = rms_norm(x_new, weight)``; returns ``(x_new, y)``.
    x and x_new fp32 (the residual stream), branch, gate and y of one 16-bit type, rows of at most 8192 elements, a multiple of 4.
    ``gate``: a tensor of branch's shape, before its sigmoid; None: no gate.  ``scale``: None, a number, or a floating tensor on x's device of one
    element or of one per column, which then has a gradient.  Statistics, sums and x_new are fp32, y and the gradients of branch and
    gate are rounded once.  The gradient of a 16-bit weight or scale is the fp32 sum, rounded."""
    if isinstance(scale, torch.Tensor):
        if gate is None:
            return N.ext().norm_add_norm_scale(x, branch, post_weight, weight, scale, float(eps))
        return N.ext().norm_add_norm_gate_scale(x, branch, post_weight, weight, gate, scale, float(eps))
    value = 1.0 if scale is None else float(scale)
    if gate is None:
        return N.ext().norm_add_norm_plain(x, branch, post_weight, weight, value, float(eps))
    return N.ext().norm_add_norm_gate(x, branch, post_weight, weight, gate, value, float(eps))


def _as_i64(seed):
    """The 64 bits of ``seed`` as the signed integer the extension takes."""
    seed = int(seed)
    if not -(1 << 63) <= seed < 1 << 64:
        raise ValueError('a dropout seed is a 64-bit integer')
    return seed - (1 << 64) if seed >= 1 << 63 else seed


def next_dropout_seed():
    """A seed from torch's default CPU generator: `torch.manual_seed` fixes the sequence, and a checkpointed forward that is run
    again draws the same ones.  No device is asked.  Refused while a CUDA graph is captured or a module traced: the seed would be a
    constant of the recording, which would drop the same elements at every run."""
    if torch.jit.is_tracing() or (torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()):
        raise RuntimeError('a captured or traced step would drop the same elements at every run: give ulm_ops.dropout and its like a seed '
                           'of your own where that is meant, or use nn.Dropout there')
    return int(torch.randint(0, 1 << 62, (), device='cpu'))         # whatever torch's default device is


class Dropout(nn.Module):
    """`nn.Dropout` on `dropout`, for CUDA fp16/bf16/fp32 tensors: the same ``p`` and the same training switch, no stored mask, a
    mask of its own per call.  Where nn.Dropout would draw anew at each replay of a captured graph, this one, at work, refuses
    the capture (`next_dropout_seed`)."""

    def __init__(self, p: float = 0.5):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f'dropout probability has to be between 0 and 1, but got {p}')
        self.p = p

    def active(self):
        return self.training and self.p > 0.0

    def forward(self, x):
        return dropout(x, self.p, next_dropout_seed()) if self.active() else x

    def extra_repr(self):
        return f'p={self.p}'


# ---------------------------------------------------------------------------
# Rotary positions of any width, pairing and frequency
# ---------------------------------------------------------------------------
def rotary_turns(rotary_dim, base=10000.0, scaling=None, device=None):
    """``(turns, factor)`` for `rotary`: how far each of the rotary_dim / 2 pairs turns per position, as an int64 tensor of 2^-64 turns,
    and what the turned vectors are multiplied by.  Pair i turns by w_i = base^(-2i / rotary_dim) radians; ``scaling`` stretches that:

      None                              as it is
      dict(kind='linear', factor=f)     w_i / f: positions f times closer together
      dict(kind='ntk', factor=f)        base * f^(rotary_dim / (rotary_dim - 2)): the slowest pair f times slower, the fastest as it is
      dict(kind='parts', factor=f, original_length=L, slow=a, fast=b)
                                        pairs that turn at least b times within L positions stay, those that turn at most a times
                                        are f times slower, those between in proportion
      dict(kind='yarn', ...)            'parts' (a = 1, b = 32 by default), and q and k multiplied by 0.1 ln f + 1 each (Peng, Quesnelle, Fan
                                        and Shippole, "YaRN: efficient context window extension of large language models", 2023)
      dict(kind='list', radians=w)      the w_i themselves, one of any sign for each pair (``base`` then does not count)

    With 'parts' and 'yarn' "in proportion" is to the number of turns, as in the paper.  Released checkpoints are mostly trained
    with ``ramp='pairs'``: in proportion to the pair's number i, from the pair that turns b times within L positions (a whole number, rounded down) to the
    one that turns a times (rounded up).  The two differ by up to a factor of two and more between the borders, and nothing in a
    checkpoint's weights tells them apart: its configuration has to.

    ``attention_factor=`` beside any of them replaces the multiplier.  Computed on the host in 64 bits."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f'rotary_dim has to be a positive even number, but got {rotary_dim}')
    if not base > 1.0 or not math.isfinite(base):
        raise ValueError(f'base has to be a finite number above 1, but got {base}')
    spec = dict(scaling or {})
    kind = spec.pop('kind', None)
    if scaling is not None and kind not in ('linear', 'ntk', 'parts', 'yarn', 'list'):
        raise ValueError(f"scaling is one of kind 'linear', 'ntk', 'parts', 'yarn' and 'list', but got {scaling}")
    multiplier = spec.pop('attention_factor', None)
    w = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if kind == 'list':
        w = [float(x) for x in spec.pop('radians', ())]
        if len(w) != rotary_dim // 2 or not all(math.isfinite(x) for x in w):
            raise ValueError(f'a list has a finite number of radians for each of the {rotary_dim // 2} pairs, but got {scaling}')
    elif kind is not None:
        f = float(spec.pop('factor', 0.0))
        if not f > 0.0 or not math.isfinite(f):
            raise ValueError(f'scaling needs a positive factor, but got {scaling}')
        if kind == 'linear':
            w = [x / f for x in w]
        elif kind == 'ntk':
            if rotary_dim > 2:
                w = [(base * f ** (rotary_dim / (rotary_dim - 2.0))) ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
        else:
            length, slow, fast = (float(spec.pop(n, d)) for n, d in (('original_length', 0.0), ('slow', 1.0), ('fast', 32.0)))
            if not length > 0.0 or not fast > slow:
                raise ValueError(f"scaling of kind '{kind}' needs an original_length and slow < fast, but got {scaling}")
            ramp = spec.pop('ramp', 'turns')
            if ramp == 'turns':
                keep = [min(1.0, max(0.0, (length * x / (2.0 * math.pi) - slow) / (fast - slow))) for x in w]
            elif ramp == 'pairs' and slow > 0.0:
                pair = lambda turns: rotary_dim * math.log(length / (2.0 * math.pi * turns)) / (2.0 * math.log(base))      # noqa: E731
                first, last = max(math.floor(pair(fast)), 0), math.ceil(pair(slow))
                keep = [1.0 if i <= first else max(0.0, (last - i) / (last - first)) if i < last else 0.0 for i in range(len(w))]
            else:
                raise ValueError(f"ramp is 'turns', or 'pairs' with a positive slow, but got {scaling}")
            w = [x * k + x / f * (1.0 - k) for x, k in zip(w, keep)]
            if kind == 'yarn' and multiplier is None:
                multiplier = 0.1 * math.log(f) + 1.0
    if spec:
        raise ValueError(f'scaling does not know {sorted(spec)}')
    multiplier = 1.0 if multiplier is None else float(multiplier)
    if not multiplier > 0.0 or not math.isfinite(multiplier):
        raise ValueError(f'the attention factor has to be a positive number, but got {multiplier}')
    # w / 2 pi of 2^64, as a signed number of the same bits: off by w's own roundings, a few 2^-53 of itself, and half of the last bit
    turns = [round(math.ldexp(x / (2.0 * math.pi), 64)) % (1 << 64) for x in w]
    return torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64, device=device), multiplier


def rotary(q, k, turns, positions=None, interleaved=False, factor=1.0, inverse=False):
    """The first columns of each head, turned by an angle that grows with the position: q (B,Hq,S,D) and k (B,Hk,S,D), fp16, bf16 or fp32
    views of any stride, of one type -> both turned, in the memory order they came in; ``k`` may be None (None comes back).
    ``turns`` (`rotary_turns`) has one number for each pair of columns: i with i + len(turns), or with ``interleaved`` 2i with 2i + 1;
    columns beyond 2 len(turns) pass through.  ``positions``: int32 or int64 [S] or [B, S] (packed sequences, single tokens of a cached
    context; negative ones turn the other way), 0, 1, 2, .. without.  The angle is positions * turns as a 64-bit fraction of a turn at any
    distance, so that what it is off by is what turns are (a few 2^-53 of themselves from `rotary_turns`); fp32 sine, cosine and products, one rounding.  ``inverse`` turns the other way (times the same ``factor``), which is also the gradient."""
    if k is None:
        return N.ext().rotary_one(q, turns, positions, bool(interleaved), float(factor), bool(inverse)), None
    return N.ext().rotary(q, k, turns, positions, bool(interleaved), float(factor), bool(inverse))


class Rotary(nn.Module):
    """`rotary` with the frequencies of `rotary_turns`, which are no parameters and not part of a state dict: a buffer that moves with the
    module, and is made anew where a module built on the meta device gets memory."""

    def __init__(self, rotary_dim, base=10000.0, interleaved=False, scaling=None):
        super().__init__()
        self.rotary_dim, self.base, self.interleaved, self.scaling = rotary_dim, base, interleaved, scaling
        turns, self.factor = rotary_turns(rotary_dim, base, scaling)
        self.register_buffer('turns', turns, persistent=False)

    def _apply(self, fn, recurse=True):
        # where fn would have the frequencies is asked with none of them, as to_empty would leave memory of any content, and nothing loads over it
        turns = self._buffers.pop('turns')
        try:
            super()._apply(fn, recurse)
            device = fn(turns[:0]).device
            if device != turns.device:
                turns = rotary_turns(self.rotary_dim, self.base, self.scaling, device)[0] if turns.is_meta else turns.to(device)
        finally:
            self._buffers['turns'] = turns
        return self

    def forward(self, q, k, positions=None):
        return rotary(q, k, self.turns, positions, self.interleaved, self.factor)

    def extra_repr(self):
        return f'{self.rotary_dim}, base={self.base}, interleaved={self.interleaved}, scaling={self.scaling}'


# ---------------------------------------------------------------------------
# Bias-free linear layers with the weight gradient accumulated where it lives
# ---------------------------------------------------------------------------
@contextlib.contextmanager
def wgrad_in_place(enabled=True):
    """While active, `linear` and `chunked_cross_entropy` add their weight gradients straight into an
    existing fp32 ``weight.grad`` with one GEMM (16-bit operands, fp32 accumulation and output, beta = 1)
    instead of returning a 16-bit product that autograd casts and adds in two more passes per parameter
    and micro-batch.  The caller owns the gradient buffers (they must exist, be zeroed per step, and no
    post-accumulate hook may be waiting for these parameters): `ulm_dp.DataParallelStep` does.  It holds for the
    calling thread and the backward passes it starts inside."""
    token = N.ext().enter_wgrad_in_place(bool(enabled)) if N.have_ext() else None
    try:
        yield
    finally:
        if token is not None:
            token.leave()


@contextlib.contextmanager
def weight_cast_scope(copies=None):
    """While active in the calling thread, `linear` keeps the 16-bit copy it makes of a weight and reuses it: the caller promises
    that the weights do not change inside the scope (one optimiser step's forward/backward calls).  Nothing
    is reused across scopes or outside one -- a parameter's version counter cannot be relied on for that
    (fused optimisers update parameters without bumping it).  ``copies``: a `weight_copies` object, which is
    refreshed here; without it each weight is cast on first use."""
    if copies is not None:
        copies.refresh()
    token = N.ext().enter_casts(copies) if N.have_ext() else None
    try:
        yield
    finally:
        if token is not None:
            token.leave()


def weight_copies(weights, dtype):
    """One buffer for the 16-bit copies of ``weights`` (fp32 CUDA parameters), kept by the caller and filled by one fused
    cast each time a `weight_cast_scope` opens with it; weights that follow one another in the list do so in the
    buffer, so that `gated_linear` runs its two projections as one GEMM.  Holds 2 bytes per weight element."""
    return N.ext().WeightCopies(list(weights), dtype)


def linear_copies(model, dtype):
    """`weight_copies` of the fp32 CUDA weights of ``model``'s linear layers (each once); None if there are none."""
    ws = {id(m.weight): m.weight for m in model.modules() if isinstance(m, nn.Linear)}
    ws = [w for w in ws.values() if w.is_cuda and w.dtype == torch.float32]
    return weight_copies(ws, dtype) if ws and dtype in _16BIT else None


def gated_linear(x, w1, w3, dropout_p=0.0, seed=0):
    """``swiglu(linear(x, w1), linear(x, w3))`` (train.py:1975) as one op: both projections write the halves of one
    [rows, 2 d_ff] matrix, which the gate's kernels read and differentiate in place of two.  ``dropout_p``, ``seed``: with the
    gate of `swiglu_dropout`."""
    if dropout_p:
        return N.ext().gated_linear_dropout(x, w1, w3, float(dropout_p), _as_i64(seed))
    return N.ext().gated_linear(x, w1, w3)


def linear(x, weight):
    """``x @ weight.T`` for the model's bias-free projections (train.py:1925-1926, 1969-1971) in the autocast
    dtype; see `wgrad_in_place` for what it does differently from ``nn.Linear`` in the backward.  On the CPU it needs no
    build of the library."""
    if not x.is_cuda and not N.have_ext():
        return nn.functional.linear(x, weight.to(x.dtype))
    return N.ext().linear(x, weight)


# ---------------------------------------------------------------------------
# Activations kept in 8 bits between forward and backward
# ---------------------------------------------------------------------------
class Packed8(typing.NamedTuple):
    """A tensor in 8 bits (`pack_8bit`): ``codes`` int8 of its shape, ``exponents`` uint8, one for every 32 elements of its row-major order,
    and the type it had.  33/32 bytes an element."""
    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype


def pack_8bit(x):
    """A CUDA fp16/bf16/fp32 tensor in 8 bits: of every 32 consecutive elements the exponent e of the largest magnitude (at least -120) and
    for each the integer nearest x / 2^(e - 6), ties to even, held to +-127.  What comes back (`unpack_8bit`) is off by at most 1/128 of the
    block's largest magnitude (1/64 where 127 holds it), and is a number of x's own type; its rms error is 0.7 % of normally distributed values.  A
    block with an infinity or a NaN comes back as NaN, so that a loss scaler sees it.  No gradient."""
    return Packed8(*N.ext().pack_8bit(x), x.dtype)


def unpack_8bit(packed, dtype=None):
    """The values that `pack_8bit` kept, in the type they had, or rounded to ``dtype``."""
    return N.ext().unpack_8bit(packed.codes, packed.exponents, packed.dtype if dtype is None else dtype)


def swiglu_8bit(a, b, p=0.0, seed=0):
    """`swiglu_dropout` (p = 0: without dropout), whose backward has a and b in 8 bits alone (`pack_8bit`): a graph keeps 2 1/16 bytes an
    element in place of two tensors.  The result is that of the operands themselves, rounded once; the gradients are those at
    the 8-bit operands."""
    return N.ext().swiglu_8bit(a, b, float(p), _as_i64(seed))


def linear_8bit(x, weight, packed=None):
    """`linear`, whose backward has its input in 8 bits alone (`pack_8bit`; nothing of it where the weight takes no gradient): the
    result and x's gradient are those of `linear`, the weight's is that of the 8-bit input.  CUDA only.  ``packed``: `pack_8bit` of x in the type of
    the product (autocast's, or x's own), for several projections of one x to keep it once between them; without it each packs its own."""
    return N.ext().linear_8bit(x, weight, *(packed or (None, None, None)))


def feed_forward_8bit(x, w1, w3, w2, dropout_p=0.0, seed=0, packed=None):
    """``linear(gated_linear(x, w1, w3, dropout_p, seed), w2)`` (train.py:1975) as one op that keeps x and the two projections in 8 bits and nothing
    else: d + 2 d_ff bytes a token (and 1/32 of that) where the ops by themselves keep 2 d + 6 d_ff.  The backward forms the gate's result
    again from the 8-bit projections, for w2's gradient.  The gate is `swiglu_8bit`'s, the products `linear`'s.  ``packed``: x as for
    `linear_8bit`.  CUDA only."""
    return N.ext().feed_forward_8bit(x, w1, w3, w2, float(dropout_p), _as_i64(seed), *(packed or (None, None, None)))


def ce_rows_forward(logits, target, ignore_index):
    """One logits tile [rows, V] -> (lse[rows], loss[rows]) in fp32."""
    lib = N.lib()
    rows, V = logits.shape
    lse = torch.empty((rows,), dtype=torch.float32, device=logits.device)
    loss = torch.empty((rows,), dtype=torch.float32, device=logits.device)
    a = N.CeFwdArgs(logits.data_ptr(), target.data_ptr(), lse.data_ptr(), loss.data_ptr(),
                    logits.stride(0), rows, V, _DT[logits.dtype], int(ignore_index), _stream())
    N.check(lib.ulm_ce_fwd(C.byref(a)), 'cross-entropy forward')
    return lse, loss


def lm_head_lse(hidden, weight, target=None, ignore_index=0, keep_logits=True):
    """The lm-head GEMM with the loss statistics taken in its epilogue (one tcgen05 kernel + a per-row
    finishing kernel): hidden [rows, d] and weight [V, d], both fp16 or both bf16 ->
    (lse [rows] fp32, loss [rows] fp32 or None, logits [rows, V] in the operands' dtype or None).
    With ``keep_logits`` the rounded logits are stored (the backward turns them into their gradient) and the
    per-row loss lse - z[target] is returned; without, only lse."""
    return N.ext().lm_head_lse(hidden, weight, target, int(ignore_index), bool(keep_logits))


def lm_head_score(hidden, weight, target, ignore_index=-100):
    """`lm_head_lse` for scoring: the per-row loss lse - z[target] (fp32, 0 on ignored rows) and whether the target has
    the row's largest logit (uint8; the lowest column counts on ties, as in ``argmax``).  The logits are never stored:
    the epilogue picks the target's and the largest out of the accumulator."""
    return N.ext().lm_head_score(hidden, weight, target, int(ignore_index))


def ce_rows_backward_(logits, target, lse, gscale_dev, ignore_index, gscale=1.0):
    """In place: logits <- (softmax - onehot) * gscale * gscale_dev[0] (0 on ignored rows)."""
    lib = N.lib()
    rows, V = logits.shape
    a = N.CeBwdArgs(logits.data_ptr(), target.data_ptr(), lse.data_ptr(),
                    gscale_dev.data_ptr() if gscale_dev is not None else None, float(gscale),
                    logits.stride(0), rows, V, _DT[logits.dtype], int(ignore_index), _stream())
    N.check(lib.ulm_ce_bwd(C.byref(a)), 'cross-entropy backward')
    return logits


# Largest [rows, V] 16-bit logits buffer the cross-entropy keeps between forward and backward.  Up to this size
# (2.1 GB for the 32768-row token budget at V = 32000: small change on a 180 GB part) the backward turns the
# kept logits into their gradient in place and runs ONE GEMM each for dH and dW over all rows; beyond it the
# loss falls back to the reference's chunk-by-chunk form, recomputing each chunk's logits in the backward.
KEEP_LOGITS_BYTES = 8 << 30

# The kept form takes its logits and their log-sum-exp from ONE kernel (`lm_head_lse`: tcgen05 GEMM with the
# statistics in its epilogue) where the shapes allow (d and V multiples of 64), instead of a library GEMM
# followed by a pass over the logits.  Measured at 32768 x 32000 x 768 in bf16 on B200: 1.44 ms against
# 1.25 + 0.45 ms, identical logits bits.
FUSED_LM_HEAD = True


class _ChunkedCE(torch.autograd.Function):
    """The chunk-by-chunk form of the loss below, for logits beyond KEEP_LOGITS_BYTES: one [chunk_rows, V] tile at a
    time; the forward keeps one fp32 lse per row and the backward recomputes each tile with the lm-head GEMM."""

    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, chunk_rows, compute_dtype, denominator):
        rows = hidden.shape[0]
        wc = N.ext().cast_cached(weight, compute_dtype)
        if denominator is None:
            n_tokens = (target != ignore_index).sum().clamp(min=1).float()
        elif torch.is_tensor(denominator):
            n_tokens = denominator.to(device=hidden.device, dtype=torch.float32)
        else:
            # a host number stays a host number: turning it into a device tensor is a pageable host-to-device
            # copy, which makes the launching thread wait for the GPU (measured: 4.6 ms per micro-batch)
            n_tokens = float(denominator)
        lse_all = torch.empty((rows,), dtype=torch.float32, device=hidden.device)
        total = torch.zeros((), dtype=torch.float32, device=hidden.device)
        for i in range(0, rows, chunk_rows):
            tile = hidden[i:i + chunk_rows].to(compute_dtype) @ wc.t()
            lse, loss = ce_rows_forward(tile, target[i:i + chunk_rows], ignore_index)
            lse_all[i:i + chunk_rows] = lse
            total = total + loss.sum()
        ctx.save_for_backward(hidden, weight, target, lse_all, *([n_tokens] if torch.is_tensor(n_tokens) else []))
        ctx.n_tokens = None if torch.is_tensor(n_tokens) else n_tokens
        ctx.ignore_index, ctx.chunk_rows, ctx.compute_dtype = ignore_index, chunk_rows, compute_dtype
        return total / n_tokens

    @staticmethod
    def backward(ctx, gout):
        hidden, weight, target, lse_all, *rest = ctx.saved_tensors
        n_tokens = ctx.n_tokens if ctx.n_tokens is not None else rest[0]
        cd = ctx.compute_dtype
        wc = N.ext().cast_cached(weight, cd)
        g = (gout.float() / n_tokens).reshape(1)
        dh = torch.empty_like(hidden)
        dw = None
        for i in range(0, hidden.shape[0], ctx.chunk_rows):
            hc = hidden[i:i + ctx.chunk_rows].to(cd)
            dl = ce_rows_backward_(hc @ wc.t(), target[i:i + ctx.chunk_rows],
                                   lse_all[i:i + ctx.chunk_rows], g, ctx.ignore_index)
            dh[i:i + ctx.chunk_rows] = dl @ wc
            part = N.ext().weight_grad(weight, dl, hc)     # None: already added into weight.grad
            if part is not None:
                dw = part.float() if dw is None else dw.add_(part)
        return dh, (None if dw is None else dw.to(weight.dtype)), None, None, None, None, None


def _loss_dtype(hidden):
    """The 16-bit type the loss computes in where none is given."""
    return torch.get_autocast_dtype('cuda') if torch.is_autocast_enabled() else (hidden.dtype if hidden.dtype in _16BIT else torch.bfloat16)


def _divided(loss_over, denominator, hidden):
    """``loss_over(device scalar or None, host number)`` for any denominator: none, a number, a tensor of any shape."""
    dev = denominator.detach() if torch.is_tensor(denominator) else None
    host, shaped = 0.0, dev is not None and dev.dim() > 0
    if dev is None and denominator is not None:
        host = float(denominator)
        if not host > 0.0:                                # the kernel counts then; a division by this number was asked for
            dev = torch.full((), host, dtype=torch.float32, device=hidden.device)
    elif shaped:                                          # one sum, divided as the tensor's shape says
        dev, host = None, 1.0
    loss = loss_over(dev, host)
    return loss / denominator.detach().to(device=hidden.device, dtype=torch.float32) if shaped else loss


def chunked_cross_entropy(hidden, weight, target, ignore_index=0, chunk_rows=2048,
                          compute_dtype=None, denominator=None):
    """hidden [rows, d], weight [V, d] (the tied lm head), target int64 [rows]
    -> CE summed over targets != ignore_index and divided by their count
    (train.py:2069-2082), or by ``denominator`` (a number or a tensor) when one is given.

    The reference loops fc_out + F.cross_entropy over row chunks so that no fp32 [rows, V] tensor is ever alive
    (autograd still keeps each chunk's fp32 log-softmax).  Here only 16-bit logits ever exist.  Two forms, same values:
      kept     logits of all rows are produced by one lm-head GEMM into one 16-bit buffer and kept; the
               backward rewrites them in place as (softmax - onehot) * g and runs one GEMM for dH and one
               for dW (no recomputation);
      chunked  one tile of rows at a time with recomputation (`_ChunkedCE`; buffers beyond KEEP_LOGITS_BYTES)."""
    if compute_dtype is None:
        compute_dtype = _loss_dtype(hidden)
    if hidden.shape[0] == 0:
        return torch.zeros((), device=hidden.device, requires_grad=True)
    target = target.contiguous()
    if hidden.shape[0] * weight.shape[0] * 2 <= KEEP_LOGITS_BYTES:
        return _divided(lambda dev, host: N.ext().kept_cross_entropy(hidden, weight, target, int(ignore_index), compute_dtype, dev, host, FUSED_LM_HEAD),
                        denominator, hidden)
    N.ext().check_target(hidden, target)
    return _ChunkedCE.apply(hidden, weight, target, int(ignore_index), int(chunk_rows), compute_dtype, denominator)


# Bytes that the backward of `streamed_cross_entropy` takes for the 16-bit softmax of one piece of the vocabulary (a piece has
# at least 256 columns, so 512 bytes a row where that is more).  Not all it takes: see there.
# At 32768 rows this is 16384 columns, two pieces of a vocabulary of 32000: 5.50 ms forward and backward against 5.67 with half
# of it, 6.15 with a quarter and 5.48 in one piece (fewer passes over dh's fp32 sum, fewer launches).
PIECE_BYTES = 1 << 30


def streamed_cross_entropy(hidden, weight, target, ignore_index=0, compute_dtype=None, denominator=None):
    """`chunked_cross_entropy` without logits: hidden [rows, d], weight [V, d], target int64 [rows] -> the mean cross-entropy over the
    targets that are not ``ignore_index`` (or the sum over ``denominator``), for any number of rows and vocabulary columns and a
    width that is a multiple of 8.  The forward keeps one fp32 log-sum-exp per row; the backward forms the logits again, one piece
    of the vocabulary at a time.  The logits are never rounded to 16 bits, so the loss is the fp32 loss of the 16-bit operands.

    Gradients: softmax - onehot is rounded once to the compute type, because the tensor cores multiply 16-bit numbers; the products'
    sums are fp32.  hidden's gradient is rounded to the compute type (and widened for an fp32 hidden), a 16-bit weight's to its own;
    an fp32 weight's is the fp32 sum of those rounded terms, under `wgrad_in_place` added into its ``grad``.  That is 2e-3 of a
    gradient in bf16 and 2.6e-4 in fp16 (2-norm against 64 bits; fp32 arithmetic throughout, rounded at the end: 1.7e-3 and 2.1e-4), up to
    4e-3 in bf16 with one to four rows, where one rounded number scales most of a gradient.

    The backward's memory beside the gradients: PIECE_BYTES for the softmax of a piece (512 bytes a row if that is more), 4 rows d
    bytes for hidden's fp32 sum where there is more than one piece, and 256 KB for each part of an output tile that is cut to fill
    the SMs (290 parts at 32768 x 768 x 32000; `ulm_streamed_ce_slots` tells how many).

    Against the kept form: a quarter more arithmetic, none of its 2 rows V bytes between forward and backward, and the backward
    may run more than once (but has no second derivative)."""
    if compute_dtype is None:
        compute_dtype = _loss_dtype(hidden)
    if hidden.shape[0] == 0:
        return torch.zeros((), device=hidden.device, requires_grad=True)
    target = target.contiguous()

    def loss_over(dev, host):
        return N.ext().streamed_cross_entropy(hidden, weight, target, int(ignore_index), compute_dtype, dev, host, int(PIECE_BYTES))
    return loss_over(None, 0.0) if denominator is None else _divided(loss_over, denominator, hidden)


def token_targets(ids, labels, padded, ignore_index):
    """The [n, L] ``ids`` as ``padded`` flat rows (0 past the end) and the label each row predicts: the next token of
    its sequence, ``ignore_index`` at a sequence's last position and on the padding rows."""
    out = N.ext().token_targets(ids, labels, padded, int(ignore_index))
    if out is not None:
        return out
    # other integer types, other devices, labels that broadcast: plain torch, whose errors come before any launch
    if labels.is_floating_point():
        raise ValueError('token_targets takes integer labels')
    n, L = ids.shape
    flat = ids.reshape(-1)
    if padded > n * L:
        flat = torch.cat([flat, flat.new_zeros(padded - n * L)])
    target = labels.new_full((padded,), ignore_index, dtype=torch.long)
    target[:n * L].view(n, L)[:, :-1] = labels[:, 1:]
    return flat, target


def grad_clip_(flat_grad, sumsq, max_norm):
    """clip_grad_norm_ on the flat gradients, given their squared norm on the device: scales them by
    min(1, max_norm / (norm + 1e-6)) and returns the norm; no pass over memory when nothing is to be clipped."""
    return N.ext().grad_clip(flat_grad, sumsq, float(max_norm))


_SUMSQ_SCRATCH = {}     # device index -> fp32 scratch for the per-CTA partial sums


def grad_unscale_sumsq_(flat_grad, inv_scale, out2):
    """flat fp32 grads *= inv_scale[0]; out2[0] += sum(g^2); out2[1] = 1 on inf/nan.
    The sum is formed in a fixed order (per-CTA partials, then one CTA), so it is
    bit-identical from call to call on the same values."""
    lib = N.lib()
    scratch = _SUMSQ_SCRATCH.get(flat_grad.device.index)
    if scratch is None:
        scratch = _SUMSQ_SCRATCH[flat_grad.device.index] = torch.empty(
            int(lib.ulm_grad_sumsq_partial_count()), dtype=torch.float32, device=flat_grad.device)
    N.check(lib.ulm_grad_unscale_sumsq(flat_grad.data_ptr(), flat_grad.numel(),
                                       inv_scale.data_ptr() if inv_scale is not None else None,
                                       out2.data_ptr(), scratch.data_ptr(), _stream()), 'grad_unscale_sumsq')
    return out2
