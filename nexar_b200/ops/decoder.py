"""Operators of a decoder block besides softmax attention: rotary positions,
counter-based dropout and attention with a decay per head.

Every function calls the sm_100a kernels on the current stream of its input's
GPU and allocates its outputs and workspaces there, so calls can be captured
into CUDA graphs and run on any stream or device. (As for every operator of torch, a
backward pass is captured only when no eager graph of the same leaves is alive.)
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch

from .. import _native


# ---------------------------------------------------------------- rotary positions
@dataclass(frozen=True)
class RotaryScaling:
    """How frequencies are stretched for contexts ``factor`` times longer than
    the ``original_length`` a model was trained on.

    ``linear``  every frequency divided by ``factor``;
    ``ntk``     the base raised to base * factor^(dim / (dim - 2)), so the
                fastest pair keeps its frequency and the slowest is divided by ``factor``;
    ``bands``   pairs that turn more than ``high`` times in the original length
                keep their frequency, those below ``low`` turns are divided by
                ``factor``, linear in the turns between;
    ``yarn``    the same idea with a ramp over the pair's index between
                ``fast`` and ``slow`` turns, and cosine and sine times
                ``magnitude`` (default 0.1 ln(factor) + 1).
    """
    kind: str
    factor: float
    original_length: int = 2048
    low: float = 1.0
    high: float = 4.0
    fast: float = 32.0
    slow: float = 1.0
    magnitude: Optional[float] = None

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "bands", "yarn"):
            raise ValueError(f"unknown rotary scaling {self.kind!r} (linear, ntk, bands, yarn)")
        if not (self.factor >= 1.0 and math.isfinite(self.factor)) or self.original_length < 1:
            raise ValueError("rotary scaling needs a finite factor >= 1 and an original length >= 1")
        if not (0 < self.low < self.high) or not (0 < self.slow < self.fast):
            raise ValueError("rotary scaling needs 0 < low < high and 0 < slow < fast")


def rotary_frequencies(dim: int, base: float = 10000.0,
                       scaling: Optional[RotaryScaling] = None) -> Tuple[List[float], float]:
    """(radians per token of each of the dim / 2 pairs, factor on cosine and sine)."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary positions turn an even number of elements, got {dim}")
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError(f"rotary base must be a finite number above 1, got {base}")
    n, magnitude = dim // 2, 1.0
    if scaling is not None and scaling.kind == "ntk" and dim > 2:
        base = base * scaling.factor ** (dim / (dim - 2))
    freq = [base ** (-2.0 * i / dim) for i in range(n)]
    if scaling is None or scaling.kind == "ntk":
        return freq, magnitude
    f, length = scaling.factor, scaling.original_length
    if scaling.kind == "linear":
        return [w / f for w in freq], magnitude
    if scaling.kind == "bands":
        keep = [min(max((length * w / (2 * math.pi) - scaling.low) / (scaling.high - scaling.low), 0.0), 1.0)
                for w in freq]
    else:
        def pair_of(turns):  # the (fractional) pair that turns this often in the original length
            return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
        first = max(math.floor(pair_of(scaling.fast)), 0)
        # the ramp may end behind the last pair (n - 1): where every pair turns more than ``slow`` times,
        # none is stretched in full
        last = min(math.ceil(pair_of(scaling.slow)), dim - 1)
        keep = [1.0 - min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0) for i in range(n)]
        magnitude = 0.1 * math.log(f) + 1.0 if scaling.magnitude is None else scaling.magnitude
    return [w / f * (1.0 - k) + w * k for w, k in zip(freq, keep)], magnitude


def rotary_table(length: int, dim: int, base: float = 10000.0, scaling: Optional[RotaryScaling] = None,
                 device=None) -> torch.Tensor:
    """fp32 [length, dim] table of (cos, sin) of every pair at positions 0 .. length - 1, angles
    computed in 64 bits. Built once and passed to :func:`rotary` / :func:`rotary_qk`; ``dim`` is how
    many elements of a head turn (the head size, or less for a partial rotation)."""
    if length < 1:
        raise ValueError(f"a rotary table needs at least one position, got {length}")
    freq, magnitude = rotary_frequencies(dim, base, scaling)
    device = torch.device("cuda") if device is None else torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"rotary tables live on a GPU, got {device}")
    table = torch.empty(length, dim, dtype=torch.float32, device=device)
    _native.cuda().rotary_table(torch.tensor(freq, dtype=torch.float64, device=table.device), table, magnitude)
    return table


def _interleaved(layout: str) -> bool:
    if layout not in ("half", "interleaved"):
        raise ValueError(f"unknown rotary layout {layout!r} (half, interleaved)")
    return layout == "interleaved"


def rotary(x, table, positions=None, start: int = 0, heads: Optional[int] = None, layout: str = "half"):
    """Rotary positions of x [T, H, D] or [B, T, H, D] (bf16, fp16 or fp32, any strides): the first
    ``table.shape[1]`` elements of a head turn by their position's angles, the rest is copied.

    ``positions`` ([T] or [B, T], int64 or int32) gives each token's row of the table; without it
    token t is at ``start + t``. A position outside the table gives NaN in the elements that turn.
    ``heads``: only the first that many heads turn, the others are copied (a packed QKV projection
    viewed as [B, T, H + 2 Hk, D] turns H + Hk of them). ``layout``: pairs (i, i + dim/2) ("half") or
    (2i, 2i + 1) ("interleaved"). Returns a contiguous tensor; differentiable in x."""
    if heads is not None and heads < 0:
        raise ValueError(f"heads must not be negative, got {heads}")
    return _native.cuda().rotary(x, None, table, positions, start, -1 if heads is None else heads,
                                 _interleaved(layout), False)[0]


def rotary_qk(q, k, table, positions=None, start: int = 0, layout: str = "half"):
    """:func:`rotary` of queries [B, T, H, D] and keys [B, T, Hk, D] in one launch: returns both."""
    return tuple(_native.cuda().rotary(q, k, table, positions, start, -1, _interleaved(layout), False))


# ---------------------------------------------------------------- dropout
class DropoutState:
    """(seed, step) of the counter-based generator, two int64 values on the GPU.

    Every call takes its numbers from (seed, step, site, element): ``site`` tells the calls of one
    step apart, :meth:`advance` moves to the next step. The kernels read the values on the device, so a
    captured graph that contains :meth:`advance` draws anew at every replay. Data-parallel ranks use
    different seeds; calls with the same seed, step (modulo 2^32) and site draw the same mask. A backward
    pass uses the values that its forward pass found; a forward pass that is run again (recomputation)
    has to run before :meth:`advance`."""

    def __init__(self, seed: int, device=None, step: int = 0):
        device = torch.device("cuda") if device is None else torch.device(device)
        self.tensor = torch.tensor(self._values(seed, step), dtype=torch.int64, device=device)

    @staticmethod
    def _values(seed: int, step: int):  # any whole numbers, as signed 64-bit ones
        return [(int(v) + (1 << 63)) % (1 << 64) - (1 << 63) for v in (seed, step)]

    def set(self, seed: int, step: int = 0) -> None:
        self.tensor.copy_(torch.tensor(self._values(seed, step), dtype=torch.int64))

    def advance(self) -> None:
        self.tensor[1:].add_(1)


def _check_dropout(p: float, state) -> None:
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    if not isinstance(state, DropoutState):
        raise TypeError("dropout needs a DropoutState")


def dropout(x, p: float, state: DropoutState, site: int = 0):
    """Zero each element of x (bf16, fp16 or fp32) with probability ``p`` (rounded to a multiple of
    2^-16) and scale the others by the inverse of the probability to be kept. No mask is stored: the
    backward draws it again from the (seed, step) that the forward used. Returns a contiguous tensor."""
    _check_dropout(p, state)
    return _native.cuda().dropout(x, state.tensor, site, p)


# ---------------------------------------------------------------- attention with a decay per head
def _decay_scale(scale, D):
    return D ** -0.5 if scale is None else float(scale)


def _decay(q, k, v, log_decay, state, lengths, scale, return_state):
    out = _native.cuda().decay_attention(q, k, v, log_decay, state, lengths, scale, return_state)
    return tuple(out) if return_state else out[0]


def decay_attention(q, k, v, log_decay, state=None, lengths=None, scale: Optional[float] = None,
                    return_state: bool = False):
    """Causal linear attention with a decay for each head (tensor-core kernels, chunked over tokens):

        S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,    o_t = scale S_t^T q_t.

    q, k, v: bf16 [B, T, H, D] of the same shape, D 64 or 128, any strides. ``log_decay``: fp32 [H],
    each at most 0 (0: no decay); not trained. ``state``: contiguous fp32 [B, H, D, D] before the first
    token (default zero). ``lengths``: int32 [B], clipped to 0 .. T; tokens from there on do not exist
    (not read, zero output and gradients, the final state is the one behind the last token). ``scale``
    defaults to D^-0.5. Returns o [B, T, H, D] bf16, or (o, final state) with ``return_state``;
    differentiable in q, k, v and state, once. Tokens are worked on in chunks of 64: a value that is
    not finite can show in the output of every token of its chunk. A kernel whose wait for its own
    products is not answered within 2 s (never seen) leaves NaN in its rows and its state and ends;
    ``_native.cuda().decay_error_flag()`` then reads 1 for the current GPU (the call synchronises)."""
    return _decay(q, k, v, log_decay, state, lengths, _decay_scale(scale, q.shape[-1]), return_state)


def decay_attention_qkv(qkv, log_decay, state=None, lengths=None, scale: Optional[float] = None,
                        return_state: bool = False):
    """:func:`decay_attention` on a packed projection qkv [B, T, 3, H, D]; the gradient comes back
    packed, in one buffer."""
    return _decay(qkv, None, None, log_decay, state, lengths, _decay_scale(scale, qkv.shape[-1]), return_state)


def decay_attention_step(q, k, v, log_decay, state, scale: Optional[float] = None):
    """One token of :func:`decay_attention` for inference: q, k, v bf16 [B, H, D]; updates ``state``
    (contiguous fp32 [B, H, D, D]) in place and returns o [B, H, D]."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay, state)):
        raise ValueError("decay_attention_step has no gradient; call it under torch.no_grad() or train with "
                         "decay_attention")
    return _native.cuda().decay_step(q, k, v, log_decay, state, _decay_scale(scale, q.shape[-1]))
