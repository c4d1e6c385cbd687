"""Rotary positions of new queries and keys.

The restore path turns cached keys by a relative shift (:func:`rope_shift_keys` and the fused
restore); this module turns a step's own queries and keys by their absolute positions before
the keys join the cache, in one launch of ``sc_rope_apply`` for both.  The half layout (the
pairing of the restore path) and the interleaved one, a rotary part smaller than the head, and
the usual ways to scale the frequencies for contexts longer than the trained ones.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import numpy as np
import torch

from .. import _lib
from .restore import DEFAULT_THETA
from .staging import Plans, integers, step_arguments
from .validation import require_apart, require_cuda, require_no_grad, same_view

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_KINDS = ("linear", "ntk", "bands", "yarn")


@dataclass(frozen=True)
class RopeScaling:
    """How the rotary frequencies ``f_i = theta^(-2i/R)`` are scaled for long contexts.

    ``kind``:

    * ``"linear"``: every frequency divided by ``factor`` (position interpolation);
    * ``"ntk"``: ``theta`` multiplied by ``factor^(R / (R - 2))``, which slows the lowest
      frequency by ``factor`` and leaves the highest;
    * ``"bands"``: by the turns a frequency makes over ``original_length`` positions: divided by
      ``factor`` below ``low_freq_factor`` turns, kept above ``high_freq_factor``, a linear
      blend between;
    * ``"yarn"``: divided by ``factor`` or kept by a linear ramp over the frequency's index,
      between the (rounded out) indices that make ``beta_fast`` and ``beta_slow`` turns over
      ``original_length`` positions; cosines and sines are multiplied by
      ``0.1 ln(factor) + 1``.

    ``attention_factor`` replaces the factor of the cosines and sines (1 but for ``"yarn"``).
    """

    kind: str
    factor: float
    original_length: int = 0
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def __post_init__(self) -> None:
        if self.kind not in _KINDS:
            raise ValueError(f"scaling kind must be one of {_KINDS}, got {self.kind!r}")
        if not (math.isfinite(self.factor) and self.factor > 0):
            raise ValueError(f"factor must be positive and finite, got {self.factor}")
        if self.kind in ("bands", "yarn") and self.original_length <= 0:
            raise ValueError(f"{self.kind!r} scaling needs original_length")
        if self.kind == "bands" and not self.high_freq_factor > self.low_freq_factor:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        if self.kind == "yarn" and not self.beta_fast > self.beta_slow > 0:
            raise ValueError("beta_fast must be above beta_slow, both positive")
        if self.attention_factor is not None and not (
                math.isfinite(self.attention_factor) and self.attention_factor > 0):
            raise ValueError(f"attention_factor must be positive and finite, got {self.attention_factor}")


def rotary_frequencies(rotary_dim: int, theta: float = DEFAULT_THETA,
                       scaling: RopeScaling | None = None) -> tuple[np.ndarray, float]:
    """float64 ``[rotary_dim / 2]`` frequencies in radians per position, and the factor of the
    cosines and sines."""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError(f"theta must be positive and finite, got {theta}")
    theta = float(theta)
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    s = scaling
    if s is not None and s.kind == "ntk" and rotary_dim > 2:
        theta *= s.factor ** (rotary_dim / (rotary_dim - 2))
    f = theta ** (-2.0 * i / rotary_dim) if rotary_dim else i
    mult = 1.0
    if s is not None:
        if s.kind == "linear":
            f = f / s.factor
        elif s.kind == "bands":
            turns = s.original_length * f / (2 * math.pi)
            keep = np.clip((turns - s.low_freq_factor) / (s.high_freq_factor - s.low_freq_factor), 0.0, 1.0)
            f = (1.0 - keep) * (f / s.factor) + keep * f
        elif s.kind == "yarn":
            if theta <= 1.0:
                raise ValueError(f"yarn scaling needs theta above 1, got {theta}")

            def index(turns: float) -> float:
                return rotary_dim * math.log(s.original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))

            lo = max(math.floor(index(s.beta_fast)), 0)
            hi = min(math.ceil(index(s.beta_slow)), rotary_dim - 1)
            slow = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
            f = slow * (f / s.factor) + (1.0 - slow) * f
            mult = 0.1 * math.log(s.factor) + 1.0 if s.factor > 1 else 1.0
        if s.attention_factor is not None:
            mult = s.attention_factor
    return np.ascontiguousarray(f), mult


_FREQUENCIES: dict[tuple, tuple[np.ndarray, int, float]] = {}


def _frequencies(rotary_dim: int, theta: float, scaling: RopeScaling | None):
    """(table, its address, factor), one table per (rotary_dim, theta, scaling)."""
    key = (rotary_dim, theta, scaling)
    hit = _FREQUENCIES.get(key)
    if hit is None:
        f, mult = rotary_frequencies(rotary_dim, theta, scaling)
        hit = _FREQUENCIES[key] = (f, f.ctypes.data, mult)
    return hit


def _layout(name: str, x: torch.Tensor) -> tuple[int, int, int, int, tuple[int, int, int, int]]:
    """(batch, tokens, heads, head_dim, strides in that order) of a 3-D or 4-D tensor."""
    if x.ndim == 3:
        s = x.stride()
        return 1, x.shape[0], x.shape[1], x.shape[2], (0, s[0], s[1], s[2])
    if x.ndim == 4:
        s = x.stride()
        return x.shape[0], x.shape[2], x.shape[1], x.shape[3], (s[0], s[2], s[1], s[3])
    raise ValueError(f"{name} must be [T, H, D] or [B, H, T, D], got {tuple(x.shape)}")


class _Plan:
    """What follows from the layouts of queries and keys alone: sizes, and strides (of the inputs
    and of new contiguous outputs) in one host array."""

    __slots__ = ("sizes", "code", "array", "q", "k", "fresh_q", "fresh_k")

    def __init__(self, q: torch.Tensor, k: torch.Tensor | None, rotary_dim: int | None) -> None:
        if q.dtype not in _DTYPES:
            raise TypeError(f"q must be float16, bfloat16 or float32, got {q.dtype}")
        self.code = _lib.DTYPE_CODE[q.dtype]
        b, t, hq, d, qs = _layout("q", q)
        hk, ks = 0, (0, 0, 0, 0)
        if k is not None:
            kb, kt, hk, kd, ks = _layout("k", k)
            if (kb, kt, kd, k.ndim) != (b, t, d, q.ndim):
                raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
            if k.dtype != q.dtype:
                raise TypeError(f"k must be {q.dtype} like q, got {k.dtype}")
            if k.device != q.device:
                raise ValueError(f"k is on {k.device}, q on {q.device}")
        rd = d if rotary_dim is None else int(rotary_dim)
        if rd < 0 or rd % 2 or rd > d:
            raise ValueError(f"rotary_dim must be even and at most head_dim {d}, got {rd}")
        self.sizes = (b, t, hq, hk, d, rd)

        def fresh(h: int) -> tuple[int, int, int, int]:  # (batch, token, head, element) strides
            return (0, h * d, d, 1) if q.ndim == 3 else (h * t * d, d, t * d, 1)

        self.array = (ctypes.c_int64 * 16)(*qs, *ks, *fresh(hq), *fresh(hk))
        base = ctypes.addressof(self.array)
        self.q, self.k, self.fresh_q, self.fresh_k = (base + 32 * i for i in range(4))


_PLANS = Plans()


def apply_rotary(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions,
    *,
    theta: float = DEFAULT_THETA,
    rotary_dim: int | None = None,
    interleaved: bool = False,
    scaling: RopeScaling | None = None,
    inverse: bool = False,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
):
    """Turn queries and keys by their positions.

    Args:
        q: float16, bfloat16 or float32 ``[T, Hq, D]``, or ``[B, Hq, T, D]`` in the model layout.
        k: keys of the same layout and dtype with their own head count, or None.
        positions: integers ``[T]`` (or ``[B, T]`` with the model layout) on the device or the
            host, or one int: the first token's position, the others follow it.
        rotary_dim: how many leading elements of a head are turned (default: all).
        interleaved: pairs are neighbours (2i, 2i + 1) instead of (i, i + rotary_dim / 2).
        scaling: a :class:`RopeScaling`; None: unscaled.
        inverse: undo the rotation (and the scaling's factor) instead.
        q_out, k_out: outputs of the inputs' shape and dtype, any strides (a cache's next slots, or
            the input itself, apart from the other input); new contiguous tensors by default.

    Angles are off by at most 2^-26 of a turn (their conversion to float32) and 2^-54 of a turn a
    position (the frequency's 53 bits); products are in float32 and rounded once.  Returns ``q_out``, or ``(q_out, k_out)`` when keys are given.
    """
    require_cuda(q)
    require_no_grad("apply_rotary", q, k, q_out, k_out)
    dev = q.device
    key = (q.shape, q.stride(), q.dtype, rotary_dim,
           None if k is None else (k.shape, k.stride(), k.dtype, k.device == dev))
    plan = _PLANS.get(key) or _PLANS.keep(key, _Plan(q, k, rotary_dim))
    if k is None and k_out is not None:
        raise ValueError("k_out given without k")
    b, t, hq, hk, d, rd = plan.sizes
    qo = torch.empty_like(q, memory_format=torch.contiguous_format) if q_out is None else q_out
    ko = k_out
    if k is not None and k_out is None:
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    if q_out is not None or k_out is not None:
        for name, x, out, given, other in (("q_out", q, qo, q_out, k), ("k_out", k, ko, k_out, q)):
            if given is None:
                continue
            if out.shape != x.shape or out.device != dev:
                raise ValueError(f"{name} must have shape {tuple(x.shape)} on {dev}, "
                                 f"got {tuple(out.shape)} on {out.device}")
            if out.dtype != x.dtype:
                raise TypeError(f"{name} must be {x.dtype}, got {out.dtype}")
            if same_view(out, x):
                require_apart(name, out, other)
            else:
                require_apart(name, out, x, other)
    if q_out is not None and k_out is not None:
        require_apart("k_out", ko, qo)

    start, pos_ptr, pos64, ps = 0, None, 0, (0, 0)
    if isinstance(positions, int):
        start = positions
    else:
        positions = integers(positions)
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.shape != (t,) and positions.shape != (b, t):
            raise ValueError(f"positions must be [{t}] or [{b}, {t}], got {tuple(positions.shape)}")
        if positions.device != dev:
            (positions,) = step_arguments("apply_rotary", [positions.contiguous()], dev)
        pos64 = 1 if positions.dtype == torch.int64 else 0
        s = positions.stride()
        ps = (0, s[0]) if len(s) == 1 else (s[0], s[1])
        pos_ptr = positions.data_ptr()
    if b * t == 0 or d == 0:
        return qo if k is None else (qo, ko)
    _, freq_ptr, mult = _frequencies(rd, float(theta), scaling)
    lib = _lib.load()
    st = _lib.stride_buffer()
    qos = plan.fresh_q if q_out is None else st.put(_layout("q_out", qo)[4])
    kos = None if ko is None else plan.fresh_k if k_out is None else st.put(_layout("k_out", ko)[4])
    with _lib.on_device(dev):
        rc = lib.sc_rope_apply(
            b, t, hq, hk, d, rd, 1 if interleaved else 0, q.data_ptr(), plan.q, _lib.ptr(k), plan.k, plan.code,
            pos_ptr, pos64, st.put(ps), start, freq_ptr, mult, 1 if inverse else 0,
            qo.data_ptr(), qos, _lib.ptr(ko), kos, _lib.stream_handle(dev))
    _lib.check(rc, "apply_rotary")
    return qo if k is None else (qo, ko)
