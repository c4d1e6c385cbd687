"""Eviction: a cache cut to its budget by accumulated attention weight."""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from .attention import _lengths, _on_device, _rows4
from .paged import _status_word
from .validation import require_apart, require_cuda, require_no_grad, same_view

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


class Evicted(NamedTuple):
    """What :func:`evict_tokens` leaves of a cache."""

    k: torch.Tensor        # [B, budget, Hkv, D]
    v: torch.Tensor
    scores: torch.Tensor   # float32 [B, Hkv, budget]
    indices: torch.Tensor  # int32 [B, Hkv, budget]: where each token was, then -1
    lens: torch.Tensor     # int32 [B]


def evict_tokens(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    scores: torch.Tensor,
    budget: int,
    cache_lens=None,
    *,
    keep_first: int = 0,
    keep_recent: int = 0,
    k_out: torch.Tensor | None = None,
    v_out: torch.Tensor | None = None,
    scores_out: torch.Tensor | None = None,
) -> Evicted:
    """Keep at most ``budget`` tokens of each sequence and KV head.

    The first ``keep_first`` and the last ``keep_recent`` tokens in use stay, and of the others
    those of the highest score (equal scores: the lower index; NaN counts as minus infinity).  What
    stays moves to the front in its order; keys keep the positions they were turned by.

    Args:
        k_cache, v_cache: ``[B, S, Hkv, D]`` float16, bfloat16 or float32 (views of a model-layout
            cache by ``transpose(1, 2)``), ``S`` up to 393216.
        scores: float32 ``[B, Hkv, S]``, as :func:`accumulate_attention_weights` gives them.
        cache_lens: ``[B]`` tokens in use (default: all).
        k_out, v_out: ``[B, budget, Hkv, D]``, and ``scores_out`` float32 ``[B, Hkv, budget]``.  An
            output may be its input's first ``budget`` tokens: then that one moves in place, and no
            other input may reach into it (one tensor as keys and values).  Rows behind a
            sequence's new length are left as they were (in outputs allocated here: zeros).

    Returns :class:`Evicted`.
    """
    require_cuda(k_cache)
    require_no_grad("evict_tokens", k_cache, v_cache, scores, k_out, v_out, scores_out)
    dev = k_cache.device
    if k_cache.ndim != 4:
        raise ValueError(f"caches must be [B, S, Hkv, D], got {tuple(k_cache.shape)}")
    if k_cache.dtype not in _DTYPES:
        raise TypeError(f"caches must be float16, bfloat16 or float32, got {k_cache.dtype}")
    b, s, h, d = k_cache.shape
    budget, keep_first, keep_recent = int(budget), int(keep_first), int(keep_recent)
    if budget < 0 or keep_first < 0 or keep_recent < 0 or keep_first + keep_recent > budget:
        raise ValueError(f"keep_first {keep_first} and keep_recent {keep_recent} must fit the budget "
                         f"of {budget} tokens")
    if d * k_cache.element_size() % 16:
        raise ValueError(f"rows of {d} x {k_cache.dtype} are no multiple of 16 bytes")
    if v_cache.shape != k_cache.shape or v_cache.device != dev:
        raise ValueError(f"v_cache {tuple(v_cache.shape)} on {v_cache.device} does not match k_cache")
    if v_cache.dtype != k_cache.dtype:
        raise TypeError(f"v_cache must be {k_cache.dtype} like k_cache, got {v_cache.dtype}")
    if scores.dtype != torch.float32:
        raise TypeError(f"scores must be float32, got {scores.dtype}")
    if scores.shape != (b, h, s) or scores.device != dev:
        raise ValueError(f"scores must be {[b, h, s]} on {dev}, got {tuple(scores.shape)} on {scores.device}")
    mask = 16 // k_cache.element_size() - 1
    st = _lib.stride_buffer()
    ks, vs = st.put(_rows4("k_cache", k_cache, mask)), st.put(_rows4("v_cache", v_cache, mask))
    lens = _lengths("cache_lens", cache_lens, b, s)
    fresh = torch.empty if lens is None and s >= budget else torch.zeros
    in_place = False
    inputs = (k_cache, v_cache, scores)
    outs: list[torch.Tensor] = []
    for role, (name, src, out) in enumerate((("k_out", k_cache, k_out), ("v_out", v_cache, v_out),
                                             ("scores_out", scores, scores_out))):
        if out is None:
            if name == "scores_out":
                out = fresh((b, h, budget), dtype=torch.float32, device=dev)
            else:
                out = fresh((b, h, budget, d), dtype=src.dtype, device=dev).transpose(1, 2)
            outs.append(out)
            continue
        want = (b, h, budget) if name == "scores_out" else (b, budget, h, d)
        if out.shape != want or out.device != dev:
            raise ValueError(f"{name} must be {list(want)} on {dev}, got {tuple(out.shape)} on {out.device}")
        if out.dtype != src.dtype:
            raise TypeError(f"{name} must be {src.dtype}, got {out.dtype}")
        if budget and same_view(out, src):
            if budget > s:
                raise ValueError(f"{name} in place cannot hold more than its {s} tokens")
            in_place = True
            # keys, values and scores move in blocks of their own, in no order among them
            require_apart(name, out, *outs, *inputs[:role], *inputs[role + 1:])
        else:
            require_apart(name, out, *outs, *inputs)
        outs.append(out)
    for name, t in (("scores", scores), ("scores_out", outs[2])):
        if t.shape[2] > 1 and t.stride(2) != 1:
            raise ValueError(f"{name} must be contiguous along its tokens, got strides {tuple(t.stride())}")
    indices = torch.empty((b, h, budget), dtype=torch.int32, device=dev)
    new_lens = torch.empty(b, dtype=torch.int32, device=dev)
    if b == 0:
        return Evicted(*outs, indices, new_lens)
    (lens,) = _on_device("evict_tokens", [lens], dev)
    ko, vo, so = outs
    kos, vos = st.put(_rows4("k_out", ko, mask)), st.put(_rows4("v_out", vo, mask))
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.sc_evict_tokens(
            b, h, s, d, k_cache.element_size(), budget, keep_first, keep_recent,
            k_cache.data_ptr(), ks, v_cache.data_ptr(), vs,
            scores.data_ptr(), st.put(scores.stride()[:2]), _lib.ptr(lens), 1 if in_place else 0,
            ko.data_ptr(), kos, vo.data_ptr(), vos,
            so.data_ptr(), st.put(so.stride()[:2]), indices.data_ptr(), new_lens.data_ptr(),
            _status_word(dev).data_ptr(), _lib.stream_handle(dev))
    _lib.check(rc, "evict_tokens")
    return Evicted(ko, vo, so, indices, new_lens)
