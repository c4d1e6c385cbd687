"""Attention over a prefix that a batch shares, and the weights it gave to cached tokens.

The restore path ends with 16-bit caches of a prompt chunk that many requests have in common.
:func:`shared_prefix_attention` reads that prefix once for all sequences of a batch, next to
each sequence's own cache (dense, or pages of a pool), for single tokens and for whole prompts.
:func:`accumulate_attention_weights` adds up, per cached token, the weight it was given: the
measure that :func:`evict_tokens` goes by.
"""

from __future__ import annotations

import ctypes
import math

import torch

from .. import _lib
from .paged import _status_word
from .staging import Plans, integers, step_arguments
from .validation import require_apart, require_cuda, require_no_grad, same_view

_DTYPES = (torch.float16, torch.bfloat16)


def _refuse_rows(name: str, t: torch.Tensor):
    raise ValueError(f"{name}: head_dim must be contiguous and rows must start at multiples of "
                     f"16 bytes, got strides {tuple(t.stride())}")


def _like(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype, dev: torch.device) -> None:
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} like q, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, q on {dev}")


def _rows3(name: str, t: torch.Tensor) -> tuple[int, int]:
    """Strides of ``[n, H, D]`` rows of 16-bit values (0 where a dimension has one entry), with
    a unit stride along the head and every row at a multiple of 16 bytes."""
    n0, n1, n2 = t.shape
    s0, s1, s2 = t.stride()
    if n0 < 2:
        s0 = 0
    if n1 < 2:
        s1 = 0
    if ((s0 | s1) & 7 or s2 != 1 or t.data_ptr() & 15) and t.numel():
        _refuse_rows(name, t)
    return s0, s1


def _rows4(name: str, t: torch.Tensor, mask: int = 7) -> tuple[int, int, int]:
    """:func:`_rows3` of ``[B, n, H, D]``; ``mask``: elements of 16 bytes, less one."""
    nb, n0, n1, n2 = t.shape
    sb, s0, s1, s2 = t.stride()
    if nb < 2:
        sb = 0
    if n0 < 2:
        s0 = 0
    if n1 < 2:
        s1 = 0
    if ((sb | s0 | s1) & mask or s2 != 1 or t.data_ptr() & 15) and t.numel():
        _refuse_rows(name, t)
    return sb, s0, s1


def _check_queries(q: torch.Tensor, kv_heads: int) -> tuple[int, int, int]:
    if q.ndim != 3:
        raise ValueError(f"q must be [tokens, heads, head_dim], got {tuple(q.shape)}")
    if q.dtype not in _DTYPES:
        raise TypeError(f"q must be float16 or bfloat16, got {q.dtype}")
    n, hq, d = q.shape
    if d == 0 or d % 8 or d > 256:
        raise ValueError(f"head_dim must be a multiple of 8 and at most 256, got {d}")
    if kv_heads == 0 or hq % kv_heads:
        raise ValueError(f"{hq} query heads are no multiple of {kv_heads} KV heads")
    return n, hq, d


def _sequence_starts(n: int, batch: int, q_lens, cu_q_lens, max_q_len):
    """(starts or None, tokens a sequence at most) from whichever the caller gave."""
    if q_lens is not None and cu_q_lens is not None:
        raise ValueError("give q_lens or cu_q_lens, not both")
    if q_lens is not None:
        if isinstance(q_lens, torch.Tensor):
            if q_lens.is_cuda:
                raise ValueError("q_lens are host values; pass device starts as cu_q_lens")
            q_lens = q_lens.reshape(-1).tolist()
        lens = [int(x) for x in q_lens]
        if len(lens) != batch or any(x < 0 for x in lens) or sum(lens) > n:
            raise ValueError(f"q_lens must be {batch} lengths of at most {n} tokens together, got "
                             f"{len(lens)} of {sum(lens)}")
        if len(set(lens)) == 1 and lens[0] * batch == n:
            return None, lens[0]
        cu = [0]
        for x in lens:
            cu.append(cu[-1] + x)
        return torch.tensor(cu, dtype=torch.int32), max(lens, default=0)
    if cu_q_lens is not None:
        if not isinstance(cu_q_lens, torch.Tensor) or cu_q_lens.dtype != torch.int32 or \
                cu_q_lens.shape != (batch + 1,):
            raise ValueError(f"cu_q_lens must be an int32 tensor [{batch + 1}]")
        if max_q_len is None:
            raise ValueError("cu_q_lens needs max_q_len")
        if not 0 <= int(max_q_len) <= n:
            raise ValueError(f"max_q_len must lie in [0, {n}], got {max_q_len}")
        return cu_q_lens.contiguous(), int(max_q_len)
    if n == 0 and batch == 0:
        return None, 0
    if batch == 0 or n % batch:
        raise ValueError(f"{n} tokens are not the same number for each of {batch} sequences; give q_lens")
    return None, n // batch


def _lengths(name: str, lens, batch: int, most: int):
    """int32 [batch] lengths; host values are checked here, device values by the kernel."""
    if lens is None or (isinstance(lens, torch.Tensor) and lens.is_cuda and lens.dtype == torch.int32 and
                        lens.shape == (batch,) and lens.stride(0) == 1):
        return lens
    lens = integers(lens)
    if lens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be integers, got {lens.dtype}")
    if lens.shape != (batch,):
        raise ValueError(f"{name} must be [{batch}], got {tuple(lens.shape)}")
    if not lens.is_cuda and batch and (int(lens.min()) < 0 or int(lens.max()) > most):
        raise ValueError(f"{name} must lie in [0, {most}]")
    return _int32(lens).contiguous()


def _int32(t: torch.Tensor) -> torch.Tensor:
    """Lengths or page ids as int32; what int32 cannot hold stays out of range."""
    return t.clamp(-1, 2 ** 31 - 1).to(torch.int32) if t.dtype == torch.int64 else t.to(torch.int32)


def _on_device(what: str, tensors: list, device: torch.device) -> list:
    """Device versions of the given (or None) small arguments."""
    for t in tensors:
        if t is not None and t.device != device:
            break
    else:
        return tensors
    there = [t for t in tensors if t is not None]
    moved = iter(step_arguments(what, there, device))
    return [None if t is None else next(moved) for t in tensors]


_LAYOUTS = Plans()
_WORKSPACES = Plans()


class _Layout:
    """Sizes of a call and its tensors' strides in one host array."""

    __slots__ = ("n", "hq", "hk", "d", "p_len", "rows", "cap", "array", "qs", "kps", "vps", "kcs", "vcs",
                 "scale")

    def __init__(self, q, k_prefix, v_prefix, k_cache, v_cache) -> None:
        ref = k_prefix if k_prefix is not None else k_cache
        if ref is None:
            raise ValueError("neither a prefix nor caches given")
        if (k_prefix is None) != (v_prefix is None) or (k_cache is None) != (v_cache is None):
            raise ValueError("keys and values must be given together")
        if ref.ndim < 2:
            raise ValueError(f"keys must be [.., Hkv, D], got {tuple(ref.shape)}")
        self.hk = hk = ref.shape[-2]
        self.n, self.hq, self.d = _check_queries(q, hk)
        d, dtype, dev = self.d, q.dtype, q.device
        self.scale = 1.0 / math.sqrt(d)
        strides = [*_rows3("q", q)]
        self.p_len = self.rows = self.cap = 0
        if k_prefix is not None:
            self.p_len = k_prefix.shape[0]
            shape = (self.p_len, hk, d)
            _like("k_prefix", k_prefix, shape, dtype, dev)
            _like("v_prefix", v_prefix, shape, dtype, dev)
            strides += [*_rows3("k_prefix", k_prefix), *_rows3("v_prefix", v_prefix)]
        else:
            strides += [0] * 4
        if k_cache is not None:
            if k_cache.ndim != 4:
                raise ValueError(f"caches must be [B, S, Hkv, D], got {tuple(k_cache.shape)}")
            self.rows, self.cap = k_cache.shape[0], k_cache.shape[1]
            shape = (self.rows, self.cap, hk, d)
            _like("k_cache", k_cache, shape, dtype, dev)
            _like("v_cache", v_cache, shape, dtype, dev)
            strides += [*_rows4("k_cache", k_cache), *_rows4("v_cache", v_cache)]
        self.array = (ctypes.c_int64 * 12)(*strides)
        base = ctypes.addressof(self.array)
        self.qs, self.kps, self.vps, self.kcs, self.vcs = (base + 8 * i for i in (0, 2, 4, 6, 9))


def _aligned(*tensors) -> bool:
    bits = 0
    for t in tensors:
        if t is not None:
            bits |= t.data_ptr()
    return not bits & 15


def shared_prefix_attention(
    q: torch.Tensor,
    k_prefix: torch.Tensor | None,
    v_prefix: torch.Tensor | None,
    k_cache: torch.Tensor | None = None,
    v_cache: torch.Tensor | None = None,
    cache_lens=None,
    *,
    q_lens=None,
    cu_q_lens: torch.Tensor | None = None,
    max_q_len: int | None = None,
    page_table=None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of ``B`` sequences over a shared prefix and their own caches.

    Args:
        q: float16 or bfloat16 ``[N, Hq, D]``, the sequences' queries one after another.
        k_prefix, v_prefix: ``[P, Hkv, D]``, seen by every query (or None).
        k_cache, v_cache: own caches ``[B, S, Hkv, D]``, or with ``page_table`` a pool
            ``[n_pages, page, Hkv, D]`` (or None).
        cache_lens: ``[B]`` tokens in use, the queries' own among them (default: all).  Query j of
            a sequence's n sees its cache's tokens ``t <= len - n + j``.
        q_lens: ``[B]`` host query counts; or ``cu_q_lens`` int32 ``[B + 1]`` starts on the device
            with ``max_q_len``.  Default: N / B each.  A sequence whose device starts decrease, lie
            outside those of the first and the last or are more than ``max_q_len`` apart has no rows
            (reported by :func:`paged_status`).  Rows of no sequence are left as they were (in
            outputs allocated here: undefined).
        page_table: int32 ``[B, max_pages]``.  A bad id's tokens count as masked, a bad device
            length as 0, both reported by :func:`paged_status`.
        scale: of the scores, default ``D ** -0.5``.
        out: ``[N, Hq, D]`` output, overlapping no input.

    Any strides with a contiguous, 16-byte aligned head; ``D`` a multiple of 8 up to 256.  Scores,
    sums and accumulators are float32.  Returns ``(out, lse)`` with float32 ``lse [N, Hq]`` (natural
    logarithm); a row that sees nothing is zero with ``lse = -inf``.  What a row does not see never
    reaches it, NaN and infinities included.
    """
    require_cuda(q)
    require_no_grad("shared_prefix_attention", q, k_prefix, v_prefix, k_cache, v_cache, out)
    dev, dtype = q.device, q.dtype
    key = [q.shape, q.stride(), dtype, dev]
    for t in (k_prefix, v_prefix, k_cache, v_cache):
        key += (None,) if t is None else (t.shape, t.stride(), t.dtype, t.device)
    key = tuple(key)
    lay = _LAYOUTS.get(key)
    if lay is None or not _aligned(q, k_prefix, v_prefix, k_cache, v_cache):
        lay = _LAYOUTS.keep(key, _Layout(q, k_prefix, v_prefix, k_cache, v_cache))
    n, hq, hk, d, p_len = lay.n, lay.hq, lay.hk, lay.d, lay.p_len
    batch, cap, page, n_pages, table, lens = 0, 0, 1, 0, None, None
    if k_cache is not None:
        if page_table is not None:
            table = integers(page_table)
            if table.dtype not in (torch.int32, torch.int64):
                raise TypeError(f"page_table must be integers, got {table.dtype}")
            if table.ndim != 2:
                raise ValueError(f"page_table must be [B, max_pages], got {tuple(table.shape)}")
            if table.dtype != torch.int32:
                table = _int32(table)
            if table.stride(1) != 1 and table.shape[1] > 1:
                table = table.contiguous()
            batch, page, n_pages = table.shape[0], lay.cap, lay.rows
            cap = table.shape[1] * page
        else:
            batch, cap = lay.rows, lay.cap
            page = max(cap, 1)
        lens = _lengths("cache_lens", cache_lens, batch, cap)
    elif page_table is not None or cache_lens is not None:
        raise ValueError("page_table and cache_lens belong to caches, none given")
    cu, nq = None, n
    if batch or q_lens is not None or cu_q_lens is not None:
        if batch == 0 and k_cache is None:
            raise ValueError("q_lens belong to caches, none given")
        cu, nq = _sequence_starts(n, batch, q_lens, cu_q_lens, max_q_len)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _like("out", out, (n, hq, d), dtype, dev)
        require_apart("out", out, q, k_prefix, v_prefix, k_cache, v_cache)
    lse = q.new_empty((n, hq), dtype=torch.float32)
    if n == 0 or hq == 0:
        return out, lse
    table, lens, cu = _on_device("shared_prefix_attention", [table, lens, cu], dev)
    if scale is None:
        scale = lay.scale
    elif not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    lib = _lib.load()
    sizes = (n, batch, hq, hk, d, nq, p_len, cap, page)
    need = _WORKSPACES.get(sizes)
    if need is None:
        size = ctypes.c_int64()
        _lib.check(lib.sc_shared_prefix_attention_workspace(*sizes, ctypes.addressof(size)),
                   "shared_prefix_attention")
        need = _WORKSPACES.keep(sizes, size.value)
    with _lib.on_device(dev):
        work = q.new_empty(need, dtype=torch.uint8) if need else None
        os = _lib.stride_buffer().put(_rows3("out", out))
        rc = lib.sc_shared_prefix_attention(
            n, batch, hq, hk, d, _lib.DTYPE_CODE[dtype], q.data_ptr(), lay.qs,
            p_len, _lib.ptr(k_prefix), lay.kps, _lib.ptr(v_prefix), lay.vps,
            cap, _lib.ptr(k_cache), lay.kcs, _lib.ptr(v_cache), lay.vcs, _lib.ptr(lens),
            _lib.ptr(table), table.stride(0) if table is not None else 0, page, n_pages,
            _lib.ptr(cu), nq, scale, out.data_ptr(), os, lse.data_ptr(),
            _lib.ptr(work), need, _status_word(dev).data_ptr(), _lib.stream_handle(dev))
    _lib.check(rc, "shared_prefix_attention")
    return out, lse


def accumulate_attention_weights(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    lse: torch.Tensor,
    scores: torch.Tensor,
    cache_lens=None,
    *,
    q_lens=None,
    cu_q_lens: torch.Tensor | None = None,
    max_q_len: int | None = None,
    causal: bool = True,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Add the weights that queries gave to cached tokens: ``out[b, h, t] = scores[b, h, t] +
    sum exp(scale * q . k_t - lse)`` over the queries of sequence ``b`` that see token ``t`` and the
    query heads of KV head ``h``.

    Args:
        q: ``[N, Hq, D]`` as given to the attention.
        k_cache: ``[B, S, Hkv, D]`` keys.  For a shared prefix: ``k_prefix[None]`` with
            ``causal=False``, whose weights are then those of the whole batch.
        lse: float32 ``[N, Hq]`` that the attention returned (over all that the queries saw).
        scores: float32 ``[B, Hkv, S]`` so far.
        cache_lens, q_lens, cu_q_lens, max_q_len, scale: as in :func:`shared_prefix_attention`.
        causal: query j of n sees ``t <= len - n + j``; otherwise every token in use.
        out: default: ``scores`` itself, added to in place.

    Tokens not in use keep their score.  No atomics are used; the same inputs give the same bits.
    """
    require_cuda(q)
    require_no_grad("accumulate_attention_weights", q, k_cache, lse, scores, out)
    dev = q.device
    if k_cache.ndim != 4:
        raise ValueError(f"k_cache must be [B, S, Hkv, D], got {tuple(k_cache.shape)}")
    batch, s, hk, _ = k_cache.shape
    n, hq, d = _check_queries(q, hk)
    _like("k_cache", k_cache, (batch, s, hk, d), q.dtype, dev)
    qs, ks = _rows3("q", q), _rows4("k_cache", k_cache)
    if out is None:
        out = scores
    for name, t, shape in (("lse", lse, (n, hq)), ("scores", scores, (batch, hk, s)),
                           ("out", out, (batch, hk, s))):
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32, got {t.dtype}")
        if t.shape != shape or t.device != dev:
            raise ValueError(f"{name} must be {list(shape)} on {dev}, got {tuple(t.shape)} on {t.device}")
    for name, t in (("scores", scores), ("out", out)):
        if t.stride(2) != 1 and s > 1:
            raise ValueError(f"{name} must be contiguous along its tokens, got strides {tuple(t.stride())}")
    if same_view(out, scores):
        require_apart("out", out, q, k_cache, lse)
    else:
        require_apart("out", out, q, k_cache, lse, scores)
    lens = _lengths("cache_lens", cache_lens, batch, s)
    cu, nq = _sequence_starts(n, batch, q_lens, cu_q_lens, max_q_len)
    if out.numel() == 0:
        return out
    lens, cu = _on_device("accumulate_attention_weights", [lens, cu], dev)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    elif not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    lib = _lib.load()
    st = _lib.stride_buffer()
    with _lib.on_device(dev):
        rc = lib.sc_accumulate_attention_weights(
            n, batch, hq, hk, d, _lib.DTYPE_CODE[q.dtype], q.data_ptr(), st.put(qs),
            s, k_cache.data_ptr(), st.put(ks), _lib.ptr(lens), _lib.ptr(cu), nq,
            1 if causal else 0, scale, lse.data_ptr(), st.put(lse.stride()),
            scores.data_ptr(), st.put(scores.stride()[:2]), out.data_ptr(), st.put(out.stride()[:2]),
            _status_word(dev).data_ptr(), _lib.stream_handle(dev))
    _lib.check(rc, "accumulate_attention_weights")
    return out
