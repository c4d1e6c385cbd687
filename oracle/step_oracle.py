"""float64 oracle of the step operators (test infrastructure, never imported by the package):
rotary positions, shared-prefix attention, accumulated attention weights and eviction, written
from their definitions with loops where that is plainer.
"""

from __future__ import annotations

import math

import torch


def rotary(x, positions, freqs, *, rotary_dim, interleaved=False, mult=1.0, inverse=False):
    """x ``[..., T, H, D]``, positions ``[..., T]``, freqs float64 ``[rotary_dim / 2]``."""
    y = x.double().clone()
    a = positions.double()[..., None, None] * torch.as_tensor(freqs, dtype=torch.float64)
    c, s = torch.cos(a), torch.sin(a)
    m = 1.0 / mult if inverse else mult
    if inverse:
        s = -s
    half = rotary_dim // 2
    i1 = torch.arange(half) * 2 if interleaved else torch.arange(half)
    i2 = i1 + 1 if interleaved else i1 + half
    x1, x2 = y[..., i1], y[..., i2]
    y[..., i1] = m * (x1 * c - x2 * s)
    y[..., i2] = m * (x2 * c + x1 * s)
    return y


def own_cache(cache, page_table, b, length):
    """``[length, Hkv, D]`` float64 of sequence b and a mask of the tokens on good pages."""
    if page_table is None:
        return cache[b, :length].double(), torch.ones(length, dtype=torch.bool)
    page = cache.shape[1]
    rows, good = [], []
    for t in range(length):
        pid = int(page_table[b, t // page])
        fine = 0 <= pid < cache.shape[0]
        rows.append(cache[pid, t % page].double() if fine else torch.zeros_like(cache[0, 0]).double())
        good.append(fine)
    if not rows:
        return cache.new_zeros((0, *cache.shape[2:])).double(), torch.zeros(0, dtype=torch.bool)
    return torch.stack(rows), torch.tensor(good)


def attention(q, k_prefix, v_prefix, k_cache, v_cache, cache_lens, q_lens, *, page_table=None, scale=None):
    """(out, lse, sum of weights times |v|, largest sum of |scale q k|), float64, on the CPU."""
    n, hq, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    ref = k_prefix if k_prefix is not None else k_cache
    hk = ref.shape[-2]
    group = hq // hk
    out, absum = torch.zeros((n, hq, d), dtype=torch.float64), torch.zeros((n, hq, d), dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    size = 0.0
    at = 0
    for b, nb in enumerate(q_lens):
        length = 0 if k_cache is None else int(cache_lens[b])
        empty = torch.zeros((0, hk, d), dtype=torch.float64)
        kp = empty if k_prefix is None else k_prefix.double()
        vp = empty if v_prefix is None else v_prefix.double()
        if k_cache is None:
            kc, vc, good = empty, empty, torch.zeros(0, dtype=torch.bool)
        else:
            kc, good = own_cache(k_cache, page_table, b, length)
            vc, _ = own_cache(v_cache, page_table, b, length)
        p = kp.shape[0]
        for j in range(nb):
            see = torch.cat((torch.ones(p, dtype=torch.bool),
                             (torch.arange(length) <= length - nb + j) & good))
            keys, values = torch.cat((kp, kc))[see], torch.cat((vp, vc))[see]
            if keys.shape[0] == 0:
                continue
            for h in range(hq):
                kv = h // group
                x = scale * (keys[:, kv] @ q[at + j, h].double())
                size = max(size, float((keys[:, kv].abs() @ q[at + j, h].double().abs()).max()) * abs(scale))
                w = torch.softmax(x, 0)
                out[at + j, h] = w @ values[:, kv]
                absum[at + j, h] = w @ values[:, kv].abs()
                lse[at + j, h] = torch.logsumexp(x, 0)
        at += nb
    return out, lse, absum, size


def weights(q, k_cache, lse, scores, cache_lens, q_lens, *, causal=True, scale=None):
    """(out, added weights, largest sum of |scale q k|)."""
    b, s, hk, d = k_cache.shape
    hq = q.shape[1]
    group = hq // hk
    scale = d ** -0.5 if scale is None else scale
    added = torch.zeros(scores.shape, dtype=torch.float64)
    size = 0.0
    at = 0
    for i, nb in enumerate(q_lens):
        length = int(cache_lens[i])
        for j in range(nb):
            see = torch.arange(length) <= (length - nb + j if causal else length)
            for h in range(hq):
                if lse[at + j, h] == -math.inf or not see.any():
                    continue
                keys = k_cache[i, :length, h // group].double()
                x = scale * (keys @ q[at + j, h].double())
                size = max(size, float((keys.abs() @ q[at + j, h].double().abs()).max()) * abs(scale))
                w = torch.exp(x - lse[at + j, h].double())
                added[i, h // group, :length] += torch.where(see, w, torch.zeros_like(w))
        at += nb
    return scores.double() + added, added, size


def evict_indices(scores, length, budget, keep_first, keep_recent):
    """Ascending list of the tokens of one (sequence, head) that stay."""
    if length <= budget:
        return list(range(length))
    forced = [t for t in range(length) if t < keep_first or t >= length - keep_recent]
    free = [t for t in range(length) if keep_first <= t < length - keep_recent]
    value = [float(x) for x in scores]
    key = [-math.inf if math.isnan(v) else v for v in value]
    free.sort(key=lambda t: (-key[t], t))
    return sorted(forced + free[:budget - len(forced)])
