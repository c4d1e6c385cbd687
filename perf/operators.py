"""The language-model operators next to the KV restore, as cases to time and to compare.

Four operators that a program calls around a restored cache:

* ``rotary``:   rotary positions of a step's queries and keys;
* ``attention``: a batch that shares a long restored prefix, each sequence with its own cache;
* ``weights``:  attention weights added up per cached token;
* ``evict``:    the cache cut to the tokens that weigh most.

``run`` computes a case in its plain form (elementary torch operations in 32 or 64 bits) or,
with ``own``, by the calls of this package.  ``exact`` computes it again in float64 from the
definitions, written apart from the plain form.
"""

from __future__ import annotations

import importlib
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
_DEVICE = "cuda"


def _package():
    return importlib.import_module("intelligent-bell_b200")


# -- cases ------------------------------------------------------------------------------------
def listed():
    return [
        # One decode step of a batch of 16: latency, wavelength-banded frequencies.
        dict(name="rotary_decode", op="rotary", batch=1, tokens=16, heads=32, kv_heads=8, dim=128,
             rotary_dim=128, interleaved=False, scaling="bands", factor=8.0, theta=500000.0,
             far=8192, layout="token", dtype="bfloat16"),
        # A whole prompt of the benchmark's length.
        dict(name="rotary_prompt", op="rotary", batch=1, tokens=8192, heads=32, kv_heads=8, dim=128,
             rotary_dim=128, interleaved=False, scaling="none", factor=1.0, theta=500000.0,
             far=0, layout="token", dtype="bfloat16"),
        # Three prompts in the model layout, half of each head rotated in adjacent pairs, at
        # positions far beyond the trained length.
        dict(name="rotary_partial", op="rotary", batch=3, tokens=1371, heads=28, kv_heads=4, dim=128,
             rotary_dim=64, interleaved=True, scaling="yarn", factor=4.0, theta=1000000.0,
             far=131072, layout="model", dtype="float16"),
        # Two users behind one short system prompt: latency.
        dict(name="attention_decode_small", op="attention", batch=2, q_len=1, ragged=True, heads=32,
             kv_heads=8, dim=128, prefix=517, cache=40, page=0, dtype="float16"),
        # 64 users behind one restored document, a decode step.
        dict(name="attention_decode", op="attention", batch=64, q_len=1, ragged=True, heads=32,
             kv_heads=8, dim=128, prefix=8192, cache=512, page=0, dtype="bfloat16"),
        # 24 users behind a long document, own tokens in pages of 64, seven query heads per KV head.
        dict(name="attention_decode_paged", op="attention", batch=24, q_len=1, ragged=True, heads=28,
             kv_heads=4, dim=128, prefix=32768, cache=2000, page=64, dtype="float16"),
        # Five draft tokens a sequence are checked at once.
        dict(name="attention_draft", op="attention", batch=16, q_len=5, ragged=False, heads=64,
             kv_heads=8, dim=64, prefix=4099, cache=700, page=0, dtype="bfloat16"),
        # Eight questions of up to 512 tokens are read behind one restored document.
        dict(name="attention_prompt", op="attention", batch=8, q_len=512, ragged=True, heads=32,
             kv_heads=8, dim=128, prefix=8192, cache=700, page=0, dtype="bfloat16"),
        # The weights of one decode step of 16 sequences.
        dict(name="weights_decode", op="weights", batch=16, q_len=1, heads=32, kv_heads=8, dim=128,
             cache=8192, dtype="bfloat16"),
        # The last 64 queries of a long prompt vote on its tokens.
        dict(name="weights_window", op="weights", batch=1, q_len=64, heads=32, kv_heads=8, dim=128,
             cache=32768, dtype="bfloat16"),
        # 16 caches of the benchmark's length are cut to a quarter.
        dict(name="evict_batch", op="evict", batch=16, kv_heads=8, dim=128, cache=8192, budget=2048,
             first=4, recent=256, ragged=True, dtype="bfloat16"),
        # One very long cache is cut to an eighth.
        dict(name="evict_long", op="evict", batch=1, kv_heads=8, dim=128, cache=131072, budget=16384,
             first=4, recent=1024, ragged=False, dtype="float16"),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def draw(rng):
    most = [work(c) for c in listed()]
    while True:  # again when a case costs more than the largest listed one
        case = _draw(rng)
        if all(work(case)[x] <= max(w[x] for w in most) for x in ("bytes", "flops")):
            return case


def _draw(rng):
    op = rng.choice(["rotary", "attention", "attention", "weights", "evict"])
    dtype = rng.choice(["float16", "bfloat16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    heads = kv_heads * group
    dim = rng.choice([64, 128])
    if op == "rotary":
        dim = rng.choice([64, 80, 128, 256])
        batch = rng.choice([1, 1, 2, 5])
        most = 8192 * 40 * 128 // (batch * (heads + kv_heads) * dim)
        return dict(op=op, batch=batch, tokens=_log(rng, 1, min(16384, most)), heads=heads,
                    kv_heads=kv_heads, dim=dim, rotary_dim=rng.choice([dim, dim, dim // 2]),
                    interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "bands", "yarn"]),
                    factor=rng.choice([2.0, 4.0, 8.0]), theta=rng.choice([10000.0, 500000.0, 1000000.0]),
                    far=rng.choice([0, 8192, 131072, 1000000]),
                    layout="model" if batch > 1 else rng.choice(["token", "model"]), dtype=dtype)
    if op == "attention":
        q_len = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 17, 512)])
        batch = _log(rng, 1, 96 if q_len <= 16 else 8)
        prefix = _log(rng, 1, 32768 if q_len <= 16 else 8192)
        return dict(op=op, batch=batch, q_len=q_len, ragged=rng.random() < 0.6, heads=heads,
                    kv_heads=kv_heads, dim=dim, prefix=prefix, cache=q_len + _log(rng, 1, 2000),
                    page=rng.choice([0, 0, 16, 64, 128]), dtype=dtype)
    if op == "weights":
        q_len = rng.choice([1, 1, _log(rng, 2, 64)])
        batch = _log(rng, 1, 24 if q_len == 1 else 2)
        return dict(op=op, batch=batch, q_len=q_len, heads=heads, kv_heads=kv_heads, dim=dim,
                    cache=q_len + _log(rng, 1, 8192 if batch > 1 else 32768), dtype=dtype)
    batch = _log(rng, 1, 24)
    cache = _log(rng, 32, 131072 // batch)
    budget = max(24, int(cache * rng.uniform(0.05, 0.6)))
    return dict(op=op, batch=batch, kv_heads=kv_heads, dim=dim, cache=cache, budget=budget,
                first=rng.choice([0, 1, 4]), recent=rng.choice([0, budget // 8, budget // 3]),
                ragged=rng.random() < 0.5, dtype=dtype)


def _lengths(case):
    """(query lengths, own cache lengths) of the case's sequences."""
    b, n, s = case["batch"], case.get("q_len", 1), case["cache"]
    if not case.get("ragged", True):
        return [n] * b, [s] * b
    rng = random.Random(1000003 * b + 1009 * n + s)
    q_lens = [n] * b if n <= 16 or case["op"] == "weights" else [rng.randint(max(1, n // 4), n) for _ in range(b)]
    q_lens[-1] = n
    if case["op"] == "evict":
        lens = [rng.randint(max(1, s // 2), s) for _ in range(b)]
    else:
        lens = [rng.randint(q, s) for q in q_lens]
    lens[0] = s
    return q_lens, lens


# -- inputs -----------------------------------------------------------------------------------
def _scaling_terms(case):
    """float64 frequencies and the factor of cos and sin, from the definitions."""
    rd, theta, factor = case["rotary_dim"], case["theta"], case["factor"]
    kind, length = case["scaling"], 8192
    i = np.arange(rd // 2, dtype=np.float64)
    if kind == "ntk":
        theta = theta * factor ** (rd / (rd - 2))
    f = theta ** (-2.0 * i / rd)
    mult = 1.0
    if kind == "linear":
        f = f / factor
    elif kind == "bands":
        # turns over the trained length: below 1 slowed down, above 4 kept, a blend between
        turns = length * f / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        f = (1 - keep) * f / factor + keep * f
    elif kind == "yarn":
        def index(turns):
            return rd * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), rd - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        f = ramp * f / factor + (1 - ramp) * f
        mult = 0.1 * math.log(factor) + 1.0
    return f, mult


def _prepare_rotary(case, g):
    dt = _DTYPES[case["dtype"]]
    b, t, d = case["batch"], case["tokens"], case["dim"]
    hq, hk = case["heads"], case["kv_heads"]
    if case["layout"] == "token":
        q = torch.randn((t, hq, d), generator=g, device=_DEVICE).to(dt)
        k = torch.randn((t, hk, d), generator=g, device=_DEVICE).to(dt)
        shape = (t,)
    else:  # [B, H, T, D] views of a projection's [B, T, H, D]
        q = torch.randn((b, t, hq, d), generator=g, device=_DEVICE).to(dt).transpose(1, 2)
        k = torch.randn((b, t, hk, d), generator=g, device=_DEVICE).to(dt).transpose(1, 2)
        shape = (b, t)
    if t <= 64 and case["layout"] == "token":  # a decode step: each token of another sequence
        pos = torch.randint(0, max(case["far"], 64), shape, generator=g, device=_DEVICE)
    else:
        start = torch.randint(0, case["far"] + 1, shape[:-1] + (1,), generator=g, device=_DEVICE)
        pos = start + torch.arange(t, device=_DEVICE)
    state = dict(case=case, q=q, k=k, positions=pos.reshape(shape))
    if own:
        scb = _package()
        kind = case["scaling"]
        if kind == "none":
            state["scaling"] = None
        elif kind in ("linear", "ntk"):
            state["scaling"] = scb.RopeScaling(kind, case["factor"])
        else:
            state["scaling"] = scb.RopeScaling(kind, case["factor"], original_length=8192)
    else:
        state["freqs"], state["mult"] = _scaling_terms(case)
    return state


def _caches(case, g, capacity, batch):
    """Token-major [B, capacity, H, D] views of model-layout caches."""
    dt = _DTYPES[case["dtype"]]
    shape = (batch, case["kv_heads"], capacity, case["dim"])
    return tuple(torch.randn(shape, generator=g, device=_DEVICE).to(dt).transpose(1, 2) for _ in range(2))


def _prepare_attention(case, g):
    dt = _DTYPES[case["dtype"]]
    q_lens, lens = _lengths(case)
    n, b, d = sum(q_lens), case["batch"], case["dim"]
    # Queries a little longer than unit variance: some tokens stand out, as in a trained model.
    q = (1.5 * torch.randn((n, case["heads"], d), generator=g, device=_DEVICE)).to(dt)
    kp, vp = (x[0] for x in _caches(case, g, case["prefix"], 1))
    state = dict(case=case, q=q, k_prefix=kp, v_prefix=vp, page_table=None,
                 cache_lens=torch.tensor(lens, dtype=torch.int32, device=_DEVICE),
                 q_lens=None if len(set(q_lens)) == 1 else q_lens)
    page = case["page"]
    if page:
        per = -(-case["cache"] // page)
        shape = (b * per, page, case["kv_heads"], d)
        state["k_cache"] = torch.randn(shape, generator=g, device=_DEVICE).to(dt)
        state["v_cache"] = torch.randn(shape, generator=g, device=_DEVICE).to(dt)
        order = torch.randperm(b * per, generator=g, device=_DEVICE)
        state["page_table"] = order.view(b, per).to(torch.int32)
    else:
        state["k_cache"], state["v_cache"] = _caches(case, g, case["cache"], b)
    return state


def _prepare_weights(case, g):
    dt = _DTYPES[case["dtype"]]
    q_lens, lens = _lengths(case)
    b, n, d, s = case["batch"], case["q_len"], case["dim"], case["cache"]
    q = (1.5 * torch.randn((b * n, case["heads"], d), generator=g, device=_DEVICE)).to(dt)
    k = _caches(case, g, s, b)[0]
    scores = torch.rand((b, case["kv_heads"], s), generator=g, device=_DEVICE) * 0.01
    lens_t = torch.tensor(lens, dtype=torch.int32, device=_DEVICE)
    # The log-sum-exp that the attention over this cache returns.
    group = case["heads"] // case["kv_heads"]
    lse = torch.empty((b * n, case["heads"]), device=_DEVICE)
    t = torch.arange(s, device=_DEVICE)
    for i in range(b):
        seen = t[None] <= lens[i] - n + torch.arange(n, device=_DEVICE)[:, None]
        for h in range(case["heads"]):
            x = q[i * n:(i + 1) * n, h].float() @ k[i, :, h // group].float().T / math.sqrt(d)
            lse[i * n:(i + 1) * n, h] = x.masked_fill(~seen, -math.inf).logsumexp(-1)
    return dict(case=case, q=q, k_cache=k, lse=lse, scores=scores, cache_lens=lens_t,
                out=torch.empty_like(scores))


def _prepare_evict(case, g):
    _, lens = _lengths(case)
    b, h, d, budget = case["batch"], case["kv_heads"], case["dim"], case["budget"]
    k, v = _caches(case, g, case["cache"], b)
    # Accumulated weights are heavy-tailed, and many tokens were never looked at.
    scores = torch.exp(2.0 * torch.randn((b, h, case["cache"]), generator=g, device=_DEVICE) - 6.0)
    scores = scores * (torch.rand(scores.shape, generator=g, device=_DEVICE) > 0.2)
    dt = _DTYPES[case["dtype"]]
    outs = [torch.zeros((b, h, budget, d), dtype=dt, device=_DEVICE).transpose(1, 2) for _ in range(2)]
    return dict(case=case, k_cache=k, v_cache=v, scores=scores, k_out=outs[0], v_out=outs[1],
                scores_out=torch.zeros((b, h, budget), device=_DEVICE),
                cache_lens=torch.tensor(lens, dtype=torch.int32, device=_DEVICE))


_PREPARE = dict(rotary=_prepare_rotary, attention=_prepare_attention, weights=_prepare_weights,
                evict=_prepare_evict)


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE)
    g.manual_seed(seed)
    return _PREPARE[case["op"]](case, g)


# -- the operators by this package ------------------------------------------------------------
def _own_rotary(st):
    c = st["case"]
    return _package().apply_rotary(st["q"], st["k"], st["positions"], theta=c["theta"],
                                   rotary_dim=c["rotary_dim"], interleaved=c["interleaved"],
                                   scaling=st["scaling"])


def _own_attention(st):
    return _package().shared_prefix_attention(
        st["q"], st["k_prefix"], st["v_prefix"], st["k_cache"], st["v_cache"], st["cache_lens"],
        q_lens=st["q_lens"], page_table=st["page_table"])


def _own_weights(st):
    return _package().accumulate_attention_weights(
        st["q"], st["k_cache"], st["lse"], st["scores"], st["cache_lens"], out=st["out"])


def _own_evict(st):
    c = st["case"]
    r = _package().evict_tokens(
        st["k_cache"], st["v_cache"], st["scores"], c["budget"], st["cache_lens"],
        keep_first=c["first"], keep_recent=c["recent"], k_out=st["k_out"], v_out=st["v_out"],
        scores_out=st["scores_out"])
    return tuple(r)


# -- the plain forms --------------------------------------------------------------------------
def _rotate_plain(x, cos, sin, c):
    """x [..., T, H, D] by cos/sin [..., T, 1, rd/2]; angles in 64 bits, products in 32."""
    rd = c["rotary_dim"]
    y = x.float()
    if c["interleaved"]:
        x1, x2 = y[..., 0:rd:2], y[..., 1:rd:2]
    else:
        x1, x2 = y[..., :rd // 2], y[..., rd // 2:rd]
    r1, r2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    turned = torch.stack((r1, r2), -1).flatten(-2) if c["interleaved"] else torch.cat((r1, r2), -1)
    return torch.cat((turned, y[..., rd:]), -1).to(x.dtype)


def _plain_rotary(st):
    c = st["case"]
    freqs = torch.as_tensor(st["freqs"], device=st["q"].device)
    angles = st["positions"].double()[..., None] * freqs
    cos, sin = (torch.cos(angles) * st["mult"]).float(), (torch.sin(angles) * st["mult"]).float()
    cos, sin = cos[..., None, :], sin[..., None, :]
    if c["layout"] == "token":
        return _rotate_plain(st["q"], cos, sin, c), _rotate_plain(st["k"], cos, sin, c)
    return tuple(_rotate_plain(x.transpose(1, 2), cos, sin, c).transpose(1, 2) for x in (st["q"], st["k"]))


def _attend_plain(q, kp, vp, kc, vc, lens):
    """q [B, n, Hq, D], prefix [P, Hkv, D], caches [B, S, Hkv, D], lens [B] -> out, lse."""
    b, n, hq, d = q.shape
    hk, s, p = kp.shape[1], kc.shape[1], kp.shape[0]
    group = hq // hk
    t = torch.arange(s, device=q.device)
    seen = t <= (lens[:, None] - n + torch.arange(n, device=q.device))[..., None]  # [B, n, S]
    seen = seen & (t < lens[:, None, None])
    hidden = ~seen.repeat_interleave(group, 1)
    out = torch.empty((b, n, hq, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((b, n, hq), dtype=torch.float32, device=q.device)
    for h in range(hk):
        qh = q[:, :, h * group:(h + 1) * group].float().reshape(b, n * group, d) / math.sqrt(d)
        x = torch.cat(((qh.reshape(-1, d) @ kp[:, h].float().T).view(b, n * group, p),
                       (qh @ kc[:, :, h].float().transpose(1, 2)).masked_fill(hidden, -math.inf)), -1)
        m = x.amax(-1, keepdim=True)
        m = torch.where(m == -math.inf, 0.0, m)
        e = torch.exp(x - m)
        total = e.sum(-1, keepdim=True)
        own_v = torch.where((t < lens[:, None])[..., None], vc[:, :, h].float(), 0.0)
        o = (e[..., :p].reshape(-1, p) @ vp[:, h].float()).view(b, n * group, d) + e[..., p:] @ own_v
        o = torch.where(total > 0, o / total, 0.0)
        out[:, :, h * group:(h + 1) * group] = o.view(b, n, group, d).to(q.dtype)
        lse[:, :, h * group:(h + 1) * group] = (m + torch.log(total)).view(b, n, group)
    return out.view(b * n, hq, d), lse.view(b * n, hq)


def _plain_attention(st):
    kc, vc, lens, table = st["k_cache"], st["v_cache"], st["cache_lens"].long(), st["page_table"]
    b = lens.shape[0]
    if table is not None:
        kc, vc = (x[table.long()].flatten(1, 2) for x in (kc, vc))
    q, kp, vp = st["q"], st["k_prefix"], st["v_prefix"]
    if st["q_lens"] is None:
        return _attend_plain(q.view(b, -1, *q.shape[1:]), kp, vp, kc, vc, lens)
    parts = [_attend_plain(x[None], kp, vp, kc[i:i + 1], vc[i:i + 1], lens[i:i + 1])
             for i, x in enumerate(q.split(st["q_lens"]))]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def _plain_weights(st):
    q, k, lse, lens = st["q"], st["k_cache"], st["lse"], st["cache_lens"].long()
    b, s, hk, d = k.shape
    n, hq = q.shape[0] // b, q.shape[1]
    group = hq // hk
    t = torch.arange(s, device=q.device)
    seen = t <= (lens[:, None] - n + torch.arange(n, device=q.device))[..., None]
    seen = (seen & (t < lens[:, None, None])).repeat_interleave(group, 1)
    added = torch.empty_like(st["scores"])
    for h in range(hk):
        pick = slice(h * group, (h + 1) * group)
        qh = q.view(b, n, hq, d)[:, :, pick].float().reshape(b, n * group, d) / math.sqrt(d)
        x = qh @ k[:, :, h].float().transpose(1, 2)
        w = torch.exp(x - lse.view(b, n, hq)[:, :, pick].reshape(b, n * group, 1))
        added[:, h] = torch.where(seen, w, 0.0).sum(1)
    return st["scores"] + added


def _plain_evict(st):
    c = st["case"]
    k, v, scores, lens = st["k_cache"], st["v_cache"], st["scores"], st["cache_lens"].long()
    b, s, h, d = k.shape
    budget = c["budget"]
    t = torch.arange(s, device=k.device)
    there = t < lens[:, None]
    forced = there & ((t < c["first"]) | (t >= (lens - c["recent"])[:, None]))
    rank = torch.where(forced, 2, torch.where(there, 1, 0))[:, None].expand(b, h, s)
    by_score = torch.sort(scores, dim=-1, descending=True, stable=True).indices
    by_rank = torch.sort(rank.gather(-1, by_score), dim=-1, descending=True, stable=True).indices
    best = by_score.gather(-1, by_rank)[..., :budget]
    n_new = torch.minimum(lens, torch.full_like(lens, budget))
    filled = torch.arange(best.shape[-1], device=k.device) < n_new[:, None, None]
    kept = torch.where(filled, best, s).sort(-1).values
    filled = kept < s
    at = torch.where(filled, kept, 0)
    rows = at.transpose(1, 2)[..., None].expand(-1, -1, -1, d)
    ok = filled.transpose(1, 2)[..., None]
    wide = at.shape[-1]
    for src, dst in ((k, st["k_out"]), (v, st["v_out"])):
        dst[:, :wide] = torch.where(ok, src.gather(1, rows), dst[:, :wide])
    st["scores_out"][..., :wide] = torch.where(filled, scores.gather(-1, at), st["scores_out"][..., :wide])
    indices = torch.full((b, h, budget), -1, dtype=torch.int32, device=k.device)
    indices[..., :wide] = torch.where(filled, kept, -1).to(torch.int32)
    return st["k_out"], st["v_out"], st["scores_out"], indices, n_new.to(torch.int32)


_OWN = dict(rotary=_own_rotary, attention=_own_attention, weights=_own_weights, evict=_own_evict)
_PLAIN = dict(rotary=_plain_rotary, attention=_plain_attention, weights=_plain_weights, evict=_plain_evict)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# -- what a pass cannot do without ------------------------------------------------------------
def work(case):
    op, d = case["op"], case["dim"]
    if op == "rotary":
        n = case["batch"] * case["tokens"]
        h = case["heads"] + case["kv_heads"]
        return {"bytes": n * (h * d * 2 * 2 + 8), "flops": n * h * case["rotary_dim"] * 3}
    q_lens, lens = _lengths(case)
    hk = case["kv_heads"]
    if op == "evict":
        kept = sum(min(x, case["budget"]) for x in lens) * hk
        return {"bytes": sum(lens) * hk * 4 + kept * (2 * 2 * d * 2 + 4 + 4), "flops": 0}
    hq, rows = case["heads"], sum(q_lens)
    pairs = sum(q * (x - q) + q * (q + 1) // 2 for q, x in zip(q_lens, lens))
    if op == "weights":
        size = rows * hq * (2 * d + 4) + sum(lens) * hk * d * 2 + case["batch"] * hk * case["cache"] * 8
        return {"bytes": size, "flops": 2 * d * hq * pairs}
    pairs += rows * case["prefix"]
    size = rows * hq * (4 * d + 4) + (case["prefix"] + sum(lens)) * hk * d * 4
    return {"bytes": size, "flops": 4 * d * hq * pairs}


# -- the definitions in 64 bits ---------------------------------------------------------------
def _exact_rotary(st):
    c = st["case"]
    freqs, mult = _scaling_terms(c)
    rd, out = c["rotary_dim"], []
    angle = st["positions"].double()[..., None] * torch.as_tensor(freqs, device=_DEVICE)
    turn = torch.polar(torch.full_like(angle, mult), angle)  # [.., T, rd/2] complex
    turn = turn.unsqueeze(-2 if c["layout"] == "token" else -3)
    for x in (st["q"], st["k"]):
        y = x.double().clone()
        if c["interleaved"]:
            z = torch.view_as_complex(y[..., :rd].reshape(*y.shape[:-1], rd // 2, 2).contiguous()) * turn
            y[..., :rd] = torch.view_as_real(z).reshape(*y.shape[:-1], rd)
        else:
            z = torch.complex(y[..., :rd // 2].contiguous(), y[..., rd // 2:rd].contiguous()) * turn
            y[..., :rd // 2], y[..., rd // 2:rd] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _own_rows(st, i, length):
    """Keys and values of sequence i's own cache, [length, Hkv, D]."""
    if st["page_table"] is None:
        return st["k_cache"][i, :length], st["v_cache"][i, :length]
    pages = st["page_table"][i].long()
    return tuple(st[x][pages].flatten(0, 1)[:length] for x in ("k_cache", "v_cache"))


def _exact_attention(st):
    c = st["case"]
    q_lens, lens = _lengths(c)
    hq, hk, d = c["heads"], c["kv_heads"], c["dim"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=_DEVICE)
    lse = torch.full(st["q"].shape[:2], -math.inf, dtype=torch.float64, device=_DEVICE)
    for h in range(hk):
        kp, vp = st["k_prefix"][:, h].double(), st["v_prefix"][:, h].double()
        at = 0
        for i, (n, length) in enumerate(zip(q_lens, lens)):
            kc, vc = _own_rows(st, i, length)
            keys, values = torch.cat((kp, kc[:, h].double())), torch.cat((vp, vc[:, h].double()))
            last = kp.shape[0] + length - n + torch.arange(n, device=_DEVICE)
            hide = torch.arange(keys.shape[0], device=_DEVICE) > last[:, None]
            for g in range(h * (hq // hk), (h + 1) * (hq // hk)):
                x = (st["q"][at:at + n, g].double() @ keys.T) * d ** -0.5
                x = x.masked_fill(hide, -math.inf)
                lse[at:at + n, g] = torch.logsumexp(x, -1)
                out[at:at + n, g] = torch.softmax(x, -1) @ values
            at += n
    return out, lse


def _exact_weights(st):
    c = st["case"]
    q_lens, lens = _lengths(c)
    hq, hk, d, n = c["heads"], c["kv_heads"], c["dim"], c["q_len"]
    total = st["scores"].double().clone()
    for i, length in enumerate(lens):
        for h in range(hq):
            kv = h * hk // hq
            x = st["k_cache"][i, :length, kv].double() @ st["q"][i * n:(i + 1) * n, h].double().T
            w = torch.exp(x * d ** -0.5 - st["lse"][i * n:(i + 1) * n, h].double())
            late = torch.arange(length, device=_DEVICE)[:, None] > length - n + torch.arange(n, device=_DEVICE)
            total[i, kv, :length] += w.masked_fill(late, 0.0).sum(1)
    return total


def _exact_evict(st):
    c = st["case"]
    _, lens = _lengths(c)
    budget, first, recent = c["budget"], c["first"], c["recent"]
    scores = st["scores"].cpu().numpy()
    b, hk, _ = scores.shape
    k, v = st["k_cache"].double(), st["v_cache"].double()
    ko = torch.zeros(st["k_out"].shape, dtype=torch.float64, device=_DEVICE)
    vo = torch.zeros_like(ko)
    so = torch.zeros((b, hk, budget), dtype=torch.float64, device=_DEVICE)
    idx = torch.full((b, hk, budget), -1, dtype=torch.int32, device=_DEVICE)
    for i, length in enumerate(lens):
        for h in range(hk):
            t = np.arange(length)
            free = (t >= first) & (t < length - recent)
            order = np.lexsort((t, -scores[i, h, :length].astype(np.float64), free))
            kept = torch.from_numpy(np.sort(order[:budget])).to(_DEVICE)
            n = kept.numel()
            ko[i, :n, h], vo[i, :n, h] = k[i, kept, h], v[i, kept, h]
            so[i, h, :n] = st["scores"][i, h, kept].double()
            idx[i, h, :n] = kept.to(torch.int32)
    new = torch.tensor([min(x, budget) for x in lens], dtype=torch.int32, device=_DEVICE)
    return ko, vo, so, idx, new


_EXACT = dict(rotary=_exact_rotary, attention=_exact_attention, weights=_exact_weights, evict=_exact_evict)


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))
