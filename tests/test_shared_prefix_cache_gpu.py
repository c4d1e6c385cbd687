"""GPU test of the step operators as a serving loop runs them: a prefix restored by the injector,
prompts and single tokens of a batch behind it, weights added up, caches cut, decoding on.

Each operator is checked on the values it was given (the caches as they are on the GPU), with the
tolerances of its own tests, so that nothing has to be said about errors that add up.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import bits_equal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ref():
    import importlib

    return importlib.import_module("oracle.step_oracle")


def restored_prefix(layers, heads, dim, dtype):
    """Three chunks of 32 tokens, quantized, stored and restored with a shift each."""
    from speccache_b200.serving import MultiLayerKVInjector, SpecDynamicCache

    g = torch.Generator().manual_seed(3)
    inj = MultiLayerKVInjector(layers, heads, dim, device=DEV, max_blocks=4, chunk_size=32, out_dtype=dtype)
    kv = [torch.randn((96, heads, dim), generator=g).to(torch.float16).to(DEV) for _ in range(2 * layers)]
    inj.offload_multi_layer([0, 1, 2], kv[:layers], kv[layers:])
    cache = SpecDynamicCache()
    inj.reconstruct_and_inject_multi_layer(cache, [2, 0, 1], [64, 0, -10])
    inj.pipeline.synchronize()
    inj.close()
    return cache


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,rotary", [
    (torch.bfloat16, 8, 2, 128, dict()),
    (torch.float16, 6, 2, 64, dict(rotary_dim=32, interleaved=True, theta=500000.0)),
])
def test_prompt_decode_evict_decode(scb, ref, dtype, heads, kv_heads, dim, rotary):
    from speccache_b200.serving import SharedPrefixCache

    layers, batch = 2, 3
    prefix = restored_prefix(layers, kv_heads, dim, dtype)
    cache = SharedPrefixCache(prefix, batch, track_weights=True, **rotary)
    freqs, mult = scb.rotary_frequencies(rotary.get("rotary_dim", dim), rotary.get("theta", 10000.0))
    g = torch.Generator().manual_seed(5)
    seen = [0] * layers
    for step, n in enumerate([40, 1, 1, 3, 1, 1]):
        if step == 4:
            before = [(cache.own[i][0].clone(), cache.own[i][1].clone(), cache.scores(i).clone())
                      for i in range(layers)]
            cache.evict(20, keep_first=2, keep_recent=6)
            for i in range(layers):
                k0, v0, s0 = before[i]
                assert cache.own.get_seq_length(i) == 20 and cache.next_position(i) == 96 + 45
                for b in range(batch):
                    for h in range(kv_heads):
                        keep = torch.tensor(ref.evict_indices(s0[b, h].cpu(), 45, 20, 2, 6), device=DEV)
                        assert bits_equal(cache.own[i][0][b, h], k0[b, h, keep])
                        assert bits_equal(cache.own[i][1][b, h], v0[b, h, keep])
                        assert bits_equal(cache.scores(i)[b, h], s0[b, h, keep])
        for layer in range(layers):
            q = torch.randn((batch, heads, n, dim), generator=g).to(dtype).to(DEV)
            k, v = (torch.randn((batch, kv_heads, n, dim), generator=g).to(dtype).to(DEV) for _ in range(2))
            at = cache.next_position(layer)
            assert at == 96 + seen[layer]
            length = cache.own.get_seq_length(layer)
            old = cache.scores(layer).clone() if length else None
            out = cache.attend(layer, q, k, v)
            seen[layer] += n
            assert out.shape == (batch, heads, n, dim)
            # the new keys and values in their slots
            keys, values = cache.own[layer]
            assert bits_equal(values[:, :, length:], v)
            pos = torch.arange(at, at + n).expand(batch, n)
            want = ref.rotary(k.transpose(1, 2).cpu(), pos, freqs, rotary_dim=2 * len(freqs),
                              interleaved=rotary.get("interleaved", False), mult=mult).transpose(1, 2)
            size = k.cpu().double().abs().amax() * 2
            assert ((keys[:, :, length:].cpu().double() - want).abs()
                    <= U[dtype] * want.abs() + 8 * 2.0 ** -23 * size).all()
            # attention over the caches as they are, with the queries as apply_rotary turns them
            tq = scb.apply_rotary(q, None, at, **rotary).transpose(1, 2).reshape(batch * n, heads, dim)
            kp, vp = (x.cpu() for x in cache.prefix_views(layer))
            kc, vc = (x.transpose(1, 2).cpu() for x in cache.own[layer])
            total = length + n
            o, lse, absum, big = ref.attention(tq.cpu(), kp, vp, kc, vc, [total] * batch, [n] * batch)
            ds = (dim + 4) * 2.0 ** -23 * big
            tol = (U[dtype] + 2 * ds + 2.0 ** -20 + 2 * (96 + total + 32) * 2.0 ** -23) * absum + U[dtype] * o.abs()
            got = out.transpose(1, 2).reshape(batch * n, heads, dim).cpu().double()
            assert ((got - o).abs() <= tol + 1e-12).all()
            # the weights on top of the old ones
            base = torch.zeros((batch, kv_heads, total))
            if old is not None:
                base[..., :length] = old.cpu()
            w, added, _ = ref.weights(tq.cpu(), kc, lse, base, [total] * batch, [n] * batch)
            rel = 2 * ds + 2.0 ** -20 + 2.0 ** -21 * float(lse.abs().max()) + (n * heads + 8) * 2.0 ** -23
            assert ((cache.scores(layer).cpu().double() - w).abs() <= rel * added + 2.0 ** -24 * w.abs()).all()
    assert scb.paged_status(DEV) == 0


def test_without_a_prefix_or_weights(scb):
    """An empty prefix is ordinary attention; evict needs the weights."""
    from speccache_b200.serving import SharedPrefixCache, SpecDynamicCache

    cache = SharedPrefixCache(SpecDynamicCache(), 2, capacity=64)
    q = torch.randn((2, 4, 5, 64), device=DEV).half()
    k, v = torch.randn((2, 2, 5, 64), device=DEV).half(), torch.randn((2, 2, 5, 64), device=DEV).half()
    out = cache.attend(0, q, k, v)
    tq, tk = scb.apply_rotary(q, k, 0)
    x = (tq.double() @ tk.double().repeat_interleave(2, 1).transpose(-1, -2)) / math.sqrt(64)
    x = x.masked_fill(torch.ones(5, 5, dtype=torch.bool, device=DEV).triu(1), -math.inf)
    w = torch.softmax(x, -1)
    vv = v.double().repeat_interleave(2, 1)
    # weights and output rounded once (2^-11 each), scores off by (64 + 4) 2^-23 times at most 64
    tol = (2.0 ** -11 + 2 * 68 * 64 * 2.0 ** -23) * (w @ vv.abs()) + 2.0 ** -11 * (w @ vv).abs()
    assert ((out.double() - w @ vv).abs() <= tol).all()
    with pytest.raises(RuntimeError, match="track"):
        cache.evict(2)
    with pytest.raises(RuntimeError, match="track"):
        cache.scores(0)
    with pytest.raises(ValueError, match="batch"):
        cache.attend(0, q[:1], k[:1], v[:1])
    with pytest.raises(ValueError, match="batch"):
        SharedPrefixCache(SpecDynamicCache(), 0)


def test_evict_keeps_short_layers(scb):
    from speccache_b200.serving import SpecDynamicCache

    cache = SpecDynamicCache()
    k = torch.randn((1, 2, 10, 64), device=DEV).half()
    cache.update(k, k, 0)
    assert cache.evict(0, torch.zeros((1, 2, 10), device=DEV), 10) is None and cache.get_seq_length(0) == 10
