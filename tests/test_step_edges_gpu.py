"""GPU tests of the step operators at their edges: shared storage, broken starts, first calls inside a
capture, values that are not finite and weights far below a row's largest."""

from __future__ import annotations

import pytest
import torch

from conftest import bits_equal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None


@pytest.fixture(scope="module")
def ref():
    import importlib

    return importlib.import_module("oracle.step_oracle")


def rand(seed, *shape, dtype=torch.float16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.mark.parametrize("dim", [1, 2, 3])
def test_eviction_in_place_of_keys_and_values_in_one_buffer(scb, dim):
    """Side by side for a sequence, a token or a head."""
    shape = [2, 900, 3, 64]
    shape.insert(dim, 2)
    kv = rand(1, *shape)
    k, v = kv.select(dim, 0), kv.select(dim, 1)
    scores = torch.rand((2, 3, 900), generator=torch.Generator().manual_seed(2)).to(DEV)
    want = scb.evict_tokens(k.clone(), v.clone(), scores, 300, keep_first=2, keep_recent=9)
    behind = kv.clone()
    got = scb.evict_tokens(k, v, scores, 300, keep_first=2, keep_recent=9, k_out=k[:, :300], v_out=v[:, :300])
    assert all(bits_equal(a, b) for a, b in zip(got, want))
    assert bits_equal(k[:, 300:], behind.select(dim, 0)[:, 300:])
    assert bits_equal(v[:, 300:], behind.select(dim, 1)[:, 300:])


def test_a_rejected_draft_leaves_the_accepted_tokens_weights(scb):
    """truncate into a draft: the scores are bit for bit those of one accumulation of the accepted rows."""
    from speccache_b200.serving import SharedPrefixCache, SpecDynamicCache

    prefix = SpecDynamicCache()
    prefix.update(rand(1, 1, 2, 90, 64), rand(2, 1, 2, 90, 64), 0)
    cache = SharedPrefixCache(prefix, 3, track_weights=True)
    cache.attend(0, rand(3, 3, 8, 20, 64), rand(4, 3, 2, 20, 64), rand(5, 3, 2, 20, 64))
    before = cache.scores(0).clone()
    q, k, v = rand(6, 3, 8, 5, 64), rand(7, 3, 2, 5, 64), rand(8, 3, 2, 5, 64)
    cache.attend(0, q, k, v)
    keys = cache.own[0][0].clone()
    tq = scb.apply_rotary(q, None, 110).transpose(1, 2).reshape(15, 8, 64)
    pre = [x[0].transpose(0, 1) for x in prefix[0]]
    _, lse = scb.shared_prefix_attention(tq, *pre, *(x.transpose(1, 2) for x in cache.own[0]))
    cache.truncate(90 + 22)
    assert cache.next_position(0) == 112 and bits_equal(cache.own[0][0], keys[:, :, :22])
    two = lambda x: x.view(3, 5, *x.shape[1:])[:, :2].reshape(6, *x.shape[1:])
    want = torch.cat((before, torch.zeros((3, 2, 2), device=DEV)), -1)
    scb.accumulate_attention_weights(two(tq), keys[:, :, :22].transpose(1, 2), two(lse), want)
    assert bits_equal(cache.scores(0), want)
    cache.truncate(90 + 20)
    assert bits_equal(cache.scores(0), before) and cache.next_position(0) == 110
    cache.attend(0, q[:, :, :1], k[:, :, :1], v[:, :, :1])
    assert bits_equal(cache.own[0][0][:, :, 20], keys[:, :, 20])
