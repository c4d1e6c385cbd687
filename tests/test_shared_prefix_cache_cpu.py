"""What SharedPrefixCache keeps of its steps, on the CPU: lengths, positions and weights, with the
operators replaced by plain ones."""

from __future__ import annotations

import importlib

import pytest
import torch

BATCH, HEADS, KV_HEADS, DIM = 2, 4, 2, 8


@pytest.fixture
def steps(scb, monkeypatch):
    """The module with plain operators; ``steps.positions`` lists the first position of each rotation and
    ``steps.refuse`` names the operator that refuses its next call."""
    module = importlib.import_module(scb.__name__ + ".serving.shared_prefix")
    kv_injector = importlib.import_module(scb.__name__ + ".serving.kv_injector")

    class Steps:
        positions: list[int] = []
        refuse: str | None = None
        SharedPrefixCache, SpecDynamicCache = module.SharedPrefixCache, module.SpecDynamicCache

    s = Steps()
    s.positions = []

    def maybe_refuse(name):
        if s.refuse == name:
            s.refuse = None
            raise ValueError(f"{name} refused")

    def rotary(q, k, position, *, q_out, k_out, **_):
        maybe_refuse("rotary")
        s.positions.append(position)
        q_out.copy_(q)
        k_out.copy_(k + position)  # a key that tells where it was turned

    def products(q, k, n):  # in 64 bits, so that only the scores' own float32 rounds
        return torch.einsum("bnhd,bshd->bnhs", q.view(-1, n, *q.shape[1:]).double(),
                            k.repeat_interleave(HEADS // KV_HEADS, 2).double())

    def attention(q, k_prefix, v_prefix, k, v, **_):
        maybe_refuse("attention")
        n = q.shape[0] // k.shape[0]
        seen = torch.arange(k.shape[1]) <= k.shape[1] - n + torch.arange(n)[:, None]       # [n, S]
        x = products(q, k, n).masked_fill(~seen[:, None], -torch.inf)
        return q.clone(), torch.logsumexp(x, -1).reshape(-1, HEADS)

    def weights(q, k, lse, scores, cache_lens=None, *, scale=None, out=None):
        maybe_refuse("weights")
        n = q.shape[0] // k.shape[0]
        seen = torch.arange(k.shape[1]) <= k.shape[1] - n + torch.arange(n)[:, None]
        w = torch.exp(products(q, k, n) - lse.view(-1, n, HEADS, 1)).masked_fill(~seen[:, None], 0.0).sum(1)
        got = scores + w.view(w.shape[0], KV_HEADS, -1, w.shape[-1]).sum(2)
        return (scores if out is None else out).copy_(got)

    def evict(k, v, scores, budget, *, keep_first, keep_recent, k_out, v_out, scores_out):
        for x in (k, v):  # any tokens do: the last ones
            x[:, :budget] = x[:, -budget:].clone()
        scores[..., :budget] = scores[..., -budget:].clone()

    monkeypatch.setattr(module, "apply_rotary", rotary)
    monkeypatch.setattr(module, "shared_prefix_attention", attention)
    monkeypatch.setattr(module, "accumulate_attention_weights", weights)
    monkeypatch.setattr(kv_injector, "evict_tokens", evict)
    return s


def prefix(steps, n=3):
    cache = steps.SpecDynamicCache()
    x = torch.zeros((1, KV_HEADS, n, DIM))
    for layer in range(2):
        cache.update(x, x, layer)
    return cache


def step(n, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((BATCH, HEADS, n, DIM), generator=g),
            *(torch.randn((BATCH, KV_HEADS, n, DIM), generator=g) for _ in range(2)))


@pytest.mark.parametrize("operator", ["rotary", "attention", "weights"])
def test_a_refused_step_leaves_nothing_behind(steps, operator):
    cache = steps.SharedPrefixCache(prefix(steps), BATCH, track_weights=True)
    twin = steps.SharedPrefixCache(prefix(steps), BATCH, track_weights=True)
    for i, n in enumerate((4, 1, 3)):
        if i:
            before = cache.own[0][0].clone(), cache.own[0][1].clone(), cache.scores(0).clone()
            steps.refuse = operator
            with pytest.raises(ValueError, match="refused"):
                cache.attend(0, *step(n, 50))
            assert cache.get_seq_length(0) == twin.get_seq_length(0)
            assert cache.next_position(0) == twin.next_position(0)
            assert all(torch.equal(a, b) for a, b in zip(before, (*cache.own[0], cache.scores(0))))
        for c in (cache, twin):
            c.attend(0, *step(n, i))
    assert cache.get_seq_length(0) == 3 + 8 and cache.next_position(0) == 11
    assert all(torch.equal(a, b) for a, b in zip(cache.own[0], twin.own[0]))
    assert torch.equal(cache.scores(0), twin.scores(0))


def test_positions_follow_truncation_and_eviction(steps):
    cache = steps.SharedPrefixCache(prefix(steps), BATCH, track_weights=True)
    for layer in range(2):
        cache.attend(layer, *step(10, 1))
        cache.attend(layer, *step(5, 2))
    cache.own.truncate(12)  # three of the five are rejected
    assert cache.next_position(0) == cache.next_position(1) == 3 + 12
    cache.attend(0, *step(1, 3))
    assert steps.positions[-1] == 15
    cache.evict(8)
    assert cache.own.get_seq_length(0) == 8 and cache.own.evicted_tokens(0) == 5 and cache.next_position(0) == 16
    assert cache.own.evicted_tokens(1) == 4 and cache.next_position(1) == 15
    cache.attend(0, *step(4, 4))
    assert steps.positions[-1] == 16
    cache.own.truncate(9)
    assert cache.next_position(0) == 17 and cache.next_position(1) == 15
    cache.own.truncate(0)  # all over again
    assert cache.next_position(0) == cache.next_position(1) == 3 and cache.own.evicted_tokens(0) == 0
    cache.attend(1, *step(2, 5))
    assert steps.positions[-1] == 3 and cache.own.evicted_tokens(7) == 0


@pytest.mark.parametrize("accepted", [0, 1, 3, 4])
def test_a_rejected_draft_is_taken_back(steps, accepted):
    """As if only the accepted tokens had been given: lengths, positions, keys and weights."""
    cache = steps.SharedPrefixCache(prefix(steps), BATCH, track_weights=True)
    twin = steps.SharedPrefixCache(prefix(steps), BATCH, track_weights=True)
    draft = step(5, 9)
    for layer in range(2):
        for c in (cache, twin):
            c.attend(layer, *step(6, 1))
        cache.attend(layer, *draft)
        if accepted:
            twin.attend(layer, *(x[:, :, :accepted] for x in draft))
    if accepted == 3:
        cache.truncate(3 + 6 + 4)  # in two goes
    cache.truncate(3 + 6 + accepted)
    for n, seed in ((1, 3), (2, 4)):
        for layer in range(2):
            assert cache.get_seq_length(layer) == twin.get_seq_length(layer)
            assert cache.next_position(layer) == twin.next_position(layer)
            assert all(torch.equal(a, b) for a, b in zip(cache.own[layer], twin.own[layer]))
            # four steps at most, each rounded once to float32 on either side: 4 x 2 x 2^-24 = 4.8e-7
            assert torch.allclose(cache.scores(layer), twin.scores(layer), rtol=1e-6, atol=0)
            for c in (cache, twin):
                c.attend(layer, *step(n, seed))


def test_what_cannot_be_taken_back_is_refused(steps):
    cache = steps.SharedPrefixCache(prefix(steps), BATCH, track_weights=True)
    cache.attend(0, *step(4, 1))
    cache.attend(0, *step(3, 2))
    cache.attend(1, *step(70, 3))
    before = cache.scores(0).clone(), cache.scores(1).clone()
    for bad in (2, 3 + 3, 3 + 5):  # into the prefix, behind layer 0's last step, into layer 1's long one
        with pytest.raises(ValueError, match="cut|part"):
            cache.truncate(bad)
        assert cache.get_seq_length(0) == 10 and cache.get_seq_length(1) == 73
        assert torch.equal(cache.scores(0), before[0]) and torch.equal(cache.scores(1), before[1])
    cache.truncate(73)
    steps.refuse = "weights"
    with pytest.raises(ValueError, match="refused"):  # a refused step between makes no difference
        cache.attend(0, *step(40, 5))
    cache.evict(4, keep_first=0, keep_recent=0)
    with pytest.raises(ValueError, match="cut back to 4"):
        cache.truncate(3 + 3)
    cache.attend(0, *step(3, 6))
    cache.attend(1, *step(3, 6))
    cache.truncate(3 + 5)
    assert cache.own.get_seq_length(0) == cache.own.get_seq_length(1) == 5
    assert cache.next_position(0) == 3 + 7 + 1 and cache.next_position(1) == 3 + 70 + 1
    plain = steps.SharedPrefixCache(prefix(steps), BATCH)  # no weights: any length
    plain.attend(0, *step(4, 1))
    plain.attend(0, *step(3, 2))
    plain.truncate(3 + 2)
    assert plain.next_position(0) == 5 and plain.get_seq_length(0) == 5


def test_a_refused_step_does_not_spoil_the_way_back(steps):
    cache = steps.SharedPrefixCache(prefix(steps), BATCH, track_weights=True)
    twin = steps.SharedPrefixCache(prefix(steps), BATCH, track_weights=True)
    for c in (cache, twin):
        c.attend(0, *step(6, 1))
    cache.attend(0, *step(5, 2))
    steps.refuse = "weights"
    with pytest.raises(ValueError, match="refused"):
        cache.attend(0, *step(60, 5))  # its scores need more room than there was
    cache.truncate(3 + 6)
    assert torch.equal(cache.scores(0), twin.scores(0)) and cache.next_position(0) == 9
