"""Calls of the step operators that host code decides on, without a GPU (what passes the checks ends at a
stand-in for the library)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from test_overlap_cpu import stand_in  # noqa: F401  (a fixture)


def calls(scb):
    """Every operator as a function of one floating input."""
    cache, scores = torch.zeros((2, 6, 2, 64), dtype=torch.float16), torch.zeros((2, 2, 6))
    q, lse = torch.zeros((2, 4, 64), dtype=torch.float16), torch.zeros((2, 4))
    return {
        "apply_rotary": (q, lambda x: scb.apply_rotary(x, None, 0)),
        "apply_rotary keys": (q, lambda x: scb.apply_rotary(q, x, 0)),
        "shared_prefix_attention": (q, lambda x: scb.shared_prefix_attention(x, cache[0], cache[0])),
        "shared_prefix_attention values": (cache, lambda x: scb.shared_prefix_attention(q, None, None, cache, x)),
        "accumulate_attention_weights": (cache, lambda x: scb.accumulate_attention_weights(q, x, lse, scores)),
        "accumulate_attention_weights lse": (lse, lambda x: scb.accumulate_attention_weights(q, cache, x, scores)),
        "evict_tokens": (cache, lambda x: scb.evict_tokens(cache, x, scores, 3)),
        "evict_tokens scores": (scores, lambda x: scb.evict_tokens(cache, cache, x, 3)),
    }


def test_calls_that_would_need_derivatives_are_refused(scb, stand_in):  # noqa: F811
    for name, (x, call) in calls(scb).items():
        call(x)
        assert stand_in
        stand_in.clear()
        with pytest.raises(RuntimeError, match="no backward"):
            call(x.clone().requires_grad_())
        with torch.no_grad():
            call(x.clone().requires_grad_())
        stand_in.clear()
        with forward_ad.dual_level():
            call(x)  # no tangent: nothing is dropped
            stand_in.clear()
            dual = forward_ad.make_dual(x.clone(), torch.ones_like(x))
            for grad in (torch.no_grad(), torch.enable_grad()):
                with grad, pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(dual)
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda y: call(y), (x.clone(),), (torch.ones_like(x),))
        assert not stand_in, name


def test_no_sequences_at_all(scb, stand_in):  # noqa: F811
    """Host lists of nothing are lengths of no sequence, not numbers of the wrong type."""
    cache, scores = torch.zeros((0, 6, 2, 64), dtype=torch.float16), torch.zeros((0, 2, 6))
    q, lse = torch.zeros((0, 4, 64), dtype=torch.float16), torch.zeros((0, 4))
    for lens in ([], None, torch.zeros(0, dtype=torch.int64)):
        r = scb.evict_tokens(cache, cache, scores, 3, lens)
        assert r.k.shape == (0, 3, 2, 64) and r.lens.shape == (0,) and r.indices.shape == (0, 2, 3)
        for q_lens in ([], None, torch.zeros(0, dtype=torch.int64)):
            out, got = scb.shared_prefix_attention(q, None, None, cache, cache, lens, q_lens=q_lens)
            assert out.shape == (0, 4, 64) and got.shape == (0, 4)
            assert scb.accumulate_attention_weights(q, cache, lse, scores, lens, q_lens=q_lens) is scores
    table = torch.zeros((0, 3), dtype=torch.int32)
    pool = torch.zeros((5, 2, 2, 64), dtype=torch.float16)
    assert scb.shared_prefix_attention(q, None, None, pool, pool, [], page_table=table, q_lens=[])[0].shape == q.shape
    assert scb.apply_rotary(q, None, []).shape == q.shape
    assert scb.apply_rotary(torch.zeros((2, 4, 0, 64)), None, [[], []]).shape == (2, 4, 0, 64)
    assert not stand_in


def test_tables_of_other_types_are_refused(scb, stand_in):  # noqa: F811
    q, pool = torch.zeros((2, 4, 64), dtype=torch.float16), torch.zeros((5, 2, 2, 64), dtype=torch.float16)
    for bad in ([[0.0, 1.5], [2.0, 3.0]], torch.zeros((2, 2)), torch.zeros((2, 2), dtype=torch.bool)):
        with pytest.raises(TypeError, match="page_table"):
            scb.shared_prefix_attention(q, None, None, pool, pool, page_table=bad)
    with pytest.raises(TypeError, match="cache_lens"):
        scb.shared_prefix_attention(q, None, None, pool, pool, [1.0, 2.0], page_table=[[0, 1], [2, 3]])
    assert not stand_in
