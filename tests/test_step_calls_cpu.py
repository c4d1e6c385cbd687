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
