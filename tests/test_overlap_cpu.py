"""Which outputs may share storage with what: decided on the host by addresses, sizes and strides, so
checked without a GPU (the calls that pass end at a stand-in for the library)."""

from __future__ import annotations

import contextlib
import importlib
import itertools
import random

import pytest
import torch


@pytest.fixture(scope="module")
def validation(scb):
    return importlib.import_module(scb.__name__ + ".kernels.validation")


def elements(t):
    return {t.data_ptr() + t.element_size() * sum(i * s for i, s in zip(at, t.stride()))
            for at in itertools.product(*(range(n) for n in t.shape))}


def apart(validation, a, b):
    try:
        validation.require_apart("out", a, b)
    except ValueError as e:
        assert "overlap" in str(e)
        return False
    return True


def test_views_side_by_side_are_apart(validation):
    kv = torch.zeros((3, 2, 16, 4, 8), dtype=torch.float16)      # pages of keys and values
    assert apart(validation, kv[:, 0], kv[:, 1]) and apart(validation, kv[:, 1], kv[:, 0])
    assert apart(validation, kv[:, 0, :7], kv[:, 1]) and not apart(validation, kv[:, 0], kv[:, 0, 3:])
    heads = torch.zeros((5, 9, 8), dtype=torch.float16)          # q, k and v of a token
    q, k, v = heads[:, :4], heads[:, 4:6], heads[:, 6:]
    assert apart(validation, q, k) and apart(validation, k, q) and apart(validation, q, v) and apart(validation, k, v)
    assert not apart(validation, q, heads[:, 3:5]) and not apart(validation, heads[:, 3:5], q)
    pairs = torch.zeros((2, 6, 3, 2, 8), dtype=torch.bfloat16)   # a head's key next to its value
    assert apart(validation, pairs[..., 0, :], pairs[..., 1, :])
    assert apart(validation, pairs[..., 0, :].transpose(1, 2), pairs[:, :4, :, 1])
    assert not apart(validation, pairs[..., 0, :], pairs[..., 0, :])
    flat = torch.zeros(64)
    assert apart(validation, flat[:32], flat[32:]) and not apart(validation, flat[:33], flat[32:])
    assert apart(validation, flat[::2], flat[1::2]) and not apart(validation, flat[::2], flat[::4])
    assert apart(validation, flat[:0], flat)


def test_no_pair_that_shares_an_element_is_called_apart(validation):
    rng = random.Random(4)
    buf = torch.zeros(400, dtype=torch.float16)
    claimed = 0
    for _ in range(4000):
        views = []
        for _ in range(2):
            shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 3))]
            strides = [rng.choice([1, 2, 3, 4, 6, 8, 12, 24, 48]) for _ in shape]
            views.append(buf.as_strided(shape, strides, rng.randint(0, 60)))
        if apart(validation, *views):
            claimed += 1
            assert not elements(views[0]) & elements(views[1])
    assert claimed > 400


@pytest.fixture
def stand_in(scb, monkeypatch):
    """Calls on CPU tensors that pass every check end here; the names of those that did."""
    reached = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: reached.append(name) or 0

    monkeypatch.setattr(scb._lib, "load", lambda: Library())
    monkeypatch.setattr(scb._lib, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(scb._lib, "stream_handle", lambda dev: None)
    for name in ("evict", "rotary", "attention"):
        module = importlib.import_module(f"{scb.__name__}.kernels.{name}")
        monkeypatch.setattr(module, "require_cuda", lambda t: None)
        if hasattr(module, "_status_word"):
            monkeypatch.setattr(module, "_status_word", lambda dev: torch.zeros(1, dtype=torch.int32))
    return reached


def test_eviction_in_place_over_the_other_cache_is_refused(scb, stand_in):
    x, scores = torch.zeros((2, 50, 3, 64), dtype=torch.float16), torch.zeros((2, 3, 50))
    for v in (x, x.view(x.shape)):
        with pytest.raises(ValueError, match="k_out must not overlap"):
            scb.evict_tokens(x, v, scores, 20, k_out=x[:, :20])
        with pytest.raises(ValueError, match="v_out must not overlap"):
            scb.evict_tokens(x, v, scores, 20, v_out=v[:, :20])
        with pytest.raises(ValueError, match="overlap"):
            scb.evict_tokens(x, v, scores, 20, k_out=x[:, :20], v_out=v[:, :20])
    longer = torch.zeros((2, 51, 3, 64), dtype=torch.float16)  # values one token behind the keys
    with pytest.raises(ValueError, match="k_out must not overlap"):
        scb.evict_tokens(longer[:, :50], longer[:, 1:], scores, 20, k_out=longer[:, :20])
    assert not stand_in
    scb.evict_tokens(x, x, scores, 20)  # nothing in place: one tensor may be both
    kv = torch.zeros((2, 50, 2, 3, 64), dtype=torch.float16)
    k, v = kv[:, :, 0], kv[:, :, 1]
    scb.evict_tokens(k, v, scores, 20, k_out=k[:, :20], v_out=v[:, :20], scores_out=scores[..., :20])
    scb.evict_tokens(k, v, scores, 20, k_out=k[:, :20])
    assert len(stand_in) == 3


def test_rotation_in_place_over_the_other_input_is_refused(scb, stand_in):
    x = torch.zeros((6, 4, 64), dtype=torch.float16)
    for kw in (dict(q_out=x), dict(k_out=x), dict(q_out=x, k_out=x)):
        with pytest.raises(ValueError, match="overlap"):
            scb.apply_rotary(x, x, 0, **kw)
    qkv = torch.zeros((6, 8, 64), dtype=torch.float16)
    q, k = qkv[:, :4], qkv[:, 4:6]
    for both in (qkv[:, 3:5], qkv[:, :6]):  # keys that reach into the queries
        with pytest.raises(ValueError, match="q_out must not overlap"):
            scb.apply_rotary(q, both, 0, q_out=q)
    assert not stand_in
    scb.apply_rotary(x, x, 0)
    for kw in (dict(q_out=q), dict(k_out=k), dict(q_out=q, k_out=k), dict(q_out=torch.zeros_like(q), k_out=k)):
        scb.apply_rotary(q, k, 0, **kw)
    wide = qkv[None].expand(1, 6, 8, 64).transpose(1, 2)  # the model layout
    scb.apply_rotary(wide[:, :4], wide[:, 4:6], 0, q_out=wide[:, :4], k_out=wide[:, 4:6])
    assert len(stand_in) == 6
