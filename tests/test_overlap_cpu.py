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
