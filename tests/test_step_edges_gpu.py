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
