"""GPU tests of evict_tokens: which tokens stay (against the oracle's sort), what moves (bit for
bit), and what is left alone.  Nothing is computed, so nothing has a tolerance."""

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


def make(seed, b, s, h, d, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((b, h, s, d), generator=g).to(dtype).to(DEV).transpose(1, 2) for _ in range(2))
    scores = torch.exp(2 * torch.randn((b, h, s), generator=g) - 6)
    scores[torch.rand((b, h, s), generator=g) < 0.3] = 0.0  # many equal ones
    return k, v, scores.to(DEV)


def check(ref, r, k, v, scores, budget, lens, first, recent):
    b, s, h, _ = k.shape
    sc = scores.cpu()
    idx = r.indices.cpu()
    for i in range(b):
        n = min(lens[i], budget)
        assert int(r.lens[i]) == n
        for j in range(h):
            want = ref.evict_indices(sc[i, j, :lens[i]], lens[i], budget, first, recent)
            assert idx[i, j, :n].tolist() == want
            assert (idx[i, j, n:] == -1).all()
            at = torch.tensor(want, dtype=torch.long, device=DEV)
            assert bits_equal(r.k[i, :n, j], k[i, at, j])
            assert bits_equal(r.v[i, :n, j], v[i, at, j])
            assert bits_equal(r.scores[i, j, :n], scores[i, j, at])


@pytest.mark.parametrize("b,s,h,d,budget,first,recent,lens,dtype", [
    (1, 1, 1, 8, 1, 0, 0, None, torch.float16),
    (2, 50, 3, 64, 20, 2, 5, None, torch.bfloat16),
    (3, 200, 2, 128, 64, 4, 16, [200, 63, 64], torch.float16),
    (2, 300, 1, 80, 100, 0, 0, [0, 300], torch.bfloat16),
    (1, 777, 4, 96, 333, 1, 331, None, torch.float16),
    (2, 100, 2, 64, 40, 40, 0, [100, 70], torch.float16),   # all forced
    (2, 100, 2, 64, 40, 0, 40, [100, 40], torch.float16),
    (1, 64, 2, 128, 64, 3, 3, None, torch.float16),         # nothing goes
    (1, 64, 2, 128, 90, 3, 3, None, torch.float32),         # a budget above the cache
    (2, 33, 1, 16, 0, 0, 0, None, torch.float16),           # nothing stays
    (1, 5000, 2, 64, 1111, 4, 100, None, torch.bfloat16),   # a cluster
    (1, 40000, 1, 8, 9999, 0, 7, None, torch.float16),
    (1, 60001, 9, 8, 20000, 4, 7, [59999], torch.float16),
])
def test_matches_the_oracle(scb, ref, b, s, h, d, budget, first, recent, lens, dtype):
    k, v, scores = make(s + budget, b, s, h, d, dtype)
    given = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    r = scb.evict_tokens(k, v, scores, budget, given, keep_first=first, keep_recent=recent)
    assert r.k.shape == (b, budget, h, d) and r.scores.shape == (b, h, budget)
    check(ref, r, k, v, scores, budget, lens or [s] * b, first, recent)
    for i, n in enumerate(lens or []):
        assert (r.k[i, min(n, budget):] == 0).all() and (r.scores[i, :, min(n, budget):] == 0).all()
    assert scb.paged_status(DEV) == 0


@pytest.mark.parametrize("d", [8, 64, 80, 128])
@pytest.mark.parametrize("s,budget", [(40, 17), (1000, 300), (6000, 5000)])
def test_in_place(scb, ref, d, s, budget):
    k, v, scores = make(s + d, 2, s, 3, d)
    k0, v0, s0 = k.clone(), v.clone(), scores.clone()
    r = scb.evict_tokens(k, v, scores, budget, keep_first=2, keep_recent=9, k_out=k[:, :budget],
                         v_out=v[:, :budget], scores_out=scores[..., :budget])
    assert r.k.data_ptr() == k.data_ptr()
    check(ref, r, k0, v0, s0, budget, [s, s], 2, 9)
    assert bits_equal(k[:, budget:], k0[:, budget:]) and bits_equal(v[:, budget:], v0[:, budget:])
    assert bits_equal(scores[..., budget:], s0[..., budget:])


def test_rows_behind_the_new_length_stay(scb, ref):
    k, v, scores = make(5, 3, 90, 2, 64)
    ko, vo = (torch.full((3, 2, 60, 64), 9.0, dtype=torch.float16, device=DEV).transpose(1, 2) for _ in range(2))
    so = torch.full((3, 2, 60), 9.0, device=DEV)
    lens = [90, 12, 0]
    r = scb.evict_tokens(k, v, scores, 60, lens, k_out=ko, v_out=vo, scores_out=so)
    check(ref, r, k, v, scores, 60, lens, 0, 0)
    assert (ko[1, 12:] == 9).all() and (vo[2] == 9).all() and (so[1, :, 12:] == 9).all()


def test_odd_scores(scb, ref):
    """Infinities, NaN, negative scores, both zeros, subnormals, all equal."""
    k, v, scores = make(6, 1, 500, 4, 16)
    scores[0, 0] = 0.25
    scores[0, 1, ::3] = float("nan")
    scores[0, 1, 1::3] = -float("inf")
    scores[0, 2] = torch.where(torch.arange(500, device=DEV) % 2 == 0, 0.0, -0.0)
    scores[0, 3] = torch.linspace(-3, 3, 500, device=DEV) * 1e-39
    scores[0, 3, 100] = float("inf")
    for budget in (100, 250, 400):
        r = scb.evict_tokens(k, v, scores, budget, keep_first=3, keep_recent=5)
        check(ref, r, k, v, scores, budget, [500], 3, 5)


def test_bad_lengths_are_reported(scb, ref):
    k, v, scores = make(7, 3, 50, 2, 64)
    scb.paged_status(DEV)
    lens = torch.tensor([50, 51, -2], dtype=torch.int32, device=DEV)
    r = scb.evict_tokens(k, v, scores, 20, lens)
    assert scb.paged_status(DEV) == scb._lib.SC_STATUS_BAD_SEQ_LEN
    check(ref, r, k, v, scores, 20, [50, 0, 0], 0, 0)


def test_captured_and_replayed(scb, ref):
    k, v, scores = make(8, 2, 400, 2, 64)
    lens = torch.tensor([400, 300], dtype=torch.int32, device=DEV)
    scb.evict_tokens(k, v, scores, 100, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = scb.evict_tokens(k, v, scores, 100, lens, keep_recent=8)
    scores.copy_(scores.flip(-1))
    lens.copy_(torch.tensor([350, 90], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    check(ref, r, k, v, scores, 100, [350, 90], 0, 8)


def test_refusals(scb):
    k, v, scores = make(9, 2, 50, 2, 64)
    call = scb.evict_tokens
    with pytest.raises(ValueError, match="budget"):
        call(k, v, scores, 10, keep_first=6, keep_recent=5)
    with pytest.raises(ValueError, match="does not match"):
        call(k, v[:, :49], scores, 10)
    with pytest.raises(TypeError, match="float32"):
        call(k, v, scores.half(), 10)
    with pytest.raises(ValueError, match="scores must be"):
        call(k, v, scores[:, :1], 10)
    with pytest.raises(ValueError, match="16 bytes"):
        call(k[..., :4], v[..., :4], scores, 10)
    with pytest.raises(ValueError, match="overlap"):
        call(k, v, scores, 10, k_out=k[:, 1:11])
    with pytest.raises(ValueError, match="overlap"):
        call(k, v, scores, 10, k_out=v[:, :10])
    with pytest.raises(ValueError, match="k_out must be"):
        call(k, v, scores, 10, k_out=k[:, :9])
    with pytest.raises(ValueError, match="lie in"):
        call(k, v, scores, 10, [50, 51])
    with pytest.raises(RuntimeError, match="backward"):
        call(k.clone().requires_grad_(), v, scores, 10)
    big = torch.empty((1, 1, 8), dtype=torch.float16, device=DEV).expand(400000, 1, 8)[None]
    with pytest.raises(RuntimeError, match="at most"):
        call(big.contiguous(), big.contiguous(), torch.zeros((1, 1, 400000), device=DEV), 10)
