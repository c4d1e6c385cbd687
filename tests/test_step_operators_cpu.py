"""Host-side checks of the step operators: refusals, frequencies and the C entries, no GPU."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch


def st(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _err(lib):
    return lib.sc_last_error().decode()


def test_operators_refuse_cpu_tensors(scb):
    q = torch.zeros((2, 4, 64), dtype=torch.float16)
    c = torch.zeros((2, 8, 2, 64), dtype=torch.float16)
    s = torch.zeros((2, 2, 8))
    for call in (lambda: scb.apply_rotary(q, None, 0),
                 lambda: scb.shared_prefix_attention(q, c[0], c[0]),
                 lambda: scb.accumulate_attention_weights(q, c, torch.zeros((2, 4)), s),
                 lambda: scb.evict_tokens(c, c, s, 4)):
        with pytest.raises(RuntimeError, match="CUDA device"):
            call()


def test_scaling_checks(scb):
    for bad in (dict(kind="other", factor=2.0), dict(kind="linear", factor=0.0),
                dict(kind="linear", factor=math.inf), dict(kind="bands", factor=2.0),
                dict(kind="yarn", factor=2.0), dict(kind="bands", factor=2.0, original_length=8,
                                                    low_freq_factor=4.0),
                dict(kind="yarn", factor=2.0, original_length=8, beta_fast=1.0),
                dict(kind="linear", factor=2.0, attention_factor=-1.0)):
        with pytest.raises(ValueError):
            scb.RopeScaling(**bad)
    with pytest.raises(ValueError, match="even"):
        scb.rotary_frequencies(7)
    with pytest.raises(ValueError, match="theta"):
        scb.rotary_frequencies(8, -1.0)


def test_frequencies(scb):
    f, m = scb.rotary_frequencies(128, 500000.0)
    assert f.dtype == np.float64 and m == 1.0
    assert np.allclose(f, [500000.0 ** (-2 * i / 128) for i in range(64)], rtol=1e-14)
    g, m = scb.rotary_frequencies(128, 500000.0, scb.RopeScaling("linear", 4.0))
    assert np.allclose(g, f / 4) and m == 1.0
    g, _ = scb.rotary_frequencies(128, 500000.0, scb.RopeScaling("ntk", 8.0))
    assert g[0] == f[0] and abs(g[-1] * 8 / f[-1] - 1) < 1e-12  # the slowest by the whole factor
    g, _ = scb.rotary_frequencies(128, 500000.0, scb.RopeScaling("bands", 8.0, original_length=8192))
    turns = 8192 * f / (2 * math.pi)
    assert np.array_equal(g[turns > 4], f[turns > 4]) and np.allclose(g[turns < 1] * 8, f[turns < 1])
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and ((g[mid] < f[mid]) & (g[mid] > f[mid] / 8)).all()
    g, m = scb.rotary_frequencies(128, 500000.0, scb.RopeScaling("yarn", 4.0, original_length=4096))
    assert abs(m - (0.1 * math.log(4.0) + 1)) < 1e-15
    assert g[0] == f[0] and abs(g[-1] * 4 / f[-1] - 1) < 1e-12 and (np.diff(g) < 0).all()
    _, m = scb.rotary_frequencies(128, scaling=scb.RopeScaling("yarn", 4.0, 4096, attention_factor=1.5))
    assert m == 1.5


def test_c_rotary_refusals(scb):
    lib, bad = scb._lib.load(), scb._lib.SC_ERR_INVALID_ARGUMENT
    f = (ctypes.c_double * 32)(*([0.1] * 32))
    s4 = st(0, 128, 64, 1)

    def call(batch=1, t=4, hq=2, hk=0, d=64, rd=64, q=16, qs=s4, dtype=0, freq=f, factor=1.0, out=16):
        return lib.sc_rope_apply(batch, t, hq, hk, d, rd, 0, q, qs, None, None, dtype, None, 0, None, 0, freq,
                                 factor, 0, out, s4, None, None, None)

    assert call(t=-1) == bad and call(rd=63) == bad and call(rd=66) == bad
    assert call(q=None) == bad and "null" in _err(lib)
    assert call(out=None) == bad and call(qs=None) == bad and call(freq=None) == bad
    assert call(factor=0.0) == bad and call(factor=math.nan) == bad
    assert call(dtype=7) == scb._lib.SC_ERR_INVALID_DTYPE
    assert call(d=2048, rd=0) == scb._lib.SC_ERR_UNSUPPORTED
    assert call(d=1024, rd=1024) == scb._lib.SC_ERR_UNSUPPORTED
    assert call(batch=2 ** 31 - 1, t=2 ** 62) == bad and "rows" in _err(lib)
    assert call(freq=(ctypes.c_double * 32)(*([math.inf] * 32))) == bad
    assert call(t=0) == 0 and call(hq=0) == 0


def test_c_attention_refusals(scb):
    lib, bad = scb._lib.load(), scb._lib.SC_ERR_INVALID_ARGUMENT
    size = ctypes.c_int64()

    def ws(n=8, b=2, hq=4, hk=2, d=64, nq=4, p=100, cap=10, page=10):
        return lib.sc_shared_prefix_attention_workspace(n, b, hq, hk, d, nq, p, cap, page,
                                                        ctypes.addressof(size))

    assert ws() == 0 and size.value >= 2 * 8 * 4 * 66 * 4
    assert ws(hq=5) == bad and ws(n=-1) == bad and ws(n=2 ** 62) == bad and ws(p=2 ** 40) == bad
    assert ws(d=60) == scb._lib.SC_ERR_UNSUPPORTED and ws(d=264) == scb._lib.SC_ERR_UNSUPPORTED
    assert ws(page=0) == bad
    assert lib.sc_shared_prefix_attention_workspace(8, 2, 4, 2, 64, 4, 100, 10, 10, None) == bad
    ws()
    need = size.value

    def call(n=8, b=2, hq=4, hk=2, d=64, dtype=0, q=16, qs=st(256, 64), p=100, kp=16, kps=st(128, 64),
             cap=10, kc=16, kcs=st(1280, 128, 64), page=10, cu=None, nq=4, scale=0.1, out=1 << 20, work=16,
             have=None):
        return lib.sc_shared_prefix_attention(
            n, b, hq, hk, d, dtype, q, qs, p, kp, kps, kp, kps, cap, kc, kcs, kc, kcs, None, None, 0, page, 0,
            cu, nq, scale, out, st(256, 64), None, work, need if have is None else have, None, None)

    assert call(have=need - 1) == bad and "workspace" in _err(lib)
    assert call(work=None) == bad and call(work=24) == bad
    assert call(q=None) == bad and call(out=None) == bad and call(kp=None) == bad and call(kc=None) == bad
    assert call(q=8) == bad and "16 bytes" in _err(lib)
    assert call(qs=st(256, 63)) == bad and call(kcs=st(1280, 4, 64)) == bad
    assert call(nq=3) == bad and call(scale=math.inf) == bad and call(page=0) == bad
    assert call(b=0, cu=16) == bad
    assert call(dtype=2) == scb._lib.SC_ERR_INVALID_DTYPE
    assert call(n=0, nq=0) == 0


def test_c_weights_refusals(scb):
    lib, bad = scb._lib.load(), scb._lib.SC_ERR_INVALID_ARGUMENT

    def call(n=8, b=2, hq=4, hk=2, d=64, dtype=0, q=16, qs=st(256, 64), s=10, k=16, ks=st(1280, 128, 64),
             nq=4, scale=0.1, lse=16, scores=16, out=16, status=16):
        return lib.sc_accumulate_attention_weights(
            n, b, hq, hk, d, dtype, q, qs, s, k, ks, None, None, nq, 1, scale, lse, st(4, 1), scores,
            st(20, 10), out, st(20, 10), status, None)

    assert call(n=-1) == bad and call(hq=5) == bad and call(nq=3) == bad and call(scale=math.nan) == bad
    assert call(d=12) == scb._lib.SC_ERR_UNSUPPORTED and call(dtype=2) == scb._lib.SC_ERR_INVALID_DTYPE
    assert call(q=None) == bad and call(lse=None) == bad and call(scores=None) == bad
    assert call(out=None) == bad and call(status=None) == bad and call(q=8) == bad
    assert call(ks=st(1280, 128, 60)) == bad and call(s=2 ** 31) == bad and call(n=2 ** 61, nq=2 ** 60) == bad
    assert call(s=0) == 0 and call(b=0, n=0) == 0


def test_c_evict_refusals(scb):
    lib, bad = scb._lib.load(), scb._lib.SC_ERR_INVALID_ARGUMENT
    s3 = st(5120, 128, 64)

    def call(b=1, h=2, s=40, d=64, e=2, budget=10, first=0, recent=0, k=16, ks=s3, scores=16, ko=16, idx=16,
             lens=16, status=16, so=16):
        return lib.sc_evict_tokens(b, h, s, d, e, budget, first, recent, k, ks, k, ks, scores, st(80, 40), None,
                                   0, ko, s3, ko, s3, so, st(20, 10), idx, lens, status, None)

    assert call(b=-1) == bad and call(first=6, recent=5) == bad and "budget" in _err(lib)
    assert call(first=2 ** 62, recent=2 ** 62) == bad
    assert call(e=3) == scb._lib.SC_ERR_INVALID_DTYPE
    assert call(d=4) == scb._lib.SC_ERR_UNSUPPORTED and call(s=400000) == scb._lib.SC_ERR_UNSUPPORTED
    assert call(d=2048) == scb._lib.SC_ERR_UNSUPPORTED
    assert call(k=None) == bad and call(scores=None) == bad and call(ko=None) == bad and call(idx=None) == bad
    assert call(lens=None) == bad and call(status=None) == bad and call(so=None) == bad
    assert call(k=8) == bad and call(ks=st(5120, 4, 64)) == bad and call(b=65535, h=2) == bad
    assert call(budget=2 ** 40) == bad and call(b=0) == 0
