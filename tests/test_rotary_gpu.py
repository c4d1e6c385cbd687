"""GPU tests of apply_rotary against the float64 oracle.

Tolerance per element: one rounding to the output type (eps / 2 relative), and fp32 products with
cosines whose angle is off by at most 2^-25 half turns (the conversion to fp32) and whose value
is off by 2 ulp: together below 8 * 2^-23 (|x1| + |x2|) m.
"""

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


def _partner(x, rd, interleaved):
    y = x.double().abs().clone()
    half = rd // 2
    i1 = torch.arange(half) * 2 if interleaved else torch.arange(half)
    i2 = i1 + 1 if interleaved else i1 + half
    total = y[..., i1] + y[..., i2]
    size = torch.zeros_like(y)
    size[..., i1], size[..., i2] = total, total
    return size


def check(ref, got, x, positions, freqs, mult, rd, interleaved, inverse=False):
    want = ref.rotary(x.cpu(), positions.cpu(), freqs, rotary_dim=rd, interleaved=interleaved, mult=mult,
                      inverse=inverse)
    m = 1.0 / mult if inverse else mult
    fi = torch.finfo(x.dtype)
    tol = fi.eps / 2 * want.abs() + 8 * 2.0 ** -23 * m * _partner(x.cpu(), rd, interleaved) + fi.tiny * fi.eps
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), f"{err.max()} of {tol.max()}, {(err > tol).sum()} values"
    if rd < x.shape[-1]:
        assert bits_equal(got[..., rd:], x[..., rd:])


def scalings(scb):
    return {None: None, "linear": scb.RopeScaling("linear", 4.0), "ntk": scb.RopeScaling("ntk", 8.0),
            "bands": scb.RopeScaling("bands", 8.0, original_length=8192),
            "yarn": scb.RopeScaling("yarn", 4.0, original_length=4096)}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,hq,hk,d,rd,interleaved,kind", [
    (1, 1, 1, 2, 2, False, None), (1, 32, 8, 128, 128, False, "bands"), (33, 5, 1, 128, 64, True, "yarn"),
    (7, 3, 3, 80, 40, False, "linear"), (19, 4, 2, 96, 96, True, "ntk"), (5, 2, 2, 34, 34, False, None),
    (3, 70, 10, 256, 256, False, "linear"), (130, 1, 1, 64, 32, False, None), (9, 2, 1, 128, 0, False, None),
    (4, 3, 1, 33, 32, True, None), (2, 9, 9, 512, 512, False, "bands"), (257, 2, 2, 8, 8, True, None)])
def test_matches_the_oracle(scb, ref, dtype, t, hq, hk, d, rd, interleaved, kind):
    g = torch.Generator().manual_seed(t * 1000 + d)
    q = torch.randn((t, hq, d), generator=g).to(dtype).to(DEV)
    k = torch.randn((t, hk, d), generator=g).to(dtype).to(DEV)
    pos = torch.randint(0, 200000, (t,), generator=g).to(DEV)
    s = scalings(scb)[kind]
    qo, ko = scb.apply_rotary(q, k, pos, theta=500000.0, rotary_dim=rd, interleaved=interleaved, scaling=s)
    f, mult = scb.rotary_frequencies(rd, 500000.0, s)
    check(ref, qo, q, pos, f, mult, rd, interleaved)
    check(ref, ko, k, pos, f, mult, rd, interleaved)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_far_and_negative_positions(scb, ref, dtype):
    g = torch.Generator().manual_seed(1)
    pos = torch.tensor([0, 1, -1, 1000003, 16777217, 2 ** 31 - 1, -(2 ** 31)])
    x = torch.randn((7, 2, 64), generator=g).to(dtype).to(DEV)
    f, mult = scb.rotary_frequencies(64)
    # float64 angles of positions near 2^31 are themselves off by 2^31 * 2^-53 radians: nothing.
    check(ref, scb.apply_rotary(x, None, pos.to(DEV)), x, pos, f, mult, 64, False)
    got32 = scb.apply_rotary(x, None, pos.to(torch.int32).to(DEV))
    assert bits_equal(got32, scb.apply_rotary(x, None, pos.to(DEV)))
    assert bits_equal(got32, scb.apply_rotary(x, None, pos.tolist()))


def test_model_layout_strides_and_cache_slots(scb, ref):
    g = torch.Generator().manual_seed(2)
    b, t, hq, hk, d = 3, 21, 6, 2, 128
    q = torch.randn((b, t, hq, d), generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2)
    k = torch.randn((b, t, hk, d), generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2)
    pos = torch.randint(0, 9000, (b, t), generator=g).to(DEV)
    f, mult = scb.rotary_frequencies(d)
    cache = torch.full((b, hk, 64, d), 7.0, dtype=torch.bfloat16, device=DEV)
    qo, ko = scb.apply_rotary(q, k, pos, k_out=cache[:, :, 11:11 + t])
    check(ref, qo.transpose(1, 2), q.transpose(1, 2), pos, f, mult, d, False)
    check(ref, ko.transpose(1, 2), k.transpose(1, 2), pos, f, mult, d, False)
    assert ko.data_ptr() == cache[:, :, 11:].data_ptr()
    assert (cache[:, :, :11] == 7).all() and (cache[:, :, 11 + t:] == 7).all()
    # one row of positions for every sequence; the first position as a number
    same = scb.apply_rotary(q, None, torch.arange(40, 40 + t, device=DEV))
    assert bits_equal(same, scb.apply_rotary(q, None, 40))
    check(ref, same.transpose(1, 2), q.transpose(1, 2), torch.arange(40, 40 + t).expand(b, t), f, mult, d, False)


def test_views_of_a_fused_projection_in_place(scb, ref):
    g = torch.Generator().manual_seed(3)
    t, hq, hk, d = 50, 4, 2, 64
    qkv = torch.randn((t, hq + 2 * hk, d), generator=g).to(torch.float16).to(DEV)
    before = qkv.clone()
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    pos = torch.arange(t, device=DEV) * 3
    scb.apply_rotary(q, k, pos, q_out=q, k_out=k)
    f, mult = scb.rotary_frequencies(d)
    check(ref, qkv[:, :hq], before[:, :hq], pos, f, mult, d, False)
    check(ref, qkv[:, hq:hq + hk], before[:, hq:hq + hk], pos, f, mult, d, False)
    assert bits_equal(qkv[:, hq + hk:], before[:, hq + hk:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_odd_strides_and_unaligned_views(scb, ref, interleaved):
    g = torch.Generator().manual_seed(4)
    big = torch.randn((11, 5, 131), generator=g).to(torch.float16).to(DEV)
    f, mult = scb.rotary_frequencies(64)
    pos = torch.arange(11, device=DEV)
    for x in (big[:, :, 1:65], big[:, ::2, 3:131:2], big.transpose(0, 1)[:, :, 2:66].transpose(0, 1)):
        got = scb.apply_rotary(x, None, pos, interleaved=interleaved)
        check(ref, got, x, pos, f, mult, 64, interleaved)


@pytest.mark.parametrize("kind", [None, "yarn"])
def test_inverse_returns(scb, ref, kind):
    g = torch.Generator().manual_seed(5)
    s = scalings(scb)[kind]
    x = torch.randn((40, 3, 128), generator=g).to(DEV)
    pos = torch.randint(0, 100000, (40,), generator=g).to(DEV)
    f, mult = scb.rotary_frequencies(128, scaling=s)
    turned = scb.apply_rotary(x, None, pos, scaling=s)
    back = scb.apply_rotary(turned, None, pos, scaling=s, inverse=True)
    check(ref, back, turned, pos, f, mult, 128, False, inverse=True)
    # two rotations of fp32 values: twice the products' bound
    assert ((back - x).abs() <= 40 * 2.0 ** -23 * _partner(x.cpu(), 128, False).to(DEV).float()).all()


def test_agrees_with_the_shift_of_cached_keys(scb):
    """Turning at p + delta equals turning at p and shifting the cached key by delta, up to the
    fp16 tables (2^-11) and two roundings of the shift."""
    g = torch.Generator().manual_seed(6)
    k = torch.randn((64, 8, 128), generator=g).to(torch.float16).to(DEV)
    pos = torch.arange(64, device=DEV)
    moved = scb.rope_shift_keys(scb.apply_rotary(k, None, pos), 700)
    direct = scb.apply_rotary(k, None, pos + 700)
    size = _partner(k.cpu(), 128, False).to(DEV)
    assert ((moved.double() - direct.double()).abs() <= (2 * 2.0 ** -11 + 2.0 ** -10) * size).all()


def test_empty_and_large_batches(scb, ref):
    for shape in ((0, 4, 64), (3, 0, 64)):
        assert scb.apply_rotary(torch.empty(shape, dtype=torch.float16, device=DEV), None, 5).shape == shape
    g = torch.Generator().manual_seed(7)
    x = torch.randn((4099, 1, 16), generator=g).to(torch.bfloat16).to(DEV)
    f, mult = scb.rotary_frequencies(16)
    check(ref, scb.apply_rotary(x, None, 3), x, torch.arange(3, 4102), f, mult, 16, False)


def test_captured_and_replayed(scb):
    q = torch.randn((16, 8, 128), device=DEV).to(torch.bfloat16)
    pos = torch.arange(16, device=DEV)
    out = torch.empty_like(q)
    scb.apply_rotary(q, None, pos, q_out=out)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            scb.apply_rotary(q, None, pos, q_out=out)
            with pytest.raises(RuntimeError, match="captured"):
                scb.apply_rotary(q, None, list(range(16)), q_out=out)
    pos.add_(1000)
    q.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert bits_equal(out, scb.apply_rotary(q, None, pos))


def test_refusals_on_the_gpu(scb):
    q = torch.zeros((4, 2, 64), dtype=torch.float16, device=DEV)
    with pytest.raises(TypeError, match="float16, bfloat16 or float32"):
        scb.apply_rotary(q.to(torch.float64), None, 0)
    with pytest.raises(ValueError, match="does not match"):
        scb.apply_rotary(q, q[:3], 0)
    with pytest.raises(TypeError, match="like q"):
        scb.apply_rotary(q, q.float(), 0)
    with pytest.raises(ValueError, match="rotary_dim"):
        scb.apply_rotary(q, None, 0, rotary_dim=31)
    with pytest.raises(ValueError, match="positions must be"):
        scb.apply_rotary(q, None, torch.arange(5, device=DEV))
    with pytest.raises(TypeError, match="int32 or int64"):
        scb.apply_rotary(q, None, torch.zeros(4, device=DEV))
    with pytest.raises(ValueError, match="overlap"):
        scb.apply_rotary(q[:3], None, 0, q_out=q[1:])
    with pytest.raises(ValueError, match="expanded"):
        scb.apply_rotary(q, None, 0, q_out=torch.zeros((1, 2, 64), dtype=torch.float16, device=DEV).expand(4, 2, 64))
    with pytest.raises(RuntimeError, match="backward"):
        scb.apply_rotary(q.clone().requires_grad_(), None, 0)
    with torch.no_grad():
        scb.apply_rotary(q.clone().requires_grad_(), None, 0)
