"""GPU tests of the step operators at their edges: shared storage, broken starts, first calls inside a
capture, values that are not finite and weights far below a row's largest."""

from __future__ import annotations

import math

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


STARTS = [  # token starts, tokens a sequence at most
    ([0, 5, 2, 3], 3), ([0, 2, 4, 30], 4), ([2, 4, 3, 6], 3), ([-1, 2, 3, 5], 4), ([0, 3, 6, 4], 3),
    ([0, 1, 7, 8], 3), ([4, 4, 4, 4], 2), ([6, 1, 2, 3], 3), ([0, 2, 5, -1], 3), ([1, 3, 9, 9], 9)]


@pytest.mark.parametrize("page", [0, 16, 5])  # tensor maps twice, and copies without them
@pytest.mark.parametrize("scale,hq", [(1, 4), (12, 8), (1, 64), (40, 8)])  # streamed, tiles, one and two row tiles
@pytest.mark.parametrize("cap", [80, 0])
def test_rows_of_no_sequence_are_left_alone(scb, ref, scale, hq, page, cap):
    """Starts that decrease, leave the range of the first and the last or lie too far apart give no rows; the
    other sequences' rows are right, whatever the plan."""
    if cap == 0 and page:
        pytest.skip("no pages without tokens")
    hk, d, p = 2, 64, 70
    n = 10 * scale
    q, kp, vp = rand(1, n, hq, d), rand(2, p, hk, d), rand(3, p, hk, d)
    table = None
    if page:
        per = cap // page
        kc, vc = rand(4, 3 * per, page, hk, d), rand(5, 3 * per, page, hk, d)
        table = torch.arange(3 * per, dtype=torch.int32, device=DEV).view(3, per)
        dense = [x.view(3, cap, hk, d) for x in (kc, vc)]
    else:
        kc, vc = rand(4, 3, cap, hk, d), rand(5, 3, cap, hk, d)
        dense = [kc, vc]
    lens = [min(cap, x) for x in (80, 33, 61)]
    for starts, most in STARTS:
        starts, most = [x * scale for x in starts], most * scale
        first, last = max(starts[0], 0), min(max(starts[-1], 0), n)
        fine = [b for b in range(3)
                if first <= starts[b] <= starts[b + 1] <= last and starts[b + 1] - starts[b] <= most]
        scb.paged_status(DEV)
        # a larger call before it leaves its parts in the memory that the workspace comes from
        scb.shared_prefix_attention(q, kp, vp, kc, vc, lens, page_table=table, q_lens=[n - 2, 1, 1])
        out = torch.full_like(q, 5.0)
        _, lse = scb.shared_prefix_attention(q, kp, vp, kc, vc, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                             page_table=table, max_q_len=most, out=out,
                                             cu_q_lens=torch.tensor(starts, dtype=torch.int32, device=DEV))
        assert scb.paged_status(DEV) == (0 if len(fine) == 3 else scb._lib.SC_STATUS_BAD_SEQ_LEN)
        claims = torch.zeros(n, dtype=torch.int32)
        for b in fine:
            claims[starts[b]:starts[b + 1]] += 1
        for b in fine:
            a, e = starts[b], starts[b + 1]
            once = claims[a:e] == 1  # rows that two sequences claim are undefined
            if a == e:
                continue
            want, wlse, absum, size = ref.attention(*(x.cpu() for x in (q[a:e], kp, vp, dense[0][b:b + 1],
                                                                        dense[1][b:b + 1])), [lens[b]], [e - a])
            # weights and outputs rounded to 2^-11 each, scores off by (64 + 4) 2^-23 of their products' sum
            ds = (d + 4) * 2.0 ** -23 * size
            tol = (2.0 ** -11 + 2 * ds + 2.0 ** -20 + 2 * (p + cap + 32) * 2.0 ** -23) * absum + 2.0 ** -11 * want.abs()
            err = ((out[a:e].cpu().double() - want).abs() - tol)[once]
            assert float(err.max()) <= 2.0 ** -25, (starts, b)
            err = ((lse[a:e].cpu().double() - wlse).abs() - 2.0 ** -22 * wlse.abs())[once]
            assert float(err.max()) <= ds + 200 * 2.0 ** -23, (starts, b)
        assert bool((out.cpu()[claims == 0] == 5).all()), starts


def test_a_status_word_made_inside_a_capture_keeps_its_bits(scb):
    """The first call on a device may be a captured one: a replay reports and does not clear."""
    import importlib

    paged = importlib.import_module(scb.__name__ + ".kernels.paged")
    q, k, v = rand(1, 3, 4, 64), rand(2, 3, 20, 2, 64), rand(3, 3, 20, 2, 64)
    lens = torch.tensor([5, 20, 9], dtype=torch.int32, device=DEV)
    scb.shared_prefix_attention(q, None, None, k, v, lens)
    torch.cuda.synchronize()
    kept = paged._STATUS.pop(DEV.index)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scb.shared_prefix_attention(q, None, None, k, v, lens)
        graph.replay()
        assert scb.paged_status(DEV, reset=False) == 0
        lens[1] = 21
        graph.replay()
        lens[1] = 20
        graph.replay()
        assert scb.paged_status(DEV) == scb._lib.SC_STATUS_BAD_SEQ_LEN
        graph.replay()
        assert scb.paged_status(DEV) == 0
        del graph
        torch.cuda.empty_cache()
        lens[1] = -1
        scb.shared_prefix_attention(q, None, None, k, v, lens)
        assert scb.paged_status(DEV) == scb._lib.SC_STATUS_BAD_SEQ_LEN
    finally:
        torch.cuda.synchronize()
        paged._STATUS[DEV.index] = kept


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hk,d,page", [
    (1, 8, 2, 128, 0), (1, 8, 2, 64, 16), (3, 8, 2, 64, 0), (3, 8, 1, 256, 0), (9, 8, 2, 128, 0),  # streamed
    (2, 8, 2, 64, 5), (9, 8, 2, 64, 5),                        # copies without tensor maps
    (1, 64, 2, 128, 0), (30, 8, 2, 64, 0), (70, 8, 2, 128, 16)])  # tiles
def test_infinite_values_that_every_row_sees(scb, ref, dtype, n, hq, hk, d, page):
    """The sum is that infinity (both signs: not a number), wherever the token lies and whichever kernel
    takes it."""
    b, p, cap = 3, 300, 240
    q, kp, vp = rand(1, b * n, hq, d, dtype=dtype), rand(2, p, hk, d, dtype=dtype), rand(3, p, hk, d, dtype=dtype)
    table = None
    if page:
        kc, vc = (rand(i, b * cap // page, page, hk, d, dtype=dtype) for i in (4, 5))
        table = torch.arange(b * cap // page, dtype=torch.int32, device=DEV).view(b, -1)
    else:
        kc, vc = (rand(i, b, cap, hk, d, dtype=dtype) for i in (4, 5))
    lens = [240, 77, 200]
    flat = vc.view(b, cap, hk, d)
    for t, column, value in ((0, 0, "inf"), (17, 1, "-inf"), (130, 2, "inf"), (299, 3, "inf"), (64, 4, "inf"),
                             (200, 4, "-inf"), (255, 5, "-inf"), (5, 6, "inf")):
        vp[t, :, column] = float(value)
    for t, column, value in ((0, 8, "inf"), (3, 9, "-inf"), (2, 10, "inf"), (5, 10, "-inf"), (4, 6, "inf")):
        flat[:, t, :, column] = float(value)
    out, _ = scb.shared_prefix_attention(q, kp, vp, kc, vc, lens, page_table=table)
    want, _, _, _ = ref.attention(*(x.cpu() for x in (q, kp, vp, kc, vc)), lens, [n] * b,
                                  page_table=None if table is None else table.cpu())
    got = out.cpu().double()
    odd = ~torch.isfinite(want)
    assert int(odd.sum()) >= 10 * b * n * hq and bool((torch.isfinite(got) == ~odd).all())
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert bool(same[odd].all()), f"{int((odd & ~same).sum())} of {int(odd.sum())}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hk,d,page", [(1, 8, 2, 128, 0), (1, 4, 2, 64, 16), (3, 8, 1, 256, 0), (9, 4, 2, 64, 0),
                                            (3, 8, 2, 128, 5)])
def test_weights_keep_more_bits_than_the_type(scb, ref, dtype, n, hq, hk, d, page):
    """Streamed weights go into the product in two pieces: 2^-16 off instead of half a step of the type.
    Outputs are rounded once; scores are off by (d + 4) 2^-23 of their products' sum."""
    b, p, cap = 2, 60 if n > 1 else 30, 160  # fewer than 64 rows of a KV head: no tiles
    q, kp, vp = rand(1, b * n, hq, d, dtype=dtype), rand(2, p, hk, d, dtype=dtype), rand(3, p, hk, d, dtype=dtype)
    table = None
    if page:
        kc, vc = (rand(i, b * cap // page, page, hk, d, dtype=dtype) for i in (4, 5))
        table = torch.arange(b * cap // page, dtype=torch.int32, device=DEV).view(b, -1)
    else:
        kc, vc = (rand(i, b, cap, hk, d, dtype=dtype) for i in (4, 5))
    out, _ = scb.shared_prefix_attention(q, kp, vp, kc, vc, page_table=table)
    want, _, absum, size = ref.attention(*(x.cpu() for x in (q, kp, vp, kc, vc)), [cap] * b, [n] * b,
                                         page_table=None if table is None else table.cpu())
    ds = (d + 4) * 2.0 ** -23 * size
    tol = (2.0 ** -16 + 2 * ds + 2.0 ** -20 + 2 * (p + cap + 32) * 2.0 ** -23) * absum
    tol += torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -26
    err = (out.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hk", [(1, 8, 2), (2, 16, 2), (1, 256, 2), (40, 8, 2), (100, 8, 2)])  # streams, tiles
@pytest.mark.parametrize("nats", [12.0, 17.0, 19.0])
@pytest.mark.parametrize("first", [True, False])
def test_many_weights_far_below_the_largest(scb, dtype, n, hq, hk, nats, first):
    """One token takes nearly all of the weight and 6,000 others e^-nats of it each: what they add, in a column
    that is zero for the first, keeps its bits."""
    b, p, cap, d = 2, 6000, n + 3, 64
    q = torch.zeros((b * n, hq, d), dtype=dtype, device=DEV)
    q[..., 0] = nats
    kp = torch.zeros((p, hk, d), dtype=dtype, device=DEV)
    vp = torch.ones_like(kp)
    at = 0 if first else p - 1
    kp[at, :, 0] = 1.0
    vp[at, :, :32] = 0.0
    kc = torch.zeros((b, cap, hk, d), dtype=dtype, device=DEV)
    kc[..., 0] = -20.0  # own tokens: e^(-21 nats) and less, nothing
    out, lse = scb.shared_prefix_attention(q, kp, vp, kc, kc, scale=1.0)
    w = math.exp(-nats)
    rest, total = (p - 1) * w, 1 + (p - 1) * w
    want = torch.full((d,), 1.0, dtype=torch.float64)
    want[:32] = rest / total
    # A weight is off by half a step of the type (float16: or 2^-33, half a step of its end
    # lifted by 2^8) and the output once more,
    # which float16 holds in steps of 2^-24 below 2^-14; the exponentials and sums by 2^-21 + p 2^-23.
    u = torch.finfo(dtype).eps / 2
    tol = (2 * u + 2.0 ** -21 + p * 2.0 ** -23) * want + 2.0 ** -25
    tol += p * 2.0 ** -33 if dtype == torch.float16 else 0.0
    err = (out.cpu().double() - want).abs().amax((0, 1))
    assert bool((err <= tol).all()), f"{err[0].item():.3g} of {rest:.3g} (most {tol[0].item():.3g})"
    assert float((lse.cpu().double() - nats - math.log(total)).abs().max()) <= 2.0 ** -20 * nats + p * 2.0 ** -23


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hk", [(1, 8, 2), (2, 16, 2), (1, 256, 2), (40, 8, 2), (100, 8, 2)])  # streams, tiles
def test_lse_keeps_its_bits(scb, dtype, n, hq, hk):
    """Equal scores of zero over up to 300 tokens: lse is ln of their number to 2^-22 of it and 2^-21, whatever
    weights are lifted by."""
    b, d = 2, 64
    q = torch.zeros((b * n, hq, d), dtype=dtype, device=DEV)
    kv = torch.ones((b, n + 20, hk, d), dtype=dtype, device=DEV)
    for p in (1, 3, 130, 200):
        kp = torch.ones((p, hk, d), dtype=dtype, device=DEV)
        out, lse = scb.shared_prefix_attention(q, kp, kp, kv, kv)
        seen = p + 21 + torch.arange(n, dtype=torch.float64).repeat(b)[:, None].expand(-1, hq)
        # sums of ones are exact; log2 and its product with ln 2 are off by 2^-23 of a value below 2^3 each
        assert float((lse.cpu().double() - torch.log(seen)).abs().max()) <= 2.0 ** -21 + 2.0 ** -22 * math.log(p + 21 + n)
        # the weights' one rounding is a factor of both sums; the output's is half a step
        assert float((out.double() - 1).abs().max()) <= torch.finfo(dtype).eps / 2 + 2.0 ** -15


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hk,page", [(1, 8, 2, 0), (2, 16, 2, 0), (2, 16, 2, 5), (1, 256, 2, 0), (40, 8, 2, 0),
                                          (100, 8, 2, 0)])  # streams, copies without tensor maps, tiles
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_far_beyond_the_weights_range(scb, dtype, n, hq, hk, page, sign):
    """Scores of up to 2^29: the largest one's value and nothing else, in float16 as in bfloat16."""
    b, p, d, cap = 2, 301, 64, n + 20
    q = torch.zeros((b * n, hq, d), dtype=dtype, device=DEV)
    q[..., 0] = 59968.0
    kp = torch.zeros((p, hk, d), dtype=dtype, device=DEV)
    kp[..., 0] = (sign * (48000.0 - 32.0 * torch.arange(p, device=DEV))).to(dtype)[:, None]
    best = 260  # a token above all others: twice the largest, or half the smallest
    kp[best, :, 0] = 65024.0 if sign > 0 else -16000.0
    vp = (torch.arange(p * d, device=DEV).view(p, 1, d) % 7).expand(p, hk, d).to(dtype).contiguous()
    shape = (b * cap // page, page, hk, d) if page else (b, cap, hk, d)
    if page:
        cap = cap // page * page
        shape = (b * cap // page, page, hk, d)
    kc = torch.zeros(shape, dtype=dtype, device=DEV)
    kc[..., 0] = -65024.0 if sign < 0 else 1000.0
    table = torch.arange(b * cap // page, dtype=torch.int32, device=DEV).view(b, -1) if page else None
    out, lse = scb.shared_prefix_attention(q, kp, vp, kc, kc, page_table=table)
    # the largest weight is a power of two, so nothing is rounded
    assert torch.equal(out, vp[best].repeat_interleave(hq // hk, 0).expand_as(out).to(dtype))
    want = float(q[0, 0, 0]) * float(kp[best, 0, 0]) / 8
    assert float((lse.double() - want).abs().max()) <= 2.0 ** -21 * abs(want)
    # scores of 2^24, 2 apart in units of log2: the parts of a split agree on what is largest
    kp[..., 0] = 0.0
    kp[5, :, 0], kp[290, :, 0] = 1024.0, 1026.0 if dtype == torch.float16 else 1032.0
    q[..., 0] = 32768.0 * sign
    if sign > 0:
        kc[..., 0] = 0.0
        out, _ = scb.shared_prefix_attention(q, kp, vp, kc, kc, page_table=table, scale=math.log(2.0) / 2)
        assert torch.equal(out, vp[290].repeat_interleave(hq // hk, 0).expand_as(out).to(dtype))
