"""Calls of the step operators that their own files do not make: caches whose offsets pass 32 bits,
prompts in captured graphs whose lengths change, and calls on two streams at once.  What is compared is
the same kernels' work on compact copies, or called eagerly, so results are equal bit for bit."""

from __future__ import annotations

import pytest
import torch

from conftest import bits_equal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None
FAR = 2 ** 31 + 2 ** 27  # elements of a buffer that 32 bits do not reach


def rand(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.fixture(scope="module")
def far():
    """Views in one long buffer: ``far(x, dim, k)`` is x with its dimension ``dim`` spread over the
    buffer, the k-th of up to four tensors that share it."""
    buf = torch.empty(FAR, dtype=torch.bfloat16, device=DEV)

    def spread(x, dim, k=0):
        inner = [1] * x.ndim
        order = [d for d in range(x.ndim) if d != dim]
        size = 1
        for d in reversed(order):
            inner[d] = size
            size *= x.shape[d]
        last = x.shape[dim] - 1
        step = (FAR - 4 * size) // last // 64 * 64
        assert step >= 4 * size and last * step >= 2 ** 31
        inner[dim] = step
        y = buf.as_strided(x.shape, inner, k * size)
        assert y.data_ptr() % 16 == 0
        y.copy_(x)
        return y

    yield spread


@pytest.mark.parametrize("n,hq,hk,d", [(1, 4, 2, 128), (1, 64, 2, 64), (3, 8, 1, 256), (60, 8, 2, 128)])
def test_attention_over_far_tokens_and_sequences(scb, far, n, hq, hk, d):
    b, p, cap = 3, 150, 90
    q = rand(1, b * n, hq, d)
    kp, vp, kc, vc = rand(2, p, hk, d), rand(3, p, hk, d), rand(4, b, cap, hk, d), rand(5, b, cap, hk, d)
    lens = torch.tensor([90, 61, 77], dtype=torch.int32, device=DEV)
    want = scb.shared_prefix_attention(q, kp, vp, kc, vc, lens)
    got = scb.shared_prefix_attention(q, far(kp, 0), far(vp, 0, 1), kc, vc, lens)
    assert bits_equal(got[0], want[0]) and bits_equal(got[1], want[1])
    got = scb.shared_prefix_attention(q, kp, vp, far(kc, 0), far(vc, 0, 1), lens)
    assert bits_equal(got[0], want[0]) and bits_equal(got[1], want[1])
    got = scb.shared_prefix_attention(q, kp, vp, far(kc, 1), far(vc, 1, 1), lens)
    assert bits_equal(got[0], want[0]) and bits_equal(got[1], want[1])
    # one KV head for all by a stride of zero: copies without tensor maps
    one = [x[..., :1, :] for x in (kp, vp, kc, vc)]
    wide = lambda xs: [x.expand(*x.shape[:-2], hk, d) for x in xs]
    want = scb.shared_prefix_attention(q, *wide(one), lens)
    for spread in ((0, 1), (2, 3)):
        mine = [far(x, 0, i & 1) if i in spread else x for i, x in enumerate(one)]
        got = scb.shared_prefix_attention(q, *wide(mine), lens)
        assert bits_equal(got[0], want[0]) and bits_equal(got[1], want[1])


@pytest.mark.parametrize("n,page", [(1, 16), (1, 3), (60, 16), (60, 3)])
def test_attention_over_far_pages(scb, far, n, page):
    b, cap, hk, d = 3, 96, 2, 128
    q = rand(1, b * n, 8, d)
    kp, vp = rand(2, 70, hk, d), rand(3, 70, hk, d)
    per = cap // page
    kc, vc = rand(4, b * per, page, hk, d), rand(5, b * per, page, hk, d)
    table = torch.randperm(b * per, generator=torch.Generator().manual_seed(6)).view(b, per).to(torch.int32).to(DEV)
    lens = [96, 61, 77]
    want = scb.shared_prefix_attention(q, kp, vp, kc, vc, lens, page_table=table)
    got = scb.shared_prefix_attention(q, kp, vp, far(kc, 0), far(vc, 0, 1), lens, page_table=table)
    assert bits_equal(got[0], want[0]) and bits_equal(got[1], want[1])


def test_weights_eviction_and_rotary_over_far_tokens(scb, far):
    b, s, hk, d = 3, 300, 2, 128
    k, v = rand(1, b, s, hk, d), rand(2, b, s, hk, d)
    scores = torch.rand((b, hk, s), generator=torch.Generator().manual_seed(3)).to(DEV)
    for n, hq in ((1, 8), (40, 8), (2, 512)):  # few rows, many, and groups that tensor maps do not hold
        q = rand(4, b * n, hq, d)
        lse = torch.full((b * n, hq), 30.0, device=DEV)
        want = scb.accumulate_attention_weights(q, k, lse, scores, out=torch.empty_like(scores))
        for dim in (0, 1):
            got = scb.accumulate_attention_weights(q, far(k, dim), lse, scores, out=torch.empty_like(scores))
            assert bits_equal(got, want)
    want = scb.evict_tokens(k, v, scores, 100, keep_first=2, keep_recent=30)
    for dim in (0, 1):
        kf, vf = far(k, dim), far(v, dim, 1)
        got = scb.evict_tokens(kf, vf, scores, 100, keep_first=2, keep_recent=30)
        assert all(bits_equal(x, y) for x, y in zip(got, want))
        mine, near = scores.clone(), v.clone()
        got = scb.evict_tokens(kf, near, mine, 100, keep_first=2, keep_recent=30, k_out=kf[:, :100],
                               v_out=near[:, :100], scores_out=mine[..., :100])
        assert all(bits_equal(x, y) for x, y in zip(got, want))
    x = rand(5, s, hk, d)
    want = scb.apply_rotary(x, None, 7)
    xf = far(x, 0)
    assert bits_equal(scb.apply_rotary(xf, None, 7), want)
    scb.apply_rotary(xf, None, 7, q_out=xf)
    assert bits_equal(xf.contiguous(), want)


@pytest.mark.parametrize("d,page", [(128, 0), (64, 16)])
def test_captured_prompts_follow_their_lengths(scb, d, page):
    """Two graphs with a workspace each, replayed side by side with other starts and lengths."""
    hq, hk, cap, most = 8, 2, 240, 200
    sets = []
    for i in range(2):
        q = rand(10 + i, 420, hq, d)
        kp, vp = rand(12 + i, 700 + i, hk, d), rand(14 + i, 700 + i, hk, d)
        table = None
        if page:
            kc, vc = rand(16 + i, 3 * cap // page, page, hk, d), rand(18 + i, 3 * cap // page, page, hk, d)
            table = torch.arange(3 * cap // page, dtype=torch.int32, device=DEV).flip(0).view(3, -1)
        else:
            kc, vc = rand(16 + i, 3, cap, hk, d), rand(18 + i, 3, cap, hk, d)
        lens = torch.tensor([200, 100, 130], dtype=torch.int32, device=DEV)
        cu = torch.tensor([0, 200, 290, 420], dtype=torch.int32, device=DEV)
        call = lambda out, q=q, kp=kp, vp=vp, kc=kc, vc=vc, lens=lens, cu=cu, table=table: scb.shared_prefix_attention(
            q, kp, vp, kc, vc, lens, cu_q_lens=cu, max_q_len=most, page_table=table, out=out)
        out = torch.zeros_like(q)
        call(out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _, lse = call(out)
        sets.append((call, out, lse, lens, cu, graph))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for starts, lengths in (([0, 1, 200, 300], [240, 199, 5]), ([0, 0, 0, 0], [1, 2, 3]), ([0, 200, 220, 420], [200, 0, 240])):
        for _, out, lse, lens, cu, _ in sets:
            cu.copy_(torch.tensor(starts, dtype=torch.int32))
            lens.copy_(torch.tensor(lengths, dtype=torch.int32))
            out.fill_(3)
        torch.cuda.synchronize()
        for _ in range(2):
            for (*_, graph), s in zip(sets, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for call, out, lse, *_ in sets:
            again = torch.full_like(out, 3)
            _, want = call(again)
            assert bits_equal(out, again) and bits_equal(lse[:starts[-1]], want[:starts[-1]])
    assert scb.paged_status(DEV) == 0


def test_calls_on_two_streams_at_once(scb):
    work = []
    for i, (n, hq, hk, d, p, cap) in enumerate([(1, 32, 8, 128, 3000, 300), (100, 8, 2, 128, 900, 130),
                                                (5, 64, 8, 64, 1500, 200), (100, 8, 4, 64, 500, 130)]):
        b = 16
        q, kp, vp = rand(20 + i, b * n, hq, d), rand(30 + i, p, hk, d), rand(40 + i, p, hk, d)
        kc, vc = rand(50 + i, b, cap, hk, d), rand(60 + i, b, cap, hk, d)
        lens = torch.randint(n, cap + 1, (b,), generator=torch.Generator().manual_seed(i)).to(torch.int32).to(DEV)
        scores = torch.zeros((b, hk, cap), device=DEV)

        def step(q=q, kp=kp, vp=vp, kc=kc, vc=vc, lens=lens, scores=scores):
            out, lse = scb.shared_prefix_attention(q, kp, vp, kc, vc, lens)
            heavy = scb.accumulate_attention_weights(q, kc, lse, scores, lens, out=torch.empty_like(scores))
            return [out, lse, heavy, *scb.evict_tokens(kc, vc, heavy, 64, lens, keep_first=1, keep_recent=8)]

        work.append((step, step()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for turn in range(6):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                step, want = work[(turn + 2 * k + k * turn) % 4]
                got.append((step(), want))
    torch.cuda.synchronize()
    for have, want in got:
        assert all(bits_equal(x, y) for x, y in zip(have, want))
