"""GPU tests of shared_prefix_attention and accumulate_attention_weights against the float64 oracle.

Tolerances, with u = eps / 2 of the 16-bit type, Q the largest sum of |scale q k| over a score's
products and n the tokens a row sees:

* a score is a sum of D exact products in fp32, one multiplication behind it:
  ds = (D + 4) 2^-23 Q; exp2 and the maximum's subtraction add 2^-21;
* a weight goes into the product with V as 16 bits (u), sums over tokens are fp32 ((n + 32) 2^-23):
  |out - o| <= (u + 2 ds + 2^-20 + 2 (n + 32) 2^-23) sum w |v| + u |o| (the output's rounding);
* lse: ds + (n + 32) 2^-23 + 2^-22 |lse|;
* an added weight: relative ds + 2^-21 + 2^-22 |lse|, sums (rows + 8) 2^-23.
"""

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


class Case:
    """Inputs on the GPU; caches in the model layout, seen token-major."""

    def __init__(self, seed, dtype, q_lens, lens, hq, hk, d, prefix, cap, page=0):
        g = torch.Generator().manual_seed(seed)

        def rand(*shape, scale=1.0):
            return (scale * torch.randn(shape, generator=g)).to(dtype).to(DEV)

        self.q_lens, self.lens = list(q_lens), list(lens)
        b, n = len(q_lens), sum(q_lens)
        self.q = rand(n, hq, d, scale=1.5)
        self.kp = self.vp = None
        if prefix is not None:
            self.kp, self.vp = (rand(hk, prefix + 3, d).transpose(0, 1)[:prefix] for _ in range(2))
        self.kc = self.vc = self.table = None
        if cap is not None and page:
            per = -(-cap // page)
            self.kc, self.vc = rand(b * per + 2, page, hk, d), rand(b * per + 2, page, hk, d)
            self.table = torch.randperm(b * per + 2, generator=g)[:b * per].view(b, per).to(torch.int32).to(DEV)
        elif cap is not None:
            self.kc, self.vc = (rand(b, hk, cap, d).transpose(1, 2) for _ in range(2))

    def lens_t(self):
        return None if self.kc is None else torch.tensor(self.lens, dtype=torch.int32, device=DEV)

    def run(self, scb, **kw):
        given = {} if self.kc is None else dict(q_lens=self.q_lens)
        return scb.shared_prefix_attention(self.q, self.kp, self.vp, self.kc, self.vc, self.lens_t(),
                                           page_table=self.table, **{**given, **kw})

    def check(self, ref, out, lse, scale=None):
        cpu = [None if x is None else x.cpu() for x in (self.q, self.kp, self.vp, self.kc, self.vc)]
        q_lens = self.q_lens if self.kc is not None else [self.q.shape[0]]
        want, wlse, absum, size = ref.attention(*cpu, self.lens, q_lens, scale=scale,
                                                page_table=None if self.table is None else self.table.cpu())
        d = self.q.shape[2]
        n = (0 if self.kp is None else self.kp.shape[0]) + max([0] + self.lens)
        u = torch.finfo(self.q.dtype).eps / 2
        ds = (d + 4) * 2.0 ** -23 * size
        tiny = torch.finfo(self.q.dtype).tiny
        tol = (u + 2 * ds + 2.0 ** -20 + 2 * (n + 32) * 2.0 ** -23) * absum + u * want.abs() + u * tiny
        err = (out.cpu().double() - want).abs()
        assert (err <= tol).all(), f"out: {err.max()}, {(err > tol).sum()} of {err.numel()} off"
        none = torch.isinf(wlse)
        assert (lse.cpu()[none] == -math.inf).all() and (out.cpu()[none] == 0).all()
        tl = ds + (n + 32) * 2.0 ** -23 + 2.0 ** -22 * wlse[~none].abs()
        el = (lse.cpu().double()[~none] - wlse[~none]).abs()
        assert (el <= tl).all(), f"lse: {el.max()}"


SHAPES = [
    # q_lens, lens, hq, hk, d, prefix, cap, page
    ([1], [1], 1, 1, 64, 1, 1, 0),
    ([1, 1, 1], [5, 1, 9], 8, 2, 128, 100, 9, 0),
    ([1, 1, 1, 1], [0, 3, 17, 64], 28, 4, 128, 129, 70, 16),
    ([1] * 5, [33, 2, 40, 0, 7], 4, 4, 64, 77, 48, 8),
    ([3, 3], [3, 50], 6, 2, 64, 200, 50, 0),
    ([7, 1, 12], [20, 1, 12], 8, 1, 128, 65, 33, 7),
    ([5, 9], [2, 30], 4, 2, 128, 40, 30, 0),      # more queries than cached tokens
    ([40, 13], [45, 200], 8, 2, 128, 150, 200, 0),
    ([130], [130], 4, 1, 64, 67, 130, 0),
    ([2, 2], [70, 70], 3, 3, 80, 31, 70, 64),
    ([4], [9], 10, 2, 256, 90, 12, 0),
    ([1, 1], [300, 257], 5, 1, 96, 300, 300, 128),
    ([1, 1], [10, 10], 16, 1, 8, 20, 10, 0),
    ([1, 1], [130, 77], 8, 1, 256, 70, 140, 16),    # eight rows and fewer
    ([2, 1, 2], [65, 0, 3], 8, 2, 128, 130, 70, 24),
    ([1, 1, 1], [64, 200, 1], 5, 1, 40, 0, 200, 0),
    ([1] * 3, [1, 70, 129], 24, 2, 128, None, 130, 0),
    ([17, 31], [60, 31], 12, 4, 128, None, 64, 0),  # no prefix
    ([1, 1, 1], [0, 0, 0], 4, 2, 64, 0, 5, 0),      # nothing to see at all
    # many rows of a KV head: 256-row tiles
    ([64, 3, 70], [64, 2, 300], 8, 2, 128, 257, 300, 0),
    ([100, 1, 33], [90, 1, 40], 6, 2, 80, 129, 100, 24),
    ([65], [65], 4, 1, 96, None, 80, 0),
    ([128, 128], [128, 140], 2, 1, 64, 128, 140, 7),
    ([257], [0], 1, 1, 128, 0, 4, 0),               # rows that see nothing
    ([1] * 40, list(range(40)), 14, 2, 128, 700, 40, 8),
    ([1] * 70, [3] * 70, 4, 4, 64, 300, 3, 0),
    ([100] * 2 + [7, 0, 64] + [1] * 35 + [80], [100] * 2 + [9, 0, 70] + [3] * 35 + [300], 8, 2, 64, 400, 300, 0),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_oracle(scb, ref, dtype, shape):
    c = Case(11, dtype, *shape)
    out, lse = c.run(scb)
    c.check(ref, out, lse)
    assert scb.paged_status(DEV) == 0


@pytest.mark.parametrize("n,hq,hk,d", [(1, 8, 8, 64), (5, 16, 2, 128), (90, 7, 1, 128), (300, 2, 1, 64), (70, 2, 2, 40)])
def test_prefix_alone(scb, ref, n, hq, hk, d):
    c = Case(12, torch.bfloat16, [n], [0], hq, hk, d, 333, None)
    c.check(ref, *c.run(scb))


@pytest.mark.parametrize("n", [2, 60])
def test_scales(scb, ref, n):
    for scale in (0.0, -0.2, 1.0):
        c = Case(13, torch.float16, [n, n], [n + 7, n + 2], 4, 2, 64, 50, n + 7)
        c.check(ref, *c.run(scb, scale=scale), scale=scale)


def test_uniform_device_starts_and_padding_rows(scb, ref):
    c = Case(14, torch.bfloat16, [3, 1, 6], [10, 4, 6], 8, 2, 128, 70, 12)
    want = c.run(scb)
    pad = torch.cat((c.q, torch.full_like(c.q[:5], float("nan"))))
    out = torch.full_like(pad, 5.0)
    cu = torch.tensor([0, 3, 4, 10], dtype=torch.int32, device=DEV)
    o, lse = scb.shared_prefix_attention(pad, c.kp, c.vp, c.kc, c.vc, c.lens_t(), cu_q_lens=cu, max_q_len=6,
                                         out=out)
    assert o is out and (out[10:] == 5).all()  # rows behind the last sequence stay
    c.check(ref, out[:10], lse[:10])
    c.check(ref, *want)
    # host lengths, host list, and the same for every sequence
    c2 = Case(15, torch.float16, [4, 4], [9, 5], 4, 2, 64, 20, 9)
    a = scb.shared_prefix_attention(c2.q, c2.kp, c2.vp, c2.kc, c2.vc, [9, 5])
    b = scb.shared_prefix_attention(c2.q, c2.kp, c2.vp, c2.kc, c2.vc, c2.lens_t(), q_lens=torch.tensor([4, 4]))
    assert bits_equal(a[0], b[0]) and bits_equal(a[1], b[1])
    full = scb.shared_prefix_attention(c2.q, c2.kp, c2.vp, c2.kc, c2.vc)
    c2.lens = [9, 9]
    c2.check(ref, *full)


@pytest.mark.parametrize("page", [0, 8])
@pytest.mark.parametrize("q_len", [1, 40])
def test_nothing_is_read_behind_the_lengths(scb, ref, page, q_len):
    """NaN in unused cache rows, in unused pages and behind the prefix changes nothing."""
    c = Case(16, torch.bfloat16, [q_len, q_len], [q_len + 13, q_len + 2], 8, 2, 128, 90, q_len + 30, page)
    want = c.run(scb)
    for x in (c.kc, c.vc):
        if page:
            used = torch.zeros(x.shape[:2], dtype=torch.bool)
            for b in range(2):
                for t in range(c.lens[b]):
                    used[c.table[b, t // page], t % page] = True
            x[~used.to(DEV)] = float("nan")
        else:
            for b in range(2):
                x[b, c.lens[b]:] = float("inf")
    for x in (c.kp, c.vp):
        base = x.as_strided((93, *x.shape[1:]), x.stride())
        base[90:] = float("nan")
    got = c.run(scb)
    assert bits_equal(got[0], want[0]) and bits_equal(got[1], want[1])
    c.check(ref, *got)


def test_rows_before_the_first_sequence_and_wide_device_integers(scb, ref):
    for n, d in ((2, 128), (40, 64)):  # streamed, and 256-row tiles
        c = Case(29, torch.float16, [n, n], [n + 20, n + 3], 8, 2, d, 70, n + 20, 8)
        q = torch.cat((torch.full_like(c.q[:3], float("nan")), c.q, c.q[:2]))
        out = torch.full_like(q, 5.0)
        cu = torch.tensor([3, 3 + n, 3 + 2 * n], dtype=torch.int32, device=DEV)
        _, lse = scb.shared_prefix_attention(q, c.kp, c.vp, c.kc, c.vc, c.lens_t().long(), page_table=c.table.long(),
                                             cu_q_lens=cu, max_q_len=n, out=out)
        assert (out[:3] == 5).all() and (out[-2:] == 5).all()
        c.check(ref, out[3:-2], lse[3:-2])
    # 64-bit lengths and page ids that 32 bits cannot hold are out of range, not some others
    scb.paged_status(DEV)
    lens, table = torch.tensor([2 ** 32 + 5, 43], device=DEV), c.table.long()
    table[1, 0] += 2 ** 32
    out, lse = scb.shared_prefix_attention(c.q, c.kp, c.vp, c.kc, c.vc, lens, page_table=table, q_lens=c.q_lens)
    assert scb.paged_status(DEV) == scb._lib.SC_STATUS_BAD_SEQ_LEN | scb._lib.SC_STATUS_BAD_PAGE_ID
    c.lens, c.table = [0, 43], c.table.clone()
    c.table[1, 0] = -1
    c.check(ref, out, lse)


def test_scores_that_grow_along_the_tokens(scb, ref):
    """The running maximum is passed again and again, by little and by much."""
    for n in (1, 50):
        c = Case(28, torch.bfloat16, [n, n], [n + 30, n], 8, 2, 128, 900, n + 30)
        c.kp.mul_(torch.linspace(0.1, 6, 900, device=DEV).to(torch.bfloat16)[:, None, None])
        c.check(ref, *c.run(scb))


def test_not_a_number_reaches_its_rows_alone(scb):
    c = Case(17, torch.float16, [1, 1, 1], [8, 8, 8], 4, 2, 64, 40, 8)
    want = c.run(scb)
    c.q[1] = float("nan")
    out, lse = c.run(scb)
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    for i in (0, 2):
        assert bits_equal(out[i], want[0][i]) and bits_equal(lse[i], want[1][i])
    c = Case(17, torch.float16, [1, 1, 1], [8, 8, 8], 4, 2, 64, 40, 8)
    c.kp[3, 0] = float("inf")  # scores of +-inf or NaN in KV head 0
    out, lse = c.run(scb)
    assert torch.isfinite(out[:, 2:]).all() and bits_equal(out[:, 2:], want[0][:, 2:])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [
    # q_lens, lens, hq, hk, d, prefix, cap, page
    ([2, 3], [40, 3], 8, 4, 128, 70, 40, 0),      # 8 rows a tile
    ([4, 2], [33, 2], 8, 2, 64, 70, 40, 8),       # 16
    ([9, 5], [64, 70], 8, 2, 128, None, 70, 0),   # 32
    ([6], [17], 8, 1, 256, 30, 20, 0),
    ([6, 4], [70, 3], 8, 2, 64, 30, 70, 1),       # pages of one token
    ([150, 70], [150, 300], 4, 2, 128, 130, 300, 0),  # 256-row tiles
    ([130], [129], 4, 2, 64, 20, 140, 24),
])
@pytest.mark.parametrize("expanded", [False, True])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(scb, ref, dtype, shape, expanded):
    """NaN and infinities among the values of a sequence's last tokens: earlier rows do not see them."""
    c = Case(31, dtype, *shape)
    if expanded:  # one KV head for all, by a stride of zero
        c.kc, c.vc = c.kc[..., :1, :].expand(*c.kc.shape[:-2], shape[3], -1), c.vc[..., :1, :]
    page = shape[7]
    at = lambda b, t: (int(c.table[b, t // page]), t % page) if page else (b, t)
    for b, (n, length) in enumerate(zip(c.q_lens, c.lens)):
        for t, column, v in ((length - 1, 3, math.nan), (length - 1, 5, math.inf), (length - n // 2, 5, -math.inf),
                             (length - n // 2, 17, math.inf), (length - n + 1, 20, -math.inf)):
            if 0 <= t < length:
                i, j = at(b, t)
                c.vc[i, j, 0, column] = v
    if expanded:
        c.vc = c.vc.expand(c.kc.shape)
    out, lse = c.run(scb)
    want, _, _, _ = ref.attention(*[None if x is None else x.cpu() for x in (c.q, c.kp, c.vp, c.kc, c.vc)], c.lens,
                                  c.q_lens, page_table=None if c.table is None else c.table.cpu())
    got = out.cpu().double()
    assert not torch.isfinite(want).all() and torch.isfinite(want).any()
    # bf16 weights go into the product in two pieces, w = hi + lo with |lo| <= 2^-9 w of either sign or zero:
    # hi inf + lo inf is inf - inf or inf + 0 inf, which is NaN, where lo <= 0.
    assert (torch.isfinite(got) == torch.isfinite(want)).all()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    if dtype == torch.bfloat16:
        same |= torch.isnan(got)
    assert (same | torch.isfinite(want)).all()
    # the others as if zeros stood there
    c.vc = torch.where(torch.isfinite(c.vc), c.vc, torch.zeros_like(c.vc))
    clean, clean_lse = c.run(scb)
    c.check(ref, torch.where(torch.isfinite(want).to(DEV), out, clean), lse)
    c.check(ref, clean, clean_lse)


def test_scores_of_minus_infinity_are_hidden(scb, ref):
    """A key of -inf along a positive query hides its token, as a mask of the lowest value does."""
    c = Case(18, torch.float16, [1, 1], [5, 5], 2, 1, 64, 30, 5)
    c.q.copy_(c.q.abs() + 0.1)
    want = Case(18, torch.float16, [1, 1], [5, 5], 2, 1, 64, 30, 5)
    want.q.copy_(c.q)
    c.kp[7] = -float("inf")
    keep = torch.tensor([i for i in range(30) if i != 7])
    want.kp, want.vp = want.kp[keep].contiguous(), want.vp[keep].contiguous()
    want.check(ref, *c.run(scb))
    c.kp[:] = -float("inf")
    c.kc[:] = -float("inf")
    out, lse = c.run(scb)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_bad_pages_and_lengths_are_reported(scb, ref):
    c = Case(19, torch.bfloat16, [1, 1, 1], [20, 20, 20], 4, 2, 64, 33, 24, 8)
    scb.paged_status(DEV)
    c.table[1, 1] = 10 ** 6
    c.table[2, 0] = -5
    out, lse = c.run(scb)
    assert scb.paged_status(DEV) == scb._lib.SC_STATUS_BAD_PAGE_ID
    c.check(ref, out, lse)  # their tokens count as masked
    c = Case(20, torch.bfloat16, [1, 1, 1], [20, 6, 9], 4, 2, 64, 33, 24, 8)
    lens = torch.tensor([20, 25, -1], dtype=torch.int32, device=DEV)
    out, lse = scb.shared_prefix_attention(c.q, c.kp, c.vp, c.kc, c.vc, lens, page_table=c.table)
    assert scb.paged_status(DEV) == scb._lib.SC_STATUS_BAD_SEQ_LEN
    c.lens = [20, 0, 0]
    c.check(ref, out, lse)
    # starts that run backwards or past the end give no rows of their own and no fault
    cu = torch.tensor([0, 5, 2, 3], dtype=torch.int32, device=DEV)
    scb.shared_prefix_attention(c.q, c.kp, c.vp, c.kc, c.vc, c.lens_t(), page_table=c.table, cu_q_lens=cu,
                                max_q_len=3)
    assert scb.paged_status(DEV) == scb._lib.SC_STATUS_BAD_SEQ_LEN
    # many rows
    c = Case(27, torch.float16, [50, 60], [200, 150], 4, 2, 64, 100, 200, 16)
    c.table[0, 3] = -1
    c.table[1, 9] = c.kc.shape[0]
    out, lse = c.run(scb)
    assert scb.paged_status(DEV) == scb._lib.SC_STATUS_BAD_PAGE_ID
    c.check(ref, out, lse)


@pytest.mark.parametrize("d,n,page", [(64, 30, 16), (64, 60, 16), (64, 60, 4), (128, 30, 16), (128, 60, 16)])
def test_bad_pages_among_many_tiles(scb, ref, d, n, page):
    """Every other tile of a long own cache has a bad page of its own; one and two row tiles."""
    c = Case(33, torch.bfloat16, [n, n], [2000, 1600], 8, 2, d, 300, 2048, page)
    for b in range(2):
        for tile in range(0, 16, 2):
            c.table[b, (tile * 128 + 8 * (tile + b)) // page] = -1 if tile & 2 else 10 ** 8
    scb.paged_status(DEV)
    for _ in range(5):
        out, lse = c.run(scb)
    assert scb.paged_status(DEV) == scb._lib.SC_STATUS_BAD_PAGE_ID
    c.check(ref, out, lse)


@pytest.mark.parametrize("prefix,n,d", [(1, 30, 128), (128, 24, 64), (129, 32, 128), (1500, 31, 64), (5000, 25, 128)])
def test_one_row_tile(scb, ref, prefix, n, d):
    """Up to 128 rows of a sequence: token tiles take turns."""
    for lens in ([n, n + 3, 500], [700, n, 129]):
        c = Case(34, torch.float16, [n, n, n - 2], lens, 8, 2, d, prefix, 700)
        c.kp.mul_(torch.linspace(0.2, 4, prefix, device=DEV).to(torch.float16)[:, None, None])
        c.check(ref, *c.run(scb))
    c = Case(35, torch.bfloat16, [1] * 30, [5] * 30, 8, 2, d, prefix, 8)  # a decode of up to 128 rows
    c.check(ref, *c.run(scb))


def test_strided_queries_and_outputs(scb, ref):
    c = Case(21, torch.float16, [2, 5], [30, 6], 6, 2, 64, 44, 30)
    qkv = torch.zeros((7, 10, 64), dtype=torch.float16, device=DEV)
    qkv[:, :6] = c.q
    c.q = qkv[:, :6]
    out = torch.full((7, 8, 72), 3.0, dtype=torch.float16, device=DEV)
    got, lse = c.run(scb, out=out[:, 1:7, :64])
    c.check(ref, got, lse)
    assert (out[:, 0] == 3).all() and (out[:, 7] == 3).all() and (out[..., 64:] == 3).all()
    # query rows in another order, an expanded KV head
    c.q = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    c.kp, c.vp = c.kp[:, :1].expand(-1, 2, -1), c.vp[:, :1].expand(-1, 2, -1)
    c.check(ref, *c.run(scb))


def test_repeatable_bit_for_bit_and_on_a_side_stream(scb):
    c = Case(22, torch.bfloat16, [1] * 6, [500, 3, 77, 0, 260, 511], 32, 8, 128, 3001, 512)
    out, lse = c.run(scb)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = [c.run(scb) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    for o, l in again:
        assert bits_equal(o, out) and bits_equal(l, lse)


def test_two_captured_graphs_and_new_lengths(scb, ref):
    """Lengths live on the device: a captured call follows them; two graphs keep apart."""
    cases = [Case(23 + i, torch.float16, [1, 1, 1], [4, 9, 2], 8, 2, 128, 150 + i, 40) for i in range(2)]
    graphs, outs, lens = [], [], []
    for c in cases:
        lens.append(c.lens_t())
        scb.shared_prefix_attention(c.q, c.kp, c.vp, c.kc, c.vc, lens[-1])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(scb.shared_prefix_attention(c.q, c.kp, c.vp, c.kc, c.vc, lens[-1]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for c, ln in zip(cases, lens):
        c.lens = [40, 0, 17]
        ln.copy_(torch.tensor(c.lens, dtype=torch.int32))
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        c.check(ref, *o)


def test_more_units_than_multiprocessors(scb, ref):
    """Whole rounds of units and a last one in parts."""
    q_lens = [300, 64, 1, 257, 129, 400]
    lens = [320, 64, 1, 300, 500, 401]
    c = Case(24, torch.bfloat16, q_lens, lens, 32, 32, 64, 700, 500)
    c.check(ref, *c.run(scb))


def test_long_prefix_splits(scb):
    """A long prefix against the same attention as one call per half, joined by their lse."""
    c = Case(25, torch.bfloat16, [1] * 4, [10] * 4, 16, 4, 128, 20011, 16)
    out, lse = c.run(scb)
    cut = 7777
    a = scb.shared_prefix_attention(c.q, c.kp[:cut], c.vp[:cut])
    b = scb.shared_prefix_attention(c.q, c.kp[cut:], c.vp[cut:], c.kc, c.vc, c.lens_t())
    m = torch.maximum(a[1], b[1]).double()
    wa, wb = torch.exp(a[1].double() - m), torch.exp(b[1].double() - m)
    joined = (wa[..., None] * a[0].double() + wb[..., None] * b[0].double()) / (wa + wb)[..., None]
    assert ((m + torch.log(wa + wb)) - lse.double()).abs().max() <= 1e-4  # ds + sums, as above
    # both sides round weights and outputs: 3 u of the weighted |v|, at most 3 u max |v|
    u = 2.0 ** -8
    vmax = max(float(c.vp.abs().max()), float(c.vc.abs().max()))
    assert ((joined - out.double()).abs() <= 4 * u * joined.abs() + 3 * u * vmax / math.sqrt(500)).all()


def test_attention_refusals(scb):
    c = Case(26, torch.float16, [1, 1], [4, 4], 4, 2, 64, 20, 8)
    call = scb.shared_prefix_attention
    with pytest.raises(ValueError, match="multiple of"):
        call(c.q[:, :3], c.kp, c.vp)
    with pytest.raises(TypeError, match="like q"):
        call(c.q, c.kp.to(torch.bfloat16), c.vp.to(torch.bfloat16))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        call(c.q.float(), c.kp.float(), c.vp.float())
    with pytest.raises(ValueError, match="shape"):
        call(c.q, c.kp, c.vp[:5])
    with pytest.raises(ValueError, match="together"):
        call(c.q, c.kp, None)
    with pytest.raises(ValueError, match="neither"):
        call(c.q, None, None)
    with pytest.raises(ValueError, match="multiple of 8"):
        call(c.q[..., :60], c.kp[..., :60], c.vp[..., :60])
    with pytest.raises(ValueError, match="contiguous"):
        call(c.q[..., ::2], c.kp[..., ::2], c.vp[..., ::2])
    with pytest.raises(ValueError, match="lie in"):
        call(c.q, c.kp, c.vp, c.kc, c.vc, [4, 9])
    with pytest.raises(ValueError, match="q_lens"):
        call(c.q, c.kp, c.vp, c.kc, c.vc, [4, 4], q_lens=[2, 1])
    with pytest.raises(ValueError, match="same number"):
        call(torch.cat((c.q, c.q[:1])), c.kp, c.vp, c.kc, c.vc, [4, 4])
    with pytest.raises(ValueError, match="max_q_len"):
        call(c.q, c.kp, c.vp, c.kc, c.vc, [4, 4], cu_q_lens=torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="overlap"):
        call(c.q, c.kp, c.vp, out=c.q)
    with pytest.raises(ValueError, match="finite"):
        call(c.q, c.kp, c.vp, scale=math.nan)
    with pytest.raises(RuntimeError, match="backward"):
        call(c.q.clone().requires_grad_(), c.kp, c.vp)
    with pytest.raises(ValueError, match="none given"):
        call(c.q, c.kp, c.vp, cache_lens=[1, 1])


# -- accumulated weights --------------------------------------------------------------------------
def _weights_case(scb, seed, dtype, q_lens, lens, hq, hk, d, cap, causal=True):
    c = Case(seed, dtype, q_lens, lens, hq, hk, d, 20, cap)
    _, lse = c.run(scb)
    g = torch.Generator().manual_seed(seed)
    scores = torch.rand((len(lens), hk, cap), generator=g).to(DEV)
    return c, lse, scores


def _check_weights(ref, c, lse, scores, out, causal=True):
    want, added, size = ref.weights(c.q.cpu(), c.kc.cpu(), lse.cpu(), scores.cpu(), c.lens, c.q_lens, causal=causal)
    d = c.q.shape[2]
    rows = max(c.q_lens) * c.q.shape[1]
    finite = lse[torch.isfinite(lse)]
    top = float(finite.abs().max()) if finite.numel() else 0.0
    rel = (d + 4) * 2.0 ** -23 * size + 2.0 ** -21 + 2.0 ** -22 * top + (rows + 8) * 2.0 ** -23
    tol = rel * added + 2.0 ** -24 * want.abs() + 1e-30
    err = (out.cpu().double() - want).abs()
    assert (err <= tol).all(), f"{err.max()}, {(err > tol).sum()} of {err.numel()} off"
    for b, n in enumerate(c.lens):
        assert bits_equal(out[b, :, n:], scores[b, :, n:])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_lens,lens,hq,hk,d,cap", [
    ([1], [1], 1, 1, 64, 1), ([1, 1, 1], [0, 140, 33], 8, 2, 128, 150), ([1] * 4, [7, 64, 129, 2], 28, 4, 128, 130),
    ([5, 5], [3, 80], 6, 2, 80, 80), ([20, 1, 33], [60, 9, 33], 8, 1, 64, 70), ([3], [50], 10, 2, 256, 61),
    ([70, 70], [90, 200], 8, 2, 128, 200), ([1] * 9, [1000, 0, 256, 257, 5, 300, 128, 129, 700], 14, 2, 128, 1000),
    ([150, 3], [1200, 700], 12, 4, 64, 1200), ([300], [290], 5, 1, 128, 310), ([40], [900], 7, 1, 40, 1000)])
def test_weights_match_the_oracle(scb, ref, dtype, q_lens, lens, hq, hk, d, cap):
    c, lse, scores = _weights_case(scb, 31, dtype, q_lens, lens, hq, hk, d, cap)
    out = torch.full_like(scores, -1.0)
    got = scb.accumulate_attention_weights(c.q, c.kc, lse, scores, c.lens_t(), q_lens=c.q_lens, out=out)
    assert got is out
    _check_weights(ref, c, lse, scores, out)
    # in place, with the lengths from the host
    mine = scores.clone()
    assert scb.accumulate_attention_weights(c.q, c.kc, lse, mine, c.lens, q_lens=c.q_lens) is mine
    assert bits_equal(mine, out)


def test_weights_of_pages_apart_and_expanded_heads(scb, ref):
    """Layouts that tensor maps cannot say, and more sequences than are counted in shared memory."""
    c, lse, scores = _weights_case(scb, 35, torch.bfloat16, [2, 2], [60, 31], 4, 2, 64, 64)
    c.kc = c.kc[:, :, :1].expand(-1, -1, 2, -1)
    got = scb.accumulate_attention_weights(c.q, c.kc, lse, scores, c.lens_t(), out=torch.empty_like(scores))
    _check_weights(ref, c, lse, scores, got)
    b = 1030
    c, lse, scores = _weights_case(scb, 36, torch.float16, [1] * b, [i % 9 for i in range(b)], 1, 1, 64, 8)
    got = scb.accumulate_attention_weights(c.q, c.kc, lse, scores, c.lens_t(), out=torch.empty_like(scores))
    _check_weights(ref, c, lse, scores, got)


def test_weights_of_a_prefix_sum_to_the_batch(scb, ref):
    c = Case(32, torch.bfloat16, [2, 2, 2], [9, 2, 5], 8, 2, 128, 300, 16)
    _, lse = c.run(scb)
    shared = torch.zeros((1, 2, 300), device=DEV)
    scb.accumulate_attention_weights(c.q, c.kp[None], lse, shared, causal=False)
    own = torch.zeros((3, 2, 16), device=DEV)
    scb.accumulate_attention_weights(c.q, c.kc, lse, own, c.lens_t())
    # every row's weights add up to one: 6 tokens x 4 heads of each KV head
    total = shared.double().sum((0, 2)) + own.double().sum((0, 2))
    # 24 rows of weights, each off by ds + 2^-21 + 2^-22 |lse| + sums: below 2e-4 in all
    assert (total - 24).abs().max() <= 24 * 2e-4


def test_weights_skip_unused_rows_and_strided_scores(scb, ref):
    c, lse, _ = _weights_case(scb, 33, torch.float16, [1, 1], [30, 11], 4, 2, 64, 40)
    big = torch.rand((2, 3, 48), device=DEV)
    scores = big[:, 1:, 4:44]
    before = big.clone()
    for b in range(2):
        c.kc[b, c.lens[b]:] = float("nan")
    got = scb.accumulate_attention_weights(c.q, c.kc, lse, scores, c.lens_t())
    assert got is scores
    clean = Case(33, torch.float16, [1, 1], [30, 11], 4, 2, 64, 20, 40)
    _check_weights(ref, clean, lse, before[:, 1:, 4:44], scores)
    assert bits_equal(big[:, 0], before[:, 0]) and bits_equal(big[..., :4], before[..., :4])
    assert bits_equal(big[..., 44:], before[..., 44:])


def test_weights_refusals(scb):
    c, lse, scores = _weights_case(scb, 34, torch.float16, [1, 1], [4, 4], 4, 2, 64, 8)
    call = scb.accumulate_attention_weights
    with pytest.raises(TypeError, match="float32"):
        call(c.q, c.kc, lse.half(), scores)
    with pytest.raises(ValueError, match="scores must be"):
        call(c.q, c.kc, lse, scores[..., :7])
    with pytest.raises(ValueError, match="contiguous along"):
        call(c.q, c.kc, lse, torch.zeros((2, 2, 16), device=DEV)[..., ::2])
    buf = torch.zeros(40, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        call(c.q, c.kc, lse, buf[:32].view(2, 2, 8), out=buf[8:].view(2, 2, 8))
    with pytest.raises(ValueError, match="expanded"):
        call(c.q, c.kc, lse, scores, out=torch.zeros((2, 1, 8), device=DEV).expand(2, 2, 8))
    with pytest.raises(ValueError, match="lie in"):
        call(c.q, c.kc, lse, scores, [4, 9])
