"""Attention over a paged cache at the ends of what its types hold: scores and values near the largest numbers, keys and values that are none."""
import math

import pytest
import torch

from tests import paged_oracle as oracle
from tests.test_paged_gpu import check_attention, hide, on_gpu, pool, starts_of, tables
from zhilight_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def attend(q, k, v, table, lens, starts, scale, **kw):
    """From the host, to float64."""
    out = ops.paged_attention(q.cuda(), *on_gpu(k, v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts.cuda(), scale, **kw)
    return out.cpu().double()


# ---- scores far from zero -----------------------------------------------------------------------------------------------------
STEEP_SEQS = {"one": [(300, 1), (77, 1), (1000, 1)], "drafts": [(300, 4), (80, 3), (4, 4)], "portion": [(300, 150), (150, 150), (700, 33)],
              "many": [(90 + 7 * (i % 5), 1 + i % 20) for i in range(60)]}


def check_steep(dtype, q_size, k_size, dim, seqs, window=0):
    """Queries of +-q_size in every column, key j k_size * (1 + (j * 37 % 7) / 128) in every column: powers of two times whole numbers below 2^8, so that
    every product and every sum of them is exact in 32 bits.  Two scores are the same number or at least 2^15 apart: a row is the mean of the values of its
    highest scores.  Equal scores get equal exponentials, whatever those are (2^-21 covers the exponential's own error and, where those of 16 bits differ from
    the 32-bit ones that are summed, their distance: powers of two round to themselves); sums add a unit for each key, the result is rounded once."""
    g = torch.Generator().manual_seed(21)
    heads, kv_heads, page = 8, 2, 16
    lens, new = [n for n, _ in seqs], [m for _, m in seqs]
    pages = sum(-(-n // page) for n in lens) + 2
    table, starts = tables(g, lens, page, pages), starts_of(new)
    k, v = pool(g, pages, page, kv_heads, dim, dtype, "rows")
    step = lambda j: 1.0 + (j * 37 % 7) / 128.0  # noqa: E731
    for b, n in enumerate(lens):
        for j in range(n):
            k[int(table[b, j // page]), j % page] = k_size * step(j)
    hide(k, table, lens, math.nan)
    hide(v, table, lens, math.nan)
    sign = torch.tensor([1.0, -1.0] * (heads // 2))
    q = (sign[:, None] * q_size).expand(sum(new), heads, dim).contiguous().to(dtype)
    assert q_size * k_size * dim / 128 >= 2.0 ** 15
    got = attend(q, k, v, table, lens, starts, 1.0, window=window, max_new=max(new))
    for b, (n, m) in enumerate(seqs):
        vv = oracle.rows_of(v, table, b, n)
        c = torch.tensor([step(j) for j in range(n)], dtype=torch.float64)
        j, at = torch.arange(n), torch.arange(n - m, n)
        seen = (j[None] <= at[:, None]) & ((j[None] > at[:, None] - window) if window else True)
        for h in range(heads):
            s = torch.where(seen, c * float(sign[h]), -math.inf)
            p = (s == s.amax(1, keepdim=True)).double()
            p /= p.sum(1, keepdim=True)
            x = vv[:, h // (heads // kv_heads)]
            o, spread = p @ x, p @ x.abs()
            err = spread * (2.0 ** -21 + 2 * (n + 64) * 2.0 ** -24)
            far = (got[int(starts[b]):int(starts[b + 1]), h] - o).abs() - err - oracle.half_step(o.abs() + err, dtype)
            assert (far <= 0).all(), (b, h, float(far.nan_to_num(1e30).max()))


@pytest.mark.parametrize("dtype,q_size,k_size", [(F16, 2.0 ** 8, 2.0 ** 8), (F16, 2.0 ** 10, 2.0 ** 11), (F16, 2.0 ** 13, 2.0 ** 13), (F16, 2.0 ** 15, 2.0 ** 15),
                                                 (BF16, 2.0 ** 12, 2.0 ** 14), (BF16, 2.0 ** 27, 2.0 ** 27)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seqs", list(STEEP_SEQS))
def test_attention_of_large_scores(cuda, dtype, q_size, k_size, dim, seqs):
    """Scores of 2^23 to 2^62: their distances decide, and steps between 32-bit numbers of their size are larger than any exponent."""
    check_steep(dtype, q_size, k_size, dim, STEEP_SEQS[seqs])


@pytest.mark.parametrize("q_size,k_size", [(2.0 ** 34, 2.0 ** 34), (2.0 ** 50, 2.0 ** 58), (2.0 ** 60, 2.0 ** 59)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seqs", list(STEEP_SEQS))
@pytest.mark.parametrize("window", [0, 40])
def test_attention_of_scores_near_the_largest_numbers(cuda, q_size, k_size, dim, seqs, window):
    """Scores of 2^74 to 2^126 on both sides of zero: rows whose scores all lie far below it are softmaxes like others."""
    check_steep(BF16, q_size, k_size, dim, STEEP_SEQS[seqs], window)


# ---- values of any size ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("size", [2.0 ** 127, 2.0 ** 100, 2.0 ** -70])
@pytest.mark.parametrize("new", [1, 4, 150])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_large_and_small_values(cuda, size, new, dim):
    """bf16 values up to the largest number: a mean of them is one that fits, whatever the sum is.  Small ones keep their bits."""
    g = torch.Generator().manual_seed(22)
    heads, kv_heads, page, seqs = 8, 2, 16, [(3000, new), (200, new), (new, new)]
    lens = [n for n, _ in seqs]
    pages = sum(-(-n // page) for n in lens) + 2
    table, starts = tables(g, lens, page, pages), starts_of([new] * 3)
    k, v = pool(g, pages, page, kv_heads, dim, BF16, "rows")
    k.mul_(3.0)                                                      # maxima that grow from tile to tile
    v.copy_(((torch.rand(v.shape, generator=g) + 0.99).double() * size).clamp(max=torch.finfo(BF16).max))
    hide(k, table, lens, math.nan)
    hide(v, table, lens, math.nan)
    q = torch.randn(3 * new, heads, dim, generator=g).to(BF16)
    got = attend(q, k, v, table, lens, starts, dim ** -0.5, max_new=new)
    want, off = oracle.attention(q, k, v, table, lens, starts, dim ** -0.5, 0)
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= off).all(), float(((got - want).abs() - off).max() / size)


# ---- keys and values that are no numbers ----------------------------------------------------------------------------------------
def softmax_of(q, k, v, table, lens, starts, scale, window):
    """oracle.attention where keys and values may be no numbers: a row's column is what 0 < p times the values it sees adds up to (NaN, or an infinity)."""
    out, off = oracle.attention(q, k, v, table, lens, starts, scale, window)
    for b, n in enumerate(lens):
        lo, hi = int(starts[b]), int(starts[b + 1])
        kk, vv = oracle.rows_of(k, table, b, n), oracle.rows_of(v, table, b, n)
        at, j = torch.arange(n - (hi - lo), n), torch.arange(n)
        seen = (j[None] <= at[:, None]) & ((j[None] > at[:, None] - window) if window else True)
        for x in range(kk.shape[1]):
            heads = slice(x * (q.shape[1] // kk.shape[1]), (x + 1) * (q.shape[1] // kk.shape[1]))
            for row in torch.nonzero(~torch.isfinite(vv[:, x]).all(1))[:, 0].tolist():
                add = torch.where(torch.isfinite(vv[row, x]), 0.0, vv[row, x])
                out[lo:hi, heads] += torch.where(seen[:, row, None], add, 0.0)[:, None]
            bad = ~torch.isfinite(kk[:, x]).all(1)
            out[lo:hi, heads] += torch.where((seen & bad).any(1), math.nan, 0.0)[:, None, None]
    return out, off


def same(got, want, off):
    """Numbers within `off`, infinities and NaN where they are wanted."""
    number = torch.isfinite(want)
    return bool(((got - want).abs() <= off)[number].all()) and torch.equal(got[~number].nan_to_num(0, 1, -1), want[~number].nan_to_num(0, 1, -1)) and \
        torch.equal(torch.isnan(got), torch.isnan(want))


@pytest.mark.parametrize("new,heads,kv_heads,page,window", [
    (1, 8, 2, 16, 0), (1, 8, 2, 16, 30), (4, 8, 2, 20, 0), (9, 2, 2, 16, 25), (6, 8, 1, 64, 0), (6, 8, 1, 5, 20), (40, 8, 2, 32, 0), (64, 8, 2, 16, 0), (64, 8, 2, 3, 0),
    (150, 8, 2, 64, 0), (150, 4, 2, 20, 50), (300, 2, 2, 128, 0), (300, 8, 1, 16, 33), (33, 40, 1, 256, 0)])
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 128)])
@pytest.mark.parametrize("before", [0, 200])
def test_attention_of_values_that_are_no_numbers(cuda, new, heads, kv_heads, page, window, dtype, dim, before):
    """In whole rows and in single columns, of new and of old tokens: rows that see them have them in their columns, other rows are as exact as ever."""
    g = torch.Generator().manual_seed(new + page)
    lens = [before + new, before + 37 + new, new]
    pages = sum(-(-n // page) for n in lens) + 2
    table, starts = tables(g, lens, page, pages), starts_of([new] * 3)
    q = torch.randn(3 * new, heads, dim, generator=g).to(dtype)
    for bad in (math.nan, math.inf, -math.inf):
        k, v = pool(g, pages, page, kv_heads, dim, dtype, "rows")
        for b, where in ((0, lens[0] - 1), (0, lens[0] - 1 - new // 3), (1, max(0, before - 10)), (2, new // 2)):
            row = (int(table[b, where // page]), where % page, b % kv_heads)
            if b == 1:
                v[row] = bad
            else:
                v[row][[3, dim - 1]] = torch.tensor([bad, -bad], dtype=dtype)
        hide(k, table, lens, math.nan)
        hide(v, table, lens, math.nan)
        got = attend(q, k, v, table, lens, starts, dim ** -0.5, window=window, max_new=new)
        assert same(got, *softmax_of(q, k, v, table, lens, starts, dim ** -0.5, window)), bad


@pytest.mark.parametrize("new,heads", [(1, 4), (3, 4), (64, 4), (300, 2)])
@pytest.mark.parametrize("what", ["last value", "old value", "old key", "window"])
def test_attention_of_long_sequences_with_a_broken_token(cuda, new, heads, what):
    """One token that is no number behind 130000: right for its own sequence and for others, no wait gave up, and it takes about as long as it does without."""
    g = torch.Generator().manual_seed(23)
    page, dim, window = 64, 64, 100000 if what == "window" else 0
    lens = [130000 + new, 500 + new, 70 + new]
    pages = sum(-(-n // page) for n in lens)
    table, starts = tables(g, lens, page, pages), starts_of([new] * 3)
    k, v = pool(g, pages, page, 1, dim, BF16, "rows")
    q = torch.randn(3 * new, heads, dim, generator=g).to(BF16)
    dev = [x.cuda() for x in (q, k, v, table, torch.tensor(lens, dtype=torch.int32), starts)]
    where = {"last value": lens[0] - 1, "old value": 7, "old key": 1000, "window": lens[0] - new - window + 1 + new // 2}[what]
    times = []
    for broken in (False, True):
        if broken:
            x, y = (k, dev[1]) if what == "old key" else (v, dev[2])
            for z in (x, y):
                z[int(table[0, where // page]), where % page, 0, 5] = math.nan if what == "old key" else math.inf
        each = []
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            got = ops.paged_attention(*dev, dim ** -0.5, window=window, max_new=new)
            b.record()
            torch.cuda.synchronize()
            each.append(a.elapsed_time(b))
        times.append(min(each))
    ops.check_waits()
    assert same(got.cpu().double(), *softmax_of(q, k, v, table, lens, starts, dim ** -0.5, window))
    assert times[1] < 3 * times[0], times


# ---- windows of any size --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30])
@pytest.mark.parametrize("new", [1, 5, 100, 200])
def test_attention_of_the_widest_windows(cuda, window, new):
    """A window that is wider than every sequence hides nothing, also where rows stand before the first key."""
    for dim in (64, 128):
        check_attention(BF16, 8, 2, dim, 16, "rows", window, [(new // 2, new), (0, new), (new, new), (new + 300, new)])
        check_attention(F16, 8, 2, dim, 16, "rows", window, [(new // 2, new), (new - new // 4, new)], max_new=new)


def test_numbers_beyond_32_bits(cuda):
    """Python's integers do not come around: a wider window is as wide as any, a layout or a window below zero is refused."""
    from zhilight_b200 import _lib
    g = torch.Generator().manual_seed(24)
    k, v = (x.cuda() for x in pool(g, 8, 16, 2, 64, BF16, "rows"))
    table, lens, starts = torch.arange(8, dtype=torch.int32)[None].cuda(), torch.tensor([100], dtype=torch.int32).cuda(), starts_of([20]).cuda()
    q = torch.randn(20, 8 * 64, generator=g).to(BF16).cuda()
    want = ops.paged_attention(q, k, v, table, lens, starts, 0.1)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 63 + 5):
        assert torch.equal(ops.paged_attention(q, k, v, table, lens, starts, 0.1, window=window), want)
    for window in (-1, -2 ** 32 + 5):
        with pytest.raises(_lib.ZLError):
            ops.paged_attention(q, k, v, table, lens, starts, 0.1, window=window)
    assert torch.equal(ops.paged_attention(q, k, v, table, lens, starts, 0.1, max_new=2 ** 32 + 1), want)
    t = torch.zeros(20, dtype=torch.int32).cuda()
    with pytest.raises(_lib.ZLError):
        ops.qkv_axes_rope_append(torch.zeros(20, 12 * 64, dtype=BF16).cuda(), t[None], torch.ones(32, dtype=torch.float64).cuda(), torch.zeros(32, dtype=torch.int32).cuda(),
                                 t, t - 1, table, k, v, 8, layout=2 ** 32)


# ---- what tells which rows are whose ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("starts", [(0, 40, 30, 60), (0, 60, 0, 60), (0, 60, 59, 60), (-7, 70, 5, 6)])
@pytest.mark.parametrize("max_new", [1, None])
def test_attention_of_more_rows_than_there_are(cuda, starts, max_new):
    """Sequences that have more rows together than q: no row is written."""
    g = torch.Generator().manual_seed(25)
    k, v = (x.cuda() for x in pool(g, 8, 16, 2, 64, BF16, "rows"))
    table, lens = torch.arange(8, dtype=torch.int32).expand(3, 8).contiguous().cuda(), torch.tensor([100, 60, 70], dtype=torch.int32).cuda()
    q, out = torch.randn(60, 4, 64, generator=g).to(BF16).cuda(), torch.full((60, 4, 64), 7.0, dtype=BF16, device="cuda")
    ops.paged_attention(q, k, v, table, lens, torch.tensor(starts, dtype=torch.int32).cuda(), 0.1, max_new=max_new, out=out)
    assert (out == 7.0).all()


@pytest.mark.parametrize("starts,lens", [((-5, 3, 20, 90), (50, 60, 70)), ((0, 0, 60, 60), (-3, 60, 2 ** 31 - 1)), ((2, 10, 11, 2 ** 31 - 1), (0, 5, -2 ** 31)),
                                         ((0, 20, 40, 60), (2 ** 31 - 1, 128, 129)), ((0, 20, 50, 0), (30, 60, 70)), ((8, 0, 8, 0), (30, 60, 70)), ((5, -1, 10, 20), (9, 60, 70)),
                                         ((60, 60, 0, 60), (9, 60, 70))])
@pytest.mark.parametrize("max_new", [1, None])
def test_attention_of_starts_and_lengths_out_of_range(cuda, starts, lens, max_new):
    """Rows before the first and behind the last one are none, lengths go as far as the table has room, a sequence that ends before it begins has no rows."""
    g = torch.Generator().manual_seed(26)
    k, v = pool(g, 8, 16, 2, 64, BF16, "rows")
    table, rows = torch.arange(8, dtype=torch.int32).expand(3, 8).contiguous(), 60
    q, out = torch.randn(rows, 4, 64, generator=g).to(BF16), torch.full((rows, 4, 64), 7.0, dtype=BF16, device="cuda")
    got = ops.paged_attention(q.cuda(), *on_gpu(k, v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), 0.1,
                              max_new=max_new, out=out).cpu().double()
    mine = torch.zeros(rows, dtype=torch.bool)
    for b, n in enumerate(lens):
        first, last = max(starts[b], 0), min(starts[b + 1], rows)
        if first >= last:
            continue
        mine[first:last] = True
        # the rows that there are, at the places that the sequence's own end gives them
        place = n - starts[b + 1] + first
        have = max(0, min(n, 128))
        kk, vv = (oracle.rows_of(x, table, b, have) for x in (k, v))
        for i in range(first, last):
            sees = max(0, min(place + i - first + 1, have))
            for h in range(4):
                p = torch.softmax(kk[:sees, h // 2] @ q[i, h].double() * 0.1, 0)
                o, spread = p @ vv[:sees, h // 2], p @ vv[:sees, h // 2].abs()
                # scores below 20 in magnitude: 2 (64 + 8) 2^-24 times that; a rounded probability, a rounded result
                err = spread * (2.0 ** -8 + 40 * 72 * 2.0 ** -24 + 2.0 ** -14)
                assert ((got[i, h] - o).abs() <= err + oracle.half_step(o.abs() + err, BF16)).all(), (b, i, h)
    assert (got[~mine] == 7.0).all()


# ---- what the kernel for few rows does not round ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,part,keys", [(BF16, 0.9 * 2.0 ** -9, 300), (BF16, 0.9 * 2.0 ** -9, 1500), (F16, 0.9 * 2.0 ** -12, 200)])
@pytest.mark.parametrize("seqs,new,heads,kv_heads", [(1, 1, 8, 2), (3, 4, 8, 2), (300, 2, 4, 2), (2, 1, 258, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_probabilities_of_few_rows_are_not_rounded_to_the_type(cuda, dtype, part, keys, seqs, new, heads, kv_heads, dim):
    """Half of the keys have probabilities of 1 and values of 1, the others just so much less that one rounding to 16 bits would make them 1 too, and values of -1: the
    result is that difference.  Carried as 16 bits and the rest in 16 bits, a probability is off by eps^2 / 4; its exponent, below 64 in size, by 2^-19, its exponential by
    2^-22 more; scores by (dim + 8) steps of 2^-24 of themselves; sums by a unit for each key; the result is rounded once."""
    g = torch.Generator().manual_seed(27)
    page = 16
    lens = [keys - 7 * (b % 3) for b in range(seqs)]
    pages = sum(-(-n // page) for n in lens)
    table, starts = tables(g, lens, page, pages), starts_of([new] * seqs)
    k, v = (x.zero_() for x in pool(g, pages, page, kv_heads, dim, dtype, "rows"))
    k[:, 1::2, :, 0] = math.log1p(-part)
    v[:, 0::2], v[:, 1::2] = 1.0, -1.0
    q = torch.zeros(seqs * new, heads, dim).to(dtype)
    q[..., 0] = 1.0
    got = attend(q, k, v, table, lens, starts, 1.0, max_new=new)
    eps = oracle.EPS[dtype]
    low = math.exp(float(k[0, 1, 0, 0]))                             # of odd keys (a page has an even number of rows)
    for b, n in enumerate(lens):
        for i in range(new):
            sees = n - new + i + 1
            even, odd = (sees + 1) // 2, sees // 2
            want = (even - odd * low) / (even + odd * low)
            off = eps * eps / 4 + 2 * (2.0 ** -19 + 2.0 ** -22 + part * (dim + 8) * 2.0 ** -24) + 2 * (sees + 64) * 2.0 ** -24
            off += (abs(want) + off) * eps / 2 + 2.0 ** -25
            assert abs((even - odd) / (even + odd) - want) > off     # one rounding would not pass
            row = got[int(starts[b]) + i]
            assert ((row - want).abs() <= off).all(), (b, i, float((row - want).abs().max()), off)


@pytest.mark.parametrize("seqs", list(STEEP_SEQS))
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (12, 4), (160, 1)])
def test_attention_in_place(cuda, seqs, heads, kv_heads):
    """out may be q itself."""
    g = torch.Generator().manual_seed(28)
    lens, new = [n for n, _ in STEEP_SEQS[seqs]], [m for _, m in STEEP_SEQS[seqs]]
    pages = sum(-(-n // 16) for n in lens)
    table, starts = tables(g, lens, 16, pages).cuda(), starts_of(new).cuda()
    k, v = (x.cuda() for x in pool(g, pages, 16, kv_heads, 64, BF16, "rows"))
    q = torch.randn(sum(new), heads, 64, generator=g).to(BF16).cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    want = ops.paged_attention(q, k, v, table, n, starts, 0.125, max_new=max(new))
    got = ops.paged_attention(q, k, v, table, n, starts, 0.125, max_new=max(new), out=q)
    assert got is q and torch.equal(q, want)
