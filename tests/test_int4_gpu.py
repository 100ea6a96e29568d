"""Operators over a paged cache of 4 bits on a GPU, against their formulas in 64 bits (paged_oracle, int4_oracle)."""
import math
from fractions import Fraction

import pytest
import torch

from tests import int4_oracle as codes
from tests import paged_oracle as oracle
from tests.test_paged_gpu import Own, Step as WideStep, both_ways, probabilities, starts_of, tables
from zhilight_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def rows_in(x, order, dtype):
    """Rows (pages, page, kv_heads, dim) -> bytes of the same order: (`rows`) as it is, (`heads`) heads outside the rows, (`wide`) within wider rows."""
    b = codes.encode(x, dtype)
    if order == "heads":
        return b.transpose(1, 2).contiguous().transpose(1, 2)
    if order == "wide":
        big = torch.full((*b.shape[:2], b.shape[2] + 1, b.shape[3] * 2), 0xa5, dtype=torch.uint8)
        big[:, :, :-1, :b.shape[3]] = b
        return big[:, :, :-1, :b.shape[3]]
    return b


def to_gpu(x):
    """The same strides on the device."""
    y = torch.empty(max(1, sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1), dtype=x.dtype, device="cuda").as_strided(x.shape, x.stride())
    return y.copy_(x)


def pool(g, pages, page, kv_heads, dim, dtype, order, spread=1.0):
    """Caches of random rows whose columns differ in their middle: keys, values."""
    middle = torch.randn(kv_heads, dim, generator=g) * spread
    k = (torch.randn(pages, page, kv_heads, dim, generator=g) + middle).to(dtype)
    return rows_in(k, order, dtype), rows_in(torch.randn(pages, page, kv_heads, dim, generator=g).to(dtype), order, dtype)


def hide(cache, table, lens, byte=0xff):
    """Bytes of 0xff (codes of 15, steps of NaN) in every row of the pool that no sequence has."""
    pages, page = cache.shape[:2]
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(n):
            if 0 <= int(table[b, i // page]) < pages:
                used[int(table[b, i // page]), i % page] = True
    cache[~used] = byte


# ---- append --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,half,adjacent,page,order,t", [
    (32, 8, 128, 64, False, 16, "rows", 1), (32, 8, 128, 64, False, 16, "heads", 37), (4, 4, 64, 16, True, 1, "rows", 9), (6, 2, 64, 20, False, 5, "wide", 33),
    (7, 1, 64, 13, True, 20, "rows", 12), (3, 3, 128, 4, False, 3, "heads", 5), (2, 1, 64, 0, False, 16, "rows", 4), (64, 8, 128, 48, False, 64, "rows", 70),
    (1, 1, 64, 32, True, 2, "rows", 3), (3, 1, 64, 31, False, 7, "heads", 300), (200, 100, 128, 64, False, 16, "heads", 5), (128, 128, 64, 32, True, 8, "rows", 400),
    (64, 8, 128, 64, False, 16, "wide", 2000)])
def test_append(cuda, dtype, heads, kv_heads, dim, half, adjacent, page, order, t):
    """Keys are turned in 64 bits and rounded to 32 and to the type: their codes, like the values', are the formula's, bit by bit."""
    g = torch.Generator().manual_seed(heads * 1000 + t)
    lens = [t, t + 11, 2 * t]
    pages = sum(-(-n // page) for n in lens) + 2
    table = tables(g, lens, page, pages)
    k, v = pool(g, pages, page, kv_heads, dim, dtype, order)
    width = (heads + 2 * kv_heads) * dim
    wide = torch.randn(t, width + 16, generator=g).to(dtype)
    pos = torch.randint(0, 5_000_000, (3, t), generator=g, dtype=torch.int32)
    axis = torch.randint(0, 3, (half,), generator=g, dtype=torch.int32)
    if half > 4:
        axis[3], axis[4] = -1, 3                                     # axes that do not exist do not turn
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    seq = torch.randint(0, 3, (t,), generator=g, dtype=torch.int32)
    place = torch.tensor([lens[int(s)] - t + i for i, s in enumerate(seq)], dtype=torch.int32)
    if t > 4:
        place[2], seq[3], place[4] = -1, 3, page * table.shape[1]    # nowhere, no such sequence, behind the table
    want_q, want_k, want_v, off_q, _ = oracle.axes_rope(wide[:, :width].contiguous(), pos, freq, axis, heads, kv_heads, dim, adjacent, 1.25)
    kd, vd = to_gpu(k), to_gpu(v)
    q = ops.qkv_axes_rope_append_int4(wide.cuda()[:, :width], pos.cuda(), freq.cuda(), axis.cuda(), seq.cuda(), place.cuda(), table.cuda(), kd, vd, heads,
                                      layout=ops.ROT_ADJACENT if adjacent else ops.ROT_HALVES, mscale=1.25).cpu().view(t, heads, dim)
    assert ((q.double() - want_q).abs() <= off_q).all()
    new_k, new_v = (codes.encode(x.float().to(dtype), dtype) for x in (want_k, want_v))
    for i in range(t):
        s, p = int(seq[i]), int(place[i])
        if 0 <= s < 3 and 0 <= p < page * table.shape[1] and 0 <= int(table[s, p // page]) < pages:
            k[int(table[s, p // page]), p % page], v[int(table[s, p // page]), p % page] = new_k[i], new_v[i]
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)     # places of no row are as they were
    for pages_of in (None, torch.randperm(pages, generator=g)[:3].to(torch.int32)):
        got = ops.int4_cache_values(kd, vd, dtype, pages_of if pages_of is None else pages_of.cuda())
        for x, y in zip(got, (k, v)):
            assert x.is_contiguous() and torch.equal(x.cpu(), codes.decode(y if pages_of is None else y[pages_of.long()], dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
def test_append_at_the_ends_of_the_type(cuda, dtype, dim):
    """Constants, the largest and smallest numbers, halves between two codes, infinities and NaN: the values that come back are the formula's."""
    g = torch.Generator().manual_seed(2)
    top, least = codes.TOP[dtype], 2.0 ** (codes.BITS[dtype][1] - codes.BITS[dtype][0] + 1)
    x = torch.randn(24, 1, dim, generator=g).to(dtype)
    x[0], x[1], x[2] = 0.0, 3.25, -top
    x[3, 0, ::2], x[3, 0, 1::2] = top, -top
    x[4] = torch.randint(0, 16, (dim,), generator=g).to(dtype) * least      # the smallest numbers
    x[5] = torch.randint(-3, 4, (dim,), generator=g).to(dtype) * least * 64
    x[6] = torch.arange(dim).remainder(31).to(dtype) * 0.5                  # steps of one: every second number between two codes
    x[7] = torch.arange(dim).remainder(16).to(dtype)
    x[8], x[8, 0, 7] = 1.0, 1.0 + 2.0 ** (1 - codes.BITS[dtype][0])
    x[9, 0, 3], x[10, 0, 35], x[11, 0, dim - 1] = math.nan, math.inf, -math.inf
    x[12, 0, :32] = math.inf
    x[13, 0, 0], x[13, 0, 1] = math.inf, -math.inf
    x[14] = (x[14].float() * 2.0 ** 13).to(dtype)
    x[15, 0, 4] = top
    x[16] *= least
    qkv = torch.cat([x[:, 0], x[:, 0], x[:, 0]], 1)                         # position 0 turns nothing
    for page, order in ((8, "rows"), (24, "heads")):
        k = rows_in(torch.zeros(24 // page, page, 1, dim, dtype=dtype), order, dtype)
        kd, vd = to_gpu(k), to_gpu(k)
        table = torch.arange(24 // page, dtype=torch.int32)[None].cuda()
        one = torch.zeros(24, dtype=torch.int32).cuda()
        q = ops.qkv_axes_rope_append_int4(qkv.cuda(), one[None], torch.ones(1, dtype=torch.float64).cuda(), one[:1] - 1, one, torch.arange(24, dtype=torch.int32).cuda(),
                                          table, kd, vd, 1)
        assert torch.equal(q.cpu().view(torch.int16)[:9], qkv[:9, :dim].view(torch.int16))
        want = codes.decode(codes.encode(x, dtype), dtype).view(24 // page, page, 1, dim)
        broken = torch.isnan(want)
        assert int(broken.sum()) == 32 * 5
        for y in ops.int4_cache_values(kd, vd, dtype):
            y = y.cpu()
            assert torch.equal(torch.isnan(y), broken) and torch.equal(y[~broken], want[~broken])


def formula_row(x, dtype):
    """A row of numbers of dtype -> its bytes, by fractions: nothing is rounded but what the formula rounds."""
    v, (bits, least), words, pairs = [Fraction(float(y)) for y in x], codes.BITS[dtype], [], []
    for i in range(0, len(v), 32):
        low, high = min(v[i:i + 32]), max(v[i:i + 32])
        part = (high - low) / 15
        power = least
        while part >= Fraction(2) ** (power + 1):
            power += 1
        unit = Fraction(2) ** (power - bits + 1)
        step = part // unit * unit
        code = [min(round((y - low) / step), 15) if step >= Fraction(2) ** -126 else 0 for y in v[i:i + 32]]   # to the nearest, ties to even
        words += [sum(c << codes.PLACE[j] for j, c in enumerate(code[k:k + 8])) for k in range(0, 32, 8)]
        pairs.append(torch.tensor([float(step), min(float(y) for y in x[i:i + 32])], dtype=dtype))   # -0 is a lowest value too
    return torch.cat([torch.tensor([w - (w >> 31 << 32) for w in words], dtype=torch.int32).view(torch.uint8), torch.cat(pairs).view(torch.uint8)])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_of_numbers_far_apart(cuda, dtype):
    """Groups whose numbers have more bits between them than 32-bit numbers: lowest values so small that the range is just below or above 15 steps of the type, values beside the
    border between two codes by as little, and any numbers of the type in one group.  Steps and codes are the formula's."""
    g = torch.Generator().manual_seed(41)
    dim, (bits, least) = 64, codes.BITS[dtype]
    tiny = 2.0 ** (least - bits + 1)                                 # the smallest number of the type
    x = torch.zeros(400, dim)
    for i in range(200):
        scale = 2.0 ** (i % 9 if dtype == F16 else i % 50 - 20)
        low = (-1.0) ** i * max(2.0 ** -(10 + i // 4 % 40), tiny)
        x[i] = torch.randint(0, 31, (dim,), generator=g) * 0.5 * scale   # whole steps and halves of them
        x[i, ::32], x[i, 1::32] = low, 15.0 * scale
        if low > 0:
            x[i].clamp_(min=low)
        elif i % 3 == 0:
            x[i, 2:9], x[i, 34:41] = -low, -low * 2
    any_bits = torch.randint(-2 ** 15, 2 ** 15, (400, dim), generator=g, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x.to(dtype)
    x[200:] = torch.where(torch.isfinite(any_bits[200:]), any_bits[200:], torch.ones((), dtype=dtype))
    x[300:] = torch.where(torch.rand(100, dim, generator=g) < 0.7, (x[300:].double().abs() ** 0.25).to(dtype), x[300:])
    x[0], x[1] = x[2], x[3]
    x[0, :3], x[1, :3] = torch.tensor([-2.0 ** -25, 15.0, 2.5]), torch.tensor([2.0 ** -25, 15.0, 2.5])
    x[0, 3:32], x[1, 3:32] = 7.5, 7.5
    kd = torch.zeros(25, 16, 1, 40, dtype=torch.uint8, device="cuda")
    vd, one = torch.zeros_like(kd), torch.zeros(400, dtype=torch.int32, device="cuda")
    ops.qkv_axes_rope_append_int4(torch.cat([x, x, x.flip(1)], 1).cuda(), one[None], torch.ones(1, dtype=torch.float64).cuda(), one[:1] - 1, one,
                                  torch.arange(400, dtype=torch.int32).cuda(), torch.arange(25, dtype=torch.int32)[None].cuda(), kd, vd, 1)
    for got, rows in ((kd, x), (vd, x.flip(1))):
        want = torch.stack([formula_row(r, dtype) for r in rows.double().tolist()])
        off = torch.nonzero((got.cpu().view(400, 40) != want).any(1)).flatten()
        assert off.numel() == 0, (off.tolist(), rows[off[0]].tolist())


def test_append_takes_pages_of_the_table_only(cuda):
    """Page numbers outside the pool take no writes and read as zeros."""
    g = torch.Generator().manual_seed(3)
    k, v = pool(g, 4, 8, 2, 64, BF16, "rows")
    kd, vd = to_gpu(k), to_gpu(v)
    table = torch.tensor([[1, -1], [4, 2 ** 31 - 1]], dtype=torch.int32)
    qkv = torch.randn(4, 8 * 64, generator=g).to(BF16)
    seq, place = torch.tensor([0, 0, 1, 1], dtype=torch.int32), torch.tensor([3, 9, 0, 12], dtype=torch.int32)
    q = ops.qkv_axes_rope_append_int4(qkv.cuda(), torch.zeros(1, 4, dtype=torch.int32).cuda(), torch.ones(32, dtype=torch.float64).cuda(),
                                      torch.zeros(32, dtype=torch.int32).cuda(), seq.cuda(), place.cuda(), table.cuda(), kd, vd, 4)
    assert torch.equal(q.cpu(), qkv[:, :4 * 64])                     # position 0 turns nothing
    k[1, 3], v[1, 3] = codes.encode(qkv[0, 4 * 64:6 * 64].view(2, 64), BF16), codes.encode(qkv[0, 6 * 64:].view(2, 64), BF16)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
    ids = torch.tensor([3, -1, 4, 1, 1, 2 ** 31 - 1], dtype=torch.int32)
    got = ops.int4_cache_values(kd, None, BF16, ids.cuda()).cpu()
    want = torch.zeros(6, 8, 2, 64, dtype=BF16)
    for i in (0, 3, 4):
        want[i] = codes.decode(k[int(ids[i])], BF16)
    assert torch.equal(got, want)


# ---- attention -----------------------------------------------------------------------------------------------------------------
def check_attention(dtype, heads, kv_heads, dim, page, order, window, seqs, seed=0, max_new=None, break_pages=False, behind=3, scale=None, extra=1):
    """seqs: [(keys, new tokens)]."""
    g = torch.Generator().manual_seed(seed)
    lens, new = [n for n, _ in seqs], [m for _, m in seqs]
    pages = sum(-(-n // page) for n in lens) + 2
    table = tables(g, lens, page, pages, extra)
    k, v = pool(g, pages, page, kv_heads, dim, dtype, order)
    if break_pages:
        table[0, 0], table[-1, 1] = pages, -1
    hide(k, table, lens)
    hide(v, table, lens)
    t = sum(new)
    q = torch.randn(t + behind, heads, dim, generator=g).to(dtype)
    starts, n = starts_of(new), torch.tensor(lens, dtype=torch.int32)
    scale = scale or dim ** -0.5
    want, off = oracle.attention(q, codes.decode(k, dtype), codes.decode(v, dtype), table, lens, starts, scale, window)
    out = torch.full_like(q, 7.0).cuda()
    got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), n.cuda(), starts.cuda(), scale, window=window, max_new=max_new, out=out)
    assert got is out
    got = got.cpu().double()
    assert (got[t:] == 7.0).all()                                    # rows behind the last sequence
    far = (got[:t] - want[:t]).abs() - off[:t]
    assert (far <= 0).all(), (float(far.nan_to_num(1e9).max()), torch.nonzero(~(far <= 0))[:5].tolist())


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(BF16, 32, 8, 128), (F16, 32, 8, 128), (BF16, 16, 16, 64), (F16, 8, 1, 64), (BF16, 28, 4, 128),
                                                      (F16, 20, 1, 128), (BF16, 3, 1, 64), (F16, 40, 1, 128), (F16, 12, 1, 64)])
@pytest.mark.parametrize("page,order", [(16, "rows"), (64, "heads"), (20, "wide"), (1, "rows"), (256, "rows"), (32, "wide"), (48, "heads")])
def test_attention_single_tokens(cuda, dtype, heads, kv_heads, dim, page, order):
    check_attention(dtype, heads, kv_heads, dim, page, order, 0, [(1, 1), (17, 1), (300, 1), (64, 1), (0, 0), (129, 1), (5, 0), (1025, 1)], max_new=1)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(BF16, 32, 8, 128), (F16, 64, 8, 128), (BF16, 8, 8, 64), (F16, 12, 4, 64)])
@pytest.mark.parametrize("window", [0, 1, 50, 1000])
def test_attention_drafts(cuda, dtype, heads, kv_heads, dim, window):
    check_attention(dtype, heads, kv_heads, dim, 16, "rows", window, [(6, 6), (200, 5), (77, 2), (500, 9), (33, 1), (1500, 4), (0, 0), (70, 7)], max_new=9)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,order", [(BF16, 8, 2, 128, 16, "rows"), (F16, 8, 2, 64, 64, "heads"), (BF16, 4, 4, 128, 20, "wide"),
                                                                 (F16, 7, 1, 128, 128, "rows"), (BF16, 16, 1, 64, 8, "rows"), (F16, 5, 5, 64, 1, "rows")])
@pytest.mark.parametrize("window", [0, 100, 300])
@pytest.mark.parametrize("seqs", [[(300, 300)], [(700, 130), (1, 1), (129, 129), (513, 257), (40, 0)], [(1000, 64), (65, 65), (128, 128)]])
def test_attention_portions(cuda, dtype, heads, kv_heads, dim, page, order, window, seqs):
    check_attention(dtype, heads, kv_heads, dim, page, order, window, seqs)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,window,seqs", [
    (BF16, 16, 2, 64, 16, 0, [(2000, 900)]), (F16, 8, 2, 128, 48, 0, [(2111, 700), (1900, 333), (1800, 1)]), (BF16, 8, 2, 128, 20, 900, [(2500, 900), (1111, 40)]),
    (F16, 64, 8, 128, 64, 0, [(1000 + 131 * i, 1 + i % 16) for i in range(10)]), (BF16, 48, 8, 64, 32, 1000, [(2000 + 77 * i, 9 + i) for i in range(6)]),
    (F16, 24, 8, 64, 256, 0, [(3001, 43), (2048, 30), (130, 130), (2500, 12)]), (BF16, 32, 8, 128, 128, 0, [(20000, 1)]), (F16, 16, 8, 64, 20, 0, [(20000, 3), (9, 1)])])
def test_attention_of_long_stretches(cuda, dtype, heads, kv_heads, dim, page, window, seqs):
    """Enough keys for every CTA to go round its buffers several times, blocks whole and cut."""
    check_attention(dtype, heads, kv_heads, dim, page, "rows", window, seqs, max_new=max(n for _, n in seqs))


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,order", [(BF16, 8, 2, 128, 16, "rows"), (F16, 8, 2, 64, 64, "heads"), (BF16, 4, 4, 128, 20, "wide"), (F16, 24, 8, 64, 32, "rows"),
                                                                 (F16, 7, 1, 128, 128, "rows"), (BF16, 16, 1, 64, 8, "rows"), (F16, 5, 5, 64, 1, "rows"), (BF16, 12, 3, 64, 16, "wide")])
@pytest.mark.parametrize("window", [0, 100, 300])
@pytest.mark.parametrize("seqs", [[(700, 700)], [(700, 130), (1, 1), (129, 129), (513, 257), (40, 0)], [(1000 + 131 * i, 1 + i % 90) for i in range(6)]])
def test_attention_behind_wide_tables(cuda, dtype, heads, kv_heads, dim, page, order, window, seqs):
    """Tables with room for far more keys than a workspace has: the tiles make codes numbers by themselves."""
    check_attention(dtype, heads, kv_heads, dim, page, order, window, seqs, extra=(1 << 30) // (page * kv_heads * dim * 4) // len(seqs))


def test_attention_behind_wide_tables_elsewhere(cuda):
    """Bad pages, rows before the first key and broken tokens on that way."""
    wide = (1 << 30) // (16 * 2 * 64 * 4)
    check_attention(F16, 8, 2, 128, 16, "rows", 0, [(200, 150), (220, 150)], break_pages=True, extra=wide)
    check_attention(BF16, 8, 2, 64, 16, "rows", 3, [(100, 200), (0, 200), (200, 200)], extra=wide)
    check_attention(BF16, 8, 2, 64, 16, "heads", 0, [(100, 200), (0, 200), (200, 200)], extra=wide)
    g = torch.Generator().manual_seed(5)
    table = tables(g, [400], 16, 40, extra=wide)
    q = torch.randn(150, 8, 64, generator=g).to(BF16)
    for where, which in ((399, 1), (300, 1), (220, 0), (399, 0)):
        k, v = pool(g, 40, 16, 2, 64, BF16, "rows")
        (k, v)[which][int(table[0, where // 16]), where % 16, 1, 36:40] = 0xff   # columns 32 to 63
        got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), torch.tensor([400], dtype=torch.int32).cuda(), starts_of([150]).cuda(), 0.125).cpu().double()
        want, off = oracle.attention(q, codes.decode(k, BF16), codes.decode(v, BF16), table, [400], starts_of([150]), 0.125, 0)
        fine = torch.ones(150, 8, 64, dtype=torch.bool)
        fine[torch.arange(250, 400) >= where, 4:, 32 if which else 0:] = False
        assert ((got - want).abs() <= off)[fine].all() and torch.isnan(got[~fine]).all()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,order", [(BF16, 8, 2, 128, 16, "rows"), (F16, 8, 2, 64, 64, "heads"), (BF16, 16, 1, 128, 20, "wide"), (F16, 32, 2, 64, 32, "rows"),
                                                                 (BF16, 5, 5, 64, 1, "rows"), (F16, 17, 1, 128, 16, "rows"), (BF16, 160, 1, 64, 16, "rows")])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("room", [2500, 20000])
@pytest.mark.parametrize("seqs", [[(700, 1), (1300, 300)], [(700, 130), (1, 1), (129, 129), (513, 257), (40, 0), (1300, 4), (300, 1)]])
def test_attention_of_few_rows_beside_portions(cuda, dtype, heads, kv_heads, dim, page, order, window, room, seqs):
    """A table with room for few keys and for more; groups of heads that count as few rows and wider ones."""
    check_attention(dtype, heads, kv_heads, dim, page, order, window, seqs, extra=room // page)


@pytest.mark.parametrize("max_new", [1, 5, 100, None])
@pytest.mark.parametrize("wide", [400, 60000])
def test_attention_of_lengths_out_of_range_behind_wide_tables(cuda, max_new, wide):
    """Lengths that the table has no room for, starts out of order: rows of q alone are touched, and the sequences in range are right."""
    g = torch.Generator().manual_seed(15)
    page, dim = 16, 64
    table = torch.full((4, wide), -1, dtype=torch.int32)
    table[:, :20] = torch.randperm(80, generator=g).view(4, 20).to(torch.int32)
    k, v = pool(g, 80, page, 2, dim, BF16, "rows")
    q = torch.randn(310, 8, dim, generator=g).to(BF16)
    kk, vv = codes.decode(k, BF16), codes.decode(v, BF16)
    for starts, lens in (((0, 300, 301, 302, 303), (320, 300, 2 ** 31 - 1, -4)), ((0, 300, 301, 301, 2 ** 31 - 1), (320, 300, 5, -2 ** 31)),
                         ((0, 300, 301, 280, 280), (320, 1, 7, 2 ** 31 - 1)), ((0, 300, 301, -2 ** 31, -2 ** 31), (320, 0, 2 ** 31 - 1, -2 ** 31)), ((0, 300, 301, 301, -2 ** 31), (320, 300, 2 ** 31 - 1, 5))):
        out = torch.full((330, 8, dim), 7.0, dtype=BF16, device="cuda")
        ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda(),
                                 0.125, max_new=max_new, out=out[:310])
        out = out.cpu().double()
        assert (out[310:] == 7.0).all()
        want, off = oracle.attention(q[:301], kk, vv, table[:2], lens[:2], starts[:3], 0.125, 0)
        assert ((out[:301] - want).abs() <= off).all()
        k16, v16 = (x.cuda() for x in (kk, vv))                       # the same over a cache of 16 bits
        got = ops.paged_attention(q.cuda(), k16, v16, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), 0.125, max_new=max_new)
        assert ((got[:301].cpu().double() - want).abs() <= off).all()


@pytest.mark.parametrize("page,dim", [(20, 64), (48, 128), (16, 64), (1, 64)])
@pytest.mark.parametrize("new", [(1, 1, 1), (150, 200, 1), (9, 3, 160), (30, 20, 8)])
@pytest.mark.parametrize("window", [0, 130])
def test_attention_of_sequences_longer_than_the_table(cuda, page, dim, new, window):
    """Keys that the table has no room for do not count, wherever its room ends in a tile: whole rows of q see what is left, or nothing of it in a window."""
    g = torch.Generator().manual_seed(page + new[0])
    columns = 613 // page
    lens = [columns * page + 7, columns * page + 190, 400]
    table = tables(g, lens, page, sum(-(-n // page) for n in lens) + 2)[:, :columns].contiguous()
    k, v = pool(g, sum(-(-n // page) for n in lens) + 2, page, 2, dim, BF16, "rows")
    used = [min(n, columns * page) for n in lens]
    hide(k, table, used), hide(v, table, used)
    q, starts = torch.randn(sum(new), 16, dim, generator=g).to(BF16), starts_of(new)
    got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts.cuda(), dim ** -0.5, window=window,
                                   max_new=max(new)).cpu().double()
    want, off = oracle.attention(q, codes.decode(k, BF16), codes.decode(v, BF16), table, lens, starts, dim ** -0.5, window)
    assert ((got - want).abs() <= off).all()


@pytest.mark.parametrize("max_new", [1, 3, 20, 200, None])
def test_attention_does_not_depend_on_the_bound_of_new_tokens(cuda, max_new):
    check_attention(BF16, 8, 2, 128, 16, "rows", 0, [(300, 200), (40, 1), (90, 3), (600, 18)], max_new=max_new)


@pytest.mark.parametrize("new", [1, 4, 150])
def test_attention_over_bad_pages(cuda, new):
    """A page number outside the pool reads as rows of zeros."""
    check_attention(F16, 8, 2, 128, 16, "rows", 0, [(200, new), (220, new)], break_pages=True)
    check_attention(BF16, 8, 2, 64, 20, "heads", 0, [(200, new), (220, new)], break_pages=True)


@pytest.mark.parametrize("new", [1, 5, 100, 200])
def test_attention_rows_before_the_first_key(cuda, new):
    """More new tokens than keys: the rows before the first key see nothing and give zeros."""
    check_attention(BF16, 8, 2, 64, 16, "rows", 0, [(new // 2, new), (0, new), (new, new)])
    check_attention(BF16, 8, 2, 64, 16, "rows", 3, [(new // 2, new), (0, new), (new, new)])


@pytest.mark.parametrize("page", [4, 8, 12, 24, 40, 56, 100, 136])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_over_pages_of_any_size(cuda, page, dim):
    seqs = [(1600 + 100 * i, 1 + 5 * i) for i in range(5)] + [(900, 200), (700, 70)]
    check_attention(BF16, 16, 2, dim, page, "rows", 0, seqs, max_new=200)
    check_attention(F16, 16, 2, dim, page, "heads", 1000, seqs[:4], max_new=16)


@pytest.mark.parametrize("new,heads,kv_heads", [(1, 4, 2), (3, 4, 1), (20, 8, 2)])
def test_attention_of_many_sequences(cuda, new, heads, kv_heads):
    """More sequences than a warp looks at at a time, some without tokens or keys, also at the ends of what is in view."""
    seqs = [(1 + (37 * i) % 150 + new, 1 + i % new) if i % 11 and i not in (127, 128, 255) else (i % 2 * 30, 0) for i in range(300)]
    check_attention(F16, heads, kv_heads, 64, 16, "rows", 0, seqs, max_new=new)
    check_attention(F16, heads, kv_heads, 64, 16, "heads", 33, seqs[:129], max_new=new)


@pytest.mark.parametrize("heads,kv_heads", [(160, 1), (129, 1), (256, 2), (65, 1)])
@pytest.mark.parametrize("new", [1, 3])
def test_attention_of_wide_groups(cuda, heads, kv_heads, new):
    check_attention(BF16, heads, kv_heads, 64, 16, "rows", 0, [(100, new), (new, new), (300, new)], max_new=new)


@pytest.mark.parametrize("window", [0, 2 ** 31 - 1, 2 ** 31 - 40])
@pytest.mark.parametrize("new", [1, 5, 100])
def test_attention_of_the_widest_windows(cuda, window, new):
    check_attention(BF16, 8, 2, 64, 16, "rows", window, [(new // 2, new), (300, new), (new, new)])


@pytest.mark.parametrize("new,dim", [(1, 128), (3, 64), (6, 128), (140, 128), (300, 64)])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("order", ["rows", "heads"])
def test_attention_rows_before_a_broken_token(cuda, new, dim, window, order):
    """Groups of keys and values that are NaN reach the rows that see them and no others."""
    g = torch.Generator().manual_seed(5)
    heads, kv_heads, page, n = 8, 2, 16, 400
    table = tables(g, [n], page, 40)
    q = torch.randn(new, heads, dim, generator=g).to(BF16)
    starts, lens = starts_of([new]), torch.tensor([n], dtype=torch.int32)
    for where in (n - new // 2 - 1, n - 1, n - new - 30):
        for which in range(2):
            k, v = pool(g, 40, page, kv_heads, dim, BF16, order)
            (k, v)[which][int(table[0, where // page]), where % page, 1, dim // 2 + 4:dim // 2 + 8] = 0xff   # columns 32 to 63
            got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), lens.cuda(), starts.cuda(), dim ** -0.5, window=window).cpu().double()
            want, off = oracle.attention(q, codes.decode(k, BF16), codes.decode(v, BF16), table, [n], starts, dim ** -0.5, window)
            at = torch.arange(n - new, n)
            sees = (at >= where) & ((at < where + window) if window else torch.ones_like(at, dtype=torch.bool))
            fine = torch.ones(new, heads, dim, dtype=torch.bool)
            fine[sees, heads // 2:, 32:64 if which else None] = False
            if not which:
                fine[sees, heads // 2:] = False
            assert ((got - want).abs() <= off)[fine].all(), (where, which)
            assert torch.isnan(got[~fine]).all()


@pytest.mark.parametrize("new,heads", [(1, 8), (20, 8), (70, 8), (9, 2)])
def test_attention_blocks_with_broken_tokens(cuda, new, heads):
    """Enough sequences for whole blocks in a CTA: broken values in the last new token of every third sequence stay with its row."""
    g = torch.Generator().manual_seed(9)
    kv_heads, dim, page, seqs = 2, 64, 32, 90
    lens = [new + 40 + 7 * (i % 5) for i in range(seqs)]
    pages = sum(-(-n // page) for n in lens)
    table, starts = tables(g, lens, page, pages), starts_of([new] * seqs)
    q = torch.randn(seqs * new, heads, dim, generator=g).to(BF16)
    k, v = pool(g, pages, page, kv_heads, dim, BF16, "rows")
    for i in range(0, seqs, 3):
        v[int(table[i, (lens[i] - 1) // page]), (lens[i] - 1) % page, 0, 32:36] = 0xff   # columns 0 to 31
    got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts.cuda(), dim ** -0.5,
                                   max_new=new).cpu().double()
    want, off = oracle.attention(q, codes.decode(k, BF16), codes.decode(v, BF16), table, lens, starts, dim ** -0.5, 0)
    fine = torch.ones(want.shape, dtype=torch.bool)
    fine[new - 1::3 * new, :heads // 2, :32] = False
    assert ((got - want).abs() <= off)[fine].all()
    assert torch.isnan(got[~fine]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("page,order", [(16, "rows"), (32, "heads"), (20, "rows"), (16, "wide")])
@pytest.mark.parametrize("new,heads,dim,extra", [(1, 8, 128, 1), (1, 8, 64, 1), (2, 8, 64, 1), (3, 8, 128, 1), (6, 8, 64, 1), (16, 8, 128, 1), (40, 8, 64, 1), (140, 8, 128, 1),
                                                 (140, 8, 128, 1 << 30), (150, 8, 64, 1), (150, 8, 64, 1 << 30), (17, 40, 64, 1)])
@pytest.mark.parametrize("window", [0, 3, 40])
def test_attention_beside_broken_groups(cuda, dtype, page, order, new, heads, dim, extra, window):
    """Broken groups of keys or values, several of them and in two pages, also behind the last key of a sequence and before the windows: rows that must not see them are what they are without.
    Blocks of 8 and of 16 rows, tiles that make numbers of codes and tiles that read them made, pages that boxes serve and others."""
    g = torch.Generator().manual_seed(new * 7 + dim + page)
    kv_heads, n, pages = 2, 400, 60
    table = tables(g, [n, n - 77], page, pages, 1 if extra == 1 else extra // (page * kv_heads * dim * 4) // 2)
    q = torch.randn(2 * new, heads, dim, generator=g).to(dtype)
    starts, lens = starts_of([new, new]), torch.tensor([n, n - 77], dtype=torch.int32)
    for wheres in ((n - new // 2 - 1,), (n - 1, n - new - 30), (n - new - 41, n - new - 42, n - 3), (n - new, n - new // 3 - 1)):
        for which in range(2):
            k, v = pool(g, pages, page, kv_heads, dim, dtype, order)
            hide(k, table, lens.tolist()), hide(v, table, lens.tolist())
            for where in wheres:
                (k, v)[which][int(table[0, where // page]), where % page, 1, dim // 2 + 4:dim // 2 + 8] = 0xff   # columns 32 to 63
            got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), lens.cuda(), starts.cuda(), dim ** -0.5, window=window, max_new=new).cpu().double()
            want, off = oracle.attention(q, codes.decode(k, dtype), codes.decode(v, dtype), table, lens.tolist(), starts, dim ** -0.5, window)
            at = torch.arange(n - new, n)[:, None]
            broken = torch.tensor(wheres)
            sees = ((at >= broken) & ((at < broken + window) if window else torch.ones((), dtype=torch.bool))).any(1)
            fine = torch.ones(2 * new, heads, dim, dtype=torch.bool)
            fine[:new][sees, heads // 2:, 32 if which else 0:64 if which else dim] = False
            assert ((got - want).abs() <= off)[fine].all(), (wheres, which)
            assert torch.isnan(got[~fine]).all(), (wheres, which)


@pytest.mark.parametrize("dtype,size", [(BF16, 2.0 ** 124), (BF16, 2.0 ** -100), (BF16, 2.0 ** -70), (F16, 2.0 ** 13), (F16, 2.0 ** -14)])
@pytest.mark.parametrize("new,heads", [(1, 4), (4, 8), (150, 8)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_large_and_small_values(cuda, dtype, size, new, heads, dim):
    """Means of values near the ends of the type stay in it and keep their bits.  Probabilities of bf16 rows carry 2^-40, the largest of a row's is that at least: a product
    or sum that 32 bits lose behind their lowest exponent is below 2^-126, so each key takes at most 2^-86 off a quotient, whatever its size is."""
    g = torch.Generator().manual_seed(31)
    lens, page = [300, new + 7], 16
    table, starts = tables(g, lens, page, 50), starts_of([new, new])
    k, _ = pool(g, 50, page, 2, dim, dtype, "rows")
    v = rows_in((torch.randn(50, page, 2, dim, generator=g).clamp(-3.9, 3.9) * size).to(dtype), "rows", dtype)
    q = torch.randn(2 * new, heads, dim, generator=g).to(dtype)
    got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts.cuda(), dim ** -0.5,
                                   max_new=new).cpu().double()
    want, off = oracle.attention(q, codes.decode(k, dtype), codes.decode(v, dtype), table, lens, starts, dim ** -0.5, 0)
    lost = 2.0 ** -86 * max(lens) if dtype == BF16 else 0.0
    assert ((got - want).abs() <= off + lost).all()


@pytest.mark.parametrize("dtype,size", [(BF16, 2.0 ** 19), (BF16, 2.0 ** 100), (F16, 2.0 ** 12)])
@pytest.mark.parametrize("new,heads,extra", [(1, 4, 1), (4, 8, 1), (150, 8, 1), (150, 8, 400000)])
def test_attention_of_large_keys(cuda, dtype, size, new, heads, extra):
    """Keys whose steps are beyond 2^15 behind ones whose steps are not, queries to match."""
    g = torch.Generator().manual_seed(33)
    lens, page = [300, new + 7], 16
    table, starts = tables(g, lens, page, 50, extra), starts_of([new, new])
    x = torch.randn(50, page, 2, 64, generator=g)
    x[:, ::3] *= 1.0 / 1024
    k, v = rows_in((x.clamp(-3.9, 3.9) * size).to(dtype), "rows", dtype), pool(g, 50, page, 2, 64, dtype, "rows")[1]
    q = (torch.randn(2 * new, heads, 64, generator=g) / size).to(dtype)
    got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts.cuda(), 0.125, max_new=new).cpu().double()
    want, off = oracle.attention(q, codes.decode(k, dtype), codes.decode(v, dtype), table, lens, starts, 0.125, 0)
    assert ((got - want).abs() <= off).all()


@pytest.mark.parametrize("dtype,scale", [(BF16, 2.0 ** 64), (BF16, 2.0 ** -60), (F16, 2.0 ** 10)])
@pytest.mark.parametrize("new,extra", [(1, 1), (9, 1), (150, 1), (150, 400000)])
def test_attention_of_large_and_small_scales(cuda, dtype, scale, new, extra):
    """Queries that the scale makes ordinary ones."""
    g = torch.Generator().manual_seed(35)
    lens, page = [300, new + 7], 16
    table, starts = tables(g, lens, page, 50, extra), starts_of([new, new])
    k, v = pool(g, 50, page, 2, 64, dtype, "rows")
    q = (torch.randn(2 * new, 8, 64, generator=g) / scale / 8).to(dtype)
    got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts.cuda(), scale, max_new=new).cpu().double()
    want, off = oracle.attention(q, codes.decode(k, dtype), codes.decode(v, dtype), table, lens, starts, scale, 0)
    assert ((got - want).abs() <= off).all()


STEEP = {"one": [(300, 1), (77, 1), (1000, 1)], "drafts": [(300, 4), (80, 3), (4, 4)], "portion": [(300, 150), (150, 150), (700, 33)],
         "many": [(90 + 7 * (i % 5), 1 + i % 20) for i in range(60)]}


@pytest.mark.parametrize("dtype,q_size,k_size", [(F16, 2.0 ** 8, 2.0 ** 8), (F16, 2.0 ** 13, 2.0 ** 13), (F16, 2.0 ** 15, 2.0 ** 15), (BF16, 2.0 ** 12, 2.0 ** 14), (BF16, 2.0 ** 27, 2.0 ** 27),
                                                 (BF16, 2.0 ** 34, 2.0 ** 34), (BF16, 2.0 ** 50, 2.0 ** 58)])
@pytest.mark.parametrize("seqs", list(STEEP))
@pytest.mark.parametrize("extra", [1, 400000])
def test_attention_of_large_scores(cuda, dtype, q_size, k_size, seqs, extra):
    """Queries of +-q_size in every column, key j k_size * (1 + (j * 37 % 7) / 128) in every column, which 4 bits hold exactly (a step of zero): products and sums of powers of two times whole
    numbers below 2^8 are exact in 32 bits, and two scores are the same number or 2^9 apart at least: a row is the mean of the values of its highest scores.  2^-21 covers the
    exponentials' own error, a half step of the type the rounding of equal ones where it is not theirs; sums add a unit for each key, the result is rounded once."""
    g = torch.Generator().manual_seed(21)
    seqs = STEEP[seqs]
    lens, new = [n for n, _ in seqs], [m for _, m in seqs]
    table, starts = tables(g, lens, 16, sum(-(-n // 16) for n in lens) + 2, extra // len(seqs)), starts_of(new)
    k = torch.zeros(sum(-(-n // 16) for n in lens) + 2, 16, 2, 64, dtype=dtype)
    step = lambda j: 1.0 + (j * 37 % 7) / 128.0  # noqa: E731
    for b, n in enumerate(lens):
        for j in range(n):
            k[int(table[b, j // 16]), j % 16] = k_size * step(j)
    v = rows_in(torch.randn(k.shape, generator=g).to(dtype), "rows", dtype)
    k = rows_in(k, "rows", dtype)
    hide(k, table, lens)
    hide(v, table, lens)
    sign = torch.tensor([1.0, -1.0] * 4)
    q = (sign[:, None] * q_size).expand(sum(new), 8, 64).contiguous().to(dtype)
    got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts.cuda(), 1.0, max_new=max(new)).cpu().double()
    vv = codes.decode(v, dtype)
    for b, (n, m) in enumerate(seqs):
        x = oracle.rows_of(vv, table, b, n)
        c = torch.tensor([step(j) for j in range(n)], dtype=torch.float64)
        seen = torch.arange(n)[None] <= torch.arange(n - m, n)[:, None]
        for h in range(8):
            s = torch.where(seen, c * float(sign[h]), -math.inf)
            p = (s == s.amax(1, keepdim=True)).double()
            p /= p.sum(1, keepdim=True)
            o, spread = p @ x[:, h // 4], p @ x[:, h // 4].abs()
            err = spread * (2.0 ** -21 + oracle.EPS[dtype] / 2 + 2 * (n + 64) * 2.0 ** -24)
            assert ((got[int(starts[b]):int(starts[b + 1]), h] - o).abs() <= err + oracle.half_step(o.abs() + err, dtype)).all(), (b, h)


@pytest.mark.parametrize("new", [1, 5, 150])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_with_equal_rows_and_large_scores(cuda, dtype, new):
    """One score far above the others, and all of them equal: no overflow, no loss."""
    g = torch.Generator().manual_seed(6)
    k = torch.randn(20, 16, 1, 128, generator=g).to(dtype)
    v = rows_in(torch.randn(20, 16, 1, 128, generator=g).to(dtype), "rows", dtype)
    table = tables(g, [300], 16, 20)
    k[int(table[0, 3]), 5] = 30.0
    k = rows_in(k, "rows", dtype)
    q = torch.full((new, 2, 128), 2.0).to(dtype)
    q[new // 2:] = 0.0
    starts, lens = starts_of([new]), torch.tensor([300], dtype=torch.int32)
    want, off = oracle.attention(q, codes.decode(k, dtype), codes.decode(v, dtype), table, [300], starts, 1.0, 0)
    got = ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), lens.cuda(), starts.cuda(), 1.0).cpu().double()
    assert ((got - want).abs() <= off).all()


def test_offsets_beyond_32_bits(cuda):
    """A pool of more than 2^32 bytes a cache, rows at its far end."""
    page, kv_heads, dim, heads, n = 64, 8, 128, 32, 150
    pages = (1 << 32) // (page * kv_heads * 80) + 200
    g = torch.Generator().manual_seed(8)
    k, v = (torch.empty(pages, page, kv_heads, 80, dtype=torch.uint8, device="cuda") for _ in range(2))
    ids = torch.tensor([pages - 1, pages - 90, pages - 3], dtype=torch.int32)
    hk, hv = pool(g, 3, page, kv_heads, dim, BF16, "rows")
    for i, p in enumerate(ids.tolist()):
        k[p], v[p] = hk[i].cuda(), hv[i].cuda()
    small = torch.arange(3, dtype=torch.int32)[None]
    for new in (1, 5, 140):
        qkv = torch.randn(new, (heads + 2 * kv_heads) * dim, generator=g).to(BF16)
        place = torch.arange(n - new, n, dtype=torch.int32)
        q = ops.qkv_axes_rope_append_int4(qkv.cuda(), torch.zeros(1, new, dtype=torch.int32).cuda(), torch.ones(64, dtype=torch.float64).cuda(),
                                          torch.zeros(64, dtype=torch.int32).cuda(), torch.zeros(new, dtype=torch.int32).cuda(), place.cuda(), ids[None].cuda(), k, v, heads)
        hk.view(-1, kv_heads, 80)[n - new:n] = codes.encode(qkv[:, heads * dim:(heads + kv_heads) * dim].view(new, kv_heads, dim), BF16)
        hv.view(-1, kv_heads, 80)[n - new:n] = codes.encode(qkv[:, (heads + kv_heads) * dim:].view(new, kv_heads, dim), BF16)
        got = ops.paged_attention_int4(q, k, v, ids[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda(), starts_of([new]).cuda(), dim ** -0.5)
        kk, vv = codes.decode(hk, BF16), codes.decode(hv, BF16)
        want, off = oracle.attention(qkv[:, :heads * dim].reshape(new, heads, dim), kk, vv, small, [n], starts_of([new]), dim ** -0.5, 0)
        assert ((got.cpu().double().view(new, heads, dim) - want).abs() <= off).all()
        for x, y in zip(ops.int4_cache_values(k, v, BF16, ids.cuda()), (kk, vv)):
            assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("starts,lens", [((-5, 3, 20, 90), (50, 60, 70)), ((0, 0, 60, 60), (-3, 60, 2 ** 31 - 1)), ((2, 10, 11, 2 ** 31 - 1), (0, 5, -2 ** 31))])
@pytest.mark.parametrize("max_new", [1, None])
def test_attention_of_starts_and_lengths_out_of_range(cuda, starts, lens, max_new):
    """Whatever the lengths and starts are, no row outside of q is touched and those of sequences in range are right."""
    g = torch.Generator().manual_seed(14)
    rows, page, dim = 60, 16, 64
    table = torch.randperm(30, generator=g)[:15].view(3, 5).to(torch.int32)
    k, v = pool(g, 30, page, 1, dim, F16, "rows")
    q = torch.randn(rows, 2, dim, generator=g).to(F16)
    out = torch.full((rows + 20, 2, dim), 7.0, dtype=F16, device="cuda")
    ops.paged_attention_int4(q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda(),
                             0.125, max_new=max_new, out=out[:rows])
    out = out.cpu().double()
    assert (out[rows:] == 7.0).all()
    kk, vv = codes.decode(k, F16), codes.decode(v, F16)
    for b in range(3):
        lo, hi = max(starts[b], 0), min(starts[b + 1], rows)
        if lo >= hi or not 0 <= lens[b] <= 80 or starts[b + 1] > rows or starts[b] < 0:
            continue
        want, off = oracle.attention(q[lo:hi], kk, vv, table[b:b + 1], [lens[b]], [0, hi - lo], 0.125, 0)
        assert ((out[lo:hi] - want).abs() <= off).all()


def test_no_rows_and_odd_forms(cuda):
    k = torch.zeros(2, 16, 1, 40, dtype=torch.uint8, device="cuda")
    table, lens = torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    q = torch.zeros(0, 64, dtype=BF16, device="cuda")
    assert ops.paged_attention_int4(q, k, k, table, lens, torch.zeros(2, dtype=torch.int32).cuda(), 1.0).shape == (0, 64)
    assert ops.qkv_axes_rope_append_int4(torch.zeros(0, 192, dtype=BF16).cuda(), torch.zeros(1, 0, dtype=torch.int32).cuda(), torch.ones(1, dtype=torch.float64).cuda(),
                                         torch.zeros(1, dtype=torch.int32).cuda(), lens[:0], lens[:0], table, k, k, 1).shape == (0, 64)
    assert ops.int4_cache_values(k, None, BF16, lens[:0]).shape == (0, 16, 1, 64)


@pytest.mark.parametrize("heads,kv_heads,new", [(8, 2, 1), (12, 4, 4), (16, 2, 40), (160, 1, 2)])
def test_attention_in_place(cuda, heads, kv_heads, new):
    g = torch.Generator().manual_seed(17)
    k, v = pool(g, 40, 16, kv_heads, 64, BF16, "rows")
    table, lens, starts = tables(g, [200, 300], 16, 40).cuda(), torch.tensor([200, 300], dtype=torch.int32).cuda(), starts_of([new, new]).cuda()
    q = torch.randn(2 * new, heads, 64, generator=g).to(BF16).cuda()
    want = ops.paged_attention_int4(q, k.cuda(), v.cuda(), table, lens, starts, 0.125, max_new=new)
    mixed = starts_of([1, new]).cuda()
    both = ops.paged_attention_int4(q, k.cuda(), v.cuda(), table, lens, mixed, 0.125)
    x = q.clone()
    got = ops.paged_attention_int4(q, k.cuda(), v.cuda(), table, lens, starts, 0.125, max_new=new, out=q)
    assert got is q and torch.equal(got, want)
    assert torch.equal(ops.paged_attention_int4(x, k.cuda(), v.cuda(), table, lens, mixed, 0.125, out=x)[:1 + new], both[:1 + new])


def test_attention_replayed_with_other_lengths(cuda):
    """A graph takes lengths, starts and pages as they are when it is replayed, whichever kernels the sequences' rows go to."""
    g = torch.Generator().manual_seed(12)
    k, v = pool(g, 120, 16, 2, 64, BF16, "rows")
    kd, vd, kk, vv = to_gpu(k), to_gpu(v), codes.decode(k, BF16), codes.decode(v, BF16)
    q = torch.randn(260, 4, 64, generator=g).to(BF16)
    for width in (50, 200000):
        table, lens, starts = torch.full((4, width), -1, dtype=torch.int32).cuda(), torch.zeros(4, dtype=torch.int32).cuda(), torch.zeros(5, dtype=torch.int32).cuda()
        out, dq, graph = torch.zeros_like(q).cuda(), q.cuda(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention_int4(dq, kd, vd, table, lens, starts, 0.125, out=out)
        for shares in ((65, 65, 65, 65), (1, 257, 0, 2), (0, 0, 3, 1), (260, 0, 0, 0)):
            n = [m + 100 * (i + 1) for i, m in enumerate(shares)]
            t, s = tables(g, n, 16, 120, extra=0), starts_of(shares)
            table[:, :t.shape[1]].copy_(t)
            lens.copy_(torch.tensor(n, dtype=torch.int32))
            starts.copy_(s)
            out.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            used = int(s[-1])
            want, off = oracle.attention(q, kk, vv, t, n, s, 0.125, 0)
            got = out.cpu().double()
            assert ((got - want).abs() <= off)[:used].all() and (got[used:] == 7.0).all()


# ---- as a program uses them ----------------------------------------------------------------------------------------------------
class Step(WideStep):
    """Rows of three users through the operators of a step: append, attend, from the last rows logits that are adjusted and become the target's probabilities, verify."""

    def __init__(self, seed, new=(3, 3, 130), before=(100, 40, 0)):
        super().__init__(seed, new=new, before=before)
        g = torch.Generator().manual_seed(seed + 100)
        self.k, self.v = pool(g, 60, 16, 2, 128, BF16, "heads")
        self.head = (torch.randn(1024, 9000, generator=g) * 0.2).to(BF16)
        self.last = (self.starts[1:, None] - 3 + torch.arange(3)).reshape(-1).long()
        self.words_of = torch.randint(0, 9000, (3, 200), generator=g, dtype=torch.int32)
        self.token_seq = torch.arange(3, dtype=torch.int32).repeat_interleave(3)
        self.token_lens = torch.tensor([50, 51, 52, 0, 1, 2, 198, 199, 200], dtype=torch.int32)
        self.prompt = torch.tensor([20] * 3 + [0] * 3 + [150] * 3, dtype=torch.int32)
        self.settings = torch.tensor([[1.2] * 3 + [1.0] * 3 + [0.9] * 3, [0.5] * 9, [0.1] * 9, [0.7] * 3 + [0.0] * 3 + [1.3] * 3])
        self.mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (2, 282), generator=g, dtype=torch.int32)
        self.mask_row = torch.tensor([0, 0, 0, 1, 1, 1, -1, -1, -1], dtype=torch.int32)
        self.dev = {n: x.cuda() for n, x in vars(self).items() if isinstance(x, torch.Tensor)}
        self.dev["k"], self.dev["v"] = to_gpu(self.k), to_gpu(self.v)

    def run(self):
        d = self.dev
        q = ops.qkv_axes_rope_append_int4(d["qkv"], d["pos"], d["freq"], d["axis"], d["seq"], d["place"], d["table"], d["k"], d["v"], self.heads, pdl=True)
        o = ops.paged_attention_int4(q, d["k"], d["v"], d["table"], d["lens"], d["starts"], self.dim ** -0.5)
        logits = torch.mm(o[d["last"]], d["head"])
        s = d["settings"]
        z = ops.adjust_logits(logits, tokens=d["words_of"], token_seq=d["token_seq"], token_lens=d["token_lens"], prompt_lens=d["prompt"], repetition=s[0], frequency=s[1],
                              presence=s[2], temperature=s[3], mask=d["mask"], mask_row=d["mask_row"], out_dtype=torch.float32)
        target = torch.softmax(z, -1).view(3, 3, 9000)
        return (q, o, logits, z, target) + ops.verify_drafts(target, d["draft"], d["words"], d["accept"], d["sample"])

    def check(self, got):
        want_q, want_k, want_v, off_q, off_k = oracle.axes_rope(self.qkv, self.pos, self.freq, self.axis, 8, 2, 128, False, 1.0)
        q, kb, vb = got[0].cpu().view(want_q.shape), self.dev["k"].cpu(), self.dev["v"].cpu()
        assert ((q.double() - want_q).abs() <= off_q).all()
        kc, vc = codes.decode(kb, BF16), codes.decode(vb, BF16)
        far_k = codes.off_by(kb, BF16)
        for i, (s, p) in enumerate(zip(self.seq.tolist(), self.place.tolist())):
            at = (int(self.table[s, p // 16]), p % 16)
            assert ((kc[at].double() - want_k[i]).abs() <= off_k[i] + far_k[at]).all()
            assert torch.equal(vb[at], codes.encode(want_v[i].to(BF16), BF16))
        want, off = oracle.attention(q, kc, vc, self.table, self.lens.tolist(), self.starts, self.dim ** -0.5, 0)
        assert ((got[1].cpu().double().view(want.shape) - want).abs() <= off).all()
        z, far = codes.adjust(got[2].cpu(), torch.float32, tokens=self.words_of, token_seq=self.token_seq, token_lens=self.token_lens, prompt_lens=self.prompt,
                              repetition=self.settings[0], frequency=self.settings[1], presence=self.settings[2], temperature=self.settings[3], mask=self.mask,
                              mask_row=self.mask_row)
        z, y = torch.from_numpy(z), got[3].cpu().double()
        assert torch.equal(z == -math.inf, y == -math.inf)
        assert ((z - y).abs() <= torch.from_numpy(far))[z > -math.inf].all()
        a, t = oracle.verify(got[4].cpu(), self.draft, self.words, self.accept, self.sample, None)
        assert got[5].tolist() == a.tolist() and got[6].tolist() == t.tolist()


def test_step(cuda):
    s = Step(0)
    s.check(s.run())


def test_step_captured_and_replayed(cuda):
    """The first step of these sizes inside a capture; replays with other inputs, and two graphs in turn."""
    steps = [Step(1, new=(3, 4, 97), before=(61, 77, 5)), Step(2, new=(3, 3, 3), before=(200, 3, 0))]
    torch.mm(steps[0].dev["head"][:9, :64].t(), steps[0].dev["head"][:9, :64])   # the library's handle is made outside of the capture
    graphs, outs = [], []
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.run())
        graphs.append(graph)
    for turn in range(3):
        for s in steps:
            s.qkv = torch.randn(s.qkv.shape, generator=torch.Generator().manual_seed(turn)).to(BF16)
            s.dev["qkv"].copy_(s.qkv)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s, out in zip(steps, outs):
            s.check(out)


def test_steps_on_streams(cuda):
    steps = [Step(i, new=(4, 200, 150), before=(300, 0, 70)) for i in range(3, 6)]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                outs.append(s.run())
    torch.cuda.synchronize()
    for s, out in zip(steps, outs):
        s.check(out)


def test_same_call_same_bits(cuda):
    s = Step(9, new=(5, 90, 64), before=(150, 0, 20))
    first = [x.clone() for x in s.run()]
    for _ in range(5):
        for a, b in zip(first, s.run()):
            assert torch.equal(a, b)


def test_both_ways_from_tensors_to_launches(cuda, monkeypatch):
    s = Step(11)
    d = dict(s.dev)
    d["q"] = torch.randn(s.qkv.shape[0], 8 * 128, device="cuda").to(BF16)
    d["pages"] = torch.tensor([4, 0, 59, 60], dtype=torch.int32).cuda()

    def append(**kw):
        e = dict(d, **kw)
        return lambda: ops.qkv_axes_rope_append_int4(e["qkv"], e["pos"], e["freq"], e["axis"], e["seq"], e["place"], e["table"], e["k"], e["v"], e.get("heads", 8),
                                                     layout=e.get("layout", 0), mscale=e.get("mscale", 1), pdl=e.get("pdl", False))

    def attend(**kw):
        e = dict(d, **kw)
        return lambda: ops.paged_attention_int4(e["q"], e["k"], e["v"], e["table"], e["lens"], e["starts"], e.get("scale", 0.1), window=e.get("window", 0),
                                                max_new=e.get("max_new"), out=e.get("out"), pdl=e.get("pdl", False))

    def values(**kw):
        e = dict(d, **kw)
        return lambda: ops.int4_cache_values(e["k"], e["v"], e.get("dtype", BF16), e["pages"], pdl=e.get("pdl", False))

    wide = torch.cat([d["qkv"], d["qkv"]], 1)[:, :12 * 128]
    for kw in (dict(), dict(mscale=1.5), dict(layout=1, pdl=True), dict(qkv=wide)):
        both_ways(monkeypatch, append(**kw))
    both_ways(monkeypatch, append(qkv=d["qkv"].as_subclass(Own)), served=False)
    for kw in (dict(layout=2), dict(qkv=wide[:, :-1]), dict(axis=d["axis"][1:]), dict(k=d["k"].view(torch.int8)), dict(freq=d["freq"].float()), dict(heads=7),
               dict(k=d["k"][..., :40], v=d["v"][..., :40]), dict(table=d["table"][:, ::2])):
        both_ways(monkeypatch, append(**kw), served="layout" in kw, refused=True)
    out = torch.zeros_like(d["q"])
    for kw in (dict(), dict(q=d["q"].view(-1, 8, 128)), dict(window=7, max_new=130, pdl=True), dict(out=out), dict(scale=1)):
        both_ways(monkeypatch, attend(**kw))
    both_ways(monkeypatch, attend(table=d["table"].as_subclass(Own)), served=False)
    for kw in (dict(scale=-1.0), dict(window=-1), dict(q=d["q"][:, :100]), dict(lens=d["lens"][1:]), dict(max_new=0), dict(out=out.float()), dict(q=d["q"].float()),
               dict(k=d["k"][:, :, :1].expand(d["k"].shape)), dict(v=d["v"].cpu())):
        both_ways(monkeypatch, attend(**kw), served=kw.get("scale", 0) < 0 or "window" in kw, refused=True)
    for kw in (dict(), dict(v=None), dict(pages=None), dict(dtype=F16, pdl=True)):
        both_ways(monkeypatch, values(**kw))
    both_ways(monkeypatch, values(pages=d["pages"][:0]), served=False)
    for kw in (dict(dtype=torch.float32), dict(pages=d["pages"].long()), dict(v=d["v"][1:]), dict(k=d["k"].cpu())):
        both_ways(monkeypatch, values(**kw), served=False, refused=True)
