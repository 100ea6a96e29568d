"""Attention over a paged cache at the ends of what its types hold: scores and values near the largest numbers, keys and values that are none."""
import math

import pytest
import torch

from tests import paged_oracle as oracle
from tests.test_paged_gpu import hide, on_gpu, pool, starts_of, tables
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
