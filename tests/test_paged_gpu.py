"""Operators over a paged cache on a GPU, against their formulas in 64 bits (paged_oracle)."""
import math

import numpy as np
import pytest
import torch

from tests import paged_oracle as oracle
from zhilight_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def pool(g, pages, page, kv_heads, dim, dtype, order, fill=None):
    """A cache on the host in the order rows, heads (`rows`), heads, rows (`heads`), or K and V of a page behind one another (`both`)."""
    if order == "both":
        x = torch.randn(pages, 2, page, kv_heads, dim, generator=g).to(dtype)
        return x[:, 0], x[:, 1]
    out = []
    for _ in range(2):
        x = torch.randn(*((pages, page, kv_heads, dim) if order == "rows" else (pages, kv_heads, page, dim)), generator=g).to(dtype)
        out.append(x if order == "rows" else x.transpose(1, 2))
    return out


def on_gpu(k, v):
    """The same strides on the device."""
    if k._base is not None and k._base is v._base:
        base = k._base.cuda()
        return base[:, 0], base[:, 1]
    return tuple(x.cuda() if x._base is None else x._base.cuda().transpose(1, 2) for x in (k, v))


def tables(g, lens, page, pages, extra=1):
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(pages, generator=g)[:sum(need)].tolist()
    table = torch.full((len(lens), max(need + [1]) + extra), -7, dtype=torch.int32)
    for b, m in enumerate(need):
        table[b, :m] = torch.tensor(ids[:m], dtype=torch.int32)
        ids = ids[m:]
    return table


def starts_of(new):
    return torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)


def hide(cache, table, lens, value):
    """`value` in every row of the pool that no sequence has."""
    pages, page = cache.shape[:2]
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(n):
            if 0 <= int(table[b, i // page]) < pages:
                used[int(table[b, i // page]), i % page] = True
    cache[~used] = value


# ---- rotation and append -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,half,adjacent,page,order,t", [
    (32, 8, 128, 64, False, 16, "rows", 1), (32, 8, 128, 64, False, 16, "heads", 37), (4, 4, 64, 16, True, 1, "rows", 9), (6, 2, 64, 20, False, 5, "both", 33),
    (7, 1, 72, 13, True, 20, "rows", 12), (3, 3, 8, 4, False, 3, "heads", 5), (2, 1, 64, 0, False, 16, "rows", 4), (64, 8, 128, 48, False, 64, "rows", 70),
    (1, 1, 1024, 512, True, 2, "rows", 3), (1, 1, 256, 128, False, 7, "heads", 300),
    (128, 128, 128, 64, False, 16, "heads", 5), (256, 128, 128, 32, True, 8, "rows", 400), (64, 8, 128, 64, False, 16, "both", 2000)])
def test_append(cuda, dtype, heads, kv_heads, dim, half, adjacent, page, order, t):
    g = torch.Generator().manual_seed(heads * 1000 + t)
    lens = [t, t + 11, 2 * t]
    pages = sum(-(-n // page) for n in lens) + 2
    table = tables(g, lens, page, pages)
    k, v = pool(g, pages, page, kv_heads, dim, dtype, order)
    width = (heads + 2 * kv_heads) * dim
    wide = torch.randn(t, width + 16, generator=g).to(dtype)
    pos = torch.randint(0, 5_000_000, (3, t), generator=g, dtype=torch.int32)
    pos[1] = torch.arange(t)
    axis = torch.randint(0, 3, (half,), generator=g, dtype=torch.int32)
    if half > 4:
        axis[3], axis[4] = -1, 3                                     # axes that do not exist do not turn
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    seq = torch.randint(0, 3, (t,), generator=g, dtype=torch.int32)
    place = torch.tensor([lens[int(s)] - t + i for i, s in enumerate(seq)], dtype=torch.int32)
    if t > 4:
        place[2], seq[3], place[4] = -1, 3, page * table.shape[1]    # nowhere, no such sequence, behind the table
    mscale = 1.25
    want_q, want_k, want_v, off_q, off_k = oracle.axes_rope(wide[:, :width].contiguous(), pos, freq, axis, heads, kv_heads, dim, adjacent, mscale)
    kd, vd = on_gpu(k, v)
    dwide = wide.cuda()
    q = ops.qkv_axes_rope_append(dwide[:, :width], pos.cuda(), freq.cuda(), axis.cuda(), seq.cuda(), place.cuda(), table.cuda(), kd, vd, heads,
                                 layout=ops.ROT_ADJACENT if adjacent else ops.ROT_HALVES, mscale=mscale)
    assert ((q.cpu().double().view(t, heads, dim) - want_q).abs() <= off_q).all()
    ek, ev, ok = k.double().clone(), v.double().clone(), torch.zeros(k.shape, dtype=torch.float64)
    for i in range(t):
        s, p = int(seq[i]), int(place[i])
        if 0 <= s < 3 and 0 <= p < page * table.shape[1] and 0 <= int(table[s, p // page]) < pages:
            at = (int(table[s, p // page]), p % page)
            ek[at], ev[at], ok[at] = want_k[i], want_v[i], off_k[i]
    assert ((kd.cpu().double() - ek).abs() <= ok).all()              # places of no row are as they were
    assert torch.equal(vd.cpu().double(), ev)


def test_append_takes_pages_of_the_table_only(cuda):
    """Page numbers outside the pool take no writes."""
    g = torch.Generator().manual_seed(3)
    k, v = pool(g, 4, 8, 2, 64, BF16, "rows")
    kd, vd = on_gpu(k, v)
    table = torch.tensor([[1, -1], [4, 2 ** 31 - 1]], dtype=torch.int32)
    qkv = torch.randn(4, 8 * 64, generator=g).to(BF16)
    seq, place = torch.tensor([0, 0, 1, 1], dtype=torch.int32), torch.tensor([3, 9, 0, 12], dtype=torch.int32)
    q = ops.qkv_axes_rope_append(qkv.cuda(), torch.zeros(1, 4, dtype=torch.int32).cuda(), torch.ones(32, dtype=torch.float64).cuda(),
                                 torch.zeros(32, dtype=torch.int32).cuda(), seq.cuda(), place.cuda(), table.cuda(), kd, vd, 4)
    assert torch.equal(q.cpu(), qkv[:, :4 * 64])                     # position 0 turns nothing
    k[1, 3], v[1, 3] = qkv[0, 4 * 64:6 * 64].view(2, 64), qkv[0, 6 * 64:].view(2, 64)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


# ---- attention -----------------------------------------------------------------------------------------------------------------
def check_attention(dtype, heads, kv_heads, dim, page, order, window, seqs, seed=0, max_new=None, hidden=math.nan, break_pages=False, behind=3):
    """seqs: [(keys, new tokens)]."""
    g = torch.Generator().manual_seed(seed)
    lens, new = [n for n, _ in seqs], [m for _, m in seqs]
    pages = sum(-(-n // page) for n in lens) + 2
    table = tables(g, lens, page, pages)
    k, v = pool(g, pages, page, kv_heads, dim, dtype, order)
    if break_pages:
        table[0, 0], table[-1, 1] = pages, -1
    hide(k, table, lens, hidden)
    hide(v, table, lens, hidden)
    t = sum(new)
    q = (torch.randn(t + behind, heads, dim, generator=g) * 1.5).to(dtype)
    starts, n = starts_of(new), torch.tensor(lens, dtype=torch.int32)
    want, off = oracle.attention(q, k, v, table, lens, starts, dim ** -0.5, window)
    kd, vd = on_gpu(k, v)
    out = torch.full_like(q, 7.0).cuda()
    got = ops.paged_attention(q.cuda(), kd, vd, table.cuda(), n.cuda(), starts.cuda(), dim ** -0.5, window=window, max_new=max_new, out=out)
    assert got is out
    got = got.cpu().double()
    assert (got[t:] == 7.0).all()                                    # rows behind the last sequence
    far = (got[:t] - want[:t]).abs() - off[:t]
    assert (far <= 0).all(), (float(far.nan_to_num(1e9).max()), torch.nonzero(~(far <= 0))[:5].tolist())


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(BF16, 32, 8, 128), (F16, 32, 8, 128), (BF16, 16, 16, 64), (F16, 8, 1, 64), (BF16, 28, 4, 128),
                                                      (F16, 20, 1, 128), (BF16, 3, 1, 64), (F16, 40, 1, 128)])
@pytest.mark.parametrize("page,order", [(16, "rows"), (64, "heads"), (20, "both"), (1, "rows"), (256, "rows")])
def test_attention_single_tokens(cuda, dtype, heads, kv_heads, dim, page, order):
    check_attention(dtype, heads, kv_heads, dim, page, order, 0, [(1, 1), (17, 1), (300, 1), (64, 1), (0, 0), (129, 1), (5, 0), (1025, 1)], max_new=1)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(BF16, 32, 8, 128), (F16, 64, 8, 128), (BF16, 8, 8, 64), (F16, 12, 4, 64)])
@pytest.mark.parametrize("window", [0, 1, 50, 1000])
def test_attention_drafts(cuda, dtype, heads, kv_heads, dim, window):
    check_attention(dtype, heads, kv_heads, dim, 16, "rows", window, [(6, 6), (200, 5), (77, 2), (500, 9), (33, 1), (1500, 4), (0, 0), (70, 7)], max_new=9)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,order", [(BF16, 8, 2, 128, 16, "rows"), (F16, 8, 2, 64, 64, "heads"), (BF16, 4, 4, 128, 20, "both"),
                                                                 (F16, 7, 1, 128, 128, "rows"), (BF16, 16, 1, 64, 8, "rows"), (F16, 5, 5, 64, 1, "rows")])
@pytest.mark.parametrize("window", [0, 100, 300])
@pytest.mark.parametrize("seqs", [[(300, 300)], [(700, 130), (1, 1), (129, 129), (513, 257), (40, 0)], [(1000, 64), (65, 65), (128, 128)]])
def test_attention_portions(cuda, dtype, heads, kv_heads, dim, page, order, window, seqs):
    check_attention(dtype, heads, kv_heads, dim, page, order, window, seqs)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,window,seqs", [
    (BF16, 16, 2, 64, 16, 0, [(3000, 1500)]), (F16, 8, 2, 128, 48, 0, [(2111, 700), (1900, 333), (1800, 1)]), (BF16, 8, 2, 128, 20, 900, [(2500, 900), (1111, 40)]),
    (F16, 64, 8, 128, 64, 0, [(1000 + 131 * i, 1 + i % 16) for i in range(10)]), (BF16, 48, 8, 64, 32, 1000, [(2000 + 77 * i, 9 + i) for i in range(6)]),
    (F16, 24, 8, 64, 256, 0, [(3001, 43), (2048, 30), (130, 130), (2500, 12)])])
def test_attention_of_long_stretches(cuda, dtype, heads, kv_heads, dim, page, window, seqs):
    """Enough keys for every CTA to go round its buffers several times, blocks of one and of two tiles, whole and cut."""
    check_attention(dtype, heads, kv_heads, dim, page, "rows", window, seqs, max_new=max(n for _, n in seqs))


@pytest.mark.parametrize("max_new", [1, 3, 20, 200, None])
def test_attention_does_not_depend_on_the_bound_of_new_tokens(cuda, max_new):
    check_attention(BF16, 8, 2, 128, 16, "rows", 0, [(300, 200), (40, 1), (90, 3), (600, 18)], max_new=max_new)


@pytest.mark.parametrize("new", [1, 4, 150])
def test_attention_over_bad_pages(cuda, new):
    """A page number outside the pool reads as rows of zeros."""
    check_attention(F16, 8, 2, 128, 16, "rows", 0, [(200, new), (220, new)], break_pages=True)


@pytest.mark.parametrize("new", [1, 5, 100, 200])
def test_attention_rows_before_the_first_key(cuda, new):
    """More new tokens than keys: the rows before the first key see nothing and give zeros."""
    check_attention(BF16, 8, 2, 64, 16, "rows", 0, [(new // 2, new), (0, new), (new, new)])
    check_attention(BF16, 8, 2, 64, 16, "rows", 3, [(new // 2, new), (0, new), (new, new)])


@pytest.mark.parametrize("hidden", [math.nan, math.inf, -math.inf, 60000.0])
@pytest.mark.parametrize("new", [1, 6, 140])
def test_attention_does_not_read_what_is_hidden(cuda, hidden, new):
    for dtype in (BF16, F16):
        check_attention(dtype, 8, 2, 128, 48, "rows", 0, [(300, new), (145, new), (new, new)], hidden=hidden)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new,dim", [(6, 128), (140, 128), (300, 64)])
@pytest.mark.parametrize("window", [0, 40])
def test_attention_rows_before_a_broken_token(cuda, bad, new, dim, window):
    """Keys and values that are not numbers reach the rows that see them and no others."""
    g = torch.Generator().manual_seed(5)
    heads, kv_heads, page, n = 8, 2, 16, 400
    table = tables(g, [n], page, 40)
    q = torch.randn(new, heads, dim, generator=g).to(BF16)
    starts, lens = starts_of([new]), torch.tensor([n], dtype=torch.int32)
    for where in (n - new // 2, n - 1, n - new - 30):
        for which in range(2):
            k, v = pool(g, 40, page, kv_heads, dim, BF16, "rows")
            (k, v)[which][int(table[0, where // page]), where % page, 1, 5] = bad
            kd, vd = on_gpu(k, v)
            got = ops.paged_attention(q.cuda(), kd, vd, table.cuda(), lens.cuda(), starts.cuda(), dim ** -0.5, window=window).cpu().double()
            want, off = oracle.attention(q, k, v, table, [n], starts, dim ** -0.5, window)
            at = torch.arange(n - new, n)
            sees = (at >= where) & ((at < where + window) if window else torch.ones_like(at, dtype=torch.bool))
            fine = torch.ones(new, heads, dim, dtype=torch.bool)
            fine[sees, heads // 2:, 5 if which else slice(None)] = False
            assert ((got - want).abs() <= off)[fine].all(), (where, which)
            if which:
                assert not torch.isfinite(got[sees][:, heads // 2:, 5]).any()


@pytest.mark.parametrize("new,heads", [(1, 8), (20, 8), (70, 8), (9, 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_blocks_with_broken_tokens(cuda, new, heads, bad):
    """Enough sequences for whole blocks in a CTA: values that are no numbers, in the last new token of every third sequence, stay with its row."""
    g = torch.Generator().manual_seed(9)
    kv_heads, dim, page, seqs = 2, 64, 32, 90
    lens = [new + 40 + 7 * (i % 5) for i in range(seqs)]
    pages = sum(-(-n // page) for n in lens)
    table, starts = tables(g, lens, page, pages), starts_of([new] * seqs)
    q = torch.randn(seqs * new, heads, dim, generator=g).to(BF16)
    k, v = pool(g, pages, page, kv_heads, dim, BF16, "rows")
    for i in range(0, seqs, 3):
        v[int(table[i, (lens[i] - 1) // page]), (lens[i] - 1) % page, 0, 7] = bad
    got = ops.paged_attention(q.cuda(), *on_gpu(k, v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts.cuda(), dim ** -0.5, max_new=new).cpu().double()
    want, off = oracle.attention(q, k, v, table, lens, starts, dim ** -0.5, 0)
    fine = torch.ones(want.shape, dtype=torch.bool)
    fine[new - 1::3 * new, :heads // 2, 7] = False
    assert ((got - want).abs() <= off)[fine].all()
    assert not torch.isfinite(got[~fine]).any()


@pytest.mark.parametrize("page", [4, 8, 12, 20, 24, 28, 40, 48, 56, 72, 100, 136])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_over_pages_of_any_size(cuda, page, dim):
    """Page borders anywhere in the tiles of blocks of one and of two tiles, for more pages than a warp holds the numbers of."""
    seqs = [(2600 + 100 * i, 1 + 5 * i) for i in range(5)] + [(1500, 200), (700, 70)]
    check_attention(BF16, 16, 2, dim, page, "rows", 0, seqs, max_new=200)
    check_attention(F16, 16, 2, dim, page, "heads", 1000, seqs[:4], max_new=16)


@pytest.mark.parametrize("new,heads,kv_heads", [(1, 4, 2), (3, 4, 1), (20, 8, 2)])
def test_attention_of_many_sequences(cuda, new, heads, kv_heads):
    """More sequences than a warp looks at at a time, some without tokens or keys, also at the ends of what is in view."""
    seqs = [(1 + (37 * i) % 150 + new, 1 + i % new) if i % 11 and i not in (127, 128, 255) else (i % 2 * 30, 0) for i in range(300)]
    check_attention(F16, heads, kv_heads, 64, 16, "rows", 0, seqs, max_new=new)
    check_attention(F16, heads, kv_heads, 64, 16, "heads", 33, seqs[:129], max_new=new)


@pytest.mark.parametrize("window", [0, 700])
def test_attention_of_a_sequence_of_many_blocks(cuda, window):
    """Blocks that a warp looks at 32 at a time, beside sequences of a few."""
    check_attention(BF16, 2, 1, 64, 64, "rows", window, [(50, 20), (4500, 4400), (300, 300), (1300, 1200)])


@pytest.mark.parametrize("heads,kv_heads", [(160, 1), (129, 1), (256, 2), (128, 1), (65, 1)])
@pytest.mark.parametrize("new", [1, 3])
def test_attention_of_wide_groups(cuda, heads, kv_heads, new):
    """Groups with more heads than a tile has rows, and those of one token a tile."""
    check_attention(BF16, heads, kv_heads, 64, 16, "rows", 0, [(100, new), (new, new), (300, new)], max_new=new)


def test_attention_with_equal_rows_and_large_scores(cuda):
    """One score far above the others, and all of them equal: no overflow, no loss."""
    g = torch.Generator().manual_seed(6)
    for dtype in (BF16, F16):
        k, v = pool(g, 20, 16, 1, 128, dtype, "rows")
        table = tables(g, [300], 16, 20)
        k[int(table[0, 3]), 5] = 30.0
        q = torch.full((150, 2, 128), 2.0).to(dtype)
        q[75:] = 0.0
        starts, lens = starts_of([150]), torch.tensor([300], dtype=torch.int32)
        want, off = oracle.attention(q, k, v, table, [300], starts, 1.0, 0)
        for rows in (150, 4):
            got = ops.paged_attention(q[-rows:].cuda(), *on_gpu(k, v), table.cuda(), lens.cuda(), starts_of([rows]).cuda(), 1.0).cpu().double()
            assert ((got - want[-rows:]).abs() <= off[-rows:]).all()
        assert ((ops.paged_attention(q[:4].cuda(), *on_gpu(k, v), table.cuda(), (lens - 146).cuda(), starts_of([4]).cuda(), 1.0).cpu().double()
                 - want[:4]).abs() <= off[:4]).all()


def test_offsets_beyond_32_bits(cuda):
    """A pool of more than 2^31 elements a cache, rows at its far end."""
    page, kv_heads, dim, heads, n = 64, 8, 128, 32, 150
    pages = (1 << 31) // (page * kv_heads * dim) + 200
    g = torch.Generator().manual_seed(8)
    k, v = (torch.empty(pages, page, kv_heads, dim, dtype=BF16, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 90, pages - 3]], dtype=torch.int32)
    hk, hv = (torch.randn(3 * page, kv_heads, dim, generator=g).to(BF16) for _ in range(2))
    for i, p in enumerate(table[0].tolist()):
        k[p], v[p] = hk[i * page:(i + 1) * page].cuda(), hv[i * page:(i + 1) * page].cuda()
    small = torch.arange(3, dtype=torch.int32)[None]
    for new in (1, 5, 140):
        qkv = torch.randn(new, (heads + 2 * kv_heads) * dim, generator=g).to(BF16)
        place = torch.arange(n - new, n, dtype=torch.int32)
        q = ops.qkv_axes_rope_append(qkv.cuda(), torch.zeros(1, new, dtype=torch.int32).cuda(), torch.ones(64, dtype=torch.float64).cuda(),
                                     torch.zeros(64, dtype=torch.int32).cuda(), torch.zeros(new, dtype=torch.int32).cuda(), place.cuda(), table.cuda(), k, v, heads)
        hk[n - new:n] = qkv[:, heads * dim:(heads + kv_heads) * dim].view(new, kv_heads, dim)
        hv[n - new:n] = qkv[:, (heads + kv_heads) * dim:].view(new, kv_heads, dim)
        got = ops.paged_attention(q, k, v, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), starts_of([new]).cuda(), dim ** -0.5)
        want, off = oracle.attention(qkv[:, :heads * dim].reshape(new, heads, dim), hk.view(3, page, kv_heads, dim), hv.view(3, page, kv_heads, dim), small, [n],
                                     starts_of([new]), dim ** -0.5, 0)
        assert ((got.cpu().double().view(new, heads, dim) - want).abs() <= off).all()


def test_attention_of_no_rows_and_odd_forms(cuda):
    k = torch.zeros(2, 16, 1, 64, dtype=BF16, device="cuda")
    table, lens = torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    q = torch.zeros(0, 64, dtype=BF16, device="cuda")
    assert ops.paged_attention(q, k, k, table, lens, torch.zeros(2, dtype=torch.int32).cuda(), 1.0).shape == (0, 64)
    assert ops.qkv_axes_rope_append(torch.zeros(0, 192, dtype=BF16).cuda(), torch.zeros(1, 0, dtype=torch.int32).cuda(), torch.ones(1, dtype=torch.float64).cuda(),
                                    torch.zeros(1, dtype=torch.int32).cuda(), lens[:0], lens[:0], table, k, k, 1).shape == (0, 64)


# ---- verification --------------------------------------------------------------------------------------------------------------
def probabilities(g, *shape, sharp=2.0):
    return torch.softmax(torch.randn(*shape, generator=g) * sharp, -1)


@pytest.mark.parametrize("seqs,drafts,vocab", [(1, 1, 5), (3, 4, 100), (7, 3, 32000), (64, 5, 1000), (5, 40, 333), (2, 2, 50257), (3, 8, 128256), (9, 0, 700),
                                               (1, 600, 17), (4, 33, 1), (2, 1, 4097)])
@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("ragged", [True, False])
def test_verification(cuda, seqs, drafts, vocab, given, ragged):
    g = torch.Generator().manual_seed(seqs * 31 + drafts)
    target = probabilities(g, seqs, drafts + 1, vocab)
    draft = torch.softmax(torch.log(target[:, :drafts]) + torch.randn(seqs, drafts, vocab, generator=g) * 0.3, -1)
    drafted = torch.zeros(seqs, drafts, dtype=torch.int32)
    if drafts:
        drafted = torch.multinomial(draft.reshape(-1, vocab), 1, generator=g).reshape(seqs, drafts).to(torch.int32)
    accept, sample = torch.rand(seqs, drafts, generator=g), torch.rand(seqs, generator=g)
    count = torch.randint(-1, drafts + 2, (seqs,), generator=g, dtype=torch.int32) if ragged else None
    for scale in (1.0, 0.0):                                         # random numbers of zero: everything with a probability is taken
        a, t = ops.verify_drafts(target.cuda(), draft.cuda() if given else None, drafted.cuda(), (accept * scale).cuda(), sample.cuda(),
                                 count.cuda() if ragged else None)
        want_a, want_t = oracle.verify(target, draft if given else None, drafted, accept * scale, sample, count)
        assert (a.cpu().numpy() == want_a).all() and (t.cpu().numpy() == want_t).all()


def test_verification_of_ties_and_leftovers(cuda):
    """Running sums that meet the random number, weights that vanish, words and numbers out of range."""
    v = 4096
    flat = torch.full((v,), 1.0 / v)
    one = torch.zeros(v)
    one[77] = 1.0
    empty = torch.zeros(v)
    odd = flat.clone()
    odd[5], odd[6], odd[v - 1] = math.nan, -1.0, math.inf
    rows, drafts, words, accept, sample = [], [], [], [], []

    def add(p0, p1, d, w, u, r):
        rows.append(torch.stack([p0, p1])), drafts.append(d[None]), words.append([w]), accept.append([u]), sample.append(r)

    add(flat, flat, flat, 9, 0.5, 0.5)            # taken; the sum of 2048 words is the number itself: the next word
    add(flat, flat, flat, 9, 1.0, 0.25)           # refused by a tie, nothing is left of the target: its own row
    add(one, flat, flat, 3, 0.0, 0.999)           # a word without a probability is refused at 0 too
    add(flat, one, flat, 3, 0.9, 0.0)             # behind the draft, the only word
    add(flat, flat, flat, v, 0.0, 0.0)            # no such word
    add(flat, flat, flat, -1, 0.0, 1.0)           # none either; a random number of one: the last word
    add(empty, flat, flat, 0, 0.0, 0.5)           # no weight anywhere
    add(odd, flat, empty, 8, 2.0, 0.99)           # what is no number has no weight
    add(flat, odd, flat, 8, 0.3, 1.0)
    target, draft = torch.stack(rows), torch.stack(drafts)
    words, accept, sample = torch.tensor(words, dtype=torch.int32), torch.tensor(accept), torch.tensor(sample)
    for given in (True, False):
        a, t = ops.verify_drafts(target.cuda(), draft.cuda() if given else None, words.cuda(), accept.cuda(), sample.cuda())
        want_a, want_t = oracle.verify(target, draft if given else None, words, accept, sample, None)
        assert a.tolist() == want_a.tolist() and t.tolist() == want_t.tolist()
    assert t.shape == (9, 2) and want_t[6].tolist() == [-1, -1]


def test_verification_of_strided_rows(cuda):
    g = torch.Generator().manual_seed(4)
    wide = probabilities(g, 3, 6, 1003)
    target, draft = wide[:, :3, 1:1002].cuda(), wide[:, 3:5, :1001].cuda()
    words, accept, sample = torch.randint(0, 1001, (3, 2), generator=g, dtype=torch.int32), torch.rand(3, 2, generator=g), torch.rand(3, generator=g)
    a, t = ops.verify_drafts(target, draft, words.cuda(), accept.cuda(), sample.cuda())
    want_a, want_t = oracle.verify(target.cpu(), draft.cpu(), words, accept, sample, None)
    assert a.tolist() == want_a.tolist() and t.tolist() == want_t.tolist()


# ---- as a program uses them ----------------------------------------------------------------------------------------------------
class Step:
    """Rows of three users through the three operators: append, attend, verify."""

    def __init__(self, seed, new=(3, 1, 130), before=(100, 40, 0)):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page = 8, 2, 128, 16
        lens = [a + b for a, b in zip(new, before)]
        t = sum(new)
        self.table = tables(g, lens, 16, 60)
        self.k, self.v = pool(g, 60, 16, 2, 128, BF16, "rows")
        self.qkv = torch.randn(t, 12 * 128, generator=g).to(BF16)
        self.pos = torch.randint(0, 3000, (3, t), generator=g, dtype=torch.int32)
        self.freq = 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
        self.axis = torch.from_numpy(ops.rope_axis_map((16, 24, 24)))
        self.seq = torch.repeat_interleave(torch.arange(3), torch.tensor(new)).to(torch.int32)
        self.place = torch.cat([torch.arange(b, b + a) for a, b in zip(new, before)]).to(torch.int32)
        self.lens, self.starts = torch.tensor(lens, dtype=torch.int32), starts_of(new)
        self.target, self.draft = probabilities(g, 3, 3, 9000), probabilities(g, 3, 2, 9000)
        self.words = torch.randint(0, 9000, (3, 2), generator=g, dtype=torch.int32)
        self.accept, self.sample = torch.rand(3, 2, generator=g) * 1e-3, torch.rand(3, generator=g)
        self.dev = {n: x.cuda() for n, x in vars(self).items() if isinstance(x, torch.Tensor)}

    def run(self):
        d = self.dev
        q = ops.qkv_axes_rope_append(d["qkv"], d["pos"], d["freq"], d["axis"], d["seq"], d["place"], d["table"], d["k"], d["v"], self.heads, pdl=True)
        o = ops.paged_attention(q, d["k"], d["v"], d["table"], d["lens"], d["starts"], self.dim ** -0.5)
        return (q, o) + ops.verify_drafts(d["target"], d["draft"], d["words"], d["accept"], d["sample"])

    def check(self, got):
        want_q, want_k, want_v, off_q, off_k = oracle.axes_rope(self.qkv, self.pos, self.freq, self.axis, 8, 2, 128, False, 1.0)
        q, kc, vc = got[0].cpu().view(want_q.shape), self.dev["k"].cpu(), self.dev["v"].cpu()
        assert ((q.double() - want_q).abs() <= off_q).all()
        for i, (s, p) in enumerate(zip(self.seq.tolist(), self.place.tolist())):
            at = (int(self.table[s, p // 16]), p % 16)
            assert ((kc[at].double() - want_k[i]).abs() <= off_k[i]).all() and torch.equal(vc[at].double(), want_v[i])
        want, off = oracle.attention(q, kc, vc, self.table, self.lens.tolist(), self.starts, self.dim ** -0.5, 0)
        assert ((got[1].cpu().double().view(want.shape) - want).abs() <= off).all()
        a, t = oracle.verify(self.target, self.draft, self.words, self.accept, self.sample, None)
        assert got[2].tolist() == a.tolist() and got[3].tolist() == t.tolist()


def test_step(cuda):
    s = Step(0)
    s.check(s.run())


def test_step_captured_and_replayed(cuda):
    """The first step of these sizes inside a capture; replays with other inputs, and two graphs in turn."""
    steps = [Step(1, new=(2, 1, 97), before=(61, 77, 5)), Step(2, new=(1, 1, 1), before=(200, 3, 0))]
    graphs, outs = [], []
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.run())
        graphs.append(graph)
    for turn in range(3):
        for s, graph, out in zip(steps, graphs, outs):
            s.qkv = torch.randn(s.qkv.shape, generator=torch.Generator().manual_seed(turn)).to(BF16)
            s.dev["qkv"].copy_(s.qkv)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s, out in zip(steps, outs):
            s.check(out)


@pytest.mark.parametrize("rows,max_new", [(12, 4), (260, None)])
def test_attention_replayed_with_other_lengths(cuda, rows, max_new):
    """A graph takes lengths, starts and pages as they are when it is replayed."""
    g = torch.Generator().manual_seed(12)
    heads, kv_heads, dim, page = 4, 2, 64, 16
    k, v = pool(g, 120, page, kv_heads, dim, BF16, "rows")
    kd, vd = on_gpu(k, v)
    q = torch.randn(rows, heads, dim, generator=g).to(BF16)
    steps = []
    for shares in ((rows // 4,) * 4, (1, rows - 3, 0, 2), (0, 0, 3, 1)) if max_new is None else ((3, 3, 3, 3), (1, 4, 0, 2), (4, 4, 4, 0)):
        lens = [n + 100 * (i + 1) for i, n in enumerate(shares)]
        steps.append((tables(g, lens, page, 120, extra=0), lens, starts_of(shares)))
    table, lens, starts = torch.full((4, 50), -1, dtype=torch.int32).cuda(), torch.zeros(4, dtype=torch.int32).cuda(), torch.zeros(5, dtype=torch.int32).cuda()
    out, dq, graph = torch.zeros_like(q).cuda(), q.cuda(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention(dq, kd, vd, table, lens, starts, dim ** -0.5, max_new=max_new, out=out)
    for t, n, s in steps:
        table[:, :t.shape[1]].copy_(t)
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        starts.copy_(s)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        used = int(s[-1])
        want, off = oracle.attention(q, k, v, t, n, s, dim ** -0.5, 0)
        got = out.cpu().double()
        assert ((got - want).abs() <= off)[:used].all() and (got[used:] == 7.0).all()


def test_steps_on_two_streams(cuda):
    steps = [Step(i, new=(4, 200, 150), before=(300, 0, 70)) for i in range(3, 7)]
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
    first = s.run()
    for _ in range(5):
        for a, b in zip(first, s.run()):
            assert torch.equal(a, b)


# ---- the native host module and the general path ---------------------------------------------------------------------------------
class Asked:
    """The native module, with a note of whether it served each call or left it to the general path."""

    def __init__(self, host):
        self.host, self.served = host, []

    def __getattr__(self, name):
        def call(*args):
            y = getattr(self.host, name)(*args)
            self.served.append(y is not None)
            return y
        return call


def both_ways(monkeypatch, f, served=True, refused=False):
    from zhilight_b200 import _lib
    asked, outs = Asked(_lib.host), []
    for host in (asked, None):
        with monkeypatch.context() as m:
            m.setattr(_lib, "host", host)
            if refused:
                with pytest.raises(_lib.ZLError):
                    f()
            else:
                y = f()
                outs.append([x.clone() for x in (y if isinstance(y, tuple) else (y,))])
    assert asked.served == [served]
    for x, y in zip(*outs) if outs else ():
        assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)


class Own(torch.Tensor):
    pass


def test_both_ways_from_tensors_to_launches(cuda, monkeypatch):
    s = Step(11)
    d = dict(s.dev)
    d["q"] = torch.randn(s.qkv.shape[0], 8 * 128, device="cuda").to(BF16)

    def append(**kw):
        e = dict(d, **kw)
        return lambda: ops.qkv_axes_rope_append(e["qkv"], e["pos"], e["freq"], e["axis"], e["seq"], e["place"], e["table"], e["k"], e["v"], e.get("heads", 8),
                                                layout=e.get("layout", 0), mscale=e.get("mscale", 1), pdl=e.get("pdl", False))

    def attend(**kw):
        e = dict(d, **kw)
        return lambda: ops.paged_attention(e["q"], e["k"], e["v"], e["table"], e["lens"], e["starts"], e.get("scale", 0.1), window=e.get("window", 0),
                                           max_new=e.get("max_new"), out=e.get("out"), pdl=e.get("pdl", False))

    def verify(**kw):
        e = dict(d, **kw)
        return lambda: ops.verify_drafts(e["target"], e["draft"], e["words"], e["accept"], e["sample"], e.get("count"), pdl=e.get("pdl", False))

    wide = torch.cat([d["qkv"], d["qkv"]], 1)[:, :12 * 128]
    for kw in (dict(), dict(mscale=1.5), dict(layout=1, pdl=True), dict(qkv=wide), dict(qkv=torch.nn.Parameter(d["qkv"], requires_grad=False))):
        both_ways(monkeypatch, append(**kw))
    both_ways(monkeypatch, append(qkv=d["qkv"].as_subclass(Own)), served=False)
    for kw in (dict(layout=2), dict(qkv=wide[:, :-1]), dict(axis=d["axis"][1:]), dict(k=d["k"].half()), dict(freq=d["freq"].float()), dict(place=d["place"].long()),
               dict(pos=d["pos"][:, 1:]), dict(heads=7), dict(qkv=d["qkv"].cpu()), dict(table=d["table"][:, ::2])):
        both_ways(monkeypatch, append(**kw), served="layout" in kw, refused=True)
    out = torch.zeros_like(d["q"])
    for kw in (dict(), dict(q=d["q"].view(-1, 8, 128)), dict(window=7, max_new=130, pdl=True), dict(out=out), dict(scale=1)):
        both_ways(monkeypatch, attend(**kw))
    both_ways(monkeypatch, attend(table=d["table"].as_subclass(Own)), served=False)
    for kw in (dict(scale=-1.0), dict(window=-1), dict(q=d["q"][:, :100]), dict(lens=d["lens"][1:]), dict(max_new=0), dict(out=out.float()),
               dict(k=d["k"][:, :, :1].expand(d["k"].shape)), dict(starts=d["starts"].long()), dict(v=d["v"].cpu())):
        both_ways(monkeypatch, attend(**kw), served=kw.get("scale", 0) < 0 or "window" in kw, refused=True)
    for kw in (dict(), dict(draft=None), dict(count=d["starts"][1:].clone()), dict(target=torch.cat([d["target"]] * 2, 2)[:, :, :9000])):
        both_ways(monkeypatch, verify(**kw))
    for kw in (dict(target=d["target"].double()), dict(draft=d["target"]), dict(words=d["words"].long()), dict(count=d["starts"]), dict(sample=d["sample"][1:])):
        both_ways(monkeypatch, verify(**kw), served=False, refused=True)
