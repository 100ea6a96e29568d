"""Penalties, biases, temperature and grammar masks on logits on a GPU, against the formula in 64 bits (int4_oracle.adjust)."""
import math

import pytest
import torch

from tests import int4_oracle as oracle
from tests.test_paged_gpu import Own, both_ways
from zhilight_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def settings(g, rows, vocab, seqs, longest, biases, masks, repeated=0.3):
    """Everything at once, on the host: words that come again, words outside the vocabulary, lengths and lists beyond their ends, neutral settings among the others."""
    words = torch.randint(-2, vocab + 2, (seqs, longest), generator=g, dtype=torch.int32)
    again = torch.rand(seqs, longest, generator=g) < repeated
    words[again] = torch.randint(0, min(vocab, 7), (int(again.sum()),), generator=g, dtype=torch.int32)
    counts = torch.randint(0, 2 * biases + 1, (rows,), generator=g)
    counts[::3] = 0
    starts = torch.zeros(rows + 1, dtype=torch.int32)
    starts[1:] = counts.cumsum(0)
    n = int(starts[-1])
    bias = torch.randn(n, generator=g) * 5
    bias[::5] = -100.0
    at = torch.randint(-1, vocab + 1, (n,), generator=g, dtype=torch.int32)
    at[::4] = torch.randint(0, min(vocab, 5), (len(at[::4]),), generator=g, dtype=torch.int32)   # words that are listed more than once
    mix = lambda lo, hi, plain: torch.where(torch.rand(rows, generator=g) < 0.3, plain, lo + (hi - lo) * torch.rand(rows, generator=g))  # noqa: E731
    return dict(tokens=words, token_seq=torch.randint(-1, seqs + 1, (rows,), generator=g, dtype=torch.int32),
                token_lens=torch.randint(-1, longest + 3, (rows,), generator=g, dtype=torch.int32),
                prompt_lens=torch.randint(-1, longest + 3, (rows,), generator=g, dtype=torch.int32), repetition=mix(0.7, 1.5, 1.0), frequency=mix(-0.3, 0.8, 0.0),
                presence=mix(-0.3, 0.8, 0.0), bias_starts=starts, bias_words=at, bias=bias, temperature=mix(0.1, 2.0, 0.0),
                mask=torch.randint(-2 ** 31, 2 ** 31 - 1, (masks, (vocab - 1) // 32 + 2), generator=g, dtype=torch.int32),
                mask_row=torch.randint(-1, masks + 1, (rows,), generator=g, dtype=torch.int32))


def on_gpu(kw):
    return {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in kw.items()}


def check(z, kw, out_dtype=None, got=None):
    kind = out_dtype or z.dtype
    got = (ops.adjust_logits(z.cuda(), out_dtype=out_dtype, **on_gpu(kw)) if got is None else got).cpu()
    assert got.dtype == kind and got.shape == z.shape
    want, off = oracle.adjust(z, kind, **kw)
    want, off, got = torch.from_numpy(want), torch.from_numpy(off), got.double()
    assert torch.equal(torch.isnan(want), torch.isnan(got)) and torch.equal(want == -math.inf, got == -math.inf) and torch.equal(want == math.inf, got == math.inf)
    fine = torch.isfinite(want)
    assert ((want - got).abs() <= off)[fine].all(), float(((want - got).abs() - off)[fine].max())


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, None), (BF16, F32), (F16, None), (F16, F32), (F32, None)])
@pytest.mark.parametrize("rows,vocab,seqs,longest", [(1, 1, 1, 1), (3, 7, 2, 5), (5, 100, 3, 70), (9, 1000, 4, 33), (4, 4099, 4, 700), (2, 32000, 2, 3000), (7, 50257, 3, 257),
                                                     (3, 128256, 2, 5000), (2, 152064, 1, 100)])
def test_adjust(cuda, dtype, out_dtype, rows, vocab, seqs, longest):
    g = torch.Generator().manual_seed(rows * 100 + vocab)
    z = (torch.randn(rows, vocab, generator=g) * 4).to(dtype)
    check(z, settings(g, rows, vocab, seqs, longest, 9, 3), out_dtype)


def test_adjust_of_the_widest_vocabularies(cuda):
    """More words than a cluster has room for at once."""
    g = torch.Generator().manual_seed(1)
    for vocab in (393216, 393248, 900001):
        z = torch.randn(2, vocab, generator=g).to(BF16)
        kw = settings(g, 2, vocab, 2, 3000, 30, 2)
        kw["token_seq"][:], kw["token_lens"][:] = torch.tensor([1, 0]), torch.tensor([3000, 2900])
        check(z, kw, F32)


@pytest.mark.parametrize("only", [(), ("tokens", "token_lens"), ("tokens", "token_lens", "repetition"), ("tokens", "token_lens", "token_seq", "frequency"),
                                  ("tokens", "token_lens", "prompt_lens", "presence"), ("bias_starts", "bias_words", "bias"), ("temperature",), ("mask",),
                                  ("mask", "mask_row", "temperature"), ("bias_starts", "bias_words", "bias", "mask")])
@pytest.mark.parametrize("vocab", [1000, 33000, 33001])
def test_adjust_by_parts(cuda, only, vocab):
    """Each argument alone: the others take no part."""
    g = torch.Generator().manual_seed(vocab)
    z = (torch.randn(6, vocab, generator=g) * 3).to(BF16)
    kw = settings(g, 6, vocab, 8, 400, 12, 7)
    check(z, {n: kw[n] for n in only})


@pytest.mark.parametrize("vocab", [64, 1003, 40000])
def test_adjust_strided_and_in_place(cuda, vocab):
    g = torch.Generator().manual_seed(4)
    for dtype in (BF16, F32):
        wide = (torch.randn(5, vocab + 24, generator=g) * 3).to(dtype)
        kw = settings(g, 5, vocab, 3, 90, 5, 2)
        kw["tokens"] = torch.cat([kw["tokens"]] * 2, 1)[:, :90]
        kw["mask"] = torch.cat([kw["mask"]] * 2, 1)[:, :kw["mask"].shape[1]]
        dev = on_gpu(kw)
        for first in (0, 8, 3):
            z = wide[:, first:first + vocab]
            dz = wide.cuda()[:, first:first + vocab]
            check(z, kw, F32, got=ops.adjust_logits(dz, out_dtype=F32, **dev))
            room = torch.full((5, vocab + 16), 9.0, dtype=dtype, device="cuda")
            got = ops.adjust_logits(dz, out=room[:, 5:vocab + 5], **dev)
            check(z, kw, got=got)
            assert (room[:, :5] == 9.0).all() and (room[:, vocab + 5:] == 9.0).all()
            got = ops.adjust_logits(dz, out=dz, **dev)
            assert got is dz
            check(z, kw, got=got)
            assert torch.equal(dz._base[:, :first].cpu(), wide[:, :first]) and torch.equal(dz._base[:, first + vocab:].cpu(), wide[:, first + vocab:])


def test_adjust_beside_itself(cuda):
    """Out in the same rows as the logits, or in them: refused where a word of one is another one's of the other."""
    g = torch.Generator().manual_seed(14)
    wide = (torch.randn(4, 2100, generator=g) * 3).to(BF16)
    kw = settings(g, 4, 1000, 3, 60, 5, 2)
    dev, dwide = on_gpu(kw), wide.cuda()
    check(wide[:, :1000], kw, got=ops.adjust_logits(dwide[:, :1000], out=dwide[:, 1000:2000], **dev))
    assert torch.equal(dwide[:, :1000].cpu(), wide[:, :1000]) and torch.equal(dwide[:, 2000:].cpu(), wide[:, 2000:])
    flat = torch.zeros(9000, dtype=BF16, device="cuda")
    for x, y in ((flat[:4000].view(4, 1000), flat[8:4008].view(4, 1000)), (flat[:4000].view(4, 1000), flat[3000:7000].view(4, 1000)), (dwide[:, 600:1600], dwide[:, :1000]),
                 (flat[:4000].view(4, 1000), flat[:8000].view(4, 2000)[:, :1000]), (flat[:1000].view(1, 1000), flat[999:1999].view(1, 1000)),
                 (flat[:1000].view(1, 1000), flat[:2000].view(torch.float32).view(1, 1000))):
        with pytest.raises(RuntimeError, match="beside"):
            ops.adjust_logits(x, out=y, out_dtype=y.dtype)
    check(torch.zeros(4, 1000, dtype=BF16), {}, got=ops.adjust_logits(flat[:4000].view(4, 1000), out=flat[4000:8000].view(4, 1000)))


def test_adjust_of_special_numbers(cuda):
    """Infinities and NaN in logits, biases and settings; masks that leave nothing or hide them; empty histories and lists."""
    vocab = 300
    z = torch.zeros(8, vocab)
    z[:, 0], z[:, 1], z[:, 2], z[:, 3], z[:, 4] = math.nan, math.inf, -math.inf, 3.0e38, -1e-42
    z[:, 5:] = torch.randn(8, vocab - 5, generator=torch.Generator().manual_seed(3))
    kw = dict(tokens=torch.arange(20, dtype=torch.int32).expand(1, 20).contiguous(), token_seq=torch.zeros(8, dtype=torch.int32),
              token_lens=torch.tensor([20, 0, 20, 20, 5, 20, 20, 20], dtype=torch.int32), prompt_lens=torch.tensor([20, 0, 0, 10, 0, 0, 0, 0], dtype=torch.int32),
              repetition=torch.tensor([1.3, 1.3, 0.5, 1.0, 2.0, 1e30, 1e-30, 1.0]), frequency=torch.tensor([0.0, 1.0, 0.5, 0.5, 0.0, 0.0, 0.0, math.inf]),
              presence=torch.zeros(8), bias_starts=torch.tensor([0, 0, 3, 3, 3, 3, 3, 3, 4], dtype=torch.int32), bias_words=torch.tensor([1, 9, 9, 40], dtype=torch.int32),
              bias=torch.tensor([-math.inf, math.inf, -1.0, math.nan]), temperature=torch.tensor([0.0, 1.0, -1.0, 1e-30, 1e-40, math.inf, 0.5, math.nan]),
              mask=torch.zeros(3, 10, dtype=torch.int32), mask_row=torch.tensor([0, 1, 2, -1, 3, 1, 2, -5], dtype=torch.int32))
    kw["mask"][1], kw["mask"][2, 0] = -1, ~0b11111
    check(z, kw)
    got = ops.adjust_logits(z.cuda(), **on_gpu(kw)).cpu()
    assert (got[0] == -math.inf).all()                               # a mask that leaves nothing
    assert (got[2, :5] == -math.inf).all() and (got[6, 32:] == -math.inf).all()


@pytest.mark.parametrize("words", ["one", "few", "all"])
@pytest.mark.parametrize("prompt", [0, 30000, 70000])
def test_adjust_of_long_histories(cuda, words, prompt):
    """Counts are whole numbers, however often a word comes."""
    g = torch.Generator().manual_seed(5)
    vocab, n = 32000, 70000
    most = {"one": 1, "few": 40, "all": vocab}[words]
    kw = dict(tokens=torch.randint(0, most, (2, n), generator=g, dtype=torch.int32), token_lens=torch.tensor([n, n - 5], dtype=torch.int32),
              prompt_lens=torch.tensor([prompt, 7], dtype=torch.int32), repetition=torch.tensor([1.1, 1.2]), frequency=torch.tensor([2.0 ** -10, 0.01]),
              presence=torch.tensor([0.5, 0.25]))
    check(torch.randn(2, vocab, generator=g), kw)


def test_adjust_of_long_bias_lists(cuda):
    """More biases than a CTA lists, all in one piece of the vocabulary, words among them twice: one after the other."""
    g = torch.Generator().manual_seed(6)
    vocab, n = 20000, 1500
    for spread in (40, 700, vocab):
        kw = dict(bias_starts=torch.tensor([0, n, n, 2 * n], dtype=torch.int32), bias_words=torch.randint(0, spread, (2 * n,), generator=g, dtype=torch.int32),
                  bias=torch.randn(2 * n, generator=g))
        check(torch.randn(3, vocab, generator=g), kw)
    kw["bias_starts"] = torch.tensor([-4, n, 2 * n + 9, 5], dtype=torch.int32)   # beyond the list's ends, and backwards
    check(torch.randn(3, vocab, generator=g), kw)


@pytest.mark.parametrize("vocab", [1000, 20000])
def test_adjust_of_bias_lists_at_the_ends_of_whole_numbers(cuda, vocab):
    """Starts near the largest and the least whole number count as the list's end and its beginning: none wraps around to a place outside of it."""
    g = torch.Generator().manual_seed(15)
    top, least, n = 2 ** 31 - 1, -2 ** 31, 700
    bias_words, bias = torch.randint(0, vocab, (n,), generator=g, dtype=torch.int32), torch.randn(n, generator=g)
    z = torch.randn(5, vocab, generator=g)
    for starts in ([top] * 6, [least] * 6, [0, top, top, least, least, top], [top - 255, top, 40, n, top - 512, least], [least, top, least + 1, 300, top - 31, n]):
        check(z, dict(bias_starts=torch.tensor(starts, dtype=torch.int32), bias_words=bias_words, bias=bias))


def some_rows(z, kw, rows):
    """The same call for some of its rows, on the host."""
    each = ("token_seq", "token_lens", "prompt_lens", "repetition", "frequency", "presence", "temperature", "mask_row")
    kw = {n: x[rows] if n in each else x for n, x in kw.items()}
    lists = [slice(int(kw["bias_starts"][r]), int(kw["bias_starts"][r + 1])) for r in rows]
    counts = torch.tensor([0] + [x.stop - x.start for x in lists])
    kw.update(bias_words=torch.cat([kw["bias_words"][x] for x in lists]), bias=torch.cat([kw["bias"][x] for x in lists]), bias_starts=counts.cumsum(0).to(torch.int32))
    return z[rows], kw


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, None), (BF16, F32), (F16, None), (F32, None)])
@pytest.mark.parametrize("rows,vocab,longest,first,different,biases", [
    (128, 32000, 9000, 200, 1400, 9), (128, 32000, 9000, 0, 2500, 9), (160, 50257, 9000, 16000, 5300, 9), (128, 32000, 9000, 21400, 5470, 9), (130, 33001, 12000, 10900, 9000, 40),
    (200, 32000, 16000, 0, 16000, 3), (400, 17000, 16000, 5, 16000, 1100), (300, 16384, 20000, 1, 16000, 9)])
def test_adjust_of_many_rows(cuda, dtype, out_dtype, rows, vocab, longest, first, different, biases):
    """Rows enough for wide pieces, histories of thousands of different words side by side: lists of marked words that a thread's registers do not hold, that fill their room,
    and that are too long for it, with counters of 16 and of 32 bits; beside the logits, over them, and from rows that begin anywhere."""
    g = torch.Generator().manual_seed(vocab + different)
    kw = settings(g, rows, vocab, 4, longest, 2, 3)
    for s in range(3):                                               # each of the words once, then some of them again; the last history is as it was
        words = first + torch.randperm(different, generator=g)
        again = words[torch.randint(0, different, (longest - different,), generator=g)]
        kw["tokens"][s] = torch.cat([words, again])[torch.randperm(longest, generator=g)]
    kw["token_seq"] = torch.arange(rows, dtype=torch.int32) % 4
    kw["token_lens"] = torch.where(torch.arange(rows) % 5 == 4, kw["token_lens"], longest).to(torch.int32)
    counts = torch.randint(0, 2 * biases + 1, (rows,), generator=g) * (torch.arange(rows) % 3 > 0)
    counts[1], counts[2] = 2 * biases, biases                        # of words behind the others, where there are any
    kw["bias_starts"][1:] = counts.cumsum(0)
    n = int(counts.sum())
    kw["bias_words"], kw["bias"] = torch.randint(min(first + different, vocab - 9), vocab, (n,), generator=g, dtype=torch.int32), torch.randn(n, generator=g)
    wide = (torch.randn(rows, vocab + 8, generator=g) * 3).to(dtype)
    sample = torch.tensor([0, 1, 2, 3, 4, rows // 2, rows - 2, rows - 1])
    dev, dwide = on_gpu(kw), wide.cuda()
    for at in (0, 3):
        z = wide[:, at:at + vocab]
        z_some, kw_some = some_rows(z, kw, sample)
        dz = dwide[:, at:at + vocab]
        check(z_some, kw_some, out_dtype, got=ops.adjust_logits(dz, out_dtype=out_dtype, **dev)[sample])
        assert torch.equal(dz.cpu(), z)
        if out_dtype is None:
            other, room = ops.adjust_logits(dz, **dev), dwide.clone()
            got = ops.adjust_logits(room[:, at:at + vocab], out=room[:, at:at + vocab], **dev)
            check(z_some, kw_some, got=got[sample])
            assert torch.equal(got.view(torch.int16 if dtype != F32 else torch.int32), other.view(torch.int16 if dtype != F32 else torch.int32))   # every row, NaN or not
            assert torch.equal(room[:, :at], dwide[:, :at]) and torch.equal(room[:, at + vocab:], dwide[:, at + vocab:])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [1003, 40000])
def test_adjust_divides(cuda, dtype, vocab):
    """Quotients by repetition and temperature are 32-bit quotients, rounded once: what torch's division on the host gives, bit by bit."""
    g = torch.Generator().manual_seed(16)
    z = torch.randn(24, vocab, generator=g) * torch.exp2(torch.randint(-3, 6, (24, vocab), generator=g).float())
    z[:, ::50], z[:, 1::50] = math.inf, -math.inf
    z, by = z.to(dtype), 0.05 + torch.rand(24, generator=g) * 2.5
    by[0], by[1], by[2], by[3] = 1.0, 2.0 ** -20, 3.0e20, 1.0 + 2.0 ** -23
    want = z.float() / by[:, None]
    assert torch.equal(ops.adjust_logits(z.cuda(), temperature=by.cuda(), out_dtype=F32).cpu(), want)
    words = torch.arange(vocab, dtype=torch.int32)[None]
    kw = dict(tokens=words, token_seq=torch.zeros(24, dtype=torch.int32), token_lens=torch.full((24,), vocab, dtype=torch.int32), repetition=by)
    want = torch.where(z.float() > 0, want, z.float() * by[:, None])
    assert torch.equal(ops.adjust_logits(z.cuda(), out_dtype=F32, **on_gpu(kw)).cpu(), want)


def test_adjust_leaves_signs_of_zeros(cuda):
    """Logits that nothing applies to are what they were to the last bit, and a quotient of zero has its sign."""
    g = torch.Generator().manual_seed(17)
    z = torch.randn(4, 1000, generator=g)
    z[:, ::7], z[:, 3::7] = 0.0, -0.0
    assert torch.equal(ops.adjust_logits(z.cuda()).cpu().view(torch.int32), z.view(torch.int32))
    by = torch.tensor([0.0, 0.3, 1.0, 7.0])
    want = torch.where(by[:, None] > 0, z / by[:, None], z)
    assert torch.equal(ops.adjust_logits(z.cuda(), temperature=by.cuda()).cpu().view(torch.int32), want.view(torch.int32))


def test_adjust_without_rows_or_histories(cuda):
    z = torch.randn(3, 40, device="cuda")
    none = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    lens, one = torch.full((3,), 5, dtype=torch.int32).cuda(), torch.full((3,), 2.0).cuda()
    assert torch.equal(ops.adjust_logits(z, tokens=none, token_lens=lens, repetition=one), z)
    assert torch.equal(ops.adjust_logits(z, bias_starts=torch.zeros(4, dtype=torch.int32).cuda(), bias_words=none[0], bias=none[0].float()), z)
    assert ops.adjust_logits(z[:0]).shape == (0, 40)


def test_adjust_captured_and_on_streams(cuda):
    """A graph takes lengths and settings as they are when it is replayed; calls on several streams at once."""
    g = torch.Generator().manual_seed(7)
    vocab, rows = 9000, 6
    cases = [((torch.randn(rows, vocab, generator=g) * 3).to(BF16), settings(g, rows, vocab, 4, 300, 60, 3)) for _ in range(3)]
    for _, kw in cases:                                              # lists of one length
        kw["bias_words"], kw["bias"] = kw["bias_words"][:20].clone(), kw["bias"][:20].clone()
        kw["bias_starts"].clamp_(max=20)
    z, kw = cases[0][0].cuda(), on_gpu(cases[0][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.adjust_logits(z, out_dtype=F32, **kw)
    for hz, hkw in cases:
        z.copy_(hz)
        for n in kw:
            kw[n].copy_(hkw[n])
        graph.replay()
        torch.cuda.synchronize()
        check(hz, hkw, F32, got=out)
    streams, dev = [torch.cuda.Stream() for _ in cases], [(hz.cuda(), on_gpu(hkw)) for hz, hkw in cases]
    torch.cuda.synchronize()
    for _ in range(4):
        outs = []
        for st, (dz, dkw) in zip(streams, dev):
            with torch.cuda.stream(st):
                outs.append(ops.adjust_logits(dz, pdl=True, **dkw))
    torch.cuda.synchronize()
    for (hz, hkw), got in zip(cases, outs):
        check(hz, hkw, got=got)


def test_adjust_same_call_same_bits(cuda):
    g = torch.Generator().manual_seed(8)
    z, kw = torch.randn(20, 30000, generator=g).cuda(), on_gpu(settings(g, 20, 30000, 5, 4000, 50, 4, repeated=0.8))
    first = ops.adjust_logits(z, **kw)
    for _ in range(5):
        assert torch.equal(first, ops.adjust_logits(z, **kw))


def test_both_ways_from_tensors_to_launches(cuda, monkeypatch):
    g = torch.Generator().manual_seed(9)
    z, kw = torch.randn(4, 600, generator=g).to(BF16).cuda(), on_gpu(settings(g, 4, 600, 5, 50, 5, 4))

    def call(**more):
        return lambda: ops.adjust_logits(**dict(dict(kw, logits=z), **more))

    for more in (dict(), dict(out_dtype=F32), dict(out_dtype=BF16, pdl=True), dict(out=torch.zeros(4, 600, device="cuda")), dict(out=torch.zeros_like(z)), dict(mask_row=None),
                 dict(mask=None, mask_row=None), dict(token_seq=None), dict(bias_starts=None, bias=None, bias_words=None), dict(prompt_lens=None, frequency=None),
                 dict(bias_words=kw["bias_words"][:0], bias=kw["bias"][:0]), dict(tokens=kw["tokens"][:, ::2][:, :1]), dict(logits=torch.cat([z, z], 1)[:, 7:607])):
        both_ways(monkeypatch, call(**more))
    for more in (dict(logits=z.as_subclass(Own)), dict(tokens=kw["tokens"][:, :0])):
        both_ways(monkeypatch, call(**more), served=False)
    for more in (dict(logits=z[0]), dict(out_dtype=F16), dict(out=torch.zeros(4, 601, device="cuda")), dict(tokens=None), dict(token_lens=None), dict(mask=None), dict(bias=None),
                 dict(bias_starts=kw["bias_starts"][1:]), dict(repetition=kw["repetition"].double()), dict(mask=kw["mask"][:, :18]), dict(temperature=kw["temperature"].cpu()),
                 dict(tokens=kw["tokens"][:1].expand(5, 50)), dict(mask=kw["mask"][:2], mask_row=None), dict(bias_starts=None), dict(out=torch.zeros(4, 600, device="cuda"), out_dtype=BF16)):
        both_ways(monkeypatch, call(**more), served=False, refused=True)
