"""Operators over a 4-bit cache and on logits, without a GPU: refusals of the C entry points and of their Python front end, the oracle's own formulas."""
import ctypes
import math

import numpy as np
import pytest
import torch

from tests import int4_oracle as oracle
from tests.test_paged_cpu import append_args, attention_args, i32
from zhilight_b200 import _lib, ops

P = ctypes.c_void_p(16)
BYTES = dict(page_stride=16 * 80, row_stride=80, head_stride=80)


@pytest.mark.parametrize("kw,code", [
    (dict(qkv=None), -1), (dict(T=0), -1), (dict(half=65), -1), (dict(axes=0), -1), (dict(ld_pos=3), -1), (dict(layout=2), -1), (dict(ldq=767), -1),
    (dict(ldq=772), -2), (dict(page_stride=1288), -2), (dict(page_size=0), -1), (dict(num_pages=0), -1), (dict(ld_table=3), -1), (dict(seqs=0), -1),
    (dict(k_cache=ctypes.c_void_p(8)), -2), (dict(dtype=ops.F32), -2), (dict(dim=96, half=8), -2), (dict(dim=256, half=4, ldq=2000), -2), (dict(axis=None), -1), (dict(row_stride=-80), -1),
    (dict(heads=460, ldq=462 * 128), -2), (dict(page_table=None), -1), (dict(v_cache=None), -1), (dict(dtype=7), -2),
])
def test_append_refuses(lib, kw, code):
    assert lib.zl_qkv_axes_rope_append_int4(*append_args(**dict(BYTES, **kw))) == code, lib.zl_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(rows=0), -1), (dict(max_new=0), -1), (dict(heads=3, kv_heads=2), -1), (dict(scale=0.0), -1), (dict(scale=-1.0), -1),
    (dict(scale=math.inf), -1), (dict(scale=math.nan), -1), (dict(window=-1), -1), (dict(dim=96), -2), (dict(dtype=ops.F32), -2),
    (dict(q=ctypes.c_void_p(8)), -2), (dict(head_stride=40), -2), (dict(max_pages=5), -1), (dict(v_cache=None), -1), (dict(page_table=None), -1), (dict(workspace=P), -1),
    (dict(max_pages=2 ** 20, ld_table=2 ** 20, page_size=2 ** 20, seqs=1000), -2),
])
def test_attention_refuses(lib, kw, code):
    assert lib.zl_paged_attention_int4(*attention_args(**dict(BYTES, **kw))) == code, lib.zl_last_error()


def test_append_refuses_rows_beyond_shared_memory(lib):
    """Two rows of 434 heads of 128, and cosines and sines of 64 frequencies: 32 elements more than there is room for."""
    assert 434 * 128 == 56288 - 12 * 64 + 32
    args = dict(BYTES, heads=432, kv_heads=1, half=64, ldq=434 * 128)
    assert lib.zl_qkv_axes_rope_append_int4(*append_args(**args)) == -2, lib.zl_last_error()


@pytest.mark.parametrize("scale", [2.0 ** 65, 3.0e38])
def test_attention_refuses_scales_beyond_its_sums(lib, scale):
    assert lib.zl_paged_attention_int4(*attention_args(**dict(BYTES, scale=scale))) == -2, lib.zl_last_error()


def values_args(**kw):
    a = dict(k_cache=P, v_cache=P, num_pages=8, page_size=16, page_stride=1280, row_stride=80, head_stride=80, pages=None, n=8, k_out=P, v_out=P, kv_heads=1,
             dim=128, dtype=ops.BF16, pdl=0, stream=None)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw,code", [(dict(k_cache=None), -1), (dict(k_out=None), -1), (dict(v_out=None), -1), (dict(n=9), -1), (dict(n=0), -1), (dict(dim=32), -2),
                                     (dict(dtype=ops.F32), -2), (dict(row_stride=72), -2), (dict(k_out=ctypes.c_void_p(8)), -2), (dict(pages=P, n=1 << 40), -2)])
def test_values_refuse(lib, kw, code):
    assert lib.zl_int4_cache_values(*values_args(**kw)) == code, lib.zl_last_error()


def adjust_args(**kw):
    a = dict(logits=P, ld_logits=100, dtype=ops.BF16, out=P, ld_out=100, out_dtype=ops.BF16, rows=4, vocab=100, tokens=None, ld_tokens=0, seqs=0, longest=0,
             token_seq=None, token_lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None, bias_starts=None, bias_words=None, bias=None, n_bias=0,
             temperature=None, mask=None, ld_mask=0, masks=0, mask_row=None, pdl=0, stream=None)
    a.update(kw)
    return tuple(a.values())


HISTORY = dict(tokens=P, ld_tokens=10, seqs=4, longest=10, token_lens=P)


@pytest.mark.parametrize("kw,code", [
    (dict(logits=None), -1), (dict(out=None), -1), (dict(rows=0), -1), (dict(vocab=0), -1), (dict(ld_logits=99), -1), (dict(ld_out=99), -1),
    (dict(HISTORY, token_lens=None), -1), (dict(HISTORY, seqs=3), -1), (dict(HISTORY, ld_tokens=9), -1), (dict(HISTORY, longest=-1), -1),
    (dict(bias_starts=P, n_bias=3), -1), (dict(bias_starts=P, n_bias=-1), -1), (dict(mask=P, ld_mask=3, masks=4), -1), (dict(mask=P, ld_mask=4, masks=3), -1),
    (dict(mask=P, ld_mask=4, masks=0, mask_row=P), -1), (dict(out_dtype=ops.F16), -2), (dict(dtype=ops.F32, out_dtype=ops.BF16), -2), (dict(dtype=9, out_dtype=9), -2),
    (dict(vocab=1 << 25, ld_logits=1 << 25, ld_out=1 << 25), -2), (dict(rows=(1 << 31) - 1, vocab=1 << 24, ld_logits=1 << 24, ld_out=1 << 24), -2)])
def test_adjust_refuses(lib, kw, code):
    assert lib.zl_adjust_logits(*adjust_args(**kw)) == code, lib.zl_last_error()


def test_front_end_refuses_shapes_types_and_cpu_tensors(lib):
    k = torch.zeros(5, 16, 2, 40, dtype=torch.uint8)
    q = torch.zeros(3, 8 * 64, dtype=torch.bfloat16)
    table, lens, starts = i32(2, 4), i32(2), i32(3)

    def attend(q=q, k=k, v=k, table=table, lens=lens, starts=starts, **kw):
        return ops.paged_attention_int4(q, k, v, table, lens, starts, 0.1, **kw)

    for bad in (dict(q=q.float()), dict(k=k[:, :, :1]), dict(q=q[:, :100]), dict(table=table.long()), dict(lens=i32(3)), dict(starts=i32(2)), dict(k=k.bfloat16(), v=k.bfloat16()),
                dict(k=k.transpose(2, 3)), dict(out=q.float()), dict(max_new=0), dict(k=k[:1].expand(5, 16, 2, 40)), dict(window=-1),
                dict(k=k[:0], v=k[:0]), dict(q=q.t()), dict(k=k[..., :39], v=k[..., :39]), dict(k=torch.zeros(5, 16, 2, 60, dtype=torch.uint8))):
        with pytest.raises(_lib.ZLError):
            attend(**bad)
    with pytest.raises(_lib.ZLError, match="CUDA tensors"):
        attend()

    qkv, pos, freq, axis = torch.zeros(3, 12 * 64, dtype=torch.bfloat16), i32(3, 3), torch.ones(32, dtype=torch.float64), i32(32)

    def append(qkv=qkv, pos=pos, freq=freq, axis=axis, seq=i32(3), place=i32(3), k=k, heads=8):
        return ops.qkv_axes_rope_append_int4(qkv, pos, freq, axis, seq, place, table, k, k, heads)

    for bad in (dict(qkv=qkv[:, :-8]), dict(pos=i32(3, 2)), dict(freq=freq.float()), dict(axis=i32(31)), dict(freq=torch.ones(33, dtype=torch.float64), axis=i32(33)),
                dict(seq=i32(2)), dict(place=i32(3).long()), dict(heads=7), dict(k=k.half()), dict(qkv=qkv.float())):
        with pytest.raises(_lib.ZLError):
            append(**bad)
    with pytest.raises(_lib.ZLError, match="CUDA tensors"):
        append()

    for bad in (dict(dtype=torch.float32), dict(dtype=None), dict(pages=i32(2).long()), dict(pages=i32(2, 1)), dict(k=k.half()), dict(v=k[1:])):
        a = dict(dict(k=k, v=k, dtype=torch.float16, pages=None), **bad)
        with pytest.raises(_lib.ZLError):
            ops.int4_cache_values(a["k"], a["v"], a["dtype"], a["pages"])
    with pytest.raises(_lib.ZLError, match="CUDA tensors"):
        ops.int4_cache_values(k, None, torch.float16)
    for dim in (0, 32, 63, 96, 256):
        with pytest.raises(_lib.ZLError):
            ops.int4_row_bytes(dim)
    assert [ops.int4_row_bytes(d) for d in (64, 128)] == [40, 80]


def test_adjust_front_end_refuses(lib):
    z, t, n, f = torch.zeros(3, 70), i32(3, 9), i32(3), torch.ones(3)
    full = dict(logits=z, tokens=t, token_seq=n, token_lens=n, prompt_lens=n, repetition=f, frequency=f, presence=f, bias_starts=i32(4), bias_words=i32(5),
                bias=torch.ones(5), temperature=f, mask=i32(2, 3), mask_row=n)
    for bad in (dict(logits=z[0]), dict(logits=z.double()), dict(logits=z.t()), dict(logits=z[:, :0]), dict(out_dtype=torch.float16), dict(out=z[:2]), dict(out=z.half()),
                dict(tokens=t.long()), dict(tokens=t[0]), dict(token_lens=None), dict(token_lens=i32(2)), dict(token_seq=None, tokens=t[:2]), dict(token_seq=n.long()),
                dict(tokens=None), dict(prompt_lens=i32(4)), dict(repetition=f[:2]), dict(frequency=f.double()), dict(presence=f.half()), dict(temperature=torch.ones(3, 1)),
                dict(bias_starts=i32(3)), dict(bias_starts=None), dict(bias_words=None), dict(bias_words=i32(4)), dict(bias=torch.ones(4)), dict(bias=torch.ones(5).half()),
                dict(mask=None), dict(mask=i32(2, 2)), dict(mask_row=None), dict(mask=i32(2, 3).long()), dict(mask=i32(0, 3)), dict(logits=z[:1].expand(3, 70)),
                dict(tokens=t[:1].expand(3, 9)), dict(mask=i32(1, 3).expand(2, 3)), dict(out=torch.zeros(1, 70).expand(3, 70)), dict(token_lens=torch.zeros(6, dtype=torch.int32)[::2])):
        with pytest.raises(_lib.ZLError):
            ops.adjust_logits(**dict(full, **bad))
    for kw in (full, dict(logits=z)):
        with pytest.raises(_lib.ZLError, match="CUDA tensors"):
            ops.adjust_logits(**kw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_oracle_rounds_as_torch_does(dtype):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(20000, generator=g) * torch.exp2(torch.randint(-30, 20, (20000,), generator=g).float())
    x[:6] = torch.tensor([0.0, -0.0, 65519.0, 65520.0, 3.3961775e38, math.inf])
    y = torch.from_numpy(oracle.to_type(x.double().numpy(), dtype))
    assert torch.equal(y, x.to(dtype).double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_oracle_rows_come_back(dtype, dim):
    """Within half a step, ends as they are or one rounding off, constants and the largest numbers exactly or nearly so, broken groups as NaN."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(50, 3, dim, generator=g) * torch.exp2(torch.randint(-9, 9, (50, 3, 1), generator=g).float())).to(dtype)
    x[0, 0], x[0, 1, :32], x[0, 2, ::2] = 3.25, oracle.TOP[dtype], -oracle.TOP[dtype]
    x[0, 2, 1::2] = oracle.TOP[dtype]
    x[1, 0, 5], x[1, 1, 40], x[1, 2, 0] = math.nan, math.inf, -math.inf
    rows = oracle.encode(x, dtype)
    assert rows.shape == (50, 3, ops.int4_row_bytes(dim)) and rows.dtype == torch.uint8
    y = oracle.decode(rows, dtype)
    bad = (~torch.isfinite(x.unflatten(-1, (-1, 32)))).any(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    assert ((y.double() - x.double()).abs() <= oracle.off_by(rows, dtype))[~bad].all()
    assert torch.equal(y[0, 0], x[0, 0]) and torch.equal(y[0, 1, :32], x[0, 1, :32])
    low = x.unflatten(-1, (-1, 32)).amin(-1)
    assert torch.equal(y.unflatten(-1, (-1, 32)).amin(-1)[2:], low[2:])


@pytest.mark.parametrize("n_bias,code", [((1 << 31) - 1, -2), ((1 << 31) - 1024, -2), (-1, -1)])
def test_adjust_refuses_lists_whose_places_do_not_fit(lib, n_bias, code):
    assert lib.zl_adjust_logits(*adjust_args(bias_starts=P, bias_words=P, bias=P, n_bias=n_bias)) == code, lib.zl_last_error()


def test_adjust_front_end_refuses_sizes_beyond_32_bits(lib):
    """Sizes that would come around as small ones, of tensors without memory."""
    def many(*shape, dtype=torch.int32):
        return torch.empty(shape, dtype=dtype, device="meta")

    n = (1 << 32) + 5
    for bad in (dict(bias_starts=i32(4), bias_words=many(n), bias=many(n, dtype=torch.float32)), dict(tokens=many(3, n), token_lens=i32(3)),
                dict(tokens=many(n, 3), token_lens=i32(3)), dict(mask=many(n, 3)), dict(logits=many(n, 70, dtype=torch.float16))):
        with pytest.raises(_lib.ZLError, match="32 bits"):
            ops.adjust_logits(**dict(dict(logits=torch.zeros(3, 70)), **bad))


def test_oracle_adjusts_logits():
    z = torch.tensor([[1.0, -2.0, 3.0, 4.0, 0.5], [1.0, 1.0, 1.0, 1.0, 1.0]])
    tokens = torch.tensor([[0, 1, 2, 2, 7, -1]], dtype=torch.int32)
    out, off = oracle.adjust(z, torch.float32, tokens=tokens, token_seq=[0, 5], token_lens=[6, 6], prompt_lens=[1, 0], repetition=[2.0, 2.0], frequency=[0.25, 1.0],
                             presence=[0.5, 1.0], bias_starts=[0, 2, 3], bias_words=[3, 3, 4], bias=[1.0, 2.0, -1.0], temperature=[0.5, 0.0],
                             mask=torch.tensor([[0b01111]], dtype=torch.int32), mask_row=[0, -1])
    assert out.tolist() == [[1.0, -9.5, 1.0, 14.0, -math.inf], [1.0, 1.0, 1.0, 1.0, 0.0]]
    assert (off[np.isfinite(out)] < 1e-5).all()
