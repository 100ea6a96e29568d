"""Operators over a paged cache, without a GPU: refusals of the C entry points and of their Python front end, the page divisor, the oracle's own formulas."""
import ctypes
import math

import numpy as np
import pytest
import torch

from tests import paged_oracle as oracle
from zhilight_b200 import _lib, ops

P = ctypes.c_void_p(16)


def append_args(**kw):
    a = dict(qkv=P, ldq=768, pos=P, ld_pos=4, axes=3, inv_freq=ctypes.cast(P, ctypes.POINTER(ctypes.c_double)), axis=P, half=64, layout=0, mscale=1.0,
             token_seq=P, placement=P, page_table=P, ld_table=4, max_pages=4, seqs=2, k_cache=P, v_cache=P, num_pages=8, page_size=16, page_stride=2048,
             row_stride=128, head_stride=128, q_out=P, T=4, heads=4, kv_heads=1, dim=128, dtype=ops.BF16, pdl=0, stream=None)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(qkv=None), -1), (dict(T=0), -1), (dict(half=65), -1), (dict(axes=0), -1), (dict(ld_pos=3), -1), (dict(layout=2), -1), (dict(ldq=767), -1),
    (dict(ldq=772), -2), (dict(page_stride=2044), -2), (dict(page_size=0), -1), (dict(num_pages=0), -1), (dict(ld_table=3), -1), (dict(seqs=0), -1),
    (dict(k_cache=ctypes.c_void_p(8)), -2), (dict(dtype=ops.F32), -2), (dict(dim=132, half=4, ldq=2000), -2), (dict(axis=None), -1), (dict(row_stride=-8), -1),
    (dict(heads=900, ldq=902 * 128), -2),
])
def test_append_refuses(lib, kw, code):
    assert lib.zl_qkv_axes_rope_append(*append_args(**kw)) == code, lib.zl_last_error()


def attention_args(**kw):
    a = dict(q=P, k_cache=P, v_cache=P, num_pages=8, page_size=16, page_stride=2048, row_stride=128, head_stride=128, page_table=P, ld_table=4, max_pages=4,
             seq_lens=P, q_starts=P, seqs=2, scale=0.1, window=0, out=P, rows=4, max_new=4, heads=4, kv_heads=1, dim=128, workspace=None,
             workspace_bytes=0, dtype=ops.BF16, pdl=0, stream=None)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(rows=0), -1), (dict(max_new=0), -1), (dict(heads=3, kv_heads=2), -1), (dict(scale=0.0), -1), (dict(scale=-1.0), -1),
    (dict(scale=math.inf), -1), (dict(scale=math.nan), -1), (dict(window=-1), -1), (dict(dim=96), -2), (dict(dtype=ops.F32), -2),
    (dict(q=ctypes.c_void_p(8)), -2), (dict(head_stride=4), -2), (dict(max_pages=5), -1), (dict(v_cache=None), -1),
])
def test_attention_refuses(lib, kw, code):
    assert lib.zl_paged_attention(*attention_args(**kw)) == code, lib.zl_last_error()


def verify_args(**kw):
    a = dict(target=P, target_seq=300, target_row=100, draft=P, draft_seq=200, draft_row=100, drafted=P, accept=P, sample=P, count=None, accepted=P, tokens=P,
             seqs=2, drafts=2, vocab=100, pdl=0, stream=None)
    a.update(kw)
    return tuple(a.values())


@pytest.mark.parametrize("kw,code", [(dict(target=None), -1), (dict(seqs=0), -1), (dict(drafts=-1), -1), (dict(vocab=0), -1), (dict(drafted=None), -1),
                                     (dict(accept=None), -1), (dict(target_row=-1), -1), (dict(vocab=(1 << 30) + 1), -2), (dict(seqs=65536), -2)])
def test_verify_refuses(lib, kw, code):
    assert lib.zl_verify_drafts(*verify_args(**kw)) == code, lib.zl_last_error()


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_front_end_refuses_shapes_types_and_cpu_tensors(lib):
    k = torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(3, 8 * 64, dtype=torch.bfloat16)
    table, lens, starts = i32(2, 4), i32(2), i32(3)

    def attend(q=q, k=k, v=k, table=table, lens=lens, starts=starts, **kw):
        return ops.paged_attention(q, k, v, table, lens, starts, 0.1, **kw)

    for bad in (dict(q=q.float()), dict(k=k[:, :, :1]), dict(q=q[:, :100]), dict(table=table.long()), dict(lens=i32(3)), dict(starts=i32(2)),
                dict(k=k.transpose(2, 3)), dict(out=q.float()), dict(max_new=0), dict(k=k.expand(5, 16, 2, 64)[:1].expand(5, 16, 2, 64)),
                dict(k=k[:0], v=k[:0]), dict(q=q.t())):
        with pytest.raises(_lib.ZLError):
            attend(**bad)
    with pytest.raises(_lib.ZLError, match="CUDA tensors"):
        attend()

    qkv, pos, freq, axis = torch.zeros(3, 12 * 64, dtype=torch.bfloat16), i32(3, 3), torch.ones(32, dtype=torch.float64), i32(32)

    def append(qkv=qkv, pos=pos, freq=freq, axis=axis, seq=i32(3), place=i32(3), k=k, heads=8):
        return ops.qkv_axes_rope_append(qkv, pos, freq, axis, seq, place, table, k, k, heads)

    for bad in (dict(qkv=qkv[:, :-8]), dict(pos=i32(3, 2)), dict(freq=freq.float()), dict(axis=i32(31)), dict(freq=torch.ones(33, dtype=torch.float64), axis=i32(33)),
                dict(seq=i32(2)), dict(place=i32(3).long()), dict(heads=7), dict(k=k.half())):
        with pytest.raises(_lib.ZLError):
            append(**bad)
    with pytest.raises(_lib.ZLError, match="CUDA tensors"):
        append()

    p, d, w = torch.zeros(2, 4, 50), torch.zeros(2, 3, 50), i32(2, 3)

    def verify(p=p, d=d, w=w, a=torch.zeros(2, 3), s=torch.zeros(2), c=None):
        return ops.verify_drafts(p, d, w, a, s, c)

    for bad in (dict(p=p.double()), dict(d=p), dict(w=i32(2, 4)), dict(a=torch.zeros(2, 4)), dict(s=torch.zeros(3)), dict(c=i32(3)), dict(p=p[:, :, ::2]),
                dict(p=p[:, :0])):
        with pytest.raises(_lib.ZLError):
            verify(**bad)
    with pytest.raises(_lib.ZLError, match="CUDA tensors"):
        verify()


def test_page_divisor_is_exact():
    """i * ceil(2^(31 + s) / d) >> (31 + s), as the kernels divide a row number by the page size."""
    rng = np.random.default_rng(0)
    for d in [1, 2, 3, 5, 7, 16, 20, 48, 100, 127, 128, 129, 1000, 4096, 65537, 2 ** 30 + 1, 2 ** 31 - 1] + [int(x) for x in rng.integers(1, 2 ** 31, 50)]:
        s = 0
        while 1 << s < d:
            s += 1
        mul = -(-(1 << (31 + s)) // d)
        assert mul < 1 << 32
        for i in [0, 1, d - 1, d, d + 1, 2 ** 31 - 1, 2 ** 31 - 2] + [int(x) for x in rng.integers(0, 2 ** 31, 50)] + [x * d + e for x in range(3) for e in (-1, 0, 1)]:
            if 0 <= i < 1 << 31:
                assert (i * mul) >> (31 + s) == i // d, (i, d)


def test_axis_map():
    assert ops.rope_axis_map((2, 3, 1)).tolist() == [0, 0, 1, 1, 1, 2]
    assert ops.rope_axis_map((4, 2, 2), interleaved=True).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    with pytest.raises(_lib.ZLError):
        ops.rope_axis_map((1, 4, 1), interleaved=True)


def test_oracle_attention_is_softmax():
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(4, 8, 2, 64, generator=g).half() for _ in range(2))
    q = torch.randn(5, 4, 64, generator=g).half()
    table = torch.tensor([[2, 0], [3, 1]])
    out, _ = oracle.attention(q, k, v, table, [13, 9], [0, 3, 5], 0.3, 0)
    for b, (lo, hi, n) in enumerate([(0, 3, 13), (3, 5, 9)]):
        kk, vv = (x[table[b]].reshape(16, 2, 64).double() for x in (k, v))
        for r in range(lo, hi):
            m = n - (hi - r) + 1
            for h in range(4):
                p = torch.softmax(q[r, h].double() @ kk[:m, h // 2].T * 0.3, -1)
                assert torch.allclose(out[r, h], p @ vv[:m, h // 2], atol=1e-12)


def test_oracle_verification_leaves_the_targets_distribution():
    """Whatever the drafts' probabilities are, a drafted word or its replacement follows the target: the sums over all random numbers agree."""
    rng = np.random.default_rng(1)
    p, d = rng.dirichlet(np.ones(4)), rng.dirichlet(np.ones(4))
    n = 60000
    words = rng.choice(4, size=(n, 1), p=d)
    target = np.broadcast_to(p, (n, 2, 4))
    acc, tok = oracle.verify(target, np.broadcast_to(d, (n, 1, 4)), words, rng.random((n, 1)), rng.random(n), None)
    share = np.bincount(tok[:, 0], minlength=4) / n
    assert np.abs(share - p).max() < 5 * 0.5 / math.sqrt(n)          # five standard deviations of a share
