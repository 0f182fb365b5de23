"""How exact kv8_attention is where its own tests leave room: rows of 16-bit types, rows that one
position carries, chunks over many tiles.  The reference and the bound are those of test_gpu_kv8's
docstring for f32 rows (weights in two 11-bit halves, sums in f32: 2^-18 of sum_j p_j |v_j|), for
every type, and one rounding of the result to its type."""
import numpy as np
import pytest
import torch

import test_gpu_kv8 as base
from test_gpu_kv8 import DT, HostCache, i32, make_pages, make_table, starts

from lama32_mojo_b200 import ops

pytestmark = pytest.mark.gpu


def attend(cuda, kv, G, hd, page, ns, ctx, dtype, seed, width=None, pages=None):
    """(outputs, reference, bound) of a call, f64 [T, heads, hd]."""
    total = sum(-(-int(c) // page) for c in ctx) + 1
    pages = pages or make_pages(cuda, total, kv, page, hd, seed)
    table = make_table(ctx, page, pages.num_pages, seed, width)
    heads, T = kv * G, int(sum(ns))
    g = torch.Generator(device=cuda).manual_seed(seed)
    q = torch.randn((T, heads * hd), device=cuda, generator=g).to(DT[dtype])
    got = ops.kv8_attention(q, i32(starts(ns), cuda), i32(ctx, cuda), heads, pages, i32(table, cuda))
    base.reference.tol16 = np.zeros((T, heads, hd))
    ref, tol = base.reference(HostCache(pages), q.double().cpu().numpy().reshape(T, heads, hd), ns, ctx, table, heads)
    info = torch.finfo(DT[dtype])
    tol = tol + info.eps / 2 * np.abs(ref) + info.smallest_normal * info.eps / 2 + 1e-37
    return got.double().cpu().numpy().reshape(T, heads, hd), ref, tol


# every form: clusters, stretches, chunks on tcgen05 (the table's width decides)
@pytest.mark.parametrize("kv,G,hd,page,ns,ctx,width", [
    (2, 4, 128, 64, [1] * 6, [1, 2, 17, 64, 200, 301], None),
    (2, 3, 64, 16, [1] * 40, list(range(1, 281, 7)), 900),
    (2, 4, 128, 64, [5, 3, 4, 1], [5, 40, 130, 77], None),
    (2, 12, 64, 32, [5] * 12, list(range(5, 245, 20)), 400),
    (1, 4, 128, 64, [70, 33], [300, 33], 400),
    (1, 4, 64, 64, [130, 64], [130, 500], 400),
])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_rows_of_16_bit_types_are_rounded_once(cuda, kv, G, hd, page, ns, ctx, width, dtype):
    got, ref, tol = attend(cuda, kv, G, hd, page, ns, ctx, dtype, G + hd, width)
    assert (np.abs(got - ref) / tol).max() <= 1


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_chunks_of_16_bit_rows_in_one_stretch(cuda, dtype, hd):
    """330 times a chunk against 6000 positions: single CTAs add up more than 64 tiles of 64 positions,
    with scores that grow along the context."""
    G, page, n, ctx, S = 4, 64, 32, 6000, 330
    pages = make_pages(cuda, 94, 1, page, hd, 6)
    pages.k_scale.mul_(torch.linspace(0.2, 3.0, 94, device=cuda)[:, None, None])
    row = np.arange(94, dtype=np.int32)
    q = torch.randn((n, G * hd), device=cuda, generator=torch.Generator(device=cuda).manual_seed(6)).to(DT[dtype])
    got = ops.kv8_attention(q.repeat(S, 1), i32(starts([n] * S), cuda), i32([ctx] * S, cuda), G, pages,
                            i32(np.tile(row, (S, 1)), cuda)).view(S, n, G, hd)
    base.reference.tol16 = np.zeros((n, G, hd))
    ref, tol = base.reference(HostCache(pages), q.double().cpu().numpy().reshape(n, G, hd), [n], [ctx], row[None], G)
    info = torch.finfo(DT[dtype])
    # sums of 64 tiles are cut off at the 24th bit some 8 times a tile: 64 * 8 * 2^-24 of sum_j p_j |v_j| at most,
    # which is 8 times the docstring's 2^-18; tol holds that once already
    mag = tol / 2.0 ** -18
    tol = tol + mag * 64 * 8 * 2.0 ** -24 + info.eps / 2 * np.abs(ref) + info.smallest_normal * info.eps / 2
    err = (got.double() - torch.from_numpy(ref).to(cuda)).abs()
    assert float((err / torch.from_numpy(tol).to(cuda)).max()) <= 1


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ctx", [40, 1000])
def test_chunk_rows_that_one_position_carries(cuda, hd, ctx):
    """f32 rows of chunks whose result is the value of one position: the first rows of fresh prompts
    (ctx 40), and rows whose scores but one are so low that the other weights are 0 (ctx 1000, the
    position in the first of 16 tiles).  The weight has 22 bits (2^-22), its two halves' products
    are cut off at 24 bits (2 * 2^-23), l's quotient and the last product round (2^-24 each), and
    exp2 of the row's largest score is one but for 2 ulps that weight and l share; 2^-24 more for
    each of the scale and the reference's own rounding."""
    G, kv, page, n, S = 4, 4, 64, 40, 64
    per = -(-ctx // page)
    pages = make_pages(cuda, per, kv, page, hd, hd)
    g = torch.Generator(device=cuda).manual_seed(hd)
    q = torch.rand((S * n, kv * G * hd), device=cuda, generator=g) + 0.5
    if ctx > n:
        pages.k.zero_()
        pages.k[0, :, 5] = 127
        pages.k_scale.fill_(1.0)
    row = np.arange(per, dtype=np.int32)
    got = ops.kv8_attention(q, i32(starts([n] * S), cuda), i32([ctx] * S, cuda), kv * G, pages,
                            i32(np.tile(row, (S, 1)), cuda)).view(S, n, kv, G, hd).double()
    at = 5 if ctx > n else 0
    want = pages.v[0, :, at].double() * pages.v_scale[0, :, at // 16, None].double()  # [kv, hd]
    if ctx == n:
        got = got[:, :1]
    err = (got - want[:, None]).abs() / want.abs().clamp(min=1e-30)[:, None]
    err = err[torch.broadcast_to(want[:, None] != 0, err.shape)]
    assert float(err.max()) <= 2.0 ** -22 + 2 * 2.0 ** -23 + 4 * 2.0 ** -24


@pytest.mark.parametrize("ns,ctx,width", [([1] * 6, [1, 2, 17, 64, 200, 301], None),
                                          ([1] * 40, list(range(1, 281, 7)), 900),
                                          ([5, 3, 4, 1], [5, 40, 130, 77], None), ([70, 130], [300, 130], 400)])
@pytest.mark.parametrize("lo,hi", [(1.3e36, 2.6e36), (1e-25, 3e-25), (1e-25, 2e36)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_of_any_size(cuda, ns, ctx, width, lo, hi, dtype):
    """Values up to f32's largest number (127 * 2.6e36), and small ones; every form."""
    pages = make_pages(cuda, 20 if width is None else 110, 2, 64, 128, 3)
    g = torch.Generator(device=cuda).manual_seed(3)
    u = torch.rand(pages.v_scale.shape, generator=g, device=cuda, dtype=torch.float64)
    pages.v_scale.copy_(torch.exp(np.log(lo) + u * (np.log(hi) - np.log(lo))))
    got, ref, tol = attend(cuda, 2, 4, 128, 64, ns, ctx, dtype, 3, width, pages)
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) / tol).max() <= 1


@pytest.mark.parametrize("deviation", [0.5, 2.0, 8.0])
def test_long_chunks_are_as_exact_as_f32_operations(cuda, deviation):
    """f32 chunks against 8000 positions, as a whole: not further from 64 bits than the same formula in
    elementary f32 operations, which round every sum where the tensor cores cut theirs off."""
    ctx, n, S, kv, G, hd, page = 8000, 256, 8, 8, 4, 128, 64
    g = torch.Generator(device=cuda).manual_seed(3)
    per = ctx // page
    shape = per, kv, page, hd

    def codes():
        return torch.randn(shape, generator=g, device=cuda).mul_(36).round_().clamp_(-127, 127).to(torch.int8)

    def scales():
        return torch.rand((per, kv, page // 16), generator=g, device=cuda) * 0.02 + 0.01

    pages = ops.KV8Pages(codes(), codes(), scales(), scales())
    q = torch.randn((n, kv * G * hd), generator=g, device=cuda) * deviation
    row = np.arange(per, dtype=np.int32)
    got = ops.kv8_attention(q.repeat(S, 1), i32(starts([n] * S), cuda), i32([ctx] * S, cuda), kv * G, pages,
                            i32(np.tile(row, (S, 1)), cuda))[:n]
    later = torch.arange(ctx, device=cuda)[None] > (ctx - n + torch.arange(n, device=cuda))[:, None]

    def plain(dtype):
        def values(c, s):
            return (c.to(dtype) * s.to(dtype).repeat_interleave(16, 2)[..., None]).transpose(1, 2).reshape(ctx, kv, hd)
        s = torch.einsum("nkgd,pkd->kgnp", q.to(dtype).view(n, kv, G, hd), values(pages.k, pages.k_scale)) / hd ** 0.5
        p = s.masked_fill_(later, float("-inf")).softmax(-1)
        return torch.einsum("kgnp,pkd->nkgd", p, values(pages.v, pages.v_scale)).reshape(n, -1).double()

    was = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    exact, near = plain(torch.float64), plain(torch.float32)
    torch.backends.cuda.matmul.allow_tf32 = was
    assert float((got.double() - exact).norm()) <= float((near - exact).norm())
