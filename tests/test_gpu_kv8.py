"""The 8-bit paged cache (kv8_append, kv8_read, kv8_attention) against plain
64-bit restatements on the host.

Append: codes and scales have one right value (the quotients are rounded as
real numbers), so they have to be equal.

Attention, per output element: with mag = sum_j p_j |v_j| and smag the largest
sum_d |q_d k_jd| / sqrt(hd) of the row,
  * a score is off by at most smag * E, E = 2^-21 (q in two 11-bit halves, or
    exact) + (hd / 16 + 3) * 2^-23 (f32 sums over hd / 16 steps of 16 products,
    scale, 1 / sqrt(hd)) and exp2 of a score of size smag adds 2 ulps of it;
    that moves every p by the factor exp(+-smag E'), so o by 2 smag E' mag;
  * p is kept in two 11-bit halves (f32 rows) or one (16-bit rows, 2^-11), the
    sums are f32 over at most a few hundred steps: 2^-18 mag covers them;
  * the weights p_j sv_j are f16 numbers lifted so that the largest lies just
    below 2^15; the f16 grid is never finer than 2^-24, so each is off by up to
    2^-25 / 2^14 = 2^-39 of the largest, however small it is, times a code of at
    most 127: positions * 2^-39 * 127 * max_j p_j sv_j.  (mag does not cover this
    where the positions that carry the weight have the code 0.)
  * the result is rounded to its type: eps / 2 of its value, and below the
    smallest normal number, where the grid stays smallest_normal * eps, half of
    that (f16: 2^-14 * 2^-10 / 2 = 2^-25; an output of 2.2e-5 lies there).
"""
import math

import numpy as np
import pytest
import torch

from lama32_mojo_b200 import _lib, ops

pytestmark = pytest.mark.gpu
B = 16
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def i32(a, cuda):
    return torch.tensor(np.asarray(a, np.int32), device=cuda)


def starts(ns):
    return np.concatenate([[0], np.cumsum(ns)]).astype(np.int32)


class HostCache:
    """Plain restatement of the cache: one append call at a time."""

    def __init__(self, pages: ops.KV8Pages):
        self.c = [t.cpu().numpy().astype(np.int64) for t in (pages.k, pages.v)]
        self.s = [t.cpu().numpy().copy() for t in (pages.k_scale, pages.v_scale)]
        self.page = pages.page

    def append(self, k, v, ns, ctx, table):
        """k, v: f64 [T, kv, hd] arrays holding the exact input values."""
        t = 0
        for b, n in enumerate(ns):
            rows = [(ctx[b] - n + i, t + i) for i in range(n) if ctx[b] - n + i >= 0]
            t += n
            for blk in sorted({p // B for p, _ in rows}):
                mine = [(p, r) for p, r in rows if p // B == blk]
                j = blk * B // self.page
                pg = table[b, j] if j < table.shape[1] else -1
                if not 0 <= pg < self.c[0].shape[0]:
                    continue
                at, in0 = blk * B % self.page, mine[0][0] % B
                for which, x in ((0, k), (1, v)):
                    new = np.stack([x[r] for _, r in mine])  # [m, kv, hd]
                    new = np.where(np.isnan(new), 0.0, new)
                    fin = np.where(np.isinf(new), 0.0, np.abs(new))
                    for h in range(new.shape[1]):
                        old = np.float32(self.s[which][pg, h, at // B]) if in0 else np.float32(0)
                        s = max(old, np.float32(fin[:, h].max() / 127.0))
                        c = self.c[which][pg, h]
                        if s != old and in0:
                            if old > 0:
                                q = c[at:at + in0] * np.float64(old) / np.float64(s)
                                c[at:at + in0] = np.clip(np.rint(q), -127, 127)
                            else:
                                c[at:at + in0] = 0
                        with np.errstate(divide="ignore", invalid="ignore"):
                            code = np.clip(np.rint(new[:, h] / np.float64(s)), -127, 127) if s > 0 else 0 * new[:, h]
                        code = np.where(np.isinf(new[:, h]), np.sign(new[:, h]) * 127, code)
                        c[at + in0:at + in0 + len(mine)] = code
                        self.s[which][pg, h, at // B] = s

    def check(self, pages):
        for a, t in zip(self.c, (pages.k, pages.v)):
            assert np.array_equal(a, t.cpu().numpy())
        for a, t in zip(self.s, (pages.k_scale, pages.v_scale)):
            assert np.array_equal(a, t.cpu().numpy())

    def scale_of(self, which, table_row, upto, h):
        """f64 [upto]: the scale of each position of a kv head (0: no page)."""
        j = [table_row[p // self.page] if p // self.page < len(table_row) else -1 for p in range(upto)]
        n = self.c[0].shape[0]
        return np.array([float(self.s[which][e, h, p % self.page // B]) if 0 <= e < n else 0.0
                         for p, e in enumerate(j)])

    def values(self, which, table_row, upto):
        """f64 [upto, kv, hd] and which positions have a page."""
        kv, page, hd = self.c[0].shape[1:]
        out, ok = np.zeros((upto, kv, hd)), np.zeros(upto, bool)
        for j in range(-(-upto // page)):
            pg = table_row[j] if j < len(table_row) else -1
            if not 0 <= pg < self.c[0].shape[0]:
                continue
            m = min(page, upto - j * page)
            s = np.repeat(self.s[which][pg].astype(np.float64), B, axis=1)[:, :m, None]
            out[j * page:j * page + m] = (self.c[which][pg][:, :m] * s).transpose(1, 0, 2)
            ok[j * page:j * page + m] = True
        return out, ok


def make_pages(cuda, total, kv, page, hd, seed=0, lo=0.005, hi=0.03):
    g = torch.Generator(device=cuda).manual_seed(seed)
    shape = (total, kv, page, hd)

    def codes():
        return torch.randint(-127, 128, shape, generator=g, device=cuda, dtype=torch.int8)

    def scales():
        return torch.rand((total, kv, page // B), generator=g, device=cuda) * (hi - lo) + lo

    return ops.KV8Pages(codes(), codes(), scales(), scales())


def make_table(lens, page, total, seed=0, width=None):
    per = [-(-max(n, 0) // page) for n in lens]
    order = np.random.default_rng(seed).permutation(total)
    assert sum(per) <= total
    table, at = np.full((len(lens), width or max(1, max(per))), -1, np.int32), 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kv,hd,page", [(8, 128, 64), (2, 64, 16), (1, 64, 48), (3, 128, 128)])
def test_append_grows_blocks(cuda, dtype, kv, hd, page):
    """Sequences grow by random counts (zero among them): full, begun and straddled blocks."""
    rng = np.random.default_rng(kv * hd + page)
    S, width = 5, -(-200 // page) + 1
    pages = ops.KV8Pages.empty(S * width + 2, kv, page, hd, cuda)
    table = np.random.default_rng(1).permutation(S * width + 2)[:S * width].reshape(S, width).astype(np.int32)
    host, ctx = HostCache(pages), np.zeros(S, np.int64)
    for step in range(6):
        ns = rng.integers(0, 4, S) if step % 2 else rng.integers(0, 37, S)
        ns[step % S] = 0
        ctx += ns
        T = int(ns.sum()) + 3  # three rows of padding
        wide = torch.randn((T, 2 * kv * hd + 5), device=cuda) * float(10.0 ** rng.integers(-2, 2))
        wide = wide.to(DT[dtype])
        # strided rows; on odd steps they do not start on a 16-byte boundary
        o = step % 2
        k, v = wide[:, o:o + kv * hd], wide[:, o + kv * hd:o + 2 * kv * hd]
        ops.kv8_append(k, v, i32(starts(ns), cuda), i32(ctx, cuda), pages, i32(table, cuda))
        f = wide.double().cpu().numpy()
        host.append(f[:, o:o + kv * hd].reshape(T, kv, hd), f[:, o + kv * hd:o + 2 * kv * hd].reshape(T, kv, hd), ns,
                    ctx, table)
        host.check(pages)


def test_append_ties_zeros_and_non_finite(cuda):
    kv, hd, page = 1, 64, 16
    pages = ops.KV8Pages.empty(8, kv, page, hd, cuda)
    host = HostCache(pages)
    table = np.arange(8, dtype=np.int32).reshape(8, 1)
    x = np.zeros((8, kv * hd), np.float32)
    x[0] = np.arange(64) - 31.5  # amax 32.5
    x[0, 0] = 127.0  # scale 1: every quotient is a tie
    x[1] = 0.0
    x[2, :4] = [np.inf, -np.inf, np.nan, 2.0]
    x[3, :3] = [np.inf, np.nan, 0.0]  # nothing finite
    x[4] = np.float32(1e-44) * np.arange(64)  # subnormal: the scale is a few units of 2^-149
    x[5, :2] = [1e-45, -1e-45]  # the scale rounds to 0
    x[6] = 3.4e38 * (np.arange(64) / 63.0)
    s = np.float32(0.37)
    x[7] = (np.float32(127) * s) * ((np.arange(64) - 32) / np.float32(127)).astype(np.float32)
    x[7, 1::2] = np.nextafter(x[7, 1::2], np.float32(1e9))
    xt = torch.from_numpy(x).to(cuda)
    ns, ctx = np.ones(8, np.int64), np.ones(8, np.int64)
    ops.kv8_append(xt, xt.flip(1).contiguous(), i32(starts(ns), cuda), i32(ctx, cuda), pages, i32(table, cuda))
    f = x.astype(np.float64).reshape(8, kv, hd)
    host.append(f, f[:, :, ::-1], ns, ctx, table)
    host.check(pages)
    # second tokens: scales grow from zero, from subnormals, by a factor with ties (2), or not at all
    y = np.zeros_like(x)
    y[0] = 254.0
    y[1], y[2], y[3] = 1.0, 1.0, 0.0
    y[4], y[5], y[6], y[7] = 1e-40, 1e-3, 0.0, 0.37 * 127 * 1.5
    yt = torch.from_numpy(y).to(cuda)
    ops.kv8_append(yt, yt, i32(starts(ns), cuda), i32(ctx + 1, cuda), pages, i32(table, cuda))
    f = y.astype(np.float64).reshape(8, kv, hd)
    host.append(f, f, ns, ctx + 1, table)
    host.check(pages)


def test_append_quotients_next_to_a_tie(cuda):
    """x = (c + 1/2) s moved by an ulp either way: f32 division alone rounds many of them to the tie."""
    rng = np.random.default_rng(5)
    kv, hd, page, S = 2, 128, 16, 40
    pages = ops.KV8Pages.empty(S, kv, page, hd, cuda)
    host = HostCache(pages)
    table = np.arange(S, dtype=np.int32).reshape(S, 1)
    amax = np.exp(rng.uniform(-20, 20, (S, kv, 1))).astype(np.float32)
    s = (amax.astype(np.float64) / 127).astype(np.float32)
    c = rng.integers(-126, 126, (S, kv, hd))
    x = ((c + 0.5) * s).astype(np.float32)
    x = np.where(rng.random(x.shape) < 0.5, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf)))
    x = np.clip(x, -amax, amax)
    x[..., 0] = amax[..., 0]
    ns = np.ones(S, np.int64)
    xt = torch.from_numpy(x.reshape(S, -1)).to(cuda)
    ops.kv8_append(xt, xt, i32(starts(ns), cuda), i32(ns, cuda), pages, i32(table, cuda))
    host.append(x.astype(np.float64), x.astype(np.float64), ns, ns, table)
    host.check(pages)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,shift", [(128, 1), (64, 3)])
def test_append_unaligned_rows(cuda, dtype, hd, shift):
    """Rows that do not begin at a multiple of 16 bytes, k and v with strides of their own."""
    kv, page, ns, ctx = 3, 32, np.array([21, 5, 40]), np.array([30, 5, 77])
    T, w = int(ns.sum()), kv * hd
    pages = make_pages(cuda, 8, kv, page, hd, shift)
    host = HostCache(pages)
    table = make_table(ctx, page, 8, shift)
    k = torch.randn((T, w + 5), device=cuda).to(DT[dtype])[:, shift:shift + w]
    v = torch.randn((T, w + 8), device=cuda).to(DT[dtype])[:, :w]
    ops.kv8_append(k, v, i32(starts(ns), cuda), i32(ctx, cuda), pages, i32(table, cuda))
    host.append(*(x.double().cpu().numpy().reshape(T, kv, hd) for x in (k, v)), ns, ctx, table)
    host.check(pages)


def test_append_leaves_out_what_has_no_page(cuda):
    kv, hd, page = 2, 64, 32
    pages = make_pages(cuda, 6, kv, page, hd)
    host = HostCache(pages)
    table = np.array([[0, -1, 1], [6, 2, -7], [3, 4, 5], [-1, -1, -1]], np.int32)  # 6 is past the pool
    ns = np.array([70, 40, 12, 5])
    ctx = np.array([90, 130, 7, 5])  # second: past its table; third: five rows before position 0
    T = int(ns.sum()) + 2
    x = torch.randn((T, 2 * kv * hd), device=cuda)
    k, v = x[:, :kv * hd], x[:, kv * hd:]
    ops.kv8_append(k, v, i32(starts(ns), cuda), i32(ctx, cuda), pages, i32(table, cuda))
    f = x.double().cpu().numpy()
    host.append(f[:, :kv * hd].reshape(T, kv, hd), f[:, kv * hd:].reshape(T, kv, hd), ns, ctx, table)
    host.check(pages)
    back = torch.full((1,), 7.0, device=cuda)
    rk, rv = ops.kv8_read(i32(starts(ns), cuda), i32(ctx, cuda), pages, i32(table, cuda), int(ns.sum()))
    t = 0
    for b, n in enumerate(ns):
        for which, got in ((0, rk), (1, rv)):
            vals, ok = host.values(which, table[b], int(ctx[b]))
            for i in range(n):
                p = ctx[b] - n + i
                want = vals[p] if p >= 0 and ok[p] else 0.0 * vals[0]
                assert np.array_equal(got[t + i].cpu().numpy(), want.astype(np.float32))
        t += n
    assert float(back) == 7.0


# ------------------------------------------------------------------ attention
def reference(host, q, ns, ctx, table, heads):
    """f64 outputs, and per element the bound of the module's docstring without the output's rounding."""
    kv, _, hd = host.c[0].shape[1:]
    G = heads // kv
    T = q.shape[0]
    out, tol = np.zeros((T, heads, hd)), np.zeros((T, heads, hd))
    t = 0
    for b, n in enumerate(ns):
        c = int(ctx[b])
        K, ok = host.values(0, table[b], max(c, 0))
        V, _ = host.values(1, table[b], max(c, 0))
        for i in range(n):
            e = c - n + i + 1
            see = ok[:max(e, 0)]
            if see.any():
                for h in range(heads):
                    k, v = K[:e, h // G][see], V[:e, h // G][see]
                    s = k @ q[t + i, h] / math.sqrt(hd)
                    smag = (np.abs(k) @ np.abs(q[t + i, h])).max() / math.sqrt(hd)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    mag = p @ np.abs(v)
                    E = 2.0 ** -21 + (hd // 16 + 3 + 2) * 2.0 ** -23
                    out[t + i, h] = p @ v
                    wmax = (p * host.scale_of(1, table[b], e, h // G)[see]).max()
                    tol[t + i, h] = mag * (2 * smag * E + 2.0 ** -18) + len(p) * 127 * 2.0 ** -39 * wmax
                    tol16 = mag * 2.0 ** -11
                    reference.tol16[t + i, h] = tol16
        t += n
    return out, tol


def run_case(cuda, kv, G, hd, page, ns, ctx, dtype="f32", seed=0, table=None, qscale=1.0, pages=None, pad=2,
             strided=False):
    ns, ctx = np.asarray(ns), np.asarray(ctx)
    total = sum(-(-max(int(c), 0) // page) for c in ctx) + 2
    pages = pages or make_pages(cuda, total, kv, page, hd, seed)
    table = make_table(ctx, page, pages.num_pages, seed) if table is None else table
    heads, T = kv * G, int(ns.sum()) + pad
    w = heads * hd
    wide = (torch.randn((T, w + 64), device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)) *
            qscale).to(DT[dtype])
    q = wide[:, 32:32 + w] if strided else wide[:, :w].contiguous()
    out = torch.full((T, w + (8 if strided else 0)), 3.0, dtype=DT[dtype], device=cuda)[:, :w]
    got = ops.kv8_attention(q, i32(starts(ns), cuda), i32(ctx, cuda), heads, pages, i32(table, cuda), out=out)
    assert got is out
    host = HostCache(pages)
    reference.tol16 = np.zeros((T, heads, hd))
    ref, tol = reference(host, q.double().cpu().numpy().reshape(T, heads, hd), ns, ctx, table, heads)
    used = int(ns.sum())
    g = got.double().cpu().numpy().reshape(T, heads, hd)
    assert np.array_equal(g[used:], np.full_like(g[used:], 3.0)), "padding rows were written"
    eps = torch.finfo(DT[dtype]).eps / 2
    tol = tol + (0 if dtype == "f32" else reference.tol16) + eps * np.abs(ref)
    tol += torch.finfo(DT[dtype]).smallest_normal * eps + 1e-37
    err = np.abs(g - ref)[:used]
    assert (err <= tol[:used]).all(), (err / tol[:used]).max()
    return g[:used], ref[:used]


@pytest.mark.parametrize("kv,G,hd,page", [(8, 4, 128, 64), (2, 3, 128, 64), (8, 4, 64, 64), (2, 1, 64, 16),
                                          (1, 8, 128, 32), (2, 2, 64, 48), (1, 16, 64, 128), (3, 5, 128, 64),
                                          (1, 71, 64, 64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_one_token(cuda, kv, G, hd, page, dtype):
    ctx = [1, 15, 16, 17, 63, 64, 65, 300, 2]
    run_case(cuda, kv, G, hd, page, [1] * len(ctx), ctx, dtype, seed=kv + G)


@pytest.mark.parametrize("kv,G,hd,page", [(2, 4, 128, 64), (1, 3, 64, 16), (2, 1, 128, 32), (1, 12, 64, 64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_several_tokens(cuda, kv, G, hd, page, dtype):
    """Drafts, chunks and empty sequences in one call; one sequence starts at position 0."""
    run_case(cuda, kv, G, hd, page, [5, 0, 1, 17, 40, 2, 9], [200, 30, 1, 17, 131, 65, 70], dtype, seed=G, strided=True)


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("gone", [0, 12])
def test_attention_long_chunks_in_one_stretch(cuda, hd, gone):
    """330 times the same chunk, so that a CTA takes all of one: sums over many tiles, with scores
    that grow along the context and, where pages are gone, none for the first tiles."""
    kv, G, page, n, ctx, S = 1, 4, 64, 32, 2000, 330
    pages = make_pages(cuda, 32, kv, page, hd, 5)
    pages.k_scale.mul_(torch.linspace(0.2, 3.0, 32, device=cuda)[:, None, None])
    row = np.arange(32, dtype=np.int32)
    row[:gone] = -1
    q = torch.randn((n, kv * G * hd), device=cuda, generator=torch.Generator(device=cuda).manual_seed(5))
    got = ops.kv8_attention(q.repeat(S, 1), i32(starts([n] * S), cuda), i32([ctx] * S, cuda), kv * G, pages,
                            i32(np.tile(row, (S, 1)), cuda)).view(S, n, G, hd)
    host = HostCache(pages)
    reference.tol16 = np.zeros((n, G, hd))
    ref, tol = reference(host, q.double().cpu().numpy().reshape(n, G, hd), [n], [ctx], row[None], G)
    tol = torch.from_numpy(tol + 2.0 ** -24 * np.abs(ref) + 1e-37).to(cuda)
    err = (got.double() - torch.from_numpy(ref).to(cuda)).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    # and as a whole within twice an f32 sum's rounding of 2000 terms at random, 2000 ** 0.5 * 2 ** -24
    assert float(err.norm() / (S ** 0.5 * np.linalg.norm(ref))) < 2 * 2000 ** 0.5 * 2.0 ** -24


@pytest.mark.parametrize("G,hd", [(3, 128), (5, 64), (7, 128), (71, 64), (128, 64), (130, 128)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width", [0, 2500])
def test_attention_chunks_of_odd_groups(cuda, G, hd, dtype, width):
    """Head groups that do not fill a tile's rows, or need several tiles, in chunks; the table's
    width decides how the call is cut up."""
    ns, ctx, page = [33, 0, 50], [120, 7, 50], 16
    pages = make_pages(cuda, 20, 1, page, hd, G)
    run_case(cuda, 1, G, hd, page, ns, ctx, dtype, G, make_table(ctx, page, 20, G, width=max(8, width)), pages=pages)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_chunks(cuda, dtype):
    run_case(cuda, 2, 4, 128, 64, [130, 67], [515, 67], dtype, seed=3)
    run_case(cuda, 1, 4, 64, 64, [257], [1000], dtype, seed=4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_missing_pages_and_empty_rows(cuda, dtype):
    """Freed pages are masked; rows without any visible position give zeros."""
    kv, G, hd, page = 2, 4, 128, 32
    pages = make_pages(cuda, 40, kv, page, hd, 7)
    ctx = [100, 64, 40, 3, 200, 0, 90]
    ns = [1, 2, 3, 5, 40, 1, 30]  # fourth: two rows before position 0; sixth: no position at all
    table = make_table(ctx, page, 40, 7, width=8)
    table[0, :2] = -1
    table[1, :] = -1
    table[2, 0] = 40  # past the pool
    table[4, 1:5] = [-1, 41, -3, table[4, 4]]
    table[6, 0] = -1
    g, ref = run_case(cuda, kv, G, hd, page, ns, ctx, dtype, 7, table, pages=pages)
    assert not g[1:3].any() and not g[6:8].any()
    # a table narrower than the length: the positions behind it are not there
    run_case(cuda, kv, G, hd, page, [2], [200], dtype, 8, table[4:5, :6].copy(), pages=pages)


def test_attention_scales_far_apart(cuda):
    """Blocks whose scales differ by many orders, zero scales, and content behind ctx that is not a number."""
    kv, G, hd, page = 1, 4, 128, 64
    pages = make_pages(cuda, 6, kv, page, hd, 9)
    g = torch.Generator(device=cuda).manual_seed(9)
    pages.v_scale.copy_(10.0 ** (torch.rand(pages.v_scale.shape, generator=g, device=cuda) * 24 - 12))
    pages.k_scale.mul_(torch.rand(pages.k_scale.shape, generator=g, device=cuda) * 2)
    pages.v_scale[1, 0, 2] = 0.0
    pages.k_scale[2, 0, 1] = 0.0
    table = np.array([[1, 2, 0, 3], [5, 4, -1, -1]], np.int32)
    # behind ctx: block 13 on of the first, block 5 on of the second sequence
    for row, blk in ((0, 13), (1, 5)):
        for j in range(blk, 16 if row == 0 else 8):
            pages.k_scale[int(table[row, j // 4]), 0, j % 4] = float("nan")
            pages.v_scale[int(table[row, j // 4]), 0, j % 4] = float("inf")
    run_case(cuda, kv, G, hd, page, [1, 3], [203, 71], "f32", 9, table, pages=pages)
    run_case(cuda, kv, G, hd, page, [20, 71], [203, 71], "f32", 9, table, pages=pages)
    # every scale of v zero
    pages.v_scale.zero_()
    got, _ = run_case(cuda, kv, G, hd, page, [1, 1], [203, 71], "f32", 9, table, pages=pages)
    assert not got.any()


@pytest.mark.parametrize("qscale", [1e-30, 1e-3, 30.0, 3e4])
def test_attention_query_sizes(cuda, qscale):
    """q far below and far above the 16-bit range; at 3e4 one position takes all the weight."""
    run_case(cuda, 2, 4, 64, 64, [1, 4], [150, 90], "f32", 11, qscale=qscale)


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_unaligned_rows(cuda, hd, dtype):
    """q and out rows that do not begin at a multiple of 16 bytes, decode rows and chunks."""
    kv, G, page, table_width = 2, 4, 64, 900
    for ns, ctx in (([1, 1, 1], [500, 64, 3]), ([70, 130], [300, 130])):
        ns, ctx = np.array(ns), np.array(ctx)
        pages = make_pages(cuda, 16, kv, page, hd, hd)
        table = make_table(ctx, page, 16, hd, width=table_width)
        heads, T = kv * G, int(ns.sum())
        w = heads * hd
        q = torch.randn((T, w + 7), device=cuda).to(DT[dtype])[:, 3:3 + w]
        args = i32(starts(ns), cuda), i32(ctx, cuda), heads, pages, i32(table, cuda)
        want = ops.kv8_attention(q.contiguous(), *args)
        out = torch.empty((T, w + 1), dtype=DT[dtype], device=cuda)[:, 1:]
        assert torch.equal(ops.kv8_attention(q, *args, out=out), want)


def test_attention_long_context_splits(cuda):
    """A few long sequences: their axis is split over CTAs and joined."""
    run_case(cuda, 2, 4, 128, 64, [1, 1, 5], [9001, 33, 4100], "f32", 12)
    run_case(cuda, 1, 2, 64, 16, [1], [20000], "bf16", 13)


def test_attention_offsets_past_32_bits(cuda):
    """Pages behind the first 2^31 code bytes of a pool."""
    kv, hd, page = 8, 128, 64
    n = 2 ** 31 // (kv * page * hd) + 3  # 65536 bytes a page and tensor
    pages = ops.KV8Pages.empty(n, kv, page, hd, cuda)
    table = np.array([[n - 1, 0, n - 2]], np.int32)
    ns, ctx = np.array([150]), np.array([150])
    x = torch.randn((150, 2 * kv * hd), device=cuda)
    ops.kv8_append(x[:, :kv * hd], x[:, kv * hd:], i32(starts(ns), cuda), i32(ctx, cuda), pages, i32(table, cuda))
    small = ops.KV8Pages(*(t[[n - 1, 0, n - 2]].contiguous() for t in pages.tensors()))
    k, v = ops.kv8_read(i32(starts(ns), cuda), i32(ctx, cuda), pages, i32(table, cuda), 150)
    # a code is off by half a step, scale / 2 = max|x| / 254 of its block; scale and product round by 2^-24 each
    half = float(x.abs().max()) / 254 * (1 + 2.0 ** -15)
    assert float((k.view(150, -1) - x[:, :kv * hd]).abs().max()) <= half and int(small.k.abs().max()) == 127
    q = torch.randn((3, 32 * hd), device=cuda)
    args = i32([0, 3], cuda), i32(ctx, cuda), 32
    a = ops.kv8_attention(q, *args, pages, i32(table, cuda))
    b = ops.kv8_attention(q, *args, small, i32([[0, 1, 2]], cuda))
    assert torch.equal(a, b)
    del pages


@pytest.mark.parametrize("hd,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("G,most,dtype", [(4, 1, "f32"), (4, 1, "bf16"), (2, 3, "f32"), (8, 24, "f32"),
                                          (8, 24, "f16")])
@pytest.mark.parametrize("width", [0, 500, 4000])
def test_attention_many_sequences(cuda, hd, page, G, most, dtype, width):
    """More sequences than threads of a CTA, empty ones among them; how the call is cut up goes
    by the table's width, whatever the sequences' lengths are."""
    rng = np.random.default_rng(G + most)
    S = 401
    ns = rng.integers(most > 1, most + 1, S)
    ns[rng.integers(0, S, 30)] = 0
    ctx = ns + rng.integers(0, 70, S)
    ctx[ns == 0] //= 8
    ctx[[7, 300, 399]] += 300
    pages = make_pages(cuda, sum(-(-int(c) // page) for c in ctx), 2, page, hd, G)
    table = make_table(ctx, page, pages.num_pages, G, width=max(width, -(-int(ctx.max()) // page)))
    run_case(cuda, 2, G, hd, page, ns, ctx, dtype, G, table, pages=pages)


@pytest.mark.parametrize("most", [1, 40])
def test_attention_wide_tables_one_sequence(cuda, most):
    """A table far wider than the one sequence, whose pages end inside a tile."""
    for c in (most, 100, 1000):
        pages = make_pages(cuda, 64, 1, 16, 128, c)
        run_case(cuda, 1, 4, 128, 16, [most], [c], "f32", c, make_table([c], 16, 64, c, width=20000), pages=pages)


def test_attention_repeats_and_streams(cuda):
    """The same call twice, on two streams at once, and replayed from two graphs: the same bits."""
    kv, G, hd, page = 8, 4, 128, 64
    ctx = np.array([5000, 17, 1, 900])
    pages = make_pages(cuda, 100, kv, page, hd, 21)
    table = i32(make_table(ctx, page, 100, 21), cuda)
    st, cx = i32(starts([1] * 4), cuda), i32(ctx, cuda)
    q = [torch.randn((4, kv * G * hd), device=cuda) for _ in range(2)]
    want = [ops.kv8_attention(x, st, cx, kv * G, pages, table) for x in q]
    graphs, outs = [], []
    for x in q:
        o = torch.empty_like(x)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            ops.kv8_attention(x, st, cx, kv * G, pages, table, out=o)
        graphs.append(g)
        outs.append(o)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for x, g in zip(s, graphs):
            with torch.cuda.stream(x):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        eager = []
        for x, st_ in zip(q, s):
            with torch.cuda.stream(st_):
                eager.append(ops.kv8_attention(x, st, cx, kv * G, pages, table))
        torch.cuda.synchronize()
        assert torch.equal(eager[0], want[0]) and torch.equal(eager[1], want[1])


@pytest.mark.parametrize("ns,ctx,width", [([300, 5, 200], [900, 70, 200], 0), ([1] * 40, list(range(1, 1600, 40)), 300),
                                          ([40] * 20, list(range(40, 1640, 80)), 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_forms_repeat_and_overlap(cuda, ns, ctx, width, dtype):
    """Chunks, many sequences and short chunks: two graphs replayed on two streams at once,
    next to calls on a third, give the bits of the first calls."""
    kv, G, hd, page = 4, 4, 128, 16
    ns, ctx = np.array(ns), np.array(ctx)
    total = int(sum(-(-c // page) for c in ctx))
    pages = make_pages(cuda, total, kv, page, hd, 31)
    table = i32(make_table(ctx, page, total, 31, width=max(width, -(-int(ctx.max()) // page))), cuda)
    st, cx = i32(starts(ns), cuda), i32(ctx, cuda)
    T = int(ns.sum())
    q = [torch.randn((T, kv * G * hd), device=cuda).to(DT[dtype]) for _ in range(3)]
    want = [ops.kv8_attention(x, st, cx, kv * G, pages, table) for x in q]
    graphs, outs = [], []
    for x in q[:2]:
        o, g = torch.empty_like(x), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            ops.kv8_attention(x, st, cx, kv * G, pages, table, out=o)
        graphs.append(g)
        outs.append(o)
    s = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for x, g in zip(s, graphs):
            with torch.cuda.stream(x):
                g.replay()
        with torch.cuda.stream(s[2]):
            third = [ops.kv8_attention(q[2], st, cx, kv * G, pages, table) for _ in range(2)]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(third[0], want[2]) and torch.equal(third[1], want[2])
    ops.device_status()


def test_attention_matches_the_f32_cache(cuda):
    """kv8_attention over appended rows against ops.attention over the values read back: the
    same numbers by two paths of the library, both f32 to about 1e-6."""
    kv, G, hd, page = 2, 4, 128, 64
    ctx = np.array([150, 64])
    pages = ops.KV8Pages.empty(8, kv, page, hd, cuda)
    table = make_table(ctx, page, 8, 3)
    T = int(ctx.sum())
    x = torch.randn((T, 2 * kv * hd), device=cuda)
    args = i32(starts(ctx), cuda), i32(ctx, cuda)
    ops.kv8_append(x[:, :kv * hd], x[:, kv * hd:], *args, pages, i32(table, cuda))
    kf, vf = ops.kv8_read(*args, pages, i32(table, cuda), T)
    kp, vp = (torch.zeros((8, kv, page, hd), device=cuda) for _ in range(2))
    t = 0
    for b, n in enumerate(ctx):
        for p in range(n):
            kp[table[b, p // page], :, p % page], vp[table[b, p // page], :, p % page] = kf[t], vf[t]
            t += 1
    q = torch.randn((2, kv * G * hd), device=cuda)
    a = ops.kv8_attention(q, i32([0, 1, 2], cuda), i32(ctx, cuda), kv * G, pages, i32(table, cuda))
    b = ops.attention(q, i32(ctx - 1, cuda), i32([0, 1], cuda), kv * G, kv, hd, kp, vp, page, i32(table, cuda))
    assert float((a - b).norm() / b.norm()) < 1e-5


def test_refusals(cuda):
    pages = ops.KV8Pages.empty(4, 2, 32, 64, cuda)
    st, cx, tb = i32([0, 1], cuda), i32([1], cuda), i32([[0]], cuda)
    q = torch.zeros((1, 256), device=cuda)
    with pytest.raises(ValueError):
        ops.kv8_attention(q, st, cx, 4, pages, tb.long())
    with pytest.raises(ValueError):
        ops.kv8_attention(q, st[:1], cx, 4, pages, tb)
    with pytest.raises(ValueError):
        ops.kv8_attention(q[:, :128], st, cx, 4, pages, tb)
    with pytest.raises(ValueError):
        ops.kv8_attention(q.double(), st, cx, 4, pages, tb)
    with pytest.raises(_lib.Q8Error):
        ops.kv8_attention(torch.zeros((1, 192), device=cuda), st, cx, 3, pages, tb)
    with pytest.raises(_lib.Q8Error):  # rows that lie on top of one another
        ops.kv8_attention(q.expand(5, 256), st, cx, 4, pages, tb)
    with pytest.raises(ValueError):
        ops.kv8_append(q[:, :128], q[:, :128].half(), st, cx, pages, tb)
    with pytest.raises(ValueError):
        ops.KV8Pages.empty(4, 2, 24, 64, cuda)
    with pytest.raises(ValueError):
        ops.KV8Pages.empty(4, 2, 32, 96, cuda)
    # nothing to do is not an error
    assert ops.kv8_attention(q[:0], i32([0, 0], cuda), cx, 4, pages, tb).shape == (0, 256)
    assert ops.kv8_read(i32([0], cuda), i32([], cuda), pages, torch.zeros((0, 3), dtype=torch.int32, device=cuda),
                        0)[0].shape == (0, 2, 64)
