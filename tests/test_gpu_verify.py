"""probs and verify against 64-bit restatements, and a whole speculative step
over the 8-bit cache.

probs: w = exp(x), x = (l - max) / temp in f32, |x| <= 16 / temp: l - max and
the quotient round by 2^-24 |x| each, expf is good to 2 ulps, the sum is 64
bits, the product rounds twice more: |p - ref| <= p (2 |x| 2^-24 + 6 2^-24).
verify: tokens and counts are whole numbers and have to be equal; its sums are
64 bits on both sides."""
import numpy as np
import pytest
import torch

from lama32_mojo_b200 import ops

pytestmark = pytest.mark.gpu


def i32(a, cuda):
    return torch.tensor(np.asarray(a, np.int32), device=cuda)


def ref_probs(l, temp):
    """f64 p, and x of each entry."""
    ok = ~np.isnan(l) & (l > -np.inf)
    if not ok.any():
        p = np.zeros(len(l))
        p[0] = 1
        return p, np.zeros(len(l))
    top = l[ok].max()
    if temp <= 0:
        p = np.zeros(len(l))
        p[np.flatnonzero(ok & (l == top))[0]] = 1
        return p, np.zeros(len(l))
    with np.errstate(invalid="ignore"):
        cand = ok & (l >= np.float32(top) - np.float32(16)) if np.isfinite(top) else ok & (l == top)
        x = np.where(cand & (l != top), (l.astype(np.float64) - np.float64(top)) / np.float64(np.float32(temp)), 0.0)
    w = np.where(cand, np.exp(x), 0.0)
    return w / w.sum(), x


def check_probs(x, temp, cuda, pad=0):
    rows, n = x.shape
    t = torch.full((rows, n + pad), 1e9, device=cuda)
    t[:, :n] = torch.from_numpy(x).to(cuda)
    got = ops.probs(t[:, :n], temp).double().cpu().numpy()
    for r in range(rows):
        p, e = ref_probs(x[r], temp)
        tol = p * (2 * np.abs(e) + 6) * 2.0 ** -24 + 2.0 ** -149
        assert (np.abs(got[r] - p) <= tol).all(), (r, temp, (np.abs(got[r] - p) / tol).max())


@pytest.mark.parametrize("n", [1, 2, 31, 1000, 4097, 50003, 128256])
@pytest.mark.parametrize("temp", [0.0, 0.3, 1.0, 2.5])
def test_probs(cuda, n, temp):
    rng = np.random.default_rng(n)
    check_probs((rng.standard_normal((3, n)) * 6).astype(np.float32), temp, cuda, pad=n % 3)


def test_probs_many_rows(cuda):
    rng = np.random.default_rng(1)
    check_probs((rng.standard_normal((700, 1003)) * 4).astype(np.float32), 0.7, cuda, pad=1)


@pytest.mark.parametrize("rows,n", [(300, 30011), (5, 200001), (2, 327680)])
@pytest.mark.parametrize("temp", [0.0, 0.9])
def test_probs_large_slices(cuda, rows, n, temp):
    """More rows than fit at once, and rows that take the larger CTAs; equal maxima in several of them."""
    x = (np.random.default_rng(n).standard_normal((rows, n)) * 3).astype(np.float32)
    x[1, [n - 1, 17, n // 2]] = 40.0
    x[0, n // 3] = np.inf
    check_probs(x, temp, cuda, pad=rows % 4)


def test_probs_in_place(cuda):
    x = torch.randn((40, 50000), device=cuda) * 4
    want = ops.probs(x, 0.8)
    assert ops.probs(x, 0.8, out=x) is x and torch.equal(x, want)


def test_probs_special_rows(cuda):
    inf, nan, low = np.inf, np.nan, np.finfo(np.float32).min
    rows = np.zeros((9, 40), np.float32)
    rows[0] = -inf
    rows[1] = nan
    rows[2, ::2] = nan
    rows[3, 5:9] = inf
    rows[4] = low
    rows[5] = -inf
    rows[5, 17] = low
    rows[6] = np.linspace(-20, 0, 40)
    rows[6, 3] = -16.0  # on the border: a candidate
    rows[7, [4, 9]] = 3.0
    rows[8] = 3e38
    rows[8, 1::2] = -3e38
    for temp in (1.0, 0.05, 0.0, 50.0, 1e-30, 1e-44):
        check_probs(rows, temp, cuda)


def ref_verify(p, q, ids, starts, u):
    taken, tokens = [], np.full(len(ids), -7)
    at = 0
    n = p.shape[1]
    for b in range(len(starts) - 1):
        lo, hi = starts[b], starts[b + 1]
        if hi <= lo:
            taken.append(0)
            continue
        r = lo
        while r < hi - 1:
            x = ids[r + 1]
            if not 0 <= x < n:
                break
            qx = 1.0 if q is None else np.float64(q[at + r - lo, x])
            if not np.float64(u[r]) * qx < np.float64(p[r, x]):
                break
            r += 1
        w = p[r].astype(np.float64)
        base = np.where(w > 0, w, 0)
        if r < hi - 1 and q is not None:
            w = w - q[at + r - lo].astype(np.float64)
        elif r < hi - 1 and 0 <= ids[r + 1] < n:
            w[ids[r + 1]] = 0
        w = np.where(w > 0, w, 0)
        if not w.sum() > 0:
            w = base
        cum = np.cumsum(w)
        over = np.flatnonzero(cum > np.float64(u[hi - 1]) * cum[-1])
        some = np.flatnonzero(w > 0)
        new = over[0] if len(over) else some[-1] if len(some) else 0
        taken.append(r - lo)
        tokens[lo:r] = ids[lo + 1:r + 1]
        tokens[r] = new
        tokens[r + 1:hi] = -1
        at += hi - lo - 1
    return np.array(taken), tokens


def check_verify(p, q, ids, starts, u, cuda, padded=0):
    def wide(x):
        t = torch.full((x.shape[0], x.shape[1] + 3), float("nan"), device=cuda)
        t[:, :x.shape[1]] = torch.from_numpy(x).to(cuda)
        return t[:, :x.shape[1]]
    a, t = ops.verify(wide(p), None if q is None else wide(q), i32(ids, cuda), i32(starts, cuda),
                      torch.from_numpy(u).to(cuda))
    wa, wt = ref_verify(p, q, ids, starts, u)
    used = int(starts[-1])
    assert np.array_equal(a.cpu().numpy(), wa)
    assert np.array_equal(t.cpu().numpy()[:used], wt[:used]), (t.cpu().numpy()[:used], wt[:used])
    return wa


def rows_of(rng, rows, n, scale=3.0):
    x = rng.standard_normal((rows, n)) * scale
    x = np.exp(x - x.max(1, keepdims=True))
    return (x / x.sum(1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("n", [1, 2, 33, 1000, 4099, 50003, 151936])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(cuda, n, certain):
    rng = np.random.default_rng(n + certain)
    counts = [5, 1, 3, 9, 1, 2, 6]
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = starts[-1] + 2  # two rows of padding
    p = rows_of(rng, rows, n)
    last = set(starts[1:] - 1)
    body = [r for r in range(starts[-1]) if r not in last]
    noisy = p[body] * np.exp(0.4 * rng.standard_normal((len(body), n)))
    q = (noisy / noisy.sum(1, keepdims=True)).astype(np.float32)
    ids = rng.integers(0, n, rows)
    for k, r in enumerate(body):
        ids[r + 1] = rng.choice(n, p=q[k].astype(np.float64) / q[k].astype(np.float64).sum())
    u = rng.random(rows).astype(np.float32)
    u[starts[1] - 1], u[starts[2] - 1] = 0.0, np.float32(1) - np.float32(2.0 ** -24)
    check_verify(p, None if certain else q, ids, starts, u, cuda)


def test_verify_edges(cuda):
    """Sequences without rows, p equal to q, drafts that cannot be, NaN, rows without weight."""
    n = 50
    rng = np.random.default_rng(2)
    counts = [2, 0, 3, 1, 0, 2, 2, 2, 2, 3, 2]
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = starts[-1]
    p = rows_of(rng, rows, n)
    body = [r for b in range(len(counts)) for r in range(starts[b], max(starts[b], starts[b + 1] - 1))]
    q = p[body].copy()
    ids = rng.integers(0, n, rows)
    u = np.full(rows, 0.5, np.float32)
    u[starts[0]] = 1.0  # refused although p == q: p itself is drawn from
    ids[starts[5] + 1] = -1
    ids[starts[6] + 1] = n
    p[starts[7]] = np.nan
    p[starts[8]] = 0.0  # refused, nothing to draw from: token 0
    q[body.index(starts[9])] = np.nan
    p[starts[10], ids[starts[10] + 1]] = 0.0
    for certain in (False, True):
        got = check_verify(p, None if certain else q, ids, starts, u, cuda)
        assert got[0] == 0
    # greedy: one-hot p, certain drafts: kept as long as they are the argmax
    logits = torch.randn((9, 1000), device=cuda)
    best = logits.argmax(-1).cpu().numpy()
    ids = np.concatenate([[3], best[:8]])
    ids[4] = (ids[4] + 1) % 1000
    a, t = ops.verify(ops.probs(logits, 0.0), None, i32(ids, cuda), i32([0, 9], cuda), torch.rand(9, device=cuda))
    assert int(a) == 3 and t.tolist() == list(best[:4]) + [-1] * 5


def test_verify_follows_the_target(cuda):
    """The first token of many calls is distributed as p, whatever q is: the counts of 40,000 draws
    stay within 5 standard deviations."""
    n, S = 8, 40000
    rng = np.random.default_rng(3)
    p, q = rows_of(rng, 2, n, 1.0), rows_of(rng, 1, n, 1.0)
    P = torch.from_numpy(p).to(cuda).repeat(S, 1)
    Q = torch.from_numpy(q).to(cuda).repeat(S, 1)
    ids = np.zeros(2 * S, np.int64)
    ids[1::2] = rng.choice(n, S, p=q[0].astype(np.float64) / q[0].astype(np.float64).sum())
    a, t = ops.verify(P, Q, i32(ids, cuda), i32(np.arange(0, 2 * S + 1, 2), cuda),
                      torch.from_numpy(rng.random(2 * S).astype(np.float32)).to(cuda))
    first = t.view(S, 2)[:, 0].cpu().numpy()
    got = np.bincount(first, minlength=n)
    want = p[0].astype(np.float64) / p[0].astype(np.float64).sum()
    assert (np.abs(got - S * want) <= 5 * np.sqrt(S * want * (1 - want))).all()
    assert 0 < int(a.sum()) < S


def test_refusals(cuda):
    p = torch.ones((3, 10), device=cuda)
    ids, st, u = i32([0, 1, 2], cuda), i32([0, 3], cuda), torch.zeros(3, device=cuda)
    a, t = ops.verify(p, p[:1] * 0, i32([0, 1, 2], cuda), st, u)  # no row of q for the second draft: refused
    assert a.tolist() == [1] and t.tolist() == [1, 0, -1]
    for bad in (lambda: ops.verify(p, p[:, :9], ids, st, u),
                lambda: ops.verify(p.double(), None, ids, st, u), lambda: ops.verify(p, None, ids.long(), st, u),
                lambda: ops.verify(p, None, ids, st, u[:2]), lambda: ops.verify(p.t(), None, ids, st, u),
                lambda: ops.probs(p.t(), 1.0), lambda: ops.probs(p.half(), 1.0),
                lambda: ops.probs(p, 1.0, out=p[:2])):
        with pytest.raises(ValueError):
            bad()
    assert ops.probs(p[:0], 1.0).shape == (0, 10)
    a, t = ops.verify(p[:0], None, ids[:0], i32([0, 0], cuda), u[:0])
    assert a.tolist() == [0] and t.numel() == 0


# ------------------------------------------------------------------ all of them together
def test_speculative_decoding_over_the_8_bit_cache(cuda):
    """A two-layer toy model decodes three sequences (two forked from the first) with drafts from
    a weaker model: pages reserved, shared pages copied, rows rotated, appended and attended to,
    distributions verified, refused positions given back.  Greedily (temp 0) the tokens have to be
    those of the same model fed one token at a time with a cache of its own."""
    nh, kv, hd, V, page, L = 4, 2, 64, 97, 16, 2
    g = torch.Generator(device=cuda).manual_seed(5)
    H, qd, kd = 128, nh * hd, kv * hd

    def rnd(*s):
        return torch.randn(s, generator=g, device=cuda) / s[-1] ** 0.5

    emb = rnd(V, H) * 8
    layers = [(rnd(qd + 2 * kd, H), rnd(H, qd)) for _ in range(L)]
    inv = 1.0 / 10000.0 ** (torch.arange(hd // 2, device=cuda).float() / (hd // 2))

    def model(ids, starts, ctx, pos, table, pages):
        h = emb[ids.long()]
        for (wqkv, wo), pg in zip(layers, pages):
            qkv = (h / h.norm(dim=-1, keepdim=True) * H ** 0.5) @ wqkv.t()
            ops.rope(qkv, pos, nh, kv, hd, inv)
            ops.kv8_append(qkv[:, qd:qd + kd], qkv[:, qd + kd:], starts, ctx, pg, table)
            h = h + ops.kv8_attention(qkv[:, :qd], starts, ctx, nh, pg, table) @ wo.t()
        return h @ emb.t()

    class Cache:
        def __init__(self, S, num):
            self.S = S
            self.pages = [ops.KV8Pages.empty(num, kv, page, hd, cuda) for _ in range(L)]
            self.table = torch.full((S, 8), -1, dtype=torch.int32, device=cuda)
            self.ctx = torch.zeros(S, dtype=torch.int32, device=cuda)
            self.refs = torch.zeros(num, dtype=torch.int32, device=cuda)

        def feed(self, rows):
            """rows: a token list per sequence; logits of all of them."""
            ns = [len(r) for r in rows]
            src, dst, status = ops.kv_reserve(self.table, self.ctx, self.refs, page, i32(ns, cuda))
            assert status[0] == 0
            ops.kv_copy_pages([t for p in self.pages for t in p.tensors()], src, dst)
            st = np.concatenate([[0], np.cumsum(ns)])
            c = self.ctx.tolist()
            pos = [c[b] - n + i for b, n in enumerate(ns) for i in range(n)]
            return model(i32([t for r in rows for t in r], cuda), i32(st, cuda), self.ctx, i32(pos, cuda),
                         self.table, self.pages), st

    prompt, S, steps = [3, 14, 15, 92, 65, 35, 89, 79, 32, 38, 46, 26, 43, 38, 32, 79, 50, 28, 84, 19], 3, 6
    # one token at a time
    plain = Cache(1, 8)
    want, logits = [], plain.feed([prompt])[0]
    for _ in range(30):
        want.append(int(logits[-1].argmax()))
        logits = plain.feed([[want[-1]]])[0]
    # drafts: what the plain run said, with mistakes put in at known places
    c = Cache(S, 20)
    logits, _ = c.feed([prompt, [], []])
    ops.kv_fork(c.table, c.ctx, c.refs, page, i32([0, 0], cuda), i32([1, 2], cuda))
    first = int(logits[-1].argmax())
    got = [[first] for _ in range(S)]
    for step in range(steps):
        rows = []
        for b in range(S):
            k = len(got[b])
            draft = want[k:k + 1 + (b + step) % 4]
            if b and draft and (step + b) % 2:
                draft[-1] = (draft[-1] + 1) % V
            rows.append([got[b][-1]] + draft)
        before = c.ctx.clone()
        logits, st = c.feed(rows)
        p = ops.probs(logits, 0.0)
        flat = [t for r in rows for t in r]
        n, tok = ops.verify(p, None, i32(flat, cuda), i32(st, cuda), torch.rand(len(flat), device=cuda))
        ops.kv_truncate(c.table, c.ctx, c.refs, page, before + n + 1)
        for b in range(S):
            got[b] += [t for t in tok[st[b]:st[b + 1]].tolist() if t >= 0]
    # 8-bit blocks round a token by its neighbours: as long as no refused draft has been in a
    # block the two runs hold the same codes; later the logits may differ by a code's rounding
    for b in range(S):
        k = min(len(got[b]), len(want))
        assert got[b][:k] == want[:k], (b, got[b], want)
    assert np.array_equal(np.bincount(c.table[c.table >= 0].cpu().numpy(), minlength=20), c.refs.cpu().numpy())


@pytest.mark.parametrize("kv,hd,normed", [(2, 64, False), (8, 128, True), (1, 128, False)])
def test_rope_rotates_as_rope_kv_append(cuda, kv, hd, normed):
    """The rotation alone, in place, has the bits of the one that writes the f32 cache; v and what
    lies behind a row stay as they were."""
    nh, T, page = 4 * kv, 21, 16
    g = torch.Generator(device=cuda).manual_seed(hd)
    w = (nh + 2 * kv) * hd
    wide = torch.randn((T, w + 32), generator=g, device=cuda)
    inv = 1.0 / 10000.0 ** (torch.arange(0, hd, 2, device=cuda) / hd)
    pos = torch.randint(0, 64, (T,), generator=g, device=cuda, dtype=torch.int32)
    qn, kn = ((torch.rand((hd,), generator=g, device=cuda) + 0.5).bfloat16() for _ in range(2)) if normed else (None, None)
    a, b = wide.clone(), wide.clone()
    ops.rope(a[:, :w], pos, nh, kv, hd, inv, qn, kn)
    kp, vp = (torch.zeros((4 * T, kv, page, hd), device=cuda) for _ in range(2))
    table = torch.arange(4 * T, device=cuda, dtype=torch.int32).view(T, 4)
    ops.rope_kv_append(b[:, :w], pos, torch.arange(T, device=cuda, dtype=torch.int32), nh, kv, hd, inv, qn, kn, 1e-6,
                       kp, vp, page, table)
    assert torch.equal(a[:, :nh * hd], b[:, :nh * hd])
    assert torch.equal(a[:, (nh + kv) * hd:], wide[:, (nh + kv) * hd:])
    for t in range(T):
        p = int(pos[t])
        assert torch.equal(a[t, nh * hd:(nh + kv) * hd].view(kv, hd), kp[4 * t + p // page, :, p % page])
