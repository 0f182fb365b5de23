"""Page tables (kv_truncate, kv_fork, kv_reserve, kv_compact, kv_copy_pages)
against a sequential restatement on the host.  Everything is a whole number or
a copied byte: results have to be equal."""
import numpy as np
import pytest
import torch

from lama32_mojo_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def i32(a, cuda):
    return torch.tensor(np.asarray(a, np.int32), device=cuda)


class Host:
    def __init__(self, S, width, pages, page):
        self.table = np.full((S, width), -1, np.int64)
        self.ctx, self.refs = np.zeros(S, np.int64), np.zeros(pages, np.int64)
        self.page = page

    def cuda(self, dev):
        return i32(self.table, dev), i32(self.ctx, dev), i32(self.refs, dev)

    def check(self, table, ctx, refs):
        assert np.array_equal(table.cpu().numpy(), self.table)
        assert np.array_equal(ctx.cpu().numpy(), self.ctx)
        assert np.array_equal(refs.cpu().numpy(), self.refs)

    def valid(self, e):
        return 0 <= e < len(self.refs)

    def truncate(self, new_len):
        for s, n in enumerate(new_len):
            if n < 0:
                continue
            self.ctx[s] = min(n, self.ctx[s])
            for j in range(-(-self.ctx[s] // self.page), self.table.shape[1]):
                if self.table[s, j] >= 0:
                    if self.valid(self.table[s, j]):
                        self.refs[self.table[s, j]] -= 1
                    self.table[s, j] = -1

    def fork(self, src, dst):
        old, lens, S = self.table.copy(), self.ctx.copy(), len(self.ctx)
        last = {b: a for a, b in zip(src, dst) if 0 <= a < S and 0 <= b < S}
        for b, a in last.items():
            for j in range(old.shape[1]):
                now = old[a, j] if j * self.page < lens[a] and self.valid(old[a, j]) else -1
                if self.valid(old[b, j]):
                    self.refs[old[b, j]] -= 1
                if now >= 0:
                    self.refs[now] += 1
                self.table[b, j] = now
            self.ctx[b] = lens[a]

    def reserve(self, n_new):
        S, width = self.table.shape
        src, dst = np.full(S, -1), np.full(S, -1)
        free = [p for p in range(len(self.refs)) if self.refs[p] == 0]
        want, over, writers = [], False, {}
        for s, n in enumerate(n_new):
            a = self.ctx[s] // self.page
            if n > 0 and (self.ctx[s] + n - 1) // self.page >= width:
                over = True
            elif n > 0 and self.ctx[s] % self.page and self.valid(self.table[s, a]):
                writers.setdefault(self.table[s, a], []).append(s)
        for s, n in enumerate(n_new):
            if n <= 0 or (self.ctx[s] + n - 1) // self.page >= width:
                continue
            a, z = self.ctx[s] // self.page, (self.ctx[s] + n - 1) // self.page
            e = self.table[s, a]
            if self.ctx[s] % self.page and self.valid(e) and self.refs[e] > 1:
                if not (len(writers[e]) == self.refs[e] and writers[e][0] == s):
                    want.append((s, a, e))
            want += [(s, j, -1) for j in range(a, z + 1) if self.table[s, j] < 0]
        if over or len(want) > len(free):
            return src, dst, [_lib.Q8_ERR_KV_FULL, len(want), len(free)]
        for (s, j, e), p in zip(want, free):
            self.table[s, j] = p
            self.refs[p] = 1
            if e >= 0:
                self.refs[e] -= 1
                src[s], dst[s] = e, p
        for s, n in enumerate(n_new):
            self.ctx[s] += max(n, 0)
        return src, dst, [0, len(want), len(free) - len(want)]

    def compact(self):
        n = int((self.refs > 0).sum())
        src = [p for p in range(n, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(n) if self.refs[p] <= 0]
        for a, b in zip(src, dst):
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.table[self.table == a] = b
        fill = [-1] * (len(self.refs) // 2 - len(src))
        return src + fill, dst + fill


@pytest.mark.parametrize("S,width,pages,page", [(1, 1, 1, 16), (7, 9, 40, 16), (64, 33, 1500, 64), (3, 2000, 5003, 1),
                                                (130, 5, 300, 48)])
def test_random_walk(cuda, S, width, pages, page):
    """Every call in random order on one state: growth, forks (permutations and duplicates among
    them), shortening, freeing and compaction; refs always count the table."""
    rng = np.random.default_rng(S * width)
    h = Host(S, width, pages, page)
    table, ctx, refs = h.cuda(cuda)
    full = 0
    for step in range(60):
        kind = rng.integers(0, 5)
        if kind in (0, 1):
            room = max(1, 2 * pages * page // (3 * S))
            n = rng.integers(-1, min(room, width * page) // 2 + 2, S)
            if rng.random() < 0.5:
                n = rng.integers(0, 2, S)
            src, dst, status = ops.kv_reserve(table, ctx, refs, page, i32(n, cuda))
            a, b, c = h.reserve(n)
            assert status.tolist() == c
            assert src.tolist() == list(a) and dst.tolist() == list(b)
            full += c[0] != 0
        elif kind == 2:
            n = int(rng.integers(1, S + 3))
            src, dst = rng.integers(-1, S + 1, n), rng.integers(-1, S + 1, n)
            if rng.random() < 0.3:
                src, dst = rng.permutation(S), np.arange(S)
            ops.kv_fork(table, ctx, refs, page, i32(src, cuda), i32(dst, cuda))
            h.fork(src, dst)
        elif kind == 3:
            n = np.where(rng.random(S) < 0.4, -1, rng.integers(0, width * page + 1, S))
            ops.kv_truncate(table, ctx, refs, page, i32(n, cuda))
            h.truncate(n)
        else:
            src, dst = ops.kv_compact(table, refs)
            a, b = h.compact()
            assert src.tolist() == a and dst.tolist() == b
        h.check(table, ctx, refs)
        assert np.array_equal(np.bincount(h.table[h.table >= 0], minlength=pages), h.refs)
    assert full or pages > 1000


def test_reserve_is_all_or_nothing(cuda):
    h = Host(3, 4, 5, 16)
    table, ctx, refs = h.cuda(cuda)
    for n, code in (([16, 1, 16], 0), ([40, 0, 1], _lib.Q8_ERR_KV_FULL), ([0, 0, 64], _lib.Q8_ERR_KV_FULL),
                    ([0, 2 ** 31 - 1, 0], _lib.Q8_ERR_KV_FULL), ([17, 0, 0], 0), ([0, 15, 1], _lib.Q8_ERR_KV_FULL),
                    ([0, 15, 0], 0)):
        src, dst, status = ops.kv_reserve(table, ctx, refs, 16, i32(n, cuda))
        _, _, want = h.reserve(n)
        assert status.tolist() == want and want[0] == code
        h.check(table, ctx, refs)


def test_shared_page_is_copied_but_for_its_last_owner(cuda):
    h = Host(4, 4, 12, 16)
    table, ctx, refs = h.cuda(cuda)
    for n in ([20, 0, 0, 0],):
        ops.kv_reserve(table, ctx, refs, 16, i32(n, cuda))
        h.reserve(n)
    pairs = np.array([0, 0, 0]), np.array([1, 2, 3])
    ops.kv_fork(table, ctx, refs, 16, *(i32(x, cuda) for x in pairs))
    h.fork(*pairs)
    # two of four sharers write: both copy; then the other two: the first keeps the page
    for n, moved in (([0, 1, 0, 1], 2), ([3, 0, 5, 0], 1), ([1, 1, 1, 1], 0)):
        src, dst, status = ops.kv_reserve(table, ctx, refs, 16, i32(n, cuda))
        a, b, c = h.reserve(n)
        assert src.tolist() == list(a) and dst.tolist() == list(b) and status.tolist() == c
        assert sum(x >= 0 for x in a) == moved
        h.check(table, ctx, refs)


def test_many_sequences_and_pages(cuda):
    rng = np.random.default_rng(3)
    S, width, pages, page = 4099, 6, 40000, 16
    h = Host(S, width, pages, page)
    table, ctx, refs = h.cuda(cuda)
    n = rng.integers(0, 60, S)
    ops.kv_reserve(table, ctx, refs, page, i32(n, cuda))
    h.reserve(n)
    src, dst = np.arange(0, 2000), np.arange(2000, 4000)
    ops.kv_fork(table, ctx, refs, page, i32(src, cuda), i32(dst, cuda))
    h.fork(src, dst)
    h.check(table, ctx, refs)
    one = np.ones(S, np.int64)
    got = ops.kv_reserve(table, ctx, refs, page, i32(one, cuda))
    want = h.reserve(one)
    assert all(g.tolist() == list(w) for g, w in zip(got, want))
    cut = rng.integers(-1, 60, S)
    ops.kv_truncate(table, ctx, refs, page, i32(cut, cuda))
    h.truncate(cut)
    src, dst = ops.kv_compact(table, refs)
    a, b = h.compact()
    assert src.tolist() == a and dst.tolist() == b
    h.check(table, ctx, refs)


@pytest.mark.parametrize("n,pages", [(1, 2), (40, 130), (700, 3000)])
def test_copy_pages(cuda, n, pages):
    rng = np.random.default_rng(n)
    pools = [torch.randn((pages, 2, 16, 64), device=cuda),
             torch.randint(-128, 128, (pages, 2, 48, 64), device=cuda, dtype=torch.int8),
             torch.randn((pages, 3), device=cuda),  # 12 bytes a page
             torch.randint(-128, 128, (pages * 7 + 1,), device=cuda, dtype=torch.int8)[1:].view(pages, 7)]
    both = rng.permutation(pages)[:2 * (min(n, pages // 2))]
    src, dst = both[:len(both) // 2].copy(), both[len(both) // 2:].copy()
    src[len(src) // 3] = src[0]  # one source twice
    want = [p.clone() for p in pools]
    for w in want:
        w[torch.from_numpy(dst).to(cuda)] = w[torch.from_numpy(src).to(cuda)]
    ops.kv_copy_pages(pools, i32(src, cuda), i32(dst, cuda))
    for p, w in zip(pools, want):
        assert torch.equal(p.view(torch.uint8), w.view(torch.uint8))


def test_copy_pages_leaves_out_what_depends_on_order(cuda):
    x = torch.arange(12, device=cuda, dtype=torch.float32)[:, None].repeat(1, 40)
    #       ok  gone gone  chain  same dst twice  itself  ok
    src = [0, -1, 3, 4, 5, 2, 7, 11, 0]
    dst = [1, 2, 12, 5, 6, 8, 8, 11, 9]
    ops.kv_copy_pages([x], i32(src, cuda), i32(dst, cuda))
    assert x[:, 0].tolist() == [0, 0, 2, 3, 4, 5, 5, 7, 8, 0, 10, 11]


def test_copy_pages_past_the_bitmap_window(cuda):
    pages = 2 ** 18 + 700
    x = torch.arange(pages, device=cuda, dtype=torch.int32)[:, None].repeat(1, 4)
    src = [5, 2 ** 18 + 3, 2 ** 18 - 1, 2 ** 18 + 600, 9]
    dst = [2 ** 18 + 4, 6, 2 ** 18, 2 ** 18 + 601, 9 + 2 ** 18]
    ops.kv_copy_pages([x], i32(src + [1, 2], cuda), i32(dst + [2 ** 18 + 9, 2 ** 18 + 10], cuda))
    assert x[dst[:4], 0].tolist() == src[:4]
    assert x[2 ** 18 + 9, 0] == 2 ** 18 + 9 and x[2 ** 18 + 10, 0] == 2  # two pairs wanted the former


@pytest.mark.parametrize("pages", [65537, 100000, 131072, 2 ** 18])
def test_copy_pages_bitmap_sizes(cuda, pages):
    x = torch.arange(pages, device=cuda, dtype=torch.int32)[:, None].repeat(1, 4)
    src, dst = [pages - 1, 3, 0], [4, pages - 2, pages // 2]
    ops.kv_copy_pages([x], i32(src, cuda), i32(dst, cuda))
    assert x[dst, 0].tolist() == src


def test_many_pools_and_refusals(cuda):
    pools = [torch.randn((9, 8), device=cuda) for _ in range(130)]
    ops.kv_copy_pages(pools, i32([3], cuda), i32([4], cuda))
    assert all(torch.equal(p[3], p[4]) for p in pools)
    t, c, r = i32([[0]], cuda), i32([1], cuda), i32([1, 0], cuda)
    with pytest.raises(ValueError):
        ops.kv_copy_pages([pools[0], pools[1][:8]], i32([3], cuda), i32([4], cuda))
    with pytest.raises(ValueError):
        ops.kv_copy_pages([pools[0].t()], i32([3], cuda), i32([4], cuda))
    with pytest.raises(ValueError):
        ops.kv_fork(t, c, r, 16, i32([0, 0], cuda), i32([0], cuda))
    with pytest.raises(ValueError):
        ops.kv_reserve(t, c, r, 16, i32([1, 1], cuda))
    with pytest.raises(_lib.Q8Error):
        ops.kv_truncate(t, c, r, 0, c)
    with pytest.raises(ValueError):
        ops.kv_truncate(t.long(), c, r, 16, c)


def test_replayed_from_a_graph(cuda):
    """A captured step (reserve, copy) replayed: the state moves on each time."""
    page = 16
    h = Host(2, 6, 12, page)
    table, ctx, refs = h.cuda(cuda)
    pool = torch.randn((12, 8), device=cuda)
    n = i32([9, 5], cuda)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        src, dst, status = ops.kv_reserve(table, ctx, refs, page, n)
        ops.kv_copy_pages([pool], src, dst)
    for _ in range(4):
        g.replay()
        torch.cuda.synchronize()
        a, b, c = h.reserve([9, 5])
        assert status.tolist() == c and src.tolist() == list(a)
        h.check(table, ctx, refs)
