"""How the Python entries of the paged-cache serving operators make their calls: what they hand to
the library stays alive until the call has returned."""
import gc
import os
import re
import textwrap
import threading
import types
import weakref

import numpy as np
import pytest
import torch

from lama32_mojo_b200 import _lib, ops


def test_attention_scratch_lives_through_the_call(monkeypatch):
    """ctypes lets other threads run during the call: a scratch that is free by then may be theirs."""
    made, seen, empty = [], [], torch.empty

    def tracked(*a, **kw):
        t = empty(*a, **kw)
        made.append((weakref.ref(t), t.data_ptr()))
        return t

    def call(fn, dev, *args):
        gc.collect()
        seen.append([r() is not None and at in args for r, at in made])

    pages = types.SimpleNamespace(head_dim=64, n_kv=1, page=64, _ref=0)
    monkeypatch.setattr(ops, "_packed", lambda *a: (1, 4, 0))
    monkeypatch.setattr(ops, "_kv8_scratch", lambda *a: 256)
    monkeypatch.setattr(ops, "_rows_of", lambda t, *a: (t.shape[0], 64))
    monkeypatch.setattr(ops, "_call", call)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    q, i = torch.zeros((1, 64)), torch.zeros(2, dtype=torch.int32)
    monkeypatch.setattr(torch, "empty", tracked)
    ops.kv8_attention(q, i, i, 1, pages, i)
    assert seen == [[True]]


@pytest.mark.gpu
def test_attention_from_two_threads_on_one_stream(cuda):
    """Two host threads on the default stream, each with calls that need a scratch and tensors of
    its own in between: the bits of calls made alone."""
    from test_gpu_kv8 import i32, make_pages, make_table, starts
    kv, G, hd, page = 4, 4, 128, 16
    work = []
    for seed, ns, ctx, width in ((1, [1] * 40, list(range(1, 1600, 40)), 300), (2, [300, 5, 200], [900, 70, 200], 57)):
        total = int(sum(-(-c // page) for c in ctx))
        pages = make_pages(cuda, total, kv, page, hd, seed)
        table = i32(make_table(ctx, page, total, seed, width=max(width, -(-max(ctx) // page))), cuda)
        q = torch.randn((sum(ns), kv * G * hd), device=cuda)
        args = q, i32(starts(np.array(ns)), cuda), i32(ctx, cuda), kv * G, pages, table
        work.append((args, ops.kv8_attention(*args)))
    torch.cuda.synchronize()
    wrong, go = [], threading.Barrier(2)

    def run(k):
        args, want = work[k]
        go.wait()
        for _ in range(60):
            got = ops.kv8_attention(*args)
            other = [torch.full((1 << s,), float(k), device=cuda) for s in range(10, 22, 2)]
            if not torch.equal(got, want):
                wrong.append(k)
            del other

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_a_refused_launch_is_not_blamed_on_the_next_call(cuda):
    """More blocks than a grid has (2^33, which an int counts as 0: nothing can run): the call says
    so, and neither torch nor the library's next call sees its error."""
    L, x = _lib.lib(), torch.randn((1, 256), device=cuda)
    pos, inv = torch.zeros(1, dtype=torch.int32, device=cuda), torch.ones(32, device=cuda)
    at = x.data_ptr()
    status = L.q8op_rope_kv_append(at, 256, 2 ** 35, pos.data_ptr(), None, 1, 1, 64, inv.data_ptr(), None, None, 1e-6,
                                   None, None, 0, None, 0, None)
    assert status == _lib.Q8_ERR_CUDA and "k_rope_kv" in _lib.last_error()
    assert int(ops.argmax(x)) == int(x.argmax())
    assert float(torch.zeros(3, device=cuda).sum()) == 0.0


@pytest.mark.gpu
def test_rope_refuses_what_its_kernel_would_misread(cuda):
    """Rows, positions and frequencies of other types or lengths reach behind their tensors."""
    nh, kv, hd, T = 4, 2, 64, 3
    w = (nh + 2 * kv) * hd
    qkv, pos = torch.randn((T, w), device=cuda), torch.arange(T, device=cuda, dtype=torch.int32)
    inv, norm = torch.rand(hd // 2, device=cuda), torch.ones(hd, device=cuda, dtype=torch.bfloat16)
    was = qkv.clone()
    for bad in (lambda: ops.rope(qkv.bfloat16(), pos, nh, kv, hd, inv), lambda: ops.rope(qkv[:, 1:], pos, nh, kv, hd, inv),
                lambda: ops.rope(qkv.t(), pos, nh, kv, hd, inv), lambda: ops.rope(qkv, pos.long(), nh, kv, hd, inv),
                lambda: ops.rope(qkv, pos[:2], nh, kv, hd, inv), lambda: ops.rope(qkv, pos, nh, kv, hd, inv[:-1]),
                lambda: ops.rope(qkv, pos, nh, kv, hd, inv.double()), lambda: ops.rope(qkv, pos, nh, kv, hd, inv, norm.float()),
                lambda: ops.rope(qkv, pos, nh, kv, hd, inv, norm, norm[:32]), lambda: ops.rope(qkv, pos.cpu(), nh, kv, hd, inv)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.Q8Error):
        ops.rope(qkv, pos, 8, 4, 32, inv[:16])
    assert torch.equal(qkv, was)
    ops.rope(qkv[:0], pos[:0], nh, kv, hd, inv)  # no rows: nothing to do
    ops.rope(qkv, pos, nh, kv, hd, inv, norm, norm)
    assert not torch.equal(qkv, was) and torch.equal(qkv[:, (nh + kv) * hd:], was[:, (nh + kv) * hd:])


@pytest.mark.gpu
def test_pages_keep_the_tensors_that_they_were_made_of(cuda):
    """The calls read the addresses of the first tensors: a replaced one would be read after it is free."""
    pages = ops.KV8Pages.empty(2, 1, 16, 64, cuda)
    k = pages.k
    for name in ("k", "v", "k_scale", "v_scale", "num_pages", "page"):
        with pytest.raises(AttributeError):
            setattr(pages, name, getattr(pages, name))
    pages.k[1] = 3
    assert pages.k is k and pages.tensors()[0] is k and int(k.sum()) == 3 * 16 * 64


def documented_step():
    """The Python blocks of the integration notes on the serving operators: set-up, one step."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")
    with open(path) as f:
        text = f.read().split("## Serving operators on a paged cache")[1].split("\n## ")[0]
    return [textwrap.dedent(b) for b in re.findall(r"```python\n(.*?)```", text, re.S)]


@pytest.mark.gpu
def test_the_documented_step_and_a_full_pool(cuda):
    """The step as the integration notes show it: drafts verified, refused positions given back.  Where the
    pool is full it leaves lengths, pages and their content as they are."""
    setup, step = documented_step()
    S, V, n = 2, 50, 3
    env = dict(torch=torch, num_pages=3, n_kv=1, head_dim=64, n_heads=2, layers=2, temp=0.0)
    env["table"] = torch.full((S, 4), -1, dtype=torch.int32, device=cuda)
    env["ctx"], env["refs"] = (torch.zeros(k, dtype=torch.int32, device=cuda) for k in (S, 3))
    exec(setup, env)
    g = torch.Generator(device=cuda).manual_seed(0)
    env["inv_freq"] = torch.rand(32, generator=g, device=cuda)
    used = 0
    for _ in range(60):
        qkv = torch.randn((S * n, 4 * 64), generator=g, device=cuda)
        env.update(qkv=qkv, q=qkv[:, :128], k=qkv[:, 128:192], v=qkv[:, 192:], n_new=env["ctx"] * 0 + n,
                   pos=(env["ctx"][:, None] + torch.arange(n, device=cuda)).flatten().int().contiguous(),
                   seq_start=torch.arange(0, S * n + 1, n, dtype=torch.int32, device=cuda), q_drafts=None,
                   logits=torch.randn((S * n, V), generator=g, device=cuda),
                   u=torch.rand(S * n, generator=g, device=cuda))
        ids = env["logits"].argmax(-1).int().roll(1)  # the first draft of each is the target's choice, the second is not
        ids[2::n] = (ids[2::n] + 1) % V
        env["ids"] = ids
        was = [t.clone() for t in (env["ctx"], env["refs"], env["table"])] + \
            [t.clone() for p in env["pages"] for t in p.tensors()]
        exec(step, env)
        now = [env["ctx"], env["refs"], env["table"]] + [t for p in env["pages"] for t in p.tensors()]
        if int(env["status"][0]) != 0:
            assert all(torch.equal(a, b) for a, b in zip(was, now))
            break
        assert env["n_accepted"].tolist() == [1, 1] and (env["ctx"] - was[0]).tolist() == [2, 2]
        used += 1
    assert int(env["status"][0]) == _lib.Q8_ERR_KV_FULL and used > 20


@pytest.mark.gpu
@pytest.mark.parametrize("kv,hd", [(2, 64), (8, 128), (3, 128)])
def test_read_leaves_rows_behind_the_last_sequence(cuda, kv, hd):
    from test_gpu_kv8 import i32, make_pages
    page, ns, ctx, tail = 32, [3, 0, 9], [40, 5, 9], 7
    pages = make_pages(cuda, 6, kv, page, hd)
    args = i32([0, 3, 3, 12], cuda), i32(ctx, cuda), pages, i32([[0, 1], [2, -1], [3, 4]], cuda)
    want = ops.kv8_read(*args, 12)
    T = 12 + tail
    k, v = (torch.full((T, kv, hd), 7.0, device=cuda) for _ in range(2))
    L, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    _lib.check(L.q8op_kv8_read(pages._ref, args[0].data_ptr(), args[1].data_ptr(), 3, args[3].data_ptr(), 2,
                               k.data_ptr(), v.data_ptr(), T, stream))
    for got, w in zip((k, v), want):
        assert torch.equal(got[:12], w) and bool((got[12:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [50, 20000])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_leaves_rows_behind_the_last_sequence(cuda, n, certain):
    """Tokens from seq_start[S] on keep what they were, and a sequence without rows touches none."""
    from test_gpu_kv8 import i32
    S, T, used = 4, 15, 9
    g = torch.Generator(device=cuda).manual_seed(n)
    p = torch.rand((T, n), generator=g, device=cuda)
    q = None if certain else p[:used - 3].clone()
    ids = p.argmax(-1).int().roll(1)
    starts, u = i32([0, 4, 4, 5, 9], cuda), torch.rand(T, generator=g, device=cuda)
    a, t = ops.verify(p[:used], q, ids[:used], starts, u[:used])
    taken = torch.full((S + 2,), -9, dtype=torch.int32, device=cuda)
    tokens = torch.full((T,), -9, dtype=torch.int32, device=cuda)
    _lib.check(_lib.lib().q8op_verify(p.data_ptr(), n, None if certain else q.data_ptr(), n, 0 if certain else used - 3,
                                      ids.data_ptr(), starts.data_ptr(), T, S, n, u.data_ptr(), taken.data_ptr(),
                                      tokens.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(taken[:S], a) and taken[S:].tolist() == [-9, -9]
    assert torch.equal(tokens[:used], t) and tokens[used:].tolist() == [-9] * (T - used)


@pytest.mark.gpu
def test_a_refused_draft_leaves_its_scale(cuda):
    """As documented: giving positions back does not shrink their block's scale, a new block starts over."""
    from test_gpu_kv8 import i32
    pages = ops.KV8Pages.empty(2, 1, 16, 64, cuda)
    table, refs, ctx, start = i32([[0, 1]], cuda), i32([1, 1], cuda), i32([3], cuda), i32([0, 3], cuda)
    x = torch.ones((3, 64), device=cuda)
    x[2] = 100.0
    ops.kv8_append(x, x, start, ctx, pages, table)
    ops.kv_truncate(table, ctx, refs, 16, i32([2], cuda))
    ctx += 15
    ops.kv8_append(x[:1].expand(15, 64).contiguous(), x[:1].expand(15, 64).contiguous(), i32([0, 15], cuda), ctx, pages,
                   i32([[0, 1]], cuda))
    s = pages.k_scale.flatten()
    assert float(s[0]) == float(np.float32(100) / np.float32(127)) and float(s[1]) == float(np.float32(1) / np.float32(127))
    assert pages.k[0, 0].unique().tolist() == [1]  # 1 / (100 / 127) rounds to 1
