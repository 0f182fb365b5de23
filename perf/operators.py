"""Workloads of the serving operators around the paged KV cache: the 8-bit
cache (append, read back, attention over it), the page tables (truncate, fork,
reserve, copy, compact) and speculative decoding (probabilities of logits,
verification of drafted tokens).

``listed()`` names the cases that are timed and ``draw(rng)`` makes more of the
same ranges.  ``run(state)`` is one pass: with ``own`` the calls a user makes
of ``lama32_mojo_b200.ops``, without it the same operators as elementary torch
operations.  ``exact(case, seed)`` computes them once more, in 64 bits, one
sequence at a time.

The operators in short (positions of a sequence are 0 .. ctx - 1; the rows
seq_start[b] .. seq_start[b + 1] - 1 of a call belong to sequence b and are
its last positions; a negative table entry is a page that is not there):

* 8-bit cache: 16 consecutive tokens of one kv head share a scale s.  Appending
  raises s to max|x| / 127 of the new rows where that is larger (a block whose
  first token is new starts from 0), codes that stay become round(c s / s'),
  new ones round(x / s'), ties to even, within +-127.
* attention: softmax(q.k / sqrt(hd)) v over the visible positions.
* pages: refs[p] counts the table entries that hold page p; 0 is free.  New
  pages are the lowest free ones, in the order of (sequence, position).
* probabilities: w = exp((l - max) / temp) for l >= max - 16, else 0; w / sum.
* verification: draft x behind row r is kept while u[r] q(x) < p(x); then one
  token from max(p - q, 0) of the first refused row, or from p of the last row.
"""
import math
import random

import torch

own = False

BLOCK = 16  # tokens of one kv head that share a scale
F32, BF16, F16 = "f32", "bf16", "f16"
DTYPES = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}
# (q heads, kv heads, head dim) of the model presets
HEADS = [(32, 8, 128), (24, 8, 128), (32, 8, 64), (16, 8, 128), (8, 2, 64), (4, 2, 128), (8, 8, 64)]
VOCABS = [128256, 151936, 50003, 2048, 1000]


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of a serving batch: a token for each of 64 sequences
        dict(name="append_decode", kind="append", seqs=64, tokens=1, ragged=False, ctx=4096, kv=8, hd=128,
             page=64, dtype=F32),
        # prompts of several thousand tokens, packed, as a prefill writes them
        dict(name="append_prompt", kind="append", seqs=5, tokens=4000, ragged=True, ctx=6000, kv=8, hd=128,
             page=64, dtype=BF16),
        # the smallest call: one user's decode step at a short context
        dict(name="attend_one", kind="attend", seqs=1, tokens=1, ragged=False, ctx=523, heads=32, kv=8, hd=64,
             page=64, dtype=F32),
        # a decode step of a full serving batch, lengths all over the range
        dict(name="attend_batch", kind="attend", seqs=64, tokens=1, ragged=False, ctx=8192, heads=32, kv=8,
             hd=128, page=64, dtype=F32),
        # drafted tokens of 16 sequences checked in one pass of the target model
        dict(name="attend_drafts", kind="attend", seqs=16, tokens=5, ragged=False, ctx=4500, heads=24, kv=8,
             hd=128, page=64, dtype=BF16),
        # two chunks of long prompts against what is cached already
        dict(name="attend_chunk", kind="attend", seqs=2, tokens=1024, ragged=False, ctx=8000, heads=32, kv=8,
             hd=128, page=64, dtype=F32),
        # beam search: three more beams of each of 16 prompts, one step
        dict(name="pages_fork", kind="fork", groups=16, beams=4, ctx=1000, kv=8, hd=128, page=64),
        # a fragmented pool is made dense after sequences have left
        dict(name="pages_compact", kind="compact", pages=3000, seqs=96, ctx=2048, kv=8, hd=128, page=64),
        # the next token's distribution for one user
        dict(name="probs_one", kind="probs", rows=1, vocab=128256, temp=0.8),
        # distributions of all rows of a batch of drafts
        dict(name="probs_batch", kind="probs", rows=320, vocab=151936, temp=1.0),
        # one user's drafts
        dict(name="verify_one", kind="verify", seqs=1, drafts=4, ragged=False, vocab=128256, draft_probs=True),
        # a serving batch with drafts of different lengths
        dict(name="verify_batch", kind="verify", seqs=64, drafts=5, ragged=True, vocab=151936, draft_probs=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "fork", "compact", "probs", "verify"])
    page = rng.choice([16, 32, 64, 64, 64, 128])
    heads, kv, hd = rng.choice(HEADS)
    if kind == "append":
        tokens = _log(rng, 1, 6000)
        return dict(kind=kind, seqs=_log(rng, 1, max(1, min(200, 20000 // tokens))), tokens=tokens,
                    ragged=rng.random() < 0.5, ctx=tokens + _log(rng, 1, 4000), kv=kv, hd=hd, page=page,
                    dtype=rng.choice([F32, BF16, F16]))
    if kind == "attend":
        tokens = rng.choice([1, 1, _log(rng, 2, 12), _log(rng, 13, 1000)])
        ctx = tokens + _log(rng, 1, 60000)
        most = 4e8 / (ctx * kv * hd * 2), 1e11 / (4.0 * tokens * ctx * heads * hd)  # 0.4 GB of codes, 0.1 TFLOP
        return dict(kind=kind, seqs=_log(rng, 1, int(max(1, min(128, *most)))), tokens=tokens,
                    ragged=rng.random() < 0.3, ctx=ctx, heads=heads, kv=kv, hd=hd, page=page,
                    dtype=rng.choice([F32, F32, BF16, F16]))
    if kind == "fork":
        return dict(kind=kind, groups=_log(rng, 1, 40), beams=rng.randint(2, 8), ctx=_log(rng, 1, 4000), kv=kv,
                    hd=hd, page=page)
    if kind == "compact":
        return dict(kind=kind, pages=_log(rng, 20, 3000), seqs=_log(rng, 1, 120), ctx=_log(rng, 16, 2048), kv=kv,
                    hd=hd, page=min(page, 64))
    vocab = rng.choice(VOCABS)
    if kind == "probs":
        return dict(kind=kind, rows=_log(rng, 1, 200), vocab=vocab, temp=rng.choice([0.0, 0.6, 1.0, 1.7]))
    return dict(kind=kind, seqs=_log(rng, 1, 48), drafts=_log(rng, 1, 8), ragged=rng.random() < 0.5, vocab=vocab,
                draft_probs=rng.random() < 0.8)


def _lengths(case):
    """Per sequence: (positions behind the call, rows of the call).  They follow from the case alone."""
    rng = random.Random(case["seqs"] * 1000003 + case["ctx"] * 31 + case["tokens"])
    got = []
    for b in range(case["seqs"]):
        n = case["tokens"] if b == 0 or not case["ragged"] else rng.randint(0, case["tokens"])
        got.append((case["ctx"] if b == 0 else rng.randint(max(n, 1), case["ctx"]), n))
    return got


def work(case):
    kind = case["kind"]
    if kind in ("append", "attend"):
        lens, kv, hd = _lengths(case), case["kv"], case["hd"]
        size = 4 if case["dtype"] == F32 else 2
        if kind == "append":  # rows in, codes out, and the read back: codes in, rows out
            back = sum(n + (c - n) % BLOCK for c, n in lens if n)
            return {"bytes": float(sum(n for _, n in lens) * 2 * kv * hd * (size + 1) + back * 2 * kv * hd * (1 + 4)),
                    "flops": float(sum(n for _, n in lens) * 2 * kv * hd * 3)}
        row = case["heads"] * hd
        pairs = sum(sum(range(c - n + 1, c + 1)) if n < 64 else n * (2 * c - n + 1) // 2 for c, n in lens)
        return {"bytes": float(sum(c for c, n in lens if n) * kv * 2 * (hd + 4 / BLOCK)
                               + sum(n for _, n in lens) * 2 * row * size),
                "flops": 4.0 * pairs * row}
    if kind == "fork":
        page = case["page"]
        per = -(-(case["ctx"] + 1) // page)
        moved = case["groups"] * (case["beams"] - 1) * (case["ctx"] % page != 0)
        return {"bytes": float(moved * 2 * 2 * case["kv"] * page * case["hd"] * 4
                               + case["groups"] * case["beams"] * per * 4 * 4), "flops": 0.0}
    if kind == "compact":
        plan = _compact_plan(case, 0)
        refs = [0] * case["pages"]
        for row in plan:
            for p in row:
                refs[p] += 1
        used = sum(r > 0 for r in refs)
        moved = sum(r > 0 for r in refs[used:])
        return {"bytes": float(moved * 2 * 2 * case["kv"] * case["page"] * case["hd"] * 4 + case["pages"] * 8
                               + sum(map(len, plan)) * 8), "flops": 0.0}
    if kind == "probs":
        n = float(case["rows"] * case["vocab"])
        return {"bytes": n * 8, "flops": n * 4}
    rows = case["seqs"] * case["vocab"]
    return {"bytes": float(rows * 4 * (2 if case["draft_probs"] else 1)), "flops": float(rows * 3)}


# ------------------------------------------------------------------ their inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    got = [0]
    for n in counts:
        got.append(got[-1] + n)
    return _ints(got)


def _codes(shape, g):
    return torch.randn(shape, generator=g, device="cuda").mul_(36).round_().clamp_(-127, 127).to(torch.int8)


def _cache(case, lens, g):
    """8-bit pages with random content and a table of shuffled pages."""
    page, kv, hd = case["page"], case["kv"], case["hd"]
    per = [-(-c // page) for c, _ in lens]
    total = sum(per) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(per)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (total, kv, page, hd)
    scales = (total, kv, page // BLOCK)
    return {"k": _codes(shape, g), "v": _codes(shape, g),
            "k_scale": torch.rand(scales, generator=g, device="cuda").mul_(0.02).add_(0.01),
            "v_scale": torch.rand(scales, generator=g, device="cuda").mul_(0.02).add_(0.01)}, table


def _compact_plan(case, seed):
    """Pages of each sequence: random lengths, scattered over the pool, at most 70 % of it in use."""
    rng = random.Random(case["pages"] * 7919 + case["seqs"])
    sizes = [rng.randint(1, -(-case["ctx"] // case["page"])) for _ in range(case["seqs"])]
    while sum(sizes) > case["pages"] * 0.7 and len(sizes) > 1:
        sizes.pop()
    sizes[0] = min(sizes[0], max(1, case["pages"] // 2))
    rng = random.Random(seed * 104729 + case["pages"])
    order = list(range(case["pages"]))
    rng.shuffle(order)
    plan, at = [], 0
    for n in sizes:
        plan.append(order[at:at + n])
        at += n
    for row in plan[1:]:  # some share a prefix, as forked sequences do
        if rng.random() < 0.25:
            k = rng.randint(0, min(len(row), len(plan[0])))
            row[:k] = plan[0][:k]
    return plan


def _pools(pages, case, g):
    shape = (pages, case["kv"], case["page"], case["hd"])
    return [torch.randn(shape, generator=g, device="cuda"), torch.randn(shape, generator=g, device="cuda")]


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    st = {"case": case, "kind": kind}
    if kind in ("append", "attend"):
        lens = _lengths(case)
        total = sum(n for _, n in lens)
        cache, st["table"] = _cache(case, lens, g)
        st["ctx"] = _ints([c for c, _ in lens])
        st["seq_start"] = _starts([n for _, n in lens])
        st["most"] = max(n for _, n in lens)
        if kind == "append":
            # k and v are columns of the rows that the q|k|v product wrote
            heads = 4 * case["kv"]
            width = (heads + 2 * case["kv"]) * case["hd"]
            rows = torch.randn((total, width), generator=g, device="cuda")
            rows *= torch.rand((total, 1), generator=g, device="cuda").add_(0.5)
            rows = rows.to(DTYPES[case["dtype"]])
            at = heads * case["hd"], (heads + case["kv"]) * case["hd"]
            st["new_k"], st["new_v"] = rows[:, at[0]:at[1]], rows[:, at[1]:]
            back = [n + (c - n) % BLOCK if n else 0 for c, n in lens]  # every token of the blocks that changed
            st["back_start"], st["back_rows"] = _starts(back), sum(back)
        else:
            st["q"] = torch.randn((total, case["heads"] * case["hd"]), generator=g, device="cuda").mul_(2).to(
                DTYPES[case["dtype"]])
        if own:
            from lama32_mojo_b200 import ops
            st["pages"] = ops.KV8Pages(**cache)
        else:
            st["pages"] = cache
    elif kind == "fork":
        page, beams, groups = case["page"], case["beams"], case["groups"]
        per = -(-(case["ctx"] + 1) // page)
        seqs = groups * beams
        pages = groups * per + seqs * 2 + 5
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        st["table"] = torch.full((seqs, per + 1), -1, dtype=torch.int32, device="cuda")
        held = -(-case["ctx"] // page)
        st["table"][::beams, :held] = order[:groups * held].view(groups, held)
        st["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
        st["refs"][order[:groups * held].long()] = 1
        st["ctx"] = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        st["ctx"][::beams] = case["ctx"]
        st["keep"] = st["ctx"].clone()
        st["one"] = torch.ones(seqs, dtype=torch.int32, device="cuda")
        child = [b for b in range(seqs) if b % beams]
        st["src"], st["dst"] = _ints([b - b % beams for b in child]), _ints(child)
        st["pools"] = _pools(pages, case, g)
    elif kind == "compact":
        plan = _compact_plan(case, seed)
        table = torch.full((len(plan), max(map(len, plan)) + 1), -1, dtype=torch.int32)
        refs = torch.zeros(case["pages"], dtype=torch.int32)
        for b, row in enumerate(plan):
            table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
            refs.index_add_(0, torch.tensor(row), torch.ones(len(row), dtype=torch.int32))
        st["table0"], st["refs0"] = table.cuda(), refs.cuda()
        st["table"], st["refs"] = torch.empty_like(st["table0"]), torch.empty_like(st["refs0"])
        st["pools"] = _pools(case["pages"], case, g)
    elif kind == "probs":
        st["logits"] = torch.randn((case["rows"], case["vocab"]), generator=g, device="cuda").mul_(2.5)
    else:
        lens = _drafts(case)
        rows = sum(n + 1 for n in lens)
        st["seq_start"] = _starts([n + 1 for n in lens])
        target = torch.randn((rows, case["vocab"]), generator=g, device="cuda").mul_(3)
        at = torch.tensor([r for r in range(rows) if r not in _last_rows(lens)], device="cuda", dtype=torch.long)
        near = target[at] + torch.randn((len(at), case["vocab"]), generator=g, device="cuda").mul_(0.7)
        st["p"], near = target.softmax(-1), near.softmax(-1)
        # the draft model's picks; row r's draft is the token fed at row r + 1
        r = torch.rand((len(at), 1), generator=g, device="cuda", dtype=torch.float64)
        picks = torch.searchsorted(near.double().cumsum(-1), r).squeeze(-1).clamp_(max=case["vocab"] - 1)
        st["ids"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        st["ids"][at + 1] = picks.to(torch.int32)
        st["q"] = near if case["draft_probs"] else None
        st["u"] = torch.rand(rows, generator=g, device="cuda")
    return st


def _drafts(case):
    rng = random.Random(case["seqs"] * 101 + case["drafts"])
    return [case["drafts"] if b == 0 or not case["ragged"] else rng.randint(0, case["drafts"])
            for b in range(case["seqs"])]


def _last_rows(lens):
    got, at = set(), -1
    for n in lens:
        at += n + 1
        got.add(at)
    return got


# ------------------------------------------------------------------ one pass
def run(st):
    kind = st["kind"]
    if own:
        from lama32_mojo_b200 import ops
        page = st["case"].get("page")
        if kind == "append":
            ops.kv8_append(st["new_k"], st["new_v"], st["seq_start"], st["ctx"], st["pages"], st["table"])
            return ops.kv8_read(st["back_start"], st["ctx"], st["pages"], st["table"], st["back_rows"])
        if kind == "attend":
            return ops.kv8_attention(st["q"], st["seq_start"], st["ctx"], st["case"]["heads"], st["pages"],
                                     st["table"])
        if kind == "fork":
            ops.kv_truncate(st["table"], st["ctx"], st["refs"], page, st["keep"])
            ops.kv_fork(st["table"], st["ctx"], st["refs"], page, st["src"], st["dst"])
            src, dst, status = ops.kv_reserve(st["table"], st["ctx"], st["refs"], page, st["one"])
            ops.kv_copy_pages(st["pools"], src, dst)
            return st["table"], st["ctx"], st["refs"], src, dst, status, st["pools"]
        if kind == "compact":
            st["table"].copy_(st["table0"])
            st["refs"].copy_(st["refs0"])
            src, dst = ops.kv_compact(st["table"], st["refs"])
            ops.kv_copy_pages(st["pools"], src, dst)
            return st["table"], st["refs"], src, dst, st["pools"]
        if kind == "probs":
            return ops.probs(st["logits"], st["case"]["temp"])
        return ops.verify(st["p"], st["q"], st["ids"], st["seq_start"], st["u"])
    if kind == "append":
        _plain_append(st["new_k"], st["pages"]["k"], st["pages"]["k_scale"], st)
        _plain_append(st["new_v"], st["pages"]["v"], st["pages"]["v_scale"], st)
        return _plain_read(st, "k"), _plain_read(st, "v")
    if kind == "attend":
        return _plain_attend(st)
    if kind == "fork":
        page = st["case"]["page"]
        _plain_truncate(st["table"], st["ctx"], st["refs"], page, st["keep"])
        _plain_fork(st["table"], st["ctx"], st["refs"], page, st["src"], st["dst"])
        src, dst, status = _plain_reserve(st["table"], st["ctx"], st["refs"], page, st["one"])
        _plain_copy(st["pools"], src, dst)
        return st["table"], st["ctx"], st["refs"], src, dst, status, st["pools"]
    if kind == "compact":
        st["table"].copy_(st["table0"])
        st["refs"].copy_(st["refs0"])
        src, dst = _plain_compact(st["table"], st["refs"])
        _plain_copy(st["pools"], src, dst)
        return st["table"], st["refs"], src, dst, st["pools"]
    if kind == "probs":
        return _plain_probs(st["logits"], st["case"]["temp"])
    return _plain_verify(st["p"], st["q"], st["ids"], st["seq_start"], st["u"])


# ------------------------------------------------------------------ plain forms: the 8-bit cache
def _places(starts, ctx, rows, table, page):
    """Of each row of a call: its page, and its position."""
    b = torch.repeat_interleave(torch.arange(ctx.numel(), device=ctx.device), starts.diff(), output_size=rows)
    pos = ctx[b] - starts[b + 1] + torch.arange(rows, device=ctx.device)
    return table[b, pos // page].long(), pos


def _plain_append(x, codes, scales, st):
    pages, kv, page, hd = codes.shape
    rows = x.shape[0]
    at, pos = _places(st["seq_start"], st["ctx"], rows, st["table"], page)
    per = page // BLOCK
    blk = at * per + (pos % page) // BLOCK  # scale block of each row, over the whole pool
    x = x.double().view(rows, kv, hd)
    high = torch.zeros((pages * per, kv), dtype=torch.float64, device=x.device)
    high.index_reduce_(0, blk, x.abs().amax(-1), "amax")
    first = torch.full((pages * per,), BLOCK, device=x.device)  # first new token of a block; BLOCK: none
    first.index_reduce_(0, blk, pos % BLOCK, "amin")
    old = scales.transpose(1, 2).reshape(pages * per, kv)
    base = torch.where((first > 0)[:, None], old, 0.0)
    new = torch.maximum(base, (high / 127.0).float())
    new = torch.where((first < BLOCK)[:, None], new, old)
    safe = torch.where(new > 0, new, 1.0).double()
    stay = torch.arange(BLOCK, device=x.device) < first[:, None]
    hit = torch.unique(blk)  # only the touched blocks are written
    view = codes.view(pages, kv, per, BLOCK, hd)
    c = view[hit // per, :, hit % per].double()
    c2 = (c * old[hit].double()[:, :, None, None] / safe[hit][:, :, None, None]).round().clamp(-127, 127)
    view[hit // per, :, hit % per] = torch.where(stay[hit][:, None, :, None], c2, c).to(torch.int8)
    scales.copy_(new.view(pages, per, kv).transpose(1, 2))
    s = safe[blk][:, :, None]
    codes[at, :, pos % page] = (x / s).round().clamp(-127, 127).to(torch.int8)


def _plain_read(st, name):
    codes, scales = st["pages"][name], st["pages"][name + "_scale"]
    page = codes.shape[2]
    at, pos = _places(st["back_start"], st["ctx"], st["back_rows"], st["table"], page)
    return codes[at, :, pos % page].float() * scales[at, :, pos % page // BLOCK][:, :, None]


def _plain_attend(st):
    case, q, table, ctx, starts = st["case"], st["q"], st["table"], st["ctx"], st["seq_start"]
    kv, hd, heads = case["kv"], case["hd"], case["heads"]
    seqs, width = table.shape
    most, rows = st["most"], q.shape[0]
    b = torch.repeat_interleave(torch.arange(seqs, device=q.device), starts.diff(), output_size=rows)
    i = torch.arange(rows, device=q.device) - starts[b]
    wide = torch.zeros((seqs, most, heads, hd), device=q.device)
    wide[b, i] = q.float().view(rows, heads, hd)
    wide = wide.view(seqs, most, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, hd)
    at = table.clamp(min=0).long()

    def rows_of(name):
        x = st["pages"][name][at].float().view(seqs, width, kv, -1, BLOCK, hd)
        x = x * st["pages"][name + "_scale"][at][:, :, :, :, None, None]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(seqs, kv, -1, hd)

    s = wide @ rows_of("k").transpose(-1, -2) * (1.0 / math.sqrt(hd))
    pos = ctx[:, None] - (starts[1:] - starts[:-1])[:, None] + torch.arange(most, device=q.device)
    seen = torch.arange(s.shape[-1], device=q.device) <= pos[..., None]  # [seqs, most, positions]
    s = s.view(seqs, kv, heads // kv, most, -1).masked_fill_(~seen[:, None, None], float("-inf"))
    s = torch.exp(s - s.amax(-1, keepdim=True))
    s = (s / s.sum(-1, keepdim=True)).nan_to_num_(0.0).view(seqs, kv, -1, s.shape[-1])
    o = (s @ rows_of("v")).view(seqs, kv, heads // kv, most, hd).permute(0, 3, 1, 2, 4)
    return o.reshape(seqs, most, heads * hd)[b, i].to(q.dtype)


# ------------------------------------------------------------------ plain forms: page tables
def _add_refs(refs, pages, valid, sign):
    refs.add_(torch.bincount(torch.where(valid, pages, -1).flatten() + 1, minlength=refs.numel() + 1)[1:]
              .to(torch.int32), alpha=sign)


def _plain_truncate(table, ctx, refs, page, keep):
    cut = torch.where(keep >= 0, torch.minimum(keep, ctx), ctx)
    col = torch.arange(table.shape[1], device=table.device)
    drop = (table >= 0) & (keep >= 0)[:, None] & (col >= ((cut + page - 1) // page)[:, None])
    _add_refs(refs, table, drop, -1)
    table.masked_fill_(drop, -1)
    ctx.copy_(cut)


def _plain_fork(table, ctx, refs, page, src, dst):
    new, lens = table.clone(), ctx.clone()
    row = table[src.long()]
    col = torch.arange(table.shape[1], device=table.device)
    row = torch.where(col < ((ctx[src.long()] + page - 1) // page)[:, None], row, -1)
    old = table[dst.long()]
    _add_refs(refs, old, old >= 0, -1)
    _add_refs(refs, row, row >= 0, 1)
    new[dst.long()] = row
    lens[dst.long()] = ctx[src.long()]
    table.copy_(new)
    ctx.copy_(lens)


def _plain_reserve(table, ctx, refs, page, n_new):
    seqs, width = table.shape
    s, col = torch.arange(seqs, device=table.device), torch.arange(width, device=table.device)
    n = n_new.clamp(min=0)
    first, last = ctx // page, (ctx + n - 1) // page
    want = (n > 0)[:, None] & (col >= first[:, None]) & (col <= last[:, None]) & (table < 0)
    # the page that the first new token shares: copied unless it is the caller's own, or the first of its last sharers
    edge = table[s, first.clamp(max=width - 1).long()]
    held = refs[edge.clamp(min=0).long()]
    cand = (n > 0) & (ctx % page != 0) & (first < width) & (edge >= 0) & (held > 1)
    same = cand[:, None] & cand[None, :] & (edge[:, None] == edge[None, :])
    keeps = cand & (same.sum(1) == held) & ((same & (s[None, :] < s[:, None])).sum(1) == 0)
    copies = cand & ~keeps
    want[s, first.clamp(max=width - 1).long()] |= copies
    rank = want.flatten().cumsum(0).view(seqs, width) - 1
    free = refs == 0
    order = torch.zeros(refs.numel() + 1, dtype=torch.int64, device=table.device)
    order[torch.where(free, free.cumsum(0) - 1, refs.numel())] = torch.arange(refs.numel(), device=table.device)
    needed, left = want.sum(), free.sum()
    fits = (needed <= left) & ~((n > 0) & (last >= width)).any()
    want &= fits
    copies &= fits
    page_of = order[rank.clamp(min=0, max=refs.numel() - 1)].to(torch.int32)
    src = torch.where(copies, edge, -1)
    _add_refs(refs, edge, copies, -1)
    _add_refs(refs, page_of, want, 1)
    table.copy_(torch.where(want, page_of, table))
    dst = torch.where(copies, table[s, first.clamp(max=width - 1).long()], -1)
    ctx.add_(torch.where(fits, n, 0))
    status = torch.stack([torch.where(fits, 0, 4), needed, left - torch.where(fits, needed, 0)]).to(torch.int32)
    return src.to(torch.int32), dst.to(torch.int32), status


def _plain_compact(table, refs):
    pages = refs.numel()
    at = torch.arange(pages, device=refs.device)
    used = refs > 0
    n = used.sum()
    out, into = used & (at >= n), ~used & (at < n)
    src = torch.full((pages // 2 + 1,), -1, dtype=torch.int32, device=refs.device)
    dst = src.clone()
    src[torch.where(out, out.cumsum(0) - 1, pages // 2)] = torch.where(out, at, -1).to(torch.int32)
    dst[torch.where(into, into.cumsum(0) - 1, pages // 2)] = torch.where(into, at, -1).to(torch.int32)
    src, dst = src[:pages // 2], dst[:pages // 2]
    move = torch.arange(pages + 1, device=refs.device, dtype=torch.int32)
    move[torch.where(src >= 0, src, pages).long()] = dst
    table.copy_(torch.where(table >= 0, move[table.clamp(min=0).long()], table))
    refs.copy_(torch.where(at < n, refs + torch.zeros_like(refs).index_add_(
        0, dst.clamp(min=0).long(), torch.where(src >= 0, refs[src.clamp(min=0).long()], 0)), 0))
    return src, dst


def _plain_copy(pools, src, dst):
    ok = (src >= 0) & (dst >= 0)
    a, b = src[ok].long(), dst[ok].long()
    pools[0][b] = pools[0][a]
    pools[1][b] = pools[1][a]


# ------------------------------------------------------------------ plain forms: speculative decoding
def _plain_probs(logits, temp):
    top = logits.amax(-1, keepdim=True)
    if temp <= 0:
        return torch.zeros_like(logits).scatter_(1, logits.argmax(-1, keepdim=True), 1.0)
    w = torch.where(logits >= top - 16.0, torch.exp((logits - top).double() / temp), 0.0)
    return (w / w.sum(-1, keepdim=True)).float()


def _plain_verify(p, q, ids, starts, u):
    rows, vocab = p.shape
    seqs = starts.numel() - 1
    s = torch.arange(seqs, device=p.device)
    b = torch.repeat_interleave(s, starts.diff(), output_size=rows)
    r = torch.arange(rows, device=p.device)
    last = r == starts[b + 1] - 1
    x = ids[(r + 1).clamp(max=rows - 1)].long()  # the draft behind each row
    qr = (r - b).clamp(max=max(rows - seqs - 1, 0))  # its row of q: q has none for a sequence's last row
    qx = 1.0 if q is None else (q[qr, x].double() if q.shape[0] else torch.zeros(rows, device=p.device))
    keep = (u.double() * qx < p[r, x].double()) & ~last
    # rows before the first refused one of each sequence
    bad = torch.where(keep, rows, r)
    stop = torch.full((seqs,), rows, device=p.device).index_reduce_(0, b, bad, "amin")
    taken = stop - starts[:-1]
    w = p[stop].double()
    sub = torch.zeros_like(w)
    if q is None:
        sub.scatter_(1, x[stop][:, None], p[stop, x[stop]].double()[:, None])
    elif q.shape[0]:
        sub = q[qr[stop]].double()
    w = torch.where(last[stop][:, None], w, w - sub).clamp(min=0)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p[stop].double())
    cum = w.cumsum(-1)
    draw_at = u[starts[1:].long() - 1].double() * cum[:, -1]
    new = torch.searchsorted(cum, draw_at[:, None], right=True).squeeze(-1)
    final = (w > 0).long().mul(torch.arange(vocab, device=p.device)).amax(-1)
    new = torch.minimum(new, final)
    out = torch.where(r < stop[b], x, torch.where(r == stop[b], new[b], -1))
    return taken.to(torch.int32), out.to(torch.int32)


# ------------------------------------------------------------------ 64 bits, one sequence at a time
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return globals()["_exact_" + case["kind"]](case, st)


def _dense(st, b, name, upto):
    """Rows 0 .. upto - 1 of sequence b: codes and scales, [positions, kv, ...]."""
    codes, scales = st["pages"][name], st["pages"][name + "_scale"]
    page = codes.shape[2]
    at = st["table"][b, :-(-upto // page)].long()
    c = codes[at].transpose(1, 2).reshape(-1, *codes.shape[1::2])[:upto].double()
    s = scales[at].transpose(1, 2).reshape(-1, codes.shape[1]).repeat_interleave(BLOCK, 0)[:upto]
    return c, s


def _exact_append(case, st):
    got = []
    for name in "kv":
        x, rows, t = st["new_" + name].double(), [], 0
        x = x.view(x.shape[0], case["kv"], case["hd"])
        for b, (c, n) in enumerate(_lengths(case)):
            if not n:
                continue
            lo = (c - n) // BLOCK * BLOCK
            codes, scales = (v[lo:] for v in _dense(st, b, name, c))
            old = c - n - lo  # tokens of the first block that stay
            new = x[t:t + n]
            t += n
            for j in range(0, c - lo, BLOCK):
                e = min(j + BLOCK, c - lo)
                stay = max(0, min(old - j, BLOCK))
                fresh = new[j + stay - old:e - old]
                was = scales[j] if stay else torch.zeros_like(scales[j])
                s = torch.maximum(was, (fresh.abs().amax((0, 2)) / 127.0).float())
                d = torch.where(s > 0, s, 1.0).double()[:, None]
                vals = torch.cat([codes[j:j + stay] * was.double()[:, None], fresh]) / d
                rows.append(torch.clamp(torch.round(vals), -127, 127) * s.double()[:, None])
        got.append(torch.cat(rows))
    return tuple(got)


def _exact_attend(case, st):
    kv, hd = case["kv"], case["hd"]
    group = case["heads"] // kv
    out, t = [], 0
    for b, (c, n) in enumerate(_lengths(case)):
        if not n:
            continue
        (kc, ks), (vc, vs) = _dense(st, b, "k", c), _dense(st, b, "v", c)
        keys, values = kc * ks.double()[:, :, None], vc * vs.double()[:, :, None]
        q = st["q"][t:t + n].double().view(n, kv, group, hd)
        t += n
        o = torch.empty_like(q)
        hidden = torch.arange(c, device=q.device)[None, :] > torch.arange(c - n, c, device=q.device)[:, None]
        for h in range(kv):
            a = torch.einsum("ngd,cd->gnc", q[:, h], keys[:, h]) / math.sqrt(hd)
            a = torch.softmax(a.masked_fill(hidden, float("-inf")), -1)
            o[:, h] = torch.einsum("gnc,cd->ngd", a, values[:, h])
        out.append(o.reshape(n, -1))
    return torch.cat(out)


def _exact_fork(case, st):
    """One sequence after the other, on the host."""
    page, beams = case["page"], case["beams"]
    table, refs, ctx = st["table"].tolist(), st["refs"].tolist(), st["ctx"].tolist()
    for a, b in zip(st["src"].tolist(), st["dst"].tolist()):  # the children hold nothing yet
        table[b], ctx[b] = list(table[a]), ctx[a]
        for p in table[b]:
            if p >= 0:
                refs[p] += 1
    writers = {}
    for b in range(len(table)):
        if ctx[b] % page:
            writers.setdefault(table[b][ctx[b] // page], []).append(b)
    before, src, dst, pending = list(refs), [-1] * len(table), [-1] * len(table), []
    for b in range(len(table)):
        j = ctx[b] // page
        old = table[b][j]
        if ctx[b] % page:
            group = writers[old]
            if before[old] == 1 or (before[old] == len(group) and group[0] == b):
                continue
            src[b] = old
            refs[old] -= 1
        pending.append((b, j))
    free = [p for p, r in enumerate(before) if r == 0]
    for (b, j), p in zip(pending, free):
        table[b][j] = p
        refs[p] += 1
        if src[b] >= 0:
            dst[b] = p
    for pool in st["pools"]:
        for a, b in zip(src, dst):
            if a >= 0:
                pool[b] = pool[a]
    status = [0, len(pending), len(free) - len(pending)]
    return (_ints(table), _ints([c + 1 for c in ctx]), _ints(refs), _ints(src), _ints(dst), _ints(status),
            [p.double() for p in st["pools"]])


def _exact_compact(case, st):
    table, refs = st["table0"].tolist(), st["refs0"].tolist()
    n = sum(r > 0 for r in refs)
    src = [p for p in range(n, len(refs)) if refs[p]]
    dst = [p for p in range(n) if not refs[p]]
    move = dict(zip(src, dst))
    table = [[move.get(p, p) for p in row] for row in table]
    for a, b in move.items():
        refs[b], refs[a] = refs[a], 0
        for pool in st["pools"]:
            pool[b] = pool[a]
    fill = [-1] * (len(refs) // 2 - len(src))
    return (_ints(table), _ints(refs), _ints(src + fill), _ints(dst + fill), [p.double() for p in st["pools"]])


def _exact_probs(case, st):
    rows = []
    for l in st["logits"]:
        if case["temp"] <= 0:
            rows.append(torch.nn.functional.one_hot(torch.argmax(l), l.numel()).double())
            continue
        top = l.max()
        w = torch.exp((l.double() - top.double()) / case["temp"]) * (l >= top - 16.0)
        rows.append(w / w.sum())
    return torch.stack(rows)


def _exact_verify(case, st):
    taken, tokens, t, at = [], [], 0, 0
    ids, u = st["ids"].tolist(), st["u"].tolist()
    for n in _drafts(case):
        kept = 0
        while kept < n:
            x = ids[t + kept + 1]
            q = 1.0 if st["q"] is None else float(st["q"][at + kept, x])
            if not u[t + kept] * q < float(st["p"][t + kept, x]):
                break
            kept += 1
        p = st["p"][t + kept].double()
        w = p.clone()
        if kept < n and st["q"] is None:
            w[ids[t + kept + 1]] = 0.0
        elif kept < n:
            w = (w - st["q"][at + kept].double()).clamp(min=0)
        if not float(w.sum()) > 0:
            w = p
        cum = torch.cumsum(w, 0)
        pick = int((cum <= u[t + n] * float(cum[-1])).sum())
        pick = min(pick, int(torch.nonzero(w > 0)[-1]))
        taken.append(kept)
        tokens += ids[t + 1:t + 1 + kept] + [pick] + [-1] * (n - kept)
        t += n + 1
        at += n
    return _ints(taken), _ints(tokens)
