"""Op-level entry points on CUDA tensors (thin wrappers over the C ABI).

Names follow the reference kernels they replace: ``pack_q8`` (quantize.py:31),
``mm_q8`` (k_mm_q8 / mm_q8_op, src/llama_q8.mojo:54-141), ``embed_q8``
(k_embed_gather_q8, :96), ``rmsnorm`` (k_rmsnorm_w, src/llama_common.mojo:197),
``rmsnorm_heads`` (k_rmsnorm2_w, :228), ``rope_kv_append`` (k_rope_qk_copy2,
:299), ``attention`` (k_scores/k_softmax_rows/k_att_out, :402-473),
``argmax`` (k_argmax, :493).  Tensors are torch CUDA tensors (torch provides
device memory and the stream); every kernel is in libq8cuda.so.

Without a counterpart in the reference: the 8-bit paged cache (``KV8Pages``,
``rope``, ``kv8_append``, ``kv8_read``, ``kv8_attention``), the page tables of either cache
(``kv_truncate``, ``kv_fork``, ``kv_reserve``, ``kv_compact``, ``kv_copy_pages``) and
speculative decoding (``probs``, ``verify``).  include/q8cuda.h says what each
does; these run on the device of their tensors, on torch's current stream
there, and may be captured into CUDA graphs.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from ._lib import check, lib

QG = 64


def _stream(t: torch.Tensor):
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("libq8cuda ops take CUDA tensors")


def row_u16(m: int) -> int:
    return m // QG + m // 2


def pack_q8(w_bf16: torch.Tensor) -> torch.Tensor:
    """bf16 [n, m] -> packed int16 [n, m/64 + m/2] (bit pattern of the reference's F16 tensor)."""
    _need_cuda(w_bf16)
    assert w_bf16.dtype == torch.bfloat16 and w_bf16.dim() == 2
    w = w_bf16.contiguous()
    n, m = w.shape
    out = torch.empty((n, row_u16(m)), dtype=torch.int16, device=w.device)
    check(lib().q8op_pack(_p(w), n, m, _p(out), _stream(w)))
    return out


def dequant_q8(packed: torch.Tensor, m: int) -> torch.Tensor:
    _need_cuda(packed)
    n = packed.shape[0]
    out = torch.empty((n, m), dtype=torch.float32, device=packed.device)
    check(lib().q8op_dequant(_p(packed), n, m, _p(out), _stream(packed)))
    return out


_DT = {torch.float32: _lib.Q8_F32, torch.bfloat16: _lib.Q8_BF16, torch.float16: _lib.Q8_F16}


def mm_q8(x: torch.Tensor, packed: torch.Tensor, m: int, out: torch.Tensor = None) -> torch.Tensor:
    """y[s, n] = x[s, m] . W[n, m]^T with W packed Q8."""
    _need_cuda(x, packed)
    assert x.dim() == 2 and x.shape[1] == m and x.stride(1) == 1
    n = packed.shape[0]
    s = x.shape[0]
    y = out if out is not None else torch.empty((s, n), dtype=torch.float32, device=x.device)
    check(lib().q8op_gemm(_p(x), _DT[x.dtype], x.stride(0), s, m, _p(packed), n, _p(y), y.stride(0), _stream(x)))
    return y


def mm_bf16(x: torch.Tensor, w_bf16: torch.Tensor, out: torch.Tensor = None) -> torch.Tensor:
    """y[s, n] = x[s, m] . W[n, m]^T with f32 x and plain bf16 W (mm_op,
    src/llama_common.mojo:636-684)."""
    _need_cuda(x, w_bf16)
    assert x.dtype == torch.float32 and w_bf16.dtype == torch.bfloat16 and x.stride(1) == 1
    assert w_bf16.is_contiguous() and x.shape[1] == w_bf16.shape[1]
    s, m = x.shape
    n = w_bf16.shape[0]
    y = out if out is not None else torch.empty((s, n), dtype=torch.float32, device=x.device)
    check(lib().q8op_gemm_bf16(_p(x), x.stride(0), s, m, _p(w_bf16), n, _p(y), y.stride(0), _stream(x)))
    return y


def mm_q8_swiglu(x: torch.Tensor, packed_gu: torch.Tensor, m: int) -> torch.Tensor:
    """silu(x.Wg^T) * (x.Wu^T) with the F gate rows then F up rows in ``packed_gu``."""
    _need_cuda(x, packed_gu)
    F = packed_gu.shape[0] // 2
    s = x.shape[0]
    y = torch.empty((s, F), dtype=torch.float32, device=x.device)
    check(lib().q8op_gemm_swiglu(_p(x), _DT[x.dtype], x.stride(0), s, m, _p(packed_gu), F, _p(y), F,
                                 _stream(x)))
    return y


def embed_q8(packed_emb: torch.Tensor, d: int, ids: torch.Tensor) -> torch.Tensor:
    _need_cuda(packed_emb, ids)
    ids = ids.to(torch.int32).contiguous()
    y = torch.empty((ids.numel(), d), dtype=torch.float32, device=ids.device)
    check(lib().q8op_embed(_p(packed_emb), packed_emb.shape[0], d, _p(ids), ids.numel(), _p(y), _stream(ids)))
    return y


def rmsnorm(x: torch.Tensor, w_bf16: torch.Tensor, eps: float, resid: torch.Tensor = None) -> torch.Tensor:
    """y = w * x / sqrt(mean(x^2) + eps); with ``resid`` x is first updated in place to x + resid."""
    _need_cuda(x, w_bf16, resid)
    assert x.is_contiguous()
    y = torch.empty_like(x)
    rows, d = x.shape
    check(lib().q8op_rmsnorm(_p(x), _p(resid), _p(w_bf16), rows, d, eps, _p(y), _stream(x)))
    return y


def rmsnorm_heads(x: torch.Tensor, w_bf16: torch.Tensor, eps: float) -> torch.Tensor:
    _need_cuda(x, w_bf16)
    hd = x.shape[-1]
    y = torch.empty_like(x)
    check(lib().q8op_rmsnorm_heads(_p(x), _p(w_bf16), x.numel() // hd, hd, eps, _p(y), _stream(x)))
    return y


def rope_inv_freq(cfg) -> torch.Tensor:
    import numpy as np
    out = np.zeros(cfg.head_dim // 2, np.float32)
    c = cfg.to_c()
    check(lib().q8_rope_inv_freq(C.byref(c), out.ctypes.data_as(C.c_void_p)))
    return torch.from_numpy(out)


def rope(qkv, pos, n_heads, n_kv, hd, inv_freq, q_norm=None, k_norm=None, eps=1e-6):
    """(QK-norm and) RoPE of the q and k heads of q|k|v rows (f32), in place, without an append."""
    dev = qkv.get_device()
    rows, width, ld = _matrix(qkv, "rope: qkv", dev)
    if width < (n_heads + 2 * n_kv) * hd:
        raise ValueError(f"rope: qkv rows of {n_heads} + 2 x {n_kv} heads of {hd} wanted, got {width} columns")
    _tensor(pos, "rope: pos", torch.int32, (rows,), dev)
    _tensor(inv_freq, "rope: inv_freq", torch.float32, (hd // 2,), dev)
    for t, what in ((q_norm, "rope: q_norm"), (k_norm, "rope: k_norm")):
        if t is not None:
            _tensor(t, what, torch.bfloat16, (hd,), dev)
    if rows:
        _call(lib().q8op_rope_kv_append, dev, qkv.data_ptr(), ld, rows, pos.data_ptr(), None, n_heads, n_kv, hd,
              inv_freq.data_ptr(), _p(q_norm), _p(k_norm), eps, None, None, 0, None, 0)


def rope_kv_append(qkv, pos, seq, n_heads, n_kv, hd, inv_freq, q_norm, k_norm, eps, k_pages, v_pages, page,
                   block_table):
    _need_cuda(qkv, pos, seq, inv_freq, k_pages, v_pages, block_table)
    T = qkv.shape[0]
    check(lib().q8op_rope_kv_append(_p(qkv), qkv.stride(0), T, _p(pos), _p(seq), n_heads, n_kv, hd, _p(inv_freq),
                                    _p(q_norm), _p(k_norm), eps, _p(k_pages), _p(v_pages), page, _p(block_table),
                                    block_table.shape[1], _stream(qkv)))


def attention(q, pos, seq, n_heads, n_kv, hd, k_pages, v_pages, page, block_table) -> torch.Tensor:
    _need_cuda(q, pos, seq, k_pages, v_pages, block_table)
    T = q.shape[0]
    out = torch.empty((T, n_heads * hd), dtype=torch.float32, device=q.device)
    check(lib().q8op_attention(_p(q), q.stride(0), T, _p(pos), _p(seq), n_heads, n_kv, hd, _p(k_pages),
                               _p(v_pages), page, _p(block_table), block_table.shape[1], _p(out), out.stride(0),
                               _stream(q)))
    return out


def argmax(logits: torch.Tensor) -> torch.Tensor:
    _need_cuda(logits)
    if logits.dim() == 1:
        logits = logits[None]
    out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    check(lib().q8op_argmax(_p(logits), logits.shape[0], logits.shape[1], logits.stride(0), _p(out),
                            _stream(logits)))
    return out


# ------------------------------------------------------------------ 8-bit paged cache
KV8_BLOCK = 16  # tokens of a kv head that share a scale (Q8_KV8_BLOCK)


def _tensor(t, what, dtype, shape, dev: int) -> None:
    """Raises unless ``t`` is a contiguous tensor of ``dtype`` (and shape) on CUDA device ``dev``."""
    try:
        if t.dtype is dtype and t.get_device() == dev and t.is_contiguous() and (shape is None or t.shape == shape):
            return
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what}: libq8cuda ops take CUDA tensors")
    if t.dtype is not dtype:
        raise ValueError(f"{what}: {dtype} wanted, got {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{what}: is on {t.device}, other tensors of the call on cuda:{dev}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: must be contiguous")
    raise ValueError(f"{what}: shape {tuple(shape)} wanted, got {tuple(t.shape)}")


_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _call(fn, dev: int, *args) -> None:
    """fn(*args, stream) on torch's current stream of device ``dev``."""
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            check(fn(*args, _raw_stream(dev)))
        return
    status = fn(*args, _raw_stream(dev))
    if status:
        check(status)


class KV8Pages:
    """One layer's pages of the 8-bit cache: int8 codes k, v [num_pages, n_kv, page, head_dim]
    and f32 scales k_scale, v_scale [num_pages, n_kv, page / 16]; a value is code * scale."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "num_pages", "n_kv", "page", "head_dim", "_c", "_ref", "_dev")

    def __init__(self, k, v, k_scale, v_scale):
        dev = k.get_device()
        _tensor(k, "KV8Pages k", torch.int8, None, max(dev, 0))
        if k.dim() != 4 or k.shape[2] == 0 or k.shape[2] % KV8_BLOCK or k.shape[3] not in (64, 128):
            raise ValueError(f"KV8Pages k: [pages, n_kv, page (a multiple of {KV8_BLOCK}), head_dim (64 or 128)] "
                             f"wanted, got {tuple(k.shape)}")
        pages, kv, page, hd = k.shape
        _tensor(v, "KV8Pages v", torch.int8, k.shape, dev)
        for t, what in ((k_scale, "KV8Pages k_scale"), (v_scale, "KV8Pages v_scale")):
            _tensor(t, what, torch.float32, (pages, kv, page // KV8_BLOCK), dev)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.n_kv, self.page, self.head_dim = pages, kv, page, hd
        self._c = _lib.q8_kv8_pages(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, kv,
                                    page, hd)
        self._ref = C.addressof(self._c)
        self._dev = dev

    def __setattr__(self, name, value):
        if hasattr(self, "_dev"):  # set last: the calls go by the addresses taken here
            raise AttributeError(f"KV8Pages: {name} cannot be replaced, make another KV8Pages")
        super().__setattr__(name, value)

    @classmethod
    def empty(cls, num_pages: int, n_kv: int, page: int = 64, head_dim: int = 128, device="cuda") -> "KV8Pages":
        """Zeroed pages."""
        shape = (num_pages, n_kv, page, head_dim)
        scales = (num_pages, n_kv, page // KV8_BLOCK)
        return cls(torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(scales, dtype=torch.float32, device=device),
                   torch.zeros(scales, dtype=torch.float32, device=device))

    @property
    def device(self) -> torch.device:
        return self.k.device

    def tensors(self) -> list:
        """The four pools, as kv_copy_pages takes them."""
        return [self.k, self.v, self.k_scale, self.v_scale]


def _packed(what, seq_start, ctx, pages, block_table):
    """Checks what every call on packed rows takes; returns (S, max_pages, device)."""
    if not isinstance(pages, KV8Pages):
        raise ValueError(f"{what}: pages must be a KV8Pages")
    dev = pages._dev
    if block_table.dim() != 2:
        raise ValueError(f"{what}: block_table [S, max_pages] wanted")
    S, width = block_table.shape
    _tensor(seq_start, what + ": seq_start", torch.int32, (S + 1,), dev)
    _tensor(ctx, what + ": ctx", torch.int32, (S,), dev)
    _tensor(block_table, what + ": block_table", torch.int32, None, dev)
    return S, width, dev


def _rows_of(t, what, width, dev: int):
    """[T, width] or [T, heads, head_dim] rows with contiguous elements: (row count, row stride)."""
    if t.get_device() != dev:
        raise ValueError(f"{what}: is on {t.device}, the pages are on cuda:{dev}")
    if t.dtype not in _DT:
        raise ValueError(f"{what}: f32, bf16 or f16 rows wanted, got {t.dtype}")
    st, sh = t.stride(), t.shape
    if len(sh) == 2 and sh[1] == width and (st[1] == 1 or width == 1):
        return sh[0], st[0] if sh[0] > 1 else max(st[0], width)
    if len(sh) == 3 and sh[1] * sh[2] == width and st[2] == 1 and (st[1] == sh[2] or sh[1] == 1):
        return sh[0], st[0] if sh[0] > 1 else max(st[0], width)
    raise ValueError(f"{what}: rows of {width} contiguous elements wanted, got shape {tuple(sh)}, strides {st}")


def kv8_append(k, v, seq_start, ctx, pages: KV8Pages, block_table) -> None:
    """Write the packed rows' (rotated) k and v, the last positions of their sequences, into
    the 8-bit pages (q8op_kv8_append).  ctx counts them already."""
    S, width, dev = _packed("kv8_append", seq_start, ctx, pages, block_table)
    w = pages.n_kv * pages.head_dim
    T, ldk = _rows_of(k, "kv8_append: k", w, dev)
    Tv, ldv = _rows_of(v, "kv8_append: v", w, dev)
    if T != Tv or k.dtype != v.dtype:
        raise ValueError("kv8_append: k and v must have the same rows and type")
    _call(lib().q8op_kv8_append, dev, k.data_ptr(), ldk, v.data_ptr(), ldv, _DT[k.dtype], T, seq_start.data_ptr(),
          ctx.data_ptr(), S, pages._ref, block_table.data_ptr(), width)


def kv8_read(seq_start, ctx, pages: KV8Pages, block_table, rows: int):
    """(k, v) f32 [rows, n_kv, head_dim]: the cached values at the packed rows' positions
    (rows behind the last sequence are not written)."""
    S, width, dev = _packed("kv8_read", seq_start, ctx, pages, block_table)
    if rows < 0:
        raise ValueError("kv8_read: rows < 0")
    k, v = torch.empty((2, rows, pages.n_kv, pages.head_dim), dtype=torch.float32, device=pages.k.device).unbind(0)
    _call(lib().q8op_kv8_read, dev, pages._ref, seq_start.data_ptr(), ctx.data_ptr(), S, block_table.data_ptr(),
          width, k.data_ptr(), v.data_ptr(), rows)
    return k, v


@functools.lru_cache(maxsize=1024)
def _kv8_scratch(dev, *shape) -> int:
    return lib().q8op_kv8_attention_workspace(*shape)


def kv8_attention(q, seq_start, ctx, n_heads: int, pages: KV8Pages, block_table, out=None) -> torch.Tensor:
    """Causal GQA attention of packed rows over the 8-bit cache (q8op_kv8_attention).  Returns
    [T, n_heads * head_dim] of q's type; ``out`` may be given (rows behind the last sequence are not written)."""
    S, width, dev = _packed("kv8_attention", seq_start, ctx, pages, block_table)
    if torch.cuda.current_device() != dev:  # the scratch's size goes by the device
        with torch.cuda.device(dev):
            return kv8_attention(q, seq_start, ctx, n_heads, pages, block_table, out)
    w = n_heads * pages.head_dim
    T, ldq = _rows_of(q, "kv8_attention: q", w, dev)
    if out is None:
        out, ldo = q.new_empty((T, w)), w
    else:
        To, ldo = _rows_of(out, "kv8_attention: out", w, dev)
        if To != T or out.dtype != q.dtype:
            raise ValueError("kv8_attention: out must have q's rows and type")
    nbytes = _kv8_scratch(dev, _DT[q.dtype], T, S, n_heads, pages.n_kv, pages.head_dim, width * pages.page)
    # held until the kernels are in the stream: the allocator may give a free block to another thread before that
    work = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _call(lib().q8op_kv8_attention, dev, q.data_ptr(), ldq, _DT[q.dtype], T, seq_start.data_ptr(), ctx.data_ptr(), S,
          n_heads, pages._ref, block_table.data_ptr(), width, out.data_ptr(), ldo,
          None if work is None else work.data_ptr(), nbytes)
    return out


# ------------------------------------------------------------------ page tables
def _state(what, block_table, ctx, refs):
    if block_table.dim() != 2 or refs.dim() != 1:
        raise ValueError(f"{what}: block_table [S, max_pages] and refs [num_pages] wanted")
    dev = block_table.get_device()
    S, width = block_table.shape
    _tensor(block_table, what + ": block_table", torch.int32, None, max(dev, 0))
    if ctx is not None:
        _tensor(ctx, what + ": ctx", torch.int32, (S,), dev)
    _tensor(refs, what + ": refs", torch.int32, None, dev)
    return S, width, refs.shape[0], dev


def kv_truncate(block_table, ctx, refs, page: int, new_len) -> None:
    """Shorten (0: free) the sequences to new_len [S] positions, in place; negative: leave alone."""
    S, width, pages, dev = _state("kv_truncate", block_table, ctx, refs)
    _tensor(new_len, "kv_truncate: new_len", torch.int32, (S,), dev)
    _call(lib().q8op_kv_truncate, dev, block_table.data_ptr(), S, width, ctx.data_ptr(), refs.data_ptr(), pages,
          page, new_len.data_ptr())


def kv_fork(block_table, ctx, refs, page: int, src, dst) -> None:
    """Sequences dst [n] become sequences src [n] as they were before the call, sharing their pages."""
    S, width, pages, dev = _state("kv_fork", block_table, ctx, refs)
    n = src.numel()
    _tensor(src, "kv_fork: src", torch.int32, (n,), dev)
    _tensor(dst, "kv_fork: dst", torch.int32, (n,), dev)
    _call(lib().q8op_kv_fork, dev, block_table.data_ptr(), S, width, ctx.data_ptr(), refs.data_ptr(), pages, page,
          src.data_ptr(), dst.data_ptr(), n)


def kv_reserve(block_table, ctx, refs, page: int, n_new):
    """Make room for n_new [S] more positions, in place; ctx grows by them.  Returns (src, dst,
    status): the page copies to make before writing (kv_copy_pages), and [0 or Q8_ERR_KV_FULL,
    pages wanted, pages free], all on the device.  When the pool is too small nothing changes."""
    S, width, pages, dev = _state("kv_reserve", block_table, ctx, refs)
    _tensor(n_new, "kv_reserve: n_new", torch.int32, (S,), dev)
    got = refs.new_empty(2 * S + 3 + pages)
    at = got.data_ptr()
    _call(lib().q8op_kv_reserve, dev, block_table.data_ptr(), S, width, ctx.data_ptr(), refs.data_ptr(), pages, page,
          n_new.data_ptr(), at, at + 4 * S, at + 8 * S, at + 8 * S + 12)
    return got.split_with_sizes((S, S, 3, pages))[:3]  # the rest is scratch


def kv_compact(block_table, refs):
    """Renumber the pages so that those in use come first, in place.  Returns (src, dst)
    [num_pages / 2], the page copies to make (kv_copy_pages), -1 behind the last."""
    S, width, pages, dev = _state("kv_compact", block_table, None, refs)
    half = pages // 2
    got = refs.new_empty(2 * half + pages)
    at = got.data_ptr()
    _call(lib().q8op_kv_compact, dev, block_table.data_ptr(), S, width, refs.data_ptr(), pages, at, at + 4 * half,
          at + 8 * half)
    return got.split_with_sizes((half, half, pages))[:2]  # the rest is scratch


def kv_copy_pages(pools, src, dst) -> None:
    """pool[dst[i]] = pool[src[i]] in every pool (contiguous, pages first); pairs with a
    negative number are left out, and so are pairs whose result would depend on the order."""
    if not pools:
        return
    dev, num_pages, n = pools[0].get_device(), pools[0].shape[0], src.numel()
    _tensor(src, "kv_copy_pages: src", torch.int32, (n,), max(dev, 0))
    _tensor(dst, "kv_copy_pages: dst", torch.int32, (n,), dev)
    addr, size = [], []
    for t in pools:
        _tensor(t, "kv_copy_pages: pool", t.dtype, None, dev)
        if t.dim() < 2 or t.shape[0] != num_pages or t.numel() == 0:
            raise ValueError("kv_copy_pages: pools of the same number of pages wanted")
        addr.append(t.data_ptr())
        size.append(t.nbytes // num_pages)
    for at in range(0, len(addr), 64):
        k = min(64, len(addr) - at)
        _call(lib().q8op_kv_copy_pages, dev, (C.c_void_p * k)(*addr[at:at + k]), (C.c_int64 * k)(*size[at:at + k]), k,
              num_pages, src.data_ptr(), dst.data_ptr(), n)


# ------------------------------------------------------------------ speculative decoding
def _matrix(t, what, dev: int):
    """f32 [rows, n] with contiguous columns: (rows, n, row stride)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what}: libq8cuda ops take CUDA tensors")
    sh, st = t.shape, t.stride()
    if t.dtype is not torch.float32 or len(sh) != 2 or sh[1] == 0 or (sh[1] > 1 and st[1] != 1):
        raise ValueError(f"{what}: f32 [rows, n] with contiguous columns wanted")
    if t.get_device() != dev:
        raise ValueError(f"{what}: is on {t.device}, other tensors of the call on cuda:{dev}")
    return sh[0], sh[1], st[0] if sh[0] > 1 else max(st[0], sh[1])


def probs(logits: torch.Tensor, temp: float, out: torch.Tensor = None) -> torch.Tensor:
    """The distributions that sampling at ``temp`` and top_p = 1 draws from (q8op_probs); ``out`` may be ``logits``."""
    dev = logits.get_device()
    rows, n, ld = _matrix(logits, "probs: logits", dev)
    if out is None:
        out, ldo = logits.new_empty((rows, n)), n
    else:
        ro, no, ldo = _matrix(out, "probs: out", dev)
        if (ro, no) != (rows, n):
            raise ValueError("probs: out must have the shape of logits")
    _call(lib().q8op_probs, dev, logits.data_ptr(), rows, n, ld, temp, out.data_ptr(), ldo)
    return out


def verify(p, q, ids, seq_start, u):
    """Verify drafted tokens against the target's distributions p [T, n] (q8op_verify): q is the
    drafts' [drafts, n] or None (certain drafts), ids [T] the tokens fed, u [T] uniform draws.
    Returns (n_accepted [S], tokens [T]: kept drafts, the next token, -1; rows behind the last sequence are
    not written)."""
    dev = p.get_device()
    rows, n, ldp = _matrix(p, "verify: p", dev)
    S = seq_start.numel() - 1
    if S < 0:
        raise ValueError("verify: seq_start [S + 1] wanted")
    _tensor(seq_start, "verify: seq_start", torch.int32, (S + 1,), dev)
    _tensor(ids, "verify: ids", torch.int32, (rows,), dev)
    _tensor(u, "verify: u", torch.float32, (rows,), dev)
    q_rows, ldq, qp = 0, 0, None
    if q is not None:
        if q.shape[0] == 0:  # no row has a draft
            ldq, qp = n, p.data_ptr()
        else:
            q_rows, nq, ldq = _matrix(q, "verify: q", dev)
            if nq != n:
                raise ValueError("verify: q must have p's columns")
            qp = q.data_ptr()
    n_accepted, tokens = ids.new_empty(S + rows).split_with_sizes((S, rows))
    _call(lib().q8op_verify, dev, p.data_ptr(), ldp, qp, ldq, q_rows, ids.data_ptr(), seq_start.data_ptr(), rows, S,
          n, u.data_ptr(), n_accepted.data_ptr(), tokens.data_ptr())
    return n_accepted, tokens


def device_status() -> None:
    """Synchronize the current device and raise if a tensor-core GEMM's bounded
    pipeline wait timed out since the last poll (q8_device_status)."""
    check(lib().q8_device_status())
