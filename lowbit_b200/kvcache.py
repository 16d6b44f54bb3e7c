"""Paged 8-bit KV cache: the pool, and the operators that fill and read it.

A cache of one layer is a pool of pages. A page holds `page` tokens of every
KV head; a block, the tokens of one page and head, shares one power-of-two
scale (E8M0 byte e, as MXFP4's): an int8 code stands for code * 2^(e - 127),
which bf16 holds exactly. Sequences own pages through a page table, so
sequences of different lengths run in one call and share prefixes.

* ``kv8_append``     bias and rotate-half position rotation of fused q/k/v rows;
                     k and v quantised into their pages, q returned rotated;
* ``kv8_attention``  causal grouped-query attention of the new tokens over the
                     pages, optionally within a sliding window;
* ``kv8_read``       pages back as values.

The new tokens of B sequences are N rows: sequence b owns rows
``starts[b]:starts[b + 1]`` (``starts`` int32 [B + 1] on the GPU; without it
every sequence has N / B), and its t-th row sits at position ``pos[b] + t``
(``pos`` int32 [B] on the GPU: the tokens already held). Position p lives in
slot p % page of page ``table[b, p // page]`` (int32 [B, width] on the GPU).
Rows at negative positions are padding (nothing stored, output 0): a fixed
batch marks its free places with ``pos`` -1. All of it is read on the device,
so a captured CUDA graph replays with new positions and tables. Ids or
positions out of range are skipped on the device and recorded in
``kernels.device_status()``.

The reference has no counterpart: its cache is one fp32 array per layer
(src/lowbit/model.py:216-230).
"""
from __future__ import annotations

import ctypes as C

import torch

from .kernels import _check, _raw_stream, lib

_device = torch._C._cuda_getDevice
PAGES = (16, 32, 64, 128)
HEAD_DIMS = (32, 64, 128)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _KV8(C.Structure):
    _fields_ = ([(f, C.c_void_p) for f in ("k", "v", "k_exp", "v_exp")]
                + [(f, C.c_longlong) for f in ("page_stride", "exp_stride")]
                + [(f, C.c_int) for f in ("pages", "page", "kv_heads", "head_dim")])


class KV8Cache:
    """One layer's pool: int8 codes ``k``, ``v`` [pages, kv_heads, page,
    head_dim] and E8M0 bytes ``k_exp``, ``v_exp`` uint8 [pages, kv_heads], all
    on one GPU. Pages may lie apart (any stride of dimension 0 that is a
    multiple of 16 bytes, the same for k and v); within a page the layout is
    contiguous."""

    __slots__ = ("k", "v", "k_exp", "v_exp", "device", "pages", "kv_heads", "page", "head_dim", "_c", "_ref",
                 "_scratch")

    def __init__(self, k, v, k_exp, v_exp):
        if k.dim() != 4 or v.shape != k.shape or k.dtype != torch.int8 or v.dtype != torch.int8:
            raise ValueError("k and v must be int8 [pages, kv_heads, page, head_dim]")
        pages, kv, page, d = k.shape
        if k_exp.shape != (pages, kv) or v_exp.shape != (pages, kv) or k_exp.dtype != torch.uint8 \
                or v_exp.dtype != torch.uint8:
            raise ValueError("k_exp and v_exp must be uint8 [pages, kv_heads]")
        if any(t.device != k.device for t in (v, k_exp, v_exp)) or not k.is_cuda:
            raise ValueError("k, v, k_exp and v_exp must be on one CUDA device")
        if page not in PAGES or d not in HEAD_DIMS or not pages or not kv:
            raise ValueError(f"page must be one of {PAGES} tokens and head_dim one of {HEAD_DIMS}")
        inner = (page * d, d, 1)[0 if kv > 1 else 1:]  # one head's stride says nothing
        if k.stride()[-len(inner):] != inner or v.stride()[-len(inner):] != inner or (pages > 1 and k.stride(0) != v.stride(0)):
            raise ValueError("k and v must be contiguous within a page, with the same page stride")
        if (kv > 1 and (k_exp.stride(1) != 1 or v_exp.stride(1) != 1)) or (pages > 1 and k_exp.stride(0) != v_exp.stride(0)):
            raise ValueError("k_exp and v_exp must be contiguous within a page, with the same page stride")
        stride = k.stride(0) if pages > 1 else kv * page * d
        if stride < kv * page * d or stride % 16 or (pages > 1 and k_exp.stride(0) < kv) \
                or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("k and v must be 16-byte aligned pages that do not overlap")
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.device, self.pages, self.kv_heads, self.page, self.head_dim = k.device, pages, kv, page, d
        self._c = _KV8(k.data_ptr(), v.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), stride,
                       k_exp.stride(0) if pages > 1 else kv, pages, page, kv, d)
        self._ref = C.byref(self._c)
        self._scratch = {}  # workspace bytes of attention calls, by their sizes

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page: int = 64, device=None) -> "KV8Cache":
        """A pool of `pages` pages, all codes and scales zero."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        shape = (int(pages), int(kv_heads), int(page), int(head_dim))
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2))
        ke, ve = (torch.zeros(shape[:2], dtype=torch.uint8, device=device) for _ in range(2))
        return cls(k, v, ke, ve)

    @property
    def nbytes(self) -> int:
        return 2 * self.pages * self.kv_heads * (self.page * self.head_dim + 1)


def _rows(cache, n, table, pos, starts, max_tokens):
    """Checks the row description; (width, B, max_tokens, starts pointer)."""
    dev, i32 = cache.device, torch.int32
    if table.dim() != 2 or table.dtype is not i32 or not table.is_contiguous() or table.device != dev:
        raise ValueError("table must be a contiguous int32 [B, pages] tensor on the cache's device")
    b, width = table.shape
    if pos.dim() != 1 or len(pos) != b or pos.dtype is not i32 or not pos.is_contiguous() or pos.device != dev:
        raise ValueError("pos must be a contiguous int32 [B] tensor on the cache's device")
    if b == 0 or width == 0:
        raise ValueError("table must hold at least one sequence and one page")
    if starts is None:
        if n % b:
            raise ValueError(f"{n} rows do not divide over {b} sequences; give starts")
        most = n // b
        if max_tokens is not None and max_tokens < most:
            raise ValueError(f"max_tokens {max_tokens} is below the {most} rows of a sequence")
        return width, b, most, None
    if starts.shape != (b + 1,) or starts.dtype != torch.int32 or not starts.is_contiguous() or starts.device != dev:
        raise ValueError("starts must be a contiguous int32 [B + 1] tensor on the cache's device")
    most = n if max_tokens is None else min(int(max_tokens), n)
    if most < 0:
        raise ValueError("max_tokens must not be negative")
    return width, b, most, starts.data_ptr()


def _out(out, shape, dtype, device):
    if out.shape != shape or out.dtype != dtype or out.device != device or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous, 16-byte aligned {dtype} tensor of shape {tuple(shape)}")
    return out


def _aligned_rows(x, inner: tuple):
    """x with its dimensions after the first contiguous and 16-byte aligned rows."""
    if x.stride()[1:] == inner and x.data_ptr() % 16 == 0 and x.stride(0) * x.element_size() % 16 == 0 \
            and x.stride(0) >= inner[0] * x.shape[1]:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _ptr(t):
    return None if t is None else t.data_ptr()


def kv8_append(qkv, cache: KV8Cache, table, pos, cos, sin, bias=None, starts=None, max_tokens: int | None = None,
               out=None):
    """Append the k and v of fused rows ``qkv`` [N, (H + 2*KV)*D] (fp32, bf16 or
    fp16; + ``bias`` fp32) to the cache and return q rotated [N, H, D] in
    qkv's type. cos, sin: fp32 [positions, D/2] (model.rope_tables).
    ``max_tokens`` bounds the rows of a sequence when ``starts`` is given."""
    kv, d, dev = cache.kv_heads, cache.head_dim, cache.device
    if qkv.dim() != 2 or qkv.dtype not in _DTYPES or qkv.device != dev:
        raise ValueError("qkv must be an fp32, bf16 or fp16 [N, (H + 2*KV)*D] tensor on the cache's device")
    n, w = qkv.shape
    heads = w // d - 2 * kv
    if heads <= 0 or w % d or heads % kv:
        raise ValueError(f"qkv has {w} columns: not (H + 2*{kv}) * {d} with H a multiple of {kv}")
    f32 = torch.float32
    if cos.dim() != 2 or cos.shape[1] * 2 != d or cos.dtype is not f32 or not cos.is_contiguous() or cos.device != dev \
            or sin.shape != cos.shape or sin.dtype is not f32 or not sin.is_contiguous() or sin.device != dev:
        raise ValueError("cos and sin must be contiguous fp32 [positions, head_dim/2] tensors on the cache's device")
    if (cos.data_ptr() | sin.data_ptr()) % 16:
        raise ValueError("cos and sin must be 16-byte aligned")
    if bias is not None and (bias.shape != (w,) or bias.dtype is not f32 or not bias.is_contiguous()
                             or bias.device != dev):
        raise ValueError("bias must be a contiguous fp32 tensor of qkv's width")
    width, b, most, sp = _rows(cache, n, table, pos, starts, max_tokens)
    q = qkv.new_empty((n, heads, d)) if out is None else _out(out, (n, heads, d), qkv.dtype, dev)
    if n == 0:
        return q
    if _device() != dev.index:
        with torch.cuda.device(dev):
            return kv8_append(qkv, cache, table, pos, cos, sin, bias, starts, max_tokens, q)
    qkv = _aligned_rows(qkv, (1,))
    rc = lib().lbc_kv8_append(cache._ref, _DTYPES[qkv.dtype], qkv.data_ptr(), qkv.stride(0), _ptr(bias), cos.data_ptr(),
                              sin.data_ptr(), cos.shape[0], table.data_ptr(), width, pos.data_ptr(), sp, b, n, most,
                              heads, q.data_ptr(), _raw_stream(dev.index))
    if rc < 0:
        _check(rc, "lbc_kv8_append")
    return q


def kv8_attention(q, cache: KV8Cache, table, pos, starts=None, max_tokens: int | None = None, window: int = 0,
                  scale: float | None = None, out=None):
    """Attention of the rows ``q`` [N, H, D] (fp32, bf16 or fp16; rows may lie
    apart), whose k and v are already appended, over the cache: [N, H, D] in
    q's type. The row at position p sees positions p - window + 1 .. p (all up
    to p without a window); scale defaults to 1/sqrt(D). Rows that see nothing
    are 0."""
    kv, d, dev, L = cache.kv_heads, cache.head_dim, cache.device, lib()
    if q.dim() != 3 or q.dtype not in _DTYPES or q.device != dev or q.shape[2] != d:
        raise ValueError(f"q must be an fp32, bf16 or fp16 [N, H, {d}] tensor on the cache's device")
    n, heads, _ = q.shape
    if heads == 0 or heads % kv:
        raise ValueError(f"{heads} query heads are not a multiple of {kv} KV heads")
    if window < 0:
        raise ValueError("window must not be negative")
    width, b, most, sp = _rows(cache, n, table, pos, starts, max_tokens)
    if out is None:
        y = torch.empty_like(q) if q.is_contiguous() else q.new_empty((n, heads, d))
    else:
        y = _out(out, (n, heads, d), q.dtype, dev)
    if n == 0:
        return y
    if _device() != dev.index:
        with torch.cuda.device(dev):
            return kv8_attention(q, cache, table, pos, starts, max_tokens, window, scale, y)
    q = _aligned_rows(q, (d, 1))
    dt = _DTYPES[q.dtype]
    sizes = (width, b, most, heads, window)
    nb = cache._scratch.get(sizes)
    if nb is None:
        nb = cache._scratch[sizes] = L.lbc_kv8_attention_workspace(cache._ref, dt, width, b, n, most, heads, window)
    # from torch's allocator: private to this call in stream order, and to a graph when captured
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    rc = L.lbc_kv8_attention(cache._ref, dt, q.data_ptr(), q.stride(0), table.data_ptr(), width, pos.data_ptr(), sp,
                             b, n, most, heads, window, d ** -0.5 if scale is None else scale, y.data_ptr(),
                             _ptr(ws), nb, _raw_stream(dev.index))
    if rc < 0:
        _check(rc, "lbc_kv8_attention")
    return y


def kv8_read(cache: KV8Cache, pages, dtype=torch.bfloat16):
    """Keys and values of the pages ``pages`` (int32 ids on the GPU), each
    [len(pages), kv_heads, page, head_dim]: exact in bf16 and fp32; fp16 rounds
    what lies outside its range."""
    dev = cache.device
    if pages.dim() != 1 or pages.dtype != torch.int32 or not pages.is_contiguous() or pages.device != dev:
        raise ValueError("pages must be a contiguous int32 tensor of ids on the cache's device")
    if dtype not in _DTYPES:
        raise ValueError("dtype must be torch.float32, bfloat16 or float16")
    n = pages.shape[0]
    shape = (n, cache.kv_heads, cache.page, cache.head_dim)
    k = torch.empty(shape, dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if n == 0:
        return k, v
    if _device() != dev.index:
        with torch.cuda.device(dev):
            return kv8_read(cache, pages, dtype)
    _check(lib().lbc_kv8_read(cache._ref, _DTYPES[dtype], pages.data_ptr(), n, k.data_ptr(), v.data_ptr(),
                              _raw_stream(dev.index)), "lbc_kv8_read")
    return k, v


class PagedKVCache:
    """The model's cache over KV8Cache pools: one pool a layer, one page table
    and one position a sequence, shared by the layers. Sequences have lengths
    of their own. Pages are handed out from a free list as sequences grow
    (``reserve``) and go back with ``release``.

    Interface of model.KVCache: ``batch``, ``capacity``, ``pos`` (int32 [batch]
    on the GPU), ``length`` (sequences of equal length), ``reset()``."""

    def __init__(self, cfg, max_len: int, batch: int = 1, page: int = 64, pages: int | None = None):
        if batch <= 0 or max_len <= 0:
            raise ValueError("a cache holds at least one sequence of one token")
        width = -(-max_len // page)
        self.batch, self.page, self._max_len = batch, page, max_len
        n = batch * width if pages is None else int(pages)
        self.layers = [KV8Cache.empty(n, cfg.num_kv_heads, cfg.head_dim, page) for _ in range(cfg.num_layers)]
        dev = self.layers[0].device
        self.table = torch.zeros((batch, width), dtype=torch.int32, device=dev)
        self.pos = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.lengths = [0] * batch
        self._owned = [[] for _ in range(batch)]
        self._free = list(range(n - 1, -1, -1))

    @property
    def capacity(self) -> int:
        return self._max_len

    @property
    def nbytes(self) -> int:
        return sum(c.nbytes for c in self.layers)

    def reserve(self, tokens) -> None:
        """Pages for ``tokens[b]`` tokens of every sequence (an int: the same
        for all); raises ValueError, with nothing changed, when they do not fit."""
        tokens = [int(tokens)] * self.batch if isinstance(tokens, int) else [int(t) for t in tokens]
        if len(tokens) != self.batch:
            raise ValueError(f"{len(tokens)} lengths for {self.batch} sequences")
        if max(tokens) > self._max_len:
            raise ValueError(f"KV cache full ({max(tokens)} > {self._max_len})")
        more = [max(0, -(-t // self.page) - len(own)) for t, own in zip(tokens, self._owned)]
        if sum(more) > len(self._free):
            raise ValueError(f"KV cache out of pages ({sum(more)} needed, {len(self._free)} free)")
        if not any(more):
            return
        for own, m in zip(self._owned, more):
            own.extend(self._free.pop() for _ in range(m))
        host = torch.zeros(self.table.shape, dtype=torch.int32)
        for b, own in enumerate(self._owned):
            host[b, :len(own)] = torch.tensor(own, dtype=torch.int32)
        self.table.copy_(host)

    def release(self, b: int) -> None:
        """Empty sequence b and return its pages."""
        self._free.extend(reversed(self._owned[b]))
        self._owned[b] = []
        self.lengths[b] = 0
        self.pos[b] = 0

    @property
    def length(self) -> int:
        if len(set(self.lengths)) > 1:
            raise ValueError("the sequences have different lengths (see lengths)")
        return self.lengths[0]

    @length.setter
    def length(self, n: int) -> None:
        self.set_lengths([int(n)] * self.batch)

    def set_lengths(self, lengths) -> None:
        self.lengths = [int(n) for n in lengths]
        self.pos.copy_(torch.tensor(self.lengths, dtype=torch.int32))

    def reset(self) -> None:
        """Empty every sequence (pools, table and pages stay, so a captured decode graph stays valid)."""
        self.length = 0
