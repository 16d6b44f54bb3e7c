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
``kernels.device_status()``; output rows that no sequence owns are not written.

The reference has no counterpart: its cache is one fp32 array per layer
(src/lowbit/model.py:216-230).
"""
from __future__ import annotations

import ctypes as C

from .kernels import lib

PAGES = (16, 32, 64, 128)
HEAD_DIMS = (32, 64, 128)
_native = None  # csrc/kv8_torch.cpp, loaded on first use


def _torch():
    # imported when a cache is made or read: the package's names can be imported without torch
    import torch
    return torch


def _load():
    """The native module (argument checks, allocation and the C ABI call), bound to the loaded library."""
    global _native
    from importlib.machinery import ExtensionFileLoader
    from importlib.util import module_from_spec, spec_from_loader

    from ._build import build_torch
    loader = ExtensionFileLoader("_kv8_torch", str(build_torch()))
    mod = module_from_spec(spec_from_loader("_kv8_torch", loader))
    loader.exec_module(mod)
    L = lib()
    mod.init(*(C.cast(getattr(L, f), C.c_void_p).value
               for f in ("lbc_kv8_append", "lbc_kv8_attention", "lbc_kv8_attention_workspace", "lbc_kv8_read",
                         "lbc_last_error")))
    _native = mod
    return mod


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

    __slots__ = ("k", "v", "k_exp", "v_exp", "device", "pages", "kv_heads", "page", "head_dim", "_c", "_at",
                 "_index")

    def __init__(self, k, v, k_exp, v_exp):
        torch = _torch()
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
        self._at, self._index = C.addressof(self._c), k.device.index

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page: int = 64, device=None) -> "KV8Cache":
        """A pool of `pages` pages, all codes and scales zero."""
        torch = _torch()
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        shape = (int(pages), int(kv_heads), int(page), int(head_dim))
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2))
        ke, ve = (torch.zeros(shape[:2], dtype=torch.uint8, device=device) for _ in range(2))
        return cls(k, v, ke, ve)

    @property
    def nbytes(self) -> int:
        return 2 * self.pages * self.kv_heads * (self.page * self.head_dim + 1)


def kv8_append(qkv, cache: KV8Cache, table, pos, cos, sin, bias=None, starts=None, max_tokens: int | None = None,
               out=None):
    """Append the k and v of fused rows ``qkv`` [N, (H + 2*KV)*D] (fp32, bf16 or
    fp16; + ``bias`` fp32; rows may lie apart) to the cache and return q rotated
    [N, H, D] in qkv's type. cos, sin: fp32 [positions, D/2] (model.rope_tables).
    ``max_tokens`` bounds the rows of a sequence when ``starts`` is given.
    Arguments of the wrong shape, type or device raise ValueError."""
    return (_native or _load()).append(cache._at, cache._index, qkv, table, pos, cos, sin, bias, starts, max_tokens, out)


def kv8_attention(q, cache: KV8Cache, table, pos, starts=None, max_tokens: int | None = None, window: int = 0,
                  scale: float | None = None, out=None):
    """Attention of the rows ``q`` [N, H, D] (fp32, bf16 or fp16; rows may lie
    apart), whose k and v are already appended, over the cache: [N, H, D] in
    q's type. The row at position p sees positions p - window + 1 .. p (all up
    to p without a window); scale defaults to 1/sqrt(D). Rows that see nothing
    are 0. Arguments of the wrong shape, type or device raise ValueError."""
    return (_native or _load()).attention(cache._at, cache._index, q, table, pos, starts, max_tokens, window, scale, out)


def kv8_read(cache: KV8Cache, pages, dtype=None):
    """Keys and values of the pages ``pages`` (int32 ids on the GPU), each
    [len(pages), kv_heads, page, head_dim]: exact in bf16 and fp32; fp16 rounds
    what lies outside its range. ``dtype`` defaults to bfloat16."""
    torch = _torch()
    ids = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, None: 1}
    if dtype not in ids:
        raise ValueError("dtype must be torch.float32, bfloat16 or float16")
    return (_native or _load()).read(cache._at, cache._index, pages, ids[dtype])


class PagedKVCache:
    """The model's cache over KV8Cache pools: one pool a layer, one page table
    and one position a sequence, shared by the layers. Sequences have lengths
    of their own. Pages are handed out from a free list as sequences grow
    (``reserve``) and go back with ``release``. Table entries without a page
    are -1: a token past its sequence's pages is not stored, and recorded
    (kernels.device_status()). A released place is padding (``pos`` -1) until
    tokens are reserved for it.

    Interface of model.KVCache: ``batch``, ``capacity``, ``pos`` (int32 [batch]
    on the GPU), ``length`` (sequences of equal length), ``reset()``."""

    def __init__(self, cfg, max_len: int, batch: int = 1, page: int = 64, pages: int | None = None):
        if batch <= 0 or max_len <= 0:
            raise ValueError("a cache holds at least one sequence of one token")
        torch = _torch()
        width = -(-max_len // page)
        self.batch, self.page, self._max_len, self._positions = batch, page, max_len, cfg.max_position
        n = batch * width if pages is None else int(pages)
        self.layers = [KV8Cache.empty(n, cfg.num_kv_heads, cfg.head_dim, page) for _ in range(cfg.num_layers)]
        dev = self.layers[0].device
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
        self.pos = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.lengths = [0] * batch
        self._owned = [[] for _ in range(batch)]
        self._released = set()
        self._free = list(range(n - 1, -1, -1))

    @property
    def capacity(self) -> int:
        return self._max_len

    @property
    def nbytes(self) -> int:
        return sum(c.nbytes for c in self.layers)

    def reserve(self, tokens) -> None:
        """Pages for ``tokens[b]`` tokens of every sequence (an int: the same
        for all); raises ValueError, with nothing changed, when they do not fit.
        A released place starts again at position 0; None leaves a place as it is."""
        tokens = [tokens] * self.batch if isinstance(tokens, int) else list(tokens)
        if len(tokens) != self.batch:
            raise ValueError(f"{len(tokens)} lengths for {self.batch} sequences")
        started = [b for b in sorted(self._released) if tokens[b] is not None]
        tokens = [0 if t is None else int(t) for t in tokens]
        if max(tokens) > self._max_len:
            raise ValueError(f"KV cache full ({max(tokens)} > {self._max_len})")
        if max(tokens) > self._positions:  # the append would store nothing past the rotation tables
            raise ValueError(f"{max(tokens)} tokens pass the model's max_position ({self._positions})")
        more = [max(0, -(-t // self.page) - len(own)) for t, own in zip(tokens, self._owned)]
        if sum(more) > len(self._free):
            raise ValueError(f"KV cache out of pages ({sum(more)} needed, {len(self._free)} free)")
        for b in started:
            self.pos[b] = 0
        self._released.difference_update(started)
        if not any(more):
            return
        for own, m in zip(self._owned, more):
            own.extend(self._free.pop() for _ in range(m))
        torch = _torch()
        host = torch.full(self.table.shape, -1, dtype=torch.int32)
        for b, own in enumerate(self._owned):
            host[b, :len(own)] = torch.tensor(own, dtype=torch.int32)
        self.table.copy_(host)

    def release(self, b: int) -> None:
        """Empty sequence b and return its pages; its place is padding from here on."""
        self._free.extend(reversed(self._owned[b]))
        self._owned[b] = []
        self._released.add(b)
        self.lengths[b] = 0
        self.table[b] = -1
        self.pos[b] = -1

    @property
    def length(self) -> int:
        if len(set(self.lengths)) > 1:
            raise ValueError("the sequences have different lengths (see lengths)")
        return self.lengths[0]

    @length.setter
    def length(self, n: int) -> None:
        self.set_lengths([int(n)] * self.batch)

    def set_lengths(self, lengths) -> None:
        """Sets the sequences' lengths; a released place of length 0 stays padding."""
        self.lengths = [int(n) for n in lengths]
        self._released = {b for b in self._released if self.lengths[b] == 0}
        torch = _torch()
        self.pos.copy_(torch.tensor([-1 if b in self._released else n for b, n in enumerate(self.lengths)], dtype=torch.int32))

    def reset(self) -> None:
        """Empty every sequence (pools, table and pages stay, so a captured decode graph stays valid)."""
        self.length = 0
