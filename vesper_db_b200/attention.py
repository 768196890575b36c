"""Answering from retrieved passages: the operators between a search and a language model's answer.

The passages that a search returns are one long prompt which many questions share.  Its keys and values are held in a
paged cache [pages, page_size, kv_heads, head_dim]:

    page_tables              which pages and slots a batch's new tokens take, from the requests' lengths
    norm_rotate              norm of each head's query and key, position rotation, write into the cache
    prompt_attention         attention over packed prompts of different lengths
    shared_prefix_attention  one token a request, over the pages that all requests share and over its own

All take torch tensors on one CUDA device, queue their work on that device's current stream through the vesper_*_device
entry points of libvesper_c.so, synchronise nothing and can be captured in a CUDA graph.  Outputs and workspaces come
from torch's allocator in that stream's order.  Arguments that do not fit raise VesperError before any work is queued.
"""
from __future__ import annotations

import functools
import struct
from typing import NamedTuple

import torch

from . import _native as N
from .index import VesperError, _check

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}

# The params structs of include/vesper_b200.h as one packed call: every field is 8 bytes wide.
_TABLES = struct.Struct("@17q")
_ROTATE = struct.Struct("@8qd" + "q" * 27)
_PROMPT = struct.Struct("@9qd" + "q" * 15)
_SHARED = struct.Struct("@6qd" + "q" * 23)


class PageTables(NamedTuple):
    table: torch.Tensor      # [requests, width] int32: the given table, with the new pages entered
    lengths: torch.Tensor    # [requests] int32: tokens of each request, the new ones included
    starts: torch.Tensor     # [requests + 1] int32: first new token of each request in the batch
    positions: torch.Tensor  # [total] int32
    slots: torch.Tensor      # [total] int64: place in the cache, -1 for none
    used: torch.Tensor       # [1] int32: pages that the batch takes from the free list


# Entry points of the library, resolved on the first call.
_lib = None


def _entries():
    global _lib
    _lib = N.load()
    return _lib


def _refuse(why: str):
    raise VesperError(N.VESPER_ERROR_INVALID_PARAM, why)


def _wrong(t: torch.Tensor, device: torch.device, dtype: torch.dtype, name: str):
    if t.device != device:
        _refuse(f"{name} is on {t.device}, not on {device}")
    _refuse(f"{name} is {t.dtype}, {dtype} expected")


def _ints(t: torch.Tensor, device: torch.device, name: str, n: int | None = None, dtype=torch.int32) -> int:
    """Address of a contiguous vector, of whole numbers unless dtype says otherwise."""
    if t.dtype is not dtype or t.device != device:
        _wrong(t, device, dtype, name)
    if t.dim() != 1 or (n is not None and t.shape[0] != n) or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous vector" + ("" if n is None else f" of {n}"))
    return t.data_ptr()


def _cuda(t: torch.Tensor, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(f"{name} must be a CUDA tensor")
    return t.device


def _odd_strides(t: torch.Tensor, name: str) -> tuple[int, ...]:
    """All strides but the last, which must be 1; those of single-element dims do not matter."""
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        _refuse(f"{name}: the last dimension must be contiguous")
    return tuple(s if n > 1 else 8 for n, s in zip(t.shape[:-1], t.stride()))


def _heads(t: torch.Tensor, device, dtype, name: str, tokens: int | None, heads: int | None, dim: int):
    """(address, token stride, head stride) of a [tokens, heads, dim] tensor."""
    if t.dtype is not dtype or t.device != device:
        _wrong(t, device, dtype, name)
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or (tokens is not None and shape[0] != tokens) or \
            (heads is not None and shape[1] != heads):
        _refuse(f"{name} has shape {tuple(shape)}: [tokens, heads, head_dim] in line with q expected")
    a, b, c = t.stride()
    if c != 1 or a % 8 or b % 8:
        a, b = _odd_strides(t, name)
    return t.data_ptr(), a, b


def _queries(q: torch.Tensor):
    """Device, dtype code, shape and fields of q."""
    dev, dt = _cuda(q, "q"), _DTYPES.get(q.dtype)
    if dt is None or q.dim() != 3:
        _refuse("q must be bf16 or f16, [tokens, heads, head_dim]")
    t, heads, dim = q.shape
    a, b, c = q.stride()
    if c != 1 or a % 8 or b % 8:
        a, b = _odd_strides(q, "q")
    return dev, dt, t, heads, dim, (q.data_ptr(), a, b)


def _caches(k_cache, v_cache, device, dtype, kv_heads: int | None, dim: int):
    """Fields of both caches, then pages and page size."""
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dtype is not dtype or t.device != device:
            _wrong(t, device, dtype, name)
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape or shape[3] != dim or (kv_heads is not None and shape[2] != kv_heads):
        _refuse(f"k_cache {tuple(shape)} and v_cache {tuple(v_cache.shape)}: "
                "[pages, page_size, kv_heads, head_dim] in line with q expected")
    a, b, c, d = k_cache.stride()
    e, f, g, h = v_cache.stride()
    if d != 1 or h != 1 or (a | b | c | e | f | g) % 8:
        a, b, c = _odd_strides(k_cache, "k_cache")
        e, f, g = _odd_strides(v_cache, "v_cache")
    return k_cache.data_ptr(), a, b, c, v_cache.data_ptr(), e, f, g, shape[0], shape[1]


def _table(table: torch.Tensor, device, n: int):
    """Address, width and row stride of a [n, width] table."""
    if table.dtype is not torch.int32 or table.device != device:
        _wrong(table, device, torch.int32, "table")
    if table.dim() != 2 or table.shape[0] != n or (table.shape[1] > 1 and table.stride(1) != 1):
        _refuse("table must be [requests, width] with contiguous rows")
    width = table.shape[1]
    return table.data_ptr(), width, table.stride(0) if n > 1 else width


def _call(fn, params: bytes, device: torch.device) -> None:
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)  # the address of torch.cuda.current_stream(device)
    if index == torch.cuda.current_device():
        status = fn(params, stream)
    else:  # the library launches on the calling thread's device
        with torch.cuda.device(device):
            status = fn(params, stream)
    if status != N.VESPER_OK:
        _check(_lib, status)


@functools.lru_cache(maxsize=4096)
def _prompt_workspace(*sizes) -> int:
    return _lib.vesper_prompt_attention_workspace(_PROMPT.pack(*sizes, *(0,) * 15))


@functools.lru_cache(maxsize=4096)
def _shared_workspace(head: tuple, n_pages: int, page_size: int, prefix_len: int, width: int) -> int:
    return _lib.vesper_shared_prefix_attention_workspace(
        _SHARED.pack(*head, *(0,) * 11, n_pages, page_size, 0, prefix_len, 0, width, *(0,) * 6))


def page_tables(cached: torch.Tensor, fresh: torch.Tensor, free: torch.Tensor, table: torch.Tensor, page_size: int,
                total: int, base: int = 0) -> PageTables:
    """Pages, cache slots and positions of a batch's new tokens (vesper_page_tables_device).

    cached, fresh: int32 [requests], tokens that each request holds and gets; free: int32, numbers of free pages, taken
    from the front; table: int32 [requests, width], written in place; total: rows of the batch (at least the sum of
    fresh; rows past it get slot -1 and position 0); base: position of a request's first token, the length of the
    prefix that it follows.  Where free does not suffice (used > len(free)), entries and slots are -1.
    """
    dev = _cuda(cached, "cached")
    n = cached.shape[0] if cached.dim() == 1 else _refuse("cached must be a vector")
    c, f, fr = _ints(cached, dev, "cached", n), _ints(fresh, dev, "fresh", n), _ints(free, dev, "free")
    if total < 0 or page_size < 0:
        _refuse("total and page_size must not be negative")
    ints = cached.new_empty(2 * n + 2 + total)
    slots = cached.new_empty(total, dtype=torch.int64)
    p = ints.data_ptr()
    _call((_lib or _entries()).vesper_page_tables_device, _TABLES.pack(
        _TABLES.size, c, f, n, fr, free.shape[0], *_table(table, dev, n), page_size, total, base, p, p + 4 * n,
        p + 8 * n + 4, slots.data_ptr(), p + 8 * n + 4 + 4 * total), dev)
    lengths, starts, positions, used = ints.split((n, n + 1, total, 1))
    return PageTables(table, lengths, starts, positions, slots, used)


def norm_rotate(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, positions: torch.Tensor, turns: torch.Tensor,
                *, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                pairs: bool = False, slots: torch.Tensor | None = None, k_cache: torch.Tensor | None = None,
                v_cache: torch.Tensor | None = None, keep_k: bool = True):
    """Norm of each head, position rotation and cache write in one pass (vesper_norm_rotate_device).

    q [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim], bf16 or f16, slices of one projection's output
    among them; positions int32 [tokens]; turns float32 [positions, turned]: cosines, then sines, of the turned / 2
    angles; pairs: rotate neighbouring values rather than halves; weights [head_dim] of q's type, None for no norm.
    With slots (int64 [tokens], -1: skip), keys and values go to the caches.  Returns (q, k) as new contiguous tensors,
    k None without keep_k.
    """
    dev, dt, t, heads, dim, fq = _queries(q)
    fk = _heads(k, dev, q.dtype, "k", t, None, dim)
    kv = k.shape[1]
    if turns.dtype is not torch.float32 or turns.device != dev:
        _wrong(turns, dev, torch.float32, "turns")
    if turns.dim() != 2 or not turns.is_contiguous():
        _refuse("turns must be [positions, turned], contiguous")
    wq = 0 if q_weight is None else _ints(q_weight, dev, "q_weight", dim, q.dtype)
    wk = 0 if k_weight is None else _ints(k_weight, dev, "k_weight", dim, q.dtype)
    if slots is not None:
        if v is None or k_cache is None or v_cache is None:
            _refuse("slots need v, k_cache and v_cache")
        fs = _ints(slots, dev, "slots", t, torch.int64)
        fv = _heads(v, dev, q.dtype, "v", t, kv, dim)
        fc = _caches(k_cache, v_cache, dev, q.dtype, kv, dim)
    else:
        fs, fv, fc = 0, (0, 0, 0), (0,) * 10
    out_q = q.new_empty((t, heads, dim))
    out_k = q.new_empty((t, kv, dim)) if keep_k else None
    _call((_lib or _entries()).vesper_norm_rotate_device, _ROTATE.pack(
        _ROTATE.size, dt, t, heads, kv, dim, turns.shape[1], 1 if pairs else 0, eps, *fq, *fk, *fv,
        _ints(positions, dev, "positions", t), turns.data_ptr(), turns.shape[0], wq, wk, fs, *fc, out_q.data_ptr(),
        out_k.data_ptr() if keep_k else 0), dev)
    return out_q, out_k


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
                     starts_k: torch.Tensor | None = None, *, causal: bool = True, scale: float | None = None,
                     stats: bool = False):
    """Attention over packed prompts (vesper_prompt_attention_device).

    q [tokens, heads, head_dim], k and v [key tokens, kv_heads, head_dim]; starts int32 [requests + 1]: request b is
    rows starts[b] to starts[b + 1] of q, and of k and v unless starts_k says otherwise.  causal: the last query of a
    request sees all its keys, each one before it one key less.  scale: 1 / sqrt(head_dim) by default.  Returns out
    [tokens, heads, head_dim], with stats (out, lse): the float32 [tokens, heads] log-sum-exp.  Rows that see no key
    are zero, their lse -inf.
    """
    dev, dt, t, heads, dim, fq = _queries(q)
    fk = _heads(k, dev, q.dtype, "k", None, None, dim)
    n_k, kv = k.shape[0], k.shape[1]
    fv = _heads(v, dev, q.dtype, "v", n_k, kv, dim)
    s = _ints(starts, dev, "starts")
    n = starts.shape[0] - 1
    if n < 0:
        _refuse("starts must hold at least one entry")
    sk = 0 if starts_k is None else _ints(starts_k, dev, "starts_k", n + 1)
    out = q.new_empty((t, heads, dim))
    lse = q.new_empty((t, heads), dtype=torch.float32) if stats else None
    lib = _lib or _entries()
    sizes = (_PROMPT.size, dt, n, t, n_k, heads, kv, dim, 1 if causal else 0, dim ** -0.5 if scale is None else scale)
    need = _prompt_workspace(*sizes)
    space = q.new_empty(need, dtype=torch.uint8) if need else None
    _call(lib.vesper_prompt_attention_device, _PROMPT.pack(
        *sizes, *fq, *fk, *fv, s, sk, out.data_ptr(), lse.data_ptr() if stats else 0, space.data_ptr() if need else 0,
        need), dev)
    return (out, lse) if stats else out


def shared_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, prefix_pages: torch.Tensor,
                            prefix_len: int, table: torch.Tensor, lengths: torch.Tensor, *, scale: float | None = None,
                            stats: bool = False):
    """One token a request over a shared prefix and its own pages (vesper_shared_prefix_attention_device).

    q [requests, heads, head_dim]; caches [pages, page_size, kv_heads, head_dim]; prefix_pages int32: the pages that
    hold the prefix_len tokens all requests begin with; table int32 [requests, width] and lengths int32 [requests]: the
    pages and the count of each request's own tokens.  Returns out [requests, heads, head_dim], with stats (out, lse).
    """
    dev, dt, b, heads, dim, fq = _queries(q)
    fc = _caches(k_cache, v_cache, dev, q.dtype, None, dim)
    pages = _ints(prefix_pages, dev, "prefix_pages")
    if prefix_len < 0 or prefix_pages.shape[0] * fc[9] < prefix_len:
        _refuse("prefix_pages do not hold prefix_len tokens")
    ft = _table(table, dev, b)
    out = q.new_empty((b, heads, dim))
    lse = q.new_empty((b, heads), dtype=torch.float32) if stats else None
    lib = _lib or _entries()
    head = (_SHARED.size, dt, b, heads, k_cache.shape[2], dim, dim ** -0.5 if scale is None else scale)
    need = _shared_workspace(head, fc[8], fc[9], prefix_len, ft[1])
    space = q.new_empty(need, dtype=torch.uint8) if need else None
    _call(lib.vesper_shared_prefix_attention_device, _SHARED.pack(
        *head, *fq, *fc, pages, prefix_len, *ft, _ints(lengths, dev, "lengths", b), out.data_ptr(),
        lse.data_ptr() if stats else 0, space.data_ptr() if need else 0, need), dev)
    return (out, lse) if stats else out
