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
There is no backward pass: where gradients are recorded, tensors that require one are refused.
The checks and the calls are native (csrc/attention_torch.cpp, built to _attention.so beside the library).
"""
from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import _native as N
from .index import _check

try:
    from . import _attention as _ops
except ImportError as e:
    raise RuntimeError("vesper_db_b200/_attention.so is missing or does not load: build it with "
                       f"`python -m vesper_db_b200.build` ({e})") from e

# The params structs of include/vesper_b200.h: every field is 8 bytes wide.
_TABLES = struct.Struct("@17q")
_ROTATE = struct.Struct("@8qd" + "q" * 27)
_PROMPT = struct.Struct("@9qd" + "q" * 15)
_SHARED = struct.Struct("@6qd" + "q" * 23)
_STRUCTS = {"page_tables": _TABLES, "norm_rotate": _ROTATE, "prompt_attention": _PROMPT,
            "shared_prefix_attention": _SHARED}


def call_device(name: str, fields, cuda_stream: int = 0) -> None:
    """vesper_<name>_device itself, for callers that hold device addresses (e.g. torch data_ptr()) instead of tensors:
    the params struct's members after struct_size, in the header's order."""
    packed = _STRUCTS[name]
    lib = N.load()
    _check(lib, getattr(lib, f"vesper_{name}_device")(packed.pack(packed.size, *fields), cuda_stream))


class PageTables(NamedTuple):
    table: torch.Tensor      # [requests, width] int32: the given table, with the new pages entered
    lengths: torch.Tensor    # [requests] int32: tokens of each request, the new ones included
    starts: torch.Tensor     # [requests + 1] int32: first new token of each request in the batch
    positions: torch.Tensor  # [total] int32
    slots: torch.Tensor      # [total] int64: place in the cache, -1 for none
    used: torch.Tensor       # [1] int32: pages that the batch takes from the free list


def page_tables(cached: torch.Tensor, fresh: torch.Tensor, free: torch.Tensor, table: torch.Tensor, page_size: int,
                total: int, base: int = 0) -> PageTables:
    """Pages, cache slots and positions of a batch's new tokens (vesper_page_tables_device).

    cached, fresh: int32 [requests], tokens that each request holds and gets; free: int32, numbers of free pages, taken
    from the front; table: int32 [requests, width], written in place; total: rows of the batch (at least the sum of
    fresh; rows past it get slot -1 and position 0); base: position of a request's first token, the length of the
    prefix that it follows.  Where free does not suffice (used > len(free)), entries and slots are -1.
    """
    return PageTables(table, *_ops.page_tables(cached, fresh, free, table, page_size, total, base))


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
    return _ops.norm_rotate(q, k, v, positions, turns, q_weight, k_weight, eps, pairs, slots, k_cache, v_cache, keep_k)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
                     starts_k: torch.Tensor | None = None, *, causal: bool = True, scale: float | None = None,
                     stats: bool = False):
    """Attention over packed prompts (vesper_prompt_attention_device).

    q [tokens, heads, head_dim], k and v [key tokens, kv_heads, head_dim]; starts int32 [requests + 1]: request b is
    rows starts[b] to starts[b + 1] of q, and of k and v unless starts_k says otherwise; neither may decrease.  causal: the last query of a
    request sees all its keys, each one before it one key less.  scale: 1 / sqrt(head_dim) by default.  Returns out
    [tokens, heads, head_dim], with stats (out, lse): the float32 [tokens, heads] log-sum-exp.  Rows that see no key
    are zero, their lse -inf.
    """
    return _ops.prompt_attention(q, k, v, starts, starts_k, causal, scale, stats)


def shared_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, prefix_pages: torch.Tensor,
                            prefix_len: int, table: torch.Tensor, lengths: torch.Tensor, *, scale: float | None = None,
                            stats: bool = False):
    """One token a request over a shared prefix and its own pages (vesper_shared_prefix_attention_device).

    q [requests, heads, head_dim]; caches [pages, page_size, kv_heads, head_dim]; prefix_pages int32: the pages that
    hold the prefix_len tokens all requests begin with; table int32 [requests, width] and lengths int32 [requests]: the
    pages and the count of each request's own tokens.  Returns out [requests, heads, head_dim], with stats (out, lse).
    """
    return _ops.shared_prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_len, table, lengths, scale, stats)
