"""Serving a paged KV pool: slot plans, the store of new tokens, attention.

The pool is the one the hook protects, ``[slots, 2 (K, V), kv_heads, head_dim]``
per layer, handed out in pages of ``page`` consecutive slots.  One layer step of
a serving batch is

* ``slots_plan``          once per step: pages, slots and positions of every new
                          token, from the requests' lengths alone;
* ``qk_norm_rope_store``  per layer: norm and rotate queries and keys, write
                          keys and values into the pool;
* ``prefix_attention``    per layer: every request's queries over the prefix
                          that all share and over the request's own tokens.

Lengths stay on the device and nothing synchronises, so a step can be captured
in a CUDA graph.  The slots of a plan are what ``codec.slots_gather`` and the
hook take.  All calls are stream-ordered on the current torch stream of the
tensors' device (or ``stream``, for which inputs must be ready); there is no CPU path.
"""
from __future__ import annotations

import importlib.util
import os
from typing import NamedTuple, Optional

import torch

from . import _lib

BIND_PATH = os.path.join(_lib.HERE, "lib", "gsec_torch.so")
_native = None


def _load():
    """The calls from torch tensors (csrc/bind.cpp); raises if they are not built."""
    global _native
    if _native is None:
        _lib.lib()
        if not os.path.exists(BIND_PATH):
            raise ImportError(f"gsec_torch.so not built at {BIND_PATH}; run 26mlsys-ae-ghostserve_b200/build.py")
        spec = importlib.util.spec_from_file_location("gsec_torch", BIND_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.setup(_lib.check, SlotPlan)
        _native = module
    return _native


def _on(stream: torch.cuda.Stream, first):
    """The context in which what a call allocates belongs to `stream` and what it launches goes there."""
    if not isinstance(first, torch.Tensor) or stream.device != first.device:
        raise ValueError("stream belongs to another device than the tensors")
    return torch.cuda.stream(stream)


class SlotPlan(NamedTuple):
    """Where a batch's new tokens go: one slot and position per token, request by
    request, padded with slot -1 and position 0."""
    slots: torch.Tensor       # int64 [tokens]
    positions: torch.Tensor   # int32 [tokens]
    cu: torch.Tensor          # int32 [batch + 1]: request i's tokens are cu[i]..cu[i + 1)
    lens: torch.Tensor        # int32 [batch]: tokens of each request, the new ones included
    cursor: torch.Tensor      # int32 [1]: free pages taken so far
    table: torch.Tensor       # int32 [batch, pages]: the caller's table, new pages filled in
    page: int


def slots_plan(lens: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free: torch.Tensor, cursor: torch.Tensor,
               page: int, tokens: int, base: int = 0, *, stream: Optional[torch.cuda.Stream] = None) -> SlotPlan:
    """Plan the slots of ``new[i]`` more tokens for each of 1 to 16384 requests, which has ``lens[i]``.

    ``table`` [batch, pages] holds the requests' pages and is filled in place with
    the pages the new tokens need, taken in request order from ``free[cursor:]``.
    ``tokens`` is the size of the per-token outputs (at least ``new.sum()``; a
    batch padded for a captured graph has more), ``base`` is added to every
    position (the length of a shared prefix). Too few free pages, a row longer
    than the table, more tokens than ``tokens``, a negative length or one that passes
    2^31 - 1 (cut to it, ``base`` included) give slot -1 where a token has no place,
    and set bit 17 of ``codec.device_status``."""
    if stream is not None:
        with _on(stream, lens):
            return slots_plan(lens, new, table, free, cursor, page, tokens, base)
    return (_native or _load()).slots_plan(lens, new, table, free, cursor, page, tokens, base)


def qk_norm_rope_store(qkv: torch.Tensor, pool: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                       cos: torch.Tensor, sin: torch.Tensor, heads: int, q_weight: Optional[torch.Tensor] = None,
                       k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                       out: Optional[torch.Tensor] = None, *,
                       stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Norm, rotate and store new tokens; returns the queries [tokens, heads, dim].

    ``qkv`` [tokens, (heads + 2 kv_heads) dim] holds every token's query, key and
    value heads (rows may be strided). Query and key heads with a weight [dim] are
    divided by their root mean square and multiplied by it; the first
    ``2 cos.shape[1]`` values of each then turn by row ``positions[t]`` of ``cos``
    and ``sin`` (fp32 [max_pos, rot / 2]): pairs (i, i + rot/2), or neighbours with
    ``interleaved``. Keys and values go to ``pool[slots[t]]``; a negative slot
    stores nothing, and no slot may appear twice. ``out`` may overlap neither ``qkv``
    nor the pool. Arithmetic in 32 bits, one
    rounding. A slot past the pool stores nothing and sets bit 16 of
    ``codec.device_status``; a position outside the tables leaves the row
    unrotated and sets bit 18."""
    if stream is not None:
        with _on(stream, qkv):
            return qk_norm_rope_store(qkv, pool, slots, positions, cos, sin, heads, q_weight, k_weight, eps, interleaved,
                                      out)
    return (_native or _load()).qk_norm_rope_store(qkv, pool, slots, positions, cos, sin, heads, q_weight, k_weight, eps,
                                                   interleaved, out)


def prefix_attention(q: torch.Tensor, pool: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor, table: torch.Tensor,
                     page: int, prefix: Optional[torch.Tensor] = None, prefix_len: int = 0,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False, *,
                     stream: Optional[torch.cuda.Stream] = None):
    """Attention of a ragged batch over the pool; returns [tokens, heads, dim].

    Request i's query tokens are ``q[cu[i]:cu[i + 1]]`` (n of them); token j sees
    the ``prefix_len`` keys on the pages ``prefix``, which all requests share, and
    the first ``lens[i] - n + j + 1`` of the request's ``lens[i]`` own keys on its
    row of ``table`` (``lens``, ``cu`` and ``table`` as ``slots_plan`` returns
    them, or slices of those for a part of a batch). ``q`` may be strided, but not
    broadcast; ``out`` may overlap neither ``q`` nor the pool. ``scale`` defaults to
    1 / sqrt(dim). With ``return_lse`` the second result is the log of each row's sum
    of exponentials, fp32 [tokens, heads]. A row that sees no key is 0 with lse -inf;
    rows before ``cu[0]`` and from ``cu[-1]`` on are left as they were. Keys and
    values inside a request's length must be finite (a non-finite value may spread to
    earlier tokens of the same request); slots outside all lengths may hold anything.
    A page outside the pool reads as zeros, a length past the table or a batch past
    ``q`` is cut; both set bit 19 of ``codec.device_status``.

    Scores, sums and accumulators are held in 32 bits and the result is rounded once.
    On the tensor core (bf16 and fp16 heads of up to 128 values, in sixteens) a key's
    weight is rounded to ``q``'s type as well before it meets the value; lse is of the
    unrounded weights. 1 to 16384 requests, fewer than 2^31 query heads in all and 2^30
    on a KV head, prefix and table together below 2^30 keys."""
    if stream is not None:
        with _on(stream, q):
            return prefix_attention(q, pool, cu, lens, table, page, prefix, prefix_len, scale, out, return_lse)
    return (_native or _load()).prefix_attention(q, pool, cu, lens, table, page, prefix, prefix_len, scale, out,
                                                 return_lse)
