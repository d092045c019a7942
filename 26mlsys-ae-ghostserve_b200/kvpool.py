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

import functools
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib, codec

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def _on_stream(fn):
    """Run fn on ``stream`` and the device of its first tensor: what it allocates
    belongs to that stream, what it launches goes there."""

    name = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, stream: Optional[torch.cuda.Stream] = None, **kwargs):
        first = args[0] if args else kwargs.get(name)
        if not isinstance(first, torch.Tensor) or not first.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if stream is not None:
            if stream.device != first.device:
                raise ValueError("stream belongs to another device than the tensors")
            with torch.cuda.stream(stream):
                return fn(*args, **kwargs)
        if first.device.index != torch.cuda.current_device():
            with torch.cuda.device(first.device):
                return fn(*args, **kwargs)
        return fn(*args, **kwargs)

    return call


def _check(t, what: str, device, dtype, shape=None) -> None:
    """A contiguous tensor of the dtype on the device, of the shape where given."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise ValueError(f"{what} must be a tensor on {device}")
    if t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {tuple(shape)}, has {tuple(t.shape)}")


def _check_table(table, batch: int, device) -> None:
    if not isinstance(table, torch.Tensor) or table.device != device or table.dtype != torch.int32 or \
            table.dim() != 2 or table.shape[0] != batch:
        raise ValueError(f"table must be an int32 tensor [{batch}, pages] on {device}")
    if table.shape[1] > 1 and table.stride(1) != 1 or batch > 1 and table.stride(0) < table.shape[1]:
        raise ValueError("the rows of table must be contiguous and must not overlap")


def _pool_record(pool, device, dtype):
    """(slot pitch, V plane offset) in bytes of a pool [slots, 2, heads, dim]."""
    if not isinstance(pool, torch.Tensor) or pool.dim() != 4 or pool.shape[1] != 2:
        raise ValueError("pool must be a CUDA tensor [slots, 2 (K, V), heads, dim]")
    if pool.device != device or pool.dtype != dtype:
        raise ValueError(f"pool must be a {dtype} tensor on {device}")
    h, d = pool.shape[2], pool.shape[3]
    s = pool.stride()
    if (d > 1 and s[3] != 1) or (h > 1 and s[2] != d):
        raise ValueError("a pool row (pool[slot, plane]) must be contiguous")
    es = pool.element_size()
    return s[0] * es, s[1] * es


@dataclass(frozen=True)
class SlotPlan:
    """Where a batch's new tokens go: one slot and position per token, request by
    request, padded with slot -1 and position 0."""
    slots: torch.Tensor       # int64 [tokens]
    positions: torch.Tensor   # int32 [tokens]
    cu: torch.Tensor          # int32 [batch + 1]: request i's tokens are cu[i]..cu[i + 1)
    lens: torch.Tensor        # int32 [batch]: tokens of each request, the new ones included
    cursor: torch.Tensor      # int32 [1]: free pages taken so far
    table: torch.Tensor       # int32 [batch, pages]: the caller's table, new pages filled in
    page: int


@_on_stream
def slots_plan(lens: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free: torch.Tensor, cursor: torch.Tensor,
               page: int, tokens: int, base: int = 0) -> SlotPlan:
    """Plan the slots of ``new[i]`` more tokens for each request that has ``lens[i]``.

    ``table`` [batch, pages] holds the requests' pages and is filled in place with
    the pages the new tokens need, taken in request order from ``free[cursor:]``.
    ``tokens`` is the size of the per-token outputs (at least ``new.sum()``; a
    batch padded for a captured graph has more), ``base`` is added to every
    position (the length of a shared prefix). Too few free pages, a row longer
    than the table, more tokens than ``tokens`` or a negative length give slot -1
    where a token has no place, and set bit 17 of ``codec.device_status``."""
    dev = lens.device
    batch = lens.numel()
    _check(lens, "lens", dev, torch.int32, (batch,))
    _check(new, "new", dev, torch.int32, (batch,))
    _check_table(table, batch, dev)
    _check(free, "free", dev, torch.int32, (free.numel(),) if isinstance(free, torch.Tensor) else None)
    _check(cursor, "cursor", dev, torch.int32, (1,))
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    slots = torch.empty(tokens, dtype=torch.int64, device=dev)
    # the four int32 outputs share one allocation; positions first, so that it is aligned
    n = -(-tokens // 4) * 4
    small = torch.empty(n + 2 * batch + 2, dtype=torch.int32, device=dev)
    positions, cu = small[:tokens], small[n:n + batch + 1]
    out, taken = small[n + batch + 1:n + 2 * batch + 1], small[n + 2 * batch + 1:]
    _lib.call("gsec_slots_plan", lens.data_ptr(), new.data_ptr(), batch, table.data_ptr(),
              max(table.stride(0), table.shape[1]), table.shape[1], free.data_ptr(), free.numel(), cursor.data_ptr(),
              int(page), int(base), slots.data_ptr(), positions.data_ptr(), tokens, cu.data_ptr(), out.data_ptr(),
              taken.data_ptr(), torch.cuda.current_stream().cuda_stream)
    return SlotPlan(slots, positions, cu, out, taken, table, int(page))


@_on_stream
def qk_norm_rope_store(qkv: torch.Tensor, pool: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                       cos: torch.Tensor, sin: torch.Tensor, heads: int, q_weight: Optional[torch.Tensor] = None,
                       k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Norm, rotate and store new tokens; returns the queries [tokens, heads, dim].

    ``qkv`` [tokens, (heads + 2 kv_heads) dim] holds every token's query, key and
    value heads (rows may be strided). Query and key heads with a weight [dim] are
    divided by their root mean square and multiplied by it; the first
    ``2 cos.shape[1]`` values of each then turn by row ``positions[t]`` of ``cos``
    and ``sin`` (fp32 [max_pos, rot / 2]): pairs (i, i + rot/2), or neighbours with
    ``interleaved``. Keys and values go to ``pool[slots[t]]``; a negative slot
    stores nothing, and no slot may appear twice. Arithmetic in 32 bits, one
    rounding. A slot past the pool stores nothing and sets bit 16 of
    ``codec.device_status``; a position outside the tables leaves the row
    unrotated and sets bit 18."""
    dev, dt = qkv.device, qkv.dtype
    if dt not in _DTYPES or qkv.dim() != 2 or qkv.shape[1] > 1 and qkv.stride(1) != 1:
        raise ValueError("qkv must be a bf16, fp16 or fp32 tensor [tokens, values] with contiguous rows")
    pitch, plane = _pool_record(pool, dev, dt)
    T, hk, D = qkv.shape[0], pool.shape[2], pool.shape[3]
    heads = int(heads)
    if qkv.shape[1] != (heads + 2 * hk) * D:
        raise ValueError(f"qkv rows hold {qkv.shape[1]} values, {heads} + 2*{hk} heads of {D} need "
                         f"{(heads + 2 * hk) * D}")
    codec._slot_list(slots, dev)
    if slots.numel() != T:
        raise ValueError(f"slots has {slots.numel()} entries for {T} tokens")
    if not isinstance(positions, torch.Tensor) or positions.device != dev or \
            positions.dtype not in (torch.int32, torch.int64) or not positions.is_contiguous() or \
            positions.numel() != T:
        raise ValueError(f"positions must be a contiguous int32 or int64 tensor of {T} entries on {dev}")
    _check(cos, "cos", dev, torch.float32)
    if cos.dim() != 2:
        raise ValueError("cos must have shape [positions, rot / 2]")
    _check(sin, "sin", dev, torch.float32, cos.shape)
    for w, what in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _check(w, what, dev, dt, (D,))
    if out is None:
        out = torch.empty(T, heads, D, dtype=dt, device=dev)
    else:
        _check(out, "out", dev, dt, (T, heads, D))
    _lib.call("gsec_qk_norm_rope_store", qkv.data_ptr(), max(qkv.stride(0), qkv.shape[1]) * qkv.element_size(), T,
              _DTYPES[dt], heads, hk, D, out.data_ptr(), pool.data_ptr(), pitch, plane, pool.shape[0],
              slots.data_ptr(), slots.element_size(), positions.data_ptr(), positions.element_size(), cos.data_ptr(),
              sin.data_ptr(), 2 * cos.shape[1], cos.shape[0], None if q_weight is None else q_weight.data_ptr(),
              None if k_weight is None else k_weight.data_ptr(), float(eps), int(bool(interleaved)),
              torch.cuda.current_stream().cuda_stream)
    return out


@_on_stream
def prefix_attention(q: torch.Tensor, pool: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor, table: torch.Tensor,
                     page: int, prefix: Optional[torch.Tensor] = None, prefix_len: int = 0,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of a ragged batch over the pool; returns [tokens, heads, dim].

    Request i's query tokens are ``q[cu[i]:cu[i + 1]]`` (n of them); token j sees
    the ``prefix_len`` keys on the pages ``prefix``, which all requests share, and
    the first ``lens[i] - n + j + 1`` of the request's ``lens[i]`` own keys on its
    row of ``table`` (``lens``, ``cu`` and ``table`` as ``slots_plan`` returns
    them). ``scale`` defaults to 1 / sqrt(dim). With ``return_lse`` the second
    result is the log of each row's sum of exponentials, fp32 [tokens, heads]. A
    row that sees no key is 0 with lse -inf; rows from ``cu[-1]`` on are left as
    they were. Keys and values inside a request's length must be finite (a
    non-finite value may spread to earlier tokens of the same request); slots outside
    all lengths may hold anything. A page outside the pool reads as zeros and a
    length past the table is cut; both set bit 19 of ``codec.device_status``."""
    dev, dt = q.device, q.dtype
    if dt not in _DTYPES or q.dim() != 3 or q.shape[2] > 1 and q.stride(2) != 1:
        raise ValueError("q must be a bf16, fp16 or fp32 tensor [tokens, heads, dim] with contiguous heads")
    pitch, plane = _pool_record(pool, dev, dt)
    T, hq, D = q.shape
    hk = pool.shape[2]
    if pool.shape[3] != D or hk == 0 or hq % hk:
        raise ValueError(f"pool heads {tuple(pool.shape[2:])} do not serve queries {tuple(q.shape[1:])}")
    batch = lens.numel() if isinstance(lens, torch.Tensor) else -1
    _check(lens, "lens", dev, torch.int32, (batch,))
    _check(cu, "cu", dev, torch.int32, (batch + 1,))
    _check_table(table, batch, dev)
    page, prefix_len = int(page), int(prefix_len)
    if prefix_len < 0 or page < 1:
        raise ValueError("prefix_len must not be negative, page must be positive")
    if prefix_len:
        if prefix is None:
            raise ValueError("prefix_len without prefix pages")
        _check(prefix, "prefix", dev, torch.int32)
        if prefix.numel() * page < prefix_len:
            raise ValueError(f"{prefix.numel()} prefix pages of {page} hold fewer than {prefix_len} keys")
    if out is None:
        out = torch.empty(T, hq, D, dtype=dt, device=dev)
    else:
        _check(out, "out", dev, dt, (T, hq, D))
    lse = torch.empty(T, hq, dtype=torch.float32, device=dev) if return_lse else None
    nbytes = _workspace_bytes(T, batch, prefix_len, _DTYPES[dt], hq, hk, D)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    es = q.element_size()
    _lib.call("gsec_prefix_attention", q.data_ptr(), q.stride(0) * es, q.stride(1) * es, T, _DTYPES[dt], hq, hk, D,
              pool.data_ptr(), pitch, plane, pool.shape[0], cu.data_ptr(), lens.data_ptr(), batch, table.data_ptr(),
              max(table.stride(0), table.shape[1]), table.shape[1], page, prefix.data_ptr() if prefix_len else None,
              prefix_len, D ** -0.5 if scale is None else float(scale), out.data_ptr(),
              lse.data_ptr() if return_lse else None, ws.data_ptr() if nbytes else None, nbytes,
              torch.cuda.current_stream().cuda_stream)
    return (out, lse) if return_lse else out


def _workspace_bytes(tokens, batch, prefix_len, dtype, hq, hk, dim) -> int:
    out = _lib.C.c_int64(0)
    _lib.call("gsec_prefix_attention_workspace", tokens, batch, prefix_len, dtype, hq, hk, dim, _lib.C.byref(out))
    return int(out.value)
