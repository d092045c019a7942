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
from typing import NamedTuple, Optional

import torch

from . import _lib, codec

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
_I32 = torch.int32

# A decode step makes these calls once per layer: the wrappers stay cheap (device
# numbers instead of device objects, one allocation for several small outputs,
# entry points looked up once).


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    return getattr(_lib.lib(), name)


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
        if first.get_device() != torch._C._cuda_getDevice():
            with torch.cuda.device(first.device):
                return fn(*args, **kwargs)
        return fn(*args, **kwargs)

    return call


def _stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _check(t, what: str, index: int, dtype, size: Optional[int] = None) -> int:
    """A contiguous tensor of the dtype on CUDA device `index`, of `size` elements
    where given; returns its address."""
    if not isinstance(t, torch.Tensor) or t.get_device() != index:
        raise ValueError(f"{what} must be a tensor on cuda:{index}")
    if t.dtype is not dtype or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor")
    if size is not None and t.numel() != size:
        raise ValueError(f"{what} must have {size} elements, has {t.numel()}")
    return t.data_ptr()


def _check_out(t, shape, index: int, dtype) -> int:
    at = _check(t, "out", index, dtype)
    if tuple(t.shape) != shape:
        raise ValueError(f"out must have shape {shape}, has {tuple(t.shape)}")
    return at


def _check_table(table, batch: int, index: int):
    """(address, row pitch, width) of a block table."""
    if not isinstance(table, torch.Tensor) or table.get_device() != index or table.dtype is not _I32 or \
            table.dim() != 2 or table.shape[0] != batch:
        raise ValueError(f"table must be an int32 tensor [{batch}, pages] on cuda:{index}")
    width = table.shape[1]
    pitch, one = table.stride()
    if width > 1 and one != 1 or batch > 1 and pitch < width:
        raise ValueError("the rows of table must be contiguous and must not overlap")
    return table.data_ptr(), (pitch if pitch > width else width), width


def _pool_record(pool, index: int, dtype):
    """(heads, dim, slot pitch, V plane offset) of a pool [slots, 2, heads, dim], the last two in bytes."""
    if not isinstance(pool, torch.Tensor) or pool.dim() != 4 or pool.shape[1] != 2:
        raise ValueError("pool must be a CUDA tensor [slots, 2 (K, V), heads, dim]")
    if pool.get_device() != index or pool.dtype is not dtype:
        raise ValueError(f"pool must be a {dtype} tensor on cuda:{index}")
    _, _, h, d = pool.shape
    pitch, plane, head, one = pool.stride()
    if (d > 1 and one != 1) or (h > 1 and head != d):
        raise ValueError("a pool row (pool[slot, plane]) must be contiguous")
    es = pool.element_size()
    return h, d, pitch * es, plane * es


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
    index, batch = lens.get_device(), lens.numel()
    if lens.dim() != 1:
        raise ValueError("lens must have one dimension")
    lens_at = _check(lens, "lens", index, _I32)
    new_at = _check(new, "new", index, _I32, batch)
    table_at, pitch, width = _check_table(table, batch, index)
    free_at = _check(free, "free", index, _I32)
    cursor_at = _check(cursor, "cursor", index, _I32, 1)
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    slots = torch.empty(tokens, dtype=torch.int64, device=lens.device)
    # the int32 outputs share one allocation, the per-token one in front
    positions, cu, out, taken = lens.new_empty(tokens + 2 * batch + 2).split_with_sizes((tokens, batch + 1, batch, 1))
    _lib.check(_entry("gsec_slots_plan")(
        lens_at, new_at, batch, table_at, pitch, width, free_at, free.numel(), cursor_at, int(page), int(base),
        slots.data_ptr(), positions.data_ptr(), tokens, cu.data_ptr(), out.data_ptr(), taken.data_ptr(),
        _stream(index)))
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
    index, dt = qkv.get_device(), qkv.dtype
    if dt not in _DTYPES or qkv.dim() != 2 or qkv.shape[1] > 1 and qkv.stride(1) != 1:
        raise ValueError("qkv must be a bf16, fp16 or fp32 tensor [tokens, values] with contiguous rows")
    hk, D, pitch, plane = _pool_record(pool, index, dt)
    T, values = qkv.shape
    heads = int(heads)
    if values != (heads + 2 * hk) * D:
        raise ValueError(f"qkv rows hold {values} values, {heads} + 2*{hk} heads of {D} need {(heads + 2 * hk) * D}")
    codec._slot_list(slots, qkv.device)
    if slots.numel() != T:
        raise ValueError(f"slots has {slots.numel()} entries for {T} tokens")
    if not isinstance(positions, torch.Tensor) or positions.get_device() != index or \
            positions.dtype not in (_I32, torch.int64) or not positions.is_contiguous() or positions.numel() != T:
        raise ValueError(f"positions must be a contiguous int32 or int64 tensor of {T} entries on cuda:{index}")
    cos_at = _check(cos, "cos", index, torch.float32)
    if cos.dim() != 2:
        raise ValueError("cos must have shape [positions, rot / 2]")
    sin_at = _check(sin, "sin", index, torch.float32)
    if sin.shape != cos.shape:
        raise ValueError(f"sin must have the shape of cos, {tuple(cos.shape)}")
    qw = None if q_weight is None else _check(q_weight, "q_weight", index, dt, D)
    kw = None if k_weight is None else _check(k_weight, "k_weight", index, dt, D)
    if out is None:
        out = torch.empty((T, heads, D), dtype=dt, device=qkv.device)
        out_at = out.data_ptr()
    else:
        out_at = _check_out(out, (T, heads, D), index, dt)
    row = qkv.stride(0)
    _lib.check(_entry("gsec_qk_norm_rope_store")(
        qkv.data_ptr(), (row if row > values else values) * qkv.element_size(), T, _DTYPES[dt], heads, hk, D, out_at,
        pool.data_ptr(), pitch, plane, pool.shape[0], slots.data_ptr(), slots.element_size(), positions.data_ptr(),
        positions.element_size(), cos_at, sin_at, 2 * cos.shape[1], cos.shape[0], qw, kw, float(eps),
        int(bool(interleaved)), _stream(index)))
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
    index, dt = q.get_device(), q.dtype
    if dt not in _DTYPES or q.dim() != 3 or q.shape[2] > 1 and q.stride(2) != 1:
        raise ValueError("q must be a bf16, fp16 or fp32 tensor [tokens, heads, dim] with contiguous heads")
    hk, d, pitch, plane = _pool_record(pool, index, dt)
    T, hq, D = q.shape
    if d != D or hk == 0 or hq % hk:
        raise ValueError(f"pool heads {(hk, d)} do not serve queries {(hq, D)}")
    lens_at = _check(lens, "lens", index, _I32)
    batch = lens.numel()
    cu_at = _check(cu, "cu", index, _I32, batch + 1)
    table_at, row, width = _check_table(table, batch, index)
    page, prefix_len = int(page), int(prefix_len)
    if prefix_len < 0 or page < 1:
        raise ValueError("prefix_len must not be negative, page must be positive")
    prefix_at = None
    if prefix_len:
        if prefix is None:
            raise ValueError("prefix_len without prefix pages")
        prefix_at = _check(prefix, "prefix", index, _I32)
        if prefix.numel() * page < prefix_len:
            raise ValueError(f"{prefix.numel()} prefix pages of {page} hold fewer than {prefix_len} keys")
    if out is None:
        out = torch.empty((T, hq, D), dtype=dt, device=q.device)
        out_at = out.data_ptr()
    else:
        out_at = _check_out(out, (T, hq, D), index, dt)
    lse = torch.empty((T, hq), dtype=torch.float32, device=q.device) if return_lse else None
    code = _DTYPES[dt]
    nbytes = _workspace_bytes(index, T, batch, prefix_len, code, hq, hk, D)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    es = q.element_size()
    q_row, q_head, _ = q.stride()
    _lib.check(_entry("gsec_prefix_attention")(
        q.data_ptr(), q_row * es, q_head * es, T, code, hq, hk, D, pool.data_ptr(), pitch, plane, pool.shape[0],
        cu_at, lens_at, batch, table_at, row, width, page, prefix_at, prefix_len,
        D ** -0.5 if scale is None else float(scale), out_at, lse.data_ptr() if return_lse else None,
        ws.data_ptr() if nbytes else None, nbytes, _stream(index)))
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(index, tokens, batch, prefix_len, dtype, hq, hk, dim) -> int:
    """Asked once per shape and device (its size goes by the number of SMs)."""
    out = _lib.C.c_int64(0)
    _lib.call("gsec_prefix_attention_workspace", tokens, batch, prefix_len, dtype, hq, hk, dim, _lib.C.byref(out))
    return int(out.value)
