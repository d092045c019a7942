"""CPU checks of the KV-pool serving operators: refusals by the C entries, before
anything could be launched, and by the Python wrappers."""
from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import pkg

P = ctypes.c_void_p
A = [P(0x10000 * (i + 1)) for i in range(16)]  # never used: every call fails before a launch


def plan_args(**kw):
    d = dict(lens=A[0], new=A[1], batch=4, table=A[2], pitch=8, width=8, free=A[3], nfree=9, cursor=A[4], page=16,
             base=0, slots=A[5], positions=A[6], capacity=64, cu=A[7], lens_out=A[8], cursor_out=A[9], stream=None)
    d.update(kw)
    return list(d.values())


def store_args(**kw):
    d = dict(qkv=A[0], pitch=12 * 128 * 2, tokens=4, dtype=0, hq=8, hk=2, dim=128, q_out=A[1], pool=A[2], slot_pitch=1024,
             plane=512, rows=100, slots=A[3], slot_bytes=8, positions=A[4], position_bytes=4, cos=A[5], sin=A[6],
             rot=128, max_pos=64, qw=None, kw=None, eps=1e-5, interleaved=0, stream=None)
    d.update(kw)
    return list(d.values())


def attn_args(**kw):
    d = dict(q=A[0], q_pitch=2048, q_head=256, tokens=4, dtype=0, hq=8, hk=2, dim=128, pool=A[1], slot_pitch=1024,
             plane=512, rows=100, cu=A[2], lens=A[3], batch=4, table=A[4], pitch=8, width=8, page=16, prefix=None,
             prefix_len=0, scale=0.1, out=A[5], lse=None, ws=A[6], ws_bytes=1 << 40, stream=None)
    d.update(kw)
    return list(d.values())


@pytest.mark.parametrize("bad,match", [
    (dict(batch=0), "batch"), (dict(batch=16385), "batch"), (dict(lens=None), "null"), (dict(table=None), "null"),
    (dict(cursor=None), "null"), (dict(free=None), "null"), (dict(slots=None), "null"), (dict(page=0), "page"),
    (dict(pitch=7), "table_pitch"), (dict(width=0), "width"), (dict(nfree=-1), "nfree"), (dict(capacity=-1), "capacity"),
    (dict(capacity=1 << 31), "capacity"), (dict(slots=P(0x50008)), "aligned"), (dict(lens_out=A[0]), "inputs"),
    (dict(cursor_out=A[4]), "inputs"),
])
def test_slots_plan_refusals(bad, match):
    with pytest.raises(ValueError, match=match):
        pkg("_lib").call("gsec_slots_plan", *plan_args(**bad))


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=3), "dtype"), (dict(hq=7), "multiple"), (dict(hk=0), "multiple"), (dict(dim=12), "16-byte"),
    (dict(dim=264), "256"), (dict(pool=None), "pool"), (dict(pool=P(0x30008)), "aligned"), (dict(plane=0), "record"),
    (dict(plane=520), "aligned"), (dict(slot_pitch=256, plane=512), "record"), (dict(plane=768), "overlap"),
    (dict(tokens=-1), "tokens"), (dict(qkv=None), "null"), (dict(q_out=None), "null"), (dict(slots=None), "null"),
    (dict(slot_bytes=2), "slot_bytes"), (dict(position_bytes=1), "position_bytes"), (dict(rot=130), "rot"),
    (dict(rot=8), "rot"), (dict(cos=None), "null"), (dict(qkv=P(0x10004)), "aligned"), (dict(pitch=3064), "aligned"),
    (dict(pitch=1536), "overlap"), (dict(qw=P(0x10002)), "aligned"),
    (dict(dtype=2, dim=256, slot_pitch=4096, plane=2048, pitch=1 << 20), "512"),
])
def test_qk_norm_rope_store_refusals(bad, match):
    with pytest.raises(ValueError, match=match):
        pkg("_lib").call("gsec_qk_norm_rope_store", *store_args(**bad))


@pytest.mark.parametrize("bad,match", [
    (dict(dtype=-1), "dtype"), (dict(hq=9), "multiple"), (dict(dim=4), "16-byte"), (dict(plane=256), "record"),
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 30), "2\\^31"), (dict(batch=0), "batch"), (dict(batch=16385), "batch"),
    (dict(rows=0), "pool_rows"), (dict(rows=1 << 31), "pool_rows"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(cu=None), "null"), (dict(lens=None), "null"), (dict(prefix_len=5), "null"), (dict(table=None), "table"),
    (dict(pitch=7), "table"), (dict(page=0), "page"), (dict(prefix=A[7], prefix_len=1 << 30), "2\\^30"),
    (dict(prefix=A[7], prefix_len=-1), "keys"), (dict(q_head=264), "aligned"), (dict(q=P(0x10008)), "aligned"),
    (dict(q_head=0), "strides"), (dict(q_pitch=0), "strides"), (dict(q_pitch=1 << 40), "strides"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(ws=None), "workspace"),
    (dict(ws_bytes=16), "workspace"), (dict(ws=P(0x70008)), "workspace"),
])
def test_prefix_attention_refusals(bad, match):
    with pytest.raises(ValueError, match=match):
        pkg("_lib").call("gsec_prefix_attention", *attn_args(**bad))


def test_prefix_attention_of_nothing_is_nothing():
    pkg("_lib").call("gsec_prefix_attention", *attn_args(tokens=0, q=None, out=None))
    pkg("_lib").call("gsec_qk_norm_rope_store", *store_args(tokens=0, qkv=None, q_out=None, slots=None, positions=None))


def test_workspace_size():
    L = pkg("_lib")
    n = ctypes.c_int64(-1)
    L.call("gsec_prefix_attention_workspace", 64, 64, 4096, 0, 32, 8, 128, ctypes.byref(n))
    assert n.value >= 2 * 64 * 32 * 128 * 4  # both parts of every row
    L.call("gsec_prefix_attention_workspace", 64, 64, 4096, 2, 32, 8, 128, ctypes.byref(n))
    assert n.value == 0  # fp32 goes row by row
    with pytest.raises(ValueError):
        L.call("gsec_prefix_attention_workspace", 64, 64, 4096, 0, 30, 8, 128, ctypes.byref(n))


def test_wrappers_need_cuda_tensors():
    k = pkg("kvpool")
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="lens must be a CUDA tensor"):
        k.slots_plan(i, i, i[None], i, i[:1], 16, 4)
    with pytest.raises(ValueError, match="qkv must be a CUDA tensor"):
        k.qk_norm_rope_store(torch.zeros(4, 64), None, i, i, None, None, 2)
    with pytest.raises(ValueError, match="q must be a CUDA tensor"):
        k.prefix_attention(q=torch.zeros(4, 2, 64), pool=None, cu=i, lens=i, table=i[None], page=16)


def test_prefix_attention_refuses_more_rows_than_it_counts():
    with pytest.raises(ValueError, match="too many"):
        pkg("_lib").call("gsec_prefix_attention", *attn_args(tokens=1 << 27, hq=8, hk=1, slot_pitch=512, plane=256))
