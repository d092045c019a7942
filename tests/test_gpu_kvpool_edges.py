"""KV-pool serving operators at the calls that the main tests leave out."""
from __future__ import annotations

import math

import pytest
import torch

import kvpool_ref as ref
from conftest import pkg
from test_gpu_kvpool import BF, F4, HF, attn_case, kv

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device_status_clean():
    """Tests that flag something on purpose clear it themselves."""
    yield
    assert pkg("codec").device_status(clear=True) == 0


def check_rows(o, lse, c, on, **kw):
    """The rows `on` [tokens, heads] of (o, lse) against the plain form."""
    want, wl, to, tl = ref.attention(**c, **kw)
    off = ((o.double() - want).abs() <= to).all(-1) | ~on
    assert bool(off.all())
    empty = wl == -math.inf
    assert bool((((lse.double() - wl).abs() <= tl) | empty | ~on).all())
    assert bool(((lse == -math.inf) == empty)[on].all())


# ---------------------------------------------------------- not a number ------
ROWS_AND_TILES = [(F4, 8, 2, 64), (F4, 1, 1, 4), (BF, 4, 2, 256), (HF, 6, 1, 136), (BF, 8, 2, 8), (BF, 8, 2, 128),
                  (HF, 6, 2, 64)]


@pytest.mark.parametrize("dtype,hq,hk,D", ROWS_AND_TILES)
@pytest.mark.parametrize("q_lens,lens,P", [([1], [1], 0), ([1, 3, 0, 20], [7, 300, 5, 20], 0),
                                           ([1, 1, 1, 1, 40], [5, 1, 128, 257, 300], 385)])
def test_a_query_that_is_not_a_number_stays_so(dtype, hq, hk, D, q_lens, lens, P):
    """All values of one head, or one value of another: the row is not a number throughout, its neighbours are as
    without it."""
    c = attn_case(q_lens, lens, P, 16, hq, hk, D, dtype)
    T = c["q"].shape[0]
    bad = torch.zeros(T, hq, dtype=torch.bool, device="cuda")
    bad[T - 1, 0] = bad[T // 2, hq - 1] = True
    q = c["q"].clone()
    q[T // 2, hq - 1, D // 2] = math.nan
    q[T - 1, 0] = math.nan
    o, lse = kv().prefix_attention(**dict(c, q=q), return_lse=True)
    assert bool(torch.isnan(o[bad]).all()) and bool(torch.isnan(lse[bad]).all())
    check_rows(o, lse, c, ~bad)


@pytest.mark.parametrize("dtype,hq,hk,D", ROWS_AND_TILES)
def test_a_key_or_value_that_is_not_a_number_shows(dtype, hq, hk, D):
    """Every row that sees the key is not a number; a value spoils its own column. Other requests and other KV heads
    are as without it."""
    c = attn_case([1, 2, 1], [3, 40, 200], 0, 16, hq, hk, D, dtype, garbage=0.0)
    group = hq // hk
    slot = int(c["table"][2, 4]) * 16 + 5
    on = torch.ones(4, hq, dtype=torch.bool, device="cuda")
    on[3, :group] = False
    pool = c["pool"].clone()
    pool[slot, 0, 0, D - 1] = math.nan
    o, lse = kv().prefix_attention(**dict(c, pool=pool), return_lse=True)
    assert bool(torch.isnan(o[~on]).all()) and bool(torch.isnan(lse[~on]).all())
    check_rows(o, lse, c, on)
    pool = c["pool"].clone()
    pool[slot, 1, 0, D - 1] = math.nan
    o, lse = kv().prefix_attention(**dict(c, pool=pool), return_lse=True)
    assert bool(torch.isnan(o[3, :group, D - 1]).all()) and not bool(torch.isnan(o[3, :group, :D - 1]).any())
    check_rows(o, lse, c, on)


def test_a_scale_next_to_nothing_keeps_what_is_not_a_number():
    c = attn_case([1, 20], [70, 20], 40, 16, 4, 2, 64, BF)
    q = c["q"].clone()
    q[3, 1] = math.nan
    o, lse = kv().prefix_attention(**dict(c, q=q), scale=1e-30, return_lse=True)
    on = torch.ones(21, 4, dtype=torch.bool, device="cuda")
    on[3, 1] = False
    assert bool(torch.isnan(o[~on]).all()) and bool(torch.isnan(lse[~on]).all())
    check_rows(o, lse, c, on, scale=1e-30)


# ------------------------------------------------------- parts of a batch -----
@pytest.mark.parametrize("dtype,hq,hk,D", [(BF, 8, 2, 128), (HF, 4, 4, 64), (F4, 4, 2, 64), (BF, 4, 2, 256)])
@pytest.mark.parametrize("P", [0, 150, 2000])
@pytest.mark.parametrize("q_lens,lens", [([1, 4, 2, 0, 1, 3], [9, 30, 70, 4, 20, 33]),
                                         ([130, 1, 140, 300], [200, 5, 140, 301])])
def test_parts_of_a_batch_share_queries_and_out(dtype, hq, hk, D, P, q_lens, lens):
    """One call for the first two requests and one for the others, on slices of cu, lens and table: each writes its own
    requests' rows and no others."""
    c = attn_case(q_lens, lens, P, 16, hq, hk, D, dtype, pad=3)
    n = sum(q_lens)
    out = torch.full_like(c["q"], 7.0)
    for part in (slice(0, 2), slice(2, None)):
        cu = c["cu"][part.start:(part.stop + 1) if part.stop else None]
        before = out.clone()
        got, lse = kv().prefix_attention(**dict(c, cu=cu, lens=c["lens"][part], table=c["table"][part]), out=out,
                                         return_lse=True)
        a, b = int(cu[0]), int(cu[-1])
        assert torch.equal(out[:a], before[:a]) and torch.equal(out[b:], before[b:])
        want, wl, to, tl = ref.attention(**dict(c, q=c["q"][:n]))
        assert bool(((got[a:b].double() - want[a:b]).abs() <= to[a:b]).all())
        seen = wl[a:b] > -math.inf
        assert bool((((lse[a:b].double() - wl[a:b]).abs() <= tl[a:b]) | ~seen).all())


# ------------------------------------------- lengths that do not fit, flagged ---
@pytest.mark.parametrize("dtype,hq,hk,D", [(BF, 4, 2, 128), (F4, 4, 2, 64), (BF, 4, 2, 256)])
@pytest.mark.parametrize("P", [0, 33])
def test_lengths_that_do_not_fit_are_cut_and_flagged(dtype, hq, hk, D, P):
    """With and without the tensor core: the same cuts, the same bit."""
    c = attn_case([1, 4, 2], [40, 20, 30], P, 16, hq, hk, D, dtype, garbage=0.0)
    status = pkg("codec").device_status
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    room = c["table"].shape[1] * 16
    c["table"] = torch.where(c["table"] < 0, 0, c["table"])
    cases = [  # what is given, what is answered
        (dict(cu=i32([0, 1, 5, 9])), dict(cu=i32([0, 1, 5, 7]))),       # the batch past the queries
        (dict(cu=i32([0, 1, 9, 9])), dict(cu=i32([0, 1, 7, 7]))),
        (dict(lens=i32([40, -3, 30])), dict(lens=i32([40, 0, 30]))),    # a negative length
        (dict(lens=i32([40, 20, room + 1])), dict(lens=i32([40, 20, room]))),
        (dict(cu=i32([0, 1, 1, 7]), lens=i32([40, room + 9, 30])),      # of a request without queries
         dict(cu=i32([0, 1, 1, 7]), lens=i32([40, room, 30]))),
    ]
    for given, cut in cases:
        want = kv().prefix_attention(**dict(c, **cut), return_lse=True)
        assert status() == 0
        got = kv().prefix_attention(**dict(c, **given), return_lse=True)
        assert status(clear=True) == 1 << 19
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ----------------------------------------------------- lengths of the work -----
@pytest.mark.parametrize("T,hq,hk", [(400_000, 32, 8), (20_000, 1024, 1), (700_000, 4, 4)])
@pytest.mark.parametrize("P", [0, 3])
def test_many_queries_on_few_keys(T, hq, hk, P):
    """All but the last 16 tokens see nothing, or the prefix alone."""
    c = attn_case([16], [16], P, 16, hq, hk, 16, BF, garbage=0.0)
    few = c["q"]
    c["q"] = torch.zeros(T, hq, 16, device="cuda", dtype=BF)
    c["q"][-16:] = few
    c["q"][:5] = few[:5]
    c["cu"] = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    o, lse = kv().prefix_attention(**c, out=torch.full_like(c["q"], 7.0), return_lse=True)
    want = attn_case([16], [16], P, 16, hq, hk, 16, BF, garbage=0.0)
    check_rows(o[-16:], lse[-16:], want, torch.ones(16, hq, dtype=torch.bool, device="cuda"))
    # zero queries weigh the prefix's values alike
    first = dict(want, lens=want["lens"] * 0, cu=torch.tensor([0, 5], dtype=torch.int32, device="cuda"), q=few[:5])
    check_rows(o[:5], lse[:5], first, torch.ones(5, hq, dtype=torch.bool, device="cuda"))
    rest, ls = o[5:-16], lse[5:-16]
    assert bool((rest == rest[:1]).all()) and bool((ls == ls[:1]).all())
    if P == 0:
        assert bool((rest[0] == 0).all()) and bool((ls[0] == -math.inf).all())
    else:  # rounding of P and of the result, and of lse: log2, a product
        slots = (c["prefix"].long()[:, None] * 16 + torch.arange(16, device="cuda")).reshape(-1)[:P]
        mean = c["pool"][slots, 1].double().mean(0).repeat_interleave(hq // hk, 0)
        big = c["pool"][slots, 1].double().abs().mean(0).repeat_interleave(hq // hk, 0)
        assert bool(((rest[0].double() - mean).abs() <= 2 * ref.half_step(BF) * big).all())
        assert bool(((ls[0].double() - math.log(P)).abs() <= 8 * 2.0 ** -24 * math.log(P)).all())


@pytest.mark.parametrize("B,hk,tokens,page", [(2048, 8, 262144, 64), (16384, 8, 32768, 16), (300, 8, 1 << 29, 1 << 17)])
def test_short_lengths_in_wide_tables(B, hk, tokens, page):
    """What a table could hold is no work: many requests with tables for long contexts are served, with the same bits
    as from narrow tables."""
    g = torch.Generator(device="cuda").manual_seed(B)
    small = min(page, 64)
    pool = torch.randn(128 * small, 2, hk, 16, generator=g, device="cuda").to(BF)
    lens = torch.randint(1, 40, (B,), generator=g, device="cuda", dtype=torch.int32)
    cu = torch.arange(B + 1, device="cuda", dtype=torch.int32)
    q = torch.randn(B, hk, 16, generator=g, device="cuda").to(BF)
    width = tokens // page
    first = torch.randint(0, 128 * small // page if page <= 64 else 1, (B, 1), generator=g, device="cuda").int()
    wide = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    need = -(-40 // page)
    wide[:, :need] = (first + torch.arange(need, device="cuda", dtype=torch.int32)) % max(1, 128 * small // page)
    got = kv().prefix_attention(q, pool, cu, lens, wide, page, return_lse=True)
    want = kv().prefix_attention(q, pool, cu, lens, wide[:, :need].contiguous(), page, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check_rows(got[0][:50], got[1][:50],
               dict(q=q[:50], pool=pool, cu=cu[:51], lens=lens[:50], table=wide[:50, :need], page=page, prefix=None,
                    prefix_len=0), torch.ones(50, hk, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("q_lens,pad", [([512] + [1] * 15, 0), ([40] + [1] * 15, 0), ([1] * 15 + [40], 1500),
                                        ([1] * 8 + [300] + [1] * 8, 3)])
def test_a_chunk_among_decodes(q_lens, pad):
    """Stacked over the prefix, or each request by itself, as the query count (padding included) has it."""
    lens = [n + 37 * i for i, n in enumerate(q_lens)]
    c = attn_case(q_lens, lens, 700, 16, 8, 2, 128, BF, pad=pad)
    n = sum(q_lens)
    o, lse = kv().prefix_attention(**c, return_lse=True)
    check_rows(o[:n], lse[:n], dict(c, q=c["q"][:n]), torch.ones(n, 8, dtype=torch.bool, device="cuda"))


def test_slots_plan_of_lengths_at_the_end_of_32_bits():
    status, top = pkg("codec").device_status, 2 ** 31 - 1
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def plan(lens, new, page, tokens, base=0, width=2):
        table = i32([[3, 5, 1, 2][:width]] * len(lens))
        p = kv().slots_plan(i32(lens), i32(new), table, i32([7, 8, 9]), i32([0]), page, tokens, base=base)
        assert table.tolist() == [[3, 5, 1, 2][:width]] * len(lens)
        return [x.tolist() for x in (p.slots, p.positions, p.cu, p.lens, p.cursor)]

    # the last length that exists
    assert plan([top - 1], [1], 1 << 30, 1) == [[5 * 2 ** 30 + 2 ** 30 - 2], [top - 1], [0, 1], [top], [0]]
    assert plan([top - 6], [1], 1 << 30, 1, base=5) == [[5 * 2 ** 30 + 2 ** 30 - 7], [top - 1], [0, 1], [top - 5], [0]]
    assert plan([top], [0], 1 << 30, 1) == [[-1], [0], [0, 0], [top], [0]]
    assert status() == 0
    # past it: cut and flagged
    assert plan([top], [1], 1 << 30, 1) == [[-1], [0], [0, 0], [top], [0]]
    assert status() == 1 << 17
    assert plan([top - 4], [3], 1 << 30, 3, base=3) == [[5 * 2 ** 30 + 2 ** 30 - 5, -1, -1], [top - 1, 0, 0], [0, 1],
                                                        [top - 3], [0]]
    assert status() == 1 << 17
    assert plan([top, 1], [top, 1], 16, 1, width=4) == [[3 * 16 + 1], [1], [0, 0, 1], [top, 2], [0]]
    assert status() == 1 << 17


# ------------------------------------------------------ errors of the calls -----
def test_an_allocation_that_fails_is_an_out_of_memory_error():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (i32([0]), i32([1]), i32([[-1]]), i32([0]), i32([0]), 16)
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.05)  # of 180 GB: below the 12 bytes of each of 2^30 tokens
    try:
        with pytest.raises(torch.OutOfMemoryError):
            kv().slots_plan(*args, 1 << 30)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert kv().slots_plan(*args, 1).slots.tolist() == [0]


def test_forward_mode_tangents_and_angle_gradients_are_refused():
    """The operators have neither a forward nor a backward derivative: none is dropped in silence."""
    import torch.autograd.forward_ad as fwd
    from test_gpu_kvpool import store_case
    c = attn_case([1, 2], [20, 30], 16, 16, 4, 2, 64, BF)
    qkv, pool, slots, positions, cos, sin, w = store_case(9, 4, 2, 64, 64, BF, True)
    base = dict(qkv=qkv, pool=pool, slots=slots, positions=positions, cos=cos, sin=sin, heads=4, q_weight=w[0],
                k_weight=w[1])
    for name in ("cos", "sin"):
        with pytest.raises(ValueError, match="gradient"):
            kv().qk_norm_rope_store(**dict(base, **{name: base[name].clone().requires_grad_()}))
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for name in ("q", "pool"):
            with pytest.raises(ValueError, match="tangent"):
                kv().prefix_attention(**dict(c, **{name: dual(c[name])}))
        with pytest.raises(ValueError, match="tangent"):
            kv().prefix_attention(**c, out=dual(torch.zeros_like(c["q"])))
        for name in ("qkv", "pool", "cos", "sin", "q_weight", "k_weight"):
            with pytest.raises(ValueError, match="tangent"):
                kv().qk_norm_rope_store(**dict(base, **{name: dual(base[name])}))
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):  # forward derivatives stay on there
            kv().prefix_attention(**dict(c, q=dual(c["q"])))
        kv().prefix_attention(**c)
        kv().qk_norm_rope_store(**base)


@pytest.mark.parametrize("dtype,hq,hk,D", [(F4, 4, 2, 64), (BF, 4, 2, 256)])
def test_pages_outside_the_pool_without_the_tensor_core(dtype, hq, hk, D):
    """They read as zeros and are flagged."""
    c = attn_case([1, 1], [40, 20], 32, 16, hq, hk, D, dtype)
    zero = c["pool"].clone()
    zero[c["table"][0, 1].item() * 16:][:16] = 0
    zero[c["prefix"][1].item() * 16:][:16] = 0
    want = kv().prefix_attention(**dict(c, pool=zero), return_lse=True)
    table, prefix = c["table"].clone(), c["prefix"].clone()
    table[0, 1], prefix[1] = -1, c["pool"].shape[0] // 16
    got = kv().prefix_attention(**dict(c, table=table, prefix=prefix), return_lse=True)
    assert pkg("codec").device_status(clear=True) == 1 << 19
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------------------- far and long --
@pytest.mark.parametrize("dtype,hk,D", [(F4, 8, 64), (BF, 8, 256)])
def test_rows_in_slots_past_32_bits(dtype, hk, D):
    """Without the tensor core: pages more than 2^32 bytes into the pool."""
    c = attn_case([1, 20], [70, 40], 300, 16, hk, hk, D, dtype)
    rows = 4_400_000_000 // (2 * hk * D * c["pool"].element_size()) // 16 * 16
    far = torch.empty(rows, 2, hk, D, dtype=dtype, device="cuda")
    shift = rows // 16 - c["pool"].shape[0] // 16
    far[shift * 16:shift * 16 + c["pool"].shape[0]] = c["pool"]
    table = torch.where(c["table"] >= 0, c["table"] + shift, -1)
    a = kv().prefix_attention(**c, return_lse=True)
    b = kv().prefix_attention(**dict(c, pool=far, table=table, prefix=c["prefix"] + shift), return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_store_in_slots_past_32_bits():
    from test_gpu_kvpool import store_case
    qkv, pool, slots, positions, cos, sin, w = store_case(50, 8, 8, 128, 128, BF, True)
    rows = 1_100_000  # 4096 bytes each
    far = torch.zeros(rows, 2, 8, 128, dtype=BF, device="cuda")
    shift = rows - pool.shape[0]
    q = kv().qk_norm_rope_store(qkv, pool, slots, positions, cos, sin, 8, q_weight=w[0], k_weight=w[1])
    f = kv().qk_norm_rope_store(qkv, far, slots + shift, positions, cos, sin, 8, q_weight=w[0], k_weight=w[1])
    assert torch.equal(q, f) and torch.equal(far[slots + shift], pool[slots])
    far[slots + shift] = 0
    assert not bool(far.any())


@pytest.mark.parametrize("P,own", [(0, 1_000_003), (600_001, 400_000)])
def test_a_million_keys(P, own):
    c = attn_case([2], [own], P, 16, 4, 1, 64, BF)
    o, lse = kv().prefix_attention(**c, return_lse=True)
    check_rows(o, lse, c, torch.ones(2, 4, dtype=torch.bool, device="cuda"))
