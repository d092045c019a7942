"""KV-pool serving operators on the GPU against their plain 64-bit forms."""
from __future__ import annotations

import math

import pytest
import torch

import kvpool_ref as ref
from conftest import pkg

pytestmark = pytest.mark.gpu

BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32
FREE_SHORT, POOL_BAD, POS_BAD, PAGE_BAD = 1 << 17, 1 << 16, 1 << 18, 1 << 19


@pytest.fixture(autouse=True)
def device_status_clean():
    """Tests that flag something on purpose clear it themselves."""
    yield
    assert pkg("codec").device_status(clear=True) == 0


def kv():
    return pkg("kvpool")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------- plan -----
def plan_case(lens, new, page, width=None, pad=0, seed=0, spare=5):
    g = gen(seed)
    width = width or max([1] + [-(-(o + n) // page) for o, n in zip(lens, new)])
    held = sum(-(-o // page) for o in lens)
    need = sum(-(-(o + n) // page) + (-o // page) for o, n in zip(lens, new))
    pages = torch.randperm(held + need + spare + 3, generator=g, device="cuda").int()
    table = torch.full((len(lens), width), -7, dtype=torch.int32, device="cuda")
    at = 0
    for i, o in enumerate(lens):
        n = -(-o // page)
        table[i, :n] = pages[at:at + n]
        at += n
    return table, pages[held:].contiguous(), i32([3]), sum(new) + pad


@pytest.mark.parametrize("lens,new,page", [
    ([0], [1], 1),
    ([5], [0], 4),
    ([0, 0, 0], [0, 0, 0], 16),
    ([15, 16, 17, 0], [1, 1, 1, 1], 16),
    ([3, 0, 7, 12, 0, 1], [5, 0, 0, 13, 24, 6], 6),
    ([0, 1], [1000, 1], 64),
    ([int(x) for x in range(700)], [(i * 37) % 5 for i in range(700)], 24),
    ([i % 97 for i in range(4097)], [(i * 7) % 3 for i in range(4097)], 1),
    ([1] * 513, [0] * 512 + [9], 128),
    ([0] * 16, [8191 + i for i in range(16)], 64),
])
@pytest.mark.parametrize("pad", [0, 7])
def test_slots_plan(lens, new, page, pad):
    table, free, cursor, tokens = plan_case(lens, new, page, pad=pad)
    want_table = table.tolist()
    slots, pos, cu, out, cur = ref.plan(lens, new, want_table, free.tolist(), 3, page, tokens, base=11)
    p = kv().slots_plan(i32(lens), i32(new), table, free, cursor, page, tokens, base=11)
    assert p.slots.tolist() == slots and p.positions.tolist() == pos
    assert p.cu.tolist() == cu and p.lens.tolist() == out and p.cursor.tolist() == [cur]
    assert p.table is table and table.tolist() == want_table


def test_slots_plan_largest_batch_and_strided_table():
    B = 16384
    lens, new = [i % 33 for i in range(B)], [1] * B
    wide, free, cursor, tokens = plan_case(lens, new, 16, width=6)
    table = wide[:, :4]  # rows 6 apart
    want = table.tolist()
    slots, pos, cu, out, cur = ref.plan(lens, new, want, free.tolist(), 3, 16, tokens)
    p = kv().slots_plan(i32(lens), i32(new), table, free, cursor, 16, tokens)
    assert p.slots.tolist() == slots and p.positions.tolist() == pos and p.cu.tolist() == cu
    assert table.tolist() == want and bool((wide[:, 4:] == -7).all())


def test_slots_plan_without_room_flags_and_gives_no_slot():
    status = pkg("codec").device_status
    # two free pages from the cursor on, four needed: the last two requests go without
    table, free, cursor, tokens = plan_case([0, 0, 0, 0], [2, 2, 2, 2], 2)
    p = kv().slots_plan(i32([0] * 4), i32([2] * 4), table, free[:5], cursor, 2, 8)
    f = free.tolist()
    assert p.slots.tolist() == [2 * f[3], 2 * f[3] + 1, 2 * f[4], 2 * f[4] + 1, -1, -1, -1, -1]
    assert table[:, 0].tolist() == [f[3], f[4], -1, -1] and status() == FREE_SHORT
    # a row longer than the table
    table, free, cursor, tokens = plan_case([1, 0], [6, 1], 2)
    p = kv().slots_plan(i32([1, 0]), i32([6, 1]), table[:, :2], free, cursor, 2, 7)
    f = free.tolist()
    assert p.slots.tolist() == [2 * int(table[0, 0]) + 1, 2 * f[3], 2 * f[3] + 1, -1, -1, -1, 2 * f[4]]
    assert status() == FREE_SHORT
    # fewer outputs than tokens; a negative length counts as none
    table, free, cursor, tokens = plan_case([0, 0], [3, 3], 4)
    p = kv().slots_plan(i32([0, 0]), i32([3, 3]), table, free, cursor, 4, 4)
    assert p.cu.tolist() == [0, 3, 6] and p.slots.tolist()[3] == 4 * free.tolist()[4] and status() == FREE_SHORT
    p = kv().slots_plan(i32([0, -4]), i32([3, -1]), table, free, cursor, 4, 4)
    assert p.cu.tolist() == [0, 3, 3] and p.lens.tolist() == [3, 0] and status() == FREE_SHORT
    # a table row without the page its tokens lie on
    p = kv().slots_plan(i32([2]), i32([1]), i32([[-1, -1]]), free, cursor, 4, 1)
    assert p.slots.tolist() == [-1] and status() == FREE_SHORT


# ------------------------------------------------------------------ store -----
def store_case(T, hq, hk, D, rot, dtype, norm, seed=0, max_pos=97, pool_rows=None):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    pool_rows = pool_rows or 2 * T + 3
    qkv = (3 * r(T, (hq + 2 * hk) * D)).to(dtype)
    pool = r(pool_rows, 2, hk, D).to(dtype)
    slots = torch.randperm(pool_rows, generator=g, device="cuda")[:T].contiguous()
    positions = torch.randint(0, max_pos, (T,), generator=g, device="cuda", dtype=torch.int32)
    ang = torch.outer(torch.arange(max_pos, device="cuda").double(), 1e4 ** (-torch.arange(rot // 2, device="cuda") * 2.0 / max(rot, 1)))
    w = [(1 + 0.3 * r(D)).to(dtype) if norm else None for _ in range(2)]
    return qkv, pool, slots, positions, ang.cos().float(), ang.sin().float(), w


def check_store(qkv, pool, slots, positions, cos, sin, w, hq, interleaved=False, eps=1e-5):
    """Run the operator and compare q, the pool's stored rows and its other rows."""
    dt, hk, D = qkv.dtype, pool.shape[2], pool.shape[3]
    before = pool.clone()
    q = kv().qk_norm_rope_store(qkv, pool, slots, positions, cos, sin, hq, q_weight=w[0], k_weight=w[1], eps=eps,
                                interleaved=interleaved)
    x = qkv.reshape(-1, hq + 2 * hk, D)
    at = positions.long()
    ok = (slots >= 0) & (slots < pool.shape[0])
    for got, part, wt in ((q, x[:, :hq], w[0]), (pool[slots.long().clamp(0, pool.shape[0] - 1), 0], x[:, hq:hq + hk], w[1])):
        want, err = ref.turned(part, wt, cos[at], sin[at], eps, interleaved)
        bound = ref.half_step(dt) * (want.abs() + err) + err + ref.tiny(dt)
        off = (got.double() - want).abs() <= bound
        assert bool((off | ~ok[:, None, None] if got is not q else off).all())
    s = slots.long()[ok]
    assert torch.equal(pool[s, 1], x[ok, hq + hk:])
    left = torch.ones(pool.shape[0], dtype=torch.bool, device="cuda")
    left[s] = False
    assert torch.equal(pool[left], before[left])
    return q


@pytest.mark.parametrize("dtype", [BF, HF, F4])
@pytest.mark.parametrize("hq,hk,D,rot", [(4, 1, 128, 128), (32, 8, 128, 128), (6, 2, 64, 32), (5, 5, 80, 64),
                                         (7, 1, 96, 96), (3, 3, 16, 16), (2, 1, 8, 0), (4, 2, 256, 64)])
@pytest.mark.parametrize("norm,interleaved", [(False, False), (True, True)])
def test_qk_norm_rope_store(dtype, hq, hk, D, rot, norm, interleaved):
    if D == 256 and dtype == F4:
        D, rot = 120, 64
    qkv, pool, slots, positions, cos, sin, w = store_case(37, hq, hk, D, rot, dtype, norm)
    check_store(qkv, pool, slots, positions, cos, sin, w, hq, interleaved)


@pytest.mark.parametrize("T", [0, 1, 2, 1023, 5000])
def test_qk_norm_rope_store_lengths_and_index_types(T):
    qkv, pool, slots, positions, cos, sin, w = store_case(T, 8, 2, 128, 128, BF, True)
    slots[::5] = -1  # rows of a padded batch
    check_store(qkv, pool, slots.int(), positions.long(), cos, sin, w, 8)


def test_qk_norm_rope_store_one_sided_weights_zero_rows_and_extremes():
    qkv, pool, slots, positions, cos, sin, w = store_case(64, 4, 2, 64, 64, BF, True)
    qkv[3] = 0
    qkv[5] *= 1e18   # squares reach 1e37: still inside fp32
    qkv[6] *= 1e-18
    check_store(qkv, pool, slots, positions, cos, sin, [w[0], None], 4)
    check_store(qkv, pool, slots, positions, cos, sin, [None, w[1]], 4)
    qkv[7, :64] = math.nan  # one head of one token: no other head sees it
    q = kv().qk_norm_rope_store(qkv, pool, slots, positions, cos, sin, 4, q_weight=w[0])
    bad = torch.isnan(q).any(-1)
    assert bool(bad[7, 0]) and int(bad.sum()) == 1


def test_qk_norm_rope_store_strides_and_pool_layouts():
    qkv, pool, slots, positions, cos, sin, w = store_case(50, 4, 2, 64, 64, HF, True)
    wide = torch.zeros(50, qkv.shape[1] + 24, dtype=HF, device="cuda")
    wide[:, 8:8 + qkv.shape[1]] = qkv
    check_store(wide[:, 8:8 + qkv.shape[1]], pool, slots, positions, cos, sin, w, 4)
    planes = torch.randn(2, 103, 2, 64, device="cuda").to(HF)  # all K rows, then all V rows
    check_store(qkv, planes.transpose(0, 1), slots, positions, cos, sin, w, 4)
    layers = torch.randn(103, 3, 2, 2, 64, device="cuda").to(HF)  # one layer of slot records that hold three
    other = layers[:, [0, 2]].clone()
    check_store(qkv, layers[:, 1], slots, positions, cos, sin, w, 4)
    assert torch.equal(layers[:, [0, 2]], other)


def test_qk_norm_rope_store_flags_bad_slots_and_positions():
    status = pkg("codec").device_status
    qkv, pool, slots, positions, cos, sin, w = store_case(9, 4, 2, 64, 64, BF, False)
    slots[4] = pool.shape[0]
    check_store(qkv, pool, slots, positions, cos, sin, w, 4)
    assert status() == POOL_BAD
    slots[4] = -1
    positions[2] = 97
    positions[3] = -1
    q = kv().qk_norm_rope_store(qkv, pool, slots, positions, cos, sin, 4)
    assert status() == POS_BAD
    assert torch.equal(q[2:4].flatten(1), qkv[2:4, :256])  # left unrotated
    assert torch.equal(pool[slots[2], 0].flatten(), qkv[2, 256:384])


# -------------------------------------------------------------- attention -----
def attn_case(q_lens, lens, P, page, hq, hk, D, dtype, seed=0, spare=2, garbage=math.nan, pad=0):
    """Pages in random order; every slot outside the lengths holds garbage."""
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    npre, need = -(-P // page), [-(-n // page) for n in lens]
    pages = torch.randperm(npre + sum(need) + spare, generator=g, device="cuda").int()
    pool = torch.full((len(pages) * page, 2, hk, D), garbage, device="cuda", dtype=dtype)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32, device="cuda")
    inner = torch.arange(page, device="cuda")
    flat = lambda p, n: (p.long()[:, None] * page + inner).reshape(-1)[:n]  # noqa: E731
    prefix = pages[:npre].contiguous()
    pool[flat(prefix, P)] = r(P, 2, hk, D).to(dtype)
    at = npre
    for i, n in enumerate(lens):
        table[i, :need[i]] = pages[at:at + need[i]]
        pool[flat(table[i, :need[i]], n)] = r(n, 2, hk, D).to(dtype)
        at += need[i]
    cu = i32([0] + torch.tensor(q_lens).cumsum(0).tolist())
    q = (1.5 * r(sum(q_lens) + pad, hq, D)).to(dtype)
    return dict(q=q, pool=pool, cu=cu, lens=i32(lens), table=table, page=page, prefix=prefix, prefix_len=P)


def check_attention(c, **kw):
    n = int(c["cu"][-1])
    out = torch.full_like(c["q"], 7.0).contiguous()
    o, lse = kv().prefix_attention(**c, out=out, return_lse=True, **kw)
    assert o is out
    live = dict(c, q=c["q"][:n])
    want, wl, to, tl = ref.attention(**live, **kw)
    assert not bool(torch.isnan(o[:n]).any())
    err = (o[:n].double() - want).abs() - to
    assert float(err.max()) <= 0 if n else True, f"o off by {float(err.max())} more than allowed"
    empty = wl == -math.inf
    assert torch.equal(lse[:n] == -math.inf, empty)
    assert bool(((lse[:n].double() - wl).abs() <= tl)[~empty].all())
    assert bool((o[n:] == 7).all())  # rows behind the last request stay as they were
    return o, lse


SHAPES = [(4, 1, 128), (32, 8, 128), (8, 8, 64), (15, 5, 64), (6, 2, 80), (8, 1, 96), (4, 2, 16), (2, 2, 40)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hk,D", SHAPES)
@pytest.mark.parametrize("q_lens,lens,P", [
    ([1], [1], 0),
    ([1, 1, 1], [1, 300, 129], 0),
    ([1, 1, 1, 1, 1], [5, 1, 128, 64, 257], 385),
    ([3, 0, 1, 40], [3, 9, 70, 300], 130),
    ([200], [200], 0),
    ([77], [200], 128),
])
def test_prefix_attention(dtype, hq, hk, D, q_lens, lens, P):
    check_attention(attn_case(q_lens, lens, P, 16, hq, hk, D, dtype))


@pytest.mark.parametrize("page", [1, 3, 16, 24, 128, 200])
def test_prefix_attention_page_sizes(page):
    check_attention(attn_case([1, 5, 1, 0, 60], [400, 131, 2, 7, 60], 333, page, 8, 2, 128, BF, seed=page))


def test_prefix_attention_fp32_and_wide_heads():
    check_attention(attn_case([1, 5, 9], [40, 131, 9], 65, 16, 8, 2, 64, F4))
    check_attention(attn_case([2, 1], [40, 131], 65, 16, 4, 2, 256, F4))
    check_attention(attn_case([2, 1], [40, 131], 65, 16, 4, 2, 256, BF))
    check_attention(attn_case([2, 1], [40, 131], 65, 16, 4, 2, 8, HF))


@pytest.mark.parametrize("dtype,hq,hk,D", [(F4, 8, 1, 128), (F4, 10, 2, 64), (BF, 12, 4, 256), (HF, 6, 1, 136), (F4, 3, 3, 4),
                                           (BF, 8, 2, 8), (F4, 14, 2, 252)])
def test_prefix_attention_rows_of_few_and_many_tokens(dtype, hq, hk, D):
    check_attention(attn_case([1, 2, 0], [40, 131, 3], 65, 16, hq, hk, D, dtype))
    check_attention(attn_case([170, 1, 3], [170, 300, 0], 33, 16, hq, hk, D, dtype, pad=2))


def test_prefix_attention_empty_rows():
    # no keys at all; more queries than own keys (the first see nothing, or the prefix alone)
    c = attn_case([2, 1, 6], [0, 0, 4], 0, 16, 4, 2, 64, BF)
    o, lse = check_attention(c)
    assert bool((o[:5] == 0).all()) and bool((lse[:5] == -math.inf).all())
    check_attention(attn_case([2, 1, 6], [0, 0, 4], 100, 16, 4, 2, 64, BF))
    check_attention(attn_case([0, 0], [5, 0], 100, 16, 4, 2, 64, BF, pad=3))


def test_prefix_attention_leaves_padding_alone():
    check_attention(attn_case([1, 3], [77, 90], 140, 16, 8, 2, 128, BF, pad=9))


@pytest.mark.parametrize("B,P,hi", [(70, 1000, 40), (300, 513, 3), (33, 5, 900)])
def test_prefix_attention_many_requests(B, P, hi):
    lens = [1 + (i * 7919) % hi for i in range(B)]
    check_attention(attn_case([1] * B, lens, P, 16, 8, 2, 128, BF))


def test_prefix_attention_long_and_mixed():
    check_attention(attn_case([1], [9000], 0, 16, 4, 1, 128, BF))
    check_attention(attn_case([1, 1], [9, 4000], 20001, 64, 8, 2, 128, BF))
    check_attention(attn_case([700, 1, 33, 1], [2000, 3, 33, 500], 1111, 16, 8, 2, 128, BF))
    check_attention(attn_case([1500], [1500], 1000, 16, 4, 1, 128, HF))


def test_prefix_attention_scores_far_apart():
    """Scores that grow along the keys (the running maximum moves at every step),
    single keys that outweigh all others, and equal scores."""
    c = attn_case([1, 200], [700, 400], 600, 16, 4, 1, 128, BF)
    steps = torch.arange(c["pool"].shape[0], device="cuda") / 40.0
    c["pool"][:, 0] = (c["pool"][:, 0].float().nan_to_num() * 0.1 + steps[:, None, None] * 0.2).to(BF)
    c["q"] = (c["q"].abs() + 0.3).to(BF)
    check_attention(c)
    c["q"][:, 1] = 0  # a head without preferences
    check_attention(c)
    check_attention(c, scale=-0.3)


def test_prefix_attention_strides():
    c = attn_case([1, 30], [70, 40], 99, 16, 6, 2, 64, BF)
    qkv = torch.randn(31, 10, 64, device="cuda").to(BF)
    qkv[:, 2:8] = c["q"]
    check_attention(dict(c, q=qkv[:, 2:8]))
    heads_first = c["q"].transpose(0, 1).contiguous().transpose(0, 1)
    check_attention(dict(c, q=heads_first))
    wide = torch.full((2, c["table"].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :c["table"].shape[1]] = c["table"]
    check_attention(dict(c, table=wide[:, :c["table"].shape[1]]))
    planes = c["pool"].transpose(0, 1).contiguous().transpose(0, 1)
    check_attention(dict(c, pool=planes))
    layers = torch.full((c["pool"].shape[0], 3, 2, 2, 64), math.nan, device="cuda", dtype=BF)
    layers[:, 1] = c["pool"]
    check_attention(dict(c, pool=layers[:, 1]))


@pytest.mark.parametrize("hq,hk,D", [(8, 8, 128), (4, 2, 64), (12, 4, 128), (24, 4, 64), (7, 1, 128), (40, 2, 64),
                                     (32, 2, 64), (32, 1, 128), (96, 2, 32), (200, 1, 16)])
def test_prefix_attention_queries_of_any_group_and_layout(hq, hk, D):
    """Whole token rows, slices of wider rows, heads first, and a token pitch that is no whole number of heads."""
    c = attn_case([1, 0, 70, 9], [300, 5, 90, 9], 150, 16, hq, hk, D, HF, seed=hq, pad=2)
    check_attention(c)
    T = c["q"].shape[0]
    for wide in (torch.zeros(T, hq * D + 3 * D, device="cuda", dtype=HF), torch.zeros(T, hq * D + 8, device="cuda", dtype=HF)):
        part = wide[:, :hq * D].view(T, hq, D)
        part.copy_(c["q"])
        check_attention(dict(c, q=part))
    check_attention(dict(c, q=c["q"].transpose(0, 1).contiguous().transpose(0, 1)))
    check_attention(dict(attn_case([1], [77], 20, 16, hq, hk, D, BF)))


@pytest.mark.parametrize("B,P", [(1000, 0), (1000, 40), (5000, 9)])
def test_prefix_attention_more_requests_than_threads(B, P):
    lens = [1 + (i * 7919) % 50 for i in range(B)]
    q_lens = [i % 3 for i in range(B)]
    check_attention(attn_case(q_lens, [max(n, m) for n, m in zip(lens, q_lens)], P, 16, 4, 2, 64, BF))


def test_prefix_attention_first_scores_far_below():
    """The first 32 scores of a row are small ones: its reference has to move in the same tile."""
    c = attn_case([1, 3], [100, 200], 0, 16, 4, 2, 128, BF, garbage=0.0)
    for i, n in enumerate((100, 200)):
        pages = c["table"][i, :-(-n // 16)].long()
        slots = (pages[:, None] * 16 + torch.arange(16, device="cuda")).reshape(-1)[:n]
        c["pool"][slots[:40], 0] *= 0.01
        c["pool"][slots[40:], 0] *= 6
    check_attention(c)


def test_out_may_not_overlap():
    c = attn_case([1, 2], [20, 30], 16, 16, 4, 2, 64, BF)
    room = torch.zeros(5, 4, 64, device="cuda", dtype=BF)
    room[:3] = c["q"]
    for q, out in ((c["q"], c["q"]), (room[:3], room[2:])):
        with pytest.raises(ValueError, match="overlaps"):
            kv().prefix_attention(**dict(c, q=q), out=out)
    with pytest.raises(ValueError, match="overlaps"):
        kv().prefix_attention(**c, out=c["pool"].view(-1)[:3 * 4 * 64].view(3, 4, 64))
    with pytest.raises(ValueError, match="gradient"):
        kv().prefix_attention(**c, out=torch.zeros(3, 4, 64, device="cuda", dtype=BF, requires_grad=True))
    with pytest.raises(ValueError, match="stride"):
        kv().prefix_attention(**dict(c, q=c["q"][:, :1].expand(-1, 4, -1)))
    qkv, pool, slots, positions, cos, sin, w = store_case(9, 4, 2, 64, 64, BF, True)
    with pytest.raises(ValueError, match="overlaps"):
        kv().qk_norm_rope_store(qkv, pool, slots, positions, cos, sin, 4, out=qkv.view(-1)[:9 * 256].view(9, 4, 64))


def test_prefix_attention_far_slots():
    """Pages more than 2^32 bytes into the pool."""
    c = attn_case([1, 20], [70, 40], 300, 16, 8, 8, 128, BF)
    rows = 1_200_000  # 4096 bytes each
    far = torch.empty(rows, 2, 8, 128, dtype=BF, device="cuda")
    shift = (rows - c["pool"].shape[0]) // 16
    far[shift * 16:shift * 16 + c["pool"].shape[0]] = c["pool"]
    table = torch.where(c["table"] >= 0, c["table"] + shift, -1)
    check_attention(dict(c, pool=far, table=table, prefix=c["prefix"] + shift))


def test_prefix_attention_flags_pages_outside_the_pool():
    status = pkg("codec").device_status
    c = attn_case([1, 1], [40, 20], 32, 16, 4, 2, 64, BF)
    zero = c["pool"].clone()
    zero[c["table"][0, 1].item() * 16:][:16] = 0
    zero[c["prefix"][1].item() * 16:][:16] = 0
    want = kv().prefix_attention(**dict(c, pool=zero))
    assert status() == 0
    table, prefix = c["table"].clone(), c["prefix"].clone()
    table[0, 1], prefix[1] = -1, c["pool"].shape[0] // 16
    got = kv().prefix_attention(**dict(c, table=table, prefix=prefix))
    assert status() == PAGE_BAD
    assert torch.equal(got, want)
    # a length past its table row is cut to it
    n = c["table"].shape[1] * 16
    full = dict(c, pool=torch.nan_to_num(c["pool"]), lens=i32([n, 20]), table=torch.where(c["table"] < 0, 0, c["table"]))
    want = kv().prefix_attention(**full)
    got = kv().prefix_attention(**dict(full, lens=i32([n + 9, 20])))
    assert status() == PAGE_BAD and torch.equal(got, want)


def test_requests_do_not_disturb_each_other():
    """A request whose values are not finite leaves the others' rows alone."""
    c = attn_case([1, 1, 40], [200, 300, 40], 150, 16, 8, 2, 128, BF)
    want = kv().prefix_attention(**c)
    c["pool"][c["table"][1, 2].item() * 16 + 3] = math.inf
    got = kv().prefix_attention(**c)
    assert torch.equal(got[[0] + list(range(2, 42))], want[[0] + list(range(2, 42))])
    assert bool(torch.isnan(got[1]).any())


# ---------------------------------------------------- streams, graphs, chain --
def test_same_inputs_same_bits():
    c = attn_case([1] * 20 + [90], [300 + i for i in range(20)] + [90], 2000, 16, 8, 2, 128, BF)
    a, b = (kv().prefix_attention(**c, return_lse=True) for _ in range(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_other_stream():
    c = attn_case([1] * 9, [300 + i for i in range(9)], 2000, 16, 8, 2, 128, BF)
    want = kv().prefix_attention(**c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = [kv().prefix_attention(**c, stream=s) for _ in range(3)]
    both = [kv().prefix_attention(**c) for _ in range(3)]  # at the same time as the others
    s.synchronize()
    assert all(torch.equal(o, want) for o in outs + both)


def test_captured_steps_replay_with_new_lengths():
    """plan -> store -> attention captured once; replays advance the batch token by
    token and give what the same calls give eagerly. Two graphs alternate."""
    k = kv()
    torch.manual_seed(5)
    B, page, hq, hk, D, P = 3, 4, 4, 2, 64, 10
    pool0 = torch.randn(200, 2, hk, D, device="cuda").to(BF)
    prefix = i32([40, 41, 42])
    free = torch.arange(0, 40, dtype=torch.int32, device="cuda")
    ang = torch.outer(torch.arange(64, device="cuda").float(), 1e4 ** (-torch.arange(32, device="cuda") / 32.0))
    cos, sin = ang.cos(), ang.sin()
    new = i32([1, 0, 1])
    steps = [torch.randn(4, (hq + 2 * hk) * D, device="cuda").to(BF) for _ in range(6)]

    def step(st, qkv):
        p = k.slots_plan(st["lens"], new, st["table"], free, st["cursor"], page, 4, base=P)
        q = k.qk_norm_rope_store(qkv, st["pool"], p.slots, p.positions, cos, sin, hq)
        st["out"].fill_(7)
        k.prefix_attention(q, st["pool"], p.cu, p.lens, p.table, page, prefix=prefix, prefix_len=P, out=st["out"])
        st["lens"].copy_(p.lens)
        st["cursor"].copy_(p.cursor)

    def fresh():
        t = torch.full((B, 4), -1, dtype=torch.int32, device="cuda")
        return dict(lens=i32([0, 0, 0]), cursor=i32([0]), table=t, pool=pool0.clone(),
                    out=torch.zeros(4, hq, D, dtype=BF, device="cuda"))

    eager, want = fresh(), []
    for x in steps:
        step(eager, x)
        want.append(eager["out"].clone())
    live, qkv = fresh(), torch.empty_like(steps[0])
    qkv.copy_(steps[0])
    warm = fresh()
    step(warm, qkv)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(live, qkv)
        graphs.append(graph)
    for i, x in enumerate(steps):
        qkv.copy_(x)
        graphs[i % 2].replay()
        assert torch.equal(live["out"], want[i]), i
    assert torch.equal(live["pool"], eager["pool"]) and torch.equal(live["table"], eager["table"])
    assert live["lens"].tolist() == [6, 0, 6]


def test_plan_store_protect_lose_recover_attend():
    """The path in one piece: plan and store a ragged batch, encode the stored rows
    with the erasure code through the plan's slots, lose the rows, rebuild them,
    and attend: the same bits as before the loss."""
    k, codec, g = kv(), pkg("codec"), pkg()
    hq, hk, D, page, P = 8, 2, 64, 16, 48
    c = attn_case([1, 20, 7], [0, 0, 0], P, page, hq, hk, D, BF, garbage=0.5, spare=40)
    new = i32([1, 20, 7])
    table = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    used = set(c["prefix"].tolist())
    free = i32([p for p in range(c["pool"].shape[0] // page) if p not in used])
    plan = k.slots_plan(i32([0, 0, 0]), new, table, free, i32([0]), page, 32, base=P)  # 4 rows of padding
    qkv = torch.randn(32, (hq + 2 * hk) * D, device="cuda").to(BF)
    ang = torch.outer(torch.arange(128, device="cuda").float(), 1e4 ** (-torch.arange(32, device="cuda") / 32.0))
    q = k.qk_norm_rope_store(qkv, c["pool"], plan.slots, plan.positions, ang.cos(), ang.sin(), hq)
    args = dict(cu=plan.cu, lens=plan.lens, table=plan.table, page=page, prefix=c["prefix"], prefix_len=P)
    check_attention(dict(args, q=q, pool=c["pool"]))
    before = k.prefix_attention(q[:28], c["pool"], **args)
    row = hk * D * 2
    shards = []
    for plane in (0, 1):
        shards.append(torch.empty(32 * row, dtype=torch.uint8, device="cuda"))
        codec.slots_gather(c["pool"], plan.slots, shards[-1], plane=plane)
    spec = g.CodeSpec.xor(2)
    parity = g.encode(spec, shards)
    c["pool"][plan.slots[:28], 0] = math.nan
    rebuilt = g.decode(spec, [None, shards[1]] + parity, [0])[0]
    codec.slots_scatter(c["pool"], plan.slots, rebuilt, plane=0)
    assert torch.equal(k.prefix_attention(q[:28], c["pool"], **args), before)


# --------------------------------------------------------------- refusals -----
def test_refusals():
    k = kv()
    c = attn_case([1, 2], [20, 30], 16, 16, 4, 2, 64, BF)
    bad = [dict(q=c["q"].float()), dict(q=c["q"].cpu()), dict(q=c["q"][0]), dict(lens=c["lens"].long()),
           dict(cu=c["cu"][:-1]), dict(table=c["table"][:1]), dict(table=c["table"].long()),
           dict(table=c["table"].t().contiguous().t()), dict(page=0), dict(prefix_len=17), dict(prefix_len=-1),
           dict(prefix=None), dict(scale=math.inf), dict(pool=c["pool"][:, :1]), dict(pool=c["pool"][:, :, :, :32]),
           dict(pool=c["pool"].transpose(2, 3).contiguous().transpose(2, 3)), dict(out=torch.empty(3, 4, 32, device="cuda", dtype=BF)),
           dict(q=torch.zeros(3, 3, 64, device="cuda", dtype=BF)),
           dict(q=torch.zeros(3, 4, 68, device="cuda", dtype=BF)[:, :, 2:66]),
           dict(q=torch.zeros(3, 4, 12, device="cuda", dtype=BF), pool=torch.zeros(64, 2, 2, 12, device="cuda", dtype=BF))]
    bad.append(dict(q=c["q"].clone().requires_grad_()))  # forward only
    for b in bad:
        with pytest.raises(ValueError):
            k.prefix_attention(**dict(c, **b))
    with torch.no_grad():
        k.prefix_attention(**dict(c, q=c["q"].clone().requires_grad_()))
    with pytest.raises(ValueError):
        k.prefix_attention(**c, scale=math.nan)
    qkv, pool, slots, positions, cos, sin, w = store_case(9, 4, 2, 64, 64, BF, True)
    base = dict(qkv=qkv, pool=pool, slots=slots, positions=positions, cos=cos, sin=sin, heads=4)
    for b in [dict(qkv=qkv.float()), dict(heads=5), dict(slots=slots[:8]), dict(slots=slots.short()),
              dict(positions=positions.float()), dict(positions=positions[:8]), dict(cos=cos.double()),
              dict(sin=sin[:, :16]), dict(cos=cos[:, :12].contiguous(), sin=sin[:, :12].contiguous()),
              dict(q_weight=w[0][:32]), dict(k_weight=w[1].float()), dict(out=torch.empty(9, 4, 32, device="cuda", dtype=BF)),
              dict(pool=pool.expand(-1, -1, -1, -1)[:, :1].expand(-1, 2, -1, -1)),
              dict(cos=torch.zeros(97, 48, device="cuda"), sin=torch.zeros(97, 48, device="cuda"))]:
        args = dict(base, **b)
        with pytest.raises(ValueError):
            k.qk_norm_rope_store(args.pop("qkv"), **args)
    table, free, cursor, tokens = plan_case([5, 0], [3, 4], 4)
    base = dict(lens=i32([5, 0]), new=i32([3, 4]), table=table, free=free, cursor=cursor, page=4, tokens=tokens)
    for b in [dict(lens=i32([5])), dict(new=torch.tensor([3, 4], device="cuda")), dict(table=table.long()), dict(page=0),
              dict(tokens=-1), dict(cursor=i32([1, 2])), dict(free=free.long()), dict(free=free[::2])]:
        args = dict(base, **b)
        with pytest.raises(ValueError):
            k.slots_plan(args.pop("lens"), **args)
