"""What attention adds to the prefill model on the KV-pool operators: every layer's
attention output and every stored key and value of a ragged batch behind a shared
prefix, against each request's whole sequence through torch's attention."""
from __future__ import annotations

import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu

SPEC = dict(layers=2, hidden=256, heads=8, kv_heads=2, head_dim=64, ffn=512, vocab=300)
P, PAGE, STEPS = 50, 16, [(7, 33, 1), (1, 1, 1), (1, 0, 40)]

# Weights of query, key, value and output projections are four times the model's own, so that queries, keys and values
# have a standard deviation of about 1.28, scores of about 1.6, and attention adds as much to a row as it holds.
#
# A rounding to bf16 is off by at most u = 2^-8, by 0.58 u in the mean square (evenly spread). Queries and keys pass
# four (norm, its weight, product, rotation), six with norms of their own: 1.2 u. A score, the mean of 64 products times
# 8, is off by 8 sqrt(2) 1.2 u 1.28^2 / 8 = 2.8 u = 0.011 and the weights by as much, relatively; values (three
# roundings), the weights' rounding and the result's add 1.3 u: 3.1 u = 0.012 a side, 0.017 for both. Three times that:
TOL_FIRST = 0.05
# Layer 2: rows off by 0.017 / sqrt(2) on either side (half of a row is attention), scores by sqrt(2) 0.012 1.64 = 0.028,
# the result by 0.031 with its roundings, 0.044 for both sides. Twice that, since it no longer is all independent:
TOL_SECOND = 0.09
# Keys and values of layer 1, at worst: four roundings (values: three) on two sides.
TOL_STORED = 2 * 4 * 2.0 ** -8


@pytest.fixture(autouse=True)
def device_status_clean():
    yield
    assert pkg("codec").device_status(clear=True) == 0


def model(attention, **kw):
    """The model, and the list that every layer's attention output goes to."""
    pre = pkg("prefill")
    m = pre.TPPrefill(pre.ModelSpec(**{**SPEC, **kw}), 512, "cuda", attention=attention)
    for layer in m.layers:
        layer["wqkv"] *= 4
        layer["wo"] *= 4
    seen, rest = [], m._after_attention

    def after(x, o, layer):
        seen.append(o.clone())
        return rest(x, o, layer)

    m._after_attention = after
    return m, seen


def tokens():
    gen = torch.Generator(device="cuda").manual_seed(9)
    ids = lambda n: torch.randint(0, 300, (n,), generator=gen, device="cuda")  # noqa: E731
    return ids(P), [[ids(n) for n in step] for step in STEPS]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def batch(m, seen, base=P, prefix_len=P, pad=0):
    """The batch on the pool: per request and layer (attention outputs, keys, values) of its own tokens."""
    kv = pkg("kvpool")
    pre_ids, steps = tokens()
    free = torch.randperm(512 // PAGE, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").int()
    table = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    first = kv.slots_plan(i32([0]), i32([P]), table, free, i32([0]), PAGE, P)
    m.extend(pre_ids, first)
    tables = torch.full((3, 5), -1, dtype=torch.int32, device="cuda")
    lens, cursor = i32([0, 0, 0]), first.cursor
    got = [[[[], [], []] for _ in range(2)] for _ in range(3)]
    for parts in steps:
        n = [len(p) for p in parts]
        plan = kv.slots_plan(lens, i32(n), tables, free, cursor, PAGE, sum(n) + pad, base=base)
        seen.clear()
        ids = torch.cat(parts + [torch.zeros(pad, dtype=torch.long, device="cuda")])
        m.extend(ids, plan, prefix=first.table[0].contiguous(), prefix_len=prefix_len)
        lens, cursor = plan.lens, plan.cursor
        live = sum(n)
        for li in range(2):
            for what, x in enumerate((seen[li][:live], m.pool[li, plan.slots[:live], 0], m.pool[li, plan.slots[:live], 1])):
                for i, part in enumerate(x.split(n)):
                    got[i][li][what].append(part)
    return [[[torch.cat(x) for x in layer] for layer in req] for req in got]


def alone(qk_norm):
    """The same of every request's whole sequence by itself, through torch's attention."""
    pre_ids, steps = tokens()
    out = []
    for i in range(3):
        m, seen = model("sdpa", qk_norm=qk_norm)
        seq = torch.cat([pre_ids] + [s[i] for s in steps])
        m.forward_chunk(seq, 0)
        own = slice(P, len(seq))
        out.append([[seen[li][own], m.pool[li, own, 0], m.pool[li, own, 1]] for li in range(2)])
    return out


def off(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("pad", [0, 5])
def test_attention_and_stored_rows_of_a_ragged_batch(qk_norm, pad):
    got, want = batch(*model("pool", qk_norm=qk_norm), pad=pad), alone(qk_norm)
    for g, w in zip(got, want):
        assert off(g[0][0], w[0][0]) <= TOL_FIRST and off(g[1][0], w[1][0]) <= TOL_SECOND
        for what in (1, 2):
            assert off(g[0][what], w[0][what]) <= TOL_STORED and off(g[1][what], w[1][what]) <= TOL_SECOND


@pytest.mark.parametrize("wrong", ["no rotation", "positions from 0", "no prefix", "a prefix key short"])
def test_what_is_wrong_exceeds_the_tolerances(wrong):
    """The comparison above would see each of these, in every request."""
    m, seen = model("pool")
    if wrong == "no rotation":
        m.cos.fill_(1)
        m.sin.zero_()
    got = batch(m, seen, base=0 if wrong == "positions from 0" else P,
                prefix_len={"no prefix": 0, "a prefix key short": P - 1}.get(wrong, P))
    for g, w in zip(got, alone(False)):
        assert off(g[0][0], w[0][0]) > TOL_FIRST and off(g[1][0], w[1][0]) > TOL_SECOND


@pytest.mark.parametrize("qk_norm", [False, True])
def test_attention_and_stored_rows_of_chunks(qk_norm):
    ids = torch.randint(0, 300, (290,), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    (a, seen_a), (b, seen_b) = model("sdpa", qk_norm=qk_norm), model("pool", qk_norm=qk_norm)
    for i in range(0, 290, 97):
        a.forward_chunk(ids[i:i + 97], i)
        b.forward_chunk(ids[i:i + 97], i)
    assert len(seen_a) == len(seen_b) == 6
    for i, (x, y) in enumerate(zip(seen_b, seen_a)):
        assert off(x, y) <= (TOL_FIRST, TOL_SECOND)[i % 2]
    for what in (0, 1):
        assert off(b.pool[0, :290, what], a.pool[0, :290, what]) <= TOL_STORED
        assert off(b.pool[1, :290, what], a.pool[1, :290, what]) <= TOL_SECOND
