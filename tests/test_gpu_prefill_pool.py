"""The prefill model on the KV-pool operators: chunks, ragged extends and decode
steps behind a shared prefix, against the same tokens through torch's attention."""
from __future__ import annotations

import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu

SPEC = dict(layers=2, hidden=256, heads=8, kv_heads=2, head_dim=64, ffn=512, vocab=300)
# Both sides round to bf16 (half a step is 2^-8) at the same places: norm, qkv, query and key, scores' weights,
# attention, two projections, two residuals, feed-forward product: ten to a layer, on two layers and two sides.
TOL = 2 * 2 * 10 * 2.0 ** -8


@pytest.fixture(autouse=True)
def device_status_clean():
    yield
    assert pkg("codec").device_status(clear=True) == 0


def model(attention, max_tokens=512, **kw):
    pre = pkg("prefill")
    return pre.TPPrefill(pre.ModelSpec(**{**SPEC, **kw}), max_tokens, "cuda", attention=attention)


def near(a, b):
    a, b = a.double(), b.double()
    assert bool(torch.isfinite(a).all())
    assert float((a - b).norm() / b.norm()) <= TOL


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("max_tokens", [512, 300])
def test_forward_chunk_on_the_pool_operators(qk_norm, max_tokens):
    ids = torch.randint(0, 300, (290,), device="cuda")
    a, b = (model(x, max_tokens, qk_norm=qk_norm) for x in ("sdpa", "pool"))
    seen = []
    for i in range(0, 290, 97):
        part = ids[i:i + 97]
        xa = a.forward_chunk(part, i)
        xb = b.forward_chunk(part, i, after_attention=lambda li, k, v: seen.append((li, k.clone(), v.clone())))
        near(xb, xa)
    for pa, pb in zip(*(sum(m.chunk_kv_parts(0, 290), []) for m in (b, a))):
        near(pa, pb)
    assert [s[0] for s in seen] == [0, 1] * 3
    assert torch.equal(seen[1][1].transpose(0, 1), b.pool[1, :97, 0]) and torch.equal(seen[1][2].transpose(0, 1), b.pool[1, :97, 1])


def test_extend_ragged_batch_behind_a_shared_prefix():
    """One prefix, three continuations of different lengths, then decode steps: every
    request's hidden states are those of its whole sequence run by itself."""
    kv = pkg("kvpool")
    m = model("pool", 512)
    page, P = 16, 50
    gen = torch.Generator(device="cuda").manual_seed(9)
    pre_ids = torch.randint(0, 300, (P,), generator=gen, device="cuda")
    own = [torch.randint(0, 300, (n,), generator=gen, device="cuda") for n in (7, 33, 1)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    free = torch.randperm(512 // page, device="cuda").int()
    table = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    first = kv.slots_plan(i32([0]), i32([P]), table, free, i32([0]), page, P)
    m.extend(pre_ids, first)
    prefix = first.table[0].contiguous()
    tables = torch.full((3, 5), -1, dtype=torch.int32, device="cuda")
    lens, cursor = i32([0, 0, 0]), first.cursor
    steps = [own, [torch.randint(0, 300, (1,), generator=gen, device="cuda") for _ in range(3)],
             [torch.randint(0, 300, (1,), generator=gen, device="cuda") for _ in range(3)]]
    got = [[], [], []]
    for parts in steps:
        n = [len(p) for p in parts]
        plan = kv.slots_plan(lens, i32(n), tables, free, cursor, page, sum(n), base=P)
        x = m.extend(torch.cat(parts), plan, prefix=prefix, prefix_len=P)
        lens, cursor = plan.lens, plan.cursor
        for i, part in enumerate(x.split(n)):
            got[i].append(part)
    assert int(cursor) == 4 + 1 + 3 + 1
    for i in range(3):
        seq = torch.cat([pre_ids] + [s[i] for s in steps])
        want = model("sdpa", 512).forward_chunk(seq, 0)
        near(torch.cat(got[i]), want[P:])


def test_run_prefill_on_the_pool_operators():
    pre = pkg("prefill")
    m = model("pool", 256)
    assert pre.run_prefill(m, 2, 200, 64, "none") == 400
    assert bool(torch.isfinite(m.pool[:, :200]).all())
