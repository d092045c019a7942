"""Measured cases of the KV-pool serving operators: slot plans, the fused norm /
rotation / store of queries and keys, and attention over a pool with a shared
prefix.

Every case is one call as a serving step makes it.  ``own`` chooses the side:
false computes the operator in plain torch operations in 32 bits, true calls the
engine.  Lengths are a fixed set per case (the seed only deals them out to the
requests), so a case's work does not depend on the seed.
"""
import importlib
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _kvpool():
    return importlib.import_module("26mlsys-ae-ghostserve_b200.kvpool")


# ------------------------------------------------------------------- cases --
def listed():
    plan = dict(op="plan")
    store = dict(op="store", dtype="bf16", hq=32, hk=8, dim=128, rot=128, norm=False, interleaved=False)
    attn = dict(op="attn", dtype="bf16", hq=32, hk=8, dim=128, page=16)
    return [
        # one decode step of 64 running requests: one new token each, a page now and then (latency)
        dict(plan, name="plan decode 64", batch=64, old_lo=1, old_hi=4096, new_lo=1, new_hi=1, page=16),
        # admission of a wave of short and empty requests, uneven lengths, odd page size
        dict(plan, name="plan ragged 3001", batch=3001, old_lo=0, old_hi=700, new_lo=0, new_hi=90, page=24),
        # 16 prompts of 32768 tokens planned at once (the prefill benchmark's batch)
        dict(plan, name="plan prompts 16x32768", batch=16, old_lo=0, old_hi=0, new_lo=32768, new_hi=32768, page=64),
        # decode step of one tensor-parallel rank of 8: 4 query heads on 1 KV head (latency)
        dict(store, name="store decode 16 tp8", tokens=16, hq=4, hk=1, max_pos=32768),
        # one 2048-token prefill chunk of the whole model, with query and key norms
        dict(store, name="store chunk 2048 norm", tokens=2048, norm=True, max_pos=32768),
        # a large ragged extend batch in fp16, half the head rotated in adjacent pairs
        dict(store, name="store extend 16381 fp16", tokens=16381, dtype="fp16", rot=64, norm=True, interleaved=True,
             max_pos=8192),
        # first tokens of a few short requests on one rank of 8, no shared prefix (latency)
        dict(attn, name="attn decode 3 short", batch=3, q_lo=1, q_hi=1, kv_lo=1, kv_hi=300, prefix=0, hq=4, hk=1),
        # 16 samples of one 32768-token prompt, a few hundred tokens in (cache-bandwidth bound)
        dict(attn, name="attn decode 16 of 32768", batch=16, q_lo=1, q_hi=1, kv_lo=100, kv_hi=600, prefix=32768),
        # 128 chats behind a 2048-token system prompt, uneven histories
        dict(attn, name="attn decode 128 ragged", batch=128, q_lo=1, q_hi=1, kv_lo=1, kv_hi=2500, prefix=2047),
        # 256 requests on one long shared document (matrix-rate bound)
        dict(attn, name="attn decode 256 of 24576", batch=256, q_lo=1, q_hi=1, kv_lo=1, kv_hi=128, prefix=24576),
        # the last 2048-token chunk of a 32768-token prompt
        dict(attn, name="attn chunk 2048 of 32768", batch=1, q_lo=2048, q_hi=2048, kv_lo=2048, kv_hi=2048,
             prefix=30720),
        # uneven extends (some of a single token) in fp16, 64-wide heads, page size 1
        dict(attn, name="attn extend 9 fp16 d64", batch=9, q_lo=1, q_hi=777, kv_lo=1100, kv_hi=1900, prefix=1000,
             dtype="fp16", hq=15, hk=5, dim=64, page=1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "store", "attn", "attn"])
    page = rng.choice([1, 16, 24, 32, 64, 128])
    if op == "plan":
        batch = _log(rng, 1, 4096)
        hi = _log(rng, 1, max(1, min(32768, 524288 // batch)))
        return dict(op=op, batch=batch, old_lo=0, old_hi=_log(rng, 1, 8192), new_lo=rng.choice([0, 1, hi]), new_hi=hi,
                    page=page)
    hk = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 4, 8])
    dim = rng.choice([64, 80, 96, 128, 128])
    if op == "store":
        # the grid's largest is 16381 tokens x 48 heads x 128
        tokens = _log(rng, 1, min(16381, 16381 * 48 * 128 // (hk * (group + 2) * dim)))
        return dict(op=op, tokens=tokens, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), hq=hk * group, hk=hk,
                    dim=dim, rot=rng.choice([dim, dim, 32, 64]), norm=rng.random() < 0.5,
                    interleaved=rng.random() < 0.3, max_pos=_log(rng, 1024, 65536))
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), hq=hk * group, hk=hk, dim=dim, page=page)
    prefix = rng.choice([0, _log(rng, 1, 32768), _log(rng, 512, 32768)])
    if rng.random() < 0.6:  # decode: at most 256 requests
        batch = _log(rng, 1, 256)
        lo = _log(rng, 1, 64)
        return dict(case, batch=batch, q_lo=1, q_hi=1, kv_lo=lo, kv_hi=lo + _log(rng, 1, max(2, min(4096, 120000 // batch))),
                    prefix=prefix)
    batch = _log(rng, 1, 12)  # extends: at most 2048 tokens in all
    q_hi = _log(rng, 2, 2048 // batch)
    kv_lo = q_hi + rng.choice([0, 0, _log(rng, 1, 2000)])
    prefix = min(prefix, 2048 * 32 * 128 * 28000 // (batch * q_hi * hk * group * dim))  # the listed chunk's work
    return dict(case, batch=batch, q_lo=rng.choice([1, q_hi]), q_hi=q_hi, kv_lo=kv_lo,
                kv_hi=kv_lo + rng.choice([0, _log(rng, 1, 1000)]), prefix=prefix)


def _spread(n, lo, hi, salt):
    """n whole numbers over [lo, hi], the same for every seed."""
    return [lo + (((i + 1) * 2654435761 + salt * 40503) % (1 << 32)) * (hi - lo + 1) // (1 << 32) for i in range(n)]


def _lengths(c):
    if c["op"] == "plan":
        return _spread(c["batch"], c["old_lo"], c["old_hi"], 1), _spread(c["batch"], c["new_lo"], c["new_hi"], 2)
    return _spread(c["batch"], c["q_lo"], c["q_hi"], 3), _spread(c["batch"], c["kv_lo"], c["kv_hi"], 4)


# ----------------------------------------------------------------- prepare --
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"plan": _prepare_plan, "store": _prepare_store, "attn": _prepare_attn}[case["op"]](case, g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).to(DEV)


def _dealt(g, a, b):
    """The pairs of two length lists, dealt out in the seed's order."""
    order = torch.randperm(len(a), generator=g, device=DEV)
    return _i32(a)[order].contiguous(), _i32(b)[order].contiguous()


def _prepare_plan(c, g):
    page, batch = c["page"], c["batch"]
    old, new = _lengths(c)
    width = max(-(-(o + n) // page) for o, n in zip(old, new)) + 2
    held = sum(-(-o // page) for o in old)
    extra = sum(-(-(o + n) // page) + (-o // page) for o, n in zip(old, new))
    tokens = sum(new)
    old, new = _dealt(g, old, new)
    pages = torch.randperm(held + extra + 40, generator=g, device=DEV).to(torch.int32)
    # rows hold the pages of the tokens so far; the rest of a row is unset
    have = (old.long() + page - 1) // page
    col = torch.arange(width, device=DEV)
    at = (torch.cumsum(have, 0) - have)[:, None] + col
    table = torch.where(col < have[:, None], pages[at.clamp(max=len(pages) - 1)], torch.full_like(pages[:1], -1))
    return dict(c=c, op="plan", old=old, new=new, table=table.contiguous(), free=pages[held:].contiguous(),
                cursor=_i32([7]), tokens=tokens + 5, page=page, base=1000)


def _prepare_store(c, g):
    T, hq, hk, D, dt = c["tokens"], c["hq"], c["hk"], c["dim"], DTYPES[c["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    slots = torch.randperm(2 * T + 3, generator=g, device=DEV)[:T].contiguous()
    positions = torch.randint(0, c["max_pos"], (T,), generator=g, device=DEV, dtype=torch.int32)
    inv = 500000.0 ** (-torch.arange(0, c["rot"], 2, device=DEV, dtype=torch.float64) / c["rot"])
    ang = torch.arange(c["max_pos"], device=DEV, dtype=torch.float64)[:, None] * inv
    weight = lambda: (1 + 0.2 * randn(D)).to(dt) if c["norm"] else None  # noqa: E731
    return dict(c=c, op="store", qkv=randn(T, (hq + 2 * hk) * D).to(dt), pool=randn(2 * T + 3, 2, hk, D).to(dt),
                slots=slots, positions=positions, cos=ang.cos().float(), sin=ang.sin().float(), hq=hq, hk=hk, D=D,
                q_weight=weight(), k_weight=weight(), eps=1e-5, interleaved=c["interleaved"])


def _prepare_attn(c, g):
    page, B, P, D, hq, hk, dt = c["page"], c["batch"], c["prefix"], c["dim"], c["hq"], c["hk"], DTYPES[c["dtype"]]
    ql, kl = _lengths(c)
    width = max(-(-k // page) for k in kl)
    np_, ns = -(-P // page), sum(-(-k // page) for k in kl)
    T, qmax = sum(ql), max(ql)
    q_lens, lens = _dealt(g, ql, kl)
    rows = (np_ + ns + 3) * page
    pages = torch.randperm(np_ + ns + 3, generator=g, device=DEV).to(torch.int32)
    pool = torch.randn(rows, 2, hk, D, generator=g, device=DEV, dtype=torch.float32 if rows < 2000 else dt).to(dt)
    have = (lens.long() + page - 1) // page
    col = torch.arange(width, device=DEV)
    at = np_ + (torch.cumsum(have, 0) - have)[:, None] + col
    table = torch.where(col < have[:, None], pages[at.clamp(max=len(pages) - 1)], torch.full_like(pages[:1], -1))
    cu = torch.cat([q_lens.new_zeros(1), torch.cumsum(q_lens, 0, dtype=torch.int32)])
    q = torch.randn(T, hq, D, generator=g, device=DEV).to(dt)
    return dict(c=c, op="attn", q=q, pool=pool, cu=cu, lens=lens, table=table.contiguous(), page=page,
                prefix=pages[:np_].contiguous(), prefix_len=P, qmax=qmax, hk=hk, D=D)


# --------------------------------------------------------------------- run --
def run(s):
    if own:
        return {"plan": _own_plan, "store": _own_store, "attn": _own_attn}[s["op"]](s)
    return {"plan": _plain_plan, "store": _plain_store, "attn": _plain_attn}[s["op"]](s)


def _own_plan(s):
    p = _kvpool().slots_plan(s["old"], s["new"], s["table"], s["free"], s["cursor"], s["page"], s["tokens"],
                             base=s["base"])
    return dict(slots=p.slots, positions=p.positions, cu=p.cu, lens=p.lens, cursor=p.cursor, table=p.table)


def _own_store(s):
    q = _kvpool().qk_norm_rope_store(s["qkv"], s["pool"], s["slots"], s["positions"], s["cos"], s["sin"], s["hq"],
                                     q_weight=s["q_weight"], k_weight=s["k_weight"], eps=s["eps"],
                                     interleaved=s["interleaved"])
    return dict(q=q, pool=s["pool"])


def _own_attn(s):
    o, lse = _kvpool().prefix_attention(s["q"], s["pool"], s["cu"], s["lens"], s["table"], s["page"],
                                        prefix=s["prefix"], prefix_len=s["prefix_len"], return_lse=True)
    return dict(o=o, lse=lse)


def _plain_plan(s):
    page, old, new = s["page"], s["old"].long(), s["new"].long()
    total = old + new
    have, want = (old + page - 1) // page, (total + page - 1) // page
    need = want - have
    first = s["cursor"].long() + torch.cumsum(need, 0) - need
    col = torch.arange(s["table"].shape[1], device=old.device)
    fresh = (col >= have[:, None]) & (col < want[:, None])
    at = (first - have)[:, None] + col
    table = torch.where(fresh, s["free"][at.clamp(0, len(s["free"]) - 1)], s["table"])
    s["table"].copy_(table)
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    t = torch.arange(s["tokens"], device=old.device)
    req = torch.searchsorted(cu[1:], t, right=True)
    live = req < len(old)
    req = req.clamp(max=len(old) - 1)
    pos = old[req] + t - cu[req]
    # a dead row's position may lie past the table
    slot = table[req, torch.where(live, pos // page, 0)].long() * page + pos % page
    return dict(slots=torch.where(live, slot, -1), positions=torch.where(live, pos + s["base"], 0).int(),
                cu=cu.int(), lens=total.int(), cursor=(s["cursor"] + need.sum()).int(), table=s["table"])


def _plain_store(s):
    hq, hk, D = s["hq"], s["hk"], s["D"]
    x = s["qkv"].float().view(-1, hq + 2 * hk, D)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    half = cos.shape[-1]

    def turned(y, w):
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + s["eps"]) * w.float()
        r, rest = y[..., :2 * half], y[..., 2 * half:]
        if s["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = r[..., :half], r[..., half:]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([r, rest], -1)

    dt = s["qkv"].dtype
    s["pool"][s["slots"]] = torch.stack([turned(k, s["k_weight"]), v], 1).to(dt)
    return dict(q=turned(q, s["q_weight"]).to(dt), pool=s["pool"])


def _plain_attn(s):
    page, hk, D, P = s["page"], s["hk"], s["D"], s["prefix_len"]
    T, B, qmax = s["q"].shape[0], s["lens"].shape[0], s["qmax"]
    dev = s["q"].device
    q = s["q"].float().view(T, hk, -1, D) / math.sqrt(D)
    g = q.shape[2]
    # the shared prefix: every query against the same keys
    at = torch.arange(P, device=dev)
    pslot = s["prefix"].long()[at // page] * page + at % page if P else at
    kp, vp = s["pool"][pslot, 0].float(), s["pool"][pslot, 1].float()
    sp = torch.einsum("tkgd,pkd->tkgp", q, kp)
    # each request's own tokens, padded to the table's width; queries padded to qmax
    L = s["table"].shape[1] * page
    col = torch.arange(L, device=dev)
    slot = (s["table"].long()[:, col // page] * page + col % page).clamp(min=0)
    seen = col < s["lens"][:, None]
    ks = s["pool"][slot, 0].float()
    vs = torch.where(seen[:, :, None, None], s["pool"][slot, 1].float(), 0.0)
    t = torch.arange(T, device=dev)
    req = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    off = t - s["cu"].long()[req]
    qp = q.new_zeros(B, qmax, hk, g, D)
    qp[req, off] = q
    ss = torch.einsum("bqkgd,blkd->bqkgl", qp, ks)[req, off]
    last = (s["lens"].long() - (s["cu"][1:] - s["cu"][:-1]).long())[req] + off
    ss = torch.where((col <= last[:, None])[:, None, None, :], ss, -math.inf)
    m = torch.cat([sp.amax(-1, keepdim=True), ss.amax(-1, keepdim=True)], -1).amax(-1, keepdim=True) if P else \
        ss.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    sp, ss = torch.exp(sp - m), torch.exp(ss - m)
    z = sp.sum(-1, keepdim=True) + ss.sum(-1, keepdim=True)
    pp = q.new_zeros(B, qmax, hk, g, L)
    pp[req, off] = ss
    o = torch.einsum("tkgp,pkd->tkgd", sp, vp) + torch.einsum("bqkgl,blkd->bqkgd", pp, vs)[req, off]
    o = torch.where(z > 0, o / z, 0.0)
    return dict(o=o.reshape(T, hk * g, D).to(s["q"].dtype), lse=(m + torch.log(z)).reshape(T, hk * g))


# -------------------------------------------------------------------- work --
def work(case):
    c = case
    if c["op"] == "plan":
        old, new = _lengths(c)
        pages = sum(-(-(o + n) // c["page"]) + (-o // c["page"]) for o, n in zip(old, new))
        # lengths in and out, offsets; new pages read and written; a slot and a position per token
        return dict(bytes=16 * c["batch"] + 8 * pages + 12 * sum(new), flops=0)
    es = 4 if c["dtype"] == "fp32" else 2
    hq, hk, D = c["hq"], c["hk"], c["dim"]
    if c["op"] == "store":
        T, row = c["tokens"], (hq + 2 * hk) * D * es
        return dict(bytes=T * (2 * row + 12) + 4 * c["rot"] * min(T, c["max_pos"]), flops=T * (hq + hk) * 6 * D)
    ql, kl = _lengths(c)
    T = sum(ql)
    pairs = T * c["prefix"] + sum(sum(max(0, k - q + j + 1) for j in range(q)) for q, k in zip(ql, kl))
    return dict(bytes=(c["prefix"] + sum(kl)) * 2 * hk * D * es + 2 * T * hq * D * es + 4 * T * hq,
                flops=4 * pairs * hq * D)


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    """The outputs from their definitions, request by request, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "store":
        return _exact_store(s)
    return _exact_attn(s)


def _exact_store(s):
    hq, hk, D = s["hq"], s["hk"], s["D"]
    x = s["qkv"].double().view(-1, hq + 2 * hk, D)
    half = s["cos"].shape[1]
    z = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()]

    def rotated(y, w):
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + s["eps"]) * w.double()
        out = y.clone()
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["interleaved"] else \
            (slice(0, half), slice(half, 2 * half))
        u = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z[:, None, :]
        out[..., first], out[..., second] = u.real, u.imag
        return out

    pool = s["pool"].double()
    pool[s["slots"], 0] = rotated(x[:, hq:hq + hk], s["k_weight"])
    pool[s["slots"], 1] = x[:, hq + hk:]
    return dict(q=rotated(x[:, :hq], s["q_weight"]), pool=pool)


def _exact_attn(s):
    page, hk, D, P = s["page"], s["hk"], s["D"], s["prefix_len"]
    T, hq = s["q"].shape[:2]
    g = hq // hk
    o = torch.zeros(T, hq, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device=s["q"].device)
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    inner = torch.arange(page, device=s["q"].device)
    flat = lambda pages: (pages.long()[:, None] * page + inner).reshape(-1)  # noqa: E731
    pre = flat(s["prefix"])[:P]
    for i, kv in enumerate(lens):
        n = cu[i + 1] - cu[i]
        mine = torch.cat([pre, flat(s["table"][i, :-(-kv // page)])[:kv]])
        kv_rows = s["pool"][mine].double()  # [keys, 2, heads, D]
        for a in range(cu[i], cu[i] + n, 512):
            b = min(a + 512, cu[i] + n)
            hidden = torch.arange(P + kv, device=o.device) > (P + kv - n + torch.arange(a - cu[i], b - cu[i],
                                                                                       device=o.device))[:, None]
            for h in range(hk):
                k, v = kv_rows[:, 0, h], kv_rows[:, 1, h]
                heads = slice(h * g, (h + 1) * g)
                x = (s["q"][a:b, heads].double() @ k.T) * D ** -0.5
                x = x.masked_fill(hidden[:, None, :], -math.inf)
                lse[a:b, heads] = torch.logsumexp(x, -1)
                o[a:b, heads] = torch.softmax(x, -1) @ v
    return dict(o=o, lse=lse)
