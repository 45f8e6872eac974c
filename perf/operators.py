"""The operators of a serving step over a paged cache whose speed matters, as data: block tables and
slot maps from request lengths, the append that uses them, prompt attention over packed sequences, and
decode attention for a batch that shares a long prefix.

``kind`` of a case:
  plan     block tables, slots and positions of a step's new tokens from the requests' lengths
  append   the new K/V rows of a packed batch written to their slots in the paged cache
  packed   causal attention of packed sequences of different lengths; keys packed like the queries, or
           (``page`` > 0) read from the paged cache, where each request has up to ``ctx`` tokens before
           its new ones
  shared   one new token per request against a paged cache whose first ``prefix`` tokens are the same
           pages for all of them

The lengths of a case's requests are log-uniform between ``lo`` and ``hi``, drawn from ``lens``; the
first request has the longest. Values are bfloat16, N(0, 1) (projections of normalised activations), and
q, k and v of a packed batch are views of one fused projection.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPE = torch.bfloat16
MAX_FLOPS = 760e9      # of a drawn case: the largest listed prompt batch
MAX_BYTES = 1.2e9      # of a drawn case: the largest listed cache
MAX_SCORES = 8.6e9     # bytes of one request's fp32 scores in the plain form


def listed() -> list[dict]:
    return [
        # A decode step of a full batch: a token per request, now and then a page. Latency.
        dict(name="plan_decode", kind="plan", B=64, lo=1, hi=1, ctx=2048, page=16, lens=1),
        # A step that takes many prompts in, of which some are the rest of cached ones.
        dict(name="plan_prompts", kind="plan", B=512, lo=1, hi=2048, ctx=1024, page=16, lens=2),
        # The append of a decode step: 64 rows per pool.
        dict(name="append_decode", kind="append", B=64, lo=1, hi=1, page=16, Hkv=8, D=128, lens=3),
        # The append of a step of prompts.
        dict(name="append_prompts", kind="append", B=128, lo=16, hi=2048, page=16, Hkv=8, D=128,
             lens=4),
        # A small model or a unit of a test suite: three short prompts. The latency of one call.
        dict(name="packed_tiny", kind="packed", B=3, lo=17, hi=200, Hq=4, Hkv=4, D=64, cap=0.0,
             window=0, page=0, ctx=0, lens=5),
        # A batch of prompts as they come in, grouped heads, sliding window with softcap: the local
        # layers of softcap models.
        dict(name="packed_window_softcap", kind="packed", B=24, lo=64, hi=2048, Hq=32, Hkv=8, D=128,
             cap=50.0, window=256, page=0, ctx=0, lens=6),
        # One long prompt among shorter ones, grouped heads: the largest prompt batch.
        dict(name="packed_long", kind="packed", B=8, lo=300, hi=8192, Hq=32, Hkv=8, D=128, cap=0.0,
             window=0, page=0, ctx=0, lens=7),
        # A mixed step: prompt chunks and single tokens of requests that have a cached context.
        dict(name="packed_chunks", kind="packed", B=32, lo=1, hi=512, Hq=32, Hkv=8, D=128, cap=0.0,
             window=0, page=16, ctx=4096, lens=8),
        # A few requests behind one system prompt, just begun.
        dict(name="shared_small", kind="shared", B=4, prefix=512, lo=1, hi=60, Hq=32, Hkv=8, D=128,
             cap=0.0, page=16, pad=0, lens=9),
        # Odd sizes: three heads per kv head, D = 64, softcap, and rows that hold no request.
        dict(name="shared_odd", kind="shared", B=37, prefix=1944, lo=1, hi=700, Hq=12, Hkv=4, D=64,
             cap=30.0, page=24, pad=3, lens=10),
        # A full batch behind a system prompt.
        dict(name="shared_batch", kind="shared", B=64, prefix=2048, lo=16, hi=1024, Hq=32, Hkv=8, D=128,
             cap=0.0, page=16, pad=0, lens=11),
        # Many questions about one long document.
        dict(name="shared_long", kind="shared", B=128, prefix=32768, lo=16, hi=2048, Hq=32, Hkv=8,
             D=128, cap=0.0, page=16, pad=0, lens=12),
    ]


def draw(rng) -> dict:
    def log_int(lo: int, hi: int) -> int:
        n = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
        return n if n != 3072 else n + 1

    kind = rng.choice(("plan", "append", "packed", "packed", "shared", "shared"))
    c = dict(kind=kind, B=0, lo=1, hi=0, page=rng.choice((8, 16, 16, 24, 32, 64)), lens=rng.randrange(1 << 30))
    if kind == "plan":
        c.update(B=log_int(1, 1024), hi=log_int(1, 2048), ctx=log_int(16, 8192))
        return c
    D = rng.choice((64, 128, 128))
    Hkv = rng.choice((1, 2, 4, 8))
    if kind == "append":
        c.update(B=log_int(1, 256), hi=log_int(1, 2048), Hkv=Hkv, D=D)
        while work(c)["bytes"] > MAX_BYTES:
            c["B"] //= 2
        return c
    c.update(Hq=Hkv * rng.choice((1, 2, 3, 4, 8)), Hkv=Hkv, D=D, cap=rng.choice((0.0, 0.0, 30.0, 50.0)))
    if kind == "packed":
        c.update(B=log_int(1, 64), hi=log_int(16, 8192), window=0, ctx=0)
        if rng.random() < 0.4:
            c.update(hi=log_int(1, 1024), ctx=log_int(64, 8192))
        else:
            c.update(page=0, window=rng.choice((0, 0, log_int(64, 1024))))
        while (work(c)["flops"] > MAX_FLOPS
               or 4 * c["Hq"] * c["hi"] * (c["hi"] + c["ctx"]) > MAX_SCORES):
            if c["B"] > 1:
                c["B"] -= 1
            else:
                c["hi"] //= 2
    else:
        c.update(B=log_int(1, 128), hi=log_int(1, 2048), pad=0)
        c["prefix"] = -(-log_int(64, 32768) // c["page"]) * c["page"]
        c["prefix"] += c["page"] * (c["prefix"] == 3072)
        c["pad"] = rng.choice((0, 0, c["B"] // 8))
        while work(c)["flops"] > MAX_FLOPS or work(c)["bytes"] > MAX_BYTES:
            c["B"] = max(c["B"] - 4, c["pad"] + 1)
            c["hi"] = max(1, c["hi"] - 64)
    return c


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and cached tokens of each request."""
    rng = random.Random(case["lens"])

    def log_uniform(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    new = [log_uniform(case["lo"], case["hi"]) for _ in range(case["B"])]
    new[0] = case["hi"]
    ctx = case.get("ctx", 0)
    held = [log_uniform(1, ctx) if ctx and rng.random() < 0.85 else 0 for _ in range(case["B"])]
    if ctx:
        held[0] = ctx
    if case["kind"] == "plan" or (case["kind"] == "packed" and case["page"]):
        for b in range(6, case["B"], 7):
            new[b] = 0                      # a request that waits in this step
    for b in range(case["B"] - case.get("pad", 0), case["B"]):
        new[b] = 0                          # a row of a padded batch that holds no request
    return new, held


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


def _plan_tokens(case: dict, new: list[int]) -> int:
    return max(8, _ceil(sum(new), 8) * 8)   # the packed batch is padded to a multiple of eight rows


# -- inputs -----------------------------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=DTYPE)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def pages(n):
        return torch.randperm(n, generator=g, device="cuda").int()

    def offsets(values):
        return torch.nn.functional.pad(ints(values).cumsum(0), (1, 0)).int()

    kind, B, P = case["kind"], case["B"], case["page"]
    new, held = _lengths(case)
    st: dict = {"kind": kind, "page": P}
    if kind == "plan":
        before = [_ceil(h, P) for h in held]
        after = [_ceil(h + n, P) for h, n in zip(held, new)]
        ids = pages(sum(after) + 64)        # the pool has a few pages left over
        table = torch.full((B, max(after) + 1), -1, dtype=torch.int32, device="cuda")
        cached = torch.arange(table.shape[1], device="cuda")[None] < ints(before)[:, None]
        table[cached] = ids[:sum(before)]
        st.update(kv_lens=ints(held), new_lens=ints(new), free=ids[sum(before):].clone(), table=table,
                  tokens=_plan_tokens(case, new))
        return st
    if kind == "append":
        Hkv, D, T = case["Hkv"], case["D"], sum(new)
        n_pages = sum(_ceil(n, P) for n in new) + 64
        pos = torch.cat([torch.arange(n) for n in new]).cuda()
        first = ints([0] + [_ceil(n, P) for n in new][:-1]).cumsum(0)
        owner = torch.repeat_interleave(torch.arange(B, device="cuda"), ints(new), output_size=T)
        slots = pages(n_pages)[first[owner] + pos // P] * P + pos % P
        qkv = normal(T, 6 * Hkv, D)         # four query heads per kv head in front of k and v
        st.update(k=qkv[:, 4 * Hkv:5 * Hkv], v=qkv[:, 5 * Hkv:], slots=slots.int(),
                  k_pool=normal(n_pages, P, Hkv, D), v_pool=normal(n_pages, P, Hkv, D))
        return st

    Hq, Hkv, D, cap = (case[n] for n in ("Hq", "Hkv", "D", "cap"))
    st.update(scale=D ** -0.5, cap=cap)
    if kind == "packed":
        T = sum(new)
        total = [n + h for n, h in zip(new, held)]
        qkv = normal(T, Hq + 2 * Hkv, D)
        st.update(new=new, total=total, window=case["window"], q=qkv[:, :Hq], cu=offsets(new))
        if not P:
            st.update(k=qkv[:, Hq:Hq + Hkv], v=qkv[:, Hq + Hkv:])
            return st
        blocks = [_ceil(t, P) for t in total]
    else:
        prefix = case["prefix"]
        total = [prefix + n if n else 0 for n in new]
        blocks = [_ceil(n, P) for n in new]
        st.update(q=normal(B, Hkv, Hq // Hkv, D), prefix=prefix, longest=max(total))
    # Every request's own pages, from all over the pool; behind a prefix, the prefix's pages come first.
    front = case.get("prefix", 0) // P
    ids = pages(front + sum(blocks) + 8)
    table = torch.zeros((B, front + max(blocks)), dtype=torch.int32, device="cuda")
    table[:, :front] = ids[:front]
    mine = torch.arange(max(blocks), device="cuda")[None] < ints(blocks)[:, None]
    table[:, front:][mine] = ids[front:front + sum(blocks)]
    st.update(table=table, lens=ints(total), k=normal(len(ids), P, Hkv, D), v=normal(len(ids), P, Hkv, D))
    return st


# -- one pass ---------------------------------------------------------------------------------------
def run(state: dict):
    return (_run_own if own else _run_plain)(state)


def _run_own(st: dict):
    from loopfuse_b200 import functional as F
    from loopfuse_b200 import spec as S

    if st["kind"] == "plan":
        plan = F.plan_pages(st["kv_lens"], st["new_lens"], st["free"], st["table"], page_size=st["page"],
                            num_tokens=st["tokens"])
        return {"table": st["table"], "cu_seqlens": plan.cu_seqlens, "seq_lens": plan.seq_lens,
                "slots": plan.slots, "positions": plan.positions, "pages_used": plan.pages_used}
    if st["kind"] == "append":
        F.kv_append_packed(st["k"], st["v"], st["k_pool"], st["v_pool"], st["slots"])
        return {"k_pool": st["k_pool"], "v_pool": st["v_pool"]}
    mods = ()
    if st["cap"]:
        mods = (S.ScoreMod(S.MOD_DIV, st["cap"]), S.ScoreMod(S.MOD_TANH), S.ScoreMod(S.MOD_MUL, st["cap"]))
    if st["kind"] == "packed":
        paged = dict(block_table=st["table"], seq_lens=st["lens"]) if st["page"] else {}
        mask = S.MASK_CAUSAL_WINDOW if st["window"] else S.MASK_CAUSAL
        return F.packed_prefill_attention(st["q"], st["k"], st["v"], st["cu"], scale=st["scale"],
                                          mods=mods, mask_kind=mask, window=st["window"], **paged)
    return F.shared_prefix_decode_attention(st["q"], st["k"], st["v"], st["table"], st["lens"],
                                            st["prefix"], scale=st["scale"], mods=mods,
                                            max_seq_len=st["longest"])


def _run_plain(st: dict):
    return {"plan": _plan, "append": _append, "packed": _packed, "shared": _shared}[st["kind"]](st)


def _plan(st: dict):
    P, held, new, table = st["page"], st["kv_lens"], st["new_lens"], st["table"]
    before, after = (held + P - 1) // P, (held + new + P - 1) // P
    ends, page_ends = new.cumsum(0), (after - before).cumsum(0)
    # Table entries: column c of a row is its (c - before)-th new page.
    col = torch.arange(table.shape[1], device=table.device)[None]
    fresh = (col >= before[:, None]) & (col < after[:, None])
    nth = (page_ends - after)[:, None] + col
    table.copy_(torch.where(fresh, st["free"][nth.clamp(0, len(st["free"]) - 1)], table))
    # Tokens: row t of the packed batch is token t - (its request's first row) of that request.
    t = torch.arange(st["tokens"], device=table.device)
    b = torch.searchsorted(ends, t, right=True).clamp(max=len(new) - 1)
    real = t < ends[-1]
    pos = torch.where(real, held[b] + t - (ends - new)[b], 0)
    slots = torch.where(real, table[b, pos // P] * P + pos % P, -1)
    cu = torch.nn.functional.pad(ends, (1, 0))
    return {"table": table, "cu_seqlens": cu.int(), "seq_lens": held + new, "slots": slots.int(),
            "positions": pos.int(), "pages_used": page_ends[-1:].int()}


def _append(st: dict):
    for rows, pool in ((st["k"], st["k_pool"]), (st["v"], st["v_pool"])):
        pool.view(-1, *pool.shape[2:])[st["slots"].long()] = rows
    return {"k_pool": st["k_pool"], "v_pool": st["v_pool"]}


def _softmax(s, seen):
    """Weights of the visible scores; a row that sees nothing gets zeros."""
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _scores(q, k, st: dict):
    s = (q @ k.transpose(-1, -2)) * st["scale"]
    return torch.tanh(s / st["cap"]) * st["cap"] if st["cap"] else s


def _packed(st: dict):
    q, k, v, P = st["q"], st["k"], st["v"], st["page"]
    Hq, Hkv, dev = q.shape[1], k.shape[-2], q.device
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    at = 0
    for b, (n, m) in enumerate(zip(st["new"], st["total"])):  # one request's scores at a time
        if not n:
            continue
        j = torch.arange(m, device=dev)
        if P:
            page = st["table"][b, j // P].long()
            kb, vb = k[page, j % P], v[page, j % P]
        else:
            kb, vb = k[at:at + n], v[at:at + n]
        qb = q[at:at + n].float().view(n, Hkv, Hq // Hkv, -1).permute(1, 2, 0, 3)     # Hkv, G, n, D
        kb, vb = (x.float().transpose(0, 1).unsqueeze(1) for x in (kb, vb))          # Hkv, 1, m, D
        i = torch.arange(n, device=dev)[:, None] + (m - n)
        seen = j <= i
        if st["window"]:
            seen &= j > i - st["window"]
        o = _softmax(_scores(qb, kb, st), seen) @ vb
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, Hq, -1).to(q.dtype)
        at += n
    return out


def _shared(st: dict):
    q, k, v, P, L, table, lens = (st[n] for n in ("q", "k", "v", "page", "prefix", "table", "lens"))
    B, Hkv, G, D = q.shape
    dev = q.device
    first = table[0, :L // P].long()
    kp, vp = (x[first].flatten(0, 1).float().transpose(0, 1) for x in (k, v))        # Hkv, L, D
    rest = table[:, L // P:].long()
    ko, vo = (x[rest].flatten(1, 2).float().transpose(1, 2) for x in (k, v))         # B, Hkv, n, D
    qf = q.float()
    # The prefix's scores of all requests are one product per kv head.
    sp = _scores(qf.transpose(0, 1).reshape(Hkv, B * G, D), kp, st).view(Hkv, B, G, L).transpose(0, 1)
    s = torch.cat((sp, _scores(qf, ko, st)), dim=-1)
    j = torch.arange(s.shape[-1], device=dev)
    w = _softmax(s, (j[None] < lens[:, None])[:, None, None])
    op = (w[..., :L].transpose(0, 1).reshape(Hkv, B * G, L) @ vp).view(Hkv, B, G, D).transpose(0, 1)
    return (op + w[..., L:] @ vo).to(q.dtype)


# -- what a pass cannot do without ------------------------------------------------------------------
def work(case: dict) -> dict:
    """Each input read once, each output written once; four operations per visible (row, key) pair and
    column."""
    kind, B, P = case["kind"], case["B"], case["page"]
    new, held = _lengths(case)
    T = sum(new)
    if kind == "plan":
        fresh = sum(_ceil(h + n, P) - _ceil(h, P) for h, n in zip(held, new))
        # lengths in and out, a free page read and a table entry written per new page, an entry read for
        # each page that is filled up, slots and positions written
        return {"bytes": 4 * (4 * B + 2 * fresh + B + 2 * _plan_tokens(case, new)), "flops": 0}
    Hkv, D = case["Hkv"], case["D"]
    if kind == "append":
        return {"bytes": 4 * T + 8 * T * Hkv * D, "flops": 0}
    Hq = case["Hq"]
    if kind == "packed":
        pairs, w = 0, case["window"]
        for n, h in zip(new, held):
            if not w or w >= h + n:
                pairs += n * h + n * (n + 1) // 2
            else:
                short = min(n, max(0, w - h))           # rows that see fewer than `window` keys
                pairs += short * h + short * (short + 1) // 2 + (n - short) * w
        keys = sum(n + h for n, h in zip(new, held) if n)
        tables = sum(_ceil(n + h, P) for n, h in zip(new, held) if n) if P else 0
        return {"bytes": 2 * (2 * T * Hq * D + 2 * keys * Hkv * D) + 4 * (tables + B),
                "flops": 4 * Hq * D * pairs}
    L = case["prefix"]
    rows = sum(n > 0 for n in new)
    return {"bytes": 2 * (2 * B * Hq * D + 2 * (L + T) * Hkv * D) + 4 * (_ceil(L + T, P) + B),
            "flops": 4 * Hq * D * (rows * L + T)}


# -- the definition, in 64 bits ---------------------------------------------------------------------
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if st["kind"] == "plan":
        return None
    if st["kind"] == "append":
        got = {}
        for rows, name in ((st["k"], "k_pool"), (st["v"], "v_pool")):
            pool = st[name].double()
            slots = st["slots"].long()
            pool[slots // st["page"], slots % st["page"]] = rows.double()
            got[name] = pool
        return got
    q, k, v = st["q"], st["k"], st["v"]
    P, cap, scale = st["page"], st["cap"], st["scale"]

    def attend(rows, keys, values, seen):
        """[r, D], [m, D], [m, D], and which keys each row sees."""
        s = torch.einsum("rd,md->rm", rows.double(), keys.double()).mul_(scale)
        if cap:
            s = cap * torch.tanh(s / cap)
        s = torch.where(seen, s, -math.inf)
        w = torch.exp(s - torch.logsumexp(s, dim=1)[:, None])
        return torch.einsum("rm,md->rd", w, values.double())

    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    if st["kind"] == "shared":
        for b, m in enumerate(st["lens"].tolist()):
            if not m:
                continue
            j = torch.arange(m, device="cuda")
            row = torch.where(j < st["prefix"], st["table"][0, j // P], st["table"][b, j // P]).long()
            for h in range(k.shape[2]):
                keys, values = k[row, j % P, h], v[row, j % P, h]
                out[b, h] = attend(q[b, h], keys, values, torch.ones_like(j, dtype=torch.bool)[None])
        return out
    at, group = 0, q.shape[1] // k.shape[-2]
    for b, (n, m) in enumerate(zip(st["new"], st["total"])):
        i = torch.arange(n, device="cuda") + m - n
        j = torch.arange(m, device="cuda")
        seen = (i[:, None] >= j) & (i[:, None] - j < (st["window"] or m + 1))
        for h in range(q.shape[1]) if n else ():
            if P:
                page = st["table"][b, j // P].long()
                keys, values = k[page, j % P, h // group], v[page, j % P, h // group]
            else:
                keys, values = k[at:at + n, h // group], v[at:at + n, h // group]
            out[at:at + n, h] = attend(q[at:at + n, h], keys, values, seen)
        at += n
    return out
