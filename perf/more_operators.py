"""The operators of a serving step over a rotated and a 4-bit cache whose speed matters, as data: norm and
rotation of queries and keys, the append that rotates on the way, the 4-bit cache with its way back to
bfloat16, and decode attention over it.

``kind`` of a case:
  norm     norm of every head of q and k, then the rotation of its position, in one pass
  append   q and k rotated, k and v stored to their slots of a bfloat16 cache
  quant    k rotated, k and v stored to a 4-bit cache, and the stored tokens read back as bfloat16: a prompt
           that attends to what the cache holds of it
  gather   keys and values of requests read back from a 4-bit cache: the context of prompt chunks
  decode   one new token per request against a paged 4-bit cache

The lengths of a case's requests are log-uniform between ``lo`` and ``hi``, drawn from ``lens``; the first
request has the longest. Values are bfloat16, N(0, 1) (projections of normalised activations), and q, k and v
of a batch are views of one fused projection. A rotated row turns its first ``rot`` columns.

A row of a 4-bit cache is a record of D / 2 + D / 8 bytes: codes c of 4 bits, then for each group of 32
columns a scale s, then for each group a midpoint z, both bfloat16. Column d stands for z + s (c - 8). The codes
of a key's eight columns 32 g + 8 i .. + 7 are the 32-bit word g of piece i (of four, D / 8 bytes each); those of
a value's four columns 32 g + 4 i .. + 3 the 16-bit word g of piece i (of eight, D / 16 bytes each); the first
column in the lowest bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPE = torch.bfloat16
EPS = 1e-6
MAX_BYTES = 0.8e9      # of a drawn case, as work() counts them
MAX_PADDED = 2.2e9     # fp32 bytes of a batch's keys, padded to the longest, in the plain form


def listed() -> list[dict]:
    return [
        # A decode step of a full batch, before its attention. Latency.
        dict(name="norm_decode", kind="norm", B=64, lo=1, hi=1, ctx=4096, Hq=32, Hkv=8, D=128, rot=128,
             pairs=False, lens=1),
        # A step of prompts of a small model that turns half of its columns, neighbours as pairs.
        dict(name="norm_odd", kind="norm", B=9, lo=3, hi=700, ctx=0, Hq=12, Hkv=4, D=64, rot=32, pairs=True,
             lens=2),
        # A step that takes many prompts in.
        dict(name="norm_prompts", kind="norm", B=32, lo=64, hi=2048, ctx=512, Hq=32, Hkv=8, D=128, rot=128,
             pairs=False, lens=3),
        # The append of a decode step.
        dict(name="append_decode", kind="append", B=64, lo=1, hi=1, ctx=4096, page=16, Hq=32, Hkv=8, D=128,
             rot=128, pairs=False, lens=4),
        # The append of a step of prompts.
        dict(name="append_prompts", kind="append", B=64, lo=16, hi=2048, ctx=0, page=16, Hq=32, Hkv=8, D=128,
             rot=128, pairs=False, lens=5),
        # Three short prompts of a small model. The latency of the two calls.
        dict(name="quant_small", kind="quant", B=3, lo=17, hi=200, ctx=0, page=16, Hkv=4, D=64, rot=64,
             pairs=False, lens=6),
        # A step of prompts over a 4-bit cache.
        dict(name="quant_prompts", kind="quant", B=64, lo=16, hi=2048, ctx=0, page=16, Hkv=8, D=128, rot=128,
             pairs=False, lens=7),
        # The contexts of a step of prompt chunks.
        dict(name="gather_chunks", kind="gather", B=32, lo=64, hi=8192, page=16, Hkv=8, D=128, lens=8),
        # A few requests just begun.
        dict(name="decode_small", kind="decode", B=4, lo=20, hi=500, Hq=32, Hkv=8, D=128, cap=0.0, window=0,
             page=16, pad=0, lens=9),
        # Odd sizes: three heads per kv head, D = 64, softcap, pages of 24, and rows that hold no request.
        dict(name="decode_odd", kind="decode", B=37, lo=1, hi=1500, Hq=12, Hkv=4, D=64, cap=30.0, window=0,
             page=24, pad=3, lens=10),
        # A full batch of running requests.
        dict(name="decode_batch", kind="decode", B=64, lo=256, hi=4096, Hq=32, Hkv=8, D=128, cap=0.0,
             window=0, page=16, pad=0, lens=11),
        # Long documents: what a 4-bit cache is for.
        dict(name="decode_long", kind="decode", B=16, lo=16384, hi=65536, Hq=32, Hkv=8, D=128, cap=0.0,
             window=0, page=16, pad=0, lens=12),
    ]


def draw(rng) -> dict:
    def log_int(lo: int, hi: int) -> int:
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(("norm", "append", "quant", "gather", "decode", "decode", "decode"))
    D = rng.choice((64, 128, 128))
    Hkv = rng.choice((1, 2, 4, 8))
    Hq = Hkv * rng.choice((1, 2, 3, 4, 8))
    c = dict(kind=kind, B=log_int(1, 64), lo=1, hi=log_int(1, 2048), Hkv=Hkv, D=D, lens=rng.randrange(1 << 30))
    if kind != "norm":
        c["page"] = rng.choice((8, 16, 16, 24, 32, 64))
    if kind in ("norm", "append", "quant"):
        c.update(ctx=rng.choice((0, log_int(16, 8192))), rot=rng.choice((D, D, D // 2, D // 4)),
                 pairs=rng.random() < 0.3)
        if kind != "quant":
            c["Hq"] = Hq
    else:
        c["hi"] = log_int(16, 16384)
    if kind == "decode":
        c.update(Hq=Hq, cap=rng.choice((0.0, 0.0, 30.0, 50.0)), window=rng.choice((0, 0, log_int(64, 4096))),
                 pad=rng.choice((0, 0, c["B"] // 8)))
    while work(c)["bytes"] > MAX_BYTES or 4 * c["B"] * c["hi"] * Hkv * D > MAX_PADDED:
        if c["B"] > 1:
            c["B"] = max(1, c["B"] // 2)
        else:
            c["hi"] //= 2
        if "pad" in c:
            c["pad"] = min(c["pad"], c["B"] // 2)
    return c


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Tokens of each request, and tokens that it had before."""
    rng = random.Random(case["lens"])

    def log_uniform(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    new = [log_uniform(case["lo"], case["hi"]) for _ in range(case["B"])]
    new[0] = case["hi"]
    ctx = case.get("ctx", 0)
    held = [log_uniform(1, ctx) if ctx else 0 for _ in range(case["B"])]
    for b in range(case["B"] - case.get("pad", 0), case["B"]):
        new[b] = 0                          # a row of a padded batch that holds no request
    return new, held


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


# -- the rows of a 4-bit cache ----------------------------------------------------------------------
def _pieces(codes, value: bool):
    """Codes [..., D] in the order of their columns -> [..., D] in the order of a record, four (eight) to a
    32-bit (16-bit) word; the same the other way round is _columns."""
    D = codes.shape[-1]
    a, b = (8, 4) if value else (4, 8)
    return codes.view(*codes.shape[:-1], D // 32, a, b).transpose(-3, -2).reshape(codes.shape)


def _columns(codes, value: bool):
    D = codes.shape[-1]
    a, b = (8, 4) if value else (4, 8)
    return codes.view(*codes.shape[:-1], a, D // 32, b).transpose(-3, -2).reshape(codes.shape)


def _encode(x, value: bool):
    """float32 [..., D] -> uint8 [..., D / 2 + D / 8]."""
    g = x.unflatten(-1, (-1, 32))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((high - low) * (1.0 / 15.0)).to(DTYPE).float()
    z = (low + 8.0 * s).to(DTYPE).float()
    inv = torch.where(s > 0, 1.0 / s, 0.0)
    codes = (torch.round((g - z) * inv) + 8.0).clamp(0.0, 15.0).to(torch.uint8).flatten(-2)
    codes = _pieces(codes, value)
    meta = torch.cat((s.squeeze(-1), z.squeeze(-1)), -1).to(DTYPE).view(torch.uint8)
    return torch.cat((codes[..., 0::2] | (codes[..., 1::2] << 4), meta), -1)


def _decode(rows, D: int, value: bool):
    """uint8 [..., D / 2 + D / 8] -> float32 [..., D]."""
    packed = rows[..., :D // 2]
    codes = _columns(torch.stack((packed & 15, packed >> 4), -1).flatten(-2), value)
    s, z = rows[..., D // 2:].contiguous().view(DTYPE).float().chunk(2, -1)
    g = codes.unflatten(-1, (-1, 32)).float() - 8.0
    return (z[..., None] + s[..., None] * g).flatten(-2)


# -- inputs -----------------------------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=DTYPE):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def pages(n):
        return torch.randperm(n, generator=g, device="cuda").int()

    kind, B, P, Hkv, D = case["kind"], case["B"], case.get("page", 0), case["Hkv"], case["D"]
    new, held = _lengths(case)
    T = sum(new)
    st: dict = {"kind": kind, "page": P, "D": D}
    if kind in ("norm", "append", "quant"):
        rot = case["rot"]
        owner = torch.repeat_interleave(torch.arange(B, device="cuda"), ints(new), output_size=T)
        first = torch.nn.functional.pad(ints(new).cumsum(0), (1, 0))
        pos = ints(held)[owner] + torch.arange(T, device="cuda") - first[owner]
        angles = torch.arange(max(n + h for n, h in zip(new, held)), device="cuda").double()[:, None] \
            * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda").double() / rot)
        st.update(positions=pos.int(), table=torch.cat((angles.cos(), angles.sin()), -1).float(),
                  rot=rot, pairs=case["pairs"])
        Hq = case.get("Hq", 4 * Hkv)
        qkv = normal(T, Hq + 2 * Hkv, D)
        st.update(q=qkv[:, :Hq], k=qkv[:, Hq:Hq + Hkv], v=qkv[:, Hq + Hkv:])
        if kind == "norm":
            st.update(qw=1 + 0.1 * normal(D), kw=1 + 0.1 * normal(D))
            return st
    # Every request's own pages, from all over the pool.
    blocks = [_ceil(n, P) for n in new]
    ids = pages(sum(blocks) + 8)
    table = torch.zeros((B, max(blocks)), dtype=torch.int32, device="cuda")
    mine = torch.arange(max(blocks), device="cuda")[None] < ints(blocks)[:, None]
    table[mine] = ids[:sum(blocks)]
    if kind in ("append", "quant"):
        at = torch.arange(T, device="cuda") - first[owner]
        st["slots"] = (table[owner, at // P] * P + at % P).int()
    if kind == "append":
        st.update(k_pool=normal(len(ids), P, Hkv, D), v_pool=normal(len(ids), P, Hkv, D))
        return st
    # [pages, page, Hkv, record], a head's rows of a page next to each other.
    for name in ("k_pool", "v_pool"):
        pool = torch.zeros((len(ids), Hkv, P, D // 2 + D // 8), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 28) // (P * Hkv * D))
        for i in range(0, len(ids) if kind != "quant" else 0, step):
            part = pool[i:i + step]
            part.copy_(_encode(normal(*part.shape[:3], D).float(), name == "v_pool"))
        st[name] = pool.transpose(1, 2)
    st.update(blocks=table)
    if kind == "decode":
        Hq = case["Hq"]
        st.update(q=normal(B, Hkv, Hq // Hkv, D), lens=ints(new), longest=max(new), scale=D ** -0.5,
                  cap=case["cap"], window=case["window"])
    else:
        st.update(cu=torch.nn.functional.pad(ints(new).cumsum(0), (1, 0)).int(), tokens=T)
    return st


# -- one pass ---------------------------------------------------------------------------------------
def run(state: dict):
    return (_run_own if own else _run_plain)(state)


def _run_own(st: dict):
    from loopfuse_b200 import functional as F
    from loopfuse_b200 import spec as S

    kind = st["kind"]
    if kind == "norm":
        q, k = F.qk_norm_rotary(st["q"], st["k"], st["positions"], st["table"], q_weight=st["qw"],
                                k_weight=st["kw"], eps=EPS, interleaved=st["pairs"])
        return {"q": q, "k": k}
    if kind == "append":
        q = F.kv_append_rotary(st["k"], st["v"], st["k_pool"], st["v_pool"], st["slots"], st["positions"],
                               st["table"], q=st["q"], interleaved=st["pairs"])
        return {"q": q, "k_pool": st["k_pool"], "v_pool": st["v_pool"]}
    if kind in ("quant", "gather"):
        if kind == "quant":
            F.kv_append_rotary(st["k"], st["v"], st["k_pool"], st["v_pool"], st["slots"], st["positions"],
                               st["table"], interleaved=st["pairs"])
        k, v = F.kv_gather_4bit(st["k_pool"], st["v_pool"], st["blocks"], st["cu"], st["tokens"])
        return {"k": k, "v": v}
    mods = ()
    if st["cap"]:
        mods = (S.ScoreMod(S.MOD_DIV, st["cap"]), S.ScoreMod(S.MOD_TANH), S.ScoreMod(S.MOD_MUL, st["cap"]))
    return F.decode_attention_4bit(st["q"], st["k_pool"], st["v_pool"], st["blocks"], st["lens"],
                                   window=st["window"], max_seq_len=st["longest"], scale=st["scale"], mods=mods)


def _run_plain(st: dict):
    return {"norm": _norm, "append": _append, "quant": _quant, "gather": _gather, "decode": _attend}[st["kind"]](st)


def _turn(x, st: dict):
    """The rotation of each row's position, in 32 bits: [T, H, D]."""
    rot = st["rot"]
    cos, sin = st["table"][st["positions"]][:, None].chunk(2, -1)
    if st["pairs"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _norm(st: dict):
    def one(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        return _turn(x, st).to(DTYPE)

    return {"q": one(st["q"], st["qw"]), "k": one(st["k"], st["kw"])}


def _append(st: dict):
    page, slot = (st["slots"] // st["page"]).long(), (st["slots"] % st["page"]).long()
    st["k_pool"][page, slot] = _turn(st["k"].float(), st).to(DTYPE)
    st["v_pool"][page, slot] = st["v"]
    return {"q": _turn(st["q"].float(), st).to(DTYPE), "k_pool": st["k_pool"], "v_pool": st["v_pool"]}


def _quant(st: dict):
    page, slot = (st["slots"] // st["page"]).long(), (st["slots"] % st["page"]).long()
    st["k_pool"][page, slot] = _encode(_turn(st["k"].float(), st), False)
    st["v_pool"][page, slot] = _encode(st["v"].float(), True)
    return _gather(st)


def _gather(st: dict):
    t = torch.arange(st["tokens"], device=st["cu"].device, dtype=torch.int32)
    b = torch.searchsorted(st["cu"][1:], t, right=True)
    at = (t - st["cu"][b]).long()
    page, slot = st["blocks"][b, at // st["page"]].long(), at % st["page"]
    return {"k": _decode(st["k_pool"][page, slot], st["D"], False).to(DTYPE),
            "v": _decode(st["v_pool"][page, slot], st["D"], True).to(DTYPE)}


def _attend(st: dict):
    q, lens, P, D = st["q"].float(), st["lens"][:, None], st["page"], st["D"]
    j = torch.arange(st["longest"], device=q.device)
    page, slot = st["blocks"][:, j // P].long(), (j % P)[None]
    k = _decode(st["k_pool"][page, slot], D, False).transpose(1, 2)                  # B, Hkv, n, D
    s = (q @ k.transpose(-1, -2)) * st["scale"]
    del k
    if st["cap"]:
        s = torch.tanh(s / st["cap"]) * st["cap"]
    seen = j[None] < lens
    if st["window"]:
        seen &= j[None] >= lens - st["window"]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    return (p @ _decode(st["v_pool"][page, slot], D, True).transpose(1, 2)).to(DTYPE)


# -- what a pass cannot do without ------------------------------------------------------------------
def work(case: dict) -> dict:
    """Each input read once, each output written once; six operations per turned pair, four per visible
    (row, key) pair and column."""
    kind, Hkv, D = case["kind"], case["Hkv"], case["D"]
    new, held = _lengths(case)
    T = sum(new)
    if kind in ("norm", "append", "quant"):
        rot = case["rot"]
        # the rows of the table that the positions name, and the positions (and slots)
        places = 4 * rot * min(T, max(n + h for n, h in zip(new, held))) + 4 * T
        heads = case.get("Hq", 0) + Hkv
        turned = 3 * T * heads * rot
        if kind == "norm":
            return {"bytes": places + 4 * T * heads * D + 4 * D, "flops": turned + 4 * T * heads * D}
        if kind == "append":
            return {"bytes": places + 4 * T + 4 * T * (heads + Hkv) * D, "flops": turned}
    records = 2 * T * Hkv * (D // 2 + D // 8)
    if kind == "quant":
        # k and v read, their records written, what these stand for written
        return {"bytes": places + 4 * T + 4 * T * Hkv * D + records + 4 * T * Hkv * D,
                "flops": turned + 2 * T * Hkv * D}
    entries = sum(_ceil(n, case["page"]) for n in new)
    if kind == "gather":
        return {"bytes": records + 4 * T * Hkv * D + 4 * (entries + case["B"]), "flops": 4 * T * Hkv * D}
    w = case["window"]
    keys = sum(min(n, w) if w else n for n in new)
    records = 2 * keys * Hkv * (D // 2 + D // 8)
    return {"bytes": records + 4 * case["B"] * case["Hq"] * D + 4 * (_ceil(keys, case["page"]) + case["B"]),
            "flops": 4 * case["Hq"] * D * keys}


# -- the definition, in 64 bits ---------------------------------------------------------------------
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    kind, D, P = st["kind"], st["D"], st["page"]

    def rotated(x):
        """[T, H, D] in float64; columns as the real and imaginary parts of numbers that are turned."""
        h = st["rot"] // 2
        re = torch.arange(h, device="cuda") * (2 if st["pairs"] else 1)
        im = re + (1 if st["pairs"] else h)
        row = st["table"][st["positions"].long()].double()
        by = torch.complex(row[:, :h], row[:, h:])[:, None]
        y = x.clone()
        num = torch.complex(x[..., re], x[..., im]) * by
        y[..., re], y[..., im] = num.real, num.imag
        return y

    def stored(x, bits):
        """What groups of 32 columns of x stand for in 4 bits."""
        out = torch.empty_like(x)
        for c in range(0, D, 32):
            g = x[..., c:c + 32]
            low = g.min(-1, keepdim=True).values
            s = ((g.max(-1, keepdim=True).values - low) / 15).to(bits).double()
            z = (low + 8 * s).to(bits).double()
            code = torch.where(s > 0, torch.round((g - z) / s), 0.0).clamp(-8, 7)
            out[..., c:c + 32] = z + s * code
        return out

    def read(pool, page, slot, value):
        """Records of tokens -> [..., Hkv, D] in float64, column by column."""
        rows = pool[page, slot]
        numbers = rows[..., D // 2:].contiguous().view(DTYPE).double()
        out = torch.empty((*rows.shape[:-1], D), dtype=torch.float64, device="cuda")
        for d in range(D):
            g, r = divmod(d, 32)
            i, n = divmod(r, 4 if value else 8)
            nibble = (i * (D // 32) + g) * (4 if value else 8) + n
            code = (rows[..., nibble // 2] >> (4 * (nibble % 2))) & 15
            out[..., d] = numbers[..., D // 32 + g] + numbers[..., g] * (code.double() - 8)
        return out

    if kind == "norm":
        got = {}
        for name in ("q", "k"):
            x = st[name].double()
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
            got[name] = rotated(x * st[name + "w"].double())
        return got
    if kind == "append":
        got = {"q": rotated(st["q"].double())}
        for name, rows in (("k_pool", rotated(st["k"].double())), ("v_pool", st["v"].double())):
            got[name] = st[name].double()
            got[name].view(-1, *rows.shape[1:])[st["slots"].long()] = rows
        return got
    if kind == "quant":
        return {"k": stored(rotated(st["k"].double()), DTYPE), "v": stored(st["v"].double(), DTYPE)}
    if kind == "gather":
        parts = {"k": [], "v": []}
        cu = st["cu"].tolist()
        for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
            j = torch.arange(hi - lo, device="cuda")
            page, slot = st["blocks"][b].long()[j // P], j % P
            for name in parts:
                parts[name].append(read(st[name + "_pool"], page, slot, name == "v"))
        return {name: torch.cat(x) for name, x in parts.items()}
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lens"].tolist()):
        if not n:
            continue
        j = torch.arange(max(0, n - st["window"]) if st["window"] else 0, n, device="cuda")
        page, slot = st["blocks"][b].long()[j // P], j % P
        keys, values = read(st["k_pool"], page, slot, False), read(st["v_pool"], page, slot, True)
        s = torch.einsum("hgd,nhd->hgn", st["q"][b].double(), keys) * st["scale"]
        if st["cap"]:
            s = st["cap"] * torch.tanh(s / st["cap"])
        weights = torch.exp(s - torch.logsumexp(s, -1, keepdim=True))
        out[b] = torch.einsum("hgn,nhd->hgd", weights, values)
    return out
