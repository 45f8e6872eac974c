"""Norm and rotation, the append that rotates, and the 4-bit cache's rows, against plain forms.

Where only a rotation is done each step is rounded once in float32, so results are compared bit for bit with the
same steps in torch. A norm's sum has an order of its own: there the tolerance is a rounding to the result's type
(bf16 2^-8 of the value) and 2^-19 of the turned columns' size for the arithmetic in float32 (a sum of 128 squares
in 12 steps, a reciprocal root within 2^-22, four products and a sum: under 32 half steps of 2^-24)."""
import pytest
import torch

from loopfuse_b200 import _native
from loopfuse_b200 import functional as F
from tests import cache4

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def rows(T, Hq, Hkv, D, seed, amp=1.0):
    """q, k, v as views of one projection."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, Hq + 2 * Hkv, D, generator=g) * amp).to(BF16).cuda()
    return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]


def positions_of(T, limit, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, limit, (T,), generator=g, dtype=torch.int32)
    p[0], p[-1] = 0, limit - 1
    return p.cuda()


SHAPES = [  # T, Hq, Hkv, D, turned columns, pairs
    (1, 1, 1, 64, 64, False), (1, 32, 8, 128, 128, False), (5, 3, 1, 64, 16, False), (7, 6, 2, 128, 96, True),
    (33, 5, 5, 128, 32, False), (129, 12, 4, 64, 32, True), (257, 8, 2, 64, 48, False), (1031, 32, 8, 128, 128, True),
    (2500, 7, 3, 128, 64, False)]


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,pairs", SHAPES)
def test_rotation_bits(T, Hq, Hkv, D, rot, pairs):
    q, k, _ = rows(T, Hq, Hkv, D, T)
    table, pos = cache4.rotary_table(4096, rot), positions_of(T, 4096, T)
    cos, sin = table[pos.long()].chunk(2, -1)
    st = F.new_status("cuda")
    got = F.qk_norm_rotary(q, k, pos, table, interleaved=pairs, status=st)
    for x, y in zip((q, k), got):
        assert y.is_contiguous() and torch.equal(y, cache4.turn(x.float(), cos, sin, pairs).to(BF16))
    F.check_status(st)
    # in place, and into given outputs of other strides
    q_out = torch.full((T, Hq, 2 * D), 7.0, dtype=BF16, device="cuda")
    both = F.qk_norm_rotary(q, k, pos, table, interleaved=pairs, q_out=q_out[..., D:], k_out=k)
    assert both[1] is k or both[1].data_ptr() == k.data_ptr()
    assert torch.equal(both[0], got[0]) and torch.equal(k, got[1]) and (q_out[..., :D] == 7).all()


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,pairs", SHAPES)
@pytest.mark.parametrize("kind", ["bf16", "f32", "q only", "k only"])
def test_norm_and_rotation(T, Hq, Hkv, D, rot, pairs, kind):
    q, k, _ = rows(T, Hq, Hkv, D, T + 1, amp=3.0)
    k[T // 2] = 0                                        # a row whose norm is eps alone
    table, pos = cache4.rotary_table(2048, rot), positions_of(T, 2048, T)
    g = torch.Generator().manual_seed(9)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(torch.float32 if kind == "f32" else BF16).cuda() for _ in "qk"]
    if kind == "q only":
        w[1] = None
    if kind == "k only":
        w[0] = None
    got = F.qk_norm_rotary(q, k, pos, table, q_weight=w[0], k_weight=w[1], eps=1e-5, interleaved=pairs)
    cos, sin = table[pos.long()].double().chunk(2, -1)
    for x, y, wt in zip((q, k), got, w):
        x = x.double()
        if wt is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * wt.double()
        want = cache4.turn(x, cos, sin, pairs)
        size = cache4.turn(x.abs(), cos.abs(), -sin.abs(), pairs).abs() + x.abs()
        assert ((y.double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -19 * size).all()
        if wt is None:
            assert torch.equal(y, cache4.turn(x.float(), cos.float(), sin.float(), pairs).to(BF16))


def test_norm_of_rows_with_infinities_and_nan_stays_in_its_row():
    q, k, _ = rows(6, 4, 2, 64, 3)
    q[2, 1, 5], q[3, 0, 7] = float("nan"), float("inf")
    table, w = cache4.rotary_table(16, 64), torch.ones(64, device="cuda")
    pos = torch.arange(6, dtype=torch.int32, device="cuda")
    y, _ = F.qk_norm_rotary(q, k, pos, table, q_weight=w)
    bad = torch.zeros(6, 4, dtype=torch.bool)
    bad[2, 1] = bad[3, 0] = True
    assert torch.equal((~y.isfinite()).any(-1).cpu(), bad)


def test_positions_outside_the_table_take_the_nearest_row():
    q, k, _ = rows(4, 2, 2, 64, 4)
    table = cache4.rotary_table(8, 64)
    pos = torch.tensor([-1, 8, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    st = F.new_status("cuda")
    got = F.qk_norm_rotary(q, k, pos, table, status=st)
    want = F.qk_norm_rotary(q, k, torch.tensor([0, 7, 7, 0], dtype=torch.int32, device="cuda"), table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(RuntimeError, match="rotation table"):
        F.check_status(st)


def pool_of(bits, pages, page, Hkv, D, layout):
    """A pair of pools full of a pattern, and the same as it was."""
    width, dtype = (D, BF16) if bits == 16 else (D // 2 + D // 8, torch.uint8)
    shape = {"page": (pages, page, Hkv), "head": (pages, Hkv, page), "slots": (page, pages, Hkv)}[layout]
    full = [torch.randint(0, 200, (*shape, width), device="cuda", dtype=torch.uint8).to(dtype) for _ in "kv"]
    perm = {"page": (0, 1, 2, 3), "head": (0, 2, 1, 3), "slots": (1, 0, 2, 3)}[layout]
    pools = [p.permute(perm) for p in full]
    return pools, [p.clone() for p in pools]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,pairs,page,layout", [
    (1, 4, 1, 64, 64, False, 16, "head"), (1, 32, 8, 128, 128, False, 16, "page"), (19, 0, 3, 128, 64, True, 1, "head"),
    (70, 6, 2, 64, 16, False, 24, "slots"), (777, 8, 5, 128, 128, False, 16, "head"),
    (1500, 0, 8, 64, 32, True, 64, "page"), (2049, 12, 4, 128, 96, False, 7, "slots"),
    (300, 4, 2, 128, 64, False, 16, "head"), (90, 0, 2, 128, 32, False, 16, "head"), (333, 2, 1, 128, 16, False, 8, "page"),
    (410, 2, 3, 64, 32, False, 16, "head"), (2100, 9, 3, 64, 48, False, 16, "slots"), (65, 5, 2, 128, 16, True, 32, "head"),
    (2300, 8, 8, 128, 48, True, 16, "page"), (2500, 16, 8, 64, 64, True, 16, "head")])
def test_append_bits(bits, T, Hq, Hkv, D, rot, pairs, page, layout):
    q, k, v = rows(T, max(Hq, 1), Hkv, D, T + 5)
    k[0], v[0] = 2.5, -0.75                              # groups of one value
    k[-1, :, :5] = 100.0                                 # columns far from the others
    table, pos = cache4.rotary_table(3000, rot), positions_of(T, 3000, T)
    pages = -(-(T + 3) // page) + 2
    (k_pool, v_pool), before = pool_of(bits, pages, page, Hkv, D, layout)
    g = torch.Generator().manual_seed(T)
    slots = torch.randperm(pages * page, generator=g)[:T].int().cuda()
    if T > 4:
        slots[T // 2] = -1                               # a row of the padding
        slots[T // 3] = -2 ** 31
    st = F.new_status("cuda")
    got = F.kv_append_rotary(k, v, k_pool, v_pool, slots, pos, table, q=q if Hq else None, interleaved=pairs, status=st)
    F.check_status(st)
    cos, sin = table[pos.long()].chunk(2, -1)
    real = slots >= 0
    at = slots[real].long()
    for x, pool, old, value in ((cache4.turn(k.float(), cos, sin, pairs), k_pool, before[0], False),
                                (v.float(), v_pool, before[1], True)):
        old[at // page, at % page] = (cache4.encode(x, value) if bits == 4 else x.to(BF16))[real]
        assert torch.equal(pool, old)
    if Hq:
        assert torch.equal(got, cache4.turn(q.float(), cos, sin, pairs).to(BF16))
    else:
        assert got is None


@pytest.mark.parametrize("D", [64, 128])
def test_append_with_norm_to_four_bits(D):
    """A normed row's bits depend on the order of a sum; what they stand for is within half a step of the value,
    or where the largest or smallest code is not enough, within the roundings of scale (15 of 2^-8, at most
    0.06 s) and midpoint (2^-8 |z|)."""
    T, Hkv = 301, 3
    _, k, v = rows(T, 1, Hkv, D, 21)
    w = (1 + 0.2 * torch.randn(D, generator=torch.Generator().manual_seed(2))).cuda()
    table, pos = cache4.rotary_table(512, D), positions_of(T, 512, 3)
    k_pool, v_pool = F.kv_cache_4bit(40, 8, Hkv, D)
    F.kv_append_rotary(k, v, k_pool, v_pool, torch.arange(T, dtype=torch.int32, device="cuda"), pos, table,
                       k_weight=w, eps=1e-6)
    cos, sin = table[pos.long()].double().chunk(2, -1)
    x = k.double()
    x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    for want, pool, value in ((cache4.turn(x, cos, sin, False), k_pool, False), (v.double(), v_pool, True)):
        _, s, z = cache4.parts(pool.reshape(-1, *pool.shape[2:])[:T], D, value)
        off = (cache4.decode(pool.reshape(-1, *pool.shape[2:])[:T], D, value) - want).abs()
        assert (off <= torch.maximum(0.5 * s + 2 ** -19 * want.abs().amax(), 0.06 * s + 2 ** -8 * z.abs())).all()
    assert torch.equal(v_pool.reshape(-1, *v_pool.shape[2:])[:T], cache4.encode(v.float(), True))


def test_groups_that_are_not_finite_stay_by_themselves():
    _, k, v = rows(4, 1, 2, 128, 30)
    v[0, 0, 3], v[1, 1, 40], v[2, 0, 127] = float("nan"), float("inf"), -float("inf")
    v[3, 0, 32], v[3, 0, 33] = 3e38, -3e38               # their range is no fp32
    k_pool, v_pool = F.kv_cache_4bit(1, 4, 2, 128)
    i = torch.arange(4, dtype=torch.int32, device="cuda")
    F.kv_append_rotary(k, v, k_pool, v_pool, i, i, cache4.rotary_table(4, 128))
    y = cache4.decode(v_pool[0], 128, True)
    bad = torch.zeros(4, 2, 4, dtype=torch.bool)
    bad[0, 0, 0] = bad[1, 1, 1] = bad[2, 0, 3] = bad[3, 0, 1] = True
    finite = y.isfinite().unflatten(-1, (4, 32)).cpu()
    assert torch.equal(~finite.all(-1), bad) and torch.equal(~finite.any(-1), bad)


def test_slots_outside_the_pool_are_reported_and_not_written():
    for bits in (4, 16):
        q, k, v = rows(3, 2, 2, 64, 8)
        (k_pool, v_pool), before = pool_of(bits, 2, 4, 2, 64, "head")
        i = torch.arange(3, dtype=torch.int32, device="cuda")
        st = F.new_status("cuda")
        got = F.kv_append_rotary(k, v, k_pool, v_pool, torch.tensor([8, 2 ** 31 - 1, -1], dtype=torch.int32,
                                 device="cuda"), i, cache4.rotary_table(4, 64), q=q, status=st)
        assert torch.equal(k_pool, before[0]) and torch.equal(v_pool, before[1])
        assert torch.equal(got, F.qk_norm_rotary(q, k, i, cache4.rotary_table(4, 64))[0])
        with pytest.raises(RuntimeError, match="page id"):
            F.check_status(st)


@pytest.mark.parametrize("D,Hkv,page,layout,lens,lead,tail", [
    (64, 1, 16, "head", [1], 0, 0), (128, 8, 16, "head", [17, 0, 200, 33], 0, 5), (128, 3, 1, "page", [5, 9], 2, 0),
    (64, 4, 24, "slots", [0, 0, 100, 1, 0, 61, 0], 0, 3), (128, 2, 64, "head", [1000, 3, 0], 4, 1)])
def test_gather_bits(D, Hkv, page, layout, lens, lead, tail):
    B, T = len(lens), lead + sum(lens) + tail
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    (k_pool, v_pool), _ = pool_of(4, pages, page, Hkv, D, layout)
    for pool in (k_pool, v_pool):                        # (random bytes are no bf16 that one compares)
        pool[..., D // 2:] = torch.randn(*pool.shape[:3], D // 16, device="cuda").bfloat16().view(torch.uint8)
    table = torch.full((B, max(need) + 1), 10 ** 6, dtype=torch.int32)
    ids = torch.randperm(pages).int()
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    table = table.cuda()
    cu = (lead + torch.tensor([0] + lens).cumsum(0)).int().cuda()
    out = [torch.full((T, Hkv, D), 5.0, dtype=BF16, device="cuda") for _ in "kv"]
    st = F.new_status("cuda")
    k, v = F.kv_gather_4bit(k_pool, v_pool, table, cu, T, k_out=out[0], v_out=out[1], status=st)
    F.check_status(st)
    t = torch.arange(T)
    mine = (t >= lead) & (t < lead + sum(lens))
    owner = torch.repeat_interleave(torch.arange(B), torch.tensor(lens)).cuda()
    j = torch.cat([torch.arange(n) for n in lens]).cuda()
    for got, pool, value in ((k, k_pool, False), (v, v_pool, True)):
        rec = pool[table[owner, j // page].long(), j % page]
        # (scale times code is exact in float32, so one rounding there, then the one to bf16)
        assert torch.equal(got[mine], cache4.decode(rec, D, value).float().to(BF16))
        assert (got[~mine] == 5).all()


def test_gather_reports_pages_that_are_not_there():
    k_pool, v_pool = F.kv_cache_4bit(4, 4, 2, 64)
    k_pool[..., 36:] = 63
    v_pool[..., 36:] = 63
    table = torch.tensor([[0, -1], [7, 1]], dtype=torch.int32, device="cuda")
    st = F.new_status("cuda")
    k, v = F.kv_gather_4bit(k_pool, v_pool, table, torch.tensor([0, 8, 20], dtype=torch.int32, device="cuda"), 20,
                            status=st)
    assert (k[:4] != 0).all() and (k[4:8] == 0).all() and (k[8:12] == 0).all() and (v[12:16] != 0).all()
    assert (v[16:] == 0).all()                            # more keys than the table has blocks for
    with pytest.raises(RuntimeError, match="page id"):
        F.check_status(st)


@pytest.mark.parametrize("cu", [[0, -5, 4], [3, 1, 8], [-2 ** 31, 2, 2 ** 31 - 1], [9, 9, 9], [0, 20, 4]])
def test_gather_of_offsets_that_make_no_sense_stays_in_its_rows(cu):
    k_pool, v_pool = F.kv_cache_4bit(4, 4, 2, 64)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    out = torch.full((3, 8, 2, 64), 5.0, dtype=BF16, device="cuda")
    F.kv_gather_4bit(k_pool, v_pool, table, torch.tensor(cu, dtype=torch.int32, device="cuda"), 8, k_out=out[1],
                     v_out=out[1].clone(), status=F.new_status("cuda"))
    assert (out[0] == 5).all() and (out[2] == 5).all()


def test_offsets_past_32_bits():
    """A cache of more than 4 GB, whose last page's first byte lies behind 2^32."""
    Hkv, D, page = 8, 128, 64
    pages = (1 << 32) // (Hkv * page * 80) + 3
    k_pool = torch.empty(pages, Hkv, page, 80, dtype=torch.uint8, device="cuda").transpose(1, 2)
    v_pool = torch.empty_like(k_pool)
    _, k, v = rows(page, 1, Hkv, D, 40)
    i = torch.arange(page, dtype=torch.int32, device="cuda")
    table = cache4.rotary_table(page, D)
    F.kv_append_rotary(k, v, k_pool, v_pool, i + (pages - 1) * page, i, table)
    cos, sin = table.chunk(2, -1)
    assert torch.equal(k_pool[-1], cache4.encode(cache4.turn(k.float(), cos, sin, False), False))
    assert torch.equal(v_pool[-1], cache4.encode(v.float(), True))
    blocks = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, page], dtype=torch.int32, device="cuda")
    assert torch.equal(F.kv_gather_4bit(k_pool, v_pool, blocks, cu, page)[1],
                       cache4.decode(v_pool[-1], D, True).float().to(BF16))


def test_refusals():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=BF16, device="cuda")  # noqa: E731
    table = torch.zeros(8, 64, device="cuda")
    q, k = bf(2, 4, 64), bf(2, 2, 64)
    k_pool, v_pool = F.kv_cache_4bit(4, 4, 2, 64)
    k16 = bf(4, 4, 2, 64)
    pos, slots = i32(0, 1), i32(0, 1)
    blocks = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    big = bf(4, 4, 64)
    bad = [
        (TypeError, lambda: F.qk_norm_rotary(q.float(), k, pos, table)),
        (TypeError, lambda: F.qk_norm_rotary(q, k, pos.long(), table)),
        (TypeError, lambda: F.qk_norm_rotary(q, k, pos, table.bfloat16())),
        (TypeError, lambda: F.qk_norm_rotary(q, k, pos, table, q_weight=torch.zeros(64, device="cuda").double())),
        (ValueError, lambda: F.qk_norm_rotary(q, k, pos, table, q_weight=torch.zeros(32, device="cuda"))),
        (ValueError, lambda: F.qk_norm_rotary(q, bf(3, 2, 64), pos, table)),
        (ValueError, lambda: F.qk_norm_rotary(q, k, i32(0), table)),
        (ValueError, lambda: F.qk_norm_rotary(q, k, pos, table[:0])),
        (ValueError, lambda: F.qk_norm_rotary(q, k, pos, table, q_out=bf(2, 3, 64))),
        (ValueError, lambda: F.qk_norm_rotary(big[:2], k, pos, table, q_out=big[1:3])),   # across its input
        (ValueError, lambda: F.qk_norm_rotary(q, k, pos, table, q_out=bf(2, 1, 64).expand(2, 4, 64))),
        (ValueError, lambda: F.qk_norm_rotary(q, k, pos, table, q_out=bf(4, 64).expand(2, 4, 64))),
        (_native.LfError, lambda: F.qk_norm_rotary(q, k, pos, table[:, :24])),
        (_native.LfError, lambda: F.qk_norm_rotary(q, k, pos, table, eps=-1.0, q_weight=table[0])),
        (ValueError, lambda: F.kv_append_rotary(k, bf(2, 1, 64), k_pool, v_pool, slots, pos, table)),
        (ValueError, lambda: F.kv_append_rotary(k, k, k_pool, v_pool, i32(0), pos, table)),
        (ValueError, lambda: F.kv_append_rotary(k, k, k_pool, v_pool[:3], slots, pos, table)),
        (TypeError, lambda: F.kv_append_rotary(k, k, k_pool, k16, slots, pos, table)),
        (TypeError, lambda: F.kv_append_rotary(k, k, k16, v_pool, slots, pos, table)),
        (ValueError, lambda: F.kv_append_rotary(bf(2, 2, 128), bf(2, 2, 128), k_pool, v_pool, slots, pos, table)),
        (ValueError, lambda: F.kv_append_rotary(k, k, k_pool, v_pool, slots, pos, table, q_weight=table[0])),
        (ValueError, lambda: F.kv_append_rotary(k, k, k_pool, v_pool, slots, pos, table, q_out=q)),
        (_native.LfError, lambda: F.kv_append_rotary(k, k, *(p.view(torch.uint8)[..., :40] for p in (
            torch.zeros(4, 4, 2, 44, dtype=torch.uint8, device="cuda"),) * 2), slots, pos, table)),
        (TypeError, lambda: F.kv_gather_4bit(k16, k16, blocks, i32(0, 4), 4)),
        (ValueError, lambda: F.kv_gather_4bit(k_pool, v_pool, blocks, i32(0, 4, 4), 4)),
        (ValueError, lambda: F.kv_gather_4bit(k_pool, v_pool, blocks, i32(0, 4), -1)),
        (ValueError, lambda: F.kv_gather_4bit(k_pool, v_pool, blocks, i32(0, 4), 4, k_out=bf(5, 2, 64))),
        (ValueError, lambda: F.kv_gather_4bit(k_pool, v_pool, blocks, i32(0, 4), 4, k_out=big[:, :2], v_out=big[:, :2])),
        (ValueError, lambda: F.kv_gather_4bit(k_pool, v_pool, blocks, i32(0, 4), 4, k_out=bf(2, 64).expand(4, 2, 64))),
        (TypeError, lambda: F.decode_attention_4bit(bf(1, 2, 2, 64), k16, k16, blocks, i32(4))),
        (ValueError, lambda: F.decode_attention_4bit(bf(1, 2, 2, 128), k_pool, v_pool, blocks, i32(4))),
        (ValueError, lambda: F.decode_attention_4bit(bf(1, 1, 2, 64), k_pool, v_pool, blocks, i32(4))),
        (ValueError, lambda: F.decode_attention_4bit(bf(1, 2, 2, 64), k_pool, v_pool, blocks, i32(4, 4))),
        (ValueError, lambda: F.decode_attention_4bit(bf(1, 2, 2, 64), k_pool, v_pool, blocks, i32(4), max_seq_len=9)),
        (ValueError, lambda: F.decode_attention_4bit(bf(1, 2, 2, 64), k_pool, v_pool, blocks, i32(4), window=-1)),
        (_native.LfError, lambda: F.decode_attention_4bit(bf(1, 2, 2, 64), k_pool, v_pool, blocks, i32(4), scale=-1.0)),
    ]
    for n, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"case {n} was taken")


def test_no_rows():
    table, none = cache4.rotary_table(4, 64), torch.empty(0, dtype=torch.int32, device="cuda")
    q, k, v = rows(0, 2, 2, 64, 1)
    assert F.qk_norm_rotary(q, k, none, table)[0].shape == (0, 2, 64)
    k_pool, v_pool = F.kv_cache_4bit(1, 4, 2, 64)
    assert F.kv_append_rotary(k, v, k_pool, v_pool, none, none, table, q=q).shape == (0, 2, 64)
    cu = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert F.kv_gather_4bit(k_pool, v_pool, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), cu, 0)[0].shape == (0, 2, 64)


def test_a_step_in_a_graph_on_another_stream():
    """Append with the norm, in place for q, then gather, recorded once and replayed on new rows."""
    T, Hq, Hkv, D = 37, 8, 2, 128
    q, k, v = rows(T, Hq, Hkv, D, 50)
    table, w = cache4.rotary_table(64, D), torch.ones(D, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    blocks, cu = torch.arange(3, device="cuda").int()[None], torch.tensor([0, T], dtype=torch.int32, device="cuda")
    pools = F.kv_cache_4bit(3, 16, Hkv, D)
    qs = q.clone()

    def step(pools, q):
        F.kv_append_rotary(k, v, *pools, pos, pos, table, q=q, q_weight=w, k_weight=w, q_out=q)
        return F.kv_gather_4bit(*pools, blocks, cu, T)

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = step(pools, qs)
    for seed in (51, 52):
        fresh = rows(T, Hq, Hkv, D, seed)
        qs.copy_(fresh[0])
        k.copy_(fresh[1])
        v.copy_(fresh[2])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        other = F.kv_cache_4bit(3, 16, Hkv, D)
        want_q = fresh[0].clone()
        want = step(other, want_q)
        assert torch.equal(qs, want_q) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert all(torch.equal(a, b) for a, b in zip(pools, other))


def test_groups_of_the_smallest_numbers():
    """Below 2^-126 numbers count as zeros: a group whose range is under 15 of these keeps its smallest column alone."""
    T, Hkv, D = 64, 4, 128
    _, k, v = rows(T, 1, Hkv, D, 60)
    i = torch.arange(T, dtype=torch.int32, device="cuda")
    table = cache4.rotary_table(T, D)
    cos, sin = table.chunk(2, -1)
    for power in (-112, -118, -121, -122, -123, -124, -126, -130):
        kk, vv = ((x.double() * 2.0 ** power).to(BF16) for x in (k, v))
        k_pool, v_pool = F.kv_cache_4bit(4, 16, Hkv, D)
        F.kv_append_rotary(kk, vv, k_pool, v_pool, i, i, table)
        for want, pool, value in ((cache4.turn(kk.double(), cos.double(), sin.double(), False), k_pool, False),
                                  (vv.double(), v_pool, True)):
            rec = pool.reshape(T, Hkv, -1)
            _, s, z = cache4.parts(rec, D, value)
            off = (cache4.decode(rec, D, value) - want).abs()
            assert (off <= 0.51 * s + 2 ** -8 * z.abs() + 2.0 ** -122 + 2 ** -20 * want.abs().amax()).all(), power
            if power == -112:
                x = cache4.turn(kk.float(), cos, sin, False) if not value else vv.float()
                assert torch.equal(rec, cache4.encode(x, value))
