"""The append with a norm of each head on the way, to bf16 and to 4-bit pools, in every layout of the rotation, with few
rows (a head an item) and with many (several). Against float64.

A norm's sum has an order of its own: 2^-19 of the turned columns' size for the arithmetic in fp32 (a sum of 128 squares in
12 steps, a reciprocal root within 2^-22, four products and a sum: under 32 half steps of 2^-24). A bf16 value is within
2^-8 of itself behind that. What a code stands for is within half a step s of its column, or where the largest or smallest
code is not enough, within the roundings of scale (15 of 2^-8, 0.0586 s) and midpoint (2^-8 |z|)."""
import pytest
import torch

from loopfuse_b200 import functional as F
from tests import cache4

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D,rot,pairs", [
    (64, 64, False), (128, 128, False), (64, 32, False), (128, 64, False), (128, 32, False), (64, 16, False),
    (64, 48, False), (128, 96, False), (128, 48, False), (64, 64, True), (128, 128, True), (64, 16, True), (128, 48, True),
    (128, 80, True)])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 4, 1), (37, 3, 2), (2500, 12, 10), (300, 0, 3)])
def test_append_with_norm(bits, D, rot, pairs, T, Hq, Hkv):
    g = torch.Generator().manual_seed(T + rot)
    x = (3 * torch.randn(T, Hq + 2 * Hkv, D, generator=g)).to(BF16).cuda()
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    k[T // 2, 0] = 0                                     # a row whose norm is eps alone
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(t).cuda() for t in ((BF16, torch.float32) if T % 2 else
                                                                     (torch.float32, BF16))]
    if T == 300:
        w[0] = None
    table, pos = cache4.rotary_table(700, rot), torch.randint(0, 700, (T,), generator=g).int().cuda()
    page, pages = 16, -(-T // 16) + 2
    slots = torch.randperm(page * pages, generator=g)[:T].int().cuda()
    if T > 1:
        slots[T // 3] = -1
    if bits == 4:
        k_pool, v_pool = F.kv_cache_4bit(pages, page, Hkv, D)
    else:
        k_pool, v_pool = torch.zeros(2, pages, page, Hkv, D, dtype=BF16, device="cuda")
    st = F.new_status("cuda")
    got_q = F.kv_append_rotary(k, v, k_pool, v_pool, slots, pos, table, q=q if Hq else None,
                               q_weight=w[0] if Hq else None, k_weight=w[1], eps=1e-5, interleaved=pairs, status=st)
    F.check_status(st)
    cos, sin = table[pos.long()].double().chunk(2, -1)

    def normed(rows, weight):
        y = rows.double()
        if weight is not None:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * weight.double()
        size = cache4.turn(y.abs(), cos.abs(), -sin.abs(), pairs).abs() + y.abs()
        return cache4.turn(y, cos, sin, pairs), size

    real = slots >= 0
    at = slots[real].long()
    want, size = (y[real] for y in normed(k, w[1]))
    if bits == 16:
        off = (k_pool[at // page, at % page].double() - want).abs()
        assert (off <= 2 ** -8 * want.abs() + 2 ** -19 * size).all()
        assert torch.equal(v_pool[at // page, at % page], v[real])
    else:
        rec = k_pool[at // page, at % page]
        _, s, z = cache4.parts(rec, D, False)
        off = (cache4.decode(rec, D, False) - want).abs()
        group = size.unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)   # what moves a group's ends
        assert (off <= torch.maximum(0.5 * s, 0.0586 * s + 2 ** -8 * z.abs()) + 2 ** -18 * group).all()
        # and scale and midpoint are those of the group: half a step of bf16 from the definition
        ends = [f(want.unflatten(-1, (-1, 32)), -1).repeat_interleave(32, -1) for f in (torch.amin, torch.amax)]
        step = (ends[1] - ends[0]) / 15
        assert ((s - step).abs() <= 2 ** -8 * step + 2 ** -20 * group).all()
        assert ((z - ends[0] - 8 * s).abs() <= 2 ** -8 * z.abs() + 2 ** -18 * group).all()
        assert torch.equal(v_pool[at // page, at % page], cache4.encode(v.float(), True)[real])
    untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    untouched[at // page, at % page] = False
    assert (k_pool[untouched] == 0).all() and (v_pool[untouched] == 0).all()
    if Hq:
        want, size = normed(q, w[0])
        assert ((got_q.double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -19 * size).all()
