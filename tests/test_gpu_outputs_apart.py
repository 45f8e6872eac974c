"""Outputs that the caller gives: rows that share elements are refused, whatever the strides that bring them together."""
import pytest
import torch

from loopfuse_b200 import functional as F
from tests import cache4

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
T, H, D = 5, 4, 64


def bf(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(BF16).cuda()


def positions():
    return torch.arange(T, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("strides", [(D, D), (0, D), (D, 0), (2 * D, D), (D, 4 * D), (3 * D, 5 * D), (D // 2, T * D),
                                     (H * D - 8, D)])
def test_rows_that_share_elements_are_refused(strides):
    q, k, table = bf(T, H, D), bf(T, 2, D, seed=1), cache4.rotary_table(8, D)
    room = torch.zeros(64 * D, dtype=BF16, device="cuda")
    out = room.as_strided((T, H, D), (*strides, 1))
    with pytest.raises(ValueError, match="q_out has rows"):
        F.qk_norm_rotary(q, k, positions(), table, q_out=out)
    pools = F.kv_cache_4bit(4, 4, H, D)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="has rows"):
        F.kv_gather_4bit(*pools, torch.zeros(1, 2, dtype=torch.int32, device="cuda"), cu, T, k_out=out)
    with pytest.raises(ValueError, match="out has rows"):
        F.decode_attention_4bit(bf(T, H, 1, D), *pools, torch.zeros(T, 2, dtype=torch.int32, device="cuda"),
                                torch.ones(T, dtype=torch.int32, device="cuda"), out=out.unsqueeze(2))


@pytest.mark.parametrize("strides", [(H * D, D), (D, T * D), (D, 7 * D), (5 * D + 8, D + 8), (8, 6 * D)])
def test_rows_of_other_orders_are_taken(strides):
    q, k, table = bf(T, H, D), bf(T, 2, D, seed=1), cache4.rotary_table(8, D)
    if strides[0] == 8:
        q, strides = q[:1], (8, 6 * D)                   # (one row: its stride says nothing)
    out = torch.zeros(64 * D, dtype=BF16, device="cuda").as_strided(q.shape, (*strides, 1))
    k = k[:len(q)]
    want = F.qk_norm_rotary(q, k, positions(), table)[0]
    assert torch.equal(F.qk_norm_rotary(q, k, positions(), table, q_out=out)[0], want)


def test_outputs_across_other_tensors_are_refused():
    """An output that lies on another input, or on the other output: refused before anything is launched."""
    table, pos = cache4.rotary_table(8, D), positions()
    x = bf(T, 3 * H, D)
    q, k, v = x.split(H, 1)
    before = x.clone()
    pools = F.kv_cache_4bit(4, 4, H, D)
    room = torch.zeros(3 * T, H, D, dtype=BF16, device="cuda")
    for call in (lambda: F.qk_norm_rotary(q, k, pos, table, q_out=k),
                 lambda: F.qk_norm_rotary(q, k, pos, table, k_out=q),
                 lambda: F.qk_norm_rotary(q, k, pos, table, q_out=room[:T], k_out=room[:T]),
                 lambda: F.qk_norm_rotary(q, k, pos, table, q_out=room[:T], k_out=room[T - 1:2 * T - 1]),
                 lambda: F.qk_norm_rotary(q, k, pos, table, q_out=x[:, 1:H + 1]),
                 lambda: F.qk_norm_rotary(q, q, pos, table, q_out=q),
                 lambda: F.kv_append_rotary(k, v, *pools, pos, pos, table, q=q, q_out=k),
                 lambda: F.kv_append_rotary(k, v, *pools, pos, pos, table, q=q, q_out=v),
                 lambda: F.kv_append_rotary(k, v, *pools, pos, pos, table, q=q, q_out=x[:, H // 2:H // 2 + H])):
        with pytest.raises(ValueError, match="apart"):
            call()
    blocks, cu = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.tensor([0, T], dtype=torch.int32, device="cuda")
    for k_out, v_out in ((room[:T], room[:T]), (room[:T], room[1:T + 1]), (room[3:T + 3], room[:T])):
        with pytest.raises(ValueError, match="share rows"):
            F.kv_gather_4bit(*pools, blocks, cu, T, k_out=k_out, v_out=v_out)
    torch.cuda.synchronize()
    assert torch.equal(x, before) and (room == 0).all() and (pools[0] == 0).all()


def test_outputs_that_lie_in_turn_with_others_are_taken():
    """Parts of one buffer: in place in a fused projection, and next to each other by tokens, heads or columns."""
    table, pos = cache4.rotary_table(8, D), positions()
    x = bf(T, 3 * H, D)
    q, k, v = x.split(H, 1)
    want = F.qk_norm_rotary(q, k, pos, table)
    both = torch.zeros(T, H, 2 * D, dtype=BF16, device="cuda")
    for q_out, k_out in ((both[..., :D], both[..., D:]), (both.view(T, 2 * H, D)[:, H:], both.view(T, 2 * H, D)[:, :H]),
                         (both.view(T, H, 2, D)[:, :, 1], both.view(T, H, 2, D)[:, :, 0])):
        got = F.qk_norm_rotary(q, k, pos, table, q_out=q_out, k_out=k_out)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert got[0].data_ptr() == q_out.data_ptr()
    pools, other = F.kv_cache_4bit(4, 4, H, D), F.kv_cache_4bit(4, 4, H, D)
    one = x.clone().split(H, 1)
    assert torch.equal(F.kv_append_rotary(one[1], one[2], *pools, pos, pos, table, q=one[0], q_out=one[0]), want[0])
    F.kv_append_rotary(k, v, *other, pos, pos, table)
    assert all(torch.equal(a, b) for a, b in zip(pools, other))
    blocks, cu = torch.arange(2, device="cuda").int()[None], torch.tensor([0, T], dtype=torch.int32, device="cuda")
    want_kv = F.kv_gather_4bit(*pools, blocks, cu, T)
    got = F.kv_gather_4bit(*pools, blocks, cu, T, k_out=both[..., :D], v_out=both[..., D:])
    assert all(torch.equal(a, b) for a, b in zip(got, want_kv))
    F.qk_norm_rotary(q, k, pos, table, q_out=q, k_out=k)            # in place, both in one projection
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, one[2])
