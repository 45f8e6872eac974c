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
