"""Requests of different lengths on the GPU, at the ends of their contracts: windows as wide as 32 bits, what
strangers and leftovers may not change, pages behind a window, lengths that are cut, offsets out of order. Most results
are compared bit by bit with those of a call that asks for the same in another way."""
import gc

import pytest
import torch

from loopfuse_b200 import functional as F
from loopfuse_b200 import spec as S

from .conftest import require_cuda

pytestmark = pytest.mark.gpu

BAD_LENGTHS = 4  # LF_DEV_BAD_LENGTHS


@pytest.fixture(autouse=True, scope="module")
def _no_garbage():
    """Tensors that cycles keep go with the module that made them, not in the middle of a later test that
    counts allocated bytes."""
    yield
    gc.collect()


@pytest.fixture(autouse=True)
def _gpu():
    require_cuda()


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).bfloat16()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def offsets(lens):
    return torch.nn.functional.pad(torch.tensor(lens).cumsum(0), (1, 0)).int().cuda()


def softcap(cap):
    return (S.ScoreMod(S.MOD_DIV, cap), S.ScoreMod(S.MOD_TANH), S.ScoreMod(S.MOD_MUL, cap))


def paged(g, keys, values, lens, P, spare=0.0):
    """Pools [pages, P, Hkv, D] that hold the requests' rows in shuffled pages, and the table. Page 0 and the slots
    that hold no key are `spare`; entries past a request's pages are -1."""
    blocks = [-(-m // P) for m in lens]
    ids = (torch.randperm(sum(blocks), generator=g, device="cuda") + 1).int()
    table = torch.full((len(lens), max(blocks) + 1), -1, dtype=torch.int32, device="cuda")
    pools = [torch.full((sum(blocks) + 1, P, *keys.shape[1:]), spare, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    at = row = 0
    for b, m in enumerate(lens):
        mine = ids[at:at + blocks[b]]
        table[b, :blocks[b]] = mine
        j = torch.arange(m, device="cuda")
        for pool, x in zip(pools, (keys, values)):
            pool[mine[j // P].long(), j % P] = x[row:row + m]
        at, row = at + blocks[b], row + m
    return pools[0], pools[1], table


# -- windows ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30 + 1, 2 ** 30])
@pytest.mark.parametrize("pages", [False, True])
def test_a_window_that_holds_every_key_is_the_causal_mask(window, pages):
    """Also for requests of more queries than keys, whose first rows see nothing."""
    g = torch.Generator(device="cuda").manual_seed(1)
    lens, keys, D = [13, 300, 5, 64], [10, 40, 5, 300], 64
    q = normal(g, sum(lens), 4, D)
    k, v = normal(g, sum(keys), 2, D), normal(g, sum(keys), 2, D)
    options = dict(cu_seqlens_k=offsets(keys))
    if pages:
        k, v, table = paged(g, k, v, keys, 16)
        options = dict(block_table=table, seq_lens=ints(keys))
    want = F.packed_prefill_attention(q, k, v, offsets(lens), scale=0.125, **options)
    got = F.packed_prefill_attention(q, k, v, offsets(lens), scale=0.125, mask_kind=S.MASK_CAUSAL_WINDOW, window=window,
                                     **options)
    assert want[3:13].abs().amax() > 0 and torch.equal(got, want)
