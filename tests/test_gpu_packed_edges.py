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


# -- what may not change a capped result ----------------------------------------------------------------
STRANGERS = [float("nan"), float("inf"), -float("inf"), 3e38, 1e4]


@pytest.mark.parametrize("bad", STRANGERS)
def test_capped_results_do_not_depend_on_neighbours(bad):
    """Logits of |x| < 0.125 of the cap, where the form of tanh that large ones take would show."""
    g = torch.Generator(device="cuda").manual_seed(2)
    lens, D = [70, 33, 130, 20], 128
    T = sum(lens)
    q, k, v = normal(g, T + 40, 4, D), normal(g, T + 40, 2, D), normal(g, T + 40, 2, D)
    cu, options = offsets(lens), dict(scale=D ** -0.5, mods=softcap(50.0))
    want = F.packed_prefill_attention(q, k, v, cu, **options)
    for b in (1, 3):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        for x in (q2, k2, v2):
            x[cu[b]:cu[b + 1]] = bad
            x[T:] = bad
        got = F.packed_prefill_attention(q2, k2, v2, cu, **options)
        for o in range(4):
            if o != b:
                assert torch.equal(got[cu[o]:cu[o + 1]], want[cu[o]:cu[o + 1]]), (b, o)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pages", [False, True])
def test_capped_results_are_those_of_the_request_alone(D, pages):
    """Requests with large keys between small ones, several per CTA: what they leave in shared memory changes
    nothing."""
    g = torch.Generator(device="cuda").manual_seed(D)
    B = 700
    lens = [70 + b % 50 if b % 2 else 200 for b in range(B)]
    T = sum(lens)
    q, k, v = normal(g, T, 4, D), normal(g, T, 2, D), normal(g, T, 2, D)
    cu = offsets(lens)
    for b in range(0, B, 2):
        k[cu[b]:cu[b + 1]] *= 200.0
    kk, vv, options = k, v, dict(scale=D ** -0.5, mods=softcap(50.0))
    if pages:
        kk, vv, table = paged(g, k, v, lens, 16)
        options.update(block_table=table, seq_lens=ints(lens))
    got = F.packed_prefill_attention(q, kk, vv, cu, **options)
    for _ in range(3):
        assert torch.equal(got, F.packed_prefill_attention(q, kk, vv, cu, **options))
    for b in range(1, B, 24):
        one = slice(int(cu[b]), int(cu[b + 1]))
        alone = F.packed_prefill_attention(q[one], k[one], v[one], ints([0, lens[b]]), scale=D ** -0.5, mods=softcap(50.0))
        assert torch.equal(got[one], alone), b


@pytest.mark.parametrize("bad", STRANGERS)
def test_capped_decode_does_not_depend_on_rows_without_a_request(bad):
    """Padding rows of the batch (length 0), and what the prefix's last page holds behind the prefix."""
    g = torch.Generator(device="cuda").manual_seed(3)
    D, P, prefix, lens = 128, 16, 200, [230, 0, 201, 200, 0, 260]
    q, kp, vp = normal(g, 6, 2, 4, D), normal(g, 80, P, 2, D), normal(g, 80, P, 2, D)
    table = torch.randperm(79, generator=g, device="cuda").int()[:60].view(6, 10).repeat(1, 2)[:, :17] + 1
    table[:, :prefix // P] = table[0, :prefix // P].clone()
    table[0, prefix // P] = 0                 # a page of row 0 alone: its first half is shared
    options = dict(scale=D ** -0.5, mods=softcap(50.0), max_seq_len=270)
    want = F.shared_prefix_decode_attention(q, kp, vp, table, ints(lens), prefix, **options)
    q2, k2 = q.clone(), kp.clone()
    q2[1] = q2[4] = bad
    got = F.shared_prefix_decode_attention(q2, kp, vp, table, ints(lens), prefix, **options)
    assert torch.equal(got, want)
    k2[0, prefix % P:] = bad
    got = F.shared_prefix_decode_attention(q, k2, vp, table, ints([200] + lens[1:]), prefix, **options)
    want = F.shared_prefix_decode_attention(q, kp, vp, table, ints([200] + lens[1:]), prefix, **options)
    assert torch.equal(got, want)


# -- pages behind the window ----------------------------------------------------------------------------
@pytest.mark.parametrize("P", [1, 4, 16, 24, 64, 128])
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 4), (128, 8, 2)])
@pytest.mark.parametrize("cap", [0.0, 50.0])
def test_pages_behind_the_window_need_not_be_there(P, D, Hq, Hkv, cap):
    """A cache that has given the pages back that no query sees any more: their entries are -1, and page 0 holds
    NaN. Short tiles, several tiles, tiles that are cut into slices."""
    g = torch.Generator(device="cuda").manual_seed(P)
    lens, keys = [1, 40, 3, 150, 1, 2], [700, 2100, 64, 900, 129, 6000]
    q = normal(g, sum(lens), Hq, D)
    k, v = normal(g, sum(keys), Hkv, D), normal(g, sum(keys), Hkv, D)
    kp, vp, table = paged(g, k, v, keys, P, spare=float("nan"))
    for window in (1, 63, 64, 100, 2500):
        options = dict(scale=D ** -0.5, mask_kind=S.MASK_CAUSAL_WINDOW, window=window, mods=softcap(cap) if cap else (),
                       seq_lens=ints(keys))
        want = F.packed_prefill_attention(q, k, v, offsets(lens), cu_seqlens_k=offsets(keys),
                                          **{n: x for n, x in options.items() if n != "seq_lens"})
        evicted = table.clone()
        for b, (n, m) in enumerate(zip(lens, keys)):
            first = max(0, m - n - (window - 1))      # that the request's first query sees
            evicted[b, :first // P] = -1
        st = F.new_status("cuda")
        got = F.packed_prefill_attention(q, kp, vp, offsets(lens), block_table=evicted, status=st, **options)
        assert int(st.item()) == 0, window
        assert torch.equal(got, want), window


# -- lengths that are cut -------------------------------------------------------------------------------
def test_shared_prefix_reports_lengths_that_it_cuts():
    """A step recorded with a bound on the lengths that they have outgrown would lose the newest keys."""
    g = torch.Generator(device="cuda").manual_seed(4)
    kp, q = normal(g, 6, 16, 2, 64), normal(g, 2, 2, 2, 64)
    table = ints([[0, 1, 2], [0, 3, 4]])
    for lens, bound, prefix, bad in (([40, 48], 48, 16, False), ([40, 48], None, 16, False), ([40, 49], None, 16, True),
                                     ([40, 33], 32, 16, True), ([17, 0], 16, 16, True), ([16, 0], 16, 16, False),
                                     ([9, 3], 8, 16, True), ([-1, 40], 48, 16, True), ([5, 0], 0, 0, True)):
        st = F.new_status("cuda")
        F.shared_prefix_decode_attention(q, kp, kp, table, ints(lens), prefix, max_seq_len=bound, status=st)
        assert int(st.item()) == (BAD_LENGTHS if bad else 0), (lens, bound)
    with pytest.raises(RuntimeError, match="max_seq_len"):
        F.check_status(ints([BAD_LENGTHS]))


def test_shared_prefix_takes_the_smallest_length_for_none():
    g = torch.Generator(device="cuda").manual_seed(5)
    kp, q = normal(g, 8, 16, 2, 64), normal(g, 2, 2, 2, 64)
    table = ints([[0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 6, 7]])
    for least in (-1, -2 ** 31, -2 ** 31 + 70):
        got = F.shared_prefix_decode_attention(q, kp, kp, table, ints([70, least]), 64)
        assert (got[1] == 0).all() and got[0].abs().amax() > 0, least


# -- page plans of more tokens than the batch has rows ------------------------------------------------------
@pytest.mark.parametrize("kv,new,num_tokens,P", [
    ([0, 0], [5, 20], 8, 4), ([3, 6, 0], [9, 30, 7], 20, 4), ([0, 5, 1], [16, 40, 3], 16, 16), ([7], [100], 0, 8),
    ([i % 9 for i in range(1300)], [i % 7 for i in range(1300)], 1000, 4),
])
def test_plan_pages_takes_pages_for_the_tokens_that_fit(kv, new, num_tokens, P):
    """Tokens past num_tokens are dropped, and with them their pages: the free list, the table and the lengths tell
    the same story."""
    kept, left = [], num_tokens
    for n in new:
        kept.append(min(n, left))
        left -= kept[-1]
    table = torch.full((len(kv), 40), -1, dtype=torch.int32, device="cuda")
    pages, at = list(range(1000, 1000 + sum(new) + len(kv))), 0
    want = [[-1] * 40 for _ in kv]
    for b, h in enumerate(kv):
        have = -(-h // P)
        table[b, :have] = torch.arange(have, device="cuda").int()
        want[b][:have] = range(have)
    free = pages[:]
    for b, (h, n) in enumerate(zip(kv, kept)):
        for c in range(-(-h // P), -(-(h + n) // P)):
            want[b][c] = free[at]
            at += 1
    st = F.new_status("cuda")
    plan = F.plan_pages(ints(kv), ints(new), ints(free), table, page_size=P, num_tokens=num_tokens, status=st)
    assert int(st.item()) == BAD_LENGTHS
    assert plan.seq_lens.tolist() == [h + n for h, n in zip(kv, kept)]
    assert plan.cu_seqlens.tolist() == [sum(kept[:b]) for b in range(len(kv) + 1)]
    assert plan.pages_used.tolist() == [at]
    assert table.tolist() == want
    assert (plan.slots >= 0).all()


# -- offsets out of order --------------------------------------------------------------------------------
def test_offsets_out_of_order_in_a_large_batch():
    """4096 requests that each claim all 524289 tokens: their tiles together pass 31 bits. No key anywhere, so every row
    that a tile holds is written as zeros. (Rows of q and out overlap: nothing reads the one, and zeros on zeros are
    zeros.)"""
    T, G, D = 524289, 128, 64
    flat = torch.full((8 * (T - 1) + G * D,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = flat.as_strided((T, G, D), (8, D, 1))
    q = torch.zeros_like(flat).as_strided((T, G, D), (8, D, 1))
    k = torch.empty(0, 1, D, dtype=torch.bfloat16, device="cuda")
    cu = ints([0, T] * 4096 + [0])
    got = F.packed_prefill_attention(q, k, k, cu, cu_seqlens_k=torch.zeros_like(cu), out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (flat == 0).all()


# -- pools whose pages are not evenly spaced ---------------------------------------------------------------
def pool_pair(layout, n, P, Hkv, D):
    """K and V pools as views [n, P, Hkv, D]: halves of each page of one tensor, heads in front of the slots, rows of a
    wider tensor, or pages with a gap between them."""
    if layout == "halves":
        both = torch.zeros(n, 2, P, Hkv, D, dtype=torch.bfloat16, device="cuda")
        return both[:, 0], both[:, 1]
    if layout == "heads first":
        return [torch.zeros(n, Hkv, P, D, dtype=torch.bfloat16, device="cuda").transpose(1, 2) for _ in "kv"]
    if layout == "one row":
        both = torch.zeros(n, P, 2 * Hkv, D, dtype=torch.bfloat16, device="cuda")
        return both[:, :, :Hkv], both[:, :, Hkv:]
    return [torch.zeros(n, P + 3, Hkv, D, dtype=torch.bfloat16, device="cuda")[:, :P] for _ in "kv"]


@pytest.mark.parametrize("layout", ["halves", "heads first", "one row", "gap"])
@pytest.mark.parametrize("P", [1, 4, 12, 16, 24, 64, 128])
@pytest.mark.parametrize("D", [64, 128])
def test_pools_of_any_strides_hold_the_same(layout, P, D):
    """Append, packed prefill and shared-prefix decode on them are those on contiguous pools, to the bit."""
    g = torch.Generator(device="cuda").manual_seed(P)
    Hkv, G, lens, keys = 2, 3, [40, 1, 150], [300, 129, 150]
    prefix = 128 // P * P
    blocks = [-(-m // P) for m in keys]
    n = sum(blocks) + 2
    table = torch.zeros(3, max(blocks), dtype=torch.int32, device="cuda")
    ids = torch.randperm(n, generator=g, device="cuda").int()
    for b, m in enumerate(blocks):
        table[b, :m] = ids[sum(blocks[:b]):sum(blocks[:b + 1])]
    T = n * P
    k, v = normal(g, T, Hkv, D), normal(g, T, Hkv, D)
    slots = torch.randperm(T, generator=g, device="cuda").int()
    q, q1 = normal(g, sum(lens), Hkv * G, D), normal(g, 3, Hkv, G, D)
    results = []
    for pools in ([torch.zeros(n, P, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in "kv"],
                  pool_pair(layout, n, P, Hkv, D)):
        st = F.new_status("cuda")
        F.kv_append_packed(k, v, *pools, slots, status=st)
        a = F.packed_prefill_attention(q, *pools, offsets(lens), block_table=table, seq_lens=ints(keys), scale=0.125,
                                       status=st)
        b = F.packed_prefill_attention(q, *pools, offsets(lens), block_table=table, seq_lens=ints(keys), scale=0.125,
                                       mask_kind=S.MASK_CAUSAL_WINDOW, window=70, mods=softcap(30.0), status=st)
        shared = table.clone()
        shared[:, :prefix // P] = shared[0, :prefix // P]
        c = F.shared_prefix_decode_attention(q1, *pools, shared, ints(keys), prefix, scale=0.125, status=st)
        assert int(st.item()) == 0
        results.append([x.contiguous() for x in pools] + [a, b, c])
    assert all(torch.equal(x, y) for x, y in zip(*results))


# -- errors ---------------------------------------------------------------------------------------------
def test_a_pool_that_runs_out_is_named_as_one():
    st = F.new_status("cuda")
    table = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    plan = F.plan_pages(ints([0]), ints([9]), ints([5, 6]), table, page_size=4, num_tokens=9, status=st)
    assert plan.pages_used.tolist() == [3] and table.tolist() == [[5, 6, -1, -1]]
    with pytest.raises(RuntimeError, match="plan_pages: .*page id.*ran out"):
        F.check_status(st, "plan_pages")
