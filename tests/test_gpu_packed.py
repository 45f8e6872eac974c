"""Requests of different lengths on the GPU: page plans, the packed append, packed prefill and
shared-prefix decode against plain computations in 64 bits, at the sizes, masks and strides where they
can go wrong.

Tolerance of an attention output, per element: the result is rounded to bf16 once and every weight of the
second product once, each by 2^-9 of its value (a rounding is at most between 2^-9 and 2^-8 of a value;
the smaller is taken): 2^-9 of the result, and 2 * 2^-9 of sum_j w_j |v_j| for the weights in the numerator
and in the row sum. What fp32 scores, exp2 and sums add is below 2^-18 of the same sums. A softcap's tanh
beyond 0.4 is the unit's (relative error 2^-11): it moves a logit s by |s| 2^-11 at most, and so every
weight by that share, twice like the rounding.
"""
import gc

import pytest
import torch

from loopfuse_b200 import functional as F
from loopfuse_b200 import spec as S

from .conftest import require_cuda

pytestmark = pytest.mark.gpu


def softcap(cap):
    return (S.ScoreMod(S.MOD_DIV, cap), S.ScoreMod(S.MOD_TANH), S.ScoreMod(S.MOD_MUL, cap))


def reference(q, k, v, scale, cap=0.0, seen=None):
    """(out, largest error) in 64 bits for q [..., n, D], k / v [..., m, D], seen [n, m]."""
    q, k, v = q.double(), k.double(), v.double()
    s = q @ k.transpose(-1, -2) * scale
    if cap:
        s = torch.tanh(s / cap) * cap
    if seen is None:
        seen = torch.ones(s.shape[-2:], dtype=torch.bool, device=s.device)
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:-1], 1), float("-inf"))
    w = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, 1.0, total)
    # (a value that no row of a query sees must not count here either)
    out, size = w @ v, w @ v.abs()
    each = 2 * 2.0 ** -9 + 2.0 ** -18
    if cap:
        x = torch.where(seen, s, 0.0).abs().amax().item() if s.numel() else 0.0
        each += 2 * x * 2.0 ** -11
    return out, 2.0 ** -9 * out.abs() + each * size + 1e-30


def check(got, want, bound, what=""):
    off = (got.double() - want).abs()
    assert not torch.isnan(off).any(), what
    assert bool((off <= bound).all()), (what, (off / bound).max().item())


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).bfloat16()


def offsets(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True, scope="module")
def _no_garbage():
    """Tensors that cycles keep (exceptions and their frames, modules) go with the module that made them, not
    in the middle of a later test that counts allocated bytes."""
    yield
    gc.collect()


@pytest.fixture(autouse=True)
def _gpu():
    require_cuda()


# -- page plans ---------------------------------------------------------------------------------------
def plan_ref(kv, new, free, table, P, num_tokens):
    table = [list(r) for r in table]
    slots, positions, cu, used = [], [], [0], 0
    for b, (h, n) in enumerate(zip(kv, new)):
        have = -(-h // P)
        for c in range(have, -(-(h + n) // P)):
            page = free[used] if used < len(free) else -1
            used += 1
            if c < len(table[b]):
                table[b][c] = page
        for i in range(n):
            pos = h + i
            page = table[b][pos // P] if pos // P < len(table[b]) else -1
            slots.append(page * P + pos % P if page >= 0 else -1)
            positions.append(pos)
        cu.append(cu[-1] + n)
    pad = num_tokens - len(slots)
    return table, cu, [h + n for h, n in zip(kv, new)], slots + [-1] * pad, positions + [0] * pad, used


def run_plan(kv, new, P, num_tokens, n_free=None, width=None, stream=None):
    g = torch.Generator().manual_seed(len(kv) * 1000 + P)
    have = [-(-h // P) for h in kv]
    need = sum(-(-(h + n) // P) - a for h, n, a in zip(kv, new, have))
    ids = torch.randperm(sum(have) + need + 3, generator=g).tolist()
    n_free = need + 3 if n_free is None else n_free
    width = max(-(-(h + n) // P) for h, n in zip(kv, new)) + 1 if width is None else width
    table, at = [[-7] * width for _ in kv], 0
    for b, a in enumerate(have):
        for c in range(min(a, width)):
            table[b][c] = ids[at]
            at += 1
    free = ids[sum(have):][:n_free]
    want = plan_ref(kv, new, free, table, P, num_tokens)
    wide = torch.full((len(kv), width + 5), -9, dtype=torch.int32, device="cuda")
    view = wide[:, 2:2 + width]      # rows of a wider table
    view.copy_(torch.tensor(table, dtype=torch.int32))
    st = F.new_status("cuda")
    plan = F.plan_pages(ints(kv), ints(new), ints(free), view, page_size=P, num_tokens=num_tokens, status=st)
    assert view.tolist() == want[0]
    assert (wide[:, :2] == -9).all() and (wide[:, 2 + width:] == -9).all()
    assert plan.cu_seqlens.tolist() == want[1]
    assert plan.seq_lens.tolist() == want[2]
    assert plan.slots.tolist() == want[3]
    assert plan.positions.tolist() == want[4]
    assert plan.pages_used.tolist() == [want[5]]
    return int(st.item())


@pytest.mark.parametrize("P", [1, 3, 16, 64])
@pytest.mark.parametrize("kv,new", [
    ([0], [1]), ([0], [0]), ([5], [0]), ([16], [1]), ([15], [1]), ([0, 0, 7], [1, 0, 130]),
    ([64, 1, 0, 63, 128], [64, 63, 0, 1, 700]),
])
def test_plan_pages_small(P, kv, new):
    assert run_plan(kv, new, P, sum(new)) == 0
    assert run_plan(kv, new, P, sum(new) + 9) == 0


@pytest.mark.parametrize("B", [31, 511, 512, 513, 1200])
def test_plan_pages_many_requests(B):
    g = torch.Generator().manual_seed(B)
    kv = torch.randint(0, 200, (B,), generator=g).tolist()
    new = (torch.randint(0, 90, (B,), generator=g) * (torch.rand(B, generator=g) < 0.8)).int().tolist()
    assert run_plan(kv, new, 16, sum(new) + 40) == 0


def test_plan_pages_more_requests_than_default_shared_memory_holds():
    B = 9000
    kv = [i % 5 for i in range(B)]
    new = [1 + (i % 2) for i in range(B)]
    assert run_plan(kv, new, 4, sum(new)) == 0


def test_plan_pages_reports_a_pool_that_runs_out_and_a_narrow_table():
    assert run_plan([0, 3, 8], [40, 9, 1], 4, 50, n_free=9) == 2        # LF_DEV_BAD_PAGE
    assert run_plan([0, 3], [40, 9], 4, 49, width=5) == 2


def test_plan_pages_cuts_lengths_that_make_no_sense():
    st = F.new_status("cuda")
    table = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    plan = F.plan_pages(ints([0, -5, 0]), ints([3, 2, -1]), ints([4, 5, 6]), table, page_size=4,
                        num_tokens=8, status=st)
    assert plan.cu_seqlens.tolist() == [0, 3, 5, 5] and plan.seq_lens.tolist() == [3, 2, 0]
    assert (int(st.item()) & 0xFF) == 4
    st.zero_()
    plan = F.plan_pages(ints([0, 0]), ints([5, 2 ** 30]), ints([1, 2, 3]), table[:2], page_size=4,
                        num_tokens=8, status=st)
    assert plan.cu_seqlens.tolist() == [0, 5, 8] and int(st.item()) != 0
    st.zero_()
    table.fill_(-1)
    plan = F.plan_pages(ints([0, 0, 0]), ints([2 ** 30] * 3), ints([7]), table, page_size=1, num_tokens=8, status=st)
    assert plan.cu_seqlens.tolist() == [0, 8, 8, 8] and plan.pages_used.tolist() == [2 ** 31 - 1]
    assert plan.slots.tolist() == [7] + [-1] * 7 and int(st.item()) != 0
    assert table[0].tolist() == [7, -1, -1, -1] and (table[1:] == -1).all()
    with pytest.raises(RuntimeError, match="length"):
        F.check_status(ints([4]))


# -- append -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,Hkv,P", [(1, 1, 1), (7, 3, 16), (130, 8, 24), (1000, 2, 64)])
def test_append_stores_rows_at_their_slots(T, Hkv, P, D):
    g = torch.Generator(device="cuda").manual_seed(T)
    n_pages = -(-T // P) + 2
    qkv = normal(g, T, 3 * Hkv, D)
    k, v = qkv[:, Hkv:2 * Hkv], qkv[:, 2 * Hkv:]
    pools = [normal(g, n_pages, P, Hkv, D) for _ in range(2)]
    slots = torch.randperm(n_pages * P, generator=g, device="cuda")[:T].int()
    slots[::5] = -1
    want = []
    for pool, rows in zip(pools, (k, v)):
        w = pool.clone()
        w.view(-1, Hkv, D)[slots[slots >= 0].long()] = rows[slots >= 0]
        want.append(w)
    st = F.new_status("cuda")
    F.kv_append_packed(k, v, pools[0], pools[1], slots, status=st)
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1]) and int(st.item()) == 0


def test_append_never_writes_outside_the_pool():
    g = torch.Generator(device="cuda").manual_seed(3)
    whole = normal(g, 6, 4, 2, 64)
    pool, before = whole[1:5], whole.clone()
    k = normal(g, 3, 2, 64)
    st = F.new_status("cuda")
    F.kv_append_packed(k, k, pool, pool, ints([16, 2 ** 31 - 1, 5]), status=st)
    assert int(st.item()) == 2
    before.view(-1, 2, 64)[4 + 5] = k[2]
    assert torch.equal(whole, before)
    F.kv_append_packed(k[:0], k[:0], pool, pool, ints([]))
    assert torch.equal(whole, before)


def test_append_to_one_token_pages():
    g = torch.Generator(device="cuda").manual_seed(4)
    pool = normal(g, 9, 2, 64)
    k = normal(g, 2, 2, 64)
    F.kv_append_packed(k, k, pool, pool, ints([8, 0]))
    assert torch.equal(pool[8], k[0]) and torch.equal(pool[0], k[1])


# -- packed prefill -----------------------------------------------------------------------------------
def heads_first(x, heads):
    """[n, H, D] -> [heads, n, D], each kv head repeated for its query heads."""
    return x.transpose(0, 1).repeat_interleave(heads // x.shape[1], dim=0)


def seen_of(n, m, mask, window):
    i = torch.arange(n, device="cuda")[:, None] + (m - n)
    j = torch.arange(m, device="cuda")[None]
    seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
    if mask != S.MASK_NONE:
        seen = j <= i
    if mask == S.MASK_CAUSAL_WINDOW:
        seen = seen & (j > i - window)
    return seen


def check_packed(got, q, keys, lens, scale, cap=0.0, mask=S.MASK_CAUSAL, window=0):
    """`keys(b)` gives the request's k and v [m, Hkv, D]."""
    at = 0
    for b, n in enumerate(lens):
        if n:
            k, v = keys(b)
            Hq = q.shape[1]
            want, bound = reference(q[at:at + n].transpose(0, 1), heads_first(k, Hq), heads_first(v, Hq), scale,
                                    cap, seen_of(n, k.shape[0], mask, window))
            check(got[at:at + n].transpose(0, 1), want, bound, (b, n))
        at += n


EDGES = [1, 0, 63, 64, 65, 31, 33, 127, 128, 129, 200, 2]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (4, 2), (3, 1), (8, 2), (7, 1), (16, 2), (128, 1)])
def test_packed_lengths_around_the_tile_edges(Hq, Hkv, D):
    g = torch.Generator(device="cuda").manual_seed(Hq * D)
    T = sum(EDGES)
    qkv = normal(g, T, Hq + 2 * Hkv, D)      # views of one projection
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    cu = offsets(EDGES)
    got = F.packed_prefill_attention(q, k, v, cu, scale=D ** -0.5)
    check_packed(got, q, lambda b: (k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]]), EDGES, D ** -0.5)


@pytest.mark.parametrize("mask,window", [(S.MASK_NONE, 0), (S.MASK_CAUSAL, 0), (S.MASK_CAUSAL_WINDOW, 1),
                                         (S.MASK_CAUSAL_WINDOW, 64), (S.MASK_CAUSAL_WINDOW, 100)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_packed_masks_and_softcap(mask, window, cap):
    g = torch.Generator(device="cuda").manual_seed(window)
    lens, D = [300, 1, 77, 450], 128
    T = sum(lens)
    q, k, v = normal(g, T, 4, D), normal(g, T, 2, D), normal(g, T, 2, D)
    cu = offsets(lens)
    got = F.packed_prefill_attention(q, k, v, cu, scale=D ** -0.5, mods=softcap(cap) if cap else (),
                                     mask_kind=mask, window=window)
    check_packed(got, q, lambda b: (k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]]), lens, D ** -0.5, cap, mask, window)


@pytest.mark.parametrize("size", [0.02, 3.0, 12.0])
@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
def test_packed_small_and_large_logits(size, cap):
    """Every form of tanh, and references that move often."""
    g = torch.Generator(device="cuda").manual_seed(9)
    lens, D = [260, 90], 64
    q, k, v = normal(g, 350, 2, D) * size, normal(g, 350, 2, D), normal(g, 350, 2, D)
    cu = offsets(lens)
    got = F.packed_prefill_attention(q, k, v, cu, scale=D ** -0.5, mods=softcap(cap) if cap else ())
    check_packed(got, q, lambda b: (k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]]), lens, D ** -0.5, cap)


@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 1)])
def test_packed_keys_of_other_lengths(Hq, Hkv):
    """Chunks behind cached keys, queries that see nothing (zeros), requests without keys."""
    g = torch.Generator(device="cuda").manual_seed(5)
    lens, keys, D = [5, 70, 40, 3, 0, 1], [200, 70, 10, 0, 9, 1], 64
    q, k, v = normal(g, sum(lens), Hq, D), normal(g, sum(keys), Hkv, D), normal(g, sum(keys), Hkv, D)
    ck = offsets(keys)
    out = torch.full_like(q, 7.0)
    got = F.packed_prefill_attention(q, k, v, offsets(lens), cu_seqlens_k=ck, scale=D ** -0.5, out=out)
    assert got.data_ptr() == out.data_ptr()
    check_packed(got, q, lambda b: (k[ck[b]:ck[b + 1]], v[ck[b]:ck[b + 1]]), lens, D ** -0.5)
    cq = offsets(lens)
    assert (got[cq[2]:cq[2] + 30] == 0).all() and (got[cq[3]:cq[4]] == 0).all()


def test_packed_neighbours_never_reach_a_result():
    """Infinities and NaN in the rows of other requests and past the last token."""
    g = torch.Generator(device="cuda").manual_seed(6)
    lens, D = [70, 33, 130, 20], 128
    T = sum(lens)
    q, k, v = normal(g, T + 40, 4, D), normal(g, T + 40, 2, D), normal(g, T + 40, 2, D)
    cu = offsets(lens)
    want = F.packed_prefill_attention(q, k, v, cu, scale=D ** -0.5)
    for bad in (float("nan"), float("inf"), -float("inf"), 3e38):
        for b in (1, 3):
            q2, k2, v2 = q.clone(), k.clone(), v.clone()
            for x in (q2, k2, v2):
                x[cu[b]:cu[b + 1]] = bad
                x[T:] = bad
            got = F.packed_prefill_attention(q2, k2, v2, cu, scale=D ** -0.5)
            for o in range(4):
                if o != b:
                    assert torch.equal(got[cu[o]:cu[o + 1]], want[cu[o]:cu[o + 1]]), (bad, b, o)


def test_packed_rows_of_no_request_are_left_alone():
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = normal(g, 50, 2, 64), normal(g, 50, 2, 64), normal(g, 50, 2, 64)
    out = torch.full_like(q, 3.0)
    F.packed_prefill_attention(q, k, v, ints([4, 10, 45]), out=out, scale=0.125)
    assert (out[:4] == 3.0).all() and (out[45:] == 3.0).all()
    before = out.clone()
    # Offsets out of order or past the end are cut to the tensors.
    F.packed_prefill_attention(q, k, v, ints([-5, 10, 7, 1000]), out=out, scale=0.125)
    assert torch.isfinite(out).all()
    F.packed_prefill_attention(q[:0], k[:0], v[:0], ints([0, 0]), out=before[:0])


@pytest.mark.parametrize("P", [1, 2, 8, 16, 24, 64, 100, 128])
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 3, 3)])
def test_packed_reads_keys_through_a_block_table(P, D, Hq, Hkv):
    """Mixed step: chunks, whole prompts, single tokens, a waiting request; unused slots hold NaN."""
    g = torch.Generator(device="cuda").manual_seed(P)
    lens, total = [40, 1, 150, 0, 17, 1], [300, 129, 150, 50, 80, 1]
    blocks = [-(-t // P) for t in total]
    n_pages = sum(blocks) + 3
    kp, vp = (torch.full((n_pages, P, Hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    ids = torch.randperm(n_pages, generator=g, device="cuda").tolist()
    table = torch.full((6, max(blocks) + 2), -1, dtype=torch.int32)
    keys = []
    for b, t in enumerate(total):
        mine = [ids.pop() for _ in range(blocks[b])]
        table[b, :blocks[b]] = torch.tensor(mine, dtype=torch.int32)
        k, v = normal(g, t, Hkv, D), normal(g, t, Hkv, D)
        keys.append((k, v))
        for j in range(t):
            kp[mine[j // P], j % P] = k[j]
            vp[mine[j // P], j % P] = v[j]
    q = normal(g, sum(lens), Hq, D)
    for mask, window, cap in ((S.MASK_CAUSAL, 0, 0.0), (S.MASK_CAUSAL_WINDOW, 90, 30.0)):
        st = F.new_status("cuda")
        got = F.packed_prefill_attention(q, kp, vp, offsets(lens), block_table=table.cuda(), seq_lens=ints(total),
                                         scale=D ** -0.5, mods=softcap(cap) if cap else (), mask_kind=mask,
                                         window=window, status=st)
        assert int(st.item()) == 0
        check_packed(got, q, lambda b: keys[b], lens, D ** -0.5, cap, mask, window)


def test_packed_paged_reports_bad_pages_and_cuts_lengths():
    g = torch.Generator(device="cuda").manual_seed(8)
    kp, q = normal(g, 4, 16, 2, 64), normal(g, 3, 2, 64)
    st = F.new_status("cuda")
    got = F.packed_prefill_attention(q, kp, kp, ints([0, 3]), block_table=ints([[1, 99]]), seq_lens=ints([20]),
                                     status=st)
    assert int(st.item()) == 2 and torch.isfinite(got).all()
    st.zero_()
    a = F.packed_prefill_attention(q, kp, kp, ints([0, 3]), block_table=ints([[1, 2]]), seq_lens=ints([5000]),
                                   status=st)
    b = F.packed_prefill_attention(q, kp, kp, ints([0, 3]), block_table=ints([[1, 2]]), seq_lens=ints([32]))
    assert torch.equal(a, b) and int(st.item()) == 0


def test_packed_batch_of_many_tiles_is_ordered_and_the_same():
    """More tiles than the machine holds: every request's result is that of the request alone."""
    g = torch.Generator(device="cuda").manual_seed(10)
    lens = [700, 3, 0, 512, 90, 1400] + [40 + 7 * i for i in range(40)]
    D, T = 64, 0
    T = sum(lens)
    q, k, v = normal(g, T, 16, D), normal(g, T, 16, D), normal(g, T, 16, D)
    cu = offsets(lens)
    assert _workspace(len(lens), T, 16, 16, D) > 0
    ws = F.DecodeWorkspace()
    got = F.packed_prefill_attention(q, k, v, cu, scale=D ** -0.5, workspace=ws)
    assert torch.equal(got, F.packed_prefill_attention(q, k, v, cu, scale=D ** -0.5, workspace=ws))
    check_packed(got, q, lambda b: (k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]]), lens, D ** -0.5)
    for b in (0, 1, 5, 20):
        one = slice(int(cu[b]), int(cu[b + 1]))
        alone = F.packed_prefill_attention(q[one], k[one], v[one], ints([0, lens[b]]), scale=D ** -0.5)
        assert torch.equal(alone, got[one]), b


def _workspace(B, T, Hq, Hkv, D):
    import ctypes

    from loopfuse_b200 import _native
    a = _native.LfPackedArgs()
    a.B, a.T, a.Tk, a.Hq, a.Hkv, a.D = B, T, T, Hq, Hkv, D
    return _native.load().lf_packed_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 4), (128, 8, 2)])
@pytest.mark.parametrize("paged", [False, True])
def test_packed_few_tokens_behind_long_contexts(D, Hq, Hkv, paged):
    """Long tiles are cut into slices of their keys, which the last one to finish joins."""
    g = torch.Generator(device="cuda").manual_seed(14)
    lens, keys, P = [3, 40, 1, 0, 200], [6000, 9001, 2049, 10, 3111], 16
    q = normal(g, sum(lens), Hq, D) * 3
    k, v = normal(g, sum(keys), Hkv, D), normal(g, sum(keys), Hkv, D)
    ck = offsets(keys)
    options = dict(cu_seqlens_k=ck)
    kk, vv = k, v
    if paged:
        blocks = [-(-m // P) for m in keys]
        ids = torch.randperm(sum(blocks), generator=g, device="cuda")
        kk, vv = (torch.full((sum(blocks), P, Hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda")
                  for _ in "kv")
        table = torch.zeros(len(keys), max(blocks), dtype=torch.int32, device="cuda")
        for b, m in enumerate(keys):
            mine = ids[sum(blocks[:b]):sum(blocks[:b + 1])]
            table[b, :len(mine)] = mine.int()
            j = torch.arange(m, device="cuda")
            kk[mine[j // P], j % P], vv[mine[j // P], j % P] = k[ck[b]:ck[b + 1]], v[ck[b]:ck[b + 1]]
        options = dict(block_table=table, seq_lens=ints(keys))
    for cap, mask, window in ((0.0, S.MASK_CAUSAL, 0), (30.0, S.MASK_CAUSAL_WINDOW, 5000)):
        st = F.new_status("cuda")
        got = F.packed_prefill_attention(q, kk, vv, offsets(lens), scale=D ** -0.5, status=st,
                                         mods=softcap(cap) if cap else (), mask_kind=mask, window=window, **options)
        again = F.packed_prefill_attention(q, kk, vv, offsets(lens), scale=D ** -0.5,
                                           mods=softcap(cap) if cap else (), mask_kind=mask, window=window, **options)
        assert int(st.item()) == 0 and torch.equal(got, again)
        check_packed(got, q, lambda b: (k[ck[b]:ck[b + 1]], v[ck[b]:ck[b + 1]]), lens, D ** -0.5, cap, mask, window)


def test_packed_many_requests_without_keys():
    """Tiles without a key block, more of them than a CTA keeps in hand at once, between ordinary ones."""
    g = torch.Generator(device="cuda").manual_seed(15)
    lens = [30] * 900
    keys = [0 if b % 9 else 30 for b in range(900)]
    q, k, v = normal(g, sum(lens), 4, 64), normal(g, sum(keys), 4, 64), normal(g, sum(keys), 4, 64)
    got = F.packed_prefill_attention(q, k, v, offsets_fast(lens), cu_seqlens_k=offsets_fast(keys), scale=0.125)
    got = got.view(900, 30, 4, 64)
    assert (got[torch.tensor([b for b in range(900) if b % 9])] == 0).all()
    want, bound = reference(q.view(900, 30, 4, 64)[::9].transpose(1, 2), k.view(100, 30, 4, 64).transpose(1, 2),
                            v.view(100, 30, 4, 64).transpose(1, 2), 0.125, 0.0, seen_of(30, 30, S.MASK_CAUSAL, 0))
    check(got[::9].transpose(1, 2), want, bound)


def test_packed_batch_beyond_the_order_kernels_requests():
    g = torch.Generator(device="cuda").manual_seed(11)
    B, D = 8300, 64
    lens = [1 + i % 3 for i in range(B)]
    T = sum(lens)
    q, k, v = normal(g, T, 1, D), normal(g, T, 1, D), normal(g, T, 1, D)
    cu = offsets_fast(lens)
    got = F.packed_prefill_attention(q, k, v, cu, scale=D ** -0.5)
    for b in list(range(0, B, 997)) + [B - 1]:
        one = slice(sum(lens[:b]), sum(lens[:b + 1]))
        want, bound = reference(q[one].transpose(0, 1), k[one].transpose(0, 1), v[one].transpose(0, 1), D ** -0.5,
                                0.0, seen_of(lens[b], lens[b], S.MASK_CAUSAL, 0))
        check(got[one].transpose(0, 1), want, bound, b)


def offsets_fast(lens):
    return torch.nn.functional.pad(torch.tensor(lens).cumsum(0), (1, 0)).int().cuda()


# -- shared prefix ------------------------------------------------------------------------------------
def shared_case(g, lens, prefix, P, Hkv, D):
    """Pools whose unused slots hold NaN, the table, and each request's keys [len, Hkv, D]."""
    whole = prefix // P                       # shared pages; a page that the prefix only begins is copied
    blocks = [max(0, -(-n // P) - whole) for n in lens]
    n_pages = whole + sum(blocks) + 4
    kp, vp = (torch.full((n_pages, P, Hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    ids = torch.randperm(n_pages, generator=g, device="cuda").tolist()
    shared = [ids.pop() for _ in range(whole)]
    table = torch.full((len(lens), whole + max(blocks + [1])), -1, dtype=torch.int32)
    pk, pv = normal(g, max(prefix, 1), Hkv, D), normal(g, max(prefix, 1), Hkv, D)
    keys = []
    for b, n in enumerate(lens):
        mine = shared + [ids.pop() for _ in range(blocks[b])]
        table[b, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
        own = max(0, n - prefix)
        k = torch.cat((pk[:min(n, prefix)], normal(g, own, Hkv, D)))
        v = torch.cat((pv[:min(n, prefix)], normal(g, own, Hkv, D)))
        keys.append((k, v))
        page = torch.tensor(mine, dtype=torch.long, device="cuda")
        j = torch.arange(n, device="cuda")
        kp[page[j // P], j % P] = k
        vp[page[j // P], j % P] = v
    # (row 0 holds the whole prefix, whatever its own length)
    j = torch.arange(whole * P, device="cuda")
    page = torch.tensor(shared + [0], dtype=torch.long, device="cuda")
    kp[page[j // P], j % P], vp[page[j // P], j % P] = pk[:whole * P], pv[:whole * P]
    return kp, vp, table.cuda(), keys


def check_shared(got, q, keys, scale, cap=0.0):
    for b, (k, v) in enumerate(keys):
        want, bound = reference(q[b], k.transpose(0, 1), v.transpose(0, 1), scale, cap)
        check(got[b], want, bound, (b, k.shape[0]))
        if not k.shape[0]:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv,G", [(1, 1), (2, 3), (2, 4), (1, 8), (1, 9), (2, 16), (1, 128)])
def test_shared_prefix_heads(Hkv, G, D):
    g = torch.Generator(device="cuda").manual_seed(G)
    prefix = 160
    lens = [prefix + n for n in (1, 64, 17, 300, 2, 65, 16, 40)]
    kp, vp, table, keys = shared_case(g, lens, prefix, 16, Hkv, D)
    q = normal(g, len(lens), Hkv, G, D)
    st = F.new_status("cuda")
    got = F.shared_prefix_decode_attention(q, kp, vp, table, ints(lens), prefix, scale=D ** -0.5,
                                           max_seq_len=max(lens), status=st)
    assert int(st.item()) == 0
    check_shared(got, q, keys, D ** -0.5)


@pytest.mark.parametrize("P", [1, 4, 16, 24, 128])
@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 200, 1000])
def test_shared_prefix_lengths(P, prefix):
    """Prefixes that end in a page and in a block; requests of length 0, inside the prefix, at its end."""
    g = torch.Generator(device="cuda").manual_seed(prefix)
    D, Hkv, G = 64, 2, 2
    lens = [prefix + 33, 0, prefix, max(prefix - 1, 0), prefix // 2, prefix + 1, prefix + 500]
    kp, vp, table, keys = shared_case(g, lens, prefix, P, Hkv, D)
    q = normal(g, len(lens), Hkv, G, D)
    for cap, bound in ((0.0, max(lens)), (30.0, None)):
        st = F.new_status("cuda")
        got = F.shared_prefix_decode_attention(q, kp, vp, table, ints(lens), prefix, scale=D ** -0.5,
                                               mods=softcap(cap) if cap else (), max_seq_len=bound, status=st)
        assert int(st.item()) == 0
        check_shared(got, q, keys, D ** -0.5, cap)


@pytest.mark.parametrize("B", [1, 5, 64, 200])
def test_shared_prefix_batches(B):
    g = torch.Generator(device="cuda").manual_seed(B)
    D, Hkv, G, prefix, P = 128, 2, 4, 640, 16
    lens = [prefix + 1 + (37 * b) % 150 for b in range(B)]
    kp, vp, table, keys = shared_case(g, lens, prefix, P, Hkv, D)
    qkv = normal(g, B, Hkv * (G + 2), D)                      # strided queries
    q = qkv[:, :Hkv * G].unflatten(1, (Hkv, G)) * 4
    q = torch.cat((q, q), dim=-1)[..., :D]
    got = F.shared_prefix_decode_attention(q, kp, vp, table, ints(lens), prefix, scale=D ** -0.5,
                                           max_seq_len=max(lens))
    check_shared(got, q, keys, D ** -0.5)
    plain = F.paged_decode_attention(q[:1], kp, vp, table[:1], seq_len=lens[0], scale=D ** -0.5)
    assert (plain[0].float() - got[0].float()).abs().max().item() <= 2e-2


def test_shared_prefix_cuts_lengths_and_reports_bad_pages():
    g = torch.Generator(device="cuda").manual_seed(12)
    kp, q = normal(g, 6, 16, 2, 64), normal(g, 2, 2, 2, 64)
    table = ints([[0, 1, 2], [0, 3, 4]])
    a = F.shared_prefix_decode_attention(q, kp, kp, table, ints([40, 900]), 16, max_seq_len=48)
    b = F.shared_prefix_decode_attention(q, kp, kp, table, ints([40, 48]), 16, max_seq_len=48)
    assert torch.equal(a, b)
    c = F.shared_prefix_decode_attention(q, kp, kp, table, ints([40, -3]), 16)
    assert torch.equal(c[0], b[0]) and (c[1] == 0).all()
    for bad in ([[99, 1, 2], [0, 3, 4]], [[0, 1, 2], [0, -1, 4]]):
        st = F.new_status("cuda")
        got = F.shared_prefix_decode_attention(q, kp, kp, ints(bad), ints([40, 40]), 16, status=st)
        assert int(st.item()) == 2 and torch.isfinite(got).all()


# -- streams and graphs -------------------------------------------------------------------------------
def _step(st):
    plan = F.plan_pages(st["kv"], st["new"], st["free"], st["table"], page_size=16, num_tokens=st["T"])
    F.kv_append_packed(st["k"], st["v"], st["kp"], st["vp"], plan.slots)
    packed = F.packed_prefill_attention(st["q"], st["kp"], st["vp"], plan.cu_seqlens, block_table=st["table"],
                                        seq_lens=plan.seq_lens, scale=0.125)
    one = F.shared_prefix_decode_attention(st["q1"], st["kp"], st["vp"], st["table"], plan.seq_lens, 32,
                                           scale=0.125, max_seq_len=160)
    return packed, one


def _step_state():
    g = torch.Generator(device="cuda").manual_seed(13)
    lens = [20, 1, 90, 64]
    table = torch.full((4, 10), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = ints([30, 31])             # two shared pages
    T = sum(lens)
    return dict(kv=ints([32] * 4), new=ints(lens), free=torch.arange(30, device="cuda").int(), table=table, T=T,
                q=normal(g, T, 4, 64), k=normal(g, T, 2, 64), v=normal(g, T, 2, 64), q1=normal(g, 4, 2, 2, 64),
                kp=normal(g, 32, 16, 2, 64), vp=normal(g, 32, 16, 2, 64))


def test_a_step_on_another_stream_and_in_a_graph():
    st = _step_state()
    want = [x.clone() for x in _step(st)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        st2 = _step_state()
        got = _step(st2)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(st)
    for x in got:
        x.zero_()
    st["table"][:, 2:] = -1
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
