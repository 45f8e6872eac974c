"""Decode attention over a 4-bit cache against float64 on the values that its records stand for.

Tolerance of an output column: its own rounding, 2^-8 |o|; the rounding of each key's weight times its scale to
fp16, 2^-11 sum_j w_j s_j c_j, or where that is subnormal 2^-33 of the largest scale, fifteen times, for each of n keys; and what an error d of the scores does to the weights, 2 d sum_j w_j |v_j|. d: the sums of the query row enter with
16 bits, 2^-16 of 8 |sum q| s and of |sum q| |z|, and sums in float32 are within 2^-20 of products of up to 15 |q| s;
with a softcap 2^-10 of the largest score (the unit's tanh is within 2^-11)."""
import math

import pytest
import torch

from loopfuse_b200 import functional as F
from loopfuse_b200 import spec as S
from tests import cache4

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


class Batch:
    def __init__(self, lens, Hkv, G, D, page, seed, layout="head", amp=1.0, spare=2, pages=None):
        g = torch.Generator().manual_seed(seed)
        self.D, self.page, self.lens = D, page, lens
        need = [-(-n // page) for n in lens]
        self.pages = pages or sum(need) + 3
        self.pools = []
        for value in (False, True):
            x = torch.randn(self.pages, page, Hkv, D, generator=g).cuda() * amp
            x[..., 3] *= 6                              # a column that sticks out, as in keys
            rec = cache4.encode(x, value)
            order = {"head": (0, 2, 1, 3), "page": (0, 1, 2, 3), "slots": (1, 0, 2, 3)}[layout]
            back = {"head": (0, 2, 1, 3), "page": (0, 1, 2, 3), "slots": (1, 0, 2, 3)}[layout]
            self.pools.append(rec.permute(order).contiguous().permute(back))
        ids = torch.randperm(self.pages, generator=g).int()
        table = torch.full((len(lens), max(max(need), 1) + spare), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = ids[at:at + n]
            at += n
        self.table = table.cuda()
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.q = torch.randn(len(lens), Hkv, G, D, generator=g).to(BF16).cuda()
        self.scale = D ** -0.5

    def check(self, out, cap=0.0, window=0, q=None, lens=None):
        q = self.q if q is None else q
        for b, n in enumerate(lens or self.lens):
            if n <= 0:
                assert (out[b] == 0).all()
                continue
            j = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
            at = self.table[b, j // self.page].long(), j % self.page
            ck, sk, zk = (x.transpose(0, 1) for x in cache4.parts(self.pools[0][at], self.D, False))
            cv, sv, zv = (x.transpose(0, 1) for x in cache4.parts(self.pools[1][at], self.D, True))
            qd = q[b].double()                          # Hkv, G, D; the others Hkv, n, D
            s = qd @ (zk + sk * ck).transpose(1, 2) * self.scale
            d = (2 ** -13 + 15 * 2 ** -20) * (qd.abs() @ sk.transpose(1, 2))
            d = (d + 2 ** -16 * (qd.abs() @ zk.abs().transpose(1, 2))) * self.scale
            d = d.amax(-1, keepdim=True)
            if cap:
                s = cap * torch.tanh(s / cap)
                d = d + 2 ** -10 * s.abs().amax(-1, keepdim=True)
            w = torch.softmax(s, -1)
            v = zv + sv * cv
            want = w @ v
            tol = 2 ** -8 * want.abs() + 2 ** -11 * (w @ (sv * (cv + 8))) + (2 * d + 2 ** -19) * (w @ v.abs())
            tol = tol + n * 2 ** -29 * sv.amax(1, keepdim=True)
            off = (out[b].double() - want).abs()
            assert (off <= tol).all(), (b, n, (off / tol).max().item())


def softcap(cap):
    return (S.ScoreMod(S.MOD_DIV, cap), S.ScoreMod(S.MOD_TANH), S.ScoreMod(S.MOD_MUL, cap)) if cap else ()


@pytest.mark.parametrize("lens,Hkv,G,D,page,layout,cap,window", [
    ([1], 1, 1, 64, 16, "head", 0.0, 0),
    ([1], 1, 1, 128, 16, "head", 0.0, 0),
    ([32, 31, 33], 2, 4, 128, 16, "head", 0.0, 0),
    ([15, 16, 17, 0, 64], 1, 8, 128, 16, "page", 0.0, 0),
    ([0, 0, 500, 0], 8, 4, 128, 16, "head", 0.0, 0),
    ([200, 3], 2, 3, 64, 24, "slots", 30.0, 0),
    ([100, 70, 1], 3, 9, 64, 1, "head", 0.0, 0),
    ([129, 260], 2, 17, 128, 7, "page", 50.0, 0),
    ([40, 300], 1, 128, 128, 32, "head", 0.0, 0),
    ([5, 64, 65, 700, 1000], 2, 4, 128, 16, "head", 0.0, 64),
    ([5, 64, 65, 700, 1000], 2, 5, 64, 24, "page", 20.0, 100),
    ([1000, 999, 998], 1, 2, 128, 8, "head", 0.0, 1),
    ([4097, 1, 2000], 4, 8, 64, 64, "head", 0.0, 0),
    ([9000], 1, 4, 128, 16, "head", 0.0, 0),
    ([20000, 30], 2, 1, 64, 16, "head", 0.0, 5000),
    ([7 * i % 90 for i in range(200)], 2, 2, 64, 16, "head", 0.0, 0),
])
def test_decode(lens, Hkv, G, D, page, layout, cap, window):
    x = Batch(lens, Hkv, G, D, page, seed=len(lens) + sum(lens), layout=layout)
    st = F.new_status("cuda")
    out = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, window=window, scale=x.scale,
                                  mods=softcap(cap), max_seq_len=max(lens), status=st)
    F.check_status(st)
    x.check(out, cap, window)
    # without a bound on the lengths, into an output of other strides, with a workspace of the caller's
    wide = torch.full((*x.q.shape[:2], G + 1, 2 * D), 3.0, dtype=BF16, device="cuda")
    ws = F.DecodeWorkspace()
    for _ in range(2):
        F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, window=window, scale=x.scale, mods=softcap(cap),
                                out=wide[:, :, :G, D:], workspace=ws, status=st)
    F.check_status(st)
    x.check(wide[:, :, :G, D:], cap, window)
    assert (wide[..., :D] == 3).all() and (wide[:, :, G] == 3).all()


@pytest.mark.parametrize("B", [32, 33, 70, 128, 129, 300])
def test_batches_around_what_is_added_up_at_once(B):
    """Lengths of 32 requests are looked at at a time, and from 129 on the join asks where parts are."""
    lens = [(37 * b * b) % 150 if b % 3 else 0 for b in range(B)]
    lens[B // 2] = 700
    x = Batch(lens, 1, 3, 64, 16, seed=B)
    for window in (0, 50):
        st = F.new_status("cuda")
        out = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, scale=x.scale, window=window, max_seq_len=700,
                                      status=st)
        F.check_status(st)
        x.check(out, window=window)


def test_two_calls_at_once_and_a_shared_row_of_the_table():
    x, y = Batch([900, 30], 2, 4, 128, 16, seed=31), Batch([64] * 5, 2, 4, 128, 16, seed=32)
    y.table = y.table[:1].expand(5, -1)                  # the same pages for all
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s, b in zip(streams, (x, y)):
            with torch.cuda.stream(s):
                outs.append((b, F.decode_attention_4bit(b.q, *b.pools, b.table, b.seq_lens, scale=b.scale)))
    torch.cuda.synchronize()
    for b, out in outs:
        assert torch.equal(out, outs[0][1] if b is x else outs[1][1])
    x.check(outs[0][1])
    y.check(outs[1][1])


def test_same_call_same_bits():
    x = Batch([700, 1300, 5], 4, 4, 128, 16, seed=3)
    one = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, scale=x.scale)
    for _ in range(5):
        assert torch.equal(one, F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, scale=x.scale))


def test_large_and_small_rows():
    """Scales far from one, scores that single out a key, and rows of zeros."""
    for amp, gain in ((1e-6, 1.0), (1e4, 1e-4), (1.0, 40.0)):
        x = Batch([300, 77], 2, 4, 128, 16, seed=5, amp=amp)
        x.q = (x.q.float() * gain).to(BF16)
        x.q[0, 0, 1] = 0
        out = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, scale=x.scale)
        x.check(out)


def test_nothing_behind_a_request_or_in_front_of_its_window_reaches_it():
    """Unused slots, pages of nobody and table entries behind the last key hold NaN scales or no page."""
    x = Batch([37, 90, 0, 150], 2, 4, 128, 16, seed=8)
    clean = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, scale=x.scale, window=40)
    used = torch.zeros(x.pages, 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate(x.lens):
        j = torch.arange(max(0, n - 40), n, device="cuda")
        used[x.table[b, j // 16].long(), j % 16] = True
    for pool in x.pools:
        pool[~used] = 0xFF                              # codes 15, scale and midpoint NaN
    table = x.table.clone()
    for b, n in enumerate(x.lens):
        table[b, :max(0, n - 40) // 16] = -1            # pages in front of the window were given back
    st = F.new_status("cuda")
    got = F.decode_attention_4bit(x.q, *x.pools, table, x.seq_lens, scale=x.scale, window=40, status=st)
    F.check_status(st)
    assert torch.equal(got, clean)
    x.check(got, window=40)


def test_lengths_and_pages_that_make_no_sense():
    x = Batch([40, 60], 1, 4, 64, 16, seed=9, spare=0)
    st = F.new_status("cuda")
    lens = torch.tensor([-5, 10 ** 9], dtype=torch.int32, device="cuda")
    out = F.decode_attention_4bit(x.q, *x.pools, x.table, lens, max_seq_len=60, scale=x.scale, status=st)
    x.check(out, lens=[0, 60])
    with pytest.raises(RuntimeError, match="max_seq_len"):
        F.check_status(st)
    st.zero_()
    table = x.table.clone()
    table[0, 1], table[1, 0] = 10 ** 6, -3
    assert F.decode_attention_4bit(x.q, *x.pools, table, x.seq_lens, scale=x.scale, status=st).isfinite().all()
    with pytest.raises(RuntimeError, match="page id"):
        F.check_status(st)
    out = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, max_seq_len=0, scale=x.scale)
    assert (out == 0).all()


@pytest.mark.parametrize("lens,Hkv,G,D,page,layout,cap,window", [
    ([0, 1, 512, 257, 33], 2, 4, 128, 16, "head", 30.0, 0),
    ([511, 480, 31, 0], 1, 11, 64, 32, "page", 0.0, 0),
    ([512, 100, 0, 7], 2, 3, 128, 24, "slots", 0.0, 0),
    ([3000, 1, 0, 496, 497, 498], 2, 8, 128, 16, "head", 0.0, 497),      # the longest that 16 groups hold
    ([3000, 1, 0, 497, 498, 499], 2, 8, 64, 16, "page", 20.0, 498),
])
def test_few_short_requests_and_the_same_among_many(lens, Hkv, G, D, page, layout, cap, window):
    """Few short requests take one launch; repeated until there are more of them than SMs, they take two. Lengths past
    the longest that the caller gives, or below zero, are cut and reported in both."""
    x = Batch(lens, Hkv, G, D, page, seed=7 + G, layout=layout)
    longest = max(lens)
    for times in (1, 80):
        tile = lambda t: t.repeat(times, *[1] * (t.dim() - 1))  # noqa: E731, B023
        q, table, seq_lens = tile(x.q), tile(x.table), tile(x.seq_lens)
        for bad in (False, True):
            st = F.new_status("cuda")
            if bad:
                seq_lens[seq_lens == longest], seq_lens[seq_lens == 0] = 2 ** 31 - 1, -1
            out = F.decode_attention_4bit(q, *x.pools, table, seq_lens, window=window, scale=x.scale,
                                          mods=softcap(cap), max_seq_len=longest, status=st)
            if bad:
                with pytest.raises(RuntimeError, match="max_seq_len"):
                    F.check_status(st)
            else:
                F.check_status(st)
            for t in (0, times - 1):
                x.check(out[t * len(lens):(t + 1) * len(lens)], cap, window)
    # a group that is infinite, in one request alone; a page that is not there
    st = F.new_status("cuda")
    short = lens.index(min(n for n in lens if n > 0))
    last = lens[short] - 1
    x.pools[1][x.table[short, last // page].item(), last % page, 0, D // 2:D // 2 + 2] = \
        torch.tensor([0x80, 0x7f], dtype=torch.uint8, device="cuda")     # its first scale
    out = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, window=window, scale=x.scale,
                                  mods=softcap(cap), max_seq_len=longest, status=st)
    F.check_status(st)
    assert not out[short, 0, :, :32].isfinite().any() and out[short, 0, :, 32:].isfinite().all()
    rest = [b for b in range(len(lens)) if b != short]
    assert out[rest].isfinite().all() and out[short, 1:].isfinite().all()
    x.table[0, 0] = 10 ** 6
    x.table[short, last // page] = -4
    F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, window=window, scale=x.scale, mods=softcap(cap),
                            max_seq_len=longest, status=st)
    with pytest.raises(RuntimeError, match="page id"):
        F.check_status(st)


def test_a_key_with_an_infinite_group_reaches_only_its_request_and_columns():
    x = Batch([20, 20], 1, 2, 64, 16, seed=12)
    at = x.table[0, 0].item()
    x.pools[1][at, 4, 0, 32:34] = torch.tensor([0x80, 0x7f], dtype=torch.uint8, device="cuda")   # its first scale
    out = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, scale=x.scale)
    assert not out[0, 0, :, :32].isfinite().any() and out[0, 0, :, 32:].isfinite().all()
    assert out[1].isfinite().all()


def test_other_stream_graph_and_shared_workspace():
    x = Batch([500, 33, 0, 1200], 4, 4, 128, 16, seed=13)
    args = (x.q, *x.pools, x.table, x.seq_lens)
    want = F.decode_attention_4bit(*args, scale=x.scale, max_seq_len=1200)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ws = F.DecodeWorkspace()
    with torch.cuda.stream(side):
        other = F.decode_attention_4bit(*args, scale=x.scale, max_seq_len=1200, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    # two graphs, each with its own memory, replayed in turn while lengths and queries change
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(F.decode_attention_4bit(*args, scale=x.scale, max_seq_len=1200))
        graphs.append(gr)
    for lens in ([500, 33, 0, 1200], [1, 1, 1, 1], [0, 0, 0, 0], [96, 32, 64, 1000]):
        x.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        x.table.copy_(torch.where(x.table < 0, 0, x.table))
        x.q.mul_(-1)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for out in outs:
            if max(lens[:3]) <= 500 and lens[1] <= 33:
                x.check(out, lens=lens)


def test_serving_steps_over_a_4bit_cache():
    """plan -> append with norm and rotation -> gather -> prompt attention, then decode steps: the same as the
    16-bit operators over what the 4-bit cache stands for."""
    Hq, Hkv, D, page, pages = 8, 2, 128, 16, 64
    g = torch.Generator().manual_seed(4)
    k_pool, v_pool = F.kv_cache_4bit(pages, page, Hkv, D)
    free = torch.randperm(pages, generator=g).int().cuda()
    prompts = [40, 3, 100]
    table = torch.full((3, 10), -1, dtype=torch.int32, device="cuda")
    rot = cache4.rotary_table(256, D)
    qw, kw = (1 + 0.1 * torch.randn(2, D, generator=g)).to(BF16).cuda()
    held = [0, 0, 0]
    st = F.new_status("cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for step, new in enumerate((prompts, [1, 1, 1], [17, 30, 1], [1, 1, 1], [1, 0, 1])):
        T = sum(new)
        qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g).to(BF16).cuda()
        q, k, v = qkv.split((Hq, Hkv, Hkv), 1)
        plan = F.plan_pages(ints(held), ints(new), free, table, page_size=page, num_tokens=T, status=st)
        free = free[int(plan.pages_used):]
        want_q, want_k = F.qk_norm_rotary(q, k, plan.positions, rot, q_weight=qw, k_weight=kw, status=st)
        q = F.kv_append_rotary(k, v, k_pool, v_pool, plan.slots, plan.positions, rot, q=q, q_weight=qw, k_weight=kw,
                               status=st)
        assert torch.equal(q, want_q)
        held = [h + n for h, n in zip(held, new)]
        cu_k = ints([0] + held).cumsum(0).int()
        keys, values = F.kv_gather_4bit(k_pool, v_pool, table, cu_k, sum(held), status=st)
        # the last rows of each request are this step's
        at = torch.cat([torch.arange(sum(held[:b + 1]) - new[b], sum(held[:b + 1])) for b in range(3)]).cuda()
        step_size = (want_k.float().unflatten(-1, (-1, 32)).amax(-1) - want_k.float().unflatten(-1, (-1, 32)).amin(-1)) / 15
        off = (keys[at].float() - want_k.float()).abs().unflatten(-1, (-1, 32)).amax(-1)
        assert (off <= 0.6 * step_size + 2 ** -6 * want_k.float().abs().amax()).all()
        o = F.packed_prefill_attention(q, keys, values, plan.cu_seqlens, cu_seqlens_k=cu_k, scale=D ** -0.5, status=st)
        if max(new) == 1:
            dec = torch.zeros(3, Hkv, Hq // Hkv, D, dtype=BF16, device="cuda")
            owner = [b for b in range(3) if new[b]]
            dec[owner] = q.unflatten(1, (Hkv, -1))
            lens = ints([h if n else 0 for h, n in zip(held, new)])
            got = F.decode_attention_4bit(dec, k_pool, v_pool, table, lens, scale=D ** -0.5, status=st)
            # both within their roundings (a few of bf16) of the same attention
            far = (got[owner].flatten(1, 2).float() - o.float()).norm() / o.float().norm()
            assert far < 4 * 2 ** -8
            assert math.isfinite(far) and (got[[b for b in range(3) if not new[b]]] == 0).all()
    F.check_status(st)


def test_scales_and_queries_from_one_end_of_their_range_to_the_other():
    """Column groups whose scales differ by 2^60 and grow from key to key, and query heads as far apart."""
    x = Batch([200, 45], 2, 4, 128, 16, seed=21)
    step = torch.linspace(-40, 40, x.pages * 16).reshape(x.pages, 16)
    for group, sign in ((0, 1), (1, -1), (3, 0)):        # group 2 as it was
        v = torch.randn(x.pages, 16, 2, 128, generator=torch.Generator().manual_seed(group)).cuda()
        v = v * 2.0 ** (sign * step.cuda() if sign else torch.full_like(step, -55.0).cuda())[..., None, None]
        rec = cache4.encode(v, True)
        meta = 64 + 2 * group
        x.pools[1][..., meta:meta + 2] = rec[..., meta:meta + 2]
        x.pools[1][..., meta + 8:meta + 10] = rec[..., meta + 8:meta + 10]
        for piece in range(8):                            # the group's 16-bit word of each piece
            b = 8 * piece + 2 * group
            x.pools[1][..., b:b + 2] = rec[..., b:b + 2]
    x.q = x.q * torch.tensor([2.0 ** -50, 1.0, 2.0 ** -10, 2.0 ** 3], device="cuda")[:, None].bfloat16()
    out = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, scale=x.scale)
    x.check(out)
    x.q[0, 0] *= 2.0 ** 40                                # and with a scale that brings them back
    x.q[1, 1] *= 2.0 ** 40
    out = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, scale=x.scale * 2.0 ** -40)
    x.scale *= 2.0 ** -40
    x.check(out)


def test_a_scale_of_zero_weighs_all_keys_alike():
    x = Batch([70, 33], 2, 4, 64, 16, seed=23)
    x.q *= 2.0 ** -30
    out = F.decode_attention_4bit(x.q, *x.pools, x.table, x.seq_lens, scale=0.0)
    x.scale = 0.0
    x.check(out)


def test_output_in_place_of_the_queries_or_apart_from_them():
    for lens in ([300, 12, 500], [2000, 12, 0]):         # one launch, and two
        x = Batch(lens, 2, 3, 64, 16, seed=41)
        args = (x.q, *x.pools, x.table, x.seq_lens)
        want = F.decode_attention_4bit(*args, scale=x.scale, max_seq_len=max(lens))
        room = torch.zeros(4, 2, 3, 64, dtype=BF16, device="cuda")
        room[:3] = x.q
        for out in (room[1:], room[:1].expand(3, -1, -1, -1), room[:3, :1].expand(-1, 2, -1, -1)):
            with pytest.raises(ValueError, match="out "):
                F.decode_attention_4bit(room[:3], *args[1:], scale=x.scale, max_seq_len=max(lens), out=out)
        with pytest.raises(ValueError, match="out "):
            F.decode_attention_4bit(*args, scale=x.scale, out=room)
        assert F.decode_attention_4bit(room[:3], *args[1:], scale=x.scale, max_seq_len=max(lens),
                                       out=room[:3]).data_ptr() == room.data_ptr()
        assert torch.equal(room[:3], want) and (room[3] == 0).all()
