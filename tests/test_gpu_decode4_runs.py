"""Decode attention over a 4-bit cache where a warp has many groups of 32 keys in a row, against float64 on the values
that the records stand for: sums that meet in the middle of a run, scales and scores that move after they did.

All requests read the same pages, so that a batch of many groups takes little memory; their lengths differ, so that
units begin anywhere in a warp's run.

Tolerance of an output column, with w the softmax weights, u those over the largest of them and S their sum:
  2^-8 |o|                                    its own rounding to bf16
  sum_j e_j (c_j + 8)                         e_j, of a key's weight times its scale: rounded to fp16, 2^-11 w_j s_j, or
                                              where that is subnormal half a step, 2^-33 of the column group's largest
                                              scale (a step is 2^-24 where that scale is 2^8 or more) over S
  2 d sum_j w_j |v_j|                         what an error d of the scores does to the weights: the sums of the query
                                              row enter with 16 bits, 2^-16 of 8 |q| s and of |q| |z|, and sums in fp32
                                              are within 2^-20 of products of up to 15 |q| s; with a softcap 2^-10
                                              of the largest score (the unit's tanh is within 2^-11)
  n_g 2^-21 sum_j w_j (|v_j| + s_j (c_j + 8)) sums in fp32 over n_g groups: four additions of a column per group (of
                                              matrix products, which may cut instead of rounding: 2^-23), as many of the
                                              bottoms and of the weights
"""
import pytest
import torch

from loopfuse_b200 import _native
from loopfuse_b200 import functional as F
from loopfuse_b200 import spec as S
from tests import cache4

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
PAGE = 16


def batch_for(run, D, Hkv, groups):
    """Requests whose units give each warp of the GPU `run` groups (12 warps an SM at D = 128, 16 at 64)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return -(-run * sms * (12 if D == 128 else 16) // (Hkv * groups))


class Shared:
    """Requests that see the first lens[b] of the same keys, k and v [n, Hkv, D]."""

    def __init__(self, k, v, lens, G, seed, page=PAGE, layout="head"):
        n, Hkv, D = k.shape
        g = torch.Generator().manual_seed(seed)
        self.D, self.n, self.page = D, n, page
        pages = -(-n // page)
        ids = torch.randperm(pages + 2, generator=g)[:pages].cuda()
        self.rec, self.pools = [], []
        for x, value in ((k, False), (v, True)):
            rec = cache4.encode(x.float().cuda(), value)
            pool = torch.full((pages + 2, page, Hkv, rec.shape[-1]), 0xFF, dtype=torch.uint8, device="cuda")
            j = torch.arange(n, device="cuda")
            pool[ids[j // page], j % page] = rec
            if layout == "head":
                pool = pool.transpose(1, 2).contiguous().transpose(1, 2)
            self.rec.append(rec)
            self.pools.append(pool)
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.table = ids.int()[None].expand(len(lens), -1)
        self.q = torch.randn(len(lens), Hkv, G, D, generator=g).to(BF16).cuda()
        self.scale = D ** -0.5

    def run(self, cap=0.0, **kw):
        st = F.new_status("cuda")
        if cap:
            kw["mods"] = (S.ScoreMod(S.MOD_DIV, cap), S.ScoreMod(S.MOD_TANH), S.ScoreMod(S.MOD_MUL, cap))
        out = F.decode_attention_4bit(self.q, *self.pools, self.table, self.lens, max_seq_len=self.n, scale=self.scale,
                                      status=st, **kw)
        F.check_status(st)
        return out

    def check(self, out, window=0, cap=0.0):
        ck, sk, zk = (x.transpose(0, 1) for x in cache4.parts(self.rec[0], self.D, False))    # Hkv, n, D
        cv, sv, zv = (x.transpose(0, 1) for x in cache4.parts(self.rec[1], self.D, True))
        keys, v = (zk + sk * ck).transpose(1, 2), zv + sv * cv
        j = torch.arange(self.n, device="cuda")
        for lo in range(0, len(self.lens), 32):
            lens = self.lens[lo:lo + 32, None]
            seen = j < lens
            if window:
                seen &= j >= lens - window
            seen = seen[:, None, None]                                              # B, 1, 1, n
            q = self.q[lo:lo + 32].double()                                         # B, Hkv, G, D
            s = q @ keys * self.scale
            if cap:
                s = cap * torch.tanh(s / cap)
            largest = s.masked_fill(~seen, 0).abs().amax(-1, keepdim=True)
            s = s.masked_fill(~seen, -torch.inf)
            u = torch.exp(s - s.amax(-1, keepdim=True))
            total = u.sum(-1, keepdim=True)
            w = u / total
            d = (2 ** -13 + 15 * 2 ** -20) * (q.abs() @ sk.transpose(1, 2)) + 2 ** -16 * (q.abs() @ zk.abs().transpose(1, 2))
            d = (d * self.scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
            if cap:
                d = d + 2 ** -10 * largest
            want = w @ v
            # rounded weights: normal ones, and subnormal ones as if all were
            highest = torch.where(seen[:, :, 0, :, None], sv[None], 0.0).amax(2)     # B, Hkv, D
            e = torch.zeros_like(want)
            for g in range(0, self.D, 32):
                each = torch.maximum(2 ** -11 * w * sv[:, None, :, g], 2 ** -33 * highest[:, :, None, g, None] / total)
                e[..., g:g + 32] = (each * seen) @ (cv + 8)[..., g:g + 32]
            groups = -(-self.n // 32)
            size = w @ (v.abs() + sv * (cv + 8))
            tol = 2 ** -8 * want.abs() + e + 2 * d * (w @ v.abs()) + groups * 2 ** -21 * size
            off = (out[lo:lo + 32].double() - want).abs()
            assert (off <= tol).all(), (lo, (off / tol).nan_to_num(torch.inf).amax((1, 2, 3)).argmax().item(),
                                        (off / tol).nan_to_num(torch.inf).max().item())


def contexts(kind, n, Hkv, D, seed):
    """Keys and values: what changes along a context, in its first third and behind it."""
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(2, n, Hkv, D, generator=g)
    j = torch.arange(n)[:, None, None].float()
    first = j < n // 3
    flat = torch.randn(n, Hkv, D // 32, generator=g).bfloat16().float().repeat_interleave(32, -1)  # one value a group
    if kind == "growing":            # scales over 2^16, and scores that rise (or fall) along the context
        v = v * 2.0 ** (16.0 * j / n - 8)
        k[..., 0] += 12.0 * j[..., 0] / n
    elif kind == "constant first":   # scales of zero and midpoints, until a meeting of the sums has come
        v = torch.where(first, flat, v)
    elif kind == "constant":
        v = flat
    elif kind == "constant, then tiny":
        v = torch.where(first, 8 * flat, v * 2.0 ** -115)
    elif kind == "tiny, then constant":
        v = torch.where(first, v * 2.0 ** -115, flat * 2.0 ** 40)
    elif kind == "tiny":
        v = v * 2.0 ** -80
    elif kind == "huge":
        v = v * 2.0 ** 80
    else:
        assert kind == "plain"
    return k, v


@pytest.mark.parametrize("run,D,Hkv,G,n,page,layout,window", [
    (17, 128, 8, 1, 1900, 16, "head", 0), (33, 64, 8, 1, 1900, 16, "head", 0), (80, 128, 8, 1, 1900, 16, "head", 0),
    (18, 128, 8, 4, 1900, 16, "head", 0), (35, 128, 4, 9, 1900, 24, "page", 0), (20, 64, 8, 3, 1500, 24, "page", 0),
    (21, 128, 8, 8, 1900, 16, "head", 1000), (100, 64, 8, 4, 3300, 16, "head", 0), (100, 128, 16, 2, 3300, 16, "head", 0)])
@pytest.mark.parametrize("kind", ["plain", "growing", "constant first", "constant"])
def test_long_runs(kind, run, D, Hkv, G, n, page, layout, window):
    k, v = contexts(kind, n, Hkv, D, run)
    B = -(-batch_for(run, D, Hkv, (window or n - 100) // 32) // -(-G // 8))
    x = Shared(k, v, [n - 7 * b % 100 for b in range(B)], G, seed=run, page=page, layout=layout)
    x.q[..., 0] = torch.where(x.q[..., 0] < 0, -8.0, 8.0)           # up or down with the keys' first column
    x.check(x.run(window=window), window)


@pytest.mark.parametrize("D,G,page", [(64, 4, 16), (128, 1, 16), (128, 3, 24)])
@pytest.mark.parametrize("kind", ["plain", "constant first"])
def test_long_runs_under_a_softcap(kind, D, G, page):
    k, v = contexts(kind, 1900, 8, D, 11)
    x = Shared(k, v, [1900 - 7 * b % 100 for b in range(batch_for(25, D, 8, 56))], G, seed=12, page=page)
    x.check(x.run(cap=20.0), cap=20.0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["constant, then tiny", "tiny, then constant", "tiny", "huge"])
def test_midpoints_and_scales_of_other_sizes(kind, D):
    """Midpoints that are many times all scales of their columns, in front of these and behind them."""
    k, v = contexts(kind, 1900, 8, D, 3)
    B = batch_for(40, D, 8, 56)
    x = Shared(k, v, [1900 - 7 * b % 100 for b in range(B)], 1, seed=4)
    x.check(x.run())


def test_queries_of_every_size():
    """The largest column of a query row anywhere in the range of bfloat16, and a scale that brings the scores back."""
    for n, D in ((300, 128), (2500, 64)):               # one launch, and two
        k, v = contexts("plain", n, 2, D, 6)
        for power in (-117, -100, -60, 90, 95, 100, 112, 120):
            x = Shared(k, v, [n, n - 50], 4, seed=7)
            x.q = (x.q.float() * 2.0 ** power).to(BF16)
            x.scale *= 2.0 ** min(-power, 96)           # (a scale is below 10^30)
            x.check(x.run())
            if x.scale / 5.0 >= 1e6:                    # (what tanh takes is refused from there)
                with pytest.raises(_native.LfError):
                    x.run(cap=5.0)
            elif power < 115:                           # (scale over cap is an fp32 above 2^-126)
                x.check(x.run(cap=5.0), cap=5.0)


@pytest.mark.parametrize("ratio", [10, 16, 22, 26, 40])
@pytest.mark.parametrize("D,n,B", [(128, 450, 3), (64, 1900, 4), (128, 1900, 0)])
def test_weights_on_keys_whose_scales_are_far_below_the_largest(ratio, D, n, B):
    """A third of the keys, in front or behind, has scales 2^ratio times the others' and weights of 2^-40: what the
    others' weights lose is what the largest scale says, and up to a ratio of 2^16 or so it is nothing."""
    for front in (True, False):
        k, v = contexts("plain", n, 8, D, ratio)
        far = torch.arange(n) < n // 3 if front else torch.arange(n) >= n - n // 3
        k[far, :, 0] = -40.0 if D == 128 else -28.0
        v[far] *= 2.0 ** ratio
        lens = [n - 7 * b % 20 for b in range(B or batch_for(20, D, 8, 58))]
        x = Shared(k, v, lens, 1, seed=ratio)
        x.q[..., 0] = 8.0
        x.check(x.run())
