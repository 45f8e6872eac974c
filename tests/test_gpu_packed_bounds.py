"""The range-checking build (liblf_sm100_dbg.so) on the entry points for requests of different lengths:
ragged sizes, results as those of the plain formula, status word zero. The library is chosen when it is
loaded, so the cases run in a child process with LF_DEBUG_BOUNDS=1."""
import os
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

CHILD = textwrap.dedent("""
    import sys, torch
    sys.path.insert(0, %r)
    from loopfuse_b200 import _native, functional as F, spec as SP
    assert _native.load().lf_debug_bounds() == 1
    g = torch.Generator(device="cuda").manual_seed(31)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    st = F.new_status("cuda")

    def attend(q, k, v, off):
        s = q.float().transpose(0, 1) @ k.float().permute(1, 2, 0) * q.shape[-1] ** -0.5
        i = torch.arange(s.shape[1], device="cuda")[:, None] + off
        s = s.masked_fill(torch.arange(s.shape[2], device="cuda") > i, float("-inf"))
        return (torch.softmax(s, -1) @ v.float().transpose(0, 1)).transpose(0, 1)

    for D, Hq, Hkv, P in ((64, 3, 1, 4), (128, 8, 2, 16), (64, 4, 4, 24)):
        held, new = [0, 37, 130, 2500], [17, 1, 129, 5]
        B, T = 4, sum(new)
        blocks = [-(-(h + n) // P) for h, n in zip(held, new)]
        have = [-(-h // P) for h in held]
        ids = torch.randperm(sum(blocks) + 3, generator=g, device="cuda").int()
        table = torch.full((B, max(blocks)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b in range(B):
            table[b, :have[b]] = ids[at:at + have[b]]
            at += have[b]
        kp, vp = mk(len(ids), P, Hkv, D), mk(len(ids), P, Hkv, D)
        plan = F.plan_pages(ints(held), ints(new), ids[at:].contiguous(), table, page_size=P, num_tokens=T + 3,
                            status=st)
        k, v, q = mk(T + 3, Hkv, D), mk(T + 3, Hkv, D), mk(T + 3, Hq, D)
        F.kv_append_packed(k, v, kp, vp, plan.slots, status=st)
        got = F.packed_prefill_attention(q, kp, vp, plan.cu_seqlens, block_table=table, seq_lens=plan.seq_lens,
                                         scale=D ** -0.5, status=st)
        at = 0
        for b in range(B):
            j = torch.arange(held[b] + new[b], device="cuda")
            page = table[b, j // P].long()
            kk, vv = (x[page, j %% P].repeat_interleave(Hq // Hkv, 1) for x in (kp, vp))
            want = attend(q[at:at + new[b]], kk, vv, held[b])
            assert (got[at:at + new[b]].float() - want).abs().max().item() <= 2e-2, (D, b)
            at += new[b]
        cu = plan.cu_seqlens
        kd, vd = mk(T, Hkv, D), mk(T, Hkv, D)
        got = F.packed_prefill_attention(q[:T], kd, vd, cu, scale=D ** -0.5, status=st)
        for b in range(B):
            one = slice(int(cu[b]), int(cu[b + 1]))
            want = attend(q[one], *(x[one].repeat_interleave(Hq // Hkv, 1) for x in (kd, vd)), 0)
            assert (got[one].float() - want).abs().max().item() <= 2e-2, (D, b)
        # The last row's pages as everybody's prefix.
        prefix = 2048
        table[:, :prefix // P] = table[3, :prefix // P]
        if table.shape[1] * P > prefix and prefix %% P == 0:
            q1 = mk(B, Hkv, Hq // Hkv, D)
            lens = [prefix + 5, 0, prefix, prefix + 400]
            table[:, prefix // P:] = table[3, prefix // P:]
            table.clamp_(min=0)
            got = F.shared_prefix_decode_attention(q1, kp, vp, table, ints(lens), prefix, scale=D ** -0.5, status=st)
            for b in range(B):
                if not lens[b]:
                    assert (got[b] == 0).all()
                    continue
                j = torch.arange(lens[b], device="cuda")
                page = table[b, j // P].long()
                kk, vv = (x[page, j %% P].repeat_interleave(Hq // Hkv, 1) for x in (kp, vp))
                want = attend(q1[b].reshape(1, Hq, D), kk, vv, lens[b])
                assert (got[b].reshape(1, Hq, D).float() - want).abs().max().item() <= 2e-2, (D, b)
    torch.cuda.synchronize()
    assert int(st.item()) == 0, int(st.item())
    print("BOUNDS_OK")
""")


@pytest.mark.gpu
def test_packed_entry_points_stay_in_range():
    from loopfuse_b200.build import DBG_LIB_PATH, build_native
    if not DBG_LIB_PATH.exists():
        build_native(debug_bounds=True)
    env = dict(os.environ, LF_DEBUG_BOUNDS="1")
    r = subprocess.run([sys.executable, "-c", CHILD % str(ROOT)], env=env, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "BOUNDS_OK" in r.stdout, r.stdout + r.stderr
