"""A small serving loop over a paged KV cache: one system prompt, several requests behind it, then a few
decode steps, with the operators for requests of different lengths.

    python examples/serve_shared_prefix.py [--requests 8] [--prefix 512] [--prompt 100] [--steps 16]

One attention layer of a model stands in for the model: hidden rows are random, q, k and v are their
projections. Each step is the same few calls, and no call reads a length back to the host:

    plan_pages                       pages, slots and offsets of the step's tokens
    kv_append_packed                 their K/V rows into the cache
    packed_prefill_attention         prompts (all lengths in one batch), or
    shared_prefix_decode_attention   one token per request, the system prompt read once for all

At the end the last step is compared with paged_decode_attention, request by request.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from loopfuse_b200 import functional as F  # noqa: E402
from loopfuse_b200 import spec as S  # noqa: E402


class Layer:
    """One attention layer and its paged cache. The host keeps the requests' lengths (it made them) and so
    knows how many pages a step takes; tables, slots and offsets stay on the device."""

    def __init__(self, hq: int, hkv: int, d: int, pages: int, page_size: int, softcap: float, seed: int):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.hq, self.hkv, self.d, self.page_size = hq, hkv, d, page_size
        hidden = hq * d
        self.qkv = torch.randn(hidden, (hq + 2 * hkv) * d, generator=g, device="cuda",
                               dtype=torch.bfloat16) * hidden ** -0.5
        self.k_pool = torch.zeros(pages, page_size, hkv, d, device="cuda", dtype=torch.bfloat16)
        self.v_pool = torch.zeros_like(self.k_pool)
        self.free = torch.randperm(pages, generator=g, device="cuda").int()
        self.options = dict(scale=d ** -0.5)
        if softcap:
            self.options["mods"] = (S.ScoreMod(S.MOD_DIV, softcap), S.ScoreMod(S.MOD_TANH),
                                    S.ScoreMod(S.MOD_MUL, softcap))
        self.workspace = F.DecodeWorkspace()
        self.status = F.new_status("cuda")

    def _pages(self, n: int) -> int:
        return -(-n // self.page_size)

    def append(self, hidden: torch.Tensor, table: torch.Tensor, held: list[int], new: list[int]):
        """Project a packed batch, find its tokens' places and store its K/V rows."""
        qkv = (hidden @ self.qkv).unflatten(1, (-1, self.d))
        q, k, v = qkv.split((self.hq, self.hkv, self.hkv), dim=1)
        lens = torch.tensor([held, new], dtype=torch.int32).cuda(non_blocking=True)
        plan = F.plan_pages(lens[0], lens[1], self.free, table, page_size=self.page_size,
                            num_tokens=sum(new), status=self.status)
        taken = sum(self._pages(h + n) - self._pages(h) for h, n in zip(held, new))
        if taken > len(self.free):
            raise RuntimeError("the cache is full")
        self.free = self.free[taken:]
        F.kv_append_packed(k, v, self.k_pool, self.v_pool, plan.slots, status=self.status)
        return q, plan

    def prefill(self, hidden, table, held, new):
        q, plan = self.append(hidden, table, held, new)
        return F.packed_prefill_attention(q, self.k_pool, self.v_pool, plan.cu_seqlens, block_table=table,
                                          seq_lens=plan.seq_lens, workspace=self.workspace,
                                          status=self.status, **self.options)

    def decode(self, hidden, table, held, prefix_len):
        q, plan = self.append(hidden, table, held, [1] * len(held))
        q = q.unflatten(1, (self.hkv, -1))
        out = F.shared_prefix_decode_attention(q, self.k_pool, self.v_pool, table, plan.seq_lens, prefix_len,
                                               max_seq_len=max(held) + 1, workspace=self.workspace,
                                               status=self.status, **self.options)
        return q, out


def serve(requests: int, prefix: int, prompt: int, steps: int, hq: int = 8, hkv: int = 2, d: int = 128,
          page_size: int = 16, softcap: float = 0.0, seed: int = 0) -> float:
    """Runs the loop; the largest difference between its last step and paged_decode_attention."""
    prefix = -(-prefix // page_size) * page_size      # shared pages are whole ones
    prompts = [1 + (prompt * (i + 1)) // requests for i in range(requests)]
    longest = prefix + max(prompts) + steps
    pages = -(-prefix // page_size) + sum(-(-(p + steps) // page_size) for p in prompts) + requests
    layer = Layer(hq, hkv, d, pages, page_size, softcap, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)

    def hidden(n):
        return torch.randn(n, hq * d, generator=g, device="cuda", dtype=torch.bfloat16)

    width = -(-longest // page_size)
    # The system prompt, as a request of its own.
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    layer.prefill(hidden(prefix), table, [0], [prefix])
    # The requests: their rows begin with its pages, and it counts as cached.
    table = table.repeat(requests, 1)
    held = [prefix] * requests
    layer.prefill(hidden(sum(prompts)), table, held, prompts)
    held = [h + p for h, p in zip(held, prompts)]
    for _ in range(steps):
        q, out = layer.decode(hidden(requests), table, held, prefix)
        held = [h + 1 for h in held]
    F.check_status(layer.status, "serving loop")
    worst = 0.0
    for b, n in enumerate(held):
        for head in range(q.shape[2]):                # (any number of query heads per kv head)
            one = slice(head, head + 1)
            want = F.paged_decode_attention(q[b:b + 1, :, one].contiguous(), layer.k_pool, layer.v_pool,
                                            table[b:b + 1], seq_len=n, **layer.options)
            worst = max(worst, (out[b:b + 1, :, one].float() - want.float()).abs().max().item())
    return worst


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--requests", type=int, default=8)
    p.add_argument("--prefix", type=int, default=512)
    p.add_argument("--prompt", type=int, default=100)
    p.add_argument("--steps", type=int, default=16)
    p.add_argument("--softcap", type=float, default=0.0)
    a = p.parse_args()
    worst = serve(a.requests, a.prefix, a.prompt, a.steps, softcap=a.softcap)
    print(f"{a.requests} requests behind {a.prefix} shared tokens, {a.steps} steps: last step within "
          f"{worst:.2e} of paged_decode_attention")


if __name__ == "__main__":
    main()
