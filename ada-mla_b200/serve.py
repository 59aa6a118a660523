"""One attention layer of a serving engine over a paged latent cache, on random weights:
prompts come in, then a tree of drafted tokens is verified.

    python ada-mla_b200/serve.py [--requests 4] [--heads 32] [--prompt 300] [--drafts 6]

Per step: ``mla_build_slots`` gives the new tokens their pages, ``mla_cache_write``
normalizes and rotates their latent rows into them, and then
* prompts attend in expanded form (``mla_prefill``: keys and values up-projected from the
  latent rows, one rope key per token), and
* drafts attend in absorbed form over the pages (``absorbed.absorb_query``,
  ``mla_decode_tree``, ``absorbed.project_output``).
The two forms are the same attention: the run ends with a check that each draft's output
is that of a prompt made of the request's tokens and the draft's ancestors.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import ada_mla  # noqa: E402
from ada_mla import absorbed  # noqa: E402

PAGE = 64
MAX_POSITIONS = 8192


def angles(n: int = MAX_POSITIONS) -> torch.Tensor:
    """[n, 64] fp32: cosines of the 32 angles of each position, then their sines."""
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    return torch.cat([a.cos(), a.sin()], 1).float().cuda()


def rotate(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor) -> torch.Tensor:
    """Rotary embedding of queries [T, n_h, 64], pairs (2i, 2i + 1)."""
    t = cos_sin[positions.long()][:, None]
    c, s, a, b = t[..., :32], t[..., 32:], x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2).to(x.dtype)


class Layer:
    """Attention weights of one layer and its page pool."""

    def __init__(self, heads: int, hidden: int, pages: int, requests: int, dtype=torch.bfloat16, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape):
            return (torch.randn(shape, generator=g, device="cuda") / shape[-2] ** 0.5).to(dtype)

        self.heads, self.dtype = heads, dtype
        self.w_q, self.w_kv = weight(hidden, heads * 192), weight(hidden, 576)
        self.w_uk, self.w_uv = weight(heads, 128, 512), weight(heads, 512, 128)
        self.norm = torch.ones(512, device="cuda", dtype=dtype)
        self.cos_sin = angles()
        self.pool = torch.zeros(pages, PAGE, 576, device="cuda", dtype=dtype)
        self.free = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.head = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.table = torch.full((requests, pages), -1, dtype=torch.int32, device="cuda")
        self.seq_lens = torch.zeros(requests, dtype=torch.int32, device="cuda")

    def append(self, x: torch.Tensor, new_lens: torch.Tensor) -> ada_mla.SlotPlan:
        """Gives the step's tokens (x [T, hidden], request by request) their slots and writes their latent rows."""
        plan = ada_mla.mla_build_slots(self.seq_lens, new_lens, self.table, self.free, PAGE, x.shape[0], free_head=self.head)
        ada_mla.mla_cache_write(x @ self.w_kv, plan.slots, self.pool, norm_weight=self.norm, positions=plan.positions, cos_sin=self.cos_sin)
        self.seq_lens, self.head = plan.seq_lens, plan.free_head
        return plan

    def queries(self, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        q = (x @ self.w_q).view(-1, self.heads, 192)
        return torch.cat([q[..., :128], rotate(q[..., 128:], positions, self.cos_sin)], -1)

    def prompts(self, x: torch.Tensor, new_lens: torch.Tensor, longest: int) -> torch.Tensor:
        """Prompts of requests that hold nothing yet -> per-head outputs [T, n_h, 128]."""
        plan = self.append(x, new_lens)
        rows = self.pool.view(-1, 576)[plan.slots]
        # one product gives every head's keys and values
        up = torch.cat([self.w_uk, self.w_uv.transpose(1, 2)], 1).reshape(-1, 512)
        kv = (rows[:, :512] @ up.t()).view(-1, self.heads, 256)
        return ada_mla.mla_prefill(self.queries(x, plan.positions), kv[..., :128], rows[:, 512:], kv[..., 128:], plan.cu_new, plan.cu_new,
                                   max_seq_len_q=longest, max_seq_len_k=longest)

    def drafts(self, x: torch.Tensor, mask: torch.Tensor, depth: torch.Tensor, longest: int) -> torch.Tensor:
        """k drafts per request (x [B, k, hidden]) with their tree -> [B, k, n_h, 128].

        A draft stands at the position after its parent's: ``depth`` [B, k], 0 for a
        draft that follows the context.
        """
        b, k, _ = x.shape
        before = self.seq_lens
        flat = x.reshape(b * k, -1)
        plan = ada_mla.mla_build_slots(before, torch.full_like(before, k), self.table, self.free, PAGE, b * k, free_head=self.head)
        positions = (before[:, None] + depth).flatten().to(torch.int32)
        ada_mla.mla_cache_write(flat @ self.w_kv, plan.slots, self.pool, norm_weight=self.norm, positions=positions, cos_sin=self.cos_sin)
        q = self.queries(flat, positions)
        q_star = absorbed.absorb_query(q[..., :128].contiguous(), q[..., 128:].contiguous(), self.w_uk)
        o_star = ada_mla.mla_decode_tree(q_star.view(b, k, self.heads, 576), self.pool, self.table, plan.seq_lens, mask, max_seq_len=longest)
        return absorbed.project_output(o_star.view(b * k, self.heads, 512), self.w_uv).view(b, k, self.heads, 128)


def run(requests: int = 4, heads: int = 32, prompt: int = 300, drafts: int = 6, hidden: int = 512, seed: int = 0) -> float:
    """Runs prompts and one draft tree; returns the largest difference between the two
    forms of attention over the drafts, relative to the outputs' root mean square."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(max(1, prompt // 2), prompt + 1, (requests,), generator=g)
    parents = ((torch.rand(requests, drafts, generator=g) * (torch.arange(drafts) + 1)).long() - 1)
    mask = ada_mla.tree_mask(parents)
    pages = int(((lens + drafts + PAGE - 1) // PAGE).sum())
    layer = Layer(heads, hidden, pages, requests, seed=seed)
    x = torch.randn(int(lens.sum()), hidden, generator=g).cuda().to(layer.dtype)
    d = torch.randn(requests, drafts, hidden, generator=g).cuda().to(layer.dtype)
    new_lens = lens.to(torch.int32).cuda()

    out = layer.prompts(x, new_lens, int(lens.max()))
    depth = torch.tensor([[bin(int(m) & (2 ** 64 - 1)).count("1") - 1 for m in row] for row in mask.tolist()])
    got = layer.drafts(d, mask.cuda(), depth.cuda(), int(lens.max()) + drafts)
    assert out.shape == (int(lens.sum()), heads, 128) and int(layer.head) <= pages

    # each draft again, as the last token of a prompt: the request's tokens and its ancestors
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    worst, size = 0.0, got.float().square().mean().sqrt().item()
    for b in range(requests):
        for i in range(drafts):
            path = [j for j in range(drafts) if (int(mask[b, i]) >> j) & 1]
            tokens = torch.cat([x[starts[b]:starts[b + 1]], d[b, path]])
            one = Layer(heads, hidden, -(-tokens.shape[0] // PAGE), 1, seed=seed)
            want = one.prompts(tokens, torch.tensor([tokens.shape[0]], dtype=torch.int32).cuda(), tokens.shape[0])[-1]
            worst = max(worst, (got[b, i].float() - want.float()).abs().max().item())
    return worst / size


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--drafts", type=int, default=6)
    a = ap.parse_args()
    far = run(a.requests, a.heads, a.prompt, a.drafts)
    print(f"{a.requests} prompts of up to {a.prompt} tokens, {a.drafts} drafts each, {a.heads} heads: "
          f"absorbed and expanded attention differ by {far:.3g} of the outputs' size")


if __name__ == "__main__":
    main()
