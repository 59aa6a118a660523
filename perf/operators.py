"""The operators around the paged latent cache, as cases that can be timed and compared.

Four operators of a serving step of latent attention (latent row: 512 latent + 64 rope
columns; query and key heads 128 + 64 wide in expanded form, value heads 128):

  slots    pages and slot maps for the tokens a step appends to its requests
  write    RMS norm + rotary embedding of latent rows, written to their slots
  tree     attention of a tree of drafted tokens over the paged latent cache
  prefill  attention over a prompt in expanded form, the rope key shared by all heads

``run`` computes each in elementary torch operations where ``own`` is false, and through
the package's entry points where it is true.
"""
import math
import os
import sys

import torch

own = False

LAT, ROPE, ROW, NOPE, VAL = 512, 64, 576, 128, 128
SCALE = 1.0 / math.sqrt(NOPE + ROPE)
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4, "e4m3": 1}


def ada_mla():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ada-mla_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import ada_mla

    return ada_mla


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 256 requests: one token each, a new page now and then
        {"name": "slots_decode", "op": "slots", "batch": 256, "lo": 1024, "hi": 8192, "new_lo": 1, "new_hi": 1, "page": 64},
        # admission of 93 new requests with prompts of 1 to 8192 tokens
        {"name": "slots_prompts", "op": "slots", "batch": 93, "lo": 0, "hi": 0, "new_lo": 1, "new_hi": 8192, "page": 64},
        # the decode step's 256 rows
        {"name": "write_decode", "op": "write", "tokens": 256, "src": "fp16", "dst": "fp16", "page": 64},
        # the rows of a long prompt, sliced out of a wider projection
        {"name": "write_prompt", "op": "write", "tokens": 32769, "src": "bf16", "dst": "bf16", "page": 64},
        # many prompts into an 8-bit cache with a scale for each row
        {"name": "write_prompt_8bit", "op": "write", "tokens": 131072, "src": "bf16", "dst": "e4m3", "page": 64},
        # 8 drafts of one sequence, 16 heads: 128 rows over a short cache
        {"name": "tree_one", "op": "tree", "batch": 1, "drafts": 8, "heads": 16, "lo": 4096, "hi": 4096, "page": 64, "type": "fp16"},
        # 7 drafts each of 64 sequences of mixed lengths
        {"name": "tree_batch", "op": "tree", "batch": 64, "drafts": 7, "heads": 16, "lo": 1024, "hi": 8192, "page": 64, "type": "fp16"},
        # 12 drafts with 128 heads: more rows than a tile
        {"name": "tree_wide", "op": "tree", "batch": 8, "drafts": 12, "heads": 128, "lo": 2048, "hi": 8192, "page": 128, "type": "bf16"},
        # one long context
        {"name": "tree_long", "op": "tree", "batch": 1, "drafts": 4, "heads": 128, "lo": 131072, "hi": 131072, "page": 64, "type": "fp16"},
        # one short prompt
        {"name": "prefill_short", "op": "prefill", "batch": 1, "heads": 128, "q_lo": 77, "q_hi": 77, "past": 0, "type": "bf16"},
        # mixed prompts in one packed batch
        {"name": "prefill_mixed", "op": "prefill", "batch": 6, "heads": 128, "q_lo": 100, "q_hi": 2048, "past": 0, "type": "fp16"},
        # a chunk of a prompt over what is cached already
        {"name": "prefill_chunk", "op": "prefill", "batch": 1, "heads": 128, "q_lo": 2048, "q_hi": 2048, "past": 6144, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    op = rng.choice(["slots", "write", "tree", "tree", "prefill", "prefill"])
    if op == "slots":
        if rng.random() < 0.5:
            lo = _log(rng, 1, 4096)
            return {"op": op, "batch": _log(rng, 1, 1024), "lo": lo, "hi": lo + _log(rng, 1, 8192), "new_lo": 1, "new_hi": rng.choice([1, 4, 8]),
                    "page": rng.choice([32, 64, 128])}
        return {"op": op, "batch": _log(rng, 1, 93), "lo": 0, "hi": rng.choice([0, 1000]), "new_lo": 1, "new_hi": _log(rng, 16, 8192),
                "page": rng.choice([32, 64, 128])}
    if op == "write":
        return {"op": op, "tokens": _log(rng, 1, 131072), "src": rng.choice(["fp16", "bf16", "fp32"]), "dst": rng.choice(["fp16", "bf16", "e4m3"]),
                "page": rng.choice([32, 64, 128])}
    if op == "tree":
        while True:
            lo = _log(rng, 100, 65536)
            c = {"op": op, "batch": _log(rng, 1, 64), "drafts": _log(rng, 1, 32), "heads": rng.choice([8, 16, 32, 64, 128]), "lo": lo,
                 "hi": lo + _log(rng, 1, 8192), "page": rng.choice([32, 64, 128]), "type": rng.choice(["fp16", "bf16"])}
            if c["batch"] * c["hi"] <= 300000 and c["batch"] * c["hi"] * c["drafts"] * c["heads"] <= 6.0e7:
                return c
    while True:
        lo = _log(rng, 16, 4096)
        c = {"op": op, "batch": _log(rng, 1, 8), "heads": rng.choice([8, 32, 64, 128]), "q_lo": lo, "q_hi": lo + _log(rng, 1, 2048),
             "past": rng.choice([0, 0, _log(rng, 16, 8192)]), "type": rng.choice(["fp16", "bf16"])}
        if c["batch"] * c["heads"] * c["q_hi"] * (c["q_hi"] + c["past"]) <= 1.8e9:
            return c


def _spread(lo, hi, batch):
    """`batch` lengths spread evenly over lo..hi: how many tokens there are in all does not go by the seed."""
    return [lo + (hi - lo) * (2 * i + 1) // (2 * batch) for i in range(batch)]


def work(case):
    op = case["op"]
    if op == "slots":
        b, p = case["batch"], case["page"]
        tokens = sum(_spread(case["new_lo"], case["new_hi"], b))
        return {"bytes": 20 * b + 12 * tokens + 8 * tokens / p, "flops": 0}
    if op == "write":
        t = case["tokens"]
        return {"bytes": t * (ROW * (SIZE[case["src"]] + SIZE[case["dst"]]) + 12 + (4 if case["dst"] == "e4m3" else 0)) + 4 * ROPE * min(t, 8192),
                "flops": 5 * t * ROW}
    if op == "tree":
        rows = case["drafts"] * case["heads"]
        total = sum(_spread(case["lo"], case["hi"], case["batch"])) + case["batch"] * case["drafts"]
        return {"bytes": total * ROW * 2 + case["batch"] * rows * ((ROW + LAT) * 2 + 4), "flops": 2 * rows * (ROW + LAT) * total}
    h, past = case["heads"], case["past"]
    lens = _spread(case["q_lo"], case["q_hi"], case["batch"])
    pairs = sum(n * past + n * (n + 1) / 2.0 for n in lens)
    nq, nk = sum(lens), sum(lens) + past * len(lens)
    return {"bytes": 2 * (nq * h * (NOPE + ROPE + VAL) + nk * (h * (NOPE + VAL) + ROPE)) + 4 * nq * h, "flops": 2 * h * (NOPE + ROPE + VAL) * pairs}


# ----------------------------------------------------------------------------- inputs
def _cu(lens):
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens, dtype=torch.int64), 0)
    return cu.cuda()


def prepare(case, seed):
    op, dev = case["op"], "cuda"
    cpu = torch.Generator().manual_seed(seed * 104729 + 5)
    gen = torch.Generator(device=dev).manual_seed(seed * 15485863 + 3)
    s = dict(case)

    def lengths(lo, hi):
        """The case's lengths, in an order of the seed's."""
        some = _spread(lo, hi, case["batch"])
        return [some[i] for i in torch.randperm(case["batch"], generator=cpu).tolist()]

    def table_of(lens, page, extra, gen):
        """A block table over a shuffled pool with room for `extra` more pages a request: (table, pages in all)."""
        have = [-(-n // page) for n in lens]
        pages = sum(have) + extra
        perm = torch.randperm(pages, generator=gen).to(torch.int32)
        width = max(max(have), 1)
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(have):
            table[b, :n] = perm[at:at + n]
            at += n
        return table, perm[at:], pages

    def rand(*shape, type="fp16", scale=1.0):
        out = torch.empty(shape, dtype=TYPES[type], device=dev)
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 26):
            j = min(flat.numel(), i + (1 << 26))
            flat[i:j] = torch.randn(j - i, generator=gen, device=dev) * scale
        return out

    if op == "slots":
        have = lengths(case["lo"], case["hi"])
        new = lengths(case["new_lo"], case["new_hi"])
        page = case["page"]
        need = sum(-(-(h + n) // page) + (-h // page) for h, n in zip(have, new))
        table, free, _ = table_of(have, page, need + 64, cpu)
        width = -(-(case["hi"] + case["new_hi"]) // page) + 8
        wide = torch.full((case["batch"], width), -1, dtype=torch.int32)
        wide[:, :table.shape[1]] = table[:, :width]
        s.update(seq_lens=torch.tensor(have, dtype=torch.int32).cuda(), new_lens=torch.tensor(new, dtype=torch.int32).cuda(), table=wide.cuda(),
                 free=free.cuda(), head=torch.tensor([3], dtype=torch.int32).cuda(), tokens=sum(new))
    elif op == "write":
        t, page = case["tokens"], case["page"]
        pages = -(-t // page) + 16
        slots = torch.randperm(pages, generator=cpu)[:, None] * page + torch.arange(page)
        angles = torch.arange(8192, device=dev, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(0, ROPE, 2, device=dev, dtype=torch.float64) / ROPE))
        s.update(latent=rand(t, 128 + ROW, type=case["src"])[:, 128:], slots=slots.view(-1)[:t].contiguous().cuda(),
                 positions=torch.randint(0, 8192, (t,), generator=cpu).to(torch.int32).cuda(),
                 weight=(1 + rand(LAT, type="fp32", scale=0.1)).to(TYPES[case["src"]]),
                 cos_sin=torch.cat([angles.cos(), angles.sin()], 1).float().contiguous(),
                 cache=torch.zeros(pages, page, ROW, device=dev, dtype=torch.float16).to(TYPES[case["dst"]]),
                 scales=torch.ones(pages * page, device=dev) if case["dst"] == "e4m3" else None)
    elif op == "tree":
        k, h = case["drafts"], case["heads"]
        lens = [n + k for n in lengths(case["lo"], case["hi"])]
        table, _, pages = table_of(lens, case["page"], 3, cpu)
        # each draft's parent is an earlier draft or the context itself; a draft sees its ancestors and itself
        mask = torch.zeros(case["batch"], k, dtype=torch.int64)
        parent = (torch.rand(case["batch"], k, generator=cpu) * (torch.arange(k) + 1)).long() - 1
        for i in range(k):
            up = torch.gather(mask, 1, parent[:, i:i + 1].clamp(min=0))[:, 0]
            mask[:, i] = torch.where(parent[:, i] >= 0, up, 0) | (1 << i)
        s.update(query=rand(case["batch"], k, h, ROW, type=case["type"]), pages=rand(pages, case["page"], ROW, type=case["type"]), table=table.cuda(),
                 seq_lens=torch.tensor(lens, dtype=torch.int32).cuda(), mask=mask.cuda(), longest=max(lens), lens=lens)
    else:
        h, past = case["heads"], case["past"]
        lens = lengths(case["q_lo"], case["q_hi"])
        both = [n + past for n in lens]
        kv = rand(sum(both), h, NOPE + VAL, type=case["type"])  # one up-projection gives keys and values
        s.update(query=rand(sum(lens), h, NOPE + ROPE, type=case["type"]), k_nope=kv[:, :, :NOPE], v=kv[:, :, NOPE:],
                 k_rope=rand(sum(both), ROPE, type=case["type"]), cu_q=_cu(lens), cu_k=_cu(both), lens_q=lens, lens_k=both, longest_q=max(lens), longest_k=max(both))
    return s


# ----------------------------------------------------------------------------- one pass
def run(s):
    return (OWN if own else PLAIN)[s["op"]](s)


def own_slots(s):
    p = ada_mla().mla_build_slots(s["seq_lens"], s["new_lens"], s["table"], s["free"], s["page"], s["tokens"], free_head=s["head"])
    return {"slots": p.slots, "positions": p.positions, "cu_new": p.cu_new, "seq_lens": p.seq_lens, "head": p.free_head, "table": s["table"]}


def own_write(s):
    ada_mla().mla_cache_write(s["latent"], s["slots"], s["cache"], norm_weight=s["weight"], eps=1e-6, positions=s["positions"], cos_sin=s["cos_sin"],
                              kv_scales=s["scales"])
    return {"cache": s["cache"]} if s["scales"] is None else {"cache": s["cache"], "scales": s["scales"]}


def own_tree(s):
    out, lse = ada_mla().mla_decode_tree(s["query"], s["pages"], s["table"], s["seq_lens"], s["mask"], max_seq_len=s["longest"], softmax_scale=SCALE,
                                         return_lse=True)
    return {"out": out, "lse": lse}


def own_prefill(s):
    out, lse = ada_mla().mla_prefill(s["query"], s["k_nope"], s["k_rope"], s["v"], s["cu_q"], s["cu_k"], max_seq_len_q=s["longest_q"],
                                     max_seq_len_k=s["longest_k"], softmax_scale=SCALE, causal=True, return_lse=True)
    return {"out": out, "lse": lse}


def plain_slots(s):
    page, table, free = s["page"], s["table"], s["free"]
    have, new = s["seq_lens"].long(), s["new_lens"].long()
    old = (have + page - 1) // page
    need = (have + new + page - 1) // page - old
    cu = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    off = need.cumsum(0) - need
    head = s["head"].long()
    token = torch.arange(s["tokens"], device=cu.device)
    req = torch.searchsorted(cu[1:], token, right=True)
    pos = have[req] + token - cu[req]
    block = pos // page
    fresh = free[(head + off[req] + block - old[req]).clamp(0, free.numel() - 1)].long()
    at = torch.where(block >= old[req], fresh, table[req, block].long())
    table[req, block] = at.int()
    return {"slots": at * page + pos % page, "positions": pos.int(), "cu_new": cu.int(), "seq_lens": (have + new).int(), "head": (head + need.sum()).int(),
            "table": table}


def plain_write(s):
    x = s["latent"].float()
    c, r = x[:, :LAT], x[:, LAT:]
    c = c * torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-6) * s["weight"].float()
    cs = s["cos_sin"][s["positions"].long()]
    cos, sin = cs[:, :ROPE // 2], cs[:, ROPE // 2:]
    a, b = r[:, 0::2], r[:, 1::2]
    r = torch.stack([a * cos - b * sin, a * sin + b * cos], 2).flatten(1)
    row, cache = torch.cat([c, r], 1), s["cache"].view(-1, ROW)
    if s["scales"] is None:
        cache[s["slots"]] = row.to(cache.dtype)
        return {"cache": s["cache"]}
    scale = row.abs().amax(1) / 448.0
    cache.view(torch.uint8)[s["slots"]] = (row / scale[:, None]).to(cache.dtype).view(torch.uint8)
    s["scales"][s["slots"]] = scale
    return {"cache": s["cache"], "scales": s["scales"]}


def plain_tree(s):
    page, k = s["page"], s["drafts"]
    token = torch.arange(s["longest"], device=s["table"].device)
    rows = s["table"][:, token // page].long().clamp(min=0) * page + token % page
    c = s["pages"].view(-1, ROW)[rows].float()
    start = (s["seq_lens"].long() - k)[:, None]
    j = (token[None] - start).clamp(0, 63)
    draft = (s["mask"][:, :, None] >> j[:, None]) & 1
    seen = (token < start)[:, None] | ((token >= start) & (token < start + k))[:, None] & (draft == 1)
    q = s["query"].float()
    b, _, h, _ = q.shape
    x = torch.bmm(q.view(b, k * h, ROW), c.transpose(1, 2)).view(b, k, h, -1) * SCALE
    x = x.masked_fill(~seen[:, :, None], float("-inf"))
    top = x.amax(3, keepdim=True)
    x = (x - top).exp_()
    total = x.sum(3, keepdim=True)
    o = torch.bmm(x.view(b, k * h, -1), c[:, :, :LAT]).view(b, k, h, LAT) / total
    return {"out": o.to(s["query"].dtype), "lse": (top + total.log())[..., 0]}


def plain_prefill(s):
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    i = torch.arange(s["longest_q"], device=cu_q.device)
    j = torch.arange(s["longest_k"], device=cu_q.device)
    nq, nk = (cu_q[1:] - cu_q[:-1])[:, None], (cu_k[1:] - cu_k[:-1])[:, None]
    at_q = (cu_q[:-1, None] + i).clamp(max=s["query"].shape[0] - 1)
    at_k = (cu_k[:-1, None] + j).clamp(max=s["k_rope"].shape[0] - 1)
    q = s["query"][at_q].float().transpose(1, 2)                     # [B, H, Q, 192]
    key = s["k_nope"][at_k].float().permute(0, 2, 3, 1)              # [B, H, 128, K]
    rope = s["k_rope"][at_k].float().transpose(1, 2)[:, None]        # [B, 1, 64, K]
    v = s["v"][at_k].float().transpose(1, 2)
    x = torch.matmul(q[..., :NOPE], key)
    x += torch.matmul(q[..., NOPE:], rope)
    x *= SCALE
    seen = (j[None, None] <= (i[None] + nk - nq)[:, :, None]) & (j < nk)[:, None]
    x.masked_fill_(~seen[:, None], float("-inf"))
    top = x.amax(3, keepdim=True)
    x -= top
    x.exp_()
    total = x.sum(3, keepdim=True)
    o = (torch.matmul(x, v) / total).transpose(1, 2)
    real = i < nq
    return {"out": o[real].to(s["query"].dtype), "lse": (top + total.log())[..., 0].transpose(1, 2)[real]}


OWN = {"slots": own_slots, "write": own_write, "tree": own_tree, "prefill": own_prefill}
PLAIN = {"slots": plain_slots, "write": plain_write, "tree": plain_tree, "prefill": plain_prefill}


# ----------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """Each operator's outputs from its definition in 64 bits, a sequence at a time."""
    def exact_slots(s):
        have, new, page = s["seq_lens"].tolist(), s["new_lens"].tolist(), s["page"]
        table, free = s["table"].cpu().clone(), s["free"].tolist()
        head, slots, positions, cu = int(s["head"]), [], [], [0]
        for b, (n, m) in enumerate(zip(have, new)):
            for block in range(-(-n // page), -(-(n + m) // page)):
                table[b, block] = free[head]
                head += 1
            row = table[b].tolist()
            positions += range(n, n + m)
            slots += [row[p // page] * page + p % page for p in range(n, n + m)]
            cu.append(cu[-1] + m)
        whole = {"cu_new": cu, "head": [head], "positions": positions, "seq_lens": [n + m for n, m in zip(have, new)]}
        return {**{k: torch.tensor(v, dtype=torch.int32) for k, v in whole.items()}, "slots": torch.tensor(slots, dtype=torch.int64), "table": table}

    def exact_write(s):
        x, out = s["latent"].double(), s["cache"].view(-1, ROW).double()
        c = x[:, :LAT] / torch.sqrt(x[:, :LAT].pow(2).sum(1, keepdim=True) / LAT + 1e-6) * s["weight"].double()
        z = torch.complex(x[:, LAT::2], x[:, LAT + 1::2])
        t = s["cos_sin"].double()[s["positions"].long()]
        r = torch.view_as_real(z * torch.complex(t[:, :ROPE // 2], t[:, ROPE // 2:])).flatten(1)
        row = torch.cat([c, r], 1)
        if s["scales"] is None:
            out[s["slots"]] = row
            return {"cache": out.view_as(s["cache"])}
        scales = s["scales"].double()
        scales[s["slots"]] = row.abs().amax(1) / 448
        out[s["slots"]] = row / scales[s["slots"], None]
        return {"cache": out.view_as(s["cache"]), "scales": scales}

    def exact_tree(s):
        k, page, outs, lses = s["drafts"], s["page"], [], []
        for b, n in enumerate(s["lens"]):
            table = s["table"][b, :-(-n // page)].long()
            c = s["pages"][table].reshape(-1, ROW)[:n].double()
            seen = torch.ones(k, n, dtype=torch.bool, device=c.device)
            seen[:, n - k:] = torch.tensor([[(m >> j) & 1 for j in range(k)] for m in s["mask"][b].tolist()], device=c.device) == 1
            one = [torch.einsum("hd,td->ht", s["query"][b, i].double(), c[seen[i]]) * SCALE for i in range(k)]
            lses.append(torch.stack([torch.logsumexp(x, 1) for x in one]))
            outs.append(torch.stack([torch.softmax(x, 1) @ c[seen[i], :LAT] for i, x in enumerate(one)]))
        return {"out": torch.stack(outs), "lse": torch.stack(lses)}

    def exact_prefill(s):
        outs, lses, q0, k0 = [], [], 0, 0
        for nq, nk in zip(s["lens_q"], s["lens_k"]):
            o = torch.empty(nq, s["heads"], VAL, dtype=torch.float64, device="cuda")
            lse = torch.empty(nq, s["heads"], dtype=torch.float64, device="cuda")
            rope = s["k_rope"][k0:k0 + nk].double()
            late = torch.arange(nk, device="cuda")[None] > (torch.arange(nq, device="cuda") + nk - nq)[:, None]
            for h in range(s["heads"]):
                key = torch.cat([s["k_nope"][k0:k0 + nk, h].double(), rope], 1)
                x = (s["query"][q0:q0 + nq, h].double() @ key.t() * SCALE).masked_fill_(late, float("-inf"))
                lse[:, h] = torch.logsumexp(x, 1)
                o[:, h] = torch.softmax(x, 1) @ s["v"][k0:k0 + nk, h].double()
            outs.append(o)
            lses.append(lse)
            q0, k0 = q0 + nq, k0 + nk
        return {"out": torch.cat(outs), "lse": torch.cat(lses)}

    s = prepare(case, seed)
    return {"slots": exact_slots, "write": exact_write, "tree": exact_tree, "prefill": exact_prefill}[case["op"]](s)
