"""Cases of the operators of a batched decoding step over the page pool: the batch plan (page tables and slot maps), the append of new
K / V rows, attention of the new tokens over the pages, and filtered sampling of the next tokens.

``run`` computes a pass in elementary torch operations, or with ``own`` set through ``subspec_amd.ops``.  Lengths of a ragged batch come from
the case alone, values and the order of the pages from the seed."""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEVICE = "cuda:0" if torch.cuda.is_available() else "cpu"


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of a few sequences: bookkeeping before the first layer, where latency is all
        dict(name="plan 8 x 1", op="plan", batch=8, chunks=0, new=1, kv=2000, page_len=16),
        # a full server: hundreds of sequences, a few of them with long chunks of their prompts
        dict(name="plan 500 ragged", op="plan", batch=500, chunks=16, new=2000, kv=8192, page_len=16),
        # one token of each of 61 sequences, the Qwen2.5-7B cache (4 heads of 128)
        dict(name="append 61", op="append", tokens=61, pad=3, kv_heads=4, head_dim=128, page_len=16, dtype="bf16"),
        # prompts of 8191 tokens in all, 8 KV heads
        dict(name="append 8191", op="append", tokens=8191, pad=1, kv_heads=8, head_dim=128, page_len=16, dtype="fp16"),
        # one user with a long context
        dict(name="one token of 32768", op="attention", batch=1, chunks=0, new=1, kv=32768, q_heads=28, kv_heads=4, head_dim=128,
             page_len=16, window=0, sinks=0, dtype="bf16"),
        # a decoding step of a batch: bandwidth
        dict(name="64 single tokens", op="attention", batch=64, chunks=0, new=1, kv=4096, q_heads=28, kv_heads=4, head_dim=128,
             page_len=16, window=0, sinks=0, dtype="bf16"),
        # long streams that keep a window and their first tokens
        dict(name="48 single tokens, window", op="attention", batch=48, chunks=0, new=1, kv=16384, q_heads=32, kv_heads=8, head_dim=128,
             page_len=64, window=1024, sinks=4, dtype="fp16"),
        # decoding sequences and two that bring chunks of their prompts
        dict(name="16 mixed", op="attention", batch=16, chunks=2, new=500, kv=2500, q_heads=28, kv_heads=4, head_dim=128, page_len=16,
             window=0, sinks=0, dtype="bf16"),
        # the last chunk of a long prompt: matrix work
        dict(name="2048 behind 6144", op="attention", batch=1, chunks=1, new=2048, kv=8192, q_heads=28, kv_heads=4, head_dim=128,
             page_len=16, window=0, sinks=0, dtype="bf16"),
        # prompts of a small model, heads of 64, window
        dict(name="5 prompts, heads of 64", op="attention", batch=5, chunks=5, new=4096, kv=4096, q_heads=14, kv_heads=2, head_dim=64,
             page_len=16, window=1000, sinks=2, dtype="fp16"),
        # the next token of one sequence
        dict(name="sample 1 row", op="sample", rows=1, vocab=152064, dtype="fp32", temperature=0.7, top_k=50, top_p=0.9, min_p=0.0),
        # the next tokens of a batch, every row with its own settings around these
        dict(name="sample 64 rows", op="sample", rows=64, vocab=152064, dtype="bf16", temperature=1.0, top_k=0, top_p=0.95, min_p=0.02),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm, odd ones among them."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "attention", "attention", "sample", "sample"])
    if op == "plan":
        batch = _spread(rng, 1, 500)
        chunks = min(batch, rng.choice([0, 1, 3, 16]))
        return dict(op=op, batch=batch, chunks=chunks, new=_spread(rng, 2, 2000) if chunks else 1, kv=_spread(rng, 2001, 8192),
                    page_len=rng.choice([1, 4, 16, 64, 256]))
    if op == "append":
        return dict(op=op, tokens=_spread(rng, 1, 8191), pad=rng.choice([0, 1, 17]), kv_heads=rng.choice([1, 2, 4, 8]),
                    head_dim=rng.choice([64, 128]), page_len=rng.choice([1, 16, 64, 256]), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    if op == "sample":
        return dict(op=op, rows=_spread(rng, 1, 64), vocab=_spread(rng, 1000, 152064), dtype=rng.choice(["fp32", "bf16", "fp16"]),
                    temperature=rng.choice([0.0, 0.2, 0.7, 1.0, 1.5]), top_k=rng.choice([0, 1, 20, 50, 1000]),
                    top_p=rng.choice([1.0, 0.95, 0.9, 0.5]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]))
    q_heads, kv_heads, head_dim = rng.choice([(28, 4, 128), (32, 8, 128), (16, 8, 128), (64, 8, 128), (8, 1, 128), (32, 32, 128),
                                              (14, 2, 64), (32, 8, 64)])
    base = dict(op=op, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page_len=rng.choice([1, 8, 16, 64, 256]),
                window=rng.choice([0, 0, 0, 128, 1000]), sinks=rng.choice([0, 4, 64]), dtype=rng.choice(["bf16", "fp16"]))
    if base["window"] == 0:
        base["sinks"] = 0
    kind = rng.choice(["single", "single", "few", "mixed", "prompt"])
    if kind == "single":                              # one token a sequence, at most 2^20 rows of a head
        batch = _spread(rng, 1, 64)
        return dict(base, batch=batch, chunks=0, new=1, kv=_spread(rng, 16, max(32, min(32768, (1 << 20) // (batch * kv_heads)))))
    if kind == "few":                                 # a handful of tokens a sequence, as a draft's tokens under verification
        batch = _spread(rng, 1, 16)
        new = _spread(rng, 2, 33)
        return dict(base, batch=batch, chunks=batch, new=new, kv=_spread(rng, new, max(64, min(8192, (1 << 19) // (batch * kv_heads)))))
    if kind == "mixed":
        batch = _spread(rng, 2, 16)
        new = _spread(rng, 20, 500)
        return dict(base, batch=batch, chunks=rng.choice([1, 2]), new=new, kv=_spread(rng, new, 2500))
    batch = rng.choice([1, 1, 2, 5])                  # chunks of one prompt or a few
    new = _spread(rng, 64, min(2048, 2048 * 28 // (max(28, q_heads) * batch)))
    return dict(base, batch=batch, chunks=batch, new=new, kv=_spread(rng, new, min(8192, max(new + 1, 3 * new))))


def _lengths(case):
    """Rows of every sequence with its new ones, and how many are new: the first ones as long as the case says."""
    rng = random.Random("%s %s %s %s" % (case["batch"], case["chunks"], case["new"], case["kv"]))
    total, fresh = [], []
    for b in range(case["batch"]):
        n = 1 if b >= case["chunks"] else case["new"] if b == 0 else rng.randint(max(1, case["new"] // 3), case["new"])
        total.append(case["kv"] if b == 0 else max(n, rng.randint(max(1, case["kv"] // 4), case["kv"])))
        fresh.append(n)
    both = list(zip(total, fresh))
    random.Random(7).shuffle(both)
    return [t for t, _ in both], [n for _, n in both]


# ------------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=_DEVICE, dtype=torch.float32)


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    if case["op"] == "plan":
        total, fresh = _lengths(case)
        P = case["page_len"]
        have = [(t - n + P - 1) // P for t, n in zip(total, fresh)]
        width = (case["kv"] + P - 1) // P + 3
        n_pages = sum((t + P - 1) // P for t in total) + 11
        order = torch.randperm(n_pages, generator=g, device=_DEVICE).to(torch.int32)
        used = sum(have)
        cell = torch.arange(width, device=_DEVICE)[None, :]
        held = torch.tensor(have, device=_DEVICE)[:, None]
        first = torch.tensor([sum(have[:b]) for b in range(len(have))], device=_DEVICE)[:, None]
        table = torch.where(cell < held, order[(first + cell).clamp(max=n_pages - 1)], torch.full_like(order[:1], -1))
        return dict(case, table=table.contiguous(), free=order[used:].contiguous(),
                    n_free=torch.tensor([n_pages - used], dtype=torch.int32, device=_DEVICE),
                    kv_lens=torch.tensor([t - n for t, n in zip(total, fresh)], dtype=torch.int32, device=_DEVICE),
                    new_lens=torch.tensor(fresh, dtype=torch.int32, device=_DEVICE), tokens=sum(fresh))
    if case["op"] == "append":
        T, H, D, P = case["tokens"], case["kv_heads"], case["head_dim"], case["page_len"]
        dtype = _TYPES[case["dtype"]]
        pages = (T + P - 1) // P + 5
        qkv = _randn(g, T + case["pad"], 5 * H, D).to(dtype)                  # the fused projection: three times as many query heads
        slots = torch.randperm(pages, generator=g, device=_DEVICE)[:, None] * P + torch.arange(P, device=_DEVICE)[None, :]
        slots = torch.cat([slots.reshape(-1)[:T], torch.full((case["pad"],), -1, device=_DEVICE, dtype=torch.int64)])
        return dict(case, k=qkv[:, 3 * H:4 * H], v=qkv[:, 4 * H:], slots=slots, pool=_randn(g, pages, 2, P, H, D).to(dtype))
    if case["op"] == "sample":
        B, V = case["rows"], case["vocab"]
        # the logits of a language model: a wide body and a few tokens far ahead of it, on every row a different number
        logits = 2.0 * _randn(g, B, V)
        ahead = torch.randint(0, V, (B, 40), generator=g, device=_DEVICE)
        logits.scatter_add_(1, ahead, 6.0 + 2.0 * _randn(g, B, 40))
        turn = torch.arange(B, device=_DEVICE) % 4                              # every fourth row is hotter, or sees more
        temperature = torch.full((B,), float(case["temperature"]), device=_DEVICE) * torch.where(turn == 1, 1.3, 1.0)
        top_k = torch.full((B,), case["top_k"], dtype=torch.int32, device=_DEVICE) * torch.where(turn == 2, 2, 1).to(torch.int32)
        top_p = torch.where(turn == 3, torch.ones((), device=_DEVICE), torch.full((B,), float(case["top_p"]), device=_DEVICE))
        min_p = torch.full((B,), float(case["min_p"]), device=_DEVICE)
        return dict(case, logits=logits.to(_TYPES[case["dtype"]]), uniforms=torch.rand(B, generator=g, device=_DEVICE),
                    temperatures=temperature, top_ks=top_k, top_ps=top_p, min_ps=min_p)
    total, fresh = _lengths(case)
    Hq, Hkv, D, P = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_len"]
    dtype = _TYPES[case["dtype"]]
    counts = [(t + P - 1) // P for t in total]
    width, n_pages = max(counts), sum(counts) + 3
    order = torch.randperm(n_pages, generator=g, device=_DEVICE).to(torch.int32)
    cell = torch.arange(width, device=_DEVICE)[None, :]
    first = torch.tensor([sum(counts[:b]) for b in range(len(counts))], device=_DEVICE)[:, None]
    table = torch.where(cell < torch.tensor(counts, device=_DEVICE)[:, None], order[(first + cell).clamp(max=n_pages - 1)],
                        torch.full_like(order[:1], -1)).contiguous()
    pool = _randn(g, n_pages, 2, P, Hkv, D).to(dtype)
    kv_lens = torch.tensor(total, device=_DEVICE)
    # rows of a last page that no token has been written to hold whatever was there before
    row = torch.arange(P, device=_DEVICE)[None, :] + ((kv_lens + P - 1) // P - 1)[:, None] * P
    last = table.long().gather(1, ((kv_lens + P - 1) // P - 1)[:, None])[:, 0]
    stale = (row >= kv_lens[:, None])[:, None, :, None, None]
    pool[last] = torch.where(stale, torch.full_like(pool[:1, :1, :1, :1, :1], float("nan")), pool[last])
    starts = torch.tensor([sum(fresh[:b]) for b in range(len(fresh) + 1)], dtype=torch.int32, device=_DEVICE)
    T = sum(fresh)
    qkv = _randn(g, T, Hq + 2 * Hkv, D).to(dtype)                          # queries are a slice of the fused projection
    return dict(case, q=qkv[:, :Hq], pool=pool, table=table, starts=starts, kv_lens=kv_lens.to(torch.int32), max_new=max(fresh),
                max_kv=max(total), scale=2.0 / math.sqrt(D))


# ------------------------------------------------------------------------------------------------ plain forms
def _plan(s):
    """Page tables and slot maps; the free pages are a stack, handed out from its end in the order of the sequences."""
    P, T = s["page_len"], s["tokens"]
    dev = s["table"].device
    old, new = s["kv_lens"].long(), s["new_lens"].long()
    total = old + new
    have = (old + P - 1) // P
    need = (total + P - 1) // P - have
    starts = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    pages_before = need.cumsum(0) - need
    n_free = s["n_free"].long()
    cell = torch.arange(s["table"].shape[1], device=dev)[None, :]
    rank = pages_before[:, None] + cell - have[:, None]
    fresh = (cell >= have[:, None]) & (cell < (have + need)[:, None])
    table = s["table"]
    table.copy_(torch.where(fresh, s["free"][(n_free - 1 - rank).clamp(0, s["free"].numel() - 1)], table))
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(starts, t, right=True) - 1
    pos = old[seq] + t - starts[seq]
    slots = table[seq, pos // P].long() * P + pos % P
    used = need.sum()
    counts = torch.stack([starts[-1], used, n_free[0] - used, torch.zeros_like(used)])
    return dict(table=table, query_starts=starts.int(), kv_lens=total.int(), positions=pos.int(), slots=slots, sequences=seq.int(),
                counts=counts.int())


def _append(s):
    P = s["page_len"]
    slots = s["slots"]
    here = (slots >= 0).nonzero()[:, 0]
    pages, rows = slots[here] // P, slots[here] % P
    s["pool"][pages, 0, rows] = s["k"][here]
    s["pool"][pages, 1, rows] = s["v"][here]
    return s["pool"]


def _attention(s):
    """Sequences padded to the longest, in 32 bits."""
    P, N, S = s["page_len"], s["max_new"], s["max_kv"]
    dev = s["table"].device
    T, Hq, D = s["q"].shape
    Hkv = s["kv_heads"]
    G = Hq // Hkv
    starts, lens = s["starts"].long(), s["kv_lens"].long()
    B = lens.numel()
    fresh = starts[1:] - starts[:-1]
    j = torch.arange(S, device=dev)
    there = (j[None, :] < lens[:, None])[:, :, None, None]
    page = s["table"][:, j // P].long().clamp(min=0)
    k = s["pool"][page, 0, j % P].float().masked_fill(~there, 0.0)          # [B, S, Hkv, D]
    v = s["pool"][page, 1, j % P].float().masked_fill(~there, 0.0)
    i = torch.arange(N, device=dev)
    q = s["q"][(starts[:-1, None] + i[None, :]).clamp(max=T - 1)].float()   # [B, N, Hq, D]
    q = q.reshape(B, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B * Hkv, G * N, D)
    k = k.permute(0, 2, 3, 1).reshape(B * Hkv, D, S).contiguous()
    v = v.permute(0, 2, 1, 3).reshape(B * Hkv, S, D).contiguous()
    pos = (lens - fresh)[:, None] + i[None, :]                              # [B, N]
    seen = j[None, None, :] <= pos[:, :, None]
    if s["window"]:
        seen &= (j[None, None, :] > pos[:, :, None] - s["window"]) | (j < s["sinks"])
    score = torch.matmul(q, k).view(B, Hkv, G, N, S).mul_(s["scale"]).masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = score.sub_(top).exp_()
    out = torch.matmul(weight.view(B * Hkv, G * N, S), v).view(B, Hkv, G, N, D)
    mass = weight.sum(-1, keepdim=True)
    out = (out / mass.masked_fill(mass == 0, 1.0)).permute(0, 3, 1, 2, 4).reshape(B, N, Hq * D)
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(starts, t, right=True) - 1
    return out[seq, t - starts[seq]].to(s["q"].dtype)


def _sample(s):
    """In 64 bits: the order of the logits, the mass of everything before a place, the place where a number falls."""
    x = s["logits"].double()
    x = x.masked_fill(x.isnan(), float("-inf"))
    x, order = x.sort(dim=-1, descending=True, stable=True)
    V = x.shape[-1]
    top = x[:, :1]
    t = s["temperatures"].double()[:, None]
    e = ((x - top) / t.masked_fill(t == 0, 1.0)).exp().masked_fill(x == top, 1.0).masked_fill(x == float("-inf"), 0.0)
    rank = torch.arange(V, device=x.device)[None, :]
    k = s["top_ks"].long()[:, None]
    k = torch.where(t == 0, torch.ones_like(k), torch.where(k <= 0, torch.full_like(k, V), k))
    e = e.masked_fill(rank >= k, 0.0)
    before = e.cumsum(-1) - e
    p = s["top_ps"].double()[:, None]
    stays = (before < p * e.sum(-1, keepdim=True)) | (p >= 1.0) | (rank == 0)
    stays &= e >= s["min_ps"].double()[:, None]
    e = e.masked_fill(~stays, 0.0)
    mass = e.cumsum(-1)
    at = torch.searchsorted(mass, s["uniforms"].double()[:, None] * mass[:, -1:], right=True)
    at = torch.minimum(at, (e > 0).sum(-1, keepdim=True) - 1).clamp(min=0)
    some = mass[:, -1:] > 0
    token = torch.where(some, order.gather(1, at), torch.full_like(at, -1))[:, 0]
    prob = torch.where(some, e.gather(1, at) / mass[:, -1:], torch.zeros_like(mass[:, :1]))[:, 0]
    return token, prob.float()


def run(state):
    s = state
    if own:
        from subspec_amd import ops
        if s["op"] == "plan":
            out = ops.paged_batch_plan(s["kv_lens"], s["new_lens"], s["free"], s["n_free"], s["table"], s["page_len"], s["tokens"])
            return dict(out, table=s["table"])
        if s["op"] == "append":
            return ops.kv_append_paged_(s["pool"], s["k"], s["v"], s["slots"])
        if s["op"] == "attention":
            return ops.paged_attention(s["q"], s["pool"], s["table"], s["starts"], s["kv_lens"], s["max_new"], s["max_kv"],
                                       window=s["window"], sinks=s["sinks"], scale=s["scale"])
        return ops.sample_filtered(s["logits"], s["uniforms"], s["temperatures"], s["top_ks"], s["top_ps"], s["min_ps"])
    return {"plan": _plan, "append": _append, "attention": _attention, "sample": _sample}[s["op"]](s)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _seen(case, position):
    """Keys that the row at a position sees."""
    w = case["window"]
    if not w or position < w:
        return position + 1
    return w + min(case["sinks"], position + 1 - w)


def work(case):
    if case["op"] == "plan":
        total, fresh = _lengths(case)
        P = case["page_len"]
        pages = sum((t + P - 1) // P - (t - n + P - 1) // P for t, n in zip(total, fresh))
        # lengths read and written, pages taken and entered, the pages that tokens land in, 16 bytes a token
        touched = sum((t - 1) // P - (t - n) // P + 1 for t, n in zip(total, fresh))
        return {"bytes": 16 * case["batch"] + 8 * pages + 4 * touched + 16 * sum(fresh), "flops": 0}
    if case["op"] == "append":
        row = case["kv_heads"] * case["head_dim"] * (4 if case["dtype"] == "fp32" else 2)
        return {"bytes": case["tokens"] * (4 * row + 8), "flops": 0}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * (4 if case["dtype"] == "fp32" else 2) + 32), "flops": 0}
    total, fresh = _lengths(case)
    w, sinks = case["window"], case["sinks"]
    rows = pairs = 0
    for t, n in zip(total, fresh):
        low = max(0, t - n - w + 1) if w else 0
        rows += t - low + min(sinks, low)
        pairs += sum(_seen(case, p) for p in range(t - n, t))
    D, Hq, Hkv = case["head_dim"], case["q_heads"], case["kv_heads"]
    return {"bytes": rows * Hkv * D * 4 + sum(fresh) * Hq * D * 4, "flops": 4.0 * D * Hq * pairs}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    if case["op"] == "plan":
        return None                                     # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        P = case["page_len"]
        n, H, D = s["pool"].shape[0], case["kv_heads"], case["head_dim"]
        rows = s["pool"].double().transpose(1, 2).reshape(n * P, 2, H, D).clone()
        T = case["tokens"]
        rows[s["slots"][:T]] = torch.stack([s["k"][:T], s["v"][:T]], 1).double()
        return rows.view(n, P, 2, H, D).transpose(1, 2).contiguous()
    if case["op"] == "sample":
        tokens, probs = [], []
        for r in range(case["rows"]):
            l = s["logits"][r].double().cpu()
            order = torch.from_numpy(np.argsort(-l.numpy(), kind="stable"))                  # equal ones by index
            t, k = float(s["temperatures"][r]), int(s["top_ks"][r])
            x = l[order]
            e = torch.exp((x - x[0]) / t) if t > 0 else (x == x[0]).double()
            n = 1 if t == 0 else k if k > 0 else len(x)
            e = e[:n]
            mass, p = math.fsum(e.tolist()), float(s["top_ps"][r])
            before = torch.cat([torch.zeros(1, dtype=torch.float64), e.cumsum(0)[:-1]])
            n = max(1, int((before < p * mass).sum())) if p < 1 else len(e)
            n = min(n, int((e >= float(s["min_ps"][r])).sum()))
            sums, goal = e[:n].cumsum(0), float(s["uniforms"][r])
            j = min(int((sums <= goal * sums[-1]).sum()), n - 1)
            tokens.append(int(order[j]))
            probs.append(e[j] / sums[-1])
        return torch.tensor(tokens), torch.stack(probs)
    out = []
    starts, lens = s["starts"].tolist(), s["kv_lens"].tolist()
    P, Hq, Hkv, D = case["page_len"], case["q_heads"], case["kv_heads"], case["head_dim"]
    for b, total in enumerate(lens):
        n = starts[b + 1] - starts[b]
        pages = s["table"][b, :(total + P - 1) // P].long()
        kv = s["pool"][pages].transpose(0, 1).reshape(2, -1, Hkv, D)[:, :total].double()
        p = torch.arange(total - n, total, device=kv.device)[:, None]
        j = torch.arange(total, device=kv.device)[None, :]
        hidden = j > p
        if case["window"]:
            hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
        heads = []
        for h in range(Hq):
            one = s["q"][starts[b]:starts[b + 1], h].double()
            key, value = kv[0, :, h // (Hq // Hkv)].contiguous(), kv[1, :, h // (Hq // Hkv)].contiguous()
            a = (one @ key.t().contiguous() * s["scale"]).masked_fill(hidden, -math.inf).softmax(-1)
            heads.append(a @ value)
        out.append(torch.stack(heads, 1).reshape(n, Hq * D))
    return torch.cat(out)
