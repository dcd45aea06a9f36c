"""Cases of the operators of a batched step over long contexts with sampled drafts: bounds of the pages' keys, the blocks that a token
attends to by them, attention over those blocks, and verification of drafts against the target's probabilities.

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
        # a decoding step: one token a sequence, a page in sixteen is full with it (the Qwen2.5-7B cache, 4 heads of 128)
        dict(name="bounds, step of 61", op="bounds", tokens=61, first=7, stride=1, kv_heads=4, head_dim=128, page_len=16, dtype="bf16"),
        # chunks of prompts: every page of them
        dict(name="bounds, prompt of 8191", op="bounds", tokens=8191, first=0, stride=0, kv_heads=8, head_dim=128, page_len=16, dtype="fp16"),
        # one user with a long context: latency
        dict(name="select, one token of 32768", op="select", batch=1, new=1, kv=32768, q_heads=28, kv_heads=4, head_dim=128, page_len=16,
             keep=64, recent=2, dtype="bf16"),
        # a decoding step of a batch with long contexts: bandwidth
        dict(name="select, 64 tokens", op="select", batch=64, new=1, kv=32768, q_heads=28, kv_heads=4, head_dim=128, page_len=16,
             keep=64, recent=2, dtype="bf16"),
        # drafted tokens under verification, large pages
        dict(name="select, 16 x 5 drafts", op="select", batch=16, new=5, kv=16384, q_heads=32, kv_heads=8, head_dim=128, page_len=64,
             keep=32, recent=1, dtype="fp16"),
        # the same three steps' attention over what was selected
        dict(name="attend, one token of 32768", op="attend", batch=1, new=1, kv=32768, q_heads=28, kv_heads=4, head_dim=128, page_len=16,
             keep=64, recent=2, dtype="bf16"),
        dict(name="attend, 64 tokens", op="attend", batch=64, new=1, kv=16384, q_heads=28, kv_heads=4, head_dim=128, page_len=16,
             keep=64, recent=2, dtype="bf16"),
        dict(name="attend, 16 x 5 drafts", op="attend", batch=16, new=5, kv=16384, q_heads=32, kv_heads=8, head_dim=128, page_len=64,
             keep=32, recent=1, dtype="fp16"),
        # four drafts of one sequence, drawn from the draft's own probabilities
        dict(name="verify 1 x 4", op="verify", batch=1, drafts=4, vocab=152064, dtype="fp32", point=False, temperature=0.7, top_k=0, top_p=1.0,
             min_p=0.0),
        # a batch of sequences with up to eight of them
        dict(name="verify 48 x 8", op="verify", batch=48, drafts=8, vocab=152064, dtype="bf16", point=False, temperature=1.0, top_k=0,
             top_p=1.0, min_p=0.0),
        # settings of a chat, each sequence its own around these
        dict(name="verify 16 x 4, filtered", op="verify", batch=16, drafts=4, vocab=152064, dtype="bf16", point=False, temperature=0.7, top_k=50,
             top_p=0.9, min_p=0.0),
        # drafts that are the draft model's best tokens, not drawn ones
        dict(name="verify 16 x 8, best drafts", op="verify", batch=16, drafts=8, vocab=32000, dtype="fp16", point=True, temperature=1.0,
             top_k=0, top_p=0.95, min_p=0.02),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm, odd ones among them."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["bounds", "select", "select", "attend", "attend", "verify", "verify"])
    if op == "bounds":
        stride = rng.choice([0, 1])
        page_len = rng.choice([1, 4, 16] if stride else [1, 4, 16, 64, 256])
        return dict(op=op, tokens=_spread(rng, 2 * page_len, 8191), first=rng.randrange(page_len), stride=stride,      # (one full page at least)
                    kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128]), page_len=page_len, dtype=rng.choice(["bf16", "fp16"]))
    if op == "verify":
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        batch, drafts = _spread(rng, 1, 24 if dtype == "fp32" else 48), rng.choice([0, 1, 3, 4, 7, 8])
        return dict(op=op, batch=batch, drafts=drafts, vocab=_spread(rng, 1000, 152064), dtype=dtype,
                    point=rng.choice([False, False, True]), temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
                    top_k=rng.choice([0, 0, 1, 20, 1000]), top_p=rng.choice([1.0, 1.0, 0.95, 0.5]), min_p=rng.choice([0.0, 0.0, 0.05]))
    q_heads, kv_heads, head_dim = rng.choice([(28, 4, 128), (32, 8, 128), (16, 8, 128), (64, 8, 128), (8, 1, 128), (32, 32, 128),
                                              (14, 2, 64), (32, 8, 64)])
    page_len = rng.choice([4, 16, 16, 64, 256])
    batch, new = _spread(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 9])
    keep = max(2, min(128, _spread(rng, 128, 2048) // page_len))
    batch = max(1, min(batch, 1024 // (new * kv_heads), (1 << 18) // (keep * page_len * kv_heads) if op == "attend" else 64))
    least = (2 * keep + 3) * page_len                    # even the shortest sequence has more blocks than are kept
    most = min(32768, (1 << 20) // (batch * kv_heads) * (4 if page_len >= 16 and op == "select" else 1))
    return dict(op=op, batch=batch, new=new, kv=_spread(rng, least, max(least + 1, most)), q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                page_len=page_len, keep=keep, recent=rng.choice([1, 2]) if keep > 2 else 1, dtype=rng.choice(["bf16", "fp16"]))


def _lengths(case):
    """Rows of every sequence with its new ones, and how many are new: the first one as long as the case says."""
    rng = random.Random("%s %s %s" % (case["batch"], case["new"], case["kv"]))
    both = []
    for b in range(case["batch"]):
        n = case["new"] if b == 0 else rng.randint(max(1, case["new"] - 2), case["new"])
        both.append((case["kv"] if b == 0 else max(n, rng.randint(max(1, case["kv"] // 2), case["kv"])), n))
    random.Random(7).shuffle(both)
    return [t for t, _ in both], [n for _, n in both]


def _rows(case):
    """Rows of logits of every sequence: one for its last token and one for each draft."""
    rng = random.Random("%s %s" % (case["batch"], case["drafts"]))
    return [1 + (case["drafts"] if b == 0 else rng.randint(case["drafts"] // 2, case["drafts"])) for b in range(case["batch"])]


def _slots(case):
    """Rows of the pool that the call's tokens have: one a page where ``stride`` says so (sequences that decode), else one after the other."""
    P = case["page_len"]
    if case["stride"]:
        return [t * P + (case["first"] + 5 * t) % P for t in range(case["tokens"])]
    return [case["first"] + t for t in range(case["tokens"])]


# ------------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=_DEVICE, dtype=torch.float32)


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    if case["op"] == "bounds":
        H, D, P = case["kv_heads"], case["head_dim"], case["page_len"]
        slots = torch.tensor(_slots(case), device=_DEVICE)
        pages = int(max(_slots(case))) // P + 3
        order = torch.randperm(pages, generator=g, device=_DEVICE)
        return dict(case, slots=order[slots // P] * P + slots % P, pool=_randn(g, pages, 2, P, H, D).to(dtype),
                    bounds=torch.zeros(pages, H, 2, D, dtype=dtype, device=_DEVICE))
    if case["op"] == "verify":
        rows, V = _rows(case), case["vocab"]
        T, B = sum(rows), len(rows)
        starts = torch.tensor([sum(rows[:b]) for b in range(B + 1)], dtype=torch.int32, device=_DEVICE)
        seq = torch.repeat_interleave(torch.arange(B, device=_DEVICE), torch.tensor(rows, device=_DEVICE))
        # the logits of a language model: a wide body and a few tokens far ahead of it; the draft sees them through some noise
        logits = 2.0 * _randn(g, T, V)
        logits.scatter_add_(1, torch.randint(0, V, (T, 40), generator=g, device=_DEVICE), 6.0 + 2.0 * _randn(g, T, 40))
        draft = logits + 0.5 * _randn(g, T, V)
        t = float(case["temperature"])
        per = torch.arange(B, device=_DEVICE) % 4                                # every fourth sequence is hotter, or sees more
        temperature = (torch.full((B,), t, device=_DEVICE) * torch.where(per == 1, 1.3, 1.0))[seq]
        top_k = (torch.full((B,), case["top_k"], dtype=torch.int32, device=_DEVICE) * torch.where(per == 2, 2, 1).to(torch.int32))[seq]
        top_p = torch.where(per == 3, torch.ones((), device=_DEVICE), torch.full((B,), float(case["top_p"]), device=_DEVICE))[seq]
        probs = torch.softmax(draft / (t if t > 0 else 0.5), -1)
        noise = -torch.log(torch.rand(T, V, generator=g, device=_DEVICE).clamp_(min=1e-30))
        drawn = (draft if case["point"] else probs / noise.clamp_(min=1e-30)).argmax(-1)
        del noise, draft
        tokens = torch.cat([drawn[-1:], drawn[:-1]])                              # the token behind row i is drawn from row i of the draft
        state = dict(case, logits=logits.to(dtype), tokens=tokens, starts=starts, uniforms=torch.rand(T, generator=g, device=_DEVICE),
                     draws=torch.rand(B, generator=g, device=_DEVICE), draft_probs=None if case["point"] else probs.to(dtype))
        if case["top_k"] or case["top_p"] < 1 or case["min_p"] > 0:
            # settings of every sequence, as a server keeps them
            state.update(temperature=temperature.contiguous(), top_k=top_k.contiguous(), top_p=top_p.contiguous(),
                         min_p=torch.full((T,), float(case["min_p"]), device=_DEVICE))
        return state
    total, fresh = _lengths(case)
    Hq, Hkv, D, P, keep = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_len"], case["keep"]
    counts = [(t + P - 1) // P for t in total]
    width, n_pages = max(counts), sum(counts) + 3
    order = torch.randperm(n_pages, generator=g, device=_DEVICE).to(torch.int32)
    cell = torch.arange(width, device=_DEVICE)[None, :]
    first = torch.tensor([sum(counts[:b]) for b in range(len(counts))], device=_DEVICE)[:, None]
    table = torch.where(cell < torch.tensor(counts, device=_DEVICE)[:, None], order[(first + cell).clamp(max=n_pages - 1)],
                        torch.full_like(order[:1], -1)).contiguous()
    T = sum(fresh)
    seq = [b for b, n in enumerate(fresh) for _ in range(n)]
    pos = [t - n + i for t, n in zip(total, fresh) for i in range(n)]
    qkv = _randn(g, T, Hq + 2 * Hkv, D).to(dtype)                              # queries are a slice of the fused projection
    state = dict(case, q=qkv[:, :Hq], table=table, sequences=torch.tensor(seq, dtype=torch.int32, device=_DEVICE),
                 positions=torch.tensor(pos, dtype=torch.int32, device=_DEVICE))
    if case["op"] == "select":
        centre = 0.7 * _randn(g, n_pages, Hkv, 1, D)                           # keys of a block resemble each other
        width = 1.4 + 0.3 * _randn(g, n_pages, Hkv, 1, D).abs()
        return dict(state, bounds=torch.cat([centre - width, centre + width], 2).to(dtype))
    pool = _randn(g, n_pages, 2, P, Hkv, D).to(dtype)
    # rows of a last page that no token has been written to hold whatever was there before
    kv_lens = torch.tensor(total, device=_DEVICE)
    row = torch.arange(P, device=_DEVICE)[None, :] + ((kv_lens + P - 1) // P - 1)[:, None] * P
    last = table.long().gather(1, ((kv_lens + P - 1) // P - 1)[:, None])[:, 0]
    stale = (row >= kv_lens[:, None])[:, None, :, None, None]
    pool[last] = torch.where(stale, torch.full_like(pool[:1, :1, :1, :1, :1], float("nan")), pool[last])
    # tokens of a sequence want much the same blocks
    own_block = (state["positions"] // P).long()[:, None, None]
    j = torch.arange(table.shape[1], device=_DEVICE)
    want = _randn(g, len(total), Hkv, table.shape[1])[state["sequences"].long()] + 0.3 * _randn(g, T, Hkv, table.shape[1])
    want = torch.where(j > own_block, -math.inf, torch.where(j > own_block - case["recent"], math.inf, want))
    top = want.topk(min(keep, table.shape[1]), -1)
    blocks = torch.where(top.values > -math.inf, top.indices, 1 << 30).sort(-1).values
    blocks = torch.where(blocks == 1 << 30, -1, blocks)
    blocks = torch.nn.functional.pad(blocks, (0, keep - blocks.shape[-1]), value=-1).to(torch.int32).contiguous()
    return dict(state, pool=pool, blocks=blocks, scale=2.0 / math.sqrt(D))


# ------------------------------------------------------------------------------------------------ plain forms
def _bounds(s):
    P = s["page_len"]
    full = s["slots"][s["slots"] % P == P - 1] // P
    keys = s["pool"][full, 0].float()
    s["bounds"][full] = torch.stack([keys.amin(1), keys.amax(1)], 2).to(s["bounds"].dtype)
    return s["bounds"]


def _select(s):
    """In 64 bits: which blocks stay is decided by the order of their scores."""
    P, keep, recent = s["page_len"], s["keep"], s["recent"]
    seq, c = s["sequences"].long(), (s["positions"] // P).long()
    T, Hq, D = s["q"].shape
    Hkv = s["kv_heads"]
    q = s["q"].double().view(T, Hkv, Hq // Hkv, D)
    weight = torch.cat([q.clamp(max=0).sum(2), q.clamp(min=0).sum(2)], -1)             # [T, Hkv, 2 D]: of low, of high
    N = s["table"].shape[1]
    pages = s["table"][seq].long().clamp(min=0)                                        # [T, N]
    score = torch.cat([(s["bounds"][pages[:, a:a + 256]].flatten(3).double() * weight[:, None]).sum(-1) for a in range(0, N, 256)], 1)
    score = score.transpose(1, 2)                                                       # [T, Hkv, N]
    j = torch.arange(N, device=score.device)
    c = c[:, None, None]
    score = torch.where(score.isnan(), math.inf, score)
    rank = torch.where(j > c - recent, torch.where(j > c, 2, 0), 1)                     # the last ones first, those behind the token never
    order = score.masked_fill(rank != 1, 0.0).sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, rank.expand_as(score).gather(-1, order).sort(dim=-1, stable=True).indices)[..., :keep]
    order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=N)
    order = torch.where(order > c, N, order).sort(-1).values
    return torch.where(order == N, -1, order).to(torch.int32)


def _attend(s):
    P = s["page_len"]
    T, Hq, D = s["q"].shape
    Hkv = s["kv_heads"]
    blocks, seq = s["blocks"].long(), s["sequences"].long()
    pages = s["table"].long()[seq[:, None, None], blocks.clamp(min=0)].clamp(min=0)    # [T, Hkv, keep]
    h = torch.arange(Hkv, device=pages.device)[None, :, None]
    row = (blocks[..., None] * P + torch.arange(P, device=pages.device)).flatten(2)
    seen = (blocks >= 0).repeat_interleave(P, -1) & (row <= s["positions"][:, None, None])
    k = s["pool"][pages, 0, :, h].flatten(2, 3).float().masked_fill(~seen[..., None], 0.0)      # [T, Hkv, keep P, D]
    v = s["pool"][pages, 1, :, h].flatten(2, 3).float().masked_fill(~seen[..., None], 0.0)
    S, G = k.shape[2], Hq // Hkv
    q = s["q"].float().reshape(T * Hkv, G, D)
    score = torch.matmul(q, k.view(T * Hkv, S, D).transpose(1, 2).contiguous()).view(T, Hkv, G, S).mul_(s["scale"])
    score = score.masked_fill_(~seen[:, :, None], float("-inf"))
    weight = score.sub_(score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp_()
    out = torch.matmul(weight.view(T * Hkv, G, S), v.view(T * Hkv, S, D)).view(T, Hkv, G, D)
    mass = weight.sum(-1, keepdim=True)
    return (out / mass.masked_fill(mass == 0, 1.0)).reshape(T, Hq * D).to(s["q"].dtype)


def _per_row(s, name, like):
    v = s[name]
    return v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full_like(like, float(v))


def _target_probs(s):
    """Every row's probabilities after the filters, in 64 bits: prefixes of the order of its logits."""
    x = s["logits"].double()
    x, order = x.masked_fill(x.isnan(), float("-inf")).sort(dim=-1, descending=True, stable=True)
    V, top = x.shape[-1], x[:, :1]
    t, p, m, k = (_per_row(s, name, top) for name in ("temperature", "top_p", "min_p", "top_k"))
    e = ((x - top) / t.masked_fill(t == 0, 1.0)).exp().masked_fill(x == top, 1.0).masked_fill(x == float("-inf"), 0.0)
    rank = torch.arange(V, device=x.device)[None, :]
    k = torch.where(t == 0, torch.ones_like(k), torch.where(k <= 0, torch.full_like(k, V), k))
    e = e.masked_fill(rank >= k, 0.0)
    before = e.cumsum(-1) - e
    e = e.masked_fill(~((before < p * e.sum(-1, keepdim=True)) | (p >= 1.0) | (rank == 0)), 0.0).masked_fill(e < m, 0.0)
    return torch.zeros_like(e).scatter_(1, order, e / e.sum(-1, keepdim=True))


def _verify(s):
    p = _target_probs(s)
    T, V = p.shape
    starts = s["starts"].long()
    B = starts.numel() - 1
    row = torch.arange(T, device=p.device)
    seq = torch.searchsorted(starts[1:], row, right=True)
    last = row == starts[seq + 1] - 1
    x = torch.cat([s["tokens"][1:], s["tokens"][:1]])[:, None]                          # the draft behind every row
    px = p.gather(1, x)[:, 0]
    qx = torch.ones_like(px) if s["draft_probs"] is None else s["draft_probs"].gather(1, x)[:, 0].double()
    stops = last | ~(s["uniforms"].double() * qx < px)
    at = torch.full((B,), T, device=p.device).scatter_reduce_(0, seq[stops], row[stops], "amin")      # the row that the sequence ends with
    pr = p[at]
    q = torch.zeros_like(pr).scatter_(1, x[at], 1.0) if s["draft_probs"] is None else s["draft_probs"][at].double()
    rest = (pr - q).clamp(min=0.0)
    rest = torch.where(last[at][:, None] | (rest.sum(-1, keepdim=True) == 0), pr, rest)
    mass = rest.cumsum(-1)
    token = torch.searchsorted(mass, s["draws"].double()[:, None] * mass[:, -1:], right=True).clamp(max=V - 1)
    tokens = torch.where(row < at[seq], x[:, 0], torch.where(row == at[seq], token[seq, 0], -1))
    probs = torch.where(row < at[seq], px, torch.where(row == at[seq], pr.gather(1, token)[seq, 0], 0.0))
    return dict(tokens=tokens, probs=probs.float(), accepted=(at - starts[:-1]).int())


def run(state):
    s = state
    if own:
        from subspec_amd import ops
        if s["op"] == "bounds":
            return ops.kv_page_bounds_(s["bounds"], s["pool"], s["slots"])
        if s["op"] == "select":
            return ops.select_blocks(s["q"], s["bounds"], s["table"], s["sequences"], s["positions"], s["page_len"], s["keep"], recent=s["recent"])
        if s["op"] == "attend":
            return ops.block_attention(s["q"], s["pool"], s["table"], s["blocks"], s["sequences"], s["positions"], scale=s["scale"])
        return ops.verify_drafts(s["logits"], s["tokens"], s["starts"], s["uniforms"], s["draws"], s["draft_probs"],
                                 temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"bounds": _bounds, "select": _select, "attend": _attend, "verify": _verify}[s["op"]](s)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "bounds":
        P, row = case["page_len"], case["kv_heads"] * case["head_dim"] * 2
        full = sum(s % P == P - 1 for s in _slots(case))
        return {"bytes": full * (P + 2) * row + 8 * case["tokens"], "flops": 0}
    if case["op"] == "verify":
        # every row of the logits, and the draft's row that the sequence ends with
        rows = sum(_rows(case))
        return {"bytes": (rows + (0 if case["point"] else case["batch"])) * case["vocab"] * size + 32 * rows, "flops": 0}
    total, fresh = _lengths(case)
    P, D, Hq, Hkv, keep = case["page_len"], case["head_dim"], case["q_heads"], case["kv_heads"], case["keep"]
    T = sum(fresh)
    if case["op"] == "select":
        scored = [[max(0, (t - n + i) // P + 1 - case["recent"]) for i in range(n)] for t, n in zip(total, fresh)]
        return {"bytes": sum(max(c) for c in scored) * Hkv * 4 * D + T * Hq * D * 2 + T * Hkv * keep * 4,
                "flops": 4.0 * D * Hkv * sum(sum(c) for c in scored)}
    # the rows that one token of every sequence sees (its fellows' are much the same), the products of all
    rows = [[min(t - n + i + 1, (keep - 1) * P + (t - n + i) % P + 1) for i in range(n)] for t, n in zip(total, fresh)]
    return {"bytes": sum(max(r) for r in rows) * Hkv * D * 4 + T * Hq * D * 4 + T * Hkv * keep * 4,
            "flops": 4.0 * D * Hq * sum(sum(r) for r in rows)}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    if case["op"] == "select":
        return None                                     # whole numbers
    s = prepare(case, seed)
    if case["op"] == "bounds":
        P, out = case["page_len"], s["bounds"].double()
        for slot in s["slots"].tolist():
            if slot % P == P - 1:
                keys = s["pool"][slot // P, 0].double()
                out[slot // P, :, 0], out[slot // P, :, 1] = keys.min(0).values, keys.max(0).values
        return out
    if case["op"] == "attend":
        P, Hq, Hkv, D = case["page_len"], case["q_heads"], case["kv_heads"], case["head_dim"]
        table, pos, seq, blocks = s["table"].tolist(), s["positions"].tolist(), s["sequences"].tolist(), s["blocks"].tolist()
        out = []
        for t in range(len(pos)):
            heads = []
            for h in range(Hkv):
                rows = [(table[seq[t]][b], r) for b in blocks[t][h] if b >= 0 for r in range(P) if b * P + r <= pos[t]]
                at = torch.tensor(rows, device=s["pool"].device)
                k, v = (s["pool"][at[:, 0], i, at[:, 1], h].double() for i in (0, 1))
                q = s["q"][t, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)].double()
                a = torch.softmax((k @ q.t().contiguous()).t().contiguous() * s["scale"], -1)
                heads.append(a @ v)
            out.append(torch.cat(heads).reshape(Hq * D))
        return torch.stack(out)
    rows, V = _rows(case), case["vocab"]
    tokens, probs, accepted = [], [], []
    at = 0

    def of(name, r):
        return float(s[name][r]) if isinstance(s[name], torch.Tensor) else float(s[name])

    for b, n in enumerate(rows):
        drafts = s["tokens"][at + 1:at + n].tolist()
        for i in range(n):
            l = s["logits"][at + i].double().cpu().numpy()
            t, k = of("temperature", at + i), int(of("top_k", at + i))
            e = np.exp((l - l.max()) / t) if t > 0 else (np.arange(V) == l.argmax()).astype(np.float64)
            if k > 0 or of("top_p", at + i) < 1:
                order = np.argsort(-l, kind="stable")                      # equal ones by index
                kept = order[:k] if k > 0 else order
                goal, before = of("top_p", at + i) * math.fsum(e[kept]), np.cumsum(e[kept]) - e[kept]
                if of("top_p", at + i) < 1:
                    kept = kept[:max(1, int((before < goal).sum()))]
                mask = np.zeros(V, bool)
                mask[kept] = True
                e = np.where(mask, e, 0.0)
            e = np.where(e >= of("min_p", at + i), e, 0.0)
            p = e / math.fsum(e)
            q = None
            if i < n - 1:
                x = drafts[i]
                q = np.zeros(V) if case["point"] else s["draft_probs"][at + i].double().cpu().numpy()
                if case["point"]:
                    q[x] = 1.0
                if float(s["uniforms"][at + i]) * q[x] < p[x]:
                    tokens.append(x)
                    probs.append(float(p[x]))
                    continue
            rest = p if q is None else np.maximum(p - q, 0.0)
            rest = rest if rest.sum() > 0 else p
            sums = np.cumsum(rest)
            x = min(int((sums <= float(s["draws"][b]) * sums[-1]).sum()), V - 1)
            tokens += [x] + [-1] * (n - 1 - i)
            probs += [float(p[x])] + [0.0] * (n - 1 - i)
            accepted.append(i)
            break
        at += n
    return dict(tokens=torch.tensor(tokens), probs=torch.tensor(probs, dtype=torch.float64), accepted=torch.tensor(accepted, dtype=torch.int32))
