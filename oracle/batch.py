"""Oracle: one step of a batch of sequences over a page pool, and filtered sampling.  Test infrastructure only.

Plain loops and float64, from the definitions: the page bookkeeping of
specdecodes/models/utils/flashinfer/cache_manager.py:218-240,350-372 for many sequences at once, causal attention with a
window and first tokens, and the warpers of specdecodes/models/generators/base.py:42-64 as prefixes of the sorted logits."""
import math

import torch


def plan(kv_lens, new_lens, free_pages, block_table, page_len, n_tokens):
    """``free_pages``: the free ones, the last of them is taken first.  Lists in, dictionary of lists out (``table`` is a copy)."""
    table, stack = [list(r) for r in block_table], list(free_pages)
    starts, positions, slots, sequences = [0], [], [], []
    for b, (held, new) in enumerate(zip(kv_lens, new_lens)):
        for block in range(-(-held // page_len), -(-(held + new) // page_len)):
            table[b][block] = stack.pop()
        for p in range(held, held + new):
            page = table[b][p // page_len]
            positions.append(p)
            slots.append(-1 if page < 0 else page * page_len + p % page_len)
            sequences.append(b)
        starts.append(len(positions))
    taken, pad = len(free_pages) - len(stack), n_tokens - len(positions)
    return dict(table=table, query_starts=starts, kv_lens=[a + b for a, b in zip(kv_lens, new_lens)],
                positions=positions + [0] * pad, slots=slots + [-1] * pad, sequences=sequences + [-1] * pad,
                counts=[starts[-1], taken, len(stack), 0])


def attention(q, pool_layer, block_table, query_starts, kv_lens, window=0, sinks=0, scale=None, max_kv=None):
    """(out, weight) float64 [tokens, Hq, D]: ``weight`` is the same average over |v|, what the rounding of a probability acts on; and the
    largest sum of |q_d k_d| times the scale, what the rounding of a score acts on.  ``max_kv``: rows from it on are not seen."""
    T, Hq, D = q.shape
    P, Hkv = pool_layer.shape[2], pool_layer.shape[3]
    scale = D ** -0.5 if scale is None else scale
    out, weight = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    worst = 0.0
    for b, total in enumerate(kv_lens):
        first, n = query_starts[b], query_starts[b + 1] - query_starts[b]
        if total <= 0 or n == 0:
            continue
        kv = torch.stack([pool_layer[block_table[b][j // P], :, j % P] for j in range(total)]).double()
        p, j = torch.arange(total - n, total)[:, None], torch.arange(total)[None, :]
        seen = j <= p
        if window:
            seen &= (j > p - window) | (j < sinks)
        if max_kv is not None:
            seen &= j < max_kv
        some = seen.any(1)
        if not some.any():
            continue
        for h in range(Hq):
            k, v, rows = kv[:, 0, h // (Hq // Hkv)], kv[:, 1, h // (Hq // Hkv)], q[first:first + n, h].double()[some]
            a = torch.softmax((rows @ k.t() * scale).masked_fill(~seen[some], -math.inf), 1)
            size = (rows.abs() @ k.abs().t()).masked_fill(~seen[some], 0.0)
            worst = max(worst, float(size.max()) * scale)
            out[first:first + n, h][some], weight[first:first + n, h][some] = a @ v, a @ v.abs()
    return out, weight, worst


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row of logits."""
    rows = [(l, i) for i, l in enumerate(logits.double().tolist()) if l == l and l > -math.inf]
    rows.sort(key=lambda e: (-e[0], e[1]))
    if not rows:
        return -1, 0.0
    top = rows[0][0]
    mass = [1.0 if l == top else math.exp((l - top) / temperature) if temperature > 0 and top < math.inf else 0.0 for l, _ in rows]
    n = 1 if temperature == 0 else min(top_k, len(rows)) if top_k > 0 else len(rows)
    mass = mass[:n]
    if top_p < 1:
        goal, before, kept = top_p * math.fsum(mass), 0.0, 0
        while kept < n and (kept == 0 or before < goal):
            before += mass[kept]
            kept += 1
        mass = mass[:kept]
    mass = [m for j, m in enumerate(mass) if j == 0 or m >= min_p]
    z, run = math.fsum(mass), 0.0
    last = max(j for j, m in enumerate(mass) if m > 0)
    for j, m in enumerate(mass):
        run += m
        if run > u * z or j == last:
            return rows[j][1], m / z
