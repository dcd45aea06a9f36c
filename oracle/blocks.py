"""Oracle: attention over selected blocks of long sequences, and verification of drafts by given numbers.  Test infrastructure only.

Plain loops and float64, from the definitions in include/subspec_hip.h (no form of either is in the reference)."""
import math

import torch



def page_bounds(bounds, pool_layer, slots):
    """A copy of ``bounds`` [pages, heads, 2, D] with those of every page whose last row is among the slots."""
    P, out = pool_layer.shape[2], bounds.clone()
    for s in slots:
        if 0 <= s < pool_layer.shape[0] * P and s % P == P - 1:
            keys = pool_layer[s // P, 0]
            out[s // P, :, 0], out[s // P, :, 1] = keys.amin(0), keys.amax(0)      # (a NaN stays one)
    return out


def select(q, bounds, block_table, sequences, positions, page_len, keep, recent=1, max_kv=None):
    """[tokens][kv heads][keep], -1 behind the last."""
    T, Hq, D = q.shape
    Hkv = bounds.shape[1]
    out = []
    for t in range(T):
        last = positions[t] if max_kv is None else min(positions[t], max_kv - 1)
        last = min(last, len(block_table[0]) * page_len - 1)
        seen = last // page_len + 1 if 0 <= sequences[t] < len(block_table) and last >= 0 else 0
        heads = []
        for h in range(Hkv):
            if seen <= keep:
                heads.append(list(range(seen)) + [-1] * (keep - seen))
                continue
            n = seen - recent
            rows = q[t, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)].double()
            low, high = bounds[torch.tensor(block_table[sequences[t]][:n]), h].double().unbind(1)          # [n, D]
            score = rows.clamp(max=0).sum(0) * low + rows.clamp(min=0).sum(0) * high
            score = score.sum(1)
            score = torch.where(score.isnan(), math.inf, score).tolist()
            best = sorted(range(n), key=lambda j: (-score[j], j))[:keep - recent]
            heads.append(sorted(best) + list(range(n, seen)))
        out.append(heads)
    return out


def attention(q, pool_layer, block_table, blocks, sequences, positions, scale=None):
    """(out, weight, worst) as ``oracle.batch.attention``; rows of tokens of no sequence are NaN."""
    T, Hq, D = q.shape
    P, Hkv = pool_layer.shape[2], pool_layer.shape[3]
    scale = D ** -0.5 if scale is None else scale
    out, weight, worst = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64), 0.0
    for t in range(T):
        if not 0 <= sequences[t] < len(block_table):
            out[t] = math.nan
            continue
        for h in range(Hkv):
            rows = [(block_table[sequences[t]][b], r) for b in blocks[t][h] if b >= 0 for r in range(P) if b * P + r <= positions[t]]
            if not rows:
                continue
            at = torch.tensor(rows)
            k, v = pool_layer[at[:, 0], 0, at[:, 1], h].double(), pool_layer[at[:, 0], 1, at[:, 1], h].double()
            mine = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            a = torch.softmax(q[t, mine].double() @ k.t() * scale, 1)
            worst = max(worst, float((q[t, mine].double().abs() @ k.abs().t()).max()) * scale)
            out[t, mine], weight[t, mine] = a @ v, a @ v.abs()
    return out, weight, worst


def target_probs(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Probabilities of one row after the filters (float64; zeros where nothing can be drawn).  The settings are fp32 numbers."""
    temperature, top_p, min_p = torch.tensor([temperature, top_p, min_p], dtype=torch.float32).tolist()
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    top = float(x.max())
    if top == -math.inf:
        return torch.zeros_like(x)
    if temperature == 0 or top == math.inf:
        mass = (x == top).double()
    else:
        mass = torch.exp((x - top) / temperature)
    order = torch.sort(-x, stable=True).indices
    kept = order[:1] if temperature == 0 else order[:top_k] if top_k > 0 else order
    if top_p < 1:
        m = mass[kept]
        before = m.cumsum(0) - m
        kept = kept[:max(1, int((before < top_p * math.fsum(m.tolist())).sum()))]
    p = torch.zeros_like(x)
    p[kept] = torch.where(mass[kept] >= min(min_p, 1.0), mass[kept], 0.0)
    return p / p.sum()


def verify_drafts(logits, tokens, query_starts, uniforms, draws, draft_probs=None, settings=None):
    """(tokens, probs, accepted) as lists; ``settings(row)``: keyword arguments of ``target_probs``."""
    T, V = logits.shape
    out, probs, accepted = [-1] * T, [0.0] * T, []
    for b in range(len(query_starts) - 1):
        first, n = query_starts[b], query_starts[b + 1] - query_starts[b]
        stays = 0
        for i in range(n):
            row = first + i
            p = target_probs(logits[row], **(settings(row) if settings else {}))
            rest = p
            if i < n - 1:
                x = int(tokens[row + 1])
                known = 0 <= x < V
                if draft_probs is None:
                    q = torch.zeros_like(p)
                    if known:
                        q[x] = 1.0
                else:
                    q = draft_probs[row].double()
                    q = torch.where(q > 0, q, 0.0)
                if known and float(p[x]) > 0 and float(uniforms[row]) * float(q[x]) < float(p[x]):
                    out[row], probs[row] = x, float(p[x])
                    stays += 1
                    continue
                rest = torch.clamp(p - q, min=0.0)
                if not float(rest.sum()) > 0:
                    rest = p
            total = rest.cumsum(0)
            if float(total[-1]) > 0:
                j = min(int((total <= float(draws[b]) * float(total[-1])).sum()), int(rest.nonzero().max()))
                out[row], probs[row] = j, float(p[j])
            break
        accepted.append(stays)
    return out, probs, accepted


