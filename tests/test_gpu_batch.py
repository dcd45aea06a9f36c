"""GPU: one step of a batch of sequences over a page pool -- page tables and slot maps, the append, attention of the new
tokens -- against plain loops and float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import batch as ob
from subspec_amd import _lib as L
from subspec_amd import ops

DEV = "cuda:0"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ plan
def _plan_case(g, kv, new, page_len, spare_pages, width_spare=2):
    """(block table, free pages): sequences' pages in random order, the rest free."""
    have = [-(-a // page_len) for a in kv]
    need = sum(-(-(a + b) // page_len) - h for a, b, h in zip(kv, new, have))
    order = torch.randperm(sum(have) + need + spare_pages, generator=g).tolist()
    width = max(-(-(a + b) // page_len) for a, b in zip(kv, new)) + width_spare
    table, at = [], 0
    for h in have:
        table.append(order[at:at + h] + [-7] * (width - h))
        at += h
    return table, order[at:]


@pytest.mark.parametrize("kv,new,page_len,pad", [
    ([0], [1], 16, 0), ([5], [0], 4, 3), ([0, 0, 0], [0, 0, 0], 16, 2), ([15, 16, 17, 0], [1, 1, 1, 1], 16, 0),
    ([3, 0, 100, 7], [40, 0, 1, 9], 8, 5), ([1, 2, 3], [1, 2, 3], 1, 0), ([255, 256, 0], [1, 300, 2000], 256, 1),
    (list(range(0, 130)), [(7 * i) % 5 for i in range(130)], 4, 17), ([9] * 1500, [i % 3 for i in range(1500)], 8, 1),
    ([100] * 4096, [1] * 4096, 32, 0)])
def test_plan(kv, new, page_len, pad):
    print("plan", len(kv), page_len, flush=True)
    g = torch.Generator().manual_seed(len(kv) + page_len)
    table, free = _plan_case(g, kv, new, page_len, 3)
    n = sum(new) + pad
    want = ob.plan(kv, new, free, table, page_len, n)
    wide = _i32([r + [-9] * 2 for r in table])                            # the table is a view with a longer row stride
    view = wide[:, :len(table[0])]
    free_t = _i32(free + [-11] * 4)                                       # behind the free pages anything may lie
    got = ops.paged_batch_plan(_i32(kv), _i32(new), free_t, _i32([len(free)]), view, page_len, n)
    assert view.tolist() == want.pop("table") and wide[:, -2:].eq(-9).all()
    for key, value in want.items():
        assert got[key].tolist() == value, key
    assert free_t.tolist() == free + [-11] * 4


@pytest.mark.parametrize("kv,new,change,status", [
    ([4, -1], [1, 1], {}, L.PLAN_NEGATIVE), ([4, 4], [1, -2], {}, L.PLAN_NEGATIVE), ([4, 4], [1, 100], {}, L.PLAN_TABLE),
    ([4, 4], [5, 5], {"n_free": 1}, L.PLAN_PAGES), ([4, 4], [1, 1], {"n_free": 9}, L.PLAN_PAGES), ([4, 4], [5, 5], {"n": 9}, L.PLAN_TOKENS),
    ([4, 4], [2147483647, 2147483647], {}, L.PLAN_TABLE | L.PLAN_PAGES | L.PLAN_TOKENS)])
def test_a_plan_that_does_not_fit_takes_nothing(kv, new, change, status):
    print("plan refused", kv, new, change, flush=True)
    table = _i32([[0, 1, -1, -1], [2, 3, -1, -1]])
    before = table.clone()
    n = change.get("n", 16)
    got = ops.paged_batch_plan(_i32(kv), _i32(new), _i32([4, 5, 6, 7, 8]), _i32([change.get("n_free", 5)]), table, 4, n)
    # (a length that overflows the table may also exceed the tokens or pages: only the bits asked for are certain)
    assert got["counts"][3].item() & status == status and got["counts"][:2].tolist() == [0, 0]
    assert torch.equal(table, before) and got["kv_lens"].tolist() == kv and got["query_starts"].tolist() == [0, 0, 0]
    assert got["slots"].tolist() == [-1] * n and got["sequences"].tolist() == [-1] * n and got["positions"].tolist() == [0] * n


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,D,page_len,layout", [
    (1, 1, 64, 16, "plain"), (61, 4, 128, 16, "fused"), (300, 8, 128, 64, "fused"), (7, 2, 80, 1, "plain"), (9, 3, 5, 4, "plain"),
    (33, 2, 64, 8, "heads first"), (5, 1, 1, 2, "plain"), (20, 2, 36, 4, "odd offset"), (6, 2, 64, 4, "every second element")])
def test_append(dtype, tokens, heads, D, page_len, layout):
    print("append", dtype, tokens, heads, D, page_len, layout, flush=True)
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page_len) + 3
    pool = torch.randn(pages, 2, page_len, heads, D, generator=g).to(dtype)
    kv = torch.randn(2, tokens, heads, D, generator=g).to(dtype)
    slots = torch.randperm(pages * page_len, generator=g)[:tokens]
    skipped = torch.arange(tokens) % 5 == 3
    slots[skipped] = torch.tensor([-1, pages * page_len, 1 << 40])[torch.arange(int(skipped.sum())) % 3]
    want = pool.clone()
    for t in range(tokens):
        if not skipped[t]:
            want[slots[t] // page_len, :, slots[t] % page_len] = kv[:, t]
    if layout == "fused":
        both = torch.cat([torch.zeros(tokens, heads, D, dtype=dtype), kv[0], kv[1]], 1).to(DEV)
        k, v = both[:, heads:2 * heads], both[:, 2 * heads:]
    elif layout == "heads first":
        k, v = (x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1) for x in kv)
    elif layout == "odd offset":                                          # rows that start in the middle of a 16-byte piece
        room = torch.zeros(2, tokens, heads * D + 2, dtype=dtype)
        room[:, :, 2:] = kv.reshape(2, tokens, -1)
        k, v = (x[:, 2:].view(tokens, heads, D) for x in room.to(DEV))
    elif layout == "every second element":
        k, v = (x.repeat_interleave(2, -1).to(DEV)[..., ::2] for x in kv)
    else:
        k, v = kv[0].to(DEV), kv[1].to(DEV)
    got = ops.kv_append_paged_(pool.to(DEV), k, v, slots.to(DEV))
    assert torch.equal(got.cpu(), want)


# ------------------------------------------------------------------------------------------------ attention
def _batch(g, lens, page_len, Hq, Hkv, D, dtype, spare=2):
    """Inputs on the host; pages in random order, NaN in every row that belongs to no sequence."""
    counts = [-(-max(0, t) // page_len) for t, _ in lens]
    order = torch.randperm(sum(counts) + spare, generator=g).tolist()
    width = max(counts + [1]) + 1
    table, at = [], 0
    for c in counts:
        table.append(order[at:at + c] + [-1] * (width - c))
        at += c
    pool = torch.full((len(order), 2, page_len, Hkv, D), float("nan"), dtype=dtype)
    for b, (t, _) in enumerate(lens):
        for j in range(t):
            pool[table[b][j // page_len], :, j % page_len] = torch.randn(2, Hkv, D, generator=g).to(dtype)
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    q = (torch.randn(starts[-1], Hq, D, generator=g) * 2).to(dtype)
    return q, pool, table, starts, [t for t, _ in lens]


def _tolerance(want, weight, worst, dtype, keys, top, D):
    """Per element.  The result is rounded once (half a step of its type); each probability is rounded once before it multiplies V
    (half a step of it, acting on the average of |v|; of fp16's smallest, 2^-24, where it is that small: half of that for each key,
    relative to a largest of 1); a score is a sum of D fp32 products in any order (2^-24 of the sum of their sizes for each addition),
    its exponential is good to 2^-21, and both act on numerator and denominator."""
    half = torch.finfo(dtype).eps / 2
    score = (D + 4) * 2.0 ** -24 * worst + 2.0 ** -21
    small = keys * 2.0 ** -25 * top if dtype == torch.float16 else 0.0
    return half * (want.abs() + weight) * (1 + 2 * half) + 2 * score * weight + small + 2.0 ** -24


SHAPES = [  # (rows with the new ones, new ones) of every sequence
    [(1, 1)], [(300, 1), (1, 1), (64, 1), (65, 1), (127, 1)], [(40, 0), (33, 1), (0, 0), (2, 2)], [(70, 70)], [(200, 37), (131, 131), (5, 3)],
    [(1000, 3), (17, 17), (513, 1)], [(2, 5), (90, 4)], [(700, 130)], [(2100, 1), (30, 1)]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D", [(7, 1, 128), (4, 2, 64), (3, 3, 128), (16, 1, 64), (40, 2, 128)])
@pytest.mark.parametrize("lens", SHAPES, ids=str)
@pytest.mark.parametrize("page_len,window,sinks", [(16, 0, 0), (1, 50, 0), (64, 33, 5), (8, 1, 1), (128, 64, 70)])
def test_attention(dtype, Hq, Hkv, D, lens, page_len, window, sinks):
    print("paged attention", dtype, Hq, Hkv, D, lens, page_len, window, sinks, flush=True)
    g = torch.Generator().manual_seed(sum(t for t, _ in lens) + Hq + D + page_len)
    q, pool, table, starts, kv = _batch(g, lens, page_len, Hq, Hkv, D, dtype)
    want, weight, worst = ob.attention(q, pool, table, starts, kv, window, sinks)
    got = ops.paged_attention(q.to(DEV), pool.to(DEV), _i32(table), _i32(starts), _i32(kv), max(n for _, n in lens), max(kv),
                              window=window, sinks=sinks)
    got = got.double().cpu().view(want.shape)
    tol = _tolerance(want, weight, worst, dtype, max(kv), float(pool.nan_to_num(0.0).abs().max()), D)
    off = (got - want).abs()
    assert torch.isfinite(got).all().item()
    assert (off / tol).max().item() <= 1.0
