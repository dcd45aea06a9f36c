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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_bounds_need_not_be_tight_and_rows_behind_the_last_sequence_stay(dtype):
    g = torch.Generator().manual_seed(11)
    lens = [(77, 1), (40, 40), (3, 5), (0, 0)]                             # the third brings more rows than it has: its first two see none
    q, pool, table, starts, kv = _batch(g, lens, 16, 7, 1, 128, dtype)
    q = torch.cat([q, torch.full((9, 7, 128), float("nan"), dtype=dtype)])
    want, weight, worst = ob.attention(q, pool, table, starts, kv)
    out = torch.full((q.shape[0], 7 * 128), 5.0, dtype=dtype, device=DEV)
    got = ops.paged_attention(q.to(DEV), pool.to(DEV), _i32(table), _i32(starts), _i32(kv), 1000, 5 * 16 + 3000, out=out)
    assert got.data_ptr() == out.data_ptr() and out[-9:].eq(5.0).all()
    tol = _tolerance(want, weight, worst, dtype, max(kv), float(pool.nan_to_num(0.0).abs().max()), 128)[:-9]
    off = (got.double().cpu().view(want.shape) - want).abs()[:-9]
    assert (off / tol).max().item() <= 1.0 and got[starts[2]:starts[2] + 2].eq(0).all()
    # bounds below what is there leave rows out and stay inside every tensor
    cut = ops.paged_attention(q.to(DEV), pool.to(DEV), _i32(table), _i32(starts), _i32(kv), 2, 20, out=torch.full_like(out, 6.0))
    assert cut[starts[1] + 2:starts[2]].eq(6.0).all() and cut[-9:].eq(6.0).all()


def test_attention_reads_strided_queries_and_clamps_bad_tables():
    g = torch.Generator().manual_seed(12)
    lens = [(50, 1), (30, 12)]
    q, pool, table, starts, kv = _batch(g, lens, 8, 4, 2, 64, torch.float16)
    args = (pool.to(DEV), _i32(table), _i32(starts), _i32(kv), 12, 50)
    plain = ops.paged_attention(q.to(DEV), *args)
    fused = torch.zeros(q.shape[0], 8, 64, dtype=torch.float16)
    fused[:, 2:6] = q
    assert torch.equal(ops.paged_attention(fused.to(DEV)[:, 2:6], *args), plain)
    assert torch.equal(ops.paged_attention(q.transpose(0, 1).contiguous().to(DEV).transpose(0, 1), *args), plain)
    odd = torch.zeros(q.shape[0], 4 * 64 + 1, dtype=torch.float16)
    odd[:, 1:] = q.reshape(q.shape[0], -1)
    assert torch.equal(ops.paged_attention(odd.to(DEV)[:, 1:].view(-1, 4, 64), *args), plain)
    wide = torch.cat([_i32(table), _i32([[-5] * 3] * 2)], 1)[:, :len(table[0])]     # a view with a longer row stride
    assert torch.equal(ops.paged_attention(q.to(DEV), pool.to(DEV), wide, *args[2:]), plain)
    bad = _i32([[(1 << 30) if i % 2 else -9 for i in range(len(table[0]))]] * 2)    # numbers outside the pool: other rows, no fault
    assert ops.paged_attention(q.to(DEV), pool.nan_to_num(0.0).to(DEV), bad, *args[2:]).isfinite().all()


def test_argument_errors():
    pool = torch.zeros(6, 2, 16, 2, 128, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16, device=DEV)
    table, starts, lens = _i32([[0, 1]]), _i32([0, 3]), _i32([20])
    ops.paged_attention(q, pool, table, starts, lens, 3, 32)
    for bad in [dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[:, :, :64]), dict(table=table.long()), dict(table=table[0]), dict(starts=_i32([0])),
                dict(lens=lens.long()), dict(max_new=-1), dict(window=-3), dict(sinks=4), dict(out=q.view(3, -1).float()),
                dict(pool=pool[:, :1]), dict(workspace=torch.zeros(16, dtype=torch.uint8, device=DEV), max_kv=4096), dict(scale=0.0)]:
        a = dict(q=q, pool=pool, table=table, starts=starts, lens=lens, max_new=3, max_kv=32)
        a.update(bad)
        with pytest.raises((ValueError, L.SubspecHipError)):
            ops.paged_attention(a.pop("q"), a.pop("pool"), a.pop("table"), a.pop("starts"), a.pop("lens"), a.pop("max_new"), a.pop("max_kv"), **a)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(3, device=DEV)
    for bad in [(pool, k.float(), k, slots), (pool, k[:2], k, slots), (pool, k, k, slots.int()), (pool[0], k, k, slots)]:
        with pytest.raises(ValueError):
            ops.kv_append_paged_(*bad)
    one = _i32([1])
    for bad in [(lens.long(), one, one, one, table), (lens, _i32([1, 1]), one, one, table), (lens, one, one, _i32([1, 1]), table),
                (lens, one, one, one, table.t())]:
        with pytest.raises(ValueError):
            ops.paged_batch_plan(*bad, 16, 4)
    with pytest.raises(ValueError):
        ops.paged_batch_plan(lens, one, one, one, table, 12, 4)
    with pytest.raises(ValueError):
        ops.sample_filtered(torch.zeros(2, 8, device=DEV), torch.zeros(3, device=DEV))
    with pytest.raises(ValueError):
        ops.sample_filtered(torch.zeros(2, 8, device=DEV), torch.zeros(2, device=DEV), temperature=-1.0)
    with pytest.raises(ValueError):
        ops.sample_filtered(torch.zeros(2, 8, device=DEV), torch.zeros(2, device=DEV), top_k=torch.zeros(2, device=DEV))
    with pytest.raises(L.SubspecHipError):
        ops.kv_append_paged_(pool.cpu(), k.cpu(), k.cpu(), slots.cpu())


# ------------------------------------------------------------------------------------------------ a run of them together
def _dense(q, k, v, window, sinks):
    """float64 causal attention of the last q.shape[0] rows of one sequence."""
    n, total = q.shape[0], k.shape[0]
    pool, table = torch.stack([k, v], 1).unsqueeze(0).transpose(1, 2), [[0]]
    return ob.attention(q, pool, table, [0, n], [total], window, sinks)


@pytest.mark.parametrize("page_len,window,sinks", [(16, 0, 0), (4, 20, 3)])
def test_steps_of_a_batch(page_len, window, sinks):
    """Prompts in chunks, single tokens, a sequence that rests, one that ends and one that takes its place, over two layers: every
    step's attention against the sequence's own rows in float64, and the tokens drawn from its outputs."""
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    g = torch.Generator().manual_seed(20 + page_len)
    Hq, Hkv, D, dtype = 8, 2, 128, torch.bfloat16
    pool = KvCachePool(max_pages=600 // page_len + 8, num_layers=2, num_heads=Hkv, head_dim=D, page_len=page_len, dtype=dtype, device=DEV)
    pool.cache_data.fill_(float("nan"))
    pool.allocate(3)
    batch = KvBatch(pool, 3, 400)
    head = torch.randn(200, Hq * D, generator=g) * 0.1
    rows = [[[] for _ in range(3)] for _ in range(2)]
    for new, end in [([40, 0, 7], None), ([1, 90, 1], None), ([1, 1, 33], None), ([0, 1, 1], 1), ([1, 65, 1], None), ([1, 1, 1], None)]:
        plan = batch.step(new, n_tokens=sum(new) + 2)
        T = sum(new)
        for layer in range(2):
            qkv = torch.randn(T + 2, Hq + 2 * Hkv, D, generator=g).to(dtype)
            dev = qkv.to(DEV)
            batch.append(layer, dev[:, Hq:Hq + Hkv], dev[:, Hq + Hkv:])
            out = batch.attention(layer, dev[:, :Hq], window=window, sinks=sinks, out=torch.zeros(T + 2, Hq * D, dtype=dtype, device=DEV))
            first = 0
            for b, n in enumerate(new):
                rows[layer][b] += list(qkv[first:first + n, Hq:].view(n, 2, Hkv, D))
                if n:
                    kv = torch.stack(rows[layer][b])
                    want, weight, worst = _dense(qkv[first:first + n, :Hq], kv[:, 0], kv[:, 1], window, sinks)
                    got = out[first:first + n].double().cpu().view(want.shape)
                    tol = _tolerance(want, weight, worst, dtype, kv.shape[0], float(kv.abs().max()), D)
                    assert ((got - want).abs() / tol).max().item() <= 1.0, (new, b, layer)
                first += n
            assert out[T:].eq(0).all()
        last = plan["query_starts"][1:].long().clamp(min=1) - 1
        logits = (out[last].float() @ head.t().contiguous().to(DEV)).to(dtype)
        u = torch.rand(3, generator=g)
        tokens, _ = ops.sample_filtered(logits, u.to(DEV), 0.9, 50, 0.9, 0.01)
        f = lambda x: float(torch.tensor(x, dtype=torch.float32))
        assert tokens.tolist() == [ob.sample(logits[b].cpu(), float(u[b]), f(0.9), 50, f(0.9), f(0.01))[0] for b in range(3)]
        assert plan["counts"][3].item() == 0 and plan["counts"][2].item() == batch.num_free and batch.kv_lens.tolist() == batch.lens
        if end is not None:
            batch.release(end)
            for layer in range(2):
                rows[layer][end] = []
    with pytest.raises(ValueError):
        batch.step([400, 0, 0])
    batch.close()
    assert int(pool.num_free_pages()) == pool.max_pages - 3


def test_a_captured_step_replays_as_the_batch_grows():
    """Plan, append, attention (single tokens and a longer call) and sampling in one graph; between the replays other work runs, the
    lengths move on the device, and every replay equals the eager calls."""
    g = torch.Generator().manual_seed(31)
    B, Hq, Hkv, D, P, cap = 5, 8, 2, 128, 16, 64
    dtype = torch.bfloat16
    pool = torch.randn(B * cap // P * 4, 2, P, Hkv, D, generator=g).to(dtype).to(DEV)
    table = torch.full((B, cap * 4 // P), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(pool.shape[0], generator=g).to(torch.int32).to(DEV)
    state = dict(lens=_i32([0] * B), new=_i32([1] * B), n_free=_i32([pool.shape[0]]), qkv=torch.zeros(B + 12, Hq + 2 * Hkv, D, dtype=dtype, device=DEV),
                 u=torch.zeros(B, device=DEV))
    head = (torch.randn(Hq * D, 20000, generator=g) * 0.2).to(dtype).to(DEV)

    def step(s, pool, table, plan=None):
        plan = ops.paged_batch_plan(s["lens"], s["new"], free, s["n_free"], table, P, B + 12, out=plan)
        ops.kv_append_paged_(pool, s["qkv"][:, Hq:Hq + Hkv], s["qkv"][:, Hq + Hkv:], plan["slots"])
        args = (s["qkv"][:, :Hq], pool, table, plan["query_starts"], plan["kv_lens"])
        out = ops.paged_attention(*args, 12, cap * 4, out=torch.zeros(B + 12, Hq * D, dtype=dtype, device=DEV))
        near = ops.paged_attention(*args, 12, cap * 4, window=9, sinks=2, out=torch.zeros(B + 12, Hq * D, dtype=dtype, device=DEV))
        tokens, probs = ops.sample_filtered(out[:B] @ head, s["u"], 0.8, 40, 0.95, 0.01)
        return plan, out, near, tokens, probs

    step({k: v.clone() for k, v in state.items()}, pool.clone(), table.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(state, pool, table)
        state["lens"].copy_(captured[0]["kv_lens"])
        state["n_free"].copy_(captured[0]["counts"][2:3])
    state["lens"].zero_()
    state["n_free"].fill_(pool.shape[0])
    for i, new in enumerate([[3, 1, 2, 5, 1], [1] * 5, [0, 12, 1, 0, 1], [1] * 5, [1, 1, 13, 0, 2]]):
        state["new"].copy_(_i32(new))
        state["qkv"].copy_(torch.randn(state["qkv"].shape, generator=g).to(dtype))
        state["u"].copy_(torch.rand(B, generator=g))
        mine = {k: v.clone() for k, v in state.items()}
        want = step(mine, pool_copy := pool.clone(), table_copy := table.clone())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        if max(new) <= 12:                                    # (the bound that the step is captured for)
            for a, b in zip(want[1:], captured[1:]):
                assert torch.equal(a, b), i
        for key, value in want[0].items():
            assert torch.equal(value, captured[0][key]), (i, key)
        assert torch.equal(pool, pool_copy) and torch.equal(table, table_copy)
        (torch.randn(1000, 1000, device=DEV) @ torch.randn(1000, 1000, device=DEV)).sum().item()


def test_a_step_does_not_wait_for_the_device():
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    pool = KvCachePool(max_pages=8, num_layers=1, num_heads=2, head_dim=64, page_len=16, dtype=torch.bfloat16, device=DEV)
    batch = KvBatch(pool, 2, 64)
    k = torch.randn(5, 2, 64, device=DEV).to(torch.bfloat16)
    before = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        with pytest.raises(RuntimeError):
            torch.ones(1, device=DEV).item()                   # (what the mode reports)
        batch.step([3, 2])
        batch.append(0, k, k)
        batch.attention(0, k)
        batch.release(1)
        batch.step([1, 4])
    finally:
        torch.cuda.set_sync_debug_mode(before)
    assert batch.plan["counts"].tolist() == [5, 1, 6, 0] and batch.kv_lens.tolist() == [4, 4]


def test_a_plan_is_not_written_over_its_inputs():
    table, one = _i32([[0, -1]]), _i32([1])
    plan = ops.paged_batch_plan(_i32([3]), one, _i32([5, 6]), _i32([2]), table, 16, 4)
    for change in (dict(kv=plan["kv_lens"]), dict(n_free=plan["counts"][2:3]), dict(new=plan["positions"][1:2]), dict(free=plan["sequences"])):
        a = dict(kv=_i32([3]), new=one, free=_i32([5, 6]), n_free=_i32([2]))
        a.update(change)
        with pytest.raises(ValueError, match="overlaps"):
            ops.paged_batch_plan(a["kv"], a["new"], a["free"], a["n_free"], table, 16, 4, out=plan)
    ops.paged_batch_plan(_i32([4]), one, _i32([5, 6]), _i32([2]), table, 16, 4, out=plan)
    assert plan["kv_lens"].tolist() == [5] and plan["slots"].tolist() == [4, -1, -1, -1]


def test_calls_on_two_streams_at_once():
    g = torch.Generator().manual_seed(41)
    jobs = []
    for lens in ([(900, 1)] * 6, [(300, 120), (200, 1)]):
        q, pool, table, starts, kv = _batch(g, lens, 16, 8, 2, 128, torch.bfloat16)
        jobs.append((q.to(DEV), pool.to(DEV), _i32(table), _i32(starts), _i32(kv), max(n for _, n in lens), max(kv)))
    logits = torch.randn(6, 40000, generator=g).to(DEV)
    u = torch.rand(6, generator=g).to(DEV)
    alone = [ops.paged_attention(*j) for j in jobs] + [ops.sample_filtered(logits, u, 1.0, 0, 0.9)[0]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = [[], [], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                results[i].append(ops.paged_attention(*jobs[i]) if i < 2 else ops.sample_filtered(logits, u, 1.0, 0, 0.9)[0])
    torch.cuda.synchronize()
    for want, got in zip(alone, results):
        assert all(torch.equal(want, x) for x in got)


def test_long_offsets():
    """Pool offsets beyond 2^31 elements: the pages of a sequence lie at both ends of a pool of 2.4 billion elements."""
    P, Hkv, D = 256, 8, 128
    pages = 4600                                               # 2 * 256 * 8 * 128 elements a page
    pool = torch.empty(pages, 2, P, Hkv, D, dtype=torch.bfloat16, device=DEV)
    assert pool.numel() > (1 << 31)
    g = torch.Generator().manual_seed(51)
    own = [pages - 1, 0, pages - 2, 4100]
    k, v = (torch.randn(1000, Hkv, D, generator=g).to(torch.bfloat16) for _ in range(2))
    slots = torch.tensor([own[j // P] * P + j % P for j in range(1000)])
    ops.kv_append_paged_(pool, k.to(DEV), v.to(DEV), slots.to(DEV))
    for n in (1, 40):
        q = torch.randn(n, 16, D, generator=g).to(torch.bfloat16)
        want, weight, worst = ob.attention(q, torch.stack([k, v], 1).unsqueeze(0).transpose(1, 2), [[0]], [0, n], [1000])
        got = ops.paged_attention(q.to(DEV), pool, _i32([own]), _i32([0, n]), _i32([1000]), n, 1000).double().cpu().view(want.shape)
        tol = _tolerance(want, weight, worst, torch.bfloat16, 1000, float(v.abs().max()), D)
        assert ((got - want).abs() / tol).max().item() <= 1.0


def test_pages_of_one_row_over_a_long_sequence():
    """More page numbers than LDS has room for: a chunk's keys are taken in stretches."""
    g = torch.Generator().manual_seed(61)
    lens = [(9000, 70)]
    q, pool, table, starts, kv = _batch(g, lens, 1, 7, 1, 64, torch.float16)
    want, weight, worst = ob.attention(q, pool, table, starts, kv)
    got = ops.paged_attention(q.to(DEV), pool.to(DEV), _i32(table), _i32(starts), _i32(kv), 70, 9000).double().cpu().view(want.shape)
    tol = _tolerance(want, weight, worst, torch.float16, 9000, float(pool.nan_to_num(0.0).abs().max()), 64)
    assert ((got - want).abs() / tol).max().item() <= 1.0


def test_thousands_of_sequences_under_a_large_bound():
    """So many (sequence, KV head) pairs that the partial results of key chunks would not fit: every pair takes its keys in one piece."""
    g = torch.Generator().manual_seed(62)
    B, H, D, P, long = 4096, 32, 64, 16, 1500
    n_pages = B + long // P + 1
    pool = torch.randn(n_pages, 2, P, H, D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV, dtype=torch.bfloat16)
    table = torch.full((B, 70000 // P), -1, dtype=torch.int32)
    table[:, 0] = torch.arange(B)
    table[17, 1:long // P + 1] = torch.arange(B, B + long // P)
    lens = torch.ones(B, dtype=torch.int32)
    lens[17], lens[99] = long, 0
    q = torch.randn(B, H, D, generator=g).to(torch.bfloat16)
    got = ops.paged_attention(q.to(DEV), pool, table.to(DEV), torch.arange(B + 1, dtype=torch.int32, device=DEV), lens.to(DEV), 1, 70000).view(B, H, D)
    one = torch.ones(B, dtype=torch.bool)
    one[17] = one[99] = False
    assert torch.equal(got[one.to(DEV)], pool[:B, 1, 0][one.to(DEV)])          # one key: its value, weight 1
    assert got[99].eq(0).all()                                                 # no key
    rows = table[17, :long // P + 1].tolist()
    want, weight, worst = ob.attention(q[17:18], pool[rows].cpu(), [list(range(len(rows)))], [0, 1], [long])
    tol = _tolerance(want, weight, worst, torch.bfloat16, long, float(pool.abs().max()), D)
    assert ((got[17:18].double().cpu() - want).abs() / tol).max().item() <= 1.0


@pytest.mark.parametrize("lens", [[(900, 1), (300, 2)], [(700, 130), (64, 1)]], ids=str)
def test_a_window_beyond_any_sequence_is_none(lens):
    g = torch.Generator().manual_seed(63)
    q, pool, table, starts, kv = _batch(g, lens, 16, 8, 2, 128, torch.bfloat16)
    args = (q.to(DEV), pool.to(DEV), _i32(table), _i32(starts), _i32(kv), max(n for _, n in lens), max(kv))
    plain = ops.paged_attention(*args)
    for window, sinks in [((1 << 63) - 1, 0), ((1 << 63) - 1, (1 << 63) - 1), (7, (1 << 63) - 1), (1 << 31, 5)]:
        print("window", window, sinks, flush=True)
        assert torch.equal(ops.paged_attention(*args, window=window, sinks=sinks), plain)


CUT = [[(40, 40)], [(13, 13), (1, 1)], [(100, 13), (90, 90), (30, 1)], [(900, 60), (700, 3), (900, 1), (5, 9)], [(3, 50), (2000, 300)]]


@pytest.mark.parametrize("dtype,Hq,Hkv,D", [(torch.bfloat16, 7, 1, 128), (torch.float16, 4, 2, 64)])
@pytest.mark.parametrize("lens", CUT, ids=str)
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 0), (33, 5), (64, 70), (500, 3)])
def test_bounds_leave_tokens_and_rows_out_and_move_no_position(dtype, Hq, Hkv, D, lens, window, sinks):
    """max_new and max_kv below what a sequence brings: tokens from max_new on stay as they were, rows from max_kv on are not seen (and
    hold NaN here), and every other token sees what its position says, from either kernel and where its window begins behind max_kv."""
    g = torch.Generator().manual_seed(sum(t for t, _ in lens) + Hq + window)
    q, pool, table, starts, kv = _batch(g, lens, 16, Hq, Hkv, D, dtype)
    before = pool.clone()
    most_new, most_kv = max(n for _, n in lens), max(kv)
    for max_new, max_kv in [(most_new, 20), (1, most_kv), (2, 20), (12, most_kv), (12, 64), (most_new, max(1, most_kv - 70)), (50, 333), (most_new, 1)]:
        print("cut", dtype, Hq, lens, window, sinks, max_new, max_kv, flush=True)
        pool.copy_(before)
        for b, t in enumerate(kv):
            for j in range(max_kv, t):
                pool[table[b][j // 16], :, j % 16] = float("nan")
        want, weight, worst = ob.attention(q, before, table, starts, kv, window, sinks, max_kv=max_kv)
        out = torch.full((q.shape[0], Hq * D), 6.0, dtype=dtype, device=DEV)
        ops.paged_attention(q.to(DEV), pool.to(DEV), _i32(table), _i32(starts), _i32(kv), max_new, max_kv, window=window, sinks=sinks, out=out)
        got = out.double().cpu().view(want.shape)
        tol = _tolerance(want, weight, worst, dtype, max(kv), float(before.nan_to_num(0.0).abs().max()), D)
        for b, (_, n) in enumerate(lens):
            kept = slice(starts[b], starts[b] + min(n, max_new))
            assert torch.isfinite(got[kept]).all().item(), (b, max_new, max_kv)
            assert ((got[kept] - want[kept]).abs() / tol[kept]).max().item() <= 1.0, (b, max_new, max_kv)
            assert got[kept.stop:starts[b + 1]].eq(6.0).all(), (b, max_new, max_kv)


@pytest.mark.parametrize("lens", [[(700, 130), (64, 1)], [(500, 40), (300, 300), (41, 41)], [(90, 1), (33, 1)]], ids=str)
@pytest.mark.parametrize("before", [5, 37, 100, 1000])
def test_rows_before_the_first_sequence_stay(lens, before):
    """The last sequences of a batch alone, through views of its lengths, starts and table: the tokens of the others are not theirs."""
    print("rows before", lens, before, flush=True)
    g = torch.Generator().manual_seed(before + len(lens))
    Hq, Hkv, D, dtype = 14, 2, 128, torch.bfloat16
    q, pool, table, starts, kv = _batch(g, lens, 16, Hq, Hkv, D, dtype)
    want, weight, worst = ob.attention(q, pool, table, starts, kv)
    room = torch.randn(before, Hq, D, generator=g).to(dtype)
    starts_all = _i32([0, 0] + [s + before for s in starts])                     # two others before them
    out = torch.full((before + q.shape[0], Hq * D), 6.0, dtype=dtype, device=DEV)
    lens_all = _i32([50, 60] + kv)
    table_all = _i32([[0] * len(table[0])] * 2 + table)
    ops.paged_attention(torch.cat([room, q]).to(DEV), pool.to(DEV), table_all[2:], starts_all[2:], lens_all[2:], max(n for _, n in lens), max(kv), out=out)
    assert out[:before].eq(6.0).all()
    tol = _tolerance(want, weight, worst, dtype, max(kv), float(pool.nan_to_num(0.0).abs().max()), D)
    assert ((out[before:].double().cpu().view(want.shape) - want).abs() / tol).max().item() <= 1.0


def test_a_sequence_released_between_layers_is_computed_to_the_step_s_end():
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    g = torch.Generator().manual_seed(71)
    Hq, Hkv, D, dtype = 8, 2, 64, torch.float16
    pool = KvCachePool(max_pages=20, num_layers=2, num_heads=Hkv, head_dim=D, page_len=8, dtype=dtype, device=DEV)
    batch = KvBatch(pool, 3, 60)
    qkv = torch.randn(2, 50, Hq + 2 * Hkv, D, generator=g).to(dtype).to(DEV)
    rows = [0, 21, 22, 50]
    batch.step([21, 1, 28])
    outs = []
    for layer in range(2):
        batch.append(layer, qkv[layer, :, Hq:Hq + Hkv], qkv[layer, :, Hq + Hkv:])
        outs.append(batch.attention(layer, qkv[layer, :, :Hq]))
        if layer == 0:
            batch.release(0)
    for layer, out in enumerate(outs):
        for b in range(3):
            one = qkv[layer, rows[b]:rows[b + 1]].cpu()
            want, weight, worst = _dense(one[:, :Hq], one[:, Hq:Hq + Hkv], one[:, Hq + Hkv:], 0, 0)
            tol = _tolerance(want, weight, worst, dtype, len(one), float(one.abs().max()), D)
            got = out[rows[b]:rows[b + 1]].double().cpu().view(want.shape)
            assert ((got - want).abs() / tol).max().item() <= 1.0, (layer, b)
    batch.step([0, 1, 1])                                      # the place is empty, its three pages are free
    assert batch.plan["kv_lens"].tolist() == [0, 2, 29] and batch.plan["counts"].tolist() == [2, 0, 15, 0]


def test_a_plan_into_an_earlier_one_s_outputs_looks_at_every_tensor_once(monkeypatch):
    """The checks of ``out=`` are on the path of every step: each tensor's address is asked for as often as without it, and once more for
    its bytes."""
    table, one = _i32([[0, -1], [1, -1]])[:, :2], _i32([1, 1])
    args = (_i32([3, 15]), one, _i32([5, 6]), _i32([2]), table, 16, 4)
    plan = ops.paged_batch_plan(*args)
    asked = []
    address = torch.Tensor.data_ptr
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: asked.append(1) or address(t))
    ops.paged_batch_plan(*args)
    alone = len(asked)
    again = ops.paged_batch_plan(*args, out=plan)
    assert again is plan and alone == 11 and len(asked) - alone <= 2 * alone


def test_a_batch_refuses_to_be_captured_and_its_layers_can_be():
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    g = torch.Generator().manual_seed(72)
    pool = KvCachePool(max_pages=8, num_layers=1, num_heads=2, head_dim=64, page_len=16, dtype=torch.bfloat16, device=DEV)
    batch = KvBatch(pool, 2, 64)
    qkv = torch.randn(5, 8, 64, generator=g).to(torch.bfloat16).to(DEV)
    batch.step([3, 2])

    def layer():
        batch.append(0, qkv[:, 4:6], qkv[:, 6:])
        return batch.attention(0, qkv[:, :4])

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="captured"):
            batch.step([1, 1])
        with pytest.raises(ValueError, match="captured"):
            batch.release(0)
        out = layer()
    assert batch.lens == [3, 2] and batch.num_free == 6
    for i in range(3):
        qkv.copy_(torch.randn(5, 8, 64, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(layer(), out), i
        (torch.randn(500, 500, device=DEV) @ torch.randn(500, 500, device=DEV)).sum().item()
    batch.step([1, 1])
    assert batch.plan["kv_lens"].tolist() == [4, 3]


@pytest.mark.parametrize("lens", [[(900, 1)] * 5, [(60, 1), (33, 4)], [(700, 130), (64, 1)], [(60, 40), (300, 200), (41, 1)]], ids=str)
def test_the_output_may_be_the_queries_themselves_and_nothing_else_that_is_read(lens):
    g = torch.Generator().manual_seed(73)
    q, pool, table, starts, kv = _batch(g, lens, 16, 8, 2, 128, torch.bfloat16, spare=40)
    pool, most = pool.to(DEV), (max(n for _, n in lens), max(kv))
    plain = ops.paged_attention(q.to(DEV), pool, _i32(table), _i32(starts), _i32(kv), *most)
    own = q.to(DEV)
    got = ops.paged_attention(own, pool, _i32(table), _i32(starts), _i32(kv), *most, out=own.view(len(q), -1))
    assert got.data_ptr() == own.data_ptr() and torch.equal(got, plain)
    room = torch.zeros(len(q) + 1, 8 * 128, dtype=torch.bfloat16, device=DEV)
    fused = room[:-1].view(-1, 8, 128)
    shifted = torch.zeros(len(q) * 8 * 128 * 2, dtype=torch.bfloat16, device=DEV).view(len(q), 16, 128)
    for queries, out in [(fused, room[1:]), (shifted[:, 8:], shifted.view(-1)[:len(q) * 1024].view(len(q), -1)),
                         (q.to(DEV), pool.view(-1)[:len(q) * 1024].view(len(q), -1))]:
        with pytest.raises(ValueError, match="overlaps"):
            ops.paged_attention(queries, pool, _i32(table), _i32(starts), _i32(kv), *most, out=out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_page_is_copied_to_another_of_the_same_pool(dtype):
    g = torch.Generator().manual_seed(74)
    pool = torch.randn(6, 2, 16, 3, 64, generator=g).to(dtype)
    want = pool.clone()
    want[1, :, 5:12] = pool[4, :, 2:9]
    dev = pool.to(DEV)
    ops.kv_append_paged_(dev, dev[4, 0, 2:9], dev[4, 1, 2:9], torch.arange(16 + 5, 16 + 12, device=DEV))
    assert torch.equal(dev.cpu(), want)
