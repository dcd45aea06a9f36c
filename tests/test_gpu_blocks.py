"""GPU: bounds of the pages' keys, blocks selected by them and attention over those blocks, against plain loops and float64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import blocks as ok
from subspec_amd import _lib as L
from subspec_amd import ops

DEV = "cuda:0"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ bounds
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,D,page_len", [(1, 1, 64, 1), (40, 1, 64, 16), (61, 4, 128, 16), (300, 8, 128, 64), (33, 3, 64, 2), (600, 32, 128, 256),
                                                     (9, 2, 128, 4), (5000, 2, 64, 16), (4200, 1, 128, 1)])
def test_bounds(dtype, tokens, heads, D, page_len):
    print("bounds", dtype, tokens, heads, D, page_len, flush=True)
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page_len) + 3
    pool = torch.randn(pages, 2, page_len, heads, D, generator=g).to(dtype)
    at = torch.randint(0, pool[:, 0].numel(), (3, 5), generator=g)
    for value, where in zip((math.nan, math.inf, -math.inf), at):
        keys = pool[:, 0].clone().flatten()
        keys[where] = value
        pool[:, 0] = keys.view_as(pool[:, 0])
    order = torch.randperm(pages, generator=g)
    rows = torch.arange(tokens) + page_len // 2
    slots = order[rows // page_len] * page_len + rows % page_len
    slots[torch.arange(tokens) % 11 == 7] = -1
    slots = torch.cat([slots, torch.tensor([pages * page_len - 1 + page_len, 1 << 40, -1, -page_len - 1])])
    before = torch.randn(pages, heads, 2, D, generator=g).to(dtype)
    want = ok.page_bounds(before, pool, slots.tolist())
    got = ops.kv_page_bounds_(before.to(DEV), pool.to(DEV), slots.to(DEV)).cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("dtype,nans", [(torch.bfloat16, [0x7f81, 0xff81, 0x7fff, 0xffff]), (torch.float16, [0x7c01, 0xfc01, 0x7fff, 0xffff])])
def test_bounds_of_every_nan_and_of_the_largest_numbers(dtype, nans):
    """Every kind of NaN stays one, in both; infinities, the largest and the smallest numbers of either sign and the zeros are numbers like others."""
    top = torch.finfo(dtype).max
    pool = torch.randn(12, 2, 8, 1, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    for page, bits in enumerate(nans):
        pool.view(torch.int16)[page, 0, 3, 0, 5] = bits - (1 << 16) if bits >= 1 << 15 else bits
    for page, values in ((4, [math.inf] * 8), (5, [-math.inf] * 8), (6, [math.inf, -math.inf] * 4), (7, [top, -top] * 4), (8, [-top] * 8),
                         (9, [0.0, -0.0] * 4), (10, [2.0 ** -24 if dtype is torch.float16 else 2.0 ** -133, -1.0] * 4)):
        pool[page, 0, :, 0, 9] = torch.tensor(values).to(dtype)
    slots = torch.arange(12 * 8)
    want = ok.page_bounds(torch.zeros(12, 1, 2, 64, dtype=dtype), pool, slots.tolist())
    got = ops.kv_page_bounds_(torch.zeros(12, 1, 2, 64, dtype=dtype, device=DEV), pool.to(DEV), slots.to(DEV)).cpu()
    assert got[:4, 0, :, 5].isnan().all() and torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_a_page_named_twice_and_nothing_at_all():
    pool = torch.randn(3, 2, 4, 2, 64, device=DEV).to(torch.bfloat16)
    bounds = torch.zeros(3, 2, 2, 64, device=DEV, dtype=torch.bfloat16)
    ops.kv_page_bounds_(bounds, pool, torch.empty(0, dtype=torch.int64, device=DEV))
    assert bounds.eq(0).all()
    ops.kv_page_bounds_(bounds, pool, torch.tensor([7, 7, 7], device=DEV))
    assert bounds[[0, 2]].eq(0).all() and torch.equal(bounds[1, :, 0], pool[1, 0].amin(0)) and torch.equal(bounds[1, :, 1], pool[1, 0].amax(0))


# ------------------------------------------------------------------------------------------------ selection
def _maps(g, lens, page_len, spare=2):
    """(table, sequences, positions, pages) of sequences (rows, new ones) in random pages."""
    counts = [-(-t // page_len) for t, _ in lens]
    order = torch.randperm(sum(counts) + spare, generator=g).tolist()
    width, table, at = max(counts + [1]) + 1, [], 0
    for c in counts:
        table.append(order[at:at + c] + [-1] * (width - c))
        at += c
    seq = [b for b, (_, n) in enumerate(lens) for _ in range(n)]
    pos = [t - n + i for t, n in lens for i in range(n)]
    return table, seq, pos, len(order)


SELECT = [  # (rows with the new ones, new ones) of every sequence, page_len, Hq, Hkv, D, keep, recent
    ([(1, 1)], 16, 4, 2, 64, 3, 1), ([(100, 1)], 16, 28, 4, 128, 3, 1), ([(100, 1), (7, 1), (333, 1), (64, 1), (65, 1)], 16, 28, 4, 128, 4, 2),
    ([(333, 9), (200, 5), (50, 4)], 16, 8, 8, 64, 5, 1), ([(90, 90)], 4, 4, 1, 128, 6, 3), ([(700, 3)], 1, 4, 2, 64, 65, 64),
    ([(9000, 2), (5000, 1)], 1, 2, 1, 64, 300, 1), ([(2000, 1)], 2, 64, 1, 64, 900, 7), ([(50, 2)], 8, 2, 2, 64, 3, 3), ([(600, 6)], 64, 6, 3, 128, 1, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", SELECT, ids=lambda c: f"{c[0]}-{c[1:]}")
@pytest.mark.parametrize("values", ["random", "whole", "flat"])
def test_select(dtype, case, values):
    """``whole``: sums of whole numbers, with many equal scores; ``flat``: all scores are equal but a few."""
    lens, page_len, Hq, Hkv, D, keep, recent = case
    print("select", dtype, case, values, flush=True)
    g = torch.Generator().manual_seed(7 + len(lens))
    table, seq, pos, pages = _maps(g, lens, page_len)
    T = len(seq)
    if values == "random":
        q, bounds = torch.randn(T, Hq, D, generator=g), torch.randn(pages, Hkv, 2, D, generator=g).sort(2).values
    elif values == "whole":
        q, bounds = torch.randint(-1, 2, (T, Hq, D), generator=g).float(), torch.randint(-2, 3, (pages, Hkv, 2, D), generator=g).float().sort(2).values
    else:
        q, bounds = torch.randint(-2, 3, (T, Hq, D), generator=g).float(), torch.ones(pages, Hkv, 2, D)
        bounds[torch.rand(pages, generator=g) < 0.05] += 1.0
    q, bounds = q.to(dtype), bounds.to(dtype)
    want = ok.select(q, bounds, table, seq, pos, page_len, keep, recent)
    got = ops.select_blocks(q.to(DEV), bounds.to(DEV), _i32(table), _i32(seq), _i32(pos), page_len, keep, recent=recent)
    assert got.tolist() == want


@pytest.mark.parametrize("dtype,Hq,Hkv,D,rows,batch", [(torch.bfloat16, 16, 8, 128, 1100, 24), (torch.float16, 4, 4, 64, 2600, 30)])
def test_select_where_a_workgroup_has_several_spans(dtype, Hq, Hkv, D, rows, batch):
    """More drafts' blocks than fit at once: lists as of every token by itself."""
    print("several spans", dtype, Hq, Hkv, D, rows, batch, flush=True)
    g = torch.Generator().manual_seed(rows)
    lens = [(rows - 7 * b, 1 + b % 5) for b in range(batch)]
    table, seq, pos, pages = _maps(g, lens, 1)
    q = torch.randn(len(seq), Hq, D, generator=g).to(dtype).to(DEV)
    bounds = torch.randn(pages, Hkv, 2, D, generator=g).sort(2).values.to(dtype).to(DEV)
    table, seq, pos = _i32(table), _i32(seq), _i32(pos)
    got = ops.select_blocks(q, bounds, table, seq, pos, 1, 40, recent=3)
    for t in range(len(seq)):
        assert torch.equal(ops.select_blocks(q[t:t + 1], bounds, table, seq[t:t + 1], pos[t:t + 1], 1, 40, recent=3), got[t:t + 1]), t


def test_select_with_infinities_and_nan():
    """A block whose score is NaN counts as +infinity; those behind the token's own are not looked at."""
    g = torch.Generator().manual_seed(3)
    lens, P, D = [(200, 1), (120, 2), (150, 1)], 8, 64
    table, seq, pos, pages = _maps(g, lens, P)
    q, bounds = torch.randn(4, 4, D, generator=g), torch.randn(pages, 2, 2, D, generator=g).sort(2).values
    for page, value in ((table[0][3], math.nan), (table[0][9], math.inf), (table[0][11], -math.inf), (table[1][2], math.nan), (table[1][14], math.nan),
                        (table[2][18], math.inf)):
        bounds[page, :, :, 5] = value
    q[3, 1, 7] = math.nan                                    # every block of KV head 0 scores NaN: the first ones
    want = ok.select(q.bfloat16(), bounds.bfloat16(), table, seq, pos, P, 6, 1)
    got = ops.select_blocks(q.bfloat16().to(DEV), bounds.bfloat16().to(DEV), _i32(table), _i32(seq), _i32(pos), P, 6).tolist()
    assert got == want and got[3][0] == [0, 1, 2, 3, 4, 18] and 3 in got[0][0]


def test_select_bounds_tables_and_tokens_of_nobody():
    g = torch.Generator().manual_seed(5)
    lens, P, D = [(300, 4), (280, 1)], 8, 128
    table, seq, pos, pages = _maps(g, lens, P)
    seq, pos = [-1, 0, 0, 1, 0, 5, 0, 0, 1, 1], [5, 299, 10, 279, 298, 3, -1, 4000000, 100, 2147483647]
    q, bounds = torch.randn(10, 14, D, generator=g).half(), torch.randn(pages, 2, 2, D, generator=g).sort(2).values.half()
    wide = _i32([r + [1 << 30, -5] for r in table])
    view = wide[:, :len(table[0])]
    fused = torch.zeros(10, 18, D, dtype=torch.float16, device=DEV)
    fused[:, 2:16] = q.to(DEV)
    for max_kv in (None, 300, 299, 100, 17, 8, 1, 0):
        # (columns of the table that no row fills are -1: pages clamped into the pool)
        clamped = [[max(0, p) for p in r] for r in table]
        want = ok.select(q, bounds, clamped, seq, pos, P, 5, 2, max_kv)
        got = ops.select_blocks(fused[:, 2:16], bounds.to(DEV), view, _i32(seq), _i32(pos), P, 5, recent=2, max_kv=max_kv)
        assert got.tolist() == want, max_kv
    assert ops.select_blocks(q[:0].to(DEV), bounds.to(DEV), view, _i32([]), _i32([]), P, 5).shape == (0, 2, 5)


def test_select_in_131072_blocks():
    g = torch.Generator().manual_seed(8)
    n, D = 1 << 17, 64
    q, bounds = torch.randn(2, 2, D, generator=g).bfloat16(), torch.randn(n, 1, 2, D, generator=g).sort(2).values.bfloat16()
    table = [torch.randperm(n, generator=g).tolist()]
    want = ok.select(q, bounds, table, [0, 0], [n - 1, n - 2], 1, 2000, 3)
    got = ops.select_blocks(q.to(DEV), bounds.to(DEV), _i32(table), _i32([0, 0]), _i32([n - 1, n - 2]), 1, 2000, recent=3)
    assert got.tolist() == want


# ------------------------------------------------------------------------------------------------ attention
def _tolerance(want, weight, worst, dtype, D, keys, top):
    """Per element.  The result is rounded once (half a step of its type); a probability is two numbers of the type, off by half a step of half a step (in
    fp16 by half of the smallest number, 2^-25, for each key where that is more, and the largest probability is 1 at least); a score is a sum of D
    fp32 products in any order (2^-24 of the sum of their sizes for each addition), its exponential is good to 2^-21, and both act on numerator and
    denominator."""
    half = torch.finfo(dtype).eps / 2
    score = (D + 4) * 2.0 ** -24 * worst + 2.0 ** -21
    small = keys * 2.0 ** -25 * top if dtype == torch.float16 else 0.0
    return half * want.abs() * (1 + half) + (half * half + 2 * score) * weight + small + 2.0 ** -24


def _cache(g, lens, page_len, Hq, Hkv, D, dtype):
    table, seq, pos, pages = _maps(g, lens, page_len)
    pool = torch.full((pages, 2, page_len, Hkv, D), float("nan"), dtype=dtype)
    for b, (t, _) in enumerate(lens):
        for j in range(t):
            pool[table[b][j // page_len], :, j % page_len] = torch.randn(2, Hkv, D, generator=g).to(dtype)
    q = (torch.randn(len(seq), Hq, D, generator=g) * 2).to(dtype)
    return q, pool, table, seq, pos


ATTEND = [  # lens, page_len, Hq, Hkv, D, keep
    ([(1, 1)], 16, 4, 2, 64, 1), ([(300, 1), (1, 1), (64, 1), (65, 1)], 16, 28, 4, 128, 5), ([(100, 3)], 1, 4, 4, 128, 40), ([(500, 5), (40, 2)], 64, 32, 8, 128, 4),
    ([(700, 1)], 256, 16, 1, 64, 2), ([(400, 2)], 8, 17, 1, 64, 12), ([(200, 1)], 32, 64, 1, 128, 4), ([(1500, 1)], 16, 34, 2, 128, 60),
    ([(2500, 3)], 4, 2, 1, 64, 400), ([(90, 90)], 4, 14, 2, 64, 6)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{c[0]}-{c[1:]}")
def test_attention(dtype, case):
    """Lists in any order with holes, entries behind the token, tokens with nothing; unlisted blocks and rows behind a token hold NaN."""
    lens, page_len, Hq, Hkv, D, keep = case
    print("attend", dtype, case, flush=True)
    g = torch.Generator().manual_seed(keep)
    q, pool, table, seq, pos = _cache(g, lens, page_len, Hq, Hkv, D, dtype)
    blocks = []
    for t in range(len(seq)):
        own, heads = pos[t] // page_len, []
        for h in range(Hkv):
            some = torch.randperm(own + 3, generator=g)[:keep].tolist()          # two of them behind the token
            some += [-1] * (keep - len(some))
            if (t + h) % 3 == 1:
                some[keep // 2] = -1
            if (t + h) % 5 == 4:
                some = [-1] * keep
            heads.append(some)
        blocks.append(heads)
    unlisted = pool.clone()
    for b, (total, _) in enumerate(lens):                                         # of a block that no token of the sequence lists, nothing is read
        listed = {(j, h) for t in range(len(seq)) if seq[t] == b for h in range(Hkv) for j in blocks[t][h]}
        for j in range(-(-total // page_len)):
            for h in range(Hkv):
                if (j, h) not in listed:
                    unlisted[table[b][j], :, :, h] = math.nan
    clean = [[[j if 0 <= j <= pos[t] // page_len else -1 for j in row] for row in heads] for t, heads in enumerate(blocks)]
    want, weight, worst = ok.attention(q, pool, table, clean, seq, pos)
    got = ops.block_attention(q.to(DEV), unlisted.to(DEV), _i32(table), _i32(blocks), _i32(seq), _i32(pos)).cpu().double().view_as(want)
    assert not got.isnan().any()
    off = (got - want).abs() / _tolerance(want, weight, worst, dtype, D, keep * page_len, 6.0)
    assert off.max() <= 1, float(off.max())


def test_attention_of_all_blocks_is_the_whole_caches():
    g = torch.Generator().manual_seed(2)
    lens, P = [(200, 3), (77, 1), (16, 2), (31, 31)], 16
    q, pool, table, seq, pos = _cache(g, lens, P, 28, 4, 128, torch.bfloat16)
    width = len(table[0])
    q, pool, table, seq, pos = q.to(DEV), pool.to(DEV), _i32(table), _i32(seq), _i32(pos)
    bounds = torch.zeros(pool.shape[0], 4, 2, 128, dtype=torch.bfloat16, device=DEV)
    blocks = ops.select_blocks(q, bounds, table, seq, pos, P, width)
    got = ops.block_attention(q, pool, table, blocks, seq, pos, scale=0.1)
    want = ops.paged_attention(q, pool, table, _i32([0, 3, 4, 6, 37]), _i32([t for t, _ in lens]), 31, 200, scale=0.1)
    top = float(pool.nan_to_num().float().abs().max())
    # (both against the formula: half a step of the output each, and the other's probabilities by half a step of theirs)
    assert (got.float() - want.float()).abs().max() <= 3 * 2.0 ** -9 * 2 * top


def test_attention_in_place_of_q_strides_and_tokens_of_nobody():
    g = torch.Generator().manual_seed(6)
    lens, P = [(120, 2), (300, 3)], 16
    q, pool, table, seq, pos = _cache(g, lens, P, 8, 2, 64, torch.float16)
    seq[1], seq[3] = -1, 7
    blocks = [[[0, pos[t] // P, 1, -1], [pos[t] // P, 2, -1, 0]] for t in range(5)]
    want, weight, worst = ok.attention(q, pool, table, blocks, seq, pos)
    wide = _i32([r + [9999] for r in table])[:, :len(table[0])]
    fused = torch.zeros(5, 12, 64, dtype=torch.float16, device=DEV)
    fused[:, 1:9] = q.to(DEV)
    out = torch.full((5, 512), 3.0, dtype=torch.float16, device=DEV)
    ops.block_attention(fused[:, 1:9], pool.to(DEV), wide, _i32(blocks), _i32(seq), _i32(pos), out=out)
    mine = q.to(DEV).clone()
    ops.block_attention(mine, pool.to(DEV), wide, _i32(blocks), _i32(seq), _i32(pos), out=mine.view(5, 512))
    assert out[[1, 3]].eq(3.0).all() and torch.equal(mine.view(5, 512)[[1, 3]].cpu(), q.view(5, 512)[[1, 3]])
    for got in (out, mine.view(5, 512)):
        rows = got.cpu().double().view_as(want)[[0, 2, 4]]
        assert ((rows - want[[0, 2, 4]]).abs() <= _tolerance(want, weight, worst, torch.float16, 64, 64, 6.0)[[0, 2, 4]]).all()
    none = ops.block_attention(q.to(DEV), pool.to(DEV), wide, _i32(blocks), _i32(seq), _i32([-1, 0, -7, 0, -1]))
    assert none[[0, 2, 4]].eq(0).all()
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    assert ops.block_attention(q[:0].to(DEV), pool.to(DEV), wide, _i32(blocks)[:0], empty, empty).shape == (0, 512)


def test_pages_far_into_a_pool():
    """Offsets beyond 2^32 bytes, in bounds, scores and rows."""
    D, P, H = 128, 16, 8
    pages = (5 << 30) // (2 * P * H * D * 2) + 1
    pool = torch.empty(pages, 2, P, H, D, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(9)
    far = [pages - 1 - i for i in range(6)]
    rows = torch.randn(6, 2, P, H, D, generator=g).bfloat16()
    pool[far[-1]:] = rows.flip(0).to(DEV)
    bounds = torch.empty(pages, H, 2, D, dtype=torch.bfloat16, device=DEV)
    slots = torch.tensor([p * P + P - 1 for p in far], device=DEV)
    ops.kv_page_bounds_(bounds, pool, slots)
    assert torch.equal(bounds[far[2], :, 0].cpu(), rows[2, 0].amin(0))
    table, pos = [far], [5 * P + 7]
    q = torch.randn(1, 16, D, generator=g).bfloat16()
    small = torch.stack([rows[:, 0].amin(1), rows[:, 0].amax(1)], 2)
    want = ok.select(q, small, [[0, 1, 2, 3, 4, 5]], [0], pos, P, 3)
    blocks = ops.select_blocks(q.to(DEV), bounds, _i32(table), _i32([0]), _i32(pos), P, 3)
    assert blocks.tolist() == want
    got = ops.block_attention(q.to(DEV), pool, _i32(table), blocks, _i32([0]), _i32(pos)).cpu().double().view(1, 16, D)
    want, weight, worst = ok.attention(q, rows, [[0, 1, 2, 3, 4, 5]], want, [0], pos)
    assert ((got - want).abs() <= _tolerance(want, weight, worst, torch.bfloat16, D, 48, 6.0)).all()


def test_pages_outside_the_pool_are_not_left():
    """A table of any numbers: wrong rows are read, none outside the pool."""
    g = torch.Generator().manual_seed(4)
    pool = torch.randn(3, 2, 16, 2, 64, generator=g).bfloat16().to(DEV)
    bounds = torch.zeros(3, 2, 2, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.randn(2, 4, 64, generator=g).bfloat16().to(DEV)
    table = _i32([[-2147483648, 2147483647, 3, -1], [7, 1 << 30, -9, 2]])
    blocks = ops.select_blocks(q, bounds, table, _i32([0, 1]), _i32([63, 60]), 16, 2)
    assert blocks.tolist() == [[[0, 3], [0, 3]]] * 2
    odd = _i32([[[2147483647, -2147483648], [3, 4]], [[1 << 27, 2], [3, 3]]])
    for some in (blocks, odd):
        assert ops.block_attention(q, pool, table, some, _i32([0, 1]), _i32([63, 2147483647])).isfinite().all()


def test_a_captured_step_and_another_stream():
    """Bounds, selection and attention as one graph, replayed with other lengths, against the eager calls; the same on a side stream."""
    g = torch.Generator().manual_seed(12)
    lens, P, H = [(150, 1), (333, 2), (90, 1)], 16, 4
    q, pool, table, seq, pos = _cache(g, lens, P, 28, H, 128, torch.bfloat16)
    q, pool, table, seq, pos = q.to(DEV), pool.nan_to_num().to(DEV), _i32(table), _i32(seq), _i32(pos)
    slots = torch.arange(pool.shape[0] * P, device=DEV)

    def step(bounds):
        ops.kv_page_bounds_(bounds, pool, slots)
        blocks = ops.select_blocks(q, bounds, table, seq, pos, P, 4, recent=2, max_kv=400)
        return blocks, ops.block_attention(q, pool, table, blocks, seq, pos)

    bounds = torch.zeros(pool.shape[0], H, 2, 128, dtype=torch.bfloat16, device=DEV)
    step(bounds)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(bounds)
    for turn in range(4):
        pool.normal_(generator=torch.Generator(device=DEV).manual_seed(turn))
        pos.copy_(_i32([149 - 20 * turn, 331 - turn, 332 - turn, 89 - turn]))
        graph.replay()
        want = step(torch.zeros_like(bounds))
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]), turn
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = step(torch.zeros_like(bounds))
        torch.cuda.synchronize()
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("batch,Hq,Hkv,D,P,keep,rows", [(70, 8, 8, 64, 4, 150, 900), (66, 16, 8, 128, 8, 60, 700), (150, 16, 8, 64, 1, 300, 400)])
def test_more_tiles_than_the_gpu_holds(batch, Hq, Hkv, D, P, keep, rows):
    """So many drafts that a tile is one unit of more rows than are looked up at a time, or two: as the tokens get it when each is its sequence's only one."""
    print("many tiles", batch, Hq, Hkv, D, P, keep, rows, flush=True)
    g = torch.Generator(device=DEV).manual_seed(batch)
    pages = -(-rows // P)
    pool = torch.randn(batch * pages, 2, P, Hkv, D, generator=g, device=DEV).bfloat16()
    table = torch.randperm(batch * pages, generator=g, device=DEV).int().view(batch, pages)
    new = torch.tensor([1 + b % 4 for b in range(batch)], device=DEV)
    seq = torch.repeat_interleave(torch.arange(batch, device=DEV), new).int()
    T = seq.numel()
    pos = (rows - 1 - torch.randint(0, 3 * P, (T,), generator=g, device=DEV)).int()
    q = (torch.randn(T, Hq, D, generator=g, device=DEV) * 2).bfloat16()
    want = torch.rand(batch, Hkv, pages, generator=g, device=DEV)[seq.long()] + 0.1 * torch.rand(T, Hkv, pages, generator=g, device=DEV)
    blocks = want.topk(keep, -1).indices.int()
    got = ops.block_attention(q, pool, table, blocks, seq, pos)
    assert torch.equal(got, ops.block_attention(q, pool, table, blocks, seq, pos))
    first = torch.cumsum(new, 0) - new
    for k in range(4):
        rows_of = first[new > k] + k
        alone = ops.block_attention(q[rows_of], pool, table, blocks[rows_of], seq[rows_of].contiguous(), pos[rows_of].contiguous())
        # each is off from the formula by half a step of the result (2^-8 of it) and little else
        assert ((alone.float() - got[rows_of].float()).abs() <= 2 * (2.0 ** -8 * 1.01 * alone.float().abs() + 2.0 ** -12)).all()


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (8, 4, 64)])
def test_a_replayed_graph_with_other_neighbours(Hq, Hkv, D):
    """The tokens' sequences change between replays, from one run to a token each in turn (more tiles than a batch in order has), some of nobody: as the eager
    calls, and as every token by itself up to the order of its sums."""
    g = torch.Generator().manual_seed(21)
    P, keep, rows, T = 8, 5, 330, 30
    q, pool, table, _, _ = _cache(g, [(rows, 10)] * 3, P, Hq, Hkv, D, torch.bfloat16)
    q, pool, table = q.to(DEV), pool.nan_to_num().to(DEV), _i32(table)
    bounds = ops.kv_page_bounds_(torch.zeros(pool.shape[0], Hkv, 2, D, dtype=torch.bfloat16, device=DEV), pool, torch.arange(pool.shape[0] * P, device=DEV))
    orders = [[0] * 30, [t % 3 for t in range(30)], [0] * 9 + [-1] * 3 + [1] * 17 + [2], [2] * 10 + [5] + [1, 1, 0, 0, 0, 1, 2, 2] * 2 + [-1] * 3, [-1] * 30,
              [t // 10 for t in range(30)]]
    seq, pos = _i32(orders[0]), _i32([rows - 1 - t for t in range(T)])
    out = torch.empty(T, Hq * D, dtype=torch.bfloat16, device=DEV)

    def step(out):
        blocks = ops.select_blocks(q, bounds, table, seq, pos, P, keep)
        return blocks, ops.block_attention(q, pool, table, blocks, seq, pos, out=out)

    step(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(out)
    for turn, order in enumerate(orders + orders[::-1]):
        seq.copy_(_i32(order))
        pos.copy_(_i32([rows - 1 - (7 * t + turn) % 60 for t in range(T)]))
        out.fill_(7.0)
        graph.replay()
        want = step(torch.full_like(out, 7.0))
        assert torch.equal(held[0], want[0]) and torch.equal(out, want[1]), turn
        nobody = torch.tensor([not 0 <= b < 3 for b in order], device=DEV)
        assert out[nobody].eq(7.0).all() and held[0][nobody].eq(-1).all()
        for t in range(0, T, 7):
            if 0 <= order[t] < 3:
                one = ops.select_blocks(q[t:t + 1], bounds, table, seq[t:t + 1], pos[t:t + 1], P, keep)
                assert torch.equal(one[0], held[0][t]), (turn, t)
                alone = ops.block_attention(q[t:t + 1], pool, table, one, seq[t:t + 1], pos[t:t + 1])[0]
                # each is off from the formula by half a step of the result (2^-8 of it) and little else
                assert (alone.float() - out[t].float()).abs().max() <= 2 * (2.0 ** -8 * 1.01 * float(alone.float().abs().max()) + 2.0 ** -14)


def test_many_tokens_take_several_passes():
    """More partial results and scores than are held at a time: tokens go in passes, with the same results."""
    g = torch.Generator().manual_seed(13)
    n, P, D = 700, 1, 64
    pool = torch.randn(n, 2, P, 1, D, generator=g).bfloat16().to(DEV)
    table, T = _i32([list(range(n))]), 60000
    pos = (torch.arange(T, dtype=torch.int32) % n).to(DEV)
    seq = torch.zeros(T, dtype=torch.int32, device=DEV)
    q = torch.randn(n, 32, D, generator=g).bfloat16().to(DEV)
    bounds = ops.kv_page_bounds_(torch.zeros(n, 1, 2, D, dtype=torch.bfloat16, device=DEV), pool, torch.arange(n, device=DEV))
    many = q[torch.arange(T, device=DEV) % n]
    blocks = ops.select_blocks(many, bounds, table, seq, pos, P, 500)
    one = ops.select_blocks(q, bounds, table, seq[:n], pos[:n], P, 500)
    assert torch.equal(blocks, one[torch.arange(T, device=DEV) % n])
    got = ops.block_attention(many, pool, table, blocks, seq, pos)
    part = torch.cat([ops.block_attention(many[a:a + n], pool, table, blocks[a:a + n], seq[a:a + n], pos[a:a + n]) for a in (0, 2 * n, 59500)])
    rows = torch.cat([torch.arange(a, min(a + n, T)) for a in (0, 2 * n, 59500)]).to(DEV)
    # (another call's size, other chunks: the same sums in another order)
    assert (got[rows].float() - part.float()).abs().max() <= 2.0 ** -7 * float(pool.float().abs().max())


# ------------------------------------------------------------------------------------------------ a batch
def _held(batch):
    """Pages of the sequences and the free ones, which together are the batch's, each once."""
    table, free = batch.block_table.tolist(), batch.free_pages.tolist()[:batch.num_free]
    used = [p for b, t in enumerate(batch.lens) for p in table[b][:-(-t // batch.page_len)]]
    assert sorted(used + free) == sorted(batch.pages) and int(batch.n_free) == batch.num_free and batch.kv_lens.tolist() == batch.lens
    return table


def test_steps_with_drafts_over_selected_blocks():
    """Prompts, then steps of a token and drafts: append with bounds, attention over selected blocks, verification, and the drafts that did not stay taken back;
    a sequence ends and another takes its place.  Everything against the formulas, from rows kept on the host."""
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    P, Hq, Hkv, D, V, layers, B = 8, 8, 2, 64, 500, 2, 3
    pool = KvCachePool(max_pages=90, num_layers=layers, num_heads=Hkv, head_dim=D, page_len=P, dtype=torch.bfloat16, device=DEV)
    batch = KvBatch(pool, B, 300, num_pages=80, bounds=True)
    g = torch.Generator().manual_seed(21)
    rows = [[torch.zeros(0, 2, Hkv, D) for _ in range(layers)] for _ in range(B)]     # what every sequence holds

    def layer_pass(new, selected):
        plan = batch.step(new, n_tokens=sum(new) + 2)
        table, T = _held(batch), sum(new) + 2
        for layer in range(layers):
            kv, q = torch.randn(2, T, Hkv, D, generator=g).bfloat16(), torch.randn(T, Hq, D, generator=g).bfloat16()
            at = 0
            for b, n in enumerate(new):
                rows[b][layer] = torch.cat([rows[b][layer], kv[:, at:at + n].transpose(0, 1).float()])
                at += n
            batch.append(layer, kv[0].to(DEV), kv[1].to(DEV))
            got = batch.attention(layer, q.to(DEV), **(dict(blocks=selected, recent=2) if selected else {}))
            if not selected:
                continue
            mirror, bounds = torch.zeros(90, 2, P, Hkv, D, dtype=torch.bfloat16), torch.zeros(90, Hkv, 2, D, dtype=torch.bfloat16)
            for b in range(B):
                for j in range(len(rows[b][layer])):
                    mirror[table[b][j // P], :, j % P] = rows[b][layer][j].bfloat16()
                for j in range(len(rows[b][layer]) // P):
                    keys = mirror[table[b][j], 0]
                    bounds[table[b][j]] = torch.stack([keys.amin(0), keys.amax(0)], 1)
            seq, pos = plan["sequences"].tolist(), plan["positions"].tolist()
            chosen = ok.select(q, bounds, table, seq, pos, P, selected, 2)
            want, weight, worst = ok.attention(q, mirror, table, chosen, seq, pos)
            some = torch.tensor(seq) >= 0
            off = (got.cpu().double().view_as(want) - want)[some].abs() / _tolerance(want, weight, worst, torch.bfloat16, D, 0, 6.0)[some]
            assert off.max() <= 1, (layer, float(off.max()))
        return plan

    layer_pass([120, 77, 200], None)
    for cycle in range(7):
        new = [[5, 4, 0], [1, 6, 9], [9, 9, 9], [3, 0, 17], [2, 2, 2], [0, 8, 1], [4, 4, 4]][cycle]
        layer_pass(new, 6)
        T = sum(new) + 2
        logits, u, v = 2 * torch.randn(T, V, generator=g), torch.rand(T, generator=g), torch.rand(B, generator=g)
        q = torch.softmax(logits + 0.7 * torch.randn(T, V, generator=g), 1)
        tokens = torch.multinomial(q, 1, generator=g)[:, 0].roll(1)
        got = batch.verify(logits.to(DEV), tokens.to(DEV), u.to(DEV), v.to(DEV), q.to(DEV), temperature=1.0, top_p=0.98)
        starts = [0, new[0], new[0] + new[1], sum(new)]
        want = ok.verify_drafts(logits, tokens, starts, u, v, q, lambda r: dict(top_p=0.98))
        accepted = got["accepted"].tolist()
        assert got["tokens"].tolist() == want[0] and accepted == want[2]
        kept = [1 + a if n else 0 for a, n in zip(accepted, new)]
        batch.keep(kept)
        for b in range(B):
            rows[b] = [r[:len(r) - new[b] + kept[b]] for r in rows[b]]
        assert batch.lens == [len(r[0]) for r in rows]
        _held(batch)
        if cycle == 3:
            batch.release(1)
            rows[1] = [r[:0] for r in rows[1]]
            with pytest.raises(ValueError):
                batch.keep([0, 1, 0])
            layer_pass([0, 40, 0], None)
    batch.keep([0] * B)
    with pytest.raises(ValueError):
        batch.keep([1, 0, 0])
    for b in range(B):
        batch.release(b)
    _held(batch)
    assert batch.num_free == 80
    batch.close()
    with pytest.raises(ValueError):
        batch.keep([0] * B)


def test_a_kept_step_waits_for_nothing():
    """``keep`` does not wait for the device."""
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    pool = KvCachePool(max_pages=64, num_layers=1, num_heads=2, head_dim=64, page_len=4, dtype=torch.bfloat16, device=DEV)
    batch = KvBatch(pool, 2, 100)
    batch.step([30, 40])
    batch.keep([11, 40])
    batch.step([9, 9])
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        batch.keep([1, 0])
    finally:
        torch.cuda.set_sync_debug_mode("default")
    _held(batch)
    assert batch.lens == [12, 40]


def test_a_batch_refuses_selection_without_bounds():
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    pool = KvCachePool(max_pages=16, num_layers=1, num_heads=2, head_dim=64, page_len=4, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    plain = KvBatch(pool, 1, 20, num_pages=4)
    plain.step([2])
    with pytest.raises(ValueError):
        plain.attention(0, q, blocks=2)
    batch = KvBatch(pool, 1, 20, num_pages=4, bounds=True)
    batch.step([2])
    with pytest.raises(ValueError):
        batch.attention(0, q, window=4, blocks=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = q + 1
        with pytest.raises(ValueError):
            batch.keep([1])
    del x


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    g = torch.Generator().manual_seed(1)
    pool = torch.randn(4, 2, 4, 2, 64, generator=g).bfloat16().to(DEV)
    bounds = torch.zeros(4, 2, 2, 64, dtype=torch.bfloat16, device=DEV)
    table, seq, pos, slots = _i32([[0, 1, 2]]), _i32([0, 0]), _i32([8, 9]), torch.tensor([3], device=DEV)
    q = torch.randn(2, 4, 64, generator=g).bfloat16().to(DEV)
    blocks = _i32([[[0, 2], [1, 2]]] * 2)
    for bad in (dict(bounds=bounds.half()), dict(bounds=bounds[:3]), dict(bounds=bounds.transpose(1, 2)), dict(slots=slots.int()), dict(slots=slots[None]),
                dict(bounds=pool.view(-1)[:4 * 2 * 2 * 64].view(4, 2, 2, 64))):
        a = dict(bounds=bounds, slots=slots)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.kv_page_bounds_(a["bounds"], pool, a["slots"])

    def select(**change):
        a = dict(q=q, bounds=bounds, table=table, seq=seq, pos=pos, page_len=4, keep=2, recent=1, out=None, workspace=None)
        a.update(change)
        return ops.select_blocks(a["q"], a["bounds"], a["table"], a["seq"], a["pos"], a["page_len"], a["keep"], recent=a["recent"], out=a["out"],
                                 workspace=a["workspace"])

    for bad in (dict(q=q.half()), dict(q=q[:1]), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(seq=seq.long()), dict(pos=pos[:1]), dict(table=table.long()),
                dict(table=table.t()), dict(page_len=3), dict(page_len=0), dict(keep=0), dict(recent=0), dict(recent=3), dict(out=blocks.long()),
                dict(out=blocks[:1]), dict(bounds=bounds[:, :, :1])):
        with pytest.raises(ValueError):
            select(**bad)
    long = _i32([0, 0] + [0] * 6)
    with pytest.raises(ValueError):
        select(seq=long[:2], out=long.view(2, 2, 2))           # the outputs over the sequences
    with pytest.raises(L.SubspecHipError):
        select(workspace=torch.empty(16, dtype=torch.uint8, device=DEV), table=_i32([list(range(3)) * 30]))

    def attend(**change):
        a = dict(q=q, pool=pool, table=table, blocks=blocks, seq=seq, pos=pos, out=None, scale=None)
        a.update(change)
        return ops.block_attention(a["q"], a["pool"], a["table"], a["blocks"], a["seq"], a["pos"], out=a["out"], scale=a["scale"])

    for bad in (dict(q=q.half()), dict(q=q[:1]), dict(q=q[:, :3]), dict(pool=pool.transpose(0, 1)), dict(blocks=blocks.long()), dict(blocks=blocks[:, :1]),
                dict(blocks=blocks[..., :0]), dict(blocks=blocks.transpose(1, 2)), dict(seq=seq[:1]), dict(pos=pos.long()), dict(scale=0.0), dict(scale=-1.0),
                dict(out=torch.empty(2, 256, device=DEV)), dict(out=q.view(2, 256)[:1]), dict(out=pool.view(-1)[:512].view(2, 256)),
                dict(q=torch.zeros(2, 130, 64, dtype=torch.bfloat16, device=DEV))):
        with pytest.raises(ValueError):
            attend(**bad)
    shifted = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        attend(q=shifted[:2], out=shifted.view(-1)[256:768].view(2, 256))         # the outputs over part of q


@pytest.mark.parametrize("Hq,Hkv,D,P,keep", [(8, 8, 64, 4, 9), (28, 4, 128, 16, 4), (16, 2, 64, 1, 70), (32, 2, 128, 8, 5), (20, 1, 64, 8, 5)])
def test_neighbours_of_a_sequence_read_their_blocks_together(Hq, Hkv, D, P, keep):
    """Runs of every length beside each other, sequences in turn, tokens of nobody between; lists that agree, in part, or not at all."""
    print("together", Hq, Hkv, D, P, keep, flush=True)
    g = torch.Generator().manual_seed(keep)
    lens = [(260, 0), (150, 0), (77, 0)]
    _, pool, table, _, _ = _cache(g, lens, P, Hq, Hkv, D, torch.float16)
    seq = [0] * 5 + [1] * 9 + [0, 1, 0, 1, -1, -1, 2, 2, 7, 2] + [2] * 70 + [0] * 3
    pos = [int(torch.randint(-1, lens[b][0], (1,), generator=g)) if 0 <= b < 3 else 5 for b in seq]
    q = (torch.randn(len(seq), Hq, D, generator=g) * 2).half()
    base = torch.randn(3, Hkv, 260, generator=g)
    blocks = []
    for t, b in enumerate(seq):
        own = max(pos[t], 0) // P
        noise = torch.randn(Hkv, own + 1, generator=g) * (0.0, 0.3, 5.0)[t % 3]
        want = base[max(b, 0) % 3, :, :own + 1] + noise
        some = want.topk(min(keep, own + 1), 1).indices
        blocks.append(torch.nn.functional.pad(some, (0, keep - some.shape[1]), value=-1).tolist())
    clean = [[[j if j >= 0 and pos[t] >= 0 else -1 for j in row] for row in heads] for t, heads in enumerate(blocks)]
    want, weight, worst = ok.attention(q, pool, table, clean, seq, pos)
    mine = torch.tensor([0 <= b < 3 for b in seq])
    out = torch.full((len(seq), Hq * D), 7.0, dtype=torch.float16, device=DEV)
    got = ops.block_attention(q.to(DEV), pool.to(DEV), _i32(table), _i32(blocks), _i32(seq), _i32(pos), out=out).cpu()
    assert got[~mine].eq(7.0).all()
    off = (got.double().view_as(want) - want)[mine].abs() / _tolerance(want, weight, worst, torch.float16, D, keep * P, 6.0)[mine]
    assert off.max() <= 1, float(off.max())
    again = ops.block_attention(q.to(DEV), pool.to(DEV), _i32(table), _i32(blocks), _i32(seq), _i32(pos))
    assert torch.equal(again.cpu()[mine], got[mine])
    for t in (0, 4, 13, 20, 24, 93, 96):                           # a token by itself: the same but for the order of its sums
        one = ops.block_attention(q[t:t + 1].to(DEV), pool.to(DEV), _i32(table), _i32(blocks[t:t + 1]), _i32(seq[t:t + 1]), _i32(pos[t:t + 1]))
        if mine[t]:
            off = (one.cpu().double().view(Hq, D) - want[t]).abs() / _tolerance(want, weight, worst, torch.float16, D, keep * P, 6.0)[t]
            assert off.max() <= 1, (t, float(off.max()))


@pytest.mark.parametrize("D,keep,P", [(128, 6, 16), (64, 40, 16), (64, 3, 4)])
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_a_value_that_one_token_does_not_see_stays_out_of_its_sums(D, keep, P, what):
    """Drafts that share a reading: a row behind one of them, and a block that only others list, hold an infinity.  Those that see it get it, the others what they get alone."""
    print("apart", D, keep, P, what, flush=True)
    Hq, Hkv, n = 8, 2, 700
    g = torch.Generator().manual_seed(D + keep)
    _, pool, table, _, _ = _cache(g, [(n, 0), (n, 0)], P, Hq, Hkv, D, torch.bfloat16)
    seq, pos = [0] * 5 + [1] * 3, [n - 5 + i for i in range(5)] + [n - 3 + i for i in range(3)]
    q = torch.randn(8, Hq, D, generator=g).bfloat16()
    last = (n - 1) // P
    blocks = [[[j % last for j in range(t + h, t + h + keep - 1)] + [pos[t] // P] for h in range(Hkv)] for t in range(8)]
    clean = ops.block_attention(q.to(DEV), pool.to(DEV), _i32(table), _i32(blocks), _i32(seq), _i32(pos))
    hit = torch.zeros(8, Hq, dtype=torch.bool)
    bad = pool.clone()
    # the last draft's own row, head 1; a row of the first block that token 4's head 0 lists alone
    row = pos[4]
    bad[table[0][row // P], 1, row % P, 1, 3] = what
    hit[4, Hq // 2:] = True
    alone = [j for j in blocks[4][0] if all(j not in blocks[t][0] for t in range(4))]
    bad[table[0][alone[0]], 1, 1, 0, 5] = what
    hit[4, :Hq // 2] = True
    got = ops.block_attention(q.to(DEV), bad.to(DEV), _i32(table), _i32(blocks), _i32(seq), _i32(pos)).cpu().view(8, Hq, D)
    clean = clean.cpu().view(8, Hq, D)
    assert not torch.isfinite(got[hit]).all(-1).any()
    assert torch.equal(got[~hit], clean[~hit])
    fine = torch.ones(D, dtype=torch.bool)
    fine[[3, 5]] = False
    assert torch.equal(got[hit][:, fine], clean[hit][:, fine])


def test_select_for_a_million_tokens_of_32_heads():
    """2^25 lists: more than one launch of a workgroup a list can have."""
    T, H, D, P = 1 << 20, 32, 64, 16
    q = torch.ones(1, H, D, dtype=torch.bfloat16, device=DEV).expand(T, H, D)
    bounds = torch.zeros(3, H, 2, D, dtype=torch.bfloat16, device=DEV)
    seq, pos = torch.arange(T, device=DEV).int() % 3 - 1, torch.arange(T, device=DEV).int() % 40
    for keep, table in ((2, _i32([[0], [2]])), (1, _i32([[0], [1]])), (2, _i32([[0, 1], [2, 0]]))):
        print("a million tokens", keep, table.tolist(), flush=True)
        seen = torch.where(seq < 0, 0, (pos // P + 1).clamp(max=table.shape[1]))[:, None]
        j = torch.arange(keep, device=DEV)
        want = torch.where(j < seen, j, -1).int()
        got = ops.select_blocks(q, bounds, table, seq, pos, P, keep, out=torch.full((T, H, keep), -7, dtype=torch.int32, device=DEV))
        assert torch.equal(got, want[:, None].expand_as(got))


def test_attention_of_a_million_tokens_of_64_heads():
    """2^26 units of a wavefront: more than one launch can have.  Every token attends to one row and gets its value."""
    T, H, D, width = 1 << 20, 64, 64, 40000                  # (so many columns that no tokens share a unit)
    pool = torch.randn(7, 2, 1, H, D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).bfloat16()
    q = torch.ones(1, H, D, dtype=torch.bfloat16, device=DEV).expand(T, H, D)
    table = (torch.arange(width, device=DEV) % 7).int()[None]
    seq = torch.where(torch.arange(T, device=DEV) % 1000 == 999, -1, 0).int()
    pos = torch.full((T,), width - 1, dtype=torch.int32, device=DEV)
    blocks = (torch.arange(T, device=DEV)[:, None] * 5 + torch.arange(H, device=DEV)).remainder(width).int()[:, :, None].contiguous()
    out = torch.full((T, H * D), 7.0, dtype=torch.bfloat16, device=DEV)
    print("a million tokens", flush=True)
    ops.block_attention(q, pool, table, blocks, seq, pos, out=out)
    step = 1 << 16
    for t0 in range(0, T, step):
        want = pool[(blocks[t0:t0 + step, :, 0] % 7).long(), 1, 0, torch.arange(H, device=DEV)]
        want[seq[t0:t0 + step] < 0] = 7.0
        assert torch.equal(out[t0:t0 + step].view(-1, H, D), want), t0
