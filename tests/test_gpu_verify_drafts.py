"""GPU: drafts verified against the target's probabilities by given numbers, against loops in float64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import blocks as ok
from subspec_amd import ops

DEV = "cuda:0"
# Tokens have to be equal: masses are exact to 2^-42 of a row's largest, so a draw falls on the other side of an entry's border than in float64 once
# in a million rows.  Probabilities are rounded once to fp32 (2^-24 relative) from masses within 0.54 * 2^-42 of the largest each; without filters those
# of drafts that stay are over a row's mass in 32 bits.  Of that a term 2^d, d = (l - top) / (T ln 2), is off by 3 |d| 2^-24 ln 2 (the exponent's rounding, the
# factor's, a slice's largest against the row's) and 2^-23; 2^20 terms of a size below 2^-20 make no more than one, so by 20 * 3 * 2^-24 * 0.7 on average at
# most; a lane adds 32 terms, a wavefront 64 sums in a tree, a row 512 of these, 32 a lane: 2.5e-6 + 2^-23 + 74 * 2^-24 < 2^-17.


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _near(got, want, filtered=False):
    want = torch.tensor(want, dtype=torch.float64)
    return ((got.cpu().double() - want).abs() <= 2.0 ** (-23 if filtered else -17) * want + 2.0 ** -40).all()


def _case(g, rows, V, dtype, q_dtype, t=1.0, noise=0.5, first=0, behind=0):
    """Logits with a few tokens far ahead, a draft that sees them through noise, tokens drawn from it."""
    T = first + sum(rows) + behind
    logits = 2.0 * torch.randn(T, V, generator=g)
    logits.scatter_add_(1, torch.randint(0, V, (T, min(V, 12)), generator=g), 5.0 + 2.0 * torch.randn(T, min(V, 12), generator=g))
    logits = logits.to(dtype)
    probs = torch.softmax((logits.float() + noise * torch.randn(T, V, generator=g)) / max(t, 0.2), -1)
    drawn = torch.multinomial(probs, 1, generator=g)[:, 0]
    tokens = torch.cat([drawn[-1:], drawn[:-1]])
    starts = [first]
    for n in rows:
        starts.append(starts[-1] + n)
    return logits, tokens, starts, torch.rand(T, generator=g), torch.rand(len(rows), generator=g), None if q_dtype is None else probs.to(q_dtype)


def _run(case, **settings):
    logits, tokens, starts, uniforms, draws, q = case
    return ops.verify_drafts(logits.to(DEV), tokens.to(DEV), _i32(starts), uniforms.to(DEV), draws.to(DEV), None if q is None else q.to(DEV), **settings)


def _check(case, got, settings=None, filtered=False):
    tokens, probs, accepted = ok.verify_drafts(*case, settings=settings)
    assert got["accepted"].tolist() == accepted and got["tokens"].tolist() == tokens
    assert _near(got["probs"], probs, filtered)


F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("rows,V,dtype,q_dtype", [
    ([1], 1, F32, F32), ([2], 1, F32, None), ([5], 7, BF16, BF16), ([3, 0, 1, 9], 100, F32, BF16), ([0, 0], 50, F16, F16), ([4] * 5, 2048, BF16, F32),
    ([2, 5, 3], 2049, F16, F16), ([1] * 9, 8195, F32, None), ([9, 1, 4], 50001, BF16, F16), ([5], 152064, F32, F32), ([3] * 4, 152064, BF16, BF16),
    ([6, 2, 0, 7], 32000, F16, None), ([8], 1 << 20, F16, F32)])
def test_against_the_formula(rows, V, dtype, q_dtype):
    print("verify", rows, V, dtype, q_dtype, flush=True)
    for seed in range(3):
        g = torch.Generator().manual_seed(seed + V)
        for t in (1.0, 0.7):
            case = _case(g, rows, V, dtype, q_dtype, t)
            _check(case, _run(case, temperature=t), lambda row: dict(temperature=t))


@pytest.mark.parametrize("rows,V,dtype,q_dtype", [([3, 2], 60, F32, BF16), ([5], 3000, BF16, BF16), ([2] * 100, 500, F16, None), ([4, 0, 6], 30000, BF16, F32),
                                                  ([9], 152064, F32, F16)])
@pytest.mark.parametrize("top_k,top_p,min_p,t", [(0, 0.9, 0.0, 1.0), (20, 1.0, 0.0, 0.8), (0, 1.0, 0.05, 1.2), (50, 0.8, 0.02, 0.7), (1, 1.0, 0.0, 1.0),
                                                 (1 << 31, 1.0, 0.0, 1.0), (0, 0.0, 0.0, 1.0), (0, 1.0, 1.0, 2.0)])
def test_filters(rows, V, dtype, q_dtype, top_k, top_p, min_p, t):
    print("filters", rows, V, dtype, top_k, top_p, min_p, t, flush=True)
    g = torch.Generator().manual_seed(V + top_k % 97)
    case = _case(g, rows, V, dtype, q_dtype, t)
    settings = dict(temperature=t, top_k=top_k, top_p=top_p, min_p=min_p)
    _check(case, _run(case, **settings), lambda row: settings, filtered=not (top_k in (0, 1 << 31) and top_p == 1.0 and min_p == 0.0))


def test_settings_of_every_row():
    g = torch.Generator().manual_seed(1)
    rows, V = [4, 1, 6, 0, 3, 5], 4000
    case = _case(g, rows, V, F32, F32)
    T = sum(rows)
    t = torch.tensor([0.0, 0.5, 1.0, 2.0])[torch.arange(T) % 4]
    k = torch.tensor([0, 3, 5000, 40, 1], dtype=torch.int32)[torch.arange(T) % 5]
    p = torch.tensor([1.0, 0.9, 0.3])[torch.arange(T) % 3]
    m = torch.tensor([0.0, 0.1])[torch.arange(T) % 2]
    got = _run(case, temperature=t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV), min_p=m.to(DEV))
    _check(case, got, lambda r: dict(temperature=float(t[r]), top_k=int(k[r]), top_p=float(p[r]), min_p=float(m[r])))
    _check(case, _run(case, temperature=t.to(DEV)), lambda r: dict(temperature=float(t[r])))         # (no filter but the rows at T = 0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("filtered", [False, True])
def test_greedy_takes_the_first_largest(dtype, filtered):
    logits = torch.zeros(6, 5000, dtype=dtype)
    logits[0, 77] = logits[0, 4000] = 3.0                    # the drafts' row: the lower of the two
    logits[1, 4999] = 1.0
    logits[3] = -0.0
    logits[3, 9] = 0.0                                       # all equal: entry 0
    tokens = torch.tensor([5, 77, 4000, 5, 0, 1])
    settings = dict(temperature=0.0, **(dict(top_p=0.9) if filtered else {}))
    case = (logits, tokens, [0, 3, 6], torch.zeros(6), torch.full((2,), 0.999), None)
    got = _run(case, **settings)
    _check(case, got, lambda r: settings)
    assert got["tokens"].tolist() == [77, 4999, -1, 0, 0, -1] and got["accepted"].tolist() == [1, 1]


@pytest.mark.parametrize("filtered", [False, True])
def test_rows_of_infinities_and_nan(filtered):
    g = torch.Generator().manual_seed(4)
    logits, tokens, starts, u, v, q = _case(g, [3, 3, 2, 3, 2, 1], 700, F32, F32)
    logits[0, 5], logits[0, 300] = math.nan, -math.inf       # never drawn
    tokens[1] = 5                                            # ... nor kept as a draft
    logits[3] = -math.inf                                    # nothing to draw
    logits[7] = math.nan
    logits[8, 10] = logits[8, 600] = math.inf                # they share the mass
    tokens[9], q[8, 10], u[8] = 10, 0.6, 0.9                 # 0.54 < 0.5 does not hold; the rest is entry 600's 0.5 and nothing of 10's
    q[8, 600] = 0.2
    q[11, :50], q[11, 50:60], q[11, 60] = math.nan, -3.0, math.inf
    tokens[12] = 60                                          # q = inf: never kept
    logits[13, 1:] = -math.inf                               # one entry has all
    settings = dict(top_p=0.95) if filtered else {}
    case = (logits, tokens, starts, u, v, q)
    got = _run(case, **settings)
    _check(case, got, lambda r: settings)
    assert got["tokens"][3].item() == -1 and got["probs"][3].item() == 0 and got["tokens"][8].item() == 600 and got["tokens"][13].item() == 0


@pytest.mark.parametrize("bad", [-1, 300, 1 << 40, -(1 << 50)])
def test_drafts_outside_the_vocabulary_do_not_stay(bad):
    g = torch.Generator().manual_seed(5)
    for q_dtype in (F32, None):
        logits, tokens, starts, u, v, q = _case(g, [4, 3], 300, BF16, q_dtype)
        tokens[1] = tokens[6] = bad
        got = _run((logits, tokens, starts, u, v, q))
        _check((logits, tokens, starts, u, v, q), got)
        assert got["accepted"][0].item() == 0


def test_the_numbers_at_their_borders():
    """u q < p is strict; a draw of 0 takes the first entry with mass, the largest number below 1 the last."""
    V = 4
    logits, q = torch.zeros(8, V), torch.full((8, V), 0.25)
    q[2] = torch.tensor([0.5, 0.5, 0.0, 0.0])
    u = torch.tensor([0.99999994, 0.0, 0.5, 0.0, 0.0, 0.0, 0.0, 0.0])
    tokens = torch.tensor([0, 1, 2, 1, 0, 3, 0, 2])
    # sequence 0: p = q stays for all u below 1; row 2: 0.5 * 0.5 < 0.25 does not hold, the rest is entries 2 and 3
    for v0, last in ((0.0, 2), (0.5, 3), (0.49999997, 2), (0.99999994, 3)):
        got = _run((logits, tokens, [0, 4, 4, 8], u, torch.tensor([v0, 0.3, v0]), q))
        assert got["tokens"].tolist()[:4] == [1, 2, last, -1] and got["accepted"].tolist() == [2, 0, 3]
        assert got["tokens"].tolist()[4:] == [3, 0, 2, {0.0: 0, 0.5: 2, 0.49999997: 1, 0.99999994: 3}[v0]]
        assert torch.equal(got["probs"].cpu(), torch.tensor([0.25, 0.25, 0.25, 0.0, 0.25, 0.25, 0.25, 0.25]))
    # a draft that takes all of its entry leaves nothing: the row's own distribution
    q[:] = torch.tensor([1.0, 1.0, 1.0, 1.0])
    got = _run((logits, tokens, [0, 4, 4, 8], torch.full((8,), 0.9), torch.tensor([0.6, 0.0, 0.99]), q))
    assert got["accepted"].tolist() == [0, 0, 0] and got["tokens"].tolist() == [2, -1, -1, -1, 3, -1, -1, -1]
    # the draft is certain and the target has no mass there
    logits[:, 1] = -math.inf
    got = _run((logits, tokens, [0, 4, 4, 8], torch.zeros(8), torch.tensor([0.6, 0.0, 0.99]), None))
    assert got["accepted"].tolist() == [0, 0, 3] and got["tokens"].tolist()[:4] == [2, -1, -1, -1]


def test_rows_of_nobody_layouts_and_given_outputs():
    g = torch.Generator().manual_seed(6)
    rows, V = [3, 0, 5, 1], 3001
    for dtype in (F32, BF16):
        case = _case(g, rows, V, dtype, dtype, first=2, behind=3)
        logits, tokens, starts, u, v, q = case
        want = ok.verify_drafts(*case)
        wide = torch.full((14, V + 9), math.nan, dtype=dtype, device=DEV)
        wide[:, 3:V + 3] = logits.to(DEV)
        strided = torch.full((14, 2 * V), math.nan, dtype=dtype, device=DEV)[:, ::2]
        strided[:] = q.to(DEV)
        wide[:2], wide[-3:] = math.nan, math.nan               # rows of nobody
        out = dict(tokens=torch.full((14,), 5, device=DEV), probs=torch.full((14,), 5.0, device=DEV), accepted=_i32([9] * 4))
        for given in (None, out):
            got = ops.verify_drafts(wide[:, 3:V + 3], tokens.to(DEV), _i32(starts), u.to(DEV), v.to(DEV), strided, out=given)
            assert got["tokens"].tolist() == want[0] and got["accepted"].tolist() == want[2] and _near(got["probs"], want[1])
            assert given is None or got["tokens"] is out["tokens"]
    none = ops.verify_drafts(logits[:0].to(DEV), tokens[:0].to(DEV), _i32([0, 0, 0]), u[:0].to(DEV), v[:2].to(DEV), None)
    assert none["accepted"].tolist() == [0, 0] and none["tokens"].numel() == 0


@pytest.mark.parametrize("starts", [[3, 1, 9], [0, -5, 6], [0, 1 << 30, 6], [-2147483648, 2147483647, 0]])
def test_starts_out_of_order_stay_inside_the_call(starts):
    g = torch.Generator().manual_seed(7)
    case = _case(g, [3, 3], 5000, F32, F32)
    for settings in ({}, dict(top_p=0.9)):
        got = _run((case[0], case[1], starts, *case[3:]), **settings)
        assert got["tokens"].min() >= -1 and got["tokens"].max() < 5000 and got["accepted"].min() >= 0 and got["accepted"].max() < 6


@pytest.mark.parametrize("left", [-1.0, -3e38, float("nan")])
def test_starts_out_of_order_after_other_work(left):
    """A sequence whose rows begin before the first start has no sums of them: whatever the workspace held, it ends with its last row."""
    case = _case(torch.Generator().manual_seed(8), [3, 3], 5000, F32, F32)
    for _ in range(3):
        held = [torch.full((1 << 16,), left, device=DEV) for _ in range(16)]
        torch.cuda.synchronize()
        del held
        got = _run((case[0], case[1], [5, 0, 6], *case[3:]))
        assert 0 <= int(got["accepted"].min()) and int(got["accepted"].max()) < 6
        assert got["tokens"].min() >= -1 and got["tokens"].max() < 5000


def test_what_comes_out_is_distributed_like_the_target():
    """4096 sequences over one pair of distributions, three drafts each: the tokens at every place follow p (each count within five standard deviations of
    its mean: one entry in 3.5 million is further off), and as many drafts stay as sum min(p, q) says."""
    V, B = 9, 4096
    g = torch.Generator().manual_seed(8)
    logits, draft = torch.randn(4, V, generator=g), torch.randn(4, V, generator=g)
    q = torch.softmax(draft, 1)
    drawn = torch.multinomial(q.repeat(B, 1), 1, generator=g).view(B, 4)
    tokens = torch.cat([torch.zeros(B, 1, dtype=torch.int64), drawn[:, :3]], 1).reshape(-1)
    case = (logits.repeat(B, 1), tokens, list(range(0, 4 * B + 1, 4)), torch.rand(4 * B, generator=g), torch.rand(B, generator=g), q.repeat(B, 1))
    for settings in ({}, dict(top_k=5)):
        got = _run(case, **settings)
        out, accepted = got["tokens"].view(B, 4).cpu(), got["accepted"].cpu()
        left = B
        for i in range(4):
            p = ok.target_probs(logits[i], **settings)
            here = out[:, i][accepted >= i]
            assert here.numel() == left
            count = torch.bincount(here, minlength=V).double()
            assert ((count - left * p).abs() <= 5 * (left * p * (1 - p)).sqrt() + 1e-9).all(), (i, count, left * p)
            if i < 3:
                a = float(torch.minimum(p, q[i].double()).sum())
                stays = int((accepted > i).sum())
                assert abs(stays - left * a) <= 5 * math.sqrt(left * a * (1 - a))
                left = stays


def test_a_replayed_graph_other_streams_and_the_same_bits():
    g = torch.Generator().manual_seed(9)
    for settings in ({}, dict(top_p=0.9, top_k=30)):
        cases = [tuple(x.to(DEV) if isinstance(x, torch.Tensor) else x for x in _case(g, [5, 2, 7], 40000, BF16, F32)) for _ in range(4)]
        live = [x.clone() if isinstance(x, torch.Tensor) else _i32(x) for x in cases[0]]
        ops.verify_drafts(*live, **settings)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = ops.verify_drafts(*live, **settings)
        side = torch.cuda.Stream()
        for case in cases[1:] + cases[:1]:
            for i, x in enumerate(case):
                live[i].copy_(_i32(x) if i == 2 else x)
            graph.replay()
            want = ops.verify_drafts(*case[:2], _i32(case[2]), *case[3:], **settings)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                again = ops.verify_drafts(*case[:2], live[2], *case[3:], **settings)
            torch.cuda.synchronize()
            for name in want:
                assert torch.equal(held[name], want[name]) and torch.equal(again[name], want[name])
        tokens, _, accepted = ok.verify_drafts(*[x.cpu() if isinstance(x, torch.Tensor) else x for x in cases[0]], settings=lambda r: settings)
        assert want["tokens"].tolist() == tokens and want["accepted"].tolist() == accepted


def test_refusals():
    g = torch.Generator().manual_seed(1)
    logits, tokens, starts, u, v, q = (x.to(DEV) if isinstance(x, torch.Tensor) else _i32(x) for x in _case(g, [3, 2], 40, F32, F32))

    def call(out=None, workspace=None, **change):
        a = dict(logits=logits, tokens=tokens, starts=starts, u=u, v=v, q=q, settings={})
        a.update(change)
        return ops.verify_drafts(a["logits"], a["tokens"], a["starts"], a["u"], a["v"], a["q"], out=out, workspace=workspace, **a["settings"])

    good = call()
    for bad in (dict(logits=logits[0]), dict(tokens=tokens.int()), dict(tokens=tokens[:4]), dict(starts=starts.long()), dict(starts=starts[:1]), dict(u=u[:4]),
                dict(u=u.double()), dict(v=v[:1]), dict(q=q[:4]), dict(q=q[:, :39]), dict(q=q.double()), dict(logits=logits.double()),
                dict(settings=dict(temperature=-1.0)), dict(settings=dict(top_k=-1)), dict(settings=dict(top_p=-0.1)), dict(settings=dict(min_p=-1.0)),
                dict(settings=dict(temperature=torch.ones(2, device=DEV))), dict(settings=dict(top_k=torch.ones(5, device=DEV))),
                dict(out=dict(good, tokens=good["tokens"].int())), dict(out=dict(good, probs=good["probs"][:4])), dict(out=dict(good, tokens=tokens)),
                dict(out=dict(good, probs=u)), dict(out=dict(good, accepted=starts[:2]))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(Exception):
        call(workspace=torch.empty(300, dtype=torch.uint8, device=DEV))
    with pytest.raises(Exception):
        call(logits=logits.cpu())
    again = call(out=good)
    assert again["tokens"] is good["tokens"]


@pytest.mark.parametrize("V", [3000, 152064])
def test_numbers_at_the_border_in_32_bits(V):
    """u q within 2^-30 of p on either side, nearer than a row's mass in 32 bits can tell: the row's mass in 64 bits decides, draft after draft."""
    g = torch.Generator().manual_seed(V)
    logits, tokens, starts, u, v, _ = _case(g, [9, 5], V, F32, None)
    q = torch.zeros(14, V)
    side = torch.rand(14, generator=g) < 0.8
    for i in range(13):
        x = int(tokens[i + 1])
        p = float(ok.target_probs(logits[i])[x])
        u[i] = 0.75
        q[i, x] = p / 0.75                                    # rounded to fp32: 0.75 q is within 2^-24 of p, on the side that the rounding is
        while (0.75 * float(q[i, x]) < p) != bool(side[i]):
            q[i, x] = torch.nextafter(q[i, x], torch.tensor(0.0 if side[i] else 9.0))
    case = (logits, tokens, starts, u, v, q)
    got = _run(case)
    _check(case, got)
    assert got["accepted"].tolist() == [int(side[:8].int().cumprod(0).sum()), int(side[9:13].int().cumprod(0).sum())]


# ------------------------------------------------------------------------------------------------ masked vocabularies, small temperatures
def _masked(g, rows, V, dtype, q_dtype, t, value, how, best):
    """Logits of which ``how`` many are masked by a finite number, drafts that see the mask: drawn ones, or with ``best`` the rows' largest (which stay where p is 1)."""
    logits, tokens, starts, u, v, _ = _case(g, rows, V, F32, None, t)
    T = logits.shape[0]
    open_ = torch.zeros(T, V, dtype=torch.bool)
    if how == "slices":                                      # a row is looked at in slices of 2048: the odd ones, and what is left behind the last whole one
        open_[:] = torch.arange(V) // 2048 % 2 == 0
        open_[:, V // 2048 * 2048:] = V < 2048
        open_[:, 5] = True
    elif how == "all but three":
        open_.scatter_(1, torch.randint(0, V, (T, 3), generator=g), True)
    elif how == "nothing":
        open_[:] = True
    logits = torch.where(open_, logits, value).to(dtype)
    probs = torch.softmax(((logits.double() - logits.double().amax(1, keepdim=True)) / max(t, 0.2)) + 0.3 * torch.randn(T, V, generator=g), -1).float()
    drawn = logits.float().argmax(1) if best else torch.multinomial(probs, 1, generator=g)[:, 0]
    return logits, torch.cat([drawn[-1:], drawn[:-1]]), starts, u, v, None if q_dtype is None else probs.to(q_dtype)


def _both_ways(case, t):
    """The call without filters, and with one that takes nothing away and so goes by masses in 64 bits alone: the formula's, both."""
    want = ok.verify_drafts(*case, settings=lambda row: dict(temperature=t))
    for settings in ({}, dict(min_p=1e-30)):
        got = _run(case, temperature=t, **settings)
        assert got["accepted"].tolist() == want[2] and got["tokens"].tolist() == want[0], (settings, got["accepted"].tolist(), want[2])
        assert _near(got["probs"], want[1], bool(settings)), settings
    return want


MASKS = [(dtype, value) for dtype in (F32, BF16, F16) for value in (-1e4, -1e9, -1e10, -1e30, torch.finfo(dtype).min) if value >= torch.finfo(dtype).min]


@pytest.mark.parametrize("how", ["slices", "all but three", "all"])
@pytest.mark.parametrize("dtype,value", MASKS)
def test_vocabularies_masked_by_finite_numbers(dtype, value, how):
    """A mask that is no infinity leaves slices of a row, or all of it, at one large negative number."""
    stays = 0
    for V, rows in ((5000, [4, 3, 1, 5]), (2049, [6])):
        for n, t in enumerate((0.2, 0.3, 0.5, 0.7, 1.0, 1.3, 1.5)):
            g = torch.Generator().manual_seed(V + n)
            for best in (False, True):
                print("masked", dtype, how, value, V, t, best, flush=True)
                stays += sum(_both_ways(_masked(g, rows, V, dtype, None if best else F32, t, value, how, best), t)[2])
    assert stays > 20                                        # (most drafts stay, if anything is right)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t", [1e-3, 1e-6, 1e-8, 1e-9, 1e-20, 1e-37, 1.2e-38, 30.0, 1e6, 1e30])
def test_temperatures_of_any_size(dtype, t):
    """Down to the smallest that is not greedy, where one entry has all unless others equal it, and up to those where all have the same."""
    stays = 0
    for V, rows in ((5000, [4, 3, 1, 5]), (2049, [6]), (7, [3, 2])):
        g = torch.Generator().manual_seed(V)
        for best in (False, True):
            print("temperature", dtype, t, V, best, flush=True)
            stays += sum(_both_ways(_masked(g, rows, V, dtype, None if best and t < 1 else F32, t, 0.0, "nothing", best), t)[2])
    assert stays > 3


def test_a_masked_row_beside_ordinary_ones():
    """Rows of one call with temperatures of their own, some masked: nothing of one reaches another."""
    g = torch.Generator().manual_seed(12)
    rows, V = [5, 4, 6], 9000
    T = sum(rows)
    logits, tokens, starts, u, v, q = _masked(g, rows, V, F32, F32, 1.0, torch.finfo(F32).min, "slices", False)
    plain = _case(g, rows, V, F32, F32)
    some = torch.arange(T) % 3 == 1
    logits[~some], q[~some] = plain[0][~some], plain[5][~some]
    t = torch.tensor([1.0, 1e-9, 0.4, 0.0])[torch.arange(T) % 4]
    drawn = logits.argmax(1)
    case = (logits, torch.cat([drawn[-1:], drawn[:-1]]), starts, 0.02 * u, v, q)
    want = ok.verify_drafts(*case, settings=lambda r: dict(temperature=float(t[r])))
    assert want[2] == [4, 3, 5]
    for settings in ({}, dict(min_p=1e-30)):
        got = _run(case, temperature=t.to(DEV), **settings)
        assert got["accepted"].tolist() == want[2] and got["tokens"].tolist() == want[0] and _near(got["probs"], want[1], bool(settings))


@pytest.mark.parametrize("rows,V", [([4] * 25, 20000), ([5, 3], 300)])
@pytest.mark.parametrize("settings", [dict(top_p=0.99999999), dict(min_p=1e-46), dict(top_p=1 - 2.0 ** -25, min_p=5e-46)])
def test_settings_that_filter_nothing_once_they_are_32_bits(rows, V, settings):
    """A number below 1, or above 0, that fp32 does not tell from it is no filter: the call without filters, which has a workspace of another size."""
    case = _case(torch.Generator().manual_seed(V), rows, V, BF16, F32)
    got, want = _run(case, **settings), _run(case)
    assert all(torch.equal(got[name], want[name]) for name in want)
    nearly = dict(top_p=1 - 2.0 ** -24) if "top_p" in settings else dict(min_p=1e-45)                    # the next number that is one
    _check(case, _run(case, **nearly), lambda row: nearly, filtered=True)
