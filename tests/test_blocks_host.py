"""What the entry points of selected blocks and of drafts' verification refuse, from the library's host code alone, and their oracles on cases done by hand."""
import math

import pytest
import torch

from oracle import blocks as ok
from subspec_amd import _lib as L
from subspec_amd import ops

ANY = 4096                                                   # a non-null, aligned address that no refused call touches


def _bounds(**change):
    a = dict(pool=ANY, bounds=ANY, dtype=L.BF16, pages=4, page_len=16, heads=2, D=64, slots=ANY, n=3)
    a.update(change)
    return L.lib().subspec_kv_page_bounds(a["pool"], a["bounds"], a["dtype"], a["pages"], a["page_len"], a["heads"], a["D"], a["slots"], a["n"], None)


@pytest.mark.parametrize("change,code", [(dict(pool=None), -1), (dict(bounds=None), -1), (dict(slots=None), -1), (dict(dtype=L.F32), -1), (dict(D=96), -4),
                                         (dict(page_len=24), -1), (dict(page_len=0), -1), (dict(pages=0), -1), (dict(heads=0), -1), (dict(n=-1), -1),
                                         (dict(pool=ANY + 2), -1), (dict(bounds=ANY + 8), -1)])
def test_bounds_refuses(change, code):
    assert _bounds(**change) == code and b"kv_page_bounds" in L.lib().subspec_last_error()


def test_no_slots_launch_nothing():
    assert _bounds(n=0, pool=None, bounds=None, slots=None) == 0


def _select(**change):
    a = dict(q=ANY, qs=512, bounds=ANY, dtype=L.BF16, pages=4, page_len=16, max_blocks=4, stride=4, seq=ANY, batch=2, n=4, hq=4, hkv=2, D=128, kv=64, keep=2,
             recent=1, out=ANY, ws=ANY, ws_bytes=1 << 20)
    a.update(change)
    return L.lib().subspec_select_blocks(a["q"], a["qs"], 128, a["bounds"], a["dtype"], a["pages"], a["page_len"], ANY, a["max_blocks"], a["stride"], a["seq"],
                                         ANY, a["batch"], a["n"], a["hq"], a["hkv"], a["D"], a["kv"], a["keep"], a["recent"], a["out"], a["ws"],
                                         a["ws_bytes"], None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(bounds=None), -1), (dict(seq=None), -1), (dict(out=None), -1), (dict(q=ANY + 2), -1), (dict(qs=513), -1), (dict(qs=-8), -1),
    (dict(dtype=L.F32), -1), (dict(D=80), -4), (dict(page_len=3), -1), (dict(stride=3), -1), (dict(batch=0), -4), (dict(batch=L.MAX_BATCH + 1), -4),
    (dict(n=-1), -4), (dict(n=(1 << 20) + 1), -4), (dict(hq=5), -1), (dict(hkv=0), -1), (dict(kv=-1), -1), (dict(kv=(1 << 30) + 1), -1), (dict(keep=0), -1),
    (dict(recent=0), -1), (dict(recent=3), -1), (dict(keep=(1 << 17) + 1), -1), (dict(page_len=1, max_blocks=1 << 18, stride=1 << 18, kv=1 << 18), -4),
    (dict(ws=None), -2), (dict(ws_bytes=300), -2), (dict(ws=ANY + 8), -1)])
def test_select_refuses(change, code):
    assert _select(**change) == code and b"select_blocks" in L.lib().subspec_last_error()


def test_no_tokens_select_nothing():
    assert _select(n=0, q=None, out=None) == 0


def _attend(**change):
    a = dict(q=ANY, qs=512, pool=ANY, dtype=L.BF16, pages=4, page_len=16, max_blocks=4, stride=4, blocks=ANY, keep=64, batch=2, n=4, hq=4, hkv=2, D=128,
             scale=0.1, out=ANY, ws=ANY, ws_bytes=1 << 24)
    a.update(change)
    return L.lib().subspec_block_attention(a["q"], a["qs"], 128, a["pool"], a["dtype"], a["pages"], a["page_len"], ANY, a["max_blocks"], a["stride"],
                                           a["blocks"], a["keep"], ANY, ANY, a["batch"], a["n"], a["hq"], a["hkv"], a["D"], a["scale"], a["out"], a["ws"],
                                           a["ws_bytes"], None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(pool=None), -1), (dict(blocks=None), -1), (dict(out=None), -1), (dict(out=ANY + 4), -1), (dict(qs=4), -1), (dict(dtype=L.F32), -1),
    (dict(D=256), -4), (dict(pages=0), -1), (dict(stride=0), -1), (dict(batch=0), -4), (dict(n=-1), -4), (dict(hq=130, hkv=2), -4), (dict(hq=3), -1),
    (dict(keep=0), -4), (dict(keep=1 << 18), -4), (dict(keep=1 << 11, page_len=1 << 20), -4), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1),
    (dict(scale=float("inf")), -1), (dict(ws=None), -2), (dict(ws_bytes=512), -2), (dict(ws=ANY + 8), -1)])
def test_attention_refuses(change, code):
    assert _attend(**change) == code and b"block_attention" in L.lib().subspec_last_error()


def test_no_tokens_attend_to_nothing():
    assert _attend(n=0, q=None, out=None) == 0


def _verify(**change):
    a = dict(logits=ANY, dtype=L.BF16, n=4, vocab=100, stride=100, drafts=ANY, starts=ANY, batch=2, u=ANY, q=ANY, q_dtype=L.F32, qs=100, ws=ANY, ws_bytes=1 << 20,
             tokens=ANY, accepted=ANY, top_p=1.0)
    a.update(change)
    return L.lib().subspec_verify_drafts(a["logits"], a["dtype"], a["n"], a["vocab"], a["stride"], a["drafts"], a["starts"], a["batch"], a["u"], ANY, a["q"],
                                         a["q_dtype"], a["qs"], None, 1.0, None, 0, None, a["top_p"], None, 0.0, a["ws"], a["ws_bytes"], a["tokens"], ANY,
                                         a["accepted"], None)


@pytest.mark.parametrize("change,code", [
    (dict(logits=None), -1), (dict(drafts=None), -1), (dict(starts=None), -1), (dict(u=None), -1), (dict(tokens=None), -1), (dict(accepted=None), -1),
    (dict(dtype=5), -1), (dict(q_dtype=5), -1), (dict(n=-1), -4), (dict(n=(1 << 20) + 1), -4), (dict(vocab=0), -4), (dict(batch=0), -4),
    (dict(batch=L.MAX_BATCH + 1), -4), (dict(vocab=(1 << 20) + 1, stride=1 << 21, qs=1 << 21), -4), (dict(stride=99), -1), (dict(qs=99), -1),
    (dict(logits=ANY + 1), -1), (dict(q=ANY + 2), -1), (dict(ws=None), -2), (dict(ws_bytes=300), -2), (dict(ws=ANY + 8), -1),
    (dict(top_p=0.5, ws_bytes=256), -2), (dict(n=0, starts=None), -1)])
def test_verify_refuses(change, code):
    assert _verify(**change) == code and b"verify_drafts" in L.lib().subspec_last_error()


@pytest.mark.parametrize("n,vocab", [(1 << 20, 1 << 20), (1 << 20, (1 << 17) - 1), (1 << 17, 1 << 20)])
def test_verify_refuses_more_slices_than_a_launch_has_threads_for(n, vocab):
    """A row without filters is looked at by a wavefront for every 2048 entries, and a launch has below 2^32 threads."""
    assert _verify(n=n, vocab=vocab, stride=vocab, qs=vocab, ws_bytes=1 << 60) == -4 and b"verify_drafts: too large" in L.lib().subspec_last_error()


def test_host_tensors_are_refused():
    q, pool, i32 = torch.zeros(1, 2, 64).bfloat16(), torch.zeros(2, 2, 4, 1, 64).bfloat16(), torch.zeros(1, dtype=torch.int32)
    bounds, table = torch.zeros(2, 1, 2, 64).bfloat16(), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(L.SubspecHipError):
        ops.kv_page_bounds_(bounds, pool, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(L.SubspecHipError):
        ops.select_blocks(q, bounds, table, i32, i32, 4, 1)
    with pytest.raises(L.SubspecHipError):
        ops.block_attention(q, pool, table, i32.view(1, 1, 1), i32, i32)
    with pytest.raises(L.SubspecHipError):
        ops.verify_drafts(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64), torch.tensor([0, 2], dtype=torch.int32), torch.zeros(2), torch.zeros(1))


def test_oracle_select_by_hand():
    bounds = torch.zeros(6, 1, 2, 2)
    for page, (low, high) in enumerate([(-1, 1), (-3, 0), (0, 2), (-2, 2), (0, 0), (9, 9)]):
        bounds[page, 0, 0], bounds[page, 0, 1] = low, high
    q = torch.tensor([[[1.0, -1.0], [1.0, 0.0]]])             # positive parts (2, 0), negative (0, -1): 2 high - low in all
    table = [[3, 0, 4, 1, 2, 5]]                              # scores 6, 3, 0, 3, 4
    assert ok.select(q, bounds, table, [0], [11], 2, 3) == [[[0, 4, 5]]]
    assert ok.select(q, bounds, table, [0], [9], 2, 3) == [[[0, 1, 4]]]              # two of 3: the lower block
    assert ok.select(q, bounds, table, [0], [11], 2, 3, recent=3) == [[[3, 4, 5]]]
    assert ok.select(q, bounds, table, [0], [3], 2, 3) == [[[0, 1, -1]]] and ok.select(q, bounds, table, [-1], [3], 2, 3) == [[[-1, -1, -1]]]
    assert ok.select(q, bounds, table, [0], [11], 2, 2, max_kv=5) == [[[0, 2]]]


def test_oracle_attention_by_hand():
    pool = torch.zeros(3, 2, 2, 1, 2, dtype=torch.float64)
    for j, page in enumerate([2, 0, 1]):
        for r in range(2):
            pool[page, 1, r] = float(1 << (2 * j + r))
    q = torch.zeros(2, 1, 2, dtype=torch.float64)             # equal scores: the average of the values seen
    out, _, _ = ok.attention(q, pool, [[2, 0, 1]], [[[0, 2]], [[1, -1]]], [0, 0], [4, 2])
    assert out[0, 0, 0].item() == pytest.approx((1 + 2 + 16) / 3) and out[1, 0, 0].item() == 4.0


def test_oracle_verify_by_hand():
    p = torch.tensor([[0.1, 0.4, 0.3, 0.2], [0.7, 0.1, 0.1, 0.1]])
    q = torch.tensor([[0.5, 0.5, 0.0, 0.0], [0.0, 0.0, 0.0, 0.0]])
    for u, v, want in ((0.79, 0.0, ([1, 0], 1)), (0.79, 0.75, ([1, 1], 1)), (0.81, 0.0, ([2, -1], 0)), (0.81, 0.65, ([3, -1], 0))):
        tokens, probs, accepted = ok.verify_drafts(torch.log(p), [3, 1], [0, 2], [u, 0.5], [v], q)
        assert (tokens, accepted[0]) == want and probs[0] == pytest.approx(float(p[0, tokens[0]]))
    tokens, _, accepted = ok.verify_drafts(torch.log(p), [3, 1], [0, 2], [0.5, 0.5], [0.2], None)
    assert accepted == [0] and tokens == [2, -1]              # 0.5 is not below 0.4; without entry 1 0.1, 0.3, 0.2 are left
    assert math.isclose(float(ok.target_probs(torch.log(p[0]), top_k=2)[1]), 4 / 7, rel_tol=1e-6)
