"""What the batched entry points refuse, from the library's host code alone, and the oracle of the batch on small cases done by hand."""
import pytest
import torch

from oracle import batch as ob
from subspec_amd import _lib as L

ANY = 4096                                                   # a non-null, aligned address that no refused call touches


def _plan(**change):
    a = dict(batch=2, capacity=8, max_blocks=4, stride=4, page_len=16, n_tokens=8, kv=ANY, counts=ANY)
    a.update(change)
    return L.lib().subspec_paged_batch_plan(a["kv"], ANY, a["batch"], ANY, ANY, a["capacity"], ANY, a["max_blocks"], a["stride"], a["page_len"],
                                            a["n_tokens"], ANY, ANY, ANY, ANY, ANY, a["counts"], None)


@pytest.mark.parametrize("change,code", [
    (dict(kv=None), -1), (dict(counts=None), -1), (dict(batch=0), -4), (dict(batch=L.MAX_BATCH + 1), -4), (dict(page_len=12), -1),
    (dict(page_len=0), -1), (dict(max_blocks=0), -1), (dict(stride=3), -1), (dict(n_tokens=-1), -1), (dict(capacity=-1), -1)])
def test_plan_refuses(change, code):
    assert _plan(**change) == code and b"paged_batch_plan" in L.lib().subspec_last_error()


def _append(**change):
    a = dict(k=ANY, dtype=L.BF16, pages=4, page_len=16, heads=2, D=64, n=3, stride=128, slots=ANY)
    a.update(change)
    return L.lib().subspec_kv_append_paged(a["k"], a["stride"], 64, ANY, 128, 64, ANY, a["dtype"], a["pages"], a["page_len"], a["heads"], a["D"],
                                           a["slots"], a["n"], None)


@pytest.mark.parametrize("change", [dict(k=None), dict(slots=None), dict(dtype=9), dict(pages=0), dict(page_len=24), dict(heads=0), dict(D=0),
                                    dict(n=-1), dict(stride=-128), dict(k=ANY + 1)])
def test_append_refuses(change):
    assert _append(**change) == -1 and b"kv_append_paged" in L.lib().subspec_last_error()


def test_nothing_to_append_launches_nothing():
    assert _append(n=0, k=None, slots=None) == 0


def _attention(**change):
    a = dict(q=ANY, qs=512, pages=4, page_len=16, max_blocks=4, stride=4, dtype=L.BF16, batch=2, n=4, hq=4, hkv=2, D=128, new=2, kv=64,
             window=0, sinks=0, scale=0.1, ws=None, ws_bytes=0, out=ANY)
    a.update(change)
    return L.lib().subspec_paged_attention(a["q"], a["qs"], 128, ANY, a["pages"], a["page_len"], ANY, a["max_blocks"], a["stride"], ANY, ANY, a["out"],
                                           a["dtype"], a["batch"], a["n"], a["hq"], a["hkv"], a["D"], a["new"], a["kv"], a["window"], a["sinks"],
                                           a["scale"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(q=ANY + 2), -1), (dict(qs=513), -1), (dict(dtype=L.F32), -1), (dict(D=96), -4), (dict(batch=0), -4),
    (dict(hq=5), -1), (dict(hkv=0), -1), (dict(page_len=3), -1), (dict(stride=2), -1), (dict(n=-1), -1), (dict(new=-1), -1), (dict(kv=-1), -1),
    (dict(window=-1), -1), (dict(sinks=3), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(pages=0), -1)])
def test_attention_refuses(change, code):
    assert _attention(**change) == code and b"paged_attention" in L.lib().subspec_last_error()


def test_attention_over_nothing_launches_nothing():
    assert _attention(n=0, q=None) == 0 and _attention(new=0) == 0 and _attention(kv=0) == 0


def _sample(**change):
    a = dict(logits=ANY, dtype=L.BF16, rows=2, vocab=100, stride=100, u=ANY, ws=None)
    a.update(change)
    return L.lib().subspec_sample_filtered(a["logits"], a["dtype"], a["rows"], a["vocab"], a["stride"], a["u"], None, 1.0, None, 0, None, 1.0, None,
                                           0.0, a["ws"], 0, ANY, ANY, None)


@pytest.mark.parametrize("change,code", [(dict(logits=None), -1), (dict(u=None), -1), (dict(dtype=5), -1), (dict(vocab=0), -4),
                                         (dict(vocab=(1 << 20) + 1, stride=1 << 21), -4), (dict(rows=-1), -4), (dict(stride=99), -1),
                                         (dict(logits=ANY + 1), -1), (dict(vocab=50000, stride=50000), -2), (dict(ws=ANY + 8), -1)])
def test_sample_refuses(change, code):
    assert _sample(**change) == code and b"sample_filtered" in L.lib().subspec_last_error()


def test_oracle_plan_by_hand():
    got = ob.plan([3, 0, 4], [2, 0, 1], [9, 8, 7], [[5, -1], [-1, -1], [6, -1]], 4, 5)
    assert got["table"] == [[5, 7], [-1, -1], [6, 8]] and got["counts"] == [3, 2, 1, 0]
    assert got["slots"] == [5 * 4 + 3, 7 * 4, 8 * 4, -1, -1] and got["sequences"] == [0, 0, 2, -1, -1]
    assert got["positions"] == [3, 4, 4, 0, 0] and got["query_starts"] == [0, 2, 2, 3] and got["kv_lens"] == [5, 0, 5]


def test_oracle_sample_by_hand():
    x = torch.log(torch.tensor([0.1, 0.4, 0.3, 0.2], dtype=torch.float64))
    assert [ob.sample(x, u)[0] for u in (0.0, 0.39, 0.41, 0.71, 0.91)] == [1, 1, 2, 3, 0]
    assert ob.sample(x, 0.99, top_k=2)[0] == 2 and ob.sample(x, 0.99, top_p=0.35)[0] == 1 and ob.sample(x, 0.99, min_p=0.6)[0] == 2
    assert abs(ob.sample(x, 0.5, top_k=2)[1] - 0.4 / 0.7) < 1e-12 or abs(ob.sample(x, 0.5, top_k=2)[1] - 0.3 / 0.7) < 1e-12


def test_oracle_attention_window_by_hand():
    pool = torch.zeros(3, 2, 2, 1, 2, dtype=torch.float64)
    table = [[2, 0, 1]]
    for j in range(6):                                        # equal scores: the average of the values seen
        pool[table[0][j // 2], 1, j % 2] = float(1 << j)
    q = torch.zeros(2, 1, 2, dtype=torch.float64)
    out, _, _ = ob.attention(q, pool, table, [0, 2], [6], window=2, sinks=1)
    assert out[0, 0, 0].item() == pytest.approx((1 + 8 + 16) / 3) and out[1, 0, 0].item() == pytest.approx((1 + 16 + 32) / 3)


def test_a_batch_refuses_before_anything_is_launched():
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    pool = KvCachePool(max_pages=8, num_layers=1, num_heads=2, head_dim=64, page_len=4, dtype=torch.bfloat16, device="cpu")
    batch = KvBatch(pool, 2, 40, num_pages=5)
    assert int(pool.num_free_pages()) == 3 and batch.block_table.shape == (2, 10)
    for bad in ([1], [1, -1], [41, 0], [12, 9]):              # a place missing, below zero, longer than the batch allows, six pages
        with pytest.raises(ValueError):
            batch.step(bad)
    with pytest.raises(ValueError):
        batch.step([3, 3], n_tokens=5)
    assert batch.lens == [0, 0] and batch.num_free == 5
    with pytest.raises(L.SubspecHipError):                     # the device work itself has no CPU fallback
        batch.step([3, 3])
    assert batch.lens == [0, 0] and batch.num_free == 5
    batch.close()
    assert int(pool.num_free_pages()) == 8
    for places in (0, L.MAX_BATCH + 1):
        with pytest.raises(ValueError):
            KvBatch(pool, places, 40)
    assert int(pool.num_free_pages()) == 8


@pytest.mark.parametrize("hq,hkv,D", [(28, 4, 128), (32, 32, 128), (14, 2, 64), (64, 1, 128)])
def test_attention_workspace_holds_a_gigabyte_of_partials_at_most(hq, hkv, D):
    size = L.lib().subspec_paged_attention_workspace
    for batch, tokens, new in [(1, 1, 1), (64, 64, 1), (4096, 4096, 1), (1, 4096, 4096), (4096, 60000, 3000), (300, 5000, 40)]:
        for kv in (1, 100, 4096, 131072, 1 << 20):            # (those of short calls and of long ones: a gigabyte each, and the sums' share)
            assert 256 <= size(batch, tokens, hq, hkv, D, new, kv, 0, 0) <= (2 << 30) * 1.02
    assert size(1, 1, hq, hkv, D, 1, 64, 0, 0) == 256       # one chunk: nothing to keep


@pytest.mark.parametrize("tokens,new", [(1, 1), (300, 300)])
def test_a_window_or_sinks_beyond_any_sequence_are_planned_like_a_large_one(tokens, new):
    """The largest int64, as a caller without a window may write it: the same chunks and workspace as any window that no sequence fills."""
    size = lambda window, sinks, kv=32768: L.lib().subspec_paged_attention_workspace(1, tokens, 28, 4, 128, new, kv, window, sinks)
    for huge in ((1 << 31) - 1, 1 << 31, 1 << 40, (1 << 62) - 1, (1 << 63) - 200, (1 << 63) - 1):
        assert size(huge, 0) == size(1 << 30, 0) == size(0, 0) > 256
        assert size(1024, huge) == size(1024, 1 << 30) == size(0, 0)
        assert size(huge, huge) == size(0, 0)
        assert _attention(n=tokens, new=new, hq=28, hkv=4, qs=28 * 128, kv=32768, window=huge, sinks=huge) == -2       # the same workspace is asked for
    for kv in ((1 << 30) + 1, (1 << 63) - 1):                   # (the call refuses these rows: nothing to keep)
        assert size(0, 0, kv) == 256 and _attention(kv=kv) == -1


def _cpu_batch(places=2, pages=8):
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    pool = KvCachePool(max_pages=pages, num_layers=1, num_heads=2, head_dim=64, page_len=4, dtype=torch.bfloat16, device="cpu")
    return pool, KvBatch(pool, places, 40)


def test_nothing_is_appended_without_a_step_or_after_close(monkeypatch):
    """The pages of a closed batch belong to whoever asks the pool next: the last plan's slots must not reach an append."""
    from subspec_amd import ops
    calls = []
    monkeypatch.setattr(ops, "kv_append_paged_", lambda *a, **k: calls.append("append"))
    monkeypatch.setattr(ops, "paged_attention", lambda *a, **k: calls.append("attention"))
    pool, batch = _cpu_batch()
    k, q = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 4, 64, dtype=torch.bfloat16)

    def refused():
        with pytest.raises(ValueError, match="step"):
            batch.append(0, k, k)
        with pytest.raises(ValueError, match="step"):
            batch.attention(0, q)

    refused()
    batch.plan = dict(slots=torch.arange(2), query_starts=torch.tensor([0, 1, 2], dtype=torch.int32), kv_lens=torch.tensor([1, 1], dtype=torch.int32))
    batch.append(0, k, k)
    batch.attention(0, q)
    assert calls == ["append", "attention"]
    batch.close()
    assert int(pool.num_free_pages()) == 8
    refused()
    batch.close()                                              # a second time does nothing
    assert int(pool.num_free_pages()) == 8 and calls == ["append", "attention"]


def test_a_release_between_layers_leaves_the_step_its_lengths(monkeypatch):
    from subspec_amd import ops
    seen = []
    monkeypatch.setattr(ops, "paged_attention", lambda q, pool, table, starts, lens, *a, **k: seen.append((starts.tolist(), lens.tolist())))
    pool, batch = _cpu_batch()
    lens = torch.tensor([9, 5], dtype=torch.int32)
    batch.plan = dict(slots=torch.arange(3), query_starts=torch.tensor([0, 2, 3], dtype=torch.int32), kv_lens=lens)
    batch.kv_lens, batch.lens, batch.num_free = lens, [9, 5], 3
    batch.attention(0, torch.zeros(3, 4, 64))
    batch.release(0)
    batch.attention(0, torch.zeros(3, 4, 64))
    assert seen == [([0, 2, 3], [9, 5])] * 2 and batch.kv_lens.tolist() == [0, 5] and batch.lens == [0, 5]


def test_a_sequence_of_more_rows_than_32_bits_number_is_refused():
    """(token, query head of a KV head) rows: 2^30 tokens of 4 heads a KV head, though q may be an expanded view of a few."""
    assert _attention(n=1 << 30, new=1 << 30, hq=8, hkv=2, kv=64) == -4 and b"tokens of 4 query heads" in L.lib().subspec_last_error()
    assert _attention(n=1 << 30, new=(1 << 29) - 65, hq=8, hkv=2, kv=640) == -2                        # (the workspace is looked at next)
    assert _attention(n=1 << 30, new=1 << 29, hq=8, hkv=2, kv=640) == -4


def test_a_batch_that_cannot_be_made_takes_no_pages():
    """A table that does not fit into memory, a length or a number of pages below zero (which as the end of a slice means all but some)."""
    from subspec_amd.paged_cache import KvBatch, KvCachePool
    pool = KvCachePool(max_pages=8, num_layers=1, num_heads=2, head_dim=64, page_len=4, dtype=torch.bfloat16, device="cpu")
    for bad in (dict(max_len=1 << 58), dict(max_len=-1), dict(max_len=40, num_pages=-1)):
        with pytest.raises((ValueError, RuntimeError)):
            KvBatch(pool, 2, **bad)
        assert int(pool.num_free_pages()) == 8
