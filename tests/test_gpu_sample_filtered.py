"""GPU: tokens drawn after temperature, top-k, top-p and min-p against the definition in float64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import batch as ob
from subspec_amd import ops

DEV = "cuda:0"


def _check(logits, u, temperature, top_k, top_p, min_p, view=None):
    """Every row against the oracle; settings are lists, one value a row."""
    dev = lambda x, dtype: torch.tensor(x, dtype=dtype, device=DEV)
    settings = [dev(temperature, torch.float32), dev(top_k, torch.int32), dev(top_p, torch.float32), dev(min_p, torch.float32)]
    uniforms = dev(u, torch.float32)
    x = logits.to(DEV) if view is None else view(logits.to(DEV))
    tokens, probs = ops.sample_filtered(x, uniforms, *settings)
    t, k, p, m = (s.double().tolist() for s in settings)
    for r in range(logits.shape[0]):
        want, share = ob.sample(logits[r], float(uniforms[r]), t[r], int(k[r]), p[r], m[r])
        assert tokens[r].item() == want, (r, tokens[r].item(), want, t[r], k[r], p[r], m[r])
        # one rounding to fp32, and sums that are exact to 2^-42 for each entry
        assert abs(probs[r].item() - share) <= 2.0 ** -24 * share + logits.shape[1] * 2.0 ** -42, r
    return tokens, probs


def _settings(rows, g):
    pick = lambda values: [values[i] for i in torch.randint(0, len(values), (rows,), generator=g).tolist()]
    return dict(temperature=pick([0.0, 0.1, 0.7, 1.0, 1.0, 3.0]), top_k=pick([0, 0, 1, 2, 17, 50, 5000]),
                top_p=pick([1.0, 1.0, 0.95, 0.5, 0.01, 0.0]), min_p=pick([0.0, 0.0, 0.02, 0.3, 1.0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (5, 2), (40, 63), (40, 64), (30, 1000), (17, 4097), (9, 32000), (12, 50257), (6, 152064)])
def test_drawn_tokens(dtype, rows, vocab):
    print("sample", dtype, rows, vocab, flush=True)
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=g) * 2.5).to(dtype)
    u = torch.rand(rows, generator=g).tolist()
    _check(logits, u, **_settings(rows, g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [5000, 30001])
def test_many_equal_logits(dtype, vocab):
    """Ties go to the lowest index, also where more entries share a value than the kernel keeps in a list."""
    print("sample ties", dtype, vocab, flush=True)
    g = torch.Generator().manual_seed(5)
    flat = torch.zeros(6, vocab)
    few = torch.randint(0, 3, (6, vocab), generator=g).float() * 0.25 - 0.0
    few[:, ::7] = -0.0
    logits = torch.cat([flat, few]).to(dtype)
    _check(logits, [0.0, 0.3, 0.5, 0.77, 0.9999999, 0.5] * 2, [1.0, 1.0, 0.5, 2.0, 1.0, 0.0] * 2, [0, 7, 4500, 0, 0, 0] * 2,
           [1.0, 1.0, 0.9, 0.5, 1.0, 1.0] * 2, [0.0, 0.0, 0.0, 0.0, 1.0, 0.0] * 2)


def test_bounds_of_the_settings_and_of_the_numbers():
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(8, 777, generator=g)
    below_one = 1 - 2.0 ** -24
    _check(logits, [0.0, below_one, 0.0, below_one, 0.5, below_one, 0.0, 0.3], [1.0] * 8, [0, 0, 3, 3, 777, 778, 1, 0],
           [1.0, 1.0, 1.0, 1.0, 0.5, 1e-30, 1.0, below_one], [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 1.0])
    # scalars are the same setting for every row
    a = ops.sample_filtered(logits.to(DEV), torch.full((8,), 0.4, device=DEV), 0.8, 20, 0.9, 0.05)
    b = _check(logits, [0.4] * 8, [0.8] * 8, [20] * 8, [0.9] * 8, [0.05] * 8)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masked_and_infinite_logits(dtype):
    g = torch.Generator().manual_seed(3)
    V, low, inf, nan = 301, torch.finfo(dtype).min, math.inf, math.nan
    x = torch.randn(9, V, generator=g).to(dtype)
    x[0] = -inf
    x[1] = nan
    x[2, ::2] = -inf
    x[3, 1::3] = low
    x[4] = low
    x[5, 7] = x[5, 200] = inf
    x[6, ::2] = nan
    x[7] = torch.finfo(dtype).max
    x[7, 5:] = low
    x[8] = -inf
    x[8, 300] = low
    tokens, probs = _check(x, [0.6] * 9, [1.0] * 9, [0] * 9, [1.0] * 9, [0.0] * 9)
    assert tokens[:2].tolist() == [-1, -1] and probs[:2].tolist() == [0.0, 0.0]
    assert tokens[5].item() == 200 and probs[5].item() == 0.5 and tokens[8].item() == 300 and probs[8].item() == 1.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_a_wider_tensor(dtype):
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(5, 1001, generator=g).to(dtype)
    wide = torch.cat([torch.full((5, 3), 50.0).to(dtype), logits, torch.full((5, 6), 50.0).to(dtype)], 1)
    _check(logits, [0.1, 0.3, 0.5, 0.7, 0.9], [1.0] * 5, [0] * 5, [0.9] * 5, [0.0] * 5, view=lambda _: wide.to(DEV)[:, 3:1004])
    _check(logits, [0.1, 0.3, 0.5, 0.7, 0.9], [1.0] * 5, [0] * 5, [0.9] * 5, [0.0] * 5, view=lambda x: x.t().contiguous().t())
