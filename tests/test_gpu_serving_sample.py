"""Sampling against a plain 64-bit statement: settings, ties, masks, rows without a distribution."""
import math

import pytest
import torch

from qmoe_b200 import serving
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _check(logits, u, t=None, k=None, p=None, m=None):
    rows = logits.shape[0]
    got, logprob = serving.sample_tokens(logits, u, temperature=t, top_k=k, top_p=p, min_p=m, return_logprob=True)
    one = lambda x, d, i: d if x is None else (x[i].item() if isinstance(x, torch.Tensor) else  # noqa: E731
                                               (x if d == 0 and x is k else torch.tensor(x, dtype=torch.float32).item()))
    for i in range(rows):
        want, lp = ref.sample_row(logits[i].float().cpu(), one(t, 1.0, i), one(k, 0, i), one(p, 1.0, i), one(m, 0.0, i), u[i].item())
        assert int(got[i]) == want, (i, int(got[i]), want)
        if math.isnan(lp):
            assert math.isnan(float(logprob[i]))
        else:
            assert abs(float(logprob[i]) - lp) <= 2.0 ** -23 * max(1.0, abs(lp)), (i, float(logprob[i]), lp)
    return got


def _rows(rows, vocab, dtype, seed, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device=DEV) * spread).to(dtype)
    return x, torch.rand(rows, generator=g, device=DEV), g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1025, 5001])
def test_settings_together(vocab, dtype):
    x, u, g = _rows(12, vocab, dtype, vocab)
    x[::3, ::2] = -math.inf
    x[:, 0] = 0.25
    t = 0.3 + torch.rand(12, generator=g, device=DEV)
    k = torch.randint(0, 60, (12,), generator=g, device=DEV, dtype=torch.int32)
    p = torch.rand(12, generator=g, device=DEV)
    m = 0.2 * torch.rand(12, generator=g, device=DEV)
    _check(x, u)
    _check(x, u, t=t)
    _check(x, u, k=k)
    _check(x, u, p=p)
    _check(x, u, m=m)
    _check(x, u, t=t, k=k, p=p, m=m)
    _check(x, u, t=0.7, k=5, p=0.9, m=0.05)
    _check(x, u, t=0.0)


@pytest.mark.parametrize("rows,vocab", [(1, 32128), (3, 50001), (300, 700), (1, 262144)])
def test_large_rows(rows, vocab):
    x, u, _ = _rows(rows, vocab, torch.float32, vocab)
    for settings in (dict(), dict(k=50), dict(p=0.95), dict(t=0.6, k=1000, p=0.9, m=0.001)):
        some = slice(0, 4)
        got = serving.sample_tokens(x, u, temperature=settings.get("t"), top_k=settings.get("k"), top_p=settings.get("p"),
                                    min_p=settings.get("m"))
        for i in range(*some.indices(rows)):
            f = lambda name, d: d if name not in settings else torch.tensor(float(settings[name]), dtype=torch.float32).item()  # noqa: E731
            want, _ = ref.sample_row(x[i].cpu(), f("t", 1.0), settings.get("k", 0), f("p", 1.0), f("m", 0.0), u[i].item())
            assert int(got[i]) == want


def test_ties_go_to_the_lower_index():
    x = torch.zeros(6, 4096, device=DEV)
    u = torch.tensor([0.0, 0.25, 0.5, 0.999, 1 - 2.0 ** -24, 0.7], device=DEV)
    _check(x, u)                                              # 4096 equal shares: borders are hit exactly
    _check(x, u, k=100)
    _check(x, u, p=0.5)
    _check(x, u, k=64, p=0.5)
    _check(x, u, m=1.0)
    x[:, 1000:] = -1.0
    x[:, 17] = -0.0
    _check(x, u, k=1500, p=0.9)
    _check(x, u, t=0.0)
    x[:, 2000] = 5.0
    x[:, 3000] = 5.0
    _check(x, u, k=1)
    _check(x, u, k=2)
    _check(x, u, p=0.0)
    _check(x, u, t=0.0)


def test_all_equal_at_the_largest_vocabulary():
    x = torch.full((2, 262144), -3.5, device=DEV)             # the largest possible mass
    u = torch.tensor([0.5, 1 - 2.0 ** -24], device=DEV)
    got = serving.sample_tokens(x, u)
    assert got.tolist() == [131072, 262144 - 1]
    got = serving.sample_tokens(x, u, top_p=0.5)
    assert got.tolist() == [65536, 131071]


def test_masks():
    x, u, _ = _rows(5, 3000, torch.float32, 1)
    low = torch.finfo(torch.float32).min
    x[0, 1:] = -math.inf                                      # one token left
    x[1, :2999] = low
    x[2] = low                                                # every logit the lowest value: equal shares
    x[3, ::2] = low
    x[4, 100:] = -math.inf
    for settings in (dict(), dict(t=0.01), dict(k=7), dict(p=0.3), dict(m=0.5), dict(k=200, p=0.99)):
        got = _check(x, u, **settings)
        assert int(got[0]) == 0 and int(got[1]) == 2999
    half = x.clamp_min(-65504).half()
    half[0, 1:] = -math.inf
    _check(half, u, t=0.5)


def test_rows_without_a_distribution():
    x, u, _ = _rows(8, 500, torch.float32, 2)
    x[0, 77] = math.nan
    x[1, 3] = math.inf
    x[2] = -math.inf
    x[3, 499] = -math.nan
    t = torch.tensor([1.0, 1.0, 1.0, 0.0, -1.0, math.nan, math.inf, 1.0], device=DEV)
    got = _check(x, u, t=t)
    assert got[:7].tolist() == [-1] * 7 and int(got[7]) >= 0


def test_numbers_outside_their_range():
    x, u, _ = _rows(4, 500, torch.float32, 3)
    u[:] = torch.tensor([-1.0, 1.0, 2.0, math.nan], device=DEV)
    clamped = torch.tensor([0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0], device=DEV)
    got = serving.sample_tokens(x, u, top_k=20)
    last = [int(torch.topk(x[i], 20).indices.max()) for i in range(4)]        # what is kept, highest index
    first = [int(torch.topk(x[i], 20).indices.min()) for i in range(4)]
    assert got.tolist() == [first[0], last[1], last[2], first[3]]
    a = serving.sample_tokens(x, clamped)
    assert torch.equal(serving.sample_tokens(x, clamped, top_k=-5, top_p=1.5, min_p=-0.5), a)
    assert torch.equal(serving.sample_tokens(x, clamped, top_k=10 ** 9), a)
    best = x.argmax(1)
    assert torch.equal(serving.sample_tokens(x, clamped, min_p=7.0), best)
    assert torch.equal(serving.sample_tokens(x, clamped, top_p=-1.0), best)
    # very low and very high temperatures
    assert torch.equal(serving.sample_tokens(x, clamped, temperature=1e-38), best)
    _check(x, clamped, t=1e30)


def test_sampled_frequencies_follow_the_distribution():
    """The inverse distribution function at an even grid of numbers gives every token its share to
    within one grid step per border."""
    n = 4096
    row = torch.randn(1, 50, device=DEV)
    u = (torch.arange(n, device=DEV).float() + 0.5) / n
    got = serving.sample_tokens(row.expand(n, -1), u)
    share = torch.bincount(got, minlength=50).double() / n
    want = torch.softmax(row[0].double(), 0)
    assert float((share - want).abs().max()) <= 1.0 / n + 1e-9


def test_row_strides_streams_and_graphs():
    x, u, _ = _rows(6, 1001, torch.bfloat16, 4)
    want = serving.sample_tokens(x, u, top_p=0.9)
    wide = torch.zeros(6, 1500, device=DEV, dtype=torch.bfloat16)
    wide[:, 3:1004] = x
    assert torch.equal(serving.sample_tokens(wide[:, 3:1004], u, top_p=0.9), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = serving.sample_tokens(x, u, top_p=0.9)
    side = torch.cuda.Stream()
    for seed in range(3):
        u.copy_(torch.rand(6, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
            other = serving.sample_tokens(x, u, top_p=0.9)
        side.synchronize()
        assert torch.equal(held, other)
    assert serving.sample_tokens(x[:0], u[:0]).shape == (0,)
