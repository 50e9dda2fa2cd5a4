"""Prompt attention against a plain 64-bit statement: head layouts, lengths, strides, masks."""
import math
import random

import pytest
import torch

from qmoe_b200 import serving
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _cu(lens, first=0):
    c = [first]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=DEV)


def _case(lens_q, lens_k, heads, kv_heads, d, dtype, seed=0, small=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda n, h, s: (torch.randn(n, h, d, generator=g, device=DEV) * s).to(dtype)  # noqa: E731
    return mk(sum(lens_q), heads, small), mk(sum(lens_k), kv_heads, small), mk(sum(lens_k), kv_heads, 1.0)


def _check(got, q, k, v, lens_q, lens_k, scale, bias=None, exact_fn=ref.attention_fast):
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        out, size = exact_fn(q[a:a + n].double(), k[b:b + m].double(), v[b:b + m].double(), scale, bias, m - n)
        err = (got[a:a + n].double() - out).abs()
        bound = ref.attention_bound(out, size, q.dtype)
        worst = float((err - bound).max()) if n else 0.0
        assert worst <= 0, (n, m, worst, float(err.max()))
        a, b = a + n, b + m


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 65), (8, 2, 128), (3, 1, 64), (2, 2, 1), (6, 3, 40), (2, 1, 127),
                                              (2, 2, 200), (1, 1, 256), (4, 2, 80), (2, 1, 16)])
def test_packed_prompts(heads, kv_heads, d, dtype):
    lens = [1, 130, 0, 257, 64, 2, 33]
    q, k, v = _case(lens, lens, heads, kv_heads, d, dtype)
    got = serving.prompt_attention(q, k, v, _cu(lens))
    _check(got, q, k, v, lens, lens, d ** -0.5)


@pytest.mark.parametrize("n", [1, 2, 127, 128, 129, 255, 256, 257, 511, 640, 1000])
def test_lengths_at_tile_edges(n):
    q, k, v = _case([n], [n], 2, 1, 64, torch.bfloat16, seed=n)
    _check(serving.prompt_attention(q, k, v, _cu([n])), q, k, v, [n], [n], 0.125)


@pytest.mark.parametrize("d", [64, 65, 128])
def test_earlier_keys_and_queries_that_see_nothing(d):
    lens_q, lens_k = [5, 100, 300, 1, 7, 4], [200, 100, 450, 999, 3, 0]       # the last two: queries before any key
    q, k, v = _case(lens_q, lens_k, 4, 2, d, torch.bfloat16, seed=2)
    got = serving.prompt_attention(q, k, v, _cu(lens_q), _cu(lens_k))
    _check(got, q, k, v, lens_q, lens_k, d ** -0.5)
    assert bool((got[-4:] == 0).all()) and bool((got[-11:-7] == 0).all())


@pytest.mark.parametrize("n_dist", [1, 2, 33, 128, 700])
def test_relative_bias_unscaled(n_dist):
    lens_q, lens_k = [300, 17, 129], [300, 400, 700]
    q, k, v = _case(lens_q, lens_k, 4, 4, 64, torch.float16, seed=3, small=64 ** -0.25)
    bias = torch.randn(4, n_dist, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)) * 2
    got = serving.prompt_attention(q, k, v, _cu(lens_q), _cu(lens_k), scale=1.0, rel_bias=bias)
    _check(got, q, k, v, lens_q, lens_k, 1.0, bias)


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_bias_that_masks(low):
    """Distances of 40 and more are masked (a window), or everything is."""
    lens = [200, 1, 90]
    q, k, v = _case(lens, lens, 2, 1, 64, torch.bfloat16, seed=5)
    bias = torch.zeros(2, 41, device=DEV)
    bias[:, 40] = low
    got = serving.prompt_attention(q, k, v, _cu(lens), rel_bias=bias)
    _check(got, q, k, v, lens, lens, 0.125, bias, ref.attention)
    got = serving.prompt_attention(q, k, v, _cu(lens), rel_bias=torch.full((2, 1), low, device=DEV))
    if low == -math.inf:
        assert bool((got == 0).all())
    else:                                   # the lowest finite value swallows every score: plain averages
        _check(got, q, k, v, lens, lens, 0.125, torch.full((2, 1), low, device=DEV), ref.attention)


def test_strides_of_a_fused_projection_and_odd_offsets():
    lens = [70, 200]
    g = torch.Generator(device=DEV).manual_seed(6)
    for d in (64, 65, 128):
        rows = torch.randn(270, 3, 4, d, generator=g, device=DEV).bfloat16()
        q, k, v = rows[:, 0], rows[:, 1], rows[:, 2]
        want = serving.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), _cu(lens))
        assert torch.equal(serving.prompt_attention(q, k, v, _cu(lens)), want)
        # head-major storage, as a cache keeps it
        kt, vt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
        assert torch.equal(serving.prompt_attention(q, kt, vt, _cu(lens)), want)
        # tensors that begin in the middle of a 16-byte unit, rows of odd pitch
        wide = torch.zeros(270, 4, d + 3, device=DEV).bfloat16()
        odd = []
        for t in (q, k, v):
            w = wide.clone()
            w[:, :, 1:d + 1] = t
            odd.append(w[:, :, 1:d + 1])
        out = wide.clone()[:, :, 2:d + 2]
        assert torch.equal(serving.prompt_attention(*odd, _cu(lens), out=out), want)
        # one key head broadcast to all query heads by a stride of 0
        one = serving.prompt_attention(q, k[:, :1].expand(-1, 4, -1), v[:, :1].expand(-1, 4, -1), _cu(lens))
        assert torch.equal(one, serving.prompt_attention(q, k[:, :1], v[:, :1], _cu(lens)))


@pytest.mark.parametrize("d", [64, 65])
def test_rows_behind_the_last_sequence_and_before_the_first(d):
    lens = [40, 133]
    q, k, v = _case([5 + 173 + 90], [5 + 173 + 90], 2, 2, d, torch.bfloat16, seed=7)
    for t in (q, k, v):                                   # rows of nobody hold NaN
        t[:5] = math.nan
        t[178:] = math.nan
    out = torch.full_like(q, 7.0)
    serving.prompt_attention(q, k, v, _cu(lens, 5), out=out)
    assert bool((out[:5] == 7).all()) and bool((out[178:] == 7).all())
    _check(out[5:178], q[5:178], k[5:178], v[5:178], lens, lens, d ** -0.5)


@pytest.mark.parametrize("d", [64, 65, 128])
@pytest.mark.parametrize("what", ["k", "v", "kv"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_non_finite_later_keys_do_not_reach_earlier_queries(d, what, value):
    n, at = 300, 201
    q, k, v = _case([n, 50], [n, 50], 2, 1, d, torch.bfloat16, seed=8)
    clean = serving.prompt_attention(q, k, v, _cu([n, 50]))
    if "k" in what:
        k[at] = value
    if "v" in what:
        v[at] = value
    got = serving.prompt_attention(q, k, v, _cu([n, 50]))
    assert torch.equal(got[n:], clean[n:])                # another sequence
    k2, v2 = k.clone(), v.clone()
    k2[at:n], v2[at:n] = 0, 0
    _check(got[:at], q[:at], k2[:at], v2[:at], [at], [at], d ** -0.5)
    if what != "k" or not math.isinf(value):              # an infinite key may also get weight 0
        assert not bool(torch.isfinite(got[at:n]).any())


def test_large_scores_and_constant_rows():
    q, k, v = _case([260], [260], 2, 2, 64, torch.bfloat16, seed=9)
    got = serving.prompt_attention(q * 100, k * 100, v, _cu([260]))          # weights are nearly one-hot
    assert bool(torch.isfinite(got).all())
    # the score's own error grows with it: 2^-24 * |s| on the exponent, |s| up to 8e4, for near ties
    out, _ = ref.attention_fast((q * 100).double(), (k * 100).double(), v.double(), 0.125, None, 0)
    assert float(((got.double() - out).abs() > 0.05).float().mean()) < 1e-3
    got = serving.prompt_attention(torch.zeros_like(q), k, v, _cu([260]))     # plain averages
    _check(got, torch.zeros_like(q), k, v, [260], [260], 0.125)


def test_many_short_sequences():
    lens = [(7 * i) % 19 for i in range(700)]
    q, k, v = _case(lens, lens, 2, 1, 64, torch.bfloat16, seed=10)
    got = serving.prompt_attention(q, k, v, _cu(lens))
    whole = torch.cat([ref.attention_fast(q[a:a + n].double(), k[a:a + n].double(), v[a:a + n].double(), 0.125, None, 0)[0]
                       for a, n in zip(_cu(lens).tolist(), lens)])
    assert float((got.double() - whole).abs().max()) < 2.0 ** -5             # |v| < 6, weights and output at 2^-8 each


def test_empty_batches():
    q, k, v = _case([4], [4], 2, 1, 64, torch.bfloat16)
    out = torch.full_like(q, 3.0)
    assert torch.equal(serving.prompt_attention(q, k, v, _cu([]), out=out), torch.full_like(q, 3.0))
    assert torch.equal(serving.prompt_attention(q, k, v, _cu([0, 0]), out=out), torch.full_like(q, 3.0))
    assert serving.prompt_attention(q[:0], k[:0], v[:0], _cu([0])).shape == (0, 2, 64)
    got = serving.prompt_attention(q, k[:0], v[:0], _cu([4]), _cu([0]))
    assert bool((got == 0).all())


def test_offsets_outside_the_tensors_are_clamped():
    q, k, v = _case([64], [64], 2, 1, 64, torch.bfloat16, seed=11)
    want = serving.prompt_attention(q, k, v, _cu([64]))
    bad = torch.tensor([-50, 1 << 30], dtype=torch.int32, device=DEV)
    assert torch.equal(serving.prompt_attention(q, k, v, bad), want)
    falling = torch.tensor([64, 0], dtype=torch.int32, device=DEV)             # no rows at all
    out = torch.full_like(q, 2.0)
    assert torch.equal(serving.prompt_attention(q, k, v, falling, out=out), torch.full_like(q, 2.0))


def test_same_bits_again_on_another_stream_and_in_a_replayed_graph():
    lens = [300, 5, 190]
    q, k, v = _case(lens, lens, 8, 2, 128, torch.bfloat16, seed=12)
    cu = _cu(lens)
    want = serving.prompt_attention(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = serving.prompt_attention(q, k, v, cu)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = serving.prompt_attention(q, k, v, cu)
    q2, _, _ = _case(lens, lens, 8, 2, 128, torch.bfloat16, seed=13)
    want2 = serving.prompt_attention(q2, k, v, cu)
    for src, w in ((q2.clone(), want2), (q.clone(), want)):
        q.copy_(src)
        graph.replay()
        assert torch.equal(held, w)


@pytest.mark.parametrize("d", [64, 128])
def test_many_items_of_every_kind(d):
    """More pieces of work than the GPU has multiprocessors, pieces without a key between long ones, and rows that
    are computed again: one CTA works through all kinds."""
    r = random.Random(d)
    lens_q = [r.choice([0, 1, 3, 40, 128, 200, 300, 600]) for _ in range(150)]
    lens_k = [max(0, n + r.choice([-n, -200, 0, 0, 0, 1, 130, 700])) for n in lens_q]
    q, k, v = _case(lens_q, lens_k, 4, 2, d, torch.bfloat16, seed=14)
    got = serving.prompt_attention(q, k, v, _cu(lens_q), _cu(lens_k))
    _check(got, q, k, v, lens_q, lens_k, d ** -0.5)
    # the last key of every fifth sequence is infinite: only the sequence's last query sees it
    first, rows = 0, []
    spoiled = v.clone()
    for i, m in enumerate(lens_k):
        if i % 5 == 0 and m > 0 and lens_q[i] > 0:
            spoiled[first + m - 1] = math.inf
            rows.append(sum(lens_q[:i + 1]) - 1)
        first += m
    again = serving.prompt_attention(q, k, spoiled, _cu(lens_q), _cu(lens_k))
    keep = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
    keep[rows] = False
    _check(again.where(keep[:, None, None], got), q, k, v, lens_q, lens_k, d ** -0.5)
    assert not bool(again[~keep].isfinite().any())


@pytest.mark.parametrize("d", [64, 65])
def test_key_rows_far_apart(d):
    """Strides that carry the last rows more than 2^32 values behind the first."""
    n, far = 40, (1 << 27) + 8
    pool = torch.empty(far * (n - 1) + 2 * d, dtype=torch.bfloat16, device=DEV)
    q, k0, v0 = _case([n], [n], 2, 1, d, torch.bfloat16, seed=15)
    k, v = (pool[i * d:].as_strided((n, 1, d), (far, d, 1)) for i in range(2))
    k.copy_(k0)
    v.copy_(v0)
    _check(serving.prompt_attention(q, k, v, _cu([n])), q, k0, v0, [n], [n], d ** -0.5)


def test_output_refusals():
    q, k, v = _case([8], [8], 2, 1, 64, torch.bfloat16)
    for bad in (q, k.expand(8, 2, 64), torch.empty(1, 2, 64, dtype=q.dtype, device=DEV).expand(8, 2, 64), q.float(), q[:4]):
        with pytest.raises((ValueError, TypeError)):
            serving.prompt_attention(q, k, v, _cu([8]), out=bad)
    with pytest.raises(ValueError):
        serving.prompt_attention(q, k, v, _cu([8]), scale=-0.5)


@pytest.mark.parametrize("heads,kv_heads,d,dtype", [(8, 1, 128, torch.bfloat16), (3, 3, 65, torch.float16), (2, 1, 40, torch.bfloat16),
                                                    (4, 4, 64, torch.float16), (1, 1, 127, torch.bfloat16)])
@pytest.mark.parametrize("lens_q,lens_k", [([1], [5000]), ([130], [2100]), ([300], [1204]), ([600], [600]),
                                           ([40, 0, 3], [3000, 700, 2]), ([129, 200], [4000, 90])])
def test_few_queries_of_many_keys(lens_q, lens_k, heads, kv_heads, d, dtype):
    """Calls whose keys are split among CTAs; some parts hold no key of a sequence."""
    q, k, v = _case(lens_q, lens_k, heads, kv_heads, d, dtype, seed=16)
    _check(serving.prompt_attention(q, k, v, _cu(lens_q), _cu(lens_k)), q, k, v, lens_q, lens_k, d ** -0.5)


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_parts_that_a_bias_masks(low):
    """All keys but the nearest 100 are masked (whole parts of them), or all but the far ones."""
    n, m, heads, d = 70, 3100, 2, 64
    q, k, v = _case([n], [m], heads, 1, d, torch.bfloat16, seed=17)
    g = torch.Generator(device=DEV).manual_seed(18)
    bias = torch.randn(heads, 400, generator=g, device=DEV)
    bias[0, 100:] = low
    bias[1, :399] = low
    got = serving.prompt_attention(q, k, v, _cu([n]), _cu([m]), scale=1.0, rel_bias=bias)
    _check(got, q, k, v, [n], [m], 1.0, bias, exact_fn=ref.attention)
    nothing = torch.full((heads, 3), -math.inf, device=DEV)
    assert bool((serving.prompt_attention(q, k, v, _cu([n]), _cu([m]), rel_bias=nothing) == 0).all())


def test_parts_with_values_that_are_not_finite():
    n, m, heads, d = 200, 2500, 2, 128
    q, k, v = _case([n], [m], heads, 1, d, torch.bfloat16, seed=19)
    k[2400:] = math.nan                                      # seen by the last hundred queries only
    v[2450:] = math.inf
    got = serving.prompt_attention(q, k, v, _cu([n]), _cu([m]))
    _check(got[:100], q[:100], k[:2400], v[:2400], [100], [2400], d ** -0.5)
    assert bool(got[100:].isnan().all())


def test_split_calls_leave_other_rows_and_follow_replayed_offsets():
    heads, d, total = 2, 64, 150
    q, k, v = _case([total], [4000], heads, 2, d, torch.bfloat16, seed=20)
    wide = torch.full((total, heads, d + 9), 7.0, dtype=q.dtype, device=DEV)      # rows off 16-byte boundaries
    cu_q, cu_k = _cu([90], first=20), _cu([3500], first=300)
    graph = torch.cuda.CUDAGraph()
    serving.prompt_attention(q, k, v, cu_q, cu_k, out=wide[..., 3:3 + d])
    with torch.cuda.graph(graph):
        serving.prompt_attention(q, k, v, cu_q, cu_k, out=wide[..., 3:3 + d])
    for first_q, n, first_k, m in ((20, 90, 300, 3500), (0, 150, 0, 4000), (149, 1, 17, 130), (3, 5, 9, 0)):
        cu_q.copy_(_cu([n], first=first_q))
        cu_k.copy_(_cu([m], first=first_k))
        wide.fill_(7.0)
        graph.replay()
        got = wide[first_q:first_q + n, :, 3:3 + d]
        rows = slice(first_q, first_q + n), slice(first_k, first_k + m)
        _check(got, q[rows[0]], k[rows[1]], v[rows[1]], [n], [m], d ** -0.5)
        wide[first_q:first_q + n, :, 3:3 + d] = 7.0
        assert bool((wide == 7.0).all())


def test_split_calls_on_two_streams_at_once():
    q, k, v = _case([64], [6000], 2, 1, 64, torch.bfloat16, seed=21)
    cu_q, cu_k = _cu([64]), _cu([6000])
    want = serving.prompt_attention(q, k, v, cu_q, cu_k)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(serving.prompt_attention(q, k, v, cu_q, cu_k))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d,n,m,heads,n_dist", [(64, 400, 400, 2, 41), (65, 300, 300, 80, 41), (64, 70, 3100, 2, 41), (128, 2000, 2000, 40, 300),
                                                (200, 150, 150, 2, 41)])
def test_keys_that_a_bias_masks_may_hold_anything(d, n, m, heads, n_dist, value):
    """Keys and values outside a window, in the tiles, with split keys and row by row."""
    q, k, v = _case([n], [m], heads, 1, d, torch.bfloat16, seed=22)
    bias = torch.randn(heads, n_dist, generator=torch.Generator(device=DEV).manual_seed(23), device=DEV)
    bias[:, -1] = -math.inf
    spoiled = torch.zeros(m, dtype=torch.bool, device=DEV)
    at = max(0, m - n) + 7
    spoiled[[0, 5, at]] = True                                        # seen by queries up to n_dist - 2 positions on
    reach = at + n_dist - 1 - (m - n)                                 # the first query that sees none of them
    cu_q, cu_k = _cu([n]), _cu([m])
    clean = serving.prompt_attention(q, k.masked_fill(spoiled[:, None, None], 0), v, cu_q, cu_k, scale=d ** -0.5, rel_bias=bias)
    k[spoiled] = value
    got = serving.prompt_attention(q, k, v, cu_q, cu_k, scale=d ** -0.5, rel_bias=bias)
    assert 0 < reach < n and torch.equal(got[reach:], clean[reach:])
    v[spoiled] = value
    got = serving.prompt_attention(q, k, v, cu_q, cu_k, scale=d ** -0.5, rel_bias=bias)[reach:]
    some = torch.linspace(0, n - reach - 1, 12, device=DEV).long()
    k, v = (t.masked_fill(spoiled[:, None, None], 0) for t in (k, v))
    for i in some.tolist():
        _check(got[i:i + 1], q[reach + i:reach + i + 1], k[:m - n + reach + i + 1], v[:m - n + reach + i + 1], [1],
               [m - n + reach + i + 1], d ** -0.5, bias)


def _time(call):
    call()
    events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    events[0].record()
    call()
    events[1].record()
    torch.cuda.synchronize()
    return events[0].elapsed_time(events[1])


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("heads,n,m", [(32, 4096, 4096), (8, 256, 8192)])
def test_scores_that_are_not_finite_cost_no_time(heads, n, m, value):
    """A key that every query sees and whose scores are NaN, or +inf for some queries: NaN where a score is, at the
    speed of finite inputs (computed key by key, these calls would take hundreds of times as long)."""
    q, k, v = _case([n], [m], heads, heads // 4, 128, torch.bfloat16, seed=24)
    cu_q, cu_k = _cu([n]), _cu([m])
    call = lambda: serving.prompt_attention(q, k, v, cu_q, cu_k)  # noqa: E731
    clean, finite = call(), _time(call)
    k[0, :, 0] = value                                          # infinite scores of both signs
    got, spoiled = call(), _time(call)
    if math.isnan(value):
        bad = torch.ones(n, heads, dtype=torch.bool, device=DEV)
    else:
        bad = q[:, :, 0] > 0
        k[0] = 0
        k = k[1:].contiguous()                                  # -inf: as if the key were not there
        some = torch.nonzero(~bad & (torch.arange(n, device=DEV) % 97 == 40)[:, None])[:40]
        for i, a in some.tolist():
            seen = m - n + i
            _check(got[i:i + 1, a:a + 1], q[i:i + 1, a:a + 1], k[:seen, a // 4:a // 4 + 1], v[1:seen + 1, a // 4:a // 4 + 1], [1], [seen], 128 ** -0.5)
    assert bool(got[bad].isnan().all()) and not bool(got[~bad].isnan().any()) and bool(clean.isfinite().all())
    assert spoiled < 5 * finite + 0.5


@pytest.mark.parametrize("column", range(16))
@pytest.mark.parametrize("d", [64, 128])
def test_a_nan_key_in_every_column_of_a_tile(column, d):
    """Whichever way a key's weight is computed, and however many of them there are."""
    n = 400
    q, k, v = _case([n], [n], 2, 2, d, torch.bfloat16, seed=25)
    clean = serving.prompt_attention(q, k, v, _cu([n]))
    k[column, 0] = math.nan
    k[column::16, 1] = math.nan
    got = serving.prompt_attention(q, k, v, _cu([n]))
    assert torch.equal(got[:column], clean[:column]) and bool(got[column:].isnan().all())


def test_rows_computed_again_stay_within_reason():
    """An infinite value that every query sees, a key that half of them see, and a masked one: every row is computed
    again.  (One key at a time this call takes 70 ms.)"""
    n, heads = 2048, 32
    q, k, v = _case([n], [n], heads, 8, 128, torch.bfloat16, seed=26)
    v[0, :, 5] = math.inf
    v[n // 2, :, 7] = -math.inf
    v[n - 1, :, 9] = math.nan
    cu = _cu([n])
    got = serving.prompt_attention(q, k, v, cu)
    assert _time(lambda: serving.prompt_attention(q, k, v, cu)) < 35
    finite = torch.ones_like(got, dtype=torch.bool)
    finite[:, :, 5] = finite[n // 2:, :, 7] = finite[n - 1:, :, 9] = False
    assert torch.equal(got.isfinite(), finite)
    assert bool((got[:, :, 5] == math.inf).all()) and bool((got[n // 2:, :, 7] == -math.inf).all()) and bool(got[n - 1, :, 9].isnan().all())
    v[~v.isfinite()] = 0
    clean = serving.prompt_attention(q, k, v, cu)
    # two computations of the same row, each within the bound of the tests above
    size = v.abs().max().double()
    assert float((got.double() - clean.double())[finite].abs().max()) <= 2.0 ** -7 * float(size) * 2


def test_more_query_rows_than_a_grid_axis():
    """270000 rows; heads of more than 128 values are refused beyond 262140."""
    lens = [900] * 300
    q, k, v = _case(lens, lens, 2, 1, 16, torch.bfloat16, seed=27)
    got = serving.prompt_attention(q, k, v, _cu(lens))
    for i in (0, 150, 291, 299):
        rows = slice(900 * i, 900 * i + 900)
        _check(got[rows], q[rows], k[rows], v[rows], [900], [900], 0.25)
    wide = torch.zeros(1, 1, 136, dtype=torch.bfloat16, device=DEV).expand(270000, 1, 136)
    with pytest.raises(RuntimeError, match="262140"):
        serving.prompt_attention(wide, wide, wide, _cu([270000]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,m,heads", [(300, 300, 2), (300, 300, 160), (60, 3000, 2)])
@pytest.mark.parametrize("power", [0, 13, 20, 30])
def test_scores_of_any_finite_size(power, n, m, heads, dtype):
    """Products that are whole numbers times 2^power: exact in 32 bits, far apart, some of them equal."""
    d = 64
    g = torch.Generator(device=DEV).manual_seed(28)
    q, k = (torch.randint(-8, 9, (rows, h, d), generator=g, device=DEV).to(dtype) for rows, h in ((n, heads), (m, 1)))
    q, k = q * 2.0 ** (power // 2 - 3), k * 2.0 ** (power - power // 2)      # fp16: 8 * 2^15 does not fit
    if not bool(q.isfinite().all() and k.isfinite().all()):
        pytest.skip("fp16 does not hold such values")
    v = torch.randn(m, 1, d, generator=g, device=DEV).to(dtype)
    got = serving.prompt_attention(q, k, v, _cu([n]), _cu([m]), scale=1.0)
    some = torch.linspace(0, heads - 1, 2).long().tolist()
    _check(got[:, some], q[:, some], k, v, [n], [m], 1.0)
