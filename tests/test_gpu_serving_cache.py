"""The quantised cache: append, read back and the attention over it, against plain 64-bit statements."""
import copy
import math

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


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _table(capacity, page, pool, seed=0):
    """Pages in no order, -1 behind every sequence's last one."""
    need = [-(-c // page) for c in capacity]
    assert sum(need) <= pool
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    rows, at = [], 0
    for c in need:
        rows.append(perm[at:at + c] + [-1] * (max(need + [1]) - c))
        at += c
    return _ints(rows)


def _slots(table, page, seq, pos):
    return int(table[seq, pos // page]), pos % page


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,heads,page", [(65, 3, 16), (128, 2, 64), (1, 1, 16), (256, 1, 32), (40, 4, 128), (17, 2, 16), (200, 2, 16)])
def test_append_then_read(fmt, dtype, d, heads, page):
    lens, start = [1, 50, 0, 130, 16], [0, 33, 5, 0, 15]
    table = _table([s + n for s, n in zip(start, lens)], page, 40)
    cache = serving.QuantCache(40, page, heads, d, DEV, fmt=fmt)
    g = torch.Generator(device=DEV).manual_seed(1)
    kv = torch.randn(sum(lens), 2, heads, d, generator=g, device=DEV)
    kv *= torch.exp2(torch.randint(-12, 6, kv.shape[:3], generator=g, device=DEV).float())[..., None]
    kv = kv.to(dtype)
    kv[3] = 0                                                                  # rows of zeros
    k, v = kv[:, 0], kv[:, 1]                                                  # strided
    serving.cache_append(cache, k, v, _cu(lens), _ints(start), table)
    got = serving.cache_read(cache, _cu(lens), _ints(start), table, sum(lens), dtype=dtype)
    assert cache.refused() == 0
    owned = torch.zeros(cache.k_scale.shape, dtype=torch.bool)
    for x, codes, scales, back in ((k, cache.k_codes, cache.k_scale, got[0]), (v, cache.v_codes, cache.v_scale, got[1])):
        value, scale = ref.quantise(x, fmt)
        assert torch.equal(back, (value.float() * scale[..., None]).to(dtype))
        row = 0
        for s, n in enumerate(lens):
            for i in range(n):
                at, inside = _slots(table, page, s, start[s] + i)
                owned[at, :, inside] = True
                assert torch.equal(codes[at, :, inside, :d].double(), value[row])
                assert torch.equal(scales[at, :, inside], scale[row])
                row += 1
        assert bool((codes.view(torch.uint8)[..., d:] == 0).all())             # padding
        assert bool((codes.view(torch.uint8).cpu()[~owned] == 0).all()) and bool((scales.cpu()[~owned] == 0).all())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_every_tie_and_every_neighbour_of_one(fmt):
    """Rows whose scale is a power of two, so that quotients lie exactly on rounding borders, and rows
    with scales of many digits whose quotients lie next to them."""
    qmax = ref.QMAX[fmt]
    rows = []
    for mult in (1.0, 3.0, 5.0, 7.0, 13.0):
        base = torch.arange(-254, 255, dtype=torch.float64) / 2 if fmt == "int8" else torch.arange(-448, 449, dtype=torch.float64) / 2
        base = torch.cat([base, base / 64, base / 1024])
        x = (base * mult).clamp(-qmax * mult, qmax * mult)
        x = x[: x.numel() // 63 * 63].reshape(-1, 63)
        rows.append(torch.cat([x, torch.full((x.shape[0], 1), qmax * mult, dtype=torch.float64)], 1))
    x = torch.cat(rows).to(torch.float16).to(DEV)[:, None]
    n = x.shape[0]
    cache = serving.QuantCache(-(-n // 64), 64, 1, 64, DEV, fmt=fmt)
    table = _ints([list(range(cache.n_pages))])
    serving.cache_append(cache, x, x, _cu([n]), _ints([0]), table)
    value, scale = ref.quantise(x, fmt)
    assert torch.equal(cache.k_codes.reshape(-1, 64)[:n].double(), value[:, 0])
    assert torch.equal(cache.k_scale.reshape(-1)[:n], scale[:, 0])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_extreme_rows(fmt, dtype):
    big = torch.finfo(dtype).max
    tiny = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -24
    x = torch.randn(8, 1, 40, device=DEV).to(dtype)
    x[0] = big
    x[1] = tiny
    x[2, 0, 3] = math.nan
    x[3, 0, 39] = math.inf
    x[4, 0, 0] = -math.inf
    x[5] = 0
    x[6, 0, 5] = big
    cache = serving.QuantCache(2, 16, 1, 40, DEV, fmt=fmt)
    serving.cache_append(cache, x, x, _cu([8]), _ints([0]), _ints([[1]]))
    k, v = serving.cache_read(cache, _cu([8]), _ints([0]), _ints([[1]]), 8, dtype=dtype)
    for r in (2, 3, 4):
        assert bool(k[r].isnan().all()) and bool(v[r].isnan().all())
    for r in (0, 1, 5, 6, 7):
        value, scale = ref.quantise(x[r], fmt)
        assert torch.equal(k[r], (value.float() * scale[..., None]).to(dtype)), r
        assert torch.equal(v[r], k[r])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_positions_without_a_page_are_refused_and_counted(fmt):
    cache = serving.QuantCache(3, 16, 2, 64, DEV, fmt=fmt)
    before = [t.view(torch.uint8).clone() for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)]
    x = torch.randn(6, 2, 64, device=DEV).bfloat16()
    table = _ints([[-1, 0], [3, 1], [2, 1 << 30]])
    cu, start = _cu([2, 2, 2]), _ints([3, 15, 31])        # bad page; bad page then page 1; behind the last bad page / the table
    serving.cache_append(cache, x, x, cu, start, table)
    assert cache.refused(reset=True) == 5
    value, scale = ref.quantise(x[3], fmt)
    assert torch.equal(cache.k_codes[1, :, 0].double(), value)
    cache.k_codes.view(torch.uint8)[1, :, 0] = 0
    cache.v_codes.view(torch.uint8)[1, :, 0] = 0
    cache.k_scale[1, :, 0] = 0
    cache.v_scale[1, :, 0] = 0
    for t, b in zip((cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale), before):
        assert torch.equal(t.view(torch.uint8), b)
    serving.cache_append(cache, x[:1], x[:1], _cu([1]), _ints([-1]), table[:1].contiguous())
    assert cache.refused() == 1
    k, _ = serving.cache_read(cache, cu, start, table, 6)
    assert cache.refused() == 6 and bool((k == 0).all())


def test_rows_that_no_sequence_owns():
    cache = serving.QuantCache(2, 16, 1, 16, DEV)
    x = torch.randn(9, 1, 16, device=DEV).bfloat16()
    serving.cache_append(cache, x, x, _cu([4], 2), _ints([0]), _ints([[0]]))
    assert bool((cache.k_scale[0, 0, :4] > 0).all()) and bool((cache.k_scale[0, 0, 4:] == 0).all())
    assert bool((cache.k_scale[1] == 0).all()) and cache.refused() == 0


# ---- attention over the cache --------------------------------------------------------------------------
def _filled(lens, page, heads, d, fmt, pool, seed=0, width=None):
    table = _table(lens, page, pool, seed)
    if width is not None:
        table = torch.nn.functional.pad(table, (0, width - table.shape[1]), value=-1).contiguous()
    cache = serving.QuantCache(pool, page, heads, d, DEV, fmt=fmt)
    # what lies in places of nobody: codes that would be NaN
    cache.k_codes.view(torch.uint8).fill_(0x7f)
    cache.v_codes.view(torch.uint8).fill_(0x7f)
    cache.k_scale.fill_(math.nan)
    cache.v_scale.fill_(math.inf)
    g = torch.Generator(device=DEV).manual_seed(seed)
    k, v = (torch.randn(max(sum(lens), 1), heads, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    cu = _cu(lens)
    serving.cache_append(cache, k[:sum(lens)], v[:sum(lens)], cu, _ints([0] * len(lens)), table)
    kq, vq = (value * scale.double()[..., None] for value, scale in (ref.quantise(t[:sum(lens)], fmt) for t in (k, v)))
    return cache, table, kq, vq


def _check_decode(got, q, kq, vq, lens, scale, bias=None, exact_fn=ref.attention_fast):
    at = 0
    for s, n in enumerate(lens):
        out, size = exact_fn(q[s:s + 1].double(), kq[at:at + n], vq[at:at + n], scale, bias, n - 1)
        err = (got[s:s + 1].double() - out).abs()
        assert float((err - ref.attention_bound(out, size, q.dtype, torch.float16)).max()) <= 0, (s, n, float(err.max()))
        at += n


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(4, 4, 65, 16), (8, 2, 128, 64), (16, 1, 64, 32), (7, 1, 40, 16), (2, 2, 256, 16),
                                                   (24, 2, 16, 128), (6, 2, 1, 16), (34, 2, 200, 16), (5, 5, 96, 1024)])
def test_decode_lengths(heads, kv_heads, d, page, fmt):
    lens = [1, 0, 15, 16, 17, 300, 64, 1029]
    cache, table, kq, vq = _filled(lens, page, kv_heads, d, fmt, 130)
    for dtype in (torch.bfloat16, torch.float16):
        q = torch.randn(len(lens), heads, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).to(dtype)
        got = serving.decode_attention_paged(q, cache, table, _ints(lens))
        _check_decode(got, q, kq, vq, lens, d ** -0.5)
        assert bool((got[1] == 0).all())
    assert cache.refused() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_decode_long_and_wide_table(fmt):
    """Long sequences next to short ones, in a table with room for far more."""
    lens = [20000, 3, 4097]
    cache, table, kq, vq = _filled(lens, 64, 2, 64, fmt, 400, width=2000)
    q = torch.randn(3, 8, 64, device=DEV).bfloat16()
    got = serving.decode_attention_paged(q, cache, table, _ints(lens))
    _check_decode(got, q, kq, vq, lens, 0.125)
    alone = serving.decode_attention_paged(q[:1], cache, table[:1, :313].contiguous(), _ints(lens[:1]))
    _check_decode(alone, q[:1], kq[:20000], vq[:20000], lens[:1], 0.125)


@pytest.mark.parametrize("n_dist", [1, 40, 128, 3000])
def test_decode_relative_bias(n_dist):
    lens = [33, 700, 1, 2500]
    cache, table, kq, vq = _filled(lens, 16, 4, 65, "int8", 210)
    q = (torch.randn(4, 4, 65, device=DEV) * 0.3).bfloat16()
    bias = torch.randn(4, n_dist, device=DEV) * 2
    got = serving.decode_attention_paged(q, cache, table, _ints(lens), scale=1.0, rel_bias=bias)
    _check_decode(got, q, kq, vq, lens, 1.0, bias)


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_decode_bias_that_masks(low):
    lens = [33, 700, 1]
    cache, table, kq, vq = _filled(lens, 16, 2, 64, "e4m3", 60)
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    bias = torch.zeros(4, 41, device=DEV)
    bias[:, 40] = low
    got = serving.decode_attention_paged(q, cache, table, _ints(lens), rel_bias=bias)
    _check_decode(got, q, kq, vq, lens, 0.125, bias, ref.attention)
    whole = torch.full((4, 1), low, device=DEV)
    got = serving.decode_attention_paged(q, cache, table, _ints(lens), rel_bias=whole)
    if low == -math.inf:
        assert bool((got == 0).all())
    else:
        _check_decode(got, q, kq, vq, lens, 0.125, whole, ref.attention)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_decode_poisoned_rows(fmt):
    """A stored NaN row reaches the sequence and head that hold it and no other; masked by a bias it does not."""
    lens = [100, 64]
    cache, table, kq, vq = _filled(lens, 16, 2, 64, fmt, 20)
    q = torch.randn(2, 4, 64, device=DEV).bfloat16()
    clean = serving.decode_attention_paged(q, cache, table, _ints(lens))
    at, inside = _slots(table, 16, 0, 30)
    for scales in (cache.k_scale, cache.v_scale):
        held = scales[at, 1, inside].clone()
        scales[at, 1, inside] = math.nan
        got = serving.decode_attention_paged(q, cache, table, _ints(lens))
        assert bool(got[0, 2:].isnan().all())
        assert torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[1], clean[1])
        scales[at, 1, inside] = held
    bias = torch.zeros(4, 60, device=DEV)
    bias[:, 59] = -math.inf                               # positions 0 .. 40 of the first sequence
    want = serving.decode_attention_paged(q, cache, table, _ints(lens), rel_bias=bias)
    cache.v_scale[at, 1, inside] = math.nan
    got = serving.decode_attention_paged(q, cache, table, _ints(lens), rel_bias=bias)
    assert torch.equal(got, want) and bool(torch.isfinite(got).all())


def test_decode_bad_pages_and_lengths():
    lens = [100, 64, 40]
    cache, table, kq, vq = _filled(lens, 16, 2, 64, "e4m3", 20)
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    hurt = table.clone()
    hurt[0, 2] = 1 << 30                                  # positions 32 .. 47 of the first sequence
    hurt[1, 0] = -7                                       # positions 0 .. 15 of the second
    got = serving.decode_attention_paged(q, cache, hurt, _ints(lens))
    assert cache.refused(reset=True) == 4                 # two tiles, two key heads
    cut = lambda t: torch.cat([t[:32], t[48:100], t[116:]])  # noqa: E731
    _check_decode(got, q, cut(kq), cut(vq), [84, 48, 40], 0.125)
    got = serving.decode_attention_paged(q, cache, table, _ints([100, -3, 1 << 30]))
    assert bool((got[1] == 0).all()) and cache.refused(reset=True) > 0
    _check_decode(got[:1], q[:1], kq, vq, [100], 0.125)


def test_decode_strided_queries_streams_and_graphs():
    lens = [700, 64, 1, 333]
    cache, table, kq, vq = _filled(lens, 16, 2, 128, "e4m3", 80)
    qkv = torch.randn(4, 8, 3, 128, device=DEV).bfloat16()
    want = serving.decode_attention_paged(qkv[:, :, 1].contiguous(), cache, table, _ints(lens))
    assert torch.equal(serving.decode_attention_paged(qkv[:, :, 1], cache, table, _ints(lens)), want)
    odd = torch.zeros(4, 8, 131, device=DEV).bfloat16()
    odd[:, :, 1:129] = qkv[:, :, 1]
    assert torch.equal(serving.decode_attention_paged(odd[:, :, 1:129], cache, table, _ints(lens)), want)
    q, lengths = qkv[:, :, 1].contiguous(), _ints(lens)
    graphs = []
    for _ in range(2):                                    # two graphs, replayed in turn on two streams
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = serving.decode_attention_paged(q, cache, table, lengths)
        graphs.append((graph, held, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, held, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, held, _ in graphs:
        assert torch.equal(held, want)
    lengths.copy_(_ints([5, 64, 0, 100]))                 # a captured call follows its lengths
    want = serving.decode_attention_paged(q, cache, table, lengths)
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], want)


def test_offsets_beyond_32_bits():
    """A pool whose last page lies more than 2^32 bytes behind the first."""
    page, heads, d = 1024, 8, 256
    n_pages = 2100                                        # 2 MB of codes a page and tensor
    cache = serving.QuantCache(n_pages, page, heads, d, DEV)
    x = torch.randn(1500, heads, d, device=DEV).bfloat16()
    table = _ints([[n_pages - 1, n_pages - 2]])
    serving.cache_append(cache, x, x, _cu([1500]), _ints([0]), table)
    k, _ = serving.cache_read(cache, _cu([1500]), _ints([0]), table, 1500)
    value, scale = ref.quantise(x, "e4m3")
    assert torch.equal(k, (value.float() * scale[..., None]).bfloat16())
    q = torch.randn(1, 8, d, device=DEV).bfloat16()
    got = serving.decode_attention_paged(q, cache, table, _ints([1500]))
    kq = value * scale.double()[..., None]
    _check_decode(got, q, kq, kq, [1500], d ** -0.5)


def test_the_cache_keeps_its_memory():
    cache = serving.QuantCache(4, 16, 1, 64, DEV)
    for name in ("k_codes", "v_codes", "k_scale", "v_scale", "status"):
        with pytest.raises(AttributeError):
            setattr(cache, name, torch.zeros_like(getattr(cache, name)))
    with pytest.raises(AttributeError):
        cache.page_size = 32
    with pytest.raises(ValueError):
        copy.deepcopy(cache)


def test_a_cache_without_pages():
    cache = serving.QuantCache(0, 16, 2, 64, DEV)
    x = torch.randn(3, 2, 64, device=DEV).bfloat16()
    for table in (_ints([[0, 1]]), torch.empty((1, 0), dtype=torch.int32, device=DEV)):
        serving.cache_append(cache, x, x, _cu([3]), _ints([0]), table)
        assert cache.refused(reset=True) == 3
        k, v = serving.cache_read(cache, _cu([3]), _ints([0]), table, 3)
        assert bool((k == 0).all()) and bool((v == 0).all()) and cache.refused(reset=True) == 3
        assert bool((serving.decode_attention_paged(x[:1], cache, table, _ints([3])) == 0).all())
        assert cache.refused(reset=True) == 2             # one tile, or one sequence, by two key heads


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("int8", torch.float16)])
@pytest.mark.parametrize("d", [2, 15, 16, 31, 33, 48, 63, 66, 72, 79, 80, 81, 95, 96, 97, 112, 127, 129])
def test_every_row_width_and_alignment(fmt, dtype, d):
    """Rows of 1 to 9 pieces that begin on any 2-byte boundary, infinities right before and behind them."""
    n, heads, page = 70, 3, 16
    table = _table([n], page, 8)
    g = torch.Generator(device=DEV).manual_seed(d)
    for shift in range(0, 9, 1 if d < 90 else 3):
        pool = torch.full((n * 2 * heads * (d + 3) + 16,), math.inf, dtype=dtype, device=DEV)
        rows = pool[shift:shift + n * 2 * heads * (d + 3)].view(n, 2, heads, d + 3)[..., 1:1 + d]
        rows.copy_(torch.randn(n, 2, heads, d, generator=g, device=DEV))
        cache = serving.QuantCache(8, page, heads, d, DEV, fmt=fmt)
        serving.cache_append(cache, rows[:, 0], rows[:, 1], _cu([n]), _ints([0]), table)
        k, v = serving.cache_read(cache, _cu([n]), _ints([0]), table, n, dtype=dtype)
        for x, back in ((rows[:, 0], k), (rows[:, 1], v)):
            value, scale = ref.quantise(x, fmt)
            assert torch.equal(back, (value.float() * scale[..., None]).to(dtype)), shift


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("group", [2, 12])
def test_decode_keys_that_a_bias_masks_may_hold_anything(fmt, group):
    lens = [100, 3000, 64]
    cache, table, _, _ = _filled(lens, 16, 2, 64, fmt, 210)
    q = torch.randn(3, 2 * group, 64, device=DEV).bfloat16()
    bias = torch.randn(2 * group, 60, device=DEV)
    bias[:, 59] = -math.inf
    want = serving.decode_attention_paged(q, cache, table, _ints(lens), rel_bias=bias)
    assert bool(torch.isfinite(want).all())
    for value in (math.nan, math.inf):
        for seq, pos in ((0, 30), (1, 2000), (1, 2940), (2, 4)):
            at, inside = _slots(table, 16, seq, pos)
            cache.k_scale[at, 1, inside] = value
            cache.v_scale[at, 0, inside] = value
        assert torch.equal(serving.decode_attention_paged(q, cache, table, _ints(lens), rel_bias=bias), want)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("low,high", [(-30, 30), (-110, -80), (-110, 100)])
def test_decode_value_rows_of_very_different_size(fmt, dtype, low, high):
    """Three times in every sequence and head the scores rise by 40 units of log 2 and the value rows' size changes,
    at other positions everywhere, so that they lie in the middle of a warp's run of tiles."""
    if dtype == torch.float16 and high != 30:
        pytest.skip("fp16 does not hold such values")
    n_seqs, n, kv_heads, group, d, page = 40, 1000, 8, 2, 64, 64
    g = torch.Generator(device=DEV).manual_seed(31)
    direction = torch.where(torch.rand(kv_heads, d, generator=g, device=DEV) < 0.5, -1.0, 1.0)
    at = torch.randint(1, n, (n_seqs, kv_heads, 3), generator=g, device=DEV).sort(-1).values
    level = (torch.arange(n, device=DEV)[None, :, None, None] >= at[:, None]).sum(-1)               # [sequence, position, head]
    size = torch.randint(low, high + 1, (n_seqs, kv_heads, 4), generator=g, device=DEV).gather(2, level.transpose(1, 2)).transpose(1, 2)
    # q = direction / 8, |q|^2 = 1: a step of 40 * ln 2 in the scores (scale 1) is one of 40 * ln 2 * direction / 8 in k
    k = direction / 8 * (level * 40 * math.log(2.0))[..., None] + 0.05 * torch.randn(n_seqs, n, kv_heads, d, generator=g, device=DEV)
    v = torch.randn(n_seqs, n, kv_heads, d, generator=g, device=DEV) * torch.exp2(size.float())[..., None]
    if dtype == torch.float16:
        v = v / 2 ** 18                                                      # 2^-48 .. 2^14: what is too small is rounded away here
    k, v = k.to(dtype).flatten(0, 1), v.to(dtype).flatten(0, 1)
    q = (direction / 8).repeat_interleave(group, 0)[None].expand(n_seqs, -1, -1).to(dtype)
    cache = serving.QuantCache(n_seqs * 16, page, kv_heads, d, DEV, fmt=fmt)
    table = torch.arange(n_seqs * 16, dtype=torch.int32, device=DEV).view(n_seqs, 16)
    serving.cache_append(cache, k, v, _cu([n] * n_seqs), _ints([0] * n_seqs), table)
    got = serving.decode_attention_paged(q, cache, table, _ints([n] * n_seqs), scale=1.0).double()
    kq, vq = ((value * scale.double()[..., None]).view(n_seqs, n, kv_heads, d) for value, scale in (ref.quantise(t, fmt) for t in (k, v)))
    p = torch.softmax(torch.einsum("sphd,hd->shp", kq, (direction / 8).double()), -1)
    out, mean = torch.einsum("shp,sphd->shd", p, vq), torch.einsum("shp,sphd->shd", p, vq.abs())
    largest = torch.einsum("shp,sph->sh", p, vq.abs().amax(-1))[..., None]
    # half a step of the output and of the fp16 weights, 2^-12 for scores of up to 2^7, and 2^-32 of the largest
    # weight * row for each of the keys (weights that are subnormal in fp16); what the output type rounds to zero
    bound = torch.finfo(dtype).eps / 2 * out.abs() + (2.0 ** -11 + 2.0 ** -12) * mean + n * 2.0 ** -32 * largest
    bound = bound * 1.01 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    err = (got.view(n_seqs, kv_heads, group, d) - out[:, :, None]).abs()
    assert float((err / bound[:, :, None]).max()) <= 1


def test_cache_offsets_outside_the_rows_are_clamped():
    x = torch.randn(20, 2, 64, device=DEV).bfloat16()
    table, start = _ints([[0, 2], [1, 3]]), _ints([3, 5])
    bad, good = _ints([-7, 12, 1 << 30]), _ints([0, 12, 20])
    caches = [serving.QuantCache(4, 16, 2, 64, DEV) for _ in range(2)]
    for cache, cu in zip(caches, (bad, good)):
        serving.cache_append(cache, x, x, cu, start, table)
        assert cache.refused() == 0
    assert torch.equal(caches[0].k_scale, caches[1].k_scale)
    assert torch.equal(caches[0].k_codes.view(torch.uint8), caches[1].k_codes.view(torch.uint8))
    for a, b in zip(*(serving.cache_read(caches[1], cu, start, table, 20) for cu in (bad, good))):
        assert torch.equal(a, b)
    assert caches[1].refused() == 0


def test_decode_of_as_many_positions_as_a_length_can_say():
    """2^31 - 1 positions in a table that has room for them, all but 2047 without a page, next to a short sequence."""
    most, page = 2 ** 31 - 1, 1024
    cache = serving.QuantCache(3, page, 1, 16, DEV)
    table = torch.full((2, 2 ** 21), -1, dtype=torch.int32, device=DEV)
    table[0, 0], table[0, -1], table[1, 0] = 0, 1, 2
    k, v = (torch.randn(2052, 1, 16, device=DEV).bfloat16() for _ in range(2))
    serving.cache_append(cache, k[:1024], v[:1024], _cu([1024]), _ints([0]), table[:1])
    serving.cache_append(cache, k[1024:2047], v[1024:2047], _cu([1023]), _ints([most - 1023]), table[:1])   # the last page but its last place
    serving.cache_append(cache, k[2047:2052], v[2047:2052], _cu([5]), _ints([0]), table[1:])
    assert cache.refused() == 0
    q = torch.randn(2, 1, 16, device=DEV).bfloat16()
    got = serving.decode_attention_paged(q, cache, table, _ints([most, 5]))
    assert cache.refused(reset=True) == 2 ** 27 - 2 * 64                    # tiles of 16 positions without a page
    kq, vq = (value * scale.double()[..., None] for value, scale in (ref.quantise(t, "e4m3") for t in (k, v)))
    _check_decode(got, q, kq, vq, [2047, 5], 0.25)
