"""Refusals of the serving entry points, before any device is touched."""
import ctypes
import math

import pytest
import torch

from qmoe_b200 import _lib, serving

FAKE = 256                                     # an address that nothing looks at: refusals come first
PROMPT = ("q", "k", "v", "out", "cu_q", "cu_k", "bias", "work", "total_q", "total_k", "q_row", "q_head", "k_row", "k_head",
          "v_row", "v_head", "out_row", "out_head", "n_seqs", "heads", "kv_heads", "head_dim", "dtype", "n_dist", "scale")
ROWS = ("k", "v", "k_row", "k_head", "v_row", "v_head", "cu", "start", "table", "status", "n_rows", "n_seqs", "max_pages", "dtype")
PAGED = ("q", "out", "table", "lengths", "bias", "status", "work", "q_row", "q_head", "n_dist", "n_seqs", "heads", "max_pages",
         "dtype", "scale")
SAMPLE = ("logits", "temperature", "top_k", "top_p", "min_p", "uniform", "tokens", "logprob", "row_stride", "rows", "vocab", "dtype")


def _pack(layout, names, base, changes):
    unknown = set(changes) - set(names)
    assert not unknown, unknown
    return layout.pack(*[changes.get(n, base.get(n, FAKE)) for n in names])


def _shape(**kw):
    return _pack(_lib.PROMPT_ARGS, PROMPT, dict(bias=0, work=0, total_q=4, total_k=4, q_row=64, q_head=64, k_row=64, k_head=64,
                                                v_row=64, v_head=64, out_row=64, out_head=64, n_seqs=1, heads=2, kv_heads=1,
                                                head_dim=64, dtype=0, n_dist=0, scale=0.0), kw)


def _prompt(args):
    return _lib.load().qmoe_prompt_attention(args, 0, None)


def test_struct_layouts():
    assert _lib.PROMPT_ARGS.size == 8 * 18 + 4 * 8 and _lib.CACHE_ROWS.size == 8 * 11 + 16
    assert _lib.PAGED_ARGS.size == 8 * 9 + 24 and _lib.SAMPLE_ARGS.size == 8 * 9 + 16
    assert ctypes.sizeof(_lib.QuantCacheDesc) == 56


@pytest.mark.parametrize("bad,status", [
    (dict(heads=3, kv_heads=2), _lib.ERR_INVALID_ARG), (dict(kv_heads=0), _lib.ERR_INVALID_ARG),
    (dict(head_dim=0), _lib.ERR_INVALID_ARG), (dict(dtype=2), _lib.ERR_INVALID_ARG), (dict(n_seqs=-1), _lib.ERR_INVALID_ARG),
    (dict(total_q=-1), _lib.ERR_INVALID_ARG), (dict(n_dist=5), _lib.ERR_INVALID_ARG),
    (dict(scale=float("nan")), _lib.ERR_INVALID_ARG), (dict(scale=float("inf")), _lib.ERR_INVALID_ARG),
    (dict(head_dim=257), _lib.ERR_UNSUPPORTED), (dict(total_k=1 << 31), _lib.ERR_UNSUPPORTED)])
def test_prompt_refusals(bad, status):
    assert _prompt(_shape(**bad)) == status
    assert _lib.load().qmoe_last_error()


def test_prompt_null_pointers_and_empty_calls():
    assert _prompt(_shape(q=0)) == _lib.ERR_INVALID_ARG
    assert _prompt(_shape(cu_k=0)) == _lib.ERR_INVALID_ARG
    assert _prompt(_shape(bias=FAKE)) == _lib.ERR_INVALID_ARG
    assert _prompt(None) == _lib.ERR_INVALID_ARG
    assert _prompt(_shape(n_seqs=0)) == _lib.OK and _prompt(_shape(total_q=0)) == _lib.OK


def test_prompt_workspace():
    size = lambda **kw: _lib.load().qmoe_prompt_work_bytes(_shape(**kw))  # noqa: E731
    assert size() == 0
    assert size(q=258) == 4 * 2 * 64 * 2                             # q off its boundary
    assert size(k_row=65) == 4 * 64 * 2 and size(heads=4, q_head=0) == 4 * 4 * 64 * 2
    assert size(k_head=3, v_head=0) == 0                             # the stride of one head is not used
    assert size(head_dim=200, q_row=201) == 0                        # taken row by row
    assert _prompt(_shape(k_row=65)) == _lib.ERR_INVALID_ARG         # needs a workspace
    assert _prompt(_shape(k_row=65, work=258)) == _lib.ERR_INVALID_ARG


def _cache(**kw):
    base = dict(k_codes=256, v_codes=256, k_scale=256, v_scale=256, n_pages=4, page_size=16, kv_heads=2, head_dim=64, format=0)
    base.update(kw)
    return _lib.QuantCacheDesc(*[base[name] for name, _ in _lib.QuantCacheDesc._fields_])


@pytest.mark.parametrize("bad,status", [
    (dict(page_size=8), _lib.ERR_UNSUPPORTED), (dict(page_size=48), _lib.ERR_UNSUPPORTED),
    (dict(page_size=2048), _lib.ERR_UNSUPPORTED), (dict(head_dim=257), _lib.ERR_UNSUPPORTED),
    (dict(head_dim=0), _lib.ERR_INVALID_ARG), (dict(kv_heads=0), _lib.ERR_INVALID_ARG), (dict(format=2), _lib.ERR_INVALID_ARG),
    (dict(n_pages=-1), _lib.ERR_INVALID_ARG), (dict(k_codes=None), _lib.ERR_INVALID_ARG), (dict(v_scale=None), _lib.ERR_INVALID_ARG),
    (dict(k_codes=264), _lib.ERR_INVALID_ARG)])
def test_cache_refusals(bad, status):
    desc = _cache(**bad)
    assert _append(desc) == status and _read(desc) == status and _decode(desc) == status


def _rows(**kw):
    return _pack(_lib.CACHE_ROWS, ROWS, dict(k_row=1, k_head=1, v_row=1, v_head=1, n_rows=1, n_seqs=1, max_pages=1, dtype=0), kw)


def _append(desc, **kw):
    return _lib.load().qmoe_cache_append(None if desc is None else ctypes.addressof(desc), _rows(**kw), 0, None)


def _read(desc, **kw):
    return _lib.load().qmoe_cache_read(None if desc is None else ctypes.addressof(desc), _rows(**kw), 0, None)


def _decode(desc, **kw):
    args = _pack(_lib.PAGED_ARGS, PAGED, dict(bias=0, q_row=1, q_head=1, n_dist=0, n_seqs=1, heads=2, max_pages=1, dtype=0, scale=0.0), kw)
    return _lib.load().qmoe_decode_attention_paged(None if desc is None else ctypes.addressof(desc), args, 0, None)


def test_cache_call_refusals():
    c = _cache()
    for call in (_append, _read):
        assert call(None) == _lib.ERR_INVALID_ARG
        for name in ("k", "v", "cu", "start", "table", "status"):
            assert call(c, **{name: 0}) == _lib.ERR_INVALID_ARG, name
        assert call(c, dtype=2) == _lib.ERR_INVALID_ARG
        assert call(c, n_rows=-1) == _lib.ERR_INVALID_ARG and call(c, n_rows=1 << 31) == _lib.ERR_INVALID_ARG
        assert call(c, n_seqs=-1) == _lib.ERR_INVALID_ARG and call(c, max_pages=-1) == _lib.ERR_INVALID_ARG
        assert call(c, n_seqs=0, n_rows=0) == _lib.OK and call(c, n_rows=0) == _lib.OK
        assert call(_cache(kv_heads=1025)) == _lib.ERR_UNSUPPORTED
    assert _decode(None) == _lib.ERR_INVALID_ARG
    for name in ("q", "out", "table", "lengths", "status", "work"):
        assert _decode(c, **{name: 0}) == _lib.ERR_INVALID_ARG, name
    for bad in (dict(heads=3), dict(heads=0), dict(bias=FAKE), dict(n_dist=3), dict(n_dist=-1), dict(scale=float("nan")),
                dict(scale=float("-inf")), dict(dtype=2), dict(work=257), dict(n_seqs=-1)):
        assert _decode(c, **bad) == _lib.ERR_INVALID_ARG, bad
    assert _decode(c, n_seqs=4097) == _lib.ERR_UNSUPPORTED
    assert _decode(c, n_seqs=0) == _lib.OK
    size = _lib.load().qmoe_decode_paged_work_bytes
    assert size(4, 8, 2, 64, 0) > 0 and size(0, 8, 2, 64, 0) == 0 and size(4, 8, 3, 64, 0) == 0 and size(4, 8, 2, 300, 0) == 0


def test_sample_refusals():
    def call(**kw):
        base = dict(temperature=0, top_k=0, top_p=0, min_p=0, logprob=0, row_stride=8, rows=1, vocab=8, dtype=2)
        return _lib.load().qmoe_sample(_pack(_lib.SAMPLE_ARGS, SAMPLE, base, kw), 0, None)

    for bad in (dict(logits=0), dict(uniform=0), dict(tokens=0), dict(rows=-1), dict(vocab=0), dict(dtype=3), dict(row_stride=-8),
                dict(rows=1 << 30)):
        assert call(**bad) == _lib.ERR_INVALID_ARG, bad
    assert call(vocab=262145) == _lib.ERR_UNSUPPORTED
    assert call(rows=0) == _lib.OK
    assert _lib.load().qmoe_sample(None, 0, None) == _lib.ERR_INVALID_ARG


def test_python_refusals_on_cpu_tensors():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError):
        serving.prompt_attention(x, x, x, cu)
    with pytest.raises(TypeError):
        serving.prompt_attention(x.float(), x, x, cu)
    with pytest.raises(ValueError):
        serving.prompt_attention(x[0], x, x, cu)
    with pytest.raises(ValueError):
        serving.prompt_attention(x.transpose(1, 2), x, x, cu)
    with pytest.raises(RuntimeError):
        serving.sample_tokens(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(RuntimeError):
        serving.QuantCache(4, 16, 2, 64, "cpu")
    for bad in (dict(page_size=24), dict(page_size=2048), dict(head_dim=0), dict(head_dim=300), dict(kv_heads=0), dict(fmt="fp4")):
        args = dict(n_pages=4, page_size=16, kv_heads=2, head_dim=64, device="cuda:0", fmt="e4m3")
        args.update(bad)
        with pytest.raises(ValueError):
            serving.QuantCache(**args)
    with pytest.raises(TypeError):
        serving.decode_attention_paged(x, None, cu, cu)


def test_prompt_output_has_to_lie_apart():
    buffer = torch.zeros(4, 3, 2, 64)
    q, k, v = buffer[:, 0], buffer[:, 1], buffer[:, 2]
    inputs = (("q", q), ("k", k), ("v", v))
    for out in (q, v, buffer[:, 1].clone().expand(4, 2, 64)[:1].expand(4, 2, 64), torch.zeros(4, 1, 64).expand(4, 2, 64),
                torch.zeros(4 * 64 + 64).as_strided((4, 2, 64), (64, 64, 1))):
        with pytest.raises(ValueError):
            serving._check_out(out, inputs)
    for out in (torch.zeros(4, 2, 64), torch.zeros(2, 4, 64).transpose(0, 1), torch.zeros(4, 2, 80)[..., :64], torch.zeros(0, 2, 64)):
        serving._check_out(out, inputs)
    flat = torch.zeros(3 * 128)                                           # neighbours
    serving._check_out(flat[128:256].view(1, 2, 64), (("q", flat[:128].view(1, 2, 64)), ("k", flat[256:].view(1, 2, 64))))


@pytest.mark.parametrize("scale", [-1.0, float("nan"), -math.inf])
def test_scale_is_not_negative(scale):
    with pytest.raises(ValueError):
        serving._scale(scale)


def test_prompt_workspace_of_split_keys():
    size = lambda **kw: _lib.load().qmoe_prompt_work_bytes(_shape(**kw))  # noqa: E731
    one = dict(n_seqs=1, heads=2, kv_heads=2, total_q=128, total_k=8192, q_row=128, k_row=128, v_row=128, q_head=64, k_head=64, v_head=64)
    parts = lambda n, rows=128, heads=2: n * rows * heads * (64 + 2) * 4    # noqa: E731
    assert size(**one) == parts(32)                                         # 64 key tiles, at most 32 parts
    assert size(**{**one, "total_k": 1024}) == parts(4)                     # two tiles a part
    assert size(**{**one, "total_k": 255}) == 0 and size(**{**one, "total_k": 0}) == 0
    assert size(**{**one, "total_q": 20000}) == 0                           # queries enough
    assert size(**{**one, "n_seqs": 64}) == 0                               # of 128 keys each
    assert size(**{**one, "heads": 20, "kv_heads": 10, "total_q": 1280}) == 0
    assert _prompt(_shape(**one)) == _lib.ERR_INVALID_ARG                   # needs a workspace
    for bad in (dict(heads=0), dict(kv_heads=0), dict(n_seqs=0), dict(n_seqs=-1), dict(total_q=-1), dict(total_k=-1)):
        assert size(**{**one, **bad}) == 0


def test_waits_for_tensor_memory_name_the_values_they_guard():
    """A wait for loads from tensor memory that stands in a statement without the loaded registers does not keep the
    compiler from moving arithmetic on them in front of it."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(serving.__file__), "csrc")
    found = 0
    for name in os.listdir(csrc):
        with open(os.path.join(csrc, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for statement in re.findall(r"asm volatile\(.*?\);", text, re.S):
            if "tcgen05.wait::ld" in statement:
                found += 1
                assert '"+r"(v[0])' in statement or '"=r"(v[0])' in statement, (name, statement)
    assert found > 0


def test_wait_limit_is_not_negative():
    assert _lib.load().qmoe_prompt_set_wait_limit(-1) == _lib.ERR_INVALID_ARG
    assert _lib.load().qmoe_prompt_set_wait_limit(0) == _lib.OK


@pytest.mark.parametrize("rows,head_dim,status", [((1 << 25) + 1, 64, _lib.ERR_UNSUPPORTED), ((1 << 18) - 3, 129, _lib.ERR_UNSUPPORTED)])
def test_too_many_query_rows(rows, head_dim, status):
    assert _prompt(_shape(total_q=rows, head_dim=head_dim, q_row=2 * 136, q_head=136, k_row=136, k_head=136, v_row=136, v_head=136)) == status
