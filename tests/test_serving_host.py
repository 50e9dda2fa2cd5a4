"""Refusals of the serving entry points, before any device is touched."""
import ctypes

import pytest
import torch

from qmoe_b200 import _lib, serving

FAKE = ctypes.c_void_p(256)


def _shape(**kw):
    base = dict(total_q=4, total_k=4, q_row=64, q_head=64, k_row=64, k_head=64, v_row=64, v_head=64, out_row=64,
                out_head=64, n_seqs=1, heads=2, kv_heads=1, head_dim=64, dtype=0, n_dist=0, scale=0.0)
    base.update(kw)
    return _lib.PromptShape(*[base[name] for name, _ in _lib.PromptShape._fields_])


def _prompt(shape, bias=None, q=FAKE):
    return _lib.load().qmoe_prompt_attention(q, FAKE, FAKE, FAKE, FAKE, FAKE, bias, ctypes.byref(shape), 0, None)


def test_struct_layouts():
    assert ctypes.sizeof(_lib.PromptShape) == 112 and _lib.PromptShape.scale.offset == 104
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
    assert _prompt(_shape(), q=None) == _lib.ERR_INVALID_ARG
    assert _prompt(_shape(), bias=FAKE) == _lib.ERR_INVALID_ARG
    assert _lib.load().qmoe_prompt_attention(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, None, 0, None) == _lib.ERR_INVALID_ARG
    assert _prompt(_shape(n_seqs=0)) == _lib.OK and _prompt(_shape(total_q=0)) == _lib.OK


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
    lib, c = _lib.load(), ctypes.byref(_cache(**bad))
    assert lib.qmoe_cache_append(c, FAKE, FAKE, 1, 1, 1, 1, FAKE, FAKE, FAKE, FAKE, 1, 1, 1, 0, 0, None) == status
    assert lib.qmoe_cache_read(c, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1, 1, 1, 0, 0, None) == status
    assert lib.qmoe_decode_attention_paged(c, FAKE, 1, 1, FAKE, FAKE, FAKE, None, 0, FAKE, FAKE, 1, 2, 1, 0.0, 0, 0, None) == status


def test_cache_call_refusals():
    lib, c = _lib.load(), ctypes.byref(_cache())
    assert lib.qmoe_cache_append(None, FAKE, FAKE, 1, 1, 1, 1, FAKE, FAKE, FAKE, FAKE, 1, 1, 1, 0, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.qmoe_cache_append(c, FAKE, FAKE, 1, 1, 1, 1, FAKE, FAKE, FAKE, None, 1, 1, 1, 0, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.qmoe_cache_append(c, None, FAKE, 1, 1, 1, 1, FAKE, FAKE, FAKE, FAKE, 1, 1, 1, 0, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.qmoe_cache_append(c, FAKE, FAKE, 1, 1, 1, 1, FAKE, FAKE, FAKE, FAKE, 1, 1, 1, 2, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.qmoe_cache_append(c, FAKE, FAKE, 1, 1, 1, 1, FAKE, FAKE, FAKE, FAKE, 1, 1, -1, 0, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.qmoe_cache_append(c, FAKE, FAKE, 1, 1, 1, 1, FAKE, FAKE, FAKE, FAKE, 0, 1, 0, 0, 0, None) == _lib.OK
    dec = lib.qmoe_decode_attention_paged
    assert dec(c, FAKE, 1, 1, FAKE, FAKE, FAKE, None, 0, FAKE, FAKE, 1, 3, 1, 0.0, 0, 0, None) == _lib.ERR_INVALID_ARG
    assert dec(c, FAKE, 1, 1, FAKE, FAKE, FAKE, FAKE, 0, FAKE, FAKE, 1, 2, 1, 0.0, 0, 0, None) == _lib.ERR_INVALID_ARG
    assert dec(c, FAKE, 1, 1, FAKE, FAKE, FAKE, None, 0, FAKE, FAKE, 1, 2, 1, float("nan"), 0, 0, None) == _lib.ERR_INVALID_ARG
    assert dec(c, FAKE, 1, 1, None, FAKE, FAKE, None, 0, FAKE, FAKE, 1, 2, 1, 0.0, 0, 0, None) == _lib.ERR_INVALID_ARG


def test_sample_refusals():
    f = _lib.load().qmoe_sample
    ok = [FAKE, 8, 1, 8, 2, None, None, None, None, FAKE, FAKE, None, 0, None]
    for at, value, status in ((0, None, _lib.ERR_INVALID_ARG), (9, None, _lib.ERR_INVALID_ARG), (10, None, _lib.ERR_INVALID_ARG),
                              (2, -1, _lib.ERR_INVALID_ARG), (3, 0, _lib.ERR_INVALID_ARG), (4, 3, _lib.ERR_INVALID_ARG),
                              (1, -8, _lib.ERR_INVALID_ARG), (3, 262145, _lib.ERR_UNSUPPORTED), (2, 0, _lib.OK)):
        args = list(ok)
        args[at] = value
        assert f(*args) == status, (at, value)


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
