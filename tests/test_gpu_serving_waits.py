"""Bounded waits of the prompt kernel: with the bound lowered they run out although nothing hangs."""
import contextlib

import pytest
import torch

from qmoe_b200 import _lib, serving, sub1

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@contextlib.contextmanager
def wait_limit(ns):
    assert _lib.load().qmoe_prompt_set_wait_limit(ns) == _lib.OK
    try:
        yield
        torch.cuda.synchronize()
    finally:
        _lib.load().qmoe_prompt_set_wait_limit(0)


def _rows(lens, heads, kv_heads, d, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)
    mk = lambda h: torch.randn(sum(lens), h, d, generator=g, device=DEV).to(dtype)  # noqa: E731
    return mk(heads), mk(kv_heads), mk(kv_heads), cu


# whole tiles and partial ones, one item a CTA and many, keys split among CTAs, a bias
@pytest.mark.parametrize("lens,heads,kv_heads,d,n_dist", [([128, 256], 2, 2, 64, 0), ([700, 33, 0, 5], 8, 2, 128, 0), ([3000], 2, 1, 64, 0),
                                                          ([600] * 12, 16, 4, 65, 0), ([300, 900], 4, 4, 64, 40)])
def test_waits_that_run_out_are_counted_and_leave_the_gpu_usable(lens, heads, kv_heads, d, n_dist):
    q, k, v, cu = _rows(lens, heads, kv_heads, d)
    bias = torch.randn(heads, n_dist, device=DEV) if n_dist else None
    want = serving.prompt_attention(q, k, v, cu, rel_bias=bias)
    assert sub1.tile_timeouts(DEV, reset=True) == 0
    with wait_limit(1):
        serving.prompt_attention(q, k, v, cu, rel_bias=bias)
    assert sub1.tile_timeouts(DEV) > 0                     # sticky
    with pytest.raises(_lib.QmoeError, match="incomplete"):
        sub1.check_tile_status(DEV)                        # raises and clears
    assert sub1.tile_timeouts(DEV) == 0
    for ns in (1500, 15000):                               # some waits run out in the middle of the work, or none does
        with wait_limit(ns):
            got = serving.prompt_attention(q, k, v, cu, rel_bias=bias)
        assert sub1.tile_timeouts(DEV, reset=True) > 0 or torch.equal(got, want)
    for _ in range(3):                                     # and the next calls are whole again
        assert torch.equal(serving.prompt_attention(q, k, v, cu, rel_bias=bias), want)
    assert sub1.tile_timeouts(DEV) == 0


def test_rows_computed_again_take_longer_than_a_wait():
    """An infinite value sends every row to the key by key path, 100000 keys a row: far longer than the bound, which
    the tiles themselves keep to.  More items than multiprocessors, so that the next one waits."""
    heads, m = 640, 100000
    q, k, v, _ = _rows([m], heads, 1, 64)
    q = q[:1].contiguous()
    v[0] = float("inf")
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (1, m))
    serving.prompt_attention(q, k, v, cu_q, cu_k)          # brings the clocks up: the tiles then take 1.3 ms
    assert sub1.tile_timeouts(DEV, reset=True) == 0
    with wait_limit(4_000_000):
        got = serving.prompt_attention(q, k, v, cu_q, cu_k, out=torch.zeros_like(q))
    assert sub1.tile_timeouts(DEV, reset=True) == 0
    assert bool((got == float("inf")).all())


@pytest.mark.parametrize("use_graph", [False, True])
def test_generation_does_not_return_tokens_behind_a_wait_that_ran_out(use_graph):
    from qmoe_b200.decoder import SwitchDecoderLM
    model = SwitchDecoderLM(d_model=128, d_ff=256, n_experts=4, n_layers=1, n_heads=2, vocab=64, max_len=64, device=DEV, seed=1,
                            drop_reference_layout=False)
    prompts = [torch.arange(20) % 64, torch.arange(3)]
    want = model.generate_batch(prompts, 8, use_graph=use_graph)
    assert sub1.tile_timeouts(DEV, reset=True) == 0
    with wait_limit(1), pytest.raises(RuntimeError, match="gave up"):
        model.generate_batch(prompts, 8, use_graph=use_graph)
    # an earlier call's count is that caller's to clear: it does not make this one fail
    assert torch.equal(model.generate_batch(prompts, 8, use_graph=use_graph), want)
    assert sub1.tile_timeouts(DEV, reset=True) > 0
