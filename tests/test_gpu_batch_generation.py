"""Batched generation: packed prompts, the quantised caches, batched steps and sampling as they are used
together, against a plain re-statement of the stack."""
import pytest
import torch

from qmoe_b200 import serving, sub1
from qmoe_b200.decoder import SwitchDecoderLM, _rms_norm
from tests import serving_ref as ref
from tests.test_gpu_decoder import _dense_expert

pytestmark = pytest.mark.gpu
VOCAB = 512


def _model(**kw):
    args = dict(d_model=136, d_ff=256, n_experts=8, n_layers=2, n_heads=8, vocab=VOCAB, max_len=96,
                device=torch.device("cuda", 0), seed=3, drop_reference_layout=False)          # heads of 17 values
    args.update(kw)
    return SwitchDecoderLM(**args)


class _Recorder:
    """Router that notes the experts it chose."""

    def __init__(self, router):
        self.router, self.w16, self.w32, self.chosen = router, router.w16, router.w32, []

    def __call__(self, hidden):
        logits = self.router(hidden)
        self.chosen.append(torch.softmax(logits, -1).bfloat16().argmax(-1))
        return logits


def _plain_moe(moe, hm, chosen, dev):
    probs = torch.softmax(hm.float() @ moe.router.w32.t(), -1).bfloat16()
    y = torch.empty_like(hm)
    for t in range(hm.shape[0]):
        e = int(chosen[t])
        wi, wo = _dense_expert(moe.store, 2 * e, dev), _dense_expert(moe.store, 2 * e + 1, dev)
        hid = torch.relu((wi @ hm[t].float()).bfloat16()).float()
        y[t] = (probs[t, e].float() * (wo @ hid).bfloat16().float()).bfloat16()
    return y


def _plain_logits(model, ids, n_prompt, fmt, chosen):
    """Logits of every position of one sequence: prompt positions see keys and values as they are, later
    ones all positions' quantised.  ``chosen``: the expert of every block and position.  The choice is the one
    place where the stack is not continuous: two experts' probabilities that differ by less than the bf16
    rounding of the attention in front (one unit in the last place of a hidden value) may change places, and
    the token's output with them, so the statement follows the choice and states everything else."""
    dev, n = model.dev, ids.shape[0]
    x = model.embed[ids]
    for b, experts in zip(model.blocks, chosen):
        qkv = (_rms_norm(x, b["ln1"]) @ b["wqkv"].t()).view(n, 3, model.h, model.hd)
        q, k, v = qkv.unbind(1)
        att = torch.empty(n, model.h, model.hd, dtype=torch.float64, device=dev)
        out, _ = ref.attention_fast(q[:n_prompt].double(), k[:n_prompt].double(), v[:n_prompt].double(), model.hd ** -0.5, None, 0)
        att[:n_prompt] = out
        if n > n_prompt:
            kq, vq = (value * scale.double()[..., None] for value, scale in (ref.quantise(t, fmt) for t in (k, v)))
            out, _ = ref.attention_fast(q[n_prompt:].double(), kq, vq, model.hd ** -0.5, None, n_prompt)
            att[n_prompt:] = out
        x = x + att.bfloat16().reshape(n, -1) @ b["wo"].t()
        hm = _rms_norm(x, b["ln2"]).contiguous()
        probs = torch.softmax(hm.float() @ b["moe"].router.w32.t(), -1)
        of = probs.gather(1, experts[:, None])[:, 0]
        assert float((probs.amax(1) - of).max()) <= 0.02                # nearly the largest, by this statement too
        x = x + _plain_moe(b["moe"], hm, experts, dev)
    return (_rms_norm(x, model.final_norm) @ model.lm_head.t()).float()


@pytest.mark.parametrize("fmt,page", [("e4m3", 16), ("int8", 64)])
def test_packed_prefill_and_steps_match_a_plain_stack(fmt, page):
    model = _model()
    g = torch.Generator().manual_seed(1)
    lens = [5, 33, 1, 16]
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in lens]
    more = torch.randint(0, VOCAB, (3, len(lens)), generator=g).to(model.dev)
    for b in model.blocks:
        b["moe"].router = _Recorder(b["moe"].router)
    state = model.start_batch(prompts, 4, cache_format=fmt, page_size=page)
    got = [state.logits]
    for step in range(3):
        got.append(model.step_batch(state, more[step]))
        state.lengths += 1
    assert sum(c.refused() for c in state.caches) == 0
    for i, prompt in enumerate(prompts):
        ids = torch.cat([prompt.to(model.dev), more[:, i]])
        first = sum(lens[:i])
        chosen = [torch.cat([calls[0][first:first + lens[i]]] + [c[i:i + 1] for c in calls[1:4]])
                  for calls in (b["moe"].router.chosen for b in model.blocks)]
        want = _plain_logits(model, ids, lens[i], fmt, chosen)[lens[i] - 1:]
        for step in range(4):
            err = float((got[step][i] - want[step]).abs().max() / want.abs().max())
            assert err <= 2e-2, (i, step, err)                    # two blocks of bf16 arithmetic


def test_sampled_generation_graph_and_eager_agree():
    model = _model()
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (3, 20, 41)]
    u = torch.rand(9, 3, generator=g)
    kw = dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.01, uniform=u)
    eager = model.generate_batch(prompts, 9, use_graph=False, **kw)
    graphed = model.generate_batch(prompts, 9, use_graph=True, **kw)
    assert eager.shape == (3, 9) and torch.equal(eager, graphed)
    other = model.generate_batch(prompts, 9, **{**kw, "uniform": 1 - u})
    assert not torch.equal(other, eager)
    greedy = model.generate_batch(prompts, 6)
    assert torch.equal(greedy, model.generate_batch(prompts, 6, use_graph=False, uniform=torch.rand(6, 3)))
    first = torch.stack([model.forward(p.to(model.dev), torch.arange(p.numel(), device=model.dev))[-1] for p in prompts])
    top2 = first.topk(2, 1).values
    sure = (top2[:, 0] - top2[:, 1]) > 4e-2 * first.abs().amax(1)          # beyond both paths' bf16 error
    assert torch.equal(greedy[sure, 0], first.argmax(1)[sure])


def test_more_sequences_than_the_small_router_takes():
    model = _model()
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, VOCAB, (1 + i % 7,), generator=g) for i in range(40)]
    u = torch.rand(6, 40, generator=g)
    a = model.generate_batch(prompts, 6, temperature=1.0, uniform=u, use_graph=False)
    assert torch.equal(a, model.generate_batch(prompts, 6, temperature=1.0, uniform=u))


def test_batch_refusals():
    model = _model(n_layers=1)
    one = torch.zeros(3, dtype=torch.int64)
    for prompts, n_new in (([], 1), ([one, one[:0]], 1), ([one], 94), ([one], 0)):
        with pytest.raises(ValueError):
            model.generate_batch(prompts, n_new)
    with pytest.raises(ValueError):
        model.generate_batch([one], 2, uniform=torch.rand(1, 2))
    with pytest.raises(ValueError):
        model.generate_batch([one], 2, cache_format="fp4")
    assert model.generate_batch([one], 93).shape == (1, 93)               # up to max_len exactly
    assert isinstance(serving.QuantCache(0, 16, 1, 8, model.dev), serving.QuantCache)


def test_ids_and_logits_that_cannot_be_used():
    model = _model(n_layers=1)
    one = torch.zeros(3, dtype=torch.int64)
    for bad in (-1, VOCAB):
        with pytest.raises(ValueError):
            model.start_batch([one, one + bad], 1)
    for temperature in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            model.generate_batch([one], 2, temperature=temperature)
    state = model.start_batch([one, one], 4)
    with pytest.raises(ValueError):
        model.step_batch(state, torch.zeros(1, dtype=torch.int64, device=model.dev))
    ids = torch.tensor([-1, VOCAB + 7], device=model.dev)          # the nearest inside
    assert torch.equal(model.step_batch(state, ids), model.step_batch(state, torch.tensor([0, VOCAB - 1], device=model.dev)))
    model.lm_head.fill_(float("nan"))
    with pytest.raises(RuntimeError, match="no distribution"):
        model.generate_batch([one, one], 6, temperature=1.0)


def _capacity(model, tokens):
    for b in model.blocks:
        b["moe"].capacity = tokens


@pytest.mark.parametrize("lens", [[5, 9, 1], [5, 40, 1, 3, 17], [2, 2], [60]])
@pytest.mark.parametrize("capacity", [1, 3, 1024])
def test_capacity_counts_within_a_sequence(lens, capacity):
    """Packed sequences through an MoE block against each by itself."""
    model = _model(n_layers=1)
    _capacity(model, capacity)
    moe = model.blocks[0]["moe"]
    hidden = torch.randn(sum(lens), model.d, generator=torch.Generator().manual_seed(4)).bfloat16().to(model.dev)
    got = moe(hidden, lens=lens)
    rows = hidden.split(lens)
    want = torch.cat([moe(h.contiguous()) for h in rows])
    assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
    choice, _ = sub1.route_top1(moe.router(hidden).contiguous())
    dropped = torch.cat([sub1.capacity_rule(c.contiguous(), moe.n_experts, c.numel(), capacity) for c in choice.split(lens)]) < 0
    if max(lens) > capacity * moe.n_experts or max(lens) <= capacity:     # some expert has more than it takes; none can have
        assert bool(dropped.any()) == (max(lens) > capacity)
    assert torch.equal(got[dropped], want[dropped])                    # passed through
    residual = torch.randn_like(hidden)
    again = moe(hidden, residual=residual, lens=lens)
    assert float((again.float() - (residual + got).float()).abs().max()) <= 2.0 ** -7 * float((residual + got).float().abs().max())


@pytest.mark.parametrize("lens", [[7, 3, 8], [8, 8, 8, 8, 8, 8]])
def test_prompts_lose_no_tokens_to_each_other(lens):
    """Prompts of at most the capacity, together far over it: as if there were none.  Longer ones: as if alone."""
    model = _model(n_layers=1)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in lens]
    unlimited = model.start_batch(prompts, 1).logits
    _capacity(model, max(lens))
    assert torch.equal(model.start_batch(prompts, 1).logits, unlimited)
    _capacity(model, 2)
    alone = torch.cat([model.start_batch([p], 1).logits for p in prompts])
    together = model.start_batch(prompts, 1).logits
    assert float((together - alone).abs().max()) <= 2e-2 * float(alone.abs().max())
    assert not torch.equal(together, unlimited)


@pytest.mark.parametrize("n", [6, 40])
def test_a_step_is_one_token_of_every_sequence(n):
    model = _model(n_layers=1)
    g = torch.Generator().manual_seed(6)
    state = model.start_batch([torch.randint(0, VOCAB, (3,), generator=g) for _ in range(n)], 2)
    ids = torch.randint(0, VOCAB, (n,), generator=g).to(model.dev)
    want = model.step_batch(state, ids)
    _capacity(model, 1)
    assert torch.equal(model.step_batch(state, ids), want)
