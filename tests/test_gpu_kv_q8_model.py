"""The Qwen3 decoder over an 8-bit KV cache: against the one over a bf16 cache, replayed from graphs, and cut down by
accumulated attention weight."""

from __future__ import annotations

import pytest
import torch

from torch2vk_amd import kernels as K

pytestmark = pytest.mark.gpu

TINY = dict(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=128, mlp=768, vocab=1024)


@pytest.fixture(scope="module")
def weights(device):
    from torch2vk_amd.qwen3.config import Qwen3Config
    from torch2vk_amd.qwen3.weights import synthetic_weights

    return synthetic_weights(Qwen3Config("tiny", **TINY, eos_token_ids=(1023,)), device=device, seed=31, std=0.08, norm_std=0.1)


def decoder(weights, positions=512, **more):
    from torch2vk_amd.qwen3.model import Qwen3Decoder

    d = Qwen3Decoder(weights, max_positions=positions, max_new_tokens=256, persistent=False, **more)
    d.stop_on_eos = False
    return d


@pytest.mark.parametrize("chunk", [None, 150, 512])
def test_hidden_states_are_those_of_a_bf16_cache(weights, chunk):
    """The same 200 tokens, then 70 more of the bf16 decoder's choice: the last hidden state and the logits to 5 %.  A code
    is off by at most half a step of 1/127 of its block's largest value, about 4 / 127 / sqrt(12) = 0.9 % of a value's size,
    so a score of one dominant key by as much and an output by 1.3 %, in each of two layers' residuals."""
    prompt = torch.randint(0, 1000, (200,), generator=torch.Generator().manual_seed(1))
    plain, q8 = decoder(weights), decoder(weights, kv_bits=8)
    for d in (plain, q8):
        if chunk is None:
            d.prefill(prompt)
        else:
            d.prefill_chunked(prompt, chunk=chunk)
    for _ in range(70):
        q8.next_token.copy_(plain.next_token)
        for d in (plain, q8):
            d.decode_step()
    assert int(q8.position) == int(plain.position) == 270
    for got, ref in ((q8.h, plain.h), (q8.logits(), plain.logits())):
        assert float((got - ref).norm() / ref.norm()) < 0.05


def test_graphs_replay_the_eager_steps(weights):
    """Prefill and steps from graphs, over the ends of blocks and with weights kept, bit for bit."""
    prompt = torch.randint(0, 1000, (100,), generator=torch.Generator().manual_seed(2))
    runs = []
    for graphs in (False, True):
        d = decoder(weights, kv_bits=8, kv_weights=True)
        for _ in range(2 if graphs else 1):  # a second prompt over the first one's cache
            if graphs:
                d.prefill_graphed(prompt, chunk=64)
            else:
                d.prefill_chunked(prompt, chunk=64)
            d.run_steps(90, steps_per_graph=7, use_graph=graphs)
        n = int(d.position)
        runs.append((d.generated.clone(), torch.stack(d.kv_weights)[..., :n], *K.kv_cache_q8_dequantize(d.kv[1], d.position)))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("more", [20, 90])
def test_a_graphed_prompt_behind_another(weights, more):
    """The warm-up that a captured prefill begins with leaves the unfinished block and the weights of the tokens before it as
    they were."""
    g = torch.Generator().manual_seed(5)
    first, then = torch.randint(0, 1000, (100,), generator=g), torch.randint(0, 1000, (more,), generator=g)
    runs = []
    for graphs in (False, True):
        d = decoder(weights, kv_bits=8, kv_weights=True)
        d.prefill_chunked(first)
        (d.prefill_graphed if graphs else d.prefill_chunked)(then, start=100, chunk=64)
        n = int(d.position)
        assert n == 100 + more
        runs.append((d.generated.clone(), torch.stack(d.kv_weights)[..., :n], *K.kv_cache_q8_dequantize(d.kv[0], d.position),
                     *K.kv_cache_q8_dequantize(d.kv[1], d.position)))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_eviction_in_the_loop(weights):
    """A prompt, steps, an eviction and steps from the same graph: weights count every query once, positions go on, and the
    kept tokens' keys are the old ones to half a code."""
    d = decoder(weights, kv_bits=8, kv_weights=True)
    prompt = torch.randint(0, 1000, (300,), generator=torch.Generator().manual_seed(3))
    d.prefill_chunked(prompt, chunk=128)
    d.run_steps(50, steps_per_graph=5)
    n = int(d.position)
    assert n == 350
    group = TINY["heads"] // TINY["kv_heads"]
    for w in d.kv_weights:  # every query's weights sum to 1 for each q head
        assert torch.allclose(w[0, :, :n].sum(-1), torch.full((2,), float(n * group), device=w.device), rtol=1e-4)
    before, _ = K.kv_cache_q8_dequantize(d.kv[0], d.position)
    kept = d.evict_cache(2, sink=4, recent=32)
    assert int(d.position) == 128 + 350 - 320 and int(d.rope_offset) == 192
    after, _ = K.kv_cache_q8_dequantize(d.kv[0], d.position)
    for h in range(2):
        at = kept[0][0, h].long()
        assert at[:4].tolist() == [0, 1, 2, 3] and at[-32:].tolist() == list(range(288, 320))
        step = d.kv[0].k_scale[0, :2, h].repeat_interleave(64)[:, None]
        old, new = before[0, at, h].float(), after[0, :128, h].float()
        # half a code of the new scale, and each side's rounding to bf16
        tol = 0.5001 * step + torch.finfo(torch.bfloat16).eps / 2 * (old.abs() + new.abs())
        assert bool(((new - old).abs() <= tol).all())
        assert torch.equal(after[0, 128:158, h], before[0, 320:350, h])
    d.run_steps(40, steps_per_graph=5)
    assert int(d.position) == 198 and int(d.rope_offset) == 192 and torch.isfinite(d.h).all()


def test_refusals(weights):
    from torch2vk_amd.qwen3 import dispatch

    with pytest.raises(ValueError):
        decoder(weights, kv_bits=4)
    with pytest.raises(ValueError):
        decoder(weights, kv_weights=True)
    from torch2vk_amd.qwen3.model import Qwen3Decoder
    with pytest.raises(NotImplementedError):
        Qwen3Decoder(weights, max_positions=64, max_new_tokens=4, persistent=True, kv_bits=8)
    d = decoder(weights, 64, kv_bits=8)
    with pytest.raises(ValueError):
        d.evict_cache(1)
    with pytest.raises(NotImplementedError):
        d.step_logits(0, token=1)
    with pytest.raises(NotImplementedError):
        d.forward_masked(torch.zeros(4, 256, device=d.device), torch.zeros(4, 4, device=d.device))
    with pytest.raises(NotImplementedError):
        dispatch.bind_model_tensors(d)
