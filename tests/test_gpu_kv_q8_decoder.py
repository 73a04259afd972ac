"""The Qwen3 decoder over an 8-bit KV cache where a call names a place in the cache or a budget of its own."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv_q8_model import TINY, decoder, weights  # noqa: F401 (weights: a fixture)
from torch2vk_amd import kernels as K

pytestmark = pytest.mark.gpu


def prompt(n, seed):
    return torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(seed))


def held(d):
    return [t.clone() for layer in range(2) for t in K.kv_cache_q8_dequantize(d.kv[layer], d.position)]


def test_a_prefill_goes_on_from_what_the_cache_holds(weights):  # noqa: F811
    """Another start than 0 or the tokens that it holds is refused, and what it holds stays as it was."""
    d = decoder(weights, kv_bits=8, kv_weights=True)
    d.prefill_chunked(prompt(150, 1))
    d.run_steps(10, steps_per_graph=5)
    assert int(d.position) == 160
    before, w = held(d), [t.clone() for t in d.kv_weights]
    embeds = torch.zeros(3, TINY["hidden"], device=d.device)
    for start in (1, 64, 100, 159, 161, 200):
        for call in (lambda: d.prefill(prompt(3, 2), start=start), lambda: d.prefill_chunked(prompt(3, 2), start=start),
                     lambda: d.prefill_graphed(prompt(3, 2), start=start), lambda: d.prefill_embeds(embeds, start=start),
                     lambda: d.reset(position=start)):
            with pytest.raises(ValueError, match="holds 160"):
                call()
    for place in (1, 159, 162):
        with pytest.raises(ValueError, match="holds 160"):
            d.run_decode_layer(0, cache_position=place)
    assert int(d.position) == 160
    assert all(torch.equal(a, b) for a, b in zip(before, held(d))) and all(torch.equal(a, b) for a, b in zip(w, d.kv_weights))
    d.prefill_chunked(prompt(70, 3), start=160)
    assert int(d.position) == 230


def test_a_captured_prefill_is_checked_before_every_replay(weights):  # noqa: F811
    d = decoder(weights, kv_bits=8)
    d.prefill_chunked(prompt(100, 4))
    d.prefill_graphed(prompt(20, 5), start=100)
    with pytest.raises(ValueError, match="holds 120"):
        d.prefill_graphed(prompt(20, 5), start=100)
    d.prefill_chunked(prompt(100, 4))
    d.prefill_graphed(prompt(20, 6), start=100)
    plain = decoder(weights, kv_bits=8)
    plain.prefill_chunked(prompt(100, 4))
    plain.prefill_chunked(prompt(20, 6), start=100)
    assert all(torch.equal(a, b) for a, b in zip(held(d), held(plain)))


def test_layers_at_the_places_that_follow(weights):  # noqa: F811
    """A caller's own loop: every layer at the next place, and at 0 again."""
    d, ref = decoder(weights, kv_bits=8), decoder(weights, kv_bits=8)
    for _ in range(2):
        ref.prefill(prompt(70, 7))
        for place, token in enumerate(prompt(70, 7).tolist()):
            d.next_token.fill_(token)
            d.run_decode_embed()
            for layer in range(2):
                d.run_decode_layer(layer, cache_position=place)
        d.position.fill_(70)
        assert all(torch.equal(a, b) for a, b in zip(held(d), held(ref)))
    other = decoder(weights)  # a bf16 cache takes any
    other.next_token.fill_(5)
    other.run_decode_embed()
    other.run_decode_layer(0, cache_position=17)
    assert int(other.position) == 17


@pytest.mark.parametrize("keep,more,recent", [(1, {}, 60), (1, dict(sink=0), 64), (2, {}, 64), (1, dict(sink=64), 0)])
def test_default_recent_tokens_fit_the_budget(weights, keep, more, recent):  # noqa: F811
    """evict_cache's defaults: the last 64 tokens, or as many as the first ones leave of the budget."""
    d = decoder(weights, kv_bits=8, kv_weights=True)
    d.prefill_chunked(prompt(200, 8))
    kept = d.evict_cache(keep, **more)
    assert int(d.position) == 64 * keep + 8
    for layer in kept:
        for row in layer[0].tolist():
            assert row[:more.get("sink", 4)] == list(range(more.get("sink", 4)))
            assert row[len(row) - recent:] == list(range(192 - recent, 192))
    with pytest.raises(ValueError):
        decoder(weights, kv_bits=8, kv_weights=True).evict_cache(1, sink=4, recent=64)
