"""Steps of the Qwen3 decoder over trees of drafted tokens: a step's logits, cache rows and tokens against one-token steps, its
bookkeeping, replays from graphs, and generation."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = dict(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=128, mlp=768, vocab=1024)

# A layer rounds its two norms' outputs, the attention's and the activation to bf16, the head its input: over two layers 9
# roundings, of half a step each, add up to 9 * 2^-8 = 3.5 % of a logit's size at the worst, where every one falls the other way;
# the attention's weights and the cached rows, bf16 in both, another 2 * 2^-8 a layer: 5 %.
CLOSE = 0.05


@pytest.fixture(scope="module")
def weights(device):
    from torch2vk_amd.qwen3.config import Qwen3Config
    from torch2vk_amd.qwen3.weights import synthetic_weights

    return synthetic_weights(Qwen3Config("tiny", **TINY, eos_token_ids=(1023,)), device=device, seed=41, std=0.08, norm_std=0.1)


def decoder(weights, positions=256, **more):
    from torch2vk_amd.qwen3.model import Qwen3Decoder

    d = Qwen3Decoder(weights, max_positions=positions, max_new_tokens=64, persistent=False, **more)
    d.stop_on_eos = False
    return d


def prompt(n, seed=1):
    return torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(seed))


def feed(d, tokens, at):
    """One-token steps; the logits after the last."""
    for i, t in enumerate(tokens):
        d.next_token.fill_(int(t))
        d.position.fill_(at + i)
        d.run_decode_embed()
        d.run_decode_layers()
    return d.logits()


def ancestors(parents, i):
    line = []
    while i >= 0:
        line.append(i)
        i = parents[i]
    return line[::-1]


def near(got, ref, tol=CLOSE):
    assert float((got.float() - ref.float()).norm() / ref.float().norm()) < tol


TREES = {"chain": [-1, 0, 1, 2, 3], "bush": [-1, 0, 0, 0, 1, 1, 2, 4, 6, 8, 9], "one": [-1], "wide": [-1] + [0] * 20}


@pytest.mark.parametrize("shape", list(TREES))
@pytest.mark.parametrize("length", [1, 63, 100])
def test_a_steps_logits_and_rows_are_one_token_steps(weights, device, shape, length):
    """Every node's logits are those after its ancestors one by one, and the rows kept are the path's."""
    parents = TREES[shape]
    n = len(parents)
    a, b = decoder(weights), decoder(weights)
    for d in (a, b):
        d.prefill_chunked(prompt(length))
    first = int(a.next_token)
    # drafts: along one line the tokens that one-token steps choose, elsewhere others
    drafts = prompt(n, 5).tolist()
    drafts[0] = first
    for i in ancestors(parents, n - 1)[1:]:
        drafts[i] = int(feed(b, [drafts[j] for j in ancestors(parents, parents[i])], length).argmax())
    path, kept, logits = a.tree_step(torch.tensor(drafts[1:], dtype=torch.int64, device=device),
                                     parents=torch.tensor(parents, dtype=torch.int32, device=device))
    for i in range(n):
        near(logits[i], feed(b, [drafts[j] for j in ancestors(parents, i)], length))
    # the walk over these logits
    best = logits.argmax(-1).tolist()
    walk = [0]
    while True:
        child = [i for i in range(n) if parents[i] == walk[-1] and drafts[i] == best[walk[-1]]]
        if not child:
            break
        walk.append(child[0])
    assert int(kept) == len(walk) and path.tolist() == walk + [-1] * (n - len(walk))
    assert int(a.next_token) == best[walk[-1]] and int(a.position) == length + len(walk)
    assert a.generated[:int(a.length)].tolist() == [first] + [drafts[i] for i in walk[1:]] + [best[walk[-1]]]
    feed(b, [drafts[i] for i in walk], length)
    rows = slice(length, length + len(walk))
    near(a.k_cache[:, rows], b.k_cache[:, rows])
    near(a.v_cache[:, rows], b.v_cache[:, rows])
    assert torch.equal(a.k_cache[:, :length], b.k_cache[:, :length])
    near(feed(a, [int(a.next_token)], length + len(walk)), feed(b, [best[walk[-1]]], length + len(walk)))


@pytest.mark.parametrize("kept,length,stopped,stop,tokens,following", [
    (3, 0, 0, True, [5, 6, 7, 8], 9),       # two drafted tokens and one more
    (1, 4, 0, True, [5, 6, 7, 8], 9),
    (4, 1, 0, True, [5, 1, 2, 1], 9),       # 1 ends the text, in the middle
    (4, 1, 0, False, [5, 1, 2, 1], 9),
    (2, 1, 0, True, [5, 6, 7, 8], 1),       # the token that follows ends it
    (2, 1, 1, True, [5, 6, 7, 8], 9),       # ended before
    (4, 6, 0, True, [5, 6, 7, 8], 9),       # room for two
    (3, 8, 0, True, [5, 6, 7, 8], 9),       # and none
    (0, 2, 0, True, [5, 6, 7, 8], -1),      # no node had a slot
    (2, 2, 0, True, [5, 6, 7, 8], -1),      # nothing has any probability
])
def test_stored_tokens(weights, device, kept, length, stopped, stop, tokens, following):
    d = decoder(weights)
    d.stop_on_eos = stop
    d.eos = torch.tensor([1, 1023], device=device)
    d.generated = torch.arange(100, 108, device=device)
    d.length.fill_(length)
    d.stopped.fill_(stopped)
    d.position.fill_(20)
    d.next_token.fill_(tokens[0])
    path = list(range(kept)) + [-1] * (4 - kept)
    want, n, end = d.generated.tolist(), length, bool(stopped)
    for t in ([tokens[i] for i in path[1:kept]] + [following])[:kept]:
        if (stop and end) or n >= 8 or t < 0:
            break
        want[n] = t
        n, end = n + 1, end or t == 1
    i32 = dict(dtype=torch.int32, device=device)
    d._store_path(torch.tensor(tokens, device=device), torch.tensor(path, **i32), torch.tensor([kept], **i32),
                  torch.tensor([following], device=device))
    assert d.generated.tolist() == want and int(d.length) == n and int(d.position) == 20 + kept
    assert int(d.next_token) == (following if kept else tokens[0])
    if stop:
        assert bool(int(d.stopped)) == end


def test_replays_of_two_graphs_are_the_eager_steps(weights, device):
    """A chain's and a tree's graph of one decoder in turn, with eager steps and other work between, bit for bit."""
    trees = [TREES["chain"], TREES["bush"]]
    g = torch.Generator().manual_seed(3)
    steps = [(k, torch.randint(0, 1000, (len(trees[k]) - 1,), generator=g).to(device)) for k in (0, 1, 1, 0, 1, 0, 0, 1)]
    runs = []
    for graphs in (False, True):
        d = decoder(weights)
        up = [torch.tensor(t, dtype=torch.int32, device=device) for t in trees]
        bufs = [torch.zeros(len(t) - 1, dtype=torch.int64, device=device) for t in trees]
        with pytest.raises(RuntimeError):  # not without its workspace
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                d.tree_step(bufs[0])
        d.prefill_chunked(prompt(50))
        captured = []
        if graphs:
            saved = d._save_state()
            side = torch.cuda.Stream(device=device)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for b, p in zip(bufs, up):
                    d.tree_step(b, parents=p)
            torch.cuda.current_stream().wait_stream(side)
            for b, p in zip(bufs, up):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    d.tree_step(b, parents=p)
                captured.append(graph)
            d._restore_state(saved)
        for i, (k, drafts) in enumerate(steps):
            bufs[k].copy_(drafts)
            bufs[k][0] = d.generated[:1].expand(1)[0] if i % 3 else drafts[0]
            if graphs:
                captured[k].replay()
            else:
                d.tree_step(bufs[k], parents=up[k])
            if i == 3:
                d.decode_step()
            torch.randn(512, 512, device=device).sum().item()
        n = int(d.position)
        runs.append((d.generated.clone(), d.position.clone(), d.next_token.clone(), d.k_cache[:, :n].clone(), d.v_cache[:, :n].clone()))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def reference_gaps(weights, ids, tokens):
    """How far each token's logit lies below the largest after the tokens before it, in the logits' rms."""
    d = decoder(weights)
    d.prefill_chunked(ids)
    gaps, logits = [], d.logits()
    for i, t in enumerate(tokens):
        gaps.append(float((logits.max() - logits[t]) / logits.pow(2).mean().sqrt()))
        logits = feed(d, [t], ids.numel() + i)
    return gaps


@pytest.mark.parametrize("how", ["nothing", "good", "random"])
def test_generation_is_greedy_whatever_is_drafted(weights, how):
    """Two logits that are each off by 5 sigma of CLOSE * rms can change places: a token's lies at most 2 * 5 * CLOSE = 0.5 rms
    below the largest (of 1024 values that is 3 rms above their mean)."""
    ids, calls = prompt(40, 7), []
    other = decoder(weights)
    g = torch.Generator().manual_seed(11)

    def draft(text):
        calls.append(len(text))
        if how == "nothing":
            return [], None
        if how == "random":
            m = int(torch.randint(0, 64, (1,), generator=g))
            return torch.randint(0, 1024, (m,), generator=g).tolist(), [int(torch.randint(-1, i, (1,), generator=g)) if i else -1
                                                                        for i in range(m)]
        # the continuation that one-token steps choose, on nodes 1, 3, 5 .. with wrong siblings between
        line = other.generate(torch.tensor(text), 6, use_graph=False, prefill_chunk=512)
        return [t for x in line for t in ((x + 1) % 1024, x)], [p for i in range(6) for p in (2 * i - 1, 2 * i - 1)]

    d = decoder(weights)
    got = d.generate_tree(ids, 40, draft)
    assert len(got) == 40
    assert max(reference_gaps(weights, ids, got)) < 0.5
    assert len(calls) <= (39 if how != "good" else 13)
    if how == "nothing":
        assert len(calls) == 39


def test_generation_ends_with_the_text(weights):
    ids = prompt(40, 7)
    d = decoder(weights)
    free = d.generate_tree(ids, 30, lambda text: ([3, 4, 5], None))
    d.stop_on_eos = True
    d.eos = torch.tensor([free[12]], device=d.device)
    assert d.generate_tree(ids, 30, lambda text: ([3, 4, 5], None)) == free[:free.index(free[12]) + 1]


def test_drawn_tokens_follow_the_logits_and_the_numbers(weights, device):
    """A step without drafts draws by the inverse of the row's summed probabilities; a seed gives the same text again."""
    d = decoder(weights)
    d.prefill_chunked(prompt(30))
    for u in (0.0, 0.123, 0.5, 0.987):
        _, kept, logits = d.tree_step(torch.empty(0, dtype=torch.int64, device=device), temperature=0.7,
                                      uniforms=torch.tensor([u], device=device))
        upto = torch.softmax(logits[0].double() / 0.7, -1).cumsum(0)
        t = int(d.next_token)
        u = float(torch.tensor(u))
        assert int(kept) == 1 and (upto[t - 1] if t else 0.0) <= u + 1e-9 and u < upto[t] + 1e-9
    texts = []
    for seed in (1, 1, 2):
        g = torch.Generator(device=device).manual_seed(seed)
        texts.append(d.generate_tree(prompt(30), 20, lambda text: ([7, 8, 9], [-1, -1, 1]), temperature=1.0, generator=g))
    assert texts[0] == texts[1] != texts[2] and len(texts[0]) == 20


def test_drawn_drafts_of_the_same_model_are_all_accepted(weights, device):
    """Drafts drawn from this model's own logits have p = q to CLOSE: at uniforms of 0.5, u q < p holds for each."""
    d, b = decoder(weights), decoder(weights)
    for x in (d, b):
        x.prefill_chunked(prompt(30))
    tokens, rows = [int(d.next_token)], []
    for _ in range(4):
        rows.append(feed(b, tokens, 30))
        tokens.append(int(rows[-1].topk(2).indices[1]))
    path, kept, _ = d.tree_step(torch.tensor(tokens[1:], device=device), temperature=1.0, draft_logits=torch.stack(rows),
                                uniforms=torch.full((5,), 0.5, device=device))
    assert path.tolist() == [0, 1, 2, 3, 4] and d.generated[1:5].tolist() == tokens[1:]


def test_the_first_nodes_parent_is_not_looked_at(weights, device):
    runs = []
    for first in (-1, 0, 7):
        d = decoder(weights)
        d.prefill_chunked(prompt(30))
        up = torch.tensor([first, 0, 0, 1], dtype=torch.int32, device=device)
        runs.append([t.clone() for t in d.tree_step(torch.tensor([5, 6, 7], device=device), parents=up)])
        assert up[0] == first
    for run in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(run, runs[0]))


@pytest.mark.parametrize("room", [1, 3])
def test_nodes_without_a_slot(weights, device, room):
    """At the end of the cache a chain is as long as what is left, and rows before it stay."""
    a, b = decoder(weights, 40), decoder(weights, 40 - room + 8)
    for d in (a, b):
        d.prefill_chunked(prompt(40 - room))
    before = a.k_cache[:, :40 - room].clone()
    _, kept, logits = a.tree_step(torch.tensor([1, 2, 3, 4, 5, 6, 7], device=device))
    _, _, want = b.tree_step(torch.tensor([1, 2, 3, 4, 5, 6, 7], device=device))
    assert torch.equal(logits[:room], want[:room]) and 1 <= int(kept) <= room
    assert torch.equal(a.k_cache[:, :40 - room], before)
    a.position.fill_(40)
    stored = a.generated.clone()
    _, kept, _ = a.tree_step(torch.tensor([1], device=device))
    assert int(kept) == 0 and int(a.position) == 40 and torch.equal(a.generated, stored)


def test_refusals(weights, device):
    d = decoder(weights, 64)
    i32 = dict(dtype=torch.int32, device=device)
    some = torch.tensor([1, 2], device=device)
    for drafts, more in [(some.int(), {}), (some.view(1, 2), {}), (some.cpu(), {}), ([1, 2], {}),
                         (torch.zeros(64, dtype=torch.int64, device=device), {}), (some, dict(temperature=1.0)),
                         (some, dict(parents=torch.zeros(2, **i32))), (some, dict(uniforms=torch.zeros(2, device=device))),
                         (some, dict(draft_logits=torch.zeros(3, 1024, device=device))),
                         (some, dict(temperature=-1.0, uniforms=torch.zeros(3, device=device))),
                         (some, dict(parents=torch.zeros(3, **i32), draft_logits=torch.zeros(2, 1024, device=device)))]:
        with pytest.raises(ValueError):
            d.tree_step(drafts, **more)
    with pytest.raises(NotImplementedError):
        decoder(weights, 64, kv_bits=8).tree_step(some)
    with pytest.raises(NotImplementedError):
        decoder(weights, 64, kv_bits=8).generate_tree(prompt(5), 4, lambda text: ([], None))
    for n, new, draft, more in [(50, 20, lambda t: ([], None), {}), (5, 0, lambda t: ([], None), {}), (5, 65, lambda t: ([], None), {}),
                                (5, 4, lambda t: ([1] * 64, None), {}), (5, 4, lambda t: ([1024], None), {}),
                                (5, 4, lambda t: ([1, 2], [-1, 1]), {}), (5, 4, lambda t: ([1, 2], [-1]), {}),
                                (5, 4, lambda t: ([], None), dict(temperature=float("inf")))]:
        with pytest.raises(ValueError):
            d.generate_tree(prompt(n), new, draft, **more)


def test_steps_of_all_sizes_share_one_workspace(weights, device):
    """Chains of 1 to 64 nodes, largest, smallest and back, as a fresh decoder's each."""
    d = decoder(weights)
    for n in (64, 1, 9, 33, 2, 17, 64, 5):
        one = decoder(weights)
        runs = []
        for x in (d, one):
            x.prefill_chunked(prompt(100))
            runs.append(x.tree_step(prompt(n - 1, n).to(device)) if n > 1 else x.tree_step(torch.empty(0, dtype=torch.int64, device=device)))
        assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("policy", ["uniform", "q4_k_m"])
def test_steps_of_a_persistent_decoder_between_its_own(device, policy):
    """Tree steps and one-token steps of the persistent launch in turn over one cache: each node's logits are those after its
    ancestors one by one, and the text is greedy."""
    from dataclasses import replace

    from torch2vk_amd.qwen3.config import QWEN3_0_6B
    from torch2vk_amd.qwen3.model import Qwen3Decoder
    from torch2vk_amd.qwen3.weights import synthetic_weights

    cfg = replace(QWEN3_0_6B, layers=2, vocab=4096, eos_token_ids=(4095,))
    w = synthetic_weights(cfg, device=device, seed=12, std=0.02, norm_std=0.1, policy=policy)
    d, one = Qwen3Decoder(w, max_positions=256, max_new_tokens=64, persistent=True), decoder(w)
    d.stop_on_eos = False
    assert d.persistent
    ids, parents = prompt(60, 3), TREES["bush"]
    d.prefill_chunked(ids)
    decided = 1
    for turn in range(6):
        if turn % 2:
            d.decode_step()
            decided += 1
        else:
            at = int(d.position)
            one.k_cache.copy_(d.k_cache)
            one.v_cache.copy_(d.v_cache)
            drafts = prompt(len(parents), 20 + turn).tolist()
            drafts[0] = int(d.next_token)
            for i in ancestors(parents, len(parents) - 1)[1:]:
                drafts[i] = int(feed(one, [drafts[j] for j in ancestors(parents, parents[i])], at).argmax())
            _, kept, logits = d.tree_step(torch.tensor(drafts[1:], device=device),
                                          parents=torch.tensor(parents, dtype=torch.int32, device=device))
            for i in range(len(parents)):
                near(logits[i], feed(one, [drafts[j] for j in ancestors(parents, i)], at))
            decided += int(kept)
        assert int(d.length) == decided and int(d.position) == 60 + decided - 1
    d.check_status()
    assert max(reference_gaps(w, ids, d.generated[:decided].tolist())) < 0.5  # (as for generation above)
