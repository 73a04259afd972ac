"""Trees of drafted tokens on the GPU: attention over a cache, verification and keeping the accepted rows, against their
definitions in 64 bits (include/t2h.h, "trees of drafted tokens")."""

from __future__ import annotations

import math

import pytest
import torch

from torch2vk_amd import kernels as K

pytestmark = pytest.mark.gpu

D, EPS, THETA = 128, 1e-6, 1e6
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF_BF16 = torch.finfo(BF).eps / 2  # a rounding to bf16, relative to the value


# ------------------------------------------------------------------------------------------------- attention


def lineage(parents, i):
    """Node i and its ancestors, or nothing where one of them is no node."""
    line = [i]
    while True:
        up = parents[line[-1]]
        if up == -1:
            return line
        if not 0 <= up < line[-1]:
            return []
        line.append(up)


def norm_rope(x, w, pos, theta):
    """fp64 [rows, heads, D] at positions [rows]."""
    x = x.to(F64)
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.to(F64)
    if theta <= 0:
        return x
    freq = float(theta) ** (-torch.arange(D // 2, dtype=F64, device=x.device) / (D // 2))
    a = (pos.to(F64)[:, None] * freq)[:, None]
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)


class Call:
    """Inputs of one attn_tree call; slots behind each length hold NaN."""

    def __init__(self, device, n_seq, n, nh, nk, lens, s_cap, parents="tree", counts=None, norms=True, theta=THETA, seed=0,
                 spread=1.0, pad=0):
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)

        def rows(*shape):
            return torch.randn(shape, generator=gen, device=device)

        self.n_seq, self.n, self.nh, self.nk, self.s_cap, self.theta = n_seq, n, nh, nk, s_cap, theta
        self.lens = list(lens)
        self.lengths = torch.tensor(self.lens, dtype=torch.int32, device=device)
        host = torch.Generator().manual_seed(seed)
        if parents == "chain":
            up = (torch.arange(n) - 1).expand(n_seq, n)
        elif parents == "roots":
            up = torch.full((n_seq, n), -1)
        elif isinstance(parents, str):
            up = (torch.rand(n_seq, n, generator=host) * (torch.arange(n) + 1)).long() - 1
        else:
            up = torch.tensor(parents).expand(n_seq, n)
        self.up = up.tolist()
        self.parents = up.to(torch.int32).contiguous().to(device)
        self.counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=device)
        self.k_cache = torch.full((n_seq, s_cap, nk, D), math.nan, dtype=BF, device=device)
        self.v_cache = torch.full((n_seq, s_cap, nk, D), math.nan, dtype=BF, device=device)
        for i, at in enumerate(self.lens):
            if 0 < at <= s_cap:
                self.k_cache[i, :at] = rows(at, nk, D) * spread
                self.v_cache[i, :at] = rows(at, nk, D) * spread
        self.wide = rows(n_seq * n, (nh + 2 * nk) * D + pad) * 1.5
        self.q = self.wide[:, :nh * D]
        self.k = self.wide[:, nh * D:(nh + nk) * D]
        self.v = self.wide[:, (nh + nk) * D:(nh + 2 * nk) * D]
        self.norms = {} if not norms else dict(q_norm_weight=1 + 0.3 * rows(D), k_norm_weight=1 + 0.3 * rows(D))
        self.out = torch.full((n_seq, n, nh, D), 7.0, dtype=BF, device=device)
        self.workspace = K.attn_tree_workspace(n_seq, n, nh, nk, D, s_cap, device)

    def nodes(self, i):
        """(node, lineage) of sequence i's nodes."""
        at = self.lens[i]
        if not 0 <= at <= self.s_cap:
            return []
        count = self.n if self.counts is None else max(0, min(self.n, int(self.counts[i])))
        lines = ((t, lineage(self.up[i], t)) for t in range(min(count, self.s_cap - at)))
        return [(t, x) for t, x in lines if x]

    def run(self, chain=False):
        K.attn_tree(self.q, self.k, self.v, self.k_cache, self.v_cache, self.out, self.lengths, self.workspace, theta=self.theta,
                    parents=None if chain else self.parents, counts=self.counts, eps=EPS, **self.norms)
        return self.out

    def check(self, before, what=""):
        """The call's outputs; ``before``: copies of the caches."""
        w = self.norms
        for i in range(self.n_seq):
            nodes, at = self.nodes(i), self.lens[i]
            mine = {t for t, _ in nodes}
            rest = [t for t in range(self.n) if t not in mine]
            assert (self.out[i, rest] == 0).all(), f"{what}: rows that are no nodes, sequence {i}"
            written = torch.zeros(self.s_cap, dtype=torch.bool, device=self.out.device)
            if nodes:
                written[[at + t for t in mine]] = True
            for cache, old in zip((self.k_cache, self.v_cache), before):
                same = cache[i, ~written].view(torch.int16) == old[i, ~written].view(torch.int16)
                assert same.all(), f"{what}: other slots changed, sequence {i}"
            if not nodes:
                continue
            idx = torch.tensor([i * self.n + t for t, _ in nodes], device=self.out.device)
            pos = torch.tensor([at + len(x) - 1 for _, x in nodes], device=self.out.device)
            slots = [at + t for t, _ in nodes]
            q = norm_rope(self.q[idx].reshape(-1, self.nh, D), w.get("q_norm_weight"), pos, self.theta)
            k = norm_rope(self.k[idx].reshape(-1, self.nk, D), w.get("k_norm_weight"), pos, self.theta)
            got = self.k_cache[i, slots].to(F64)
            # half a step, and what 32 bits leave of norm and rotation: a sum of 128 squares, a root, two products and their sum
            tol = HALF_BF16 * 1.01 * k.abs() + 2.0 ** -18 * (k.abs() + k.roll(D // 2, -1).abs()) + 1e-30
            assert ((got - k).abs() <= tol).all(), f"{what}: k rows of sequence {i}"
            assert torch.equal(self.v_cache[i, slots], self.v[idx].reshape(-1, self.nk, D).to(BF)), f"{what}: v rows of {i}"
            keys, values = self.k_cache[i].to(F64), self.v_cache[i].to(F64)
            for r, (t, line) in enumerate(nodes):
                seen = torch.cat([torch.arange(at), torch.tensor(sorted(at + j for j in line))]).to(self.out.device)
                ks, vs = keys[seen].transpose(0, 1), values[seen].transpose(0, 1)  # [nk, seen, D]
                g = q[r].reshape(self.nk, -1, D)
                score = torch.matmul(g, ks.transpose(1, 2)) / math.sqrt(D)
                mass_qk = float(torch.matmul(g.abs(), ks.abs().transpose(1, 2)).max()) / math.sqrt(D)
                p = torch.softmax(score, -1)
                ref, mass_v = torch.matmul(p, vs), torch.matmul(p, vs.abs())
                # half a step of the output's; each p in bf16; p's relative error from scores: q in two bf16 terms (2^-16), 32-bit
                # products and sums of 128 terms (2^-17), in the numerator and in the sum
                tol = HALF_BF16 * 1.01 * ref.abs() + (HALF_BF16 * 1.01 + 2.0 ** -14 * mass_qk) * mass_v + 1e-30
                off = (self.out[i, t].reshape(self.nk, -1, D).to(F64) - ref).abs() / tol
                assert (off <= 1).all(), f"{what}: sequence {i}, node {t}: {float(off.max()):.2f} of the tolerance"


def checked(c, what="", **kw):
    before = (c.k_cache.clone(), c.v_cache.clone())
    c.run(**kw)
    c.check(before, what)


@pytest.mark.parametrize("n", [1, 2, 5, 8, 13, 16, 17, 31, 33, 64])
@pytest.mark.parametrize("nh,nk", [(16, 8), (32, 8), (20, 4), (16, 1)])
def test_attention_of_a_tree(device, n, nh, nk):
    checked(Call(device, 3, n, nh, nk, [200, 0, 77], 300, seed=n * nh + nk))


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 30, 31, 32, 33, 62, 63, 64, 65, 95, 97, 127, 128, 129, 255, 257, 1000])
def test_attention_around_tile_borders(device, length):
    for n, nh, nk in ((1, 8, 8), (7, 16, 8), (64, 32, 8)):
        checked(Call(device, 1, n, nh, nk, [length], length + n, seed=length + n), f"{n} nodes at {length}")


@pytest.mark.parametrize("n,nh,nk", [(3, 32, 8), (12, 32, 4), (26, 32, 8), (64, 32, 8), (40, 32, 2), (64, 16, 1)])
def test_attention_of_a_ragged_batch_of_long_contexts(device, n, nh, nk):
    lens = [4100, 1, 7001, 333, 0, 2048]
    checked(Call(device, 6, n, nh, nk, lens, 7200, counts=[n, n // 2, n, 1, n, 0], seed=n))


def test_attention_of_a_batch_of_more_than_64_sequences(device):
    lens = [(37 * i) % 400 for i in range(131)]
    checked(Call(device, 131, 3, 4, 2, lens, 420, counts=[i % 4 for i in range(131)], seed=5))


@pytest.mark.parametrize("n,nk", [(5, 2), (9, 2), (13, 1), (40, 2)])
def test_units_of_more_than_64_sequences_come_from_the_table(device, n, nk):
    """40 to 320 rows a KV head: units of 131 sequences, some of them empty, laid out 64 at a time."""
    lens = [(37 * i) % 400 for i in range(131)]
    checked(Call(device, 131, n, 16, nk, lens, 440, counts=[(3 * i) % (n + 1) for i in range(131)], seed=6))

def test_attention_of_one_very_long_context(device):
    checked(Call(device, 1, 9, 8, 1, [100_003], 100_100, seed=1))


@pytest.mark.parametrize("n,nh,nk", [(1, 8, 8), (8, 16, 8), (7, 32, 8), (12, 32, 8), (31, 32, 8)])
@pytest.mark.parametrize("length", [1, 40, 700, 5000])
def test_weights_of_up_to_128_rows_are_not_rounded_to_bf16(device, n, nh, nk, length):
    """Scores near 0, so that they add next to nothing: an output is off by half a step of its own, and by what two terms leave of
    a weight: 2^-8 of a rest that is less than 2^-7 of it, 2^-19 that 32-bit exponentials, sums and the rest's own 2^-20 take."""
    c = Call(device, 1, n, nh, nk, [length], length + n, norms=False, theta=0.0, seed=length + n)
    c.q *= 0.02
    c.k *= 0.5
    c.run()
    keys, values = c.k_cache[0].to(F64), c.v_cache[0].to(F64)
    for t, line in c.nodes(0):
        seen = torch.cat([torch.arange(length), torch.tensor(sorted(length + j for j in line))]).to(device)
        ks, vs = keys[seen].transpose(0, 1), values[seen].transpose(0, 1)
        q = c.q[t].reshape(nk, -1, D).to(F64)
        p = torch.softmax(torch.matmul(q, ks.transpose(1, 2)) / math.sqrt(D), -1)
        mass_qk = float(torch.matmul(q.abs(), ks.abs().transpose(1, 2)).max()) / math.sqrt(D)
        ref, mass_v = torch.matmul(p, vs), torch.matmul(p, vs.abs())
        tol = HALF_BF16 * 1.01 * ref.abs() + (2.0 ** -15 + 2.0 ** -19 + 2.0 ** -14 * mass_qk) * mass_v
        off = (c.out[0, t].reshape(nk, -1, D).to(F64) - ref).abs() / tol
        assert (off <= 1).all(), f"node {t}: {float(off.max()):.2f} of the tolerance"

def test_attention_without_norms_and_without_rotation(device):
    checked(Call(device, 2, 6, 16, 8, [50, 300], 400, norms=False, theta=0.0, seed=2))
    checked(Call(device, 2, 6, 16, 8, [50, 300], 400, norms=False, seed=3))


def test_rows_of_a_wider_product_and_a_far_position(device):
    checked(Call(device, 2, 5, 16, 8, [41_000, 40_321], 41_100, pad=37, seed=4))


def test_no_parents_is_a_chain(device):
    a, b = (Call(device, 2, 9, 16, 8, [70, 130], 200, parents="chain", counts=[9, 4], seed=6) for _ in range(2))
    checked(a, chain=True)
    b.run()
    assert torch.equal(a.out, b.out) and torch.equal(a.k_cache.view(torch.int16), b.k_cache.view(torch.int16))


def test_a_chain_of_one_is_the_decode_step(device):
    c = Call(device, 1, 1, 16, 8, [321], 400, seed=7)
    c.k_cache[:, 321:] = 0
    c.v_cache[:, 321:] = 0
    k, v, out = c.k_cache[0].clone(), c.v_cache[0].clone(), torch.empty(16 * D, dtype=BF, device=device)
    K.attn_decode(c.q.reshape(-1).contiguous(), c.k.reshape(-1).contiguous(), c.v.reshape(-1).contiguous(), k, v, out,
                  torch.tensor([321], dtype=torch.int32, device=device), K.attn_decode_workspace(16, 8, D, 400, device),
                  theta=THETA, eps=EPS, **c.norms)
    checked(c)
    far = (c.out.reshape(-1).float() - out.float()).norm() / out.float().norm()
    assert far < 3 * HALF_BF16  # two outputs' roundings, and the angle of a 32-bit product there


def test_nodes_that_hang_on_no_node_are_none(device):
    parents = [-1, 0, 5, 2, 3, -7, 1, 6, 8, 8, 9]  # 2 hangs on a later one, 3 and 4 on it, 5 on nothing, 8 on itself
    checked(Call(device, 2, 11, 16, 8, [100, 33], 150, parents=parents, seed=8))


def test_no_slot_no_node(device):
    checked(Call(device, 4, 10, 16, 8, [95, 100, 90, 99], 100, parents="roots", seed=9))


def test_lengths_outside_the_cache_take_no_part(device):
    checked(Call(device, 4, 4, 16, 8, [-1, 101, 20, 1 << 30], 100, counts=[4, 4, 4, 4], seed=10))


def test_counts_are_clamped(device):
    checked(Call(device, 4, 4, 16, 8, [10, 20, 30, 40], 100, counts=[-3, 0, 99, 1], seed=11))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n", [6, 30, 64])
def test_what_is_not_finite_reaches_the_rows_that_see_it(device, bad, n):
    """One node's value: its own dimension of the rows below it.  One node's key: the rows below it whole.  Others: bit for bit
    as without."""
    parents = [-1, 0, 0, 1, 2, 2] + [(i * 7) % 6 for i in range(6, n)]
    for part in ("v", "k"):
        clean, c = (Call(device, 2, n, 16, 8, [70, 5], 200, parents=parents, seed=12) for _ in range(2))
        getattr(c, part)[2, 3 * D + 17] = bad  # node 2 of sequence 0, KV head 3
        clean.run()
        c.run()
        below = [t for t in range(n) if 2 in lineage(parents, t)]
        hit = torch.zeros_like(c.out, dtype=torch.bool)
        for t in below:
            if part == "v":
                hit[0, t, 6:8, 17] = True
            else:
                hit[0, t, 6:8] = True
        assert torch.equal(c.out[~hit], clean.out[~hit]), f"{part}: other rows changed"
        if part == "v":
            want = torch.full_like(c.out[hit], bad)
            assert torch.equal(c.out[hit].isnan(), want.isnan()) and torch.equal(c.out[hit].nan_to_num(), want.nan_to_num())
        else:
            assert c.out[hit].isnan().all()  # the norm of a row with an infinity or a NaN leaves NaN


@pytest.mark.parametrize("length", [230, 255, 256, 480])
def test_what_is_not_finite_in_trees_that_lie_across_units(device, length):
    parents = [-1, 0, 0] + [(i - 1) // 2 for i in range(3, 64)]
    clean, c = (Call(device, 1, 64, 16, 1, [length], 600, parents=parents, seed=18) for _ in range(2))
    for node, bad in ((1, math.inf), (2, -math.inf), (40, math.nan), (63, math.inf)):
        c.v[node, 64 + node] = bad
    clean.run()
    c.run()
    for t in range(64):
        line = lineage(parents, t)
        for node, bad in ((1, math.inf), (2, -math.inf), (40, math.nan), (63, math.inf)):
            got = c.out[0, t, :, 64 + node].float()
            if node in line:
                assert got.isnan().all() if math.isnan(bad) else (got == bad).all(), (t, node)
                c.out[0, t, :, 64 + node] = clean.out[0, t, :, 64 + node]
    assert torch.equal(c.out, clean.out)


def test_an_infinity_of_each_sign_on_one_path_is_a_nan(device):
    c = Call(device, 1, 5, 8, 8, [40], 64, parents=[-1, 0, 0, 1, 2], seed=13)
    c.v[1, 5], c.v[2, 5], c.v[3, 5] = math.inf, math.inf, -math.inf
    c.run()
    got = c.out[0, :, 0, 5].float().tolist()
    assert math.isfinite(got[0]) and got[1] == math.inf and got[2] == math.inf and math.isnan(got[3]) and got[4] == math.inf
    assert torch.isfinite(c.out[0, :, 1:]).all()


def test_a_cached_value_that_is_not_finite_reaches_all_rows(device):
    c = Call(device, 2, 20, 16, 8, [300, 300], 400, seed=14)
    c.v_cache[0, 17, 2, 9] = math.inf
    c.run()
    assert (c.out[0, :, 4:6, 9] == math.inf).all()
    c.out[0, :, 4:6, 9] = 0
    assert torch.isfinite(c.out).all()


def test_large_and_small_scores(device):
    checked(Call(device, 1, 20, 16, 8, [500], 600, norms=False, spread=30.0, seed=15))
    c = Call(device, 1, 20, 16, 8, [500], 600, norms=False, seed=16)
    c.wide *= 1e-20
    checked(c)


def test_sequences_of_a_layer_major_cache(device):
    """Views whose sequences lie apart, as one layer of [n_seq, layers, s_cap, nk, d], K and V unlike."""
    c = Call(device, 3, 7, 16, 8, [90, 0, 33], 128, seed=17)
    whole_k = torch.zeros(3, 4, 128, 8, D, dtype=BF, device=device)
    whole_v = torch.zeros(4, 3, 128, 8, D, dtype=BF, device=device)
    whole_k[:, 2], whole_v[1] = c.k_cache, c.v_cache
    c.k_cache, c.v_cache = whole_k[:, 2], whole_v[1]
    checked(c)
    assert (whole_k[:, [0, 1, 3]] == 0).all() and (whole_v[[0, 2, 3]] == 0).all()


def test_places_past_32_bits(device):
    """The far end of a sequence behind 2^31 elements of another one."""
    s_cap = (1 << 31) // (8 * D) + 5000
    c = Call(device, 1, 1, 8, 8, [0], 64)
    gen = torch.Generator(device=device).manual_seed(3)
    c.n_seq, c.n, c.s_cap = 2, 3, s_cap
    c.k_cache = torch.zeros(2, s_cap, 8, D, dtype=BF, device=device)
    c.v_cache = torch.zeros(2, s_cap, 8, D, dtype=BF, device=device)
    at = s_cap - 9
    for cache in (c.k_cache, c.v_cache):
        cache[1, at - 4000:at] = torch.randn(4000, 8, D, generator=gen, device=device)
    c.lens = [3, at]
    c.lengths = torch.tensor(c.lens, dtype=torch.int32, device=device)
    c.up = [[-1, 0, 0]] * 2
    c.parents = torch.tensor(c.up, dtype=torch.int32, device=device)
    wide = torch.randn(6, 24 * D, generator=gen, device=device)
    c.q, c.k, c.v = wide[:, :8 * D], wide[:, 8 * D:16 * D], wide[:, 16 * D:]
    c.q[3:] *= 8  # scores that reach past two million keys of zero
    c.norms = {}
    c.theta = 0.0
    c.out = torch.empty(2, 3, 8, D, dtype=BF, device=device)
    c.workspace = K.attn_tree_workspace(2, 3, 8, 8, D, s_cap, device)
    c.run()
    keys, values = c.k_cache[1, :at + 3].to(F64), c.v_cache[1, :at + 3].to(F64)
    for t, line in enumerate(([0], [0, 1], [0, 2])):
        q = c.q[3 + t].reshape(8, 1, D).to(F64)
        score = torch.matmul(q, keys.permute(1, 2, 0)) / math.sqrt(D)
        score[:, :, [at + j for j in range(3) if j not in line]] = -math.inf
        p = torch.softmax(score, -1)
        ref = torch.matmul(p, values.transpose(0, 1))[:, 0]
        mass_v = torch.matmul(p, values.abs().transpose(0, 1))[:, 0]
        mass_qk = float(torch.matmul(q.abs(), keys.abs().permute(1, 2, 0)).max()) / math.sqrt(D)
        tol = HALF_BF16 * 1.01 * ref.abs() + (HALF_BF16 * 1.01 + 2.0 ** -14 * mass_qk) * mass_v
        assert ((c.out[1, t].to(F64) - ref).abs() <= tol).all()


def test_one_workspace_serves_several_shapes(device):
    shapes = [(4, 64, 32, 8, 600), (1, 3, 16, 8, 2000), (9, 5, 8, 1, 900), (1, 64, 16, 1, 1200)]
    most = max((K.attn_tree_workspace(b, n, nh, nk, D, cap, device) for b, n, nh, nk, cap in shapes), key=torch.numel)
    for turn in range(2):
        for i, (b, n, nh, nk, cap) in enumerate(shapes):
            c = Call(device, b, n, nh, nk, [(cap - n) // (j + 1) for j in range(b)], cap, seed=20 + i)
            c.workspace = most
            checked(c, f"turn {turn}, shape {i}")


def test_the_same_call_gives_the_same_bits(device):
    c = Call(device, 3, 26, 32, 8, [3000, 500, 77], 3100, seed=30)
    first = c.run().clone()
    for _ in range(5):
        assert torch.equal(c.run(), first)


def test_attention_on_another_stream(device):
    c, e = (Call(device, 2, 12, 16, 8, [700, 90], 800, seed=31) for _ in range(2))
    e.run()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        c.run()
    torch.cuda.current_stream(device).wait_stream(side)
    assert torch.equal(c.out, e.out)


def test_a_captured_call_follows_lengths_counts_and_parents(device):
    c = Call(device, 2, 8, 16, 8, [100, 100], 600, seed=32, counts=[8, 8])
    c.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run()
    for i, lens in enumerate(([90, 3], [599, 0], [500, 412], [-1, 600])):
        e = Call(device, 2, 8, 16, 8, lens, 600, seed=40 + i, counts=[8, 3 + i])
        for name in ("k_cache", "v_cache", "wide", "lengths", "parents", "counts"):
            getattr(c, name).copy_(getattr(e, name))
        for name in c.norms:
            c.norms[name].copy_(e.norms[name])
        g.replay()
        e.run()
        torch.cuda.synchronize()
        assert torch.equal(c.out, e.out) and torch.equal(c.k_cache.view(torch.int16), e.k_cache.view(torch.int16))


def test_attention_refusals(device):
    c = Call(device, 2, 4, 16, 8, [10, 20], 64, seed=33)

    def call(**kw):
        a = dict(q=c.q, k_new=c.k, v_new=c.v, k_cache=c.k_cache, v_cache=c.v_cache, out=c.out, lengths=c.lengths,
                 workspace=c.workspace, theta=THETA, parents=c.parents, counts=c.counts, **c.norms)
        K.attn_tree(**(a | kw))

    wrong = [
        (ValueError, dict(q=c.q.cpu())), (TypeError, dict(q=c.q.to(BF))), (TypeError, dict(q=None)),
        (ValueError, dict(q=c.q[:7])), (ValueError, dict(q=c.q[:, :100])), (ValueError, dict(q=c.q.t())),
        (ValueError, dict(k_new=c.k[:, :7 * D])), (ValueError, dict(v_new=c.v[:6])), (ValueError, dict(q=c.q[:1].expand(8, -1))),
        (TypeError, dict(k_cache=c.k_cache.float())), (ValueError, dict(v_cache=c.v_cache[:1])),
        (ValueError, dict(v_cache=c.v_cache[:, :60])), (ValueError, dict(k_cache=c.k_cache.transpose(1, 2))),
        (ValueError, dict(k_cache=c.k_cache[:1].expand(2, -1, -1, -1))), (ValueError, dict(k_cache=c.k_cache[0])),
        (TypeError, dict(out=c.out.float())), (ValueError, dict(out=c.out[:1])), (TypeError, dict(out=None)),
        (TypeError, dict(lengths=c.lengths.long())), (ValueError, dict(lengths=c.lengths[:1])), (TypeError, dict(lengths=None)),
        (TypeError, dict(parents=c.parents.long())), (ValueError, dict(parents=c.parents[:1])),
        (ValueError, dict(counts=c.lengths[:1])), (ValueError, dict(counts=c.lengths.cpu())),
        (TypeError, dict(workspace=c.workspace.float())), (ValueError, dict(q_norm_weight=None)),
        (ValueError, dict(k_norm_weight=torch.ones(64, device=device))),
    ]
    for error, kw in wrong:
        with pytest.raises(error):
            call(**kw)
    with pytest.raises(RuntimeError):
        call(workspace=c.workspace[:16])
    big = torch.zeros(2 * 65, 32 * D, device=device)
    with pytest.raises(ValueError):
        K.attn_tree(big[:, :16 * D], big[:, 16 * D:24 * D], big[:, 24 * D:], c.k_cache, c.v_cache,
                    torch.empty(2, 65, 16, D, dtype=BF, device=device), c.lengths, c.workspace, theta=THETA)
    with pytest.raises(ValueError):
        K.attn_tree_workspace(1, 65, 16, 8, D, 64, device)
    with pytest.raises(ValueError):
        K.attn_tree_workspace(1, 4, 34, 2, D, 64, device)


# ---------------------------------------------------------------------------------------------- verification


def reference(logits, tokens, temps, uniforms, parents=None, counts=None, draft=None):
    """The walk in 64 bits, sequence by sequence, from host copies."""
    b, n, vocab = logits.shape
    logits = torch.where(logits.isnan(), -math.inf, logits.double()).cpu()
    draft = None if draft is None else torch.where(draft.isnan(), -math.inf, draft.double()).cpu()
    tokens, temps = tokens.tolist(), [float(t) for t in temps]
    uniforms = None if uniforms is None else uniforms.double().nan_to_num(0.0).clamp(0.0, 1 - 2.0 ** -24).tolist()
    parents = [list(range(-1, n - 1))] * b if parents is None else parents.tolist()
    counts = [n] * b if counts is None else counts.tolist()

    def probabilities(row, t):
        top = row.max()
        if top == -math.inf:
            return torch.zeros_like(row)
        w = (row == math.inf).double() if top == math.inf else torch.exp((row - top) / t)
        return w / w.sum()

    def of(mass, x):
        return float(mass[x]) if 0 <= x < vocab else 0.0

    path, kept, following = torch.full((b, n), -1, dtype=torch.int32), [], []
    for i in range(b):
        count = max(0, min(n, counts[i]))
        if count == 0:
            kept.append(0)
            following.append(-1)
            continue
        at, line, t = 0, [0], temps[i]
        while True:
            row = logits[i, at]
            children = [j for j in range(at + 1, count) if parents[i][j] == at]
            step = None
            if not t > 0:
                choice = -1 if row.max() == -math.inf else int((row == row.max()).nonzero()[0, 0])
                step = next((j for j in children if choice >= 0 and tokens[i][j] == choice), None)
            else:
                mass = probabilities(row, t)
                plain = mass
                for j in children:
                    x = tokens[i][j]
                    if draft is None:
                        if uniforms[i][j] * float(mass.sum()) < of(mass, x):
                            step = j
                            break
                        mass = mass.clone()
                        if 0 <= x < vocab:
                            mass[x] = 0.0
                    else:
                        q = probabilities(draft[i, at], t)
                        if uniforms[i][j] * of(q, x) < of(mass, x):
                            step = j
                            break
                        mass = torch.clamp(mass - q, min=0.0)
                if step is None:
                    if float(mass.sum()) == 0.0:
                        mass = plain if draft is not None else mass
                    run = torch.cumsum(mass, 0)
                    over = (run > uniforms[i][0] * float(run[-1])).nonzero()
                    some = (mass > 0).nonzero()
                    choice = int(over[0, 0]) if len(over) else (int(some[-1, 0]) if len(some) else -1)
            if step is None:
                break
            at = step
            line.append(at)
        path[i, :len(line)] = torch.tensor(line, dtype=torch.int32)
        kept.append(len(line))
        following.append(choice)
    return path, torch.tensor(kept, dtype=torch.int32), torch.tensor(following)


def verify_inputs(device, b, n, vocab, *, seed=0, dtype=F32, shape="tree", spread=2.0, drawn=False, temperature=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    logits = (torch.randn(b, n, vocab, generator=gen, device=device) * spread).to(dtype)
    up = torch.arange(n).expand(b, n) - 1
    if shape == "tree":
        up = (torch.rand(b, n, generator=host) * torch.arange(n)).long().clamp(max=torch.arange(n) - 1)
    up = up.to(torch.int32).contiguous().to(device)
    likely = logits.float().topk(min(4, vocab), -1).indices  # some drafts right, some wrong, siblings now and then alike
    pick = torch.randint(0, likely.shape[-1], (b, n), generator=gen, device=device)
    rows = torch.gather(likely, 1, up.long().clamp(min=0)[..., None].expand(-1, -1, likely.shape[-1]))
    tokens = torch.gather(rows, 2, pick[..., None])[..., 0].contiguous()
    uniforms = torch.rand(b, n, generator=gen, device=device)
    draft = None
    if drawn:
        draft = (logits[:, :n - 1].float() * 0.8 + torch.randn(b, n - 1, vocab, generator=gen, device=device) * 0.7).to(dtype)
        if n > 1:
            tokens[:, 1:] = torch.distributions.Categorical(logits=(draft.float() / temperature).cpu()).sample().to(device)
    return dict(logits=logits, tokens=tokens, uniforms=uniforms, parents=up, draft=draft)


def verified(x, temps, counts=None, chain=False, **kw):
    """The call's results, equal to the reference's."""
    b, n, vocab = x["logits"].shape
    device = x["logits"].device
    chain = chain or x["draft"] is not None
    ws = kw.pop("workspace", None)
    ws = K.tree_verify_workspace(b, n, vocab, device, drawn=x["draft"] is not None) if ws is None else ws
    got = K.tree_verify(x["logits"], x["tokens"], ws, temperature=temps, uniforms=x["uniforms"], counts=counts,
                        parents=None if chain else x["parents"], draft_logits=x["draft"], **kw)
    each = [temps] * b if not isinstance(temps, torch.Tensor) else temps.tolist()
    want = reference(x["logits"], x["tokens"], each, x["uniforms"], None if chain else x["parents"], counts, x["draft"])
    for name, g, w in zip(("path", "kept", "next_token"), got, want):
        assert torch.equal(g.cpu(), w), f"{name}: {g.tolist()} for {w.tolist()}"
    return got


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 63, 257, 1000, 4099, 32001, 151936])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_verification(device, vocab, dtype):
    for n in (1, 2, 5, 26):
        for t in (0.0, 0.7, 1.0):
            verified(verify_inputs(device, 3, n, vocab, dtype=dtype, seed=vocab + n), t)
        verified(verify_inputs(device, 3, n, vocab, dtype=dtype, seed=vocab + n, drawn=True, temperature=0.9), 0.9)


@pytest.mark.parametrize("mode", ["greedy", "tree", "drawn"])
def test_verification_of_a_ragged_batch(device, mode):
    counts = torch.tensor([9, 0, 1, 5, -2, 64, 9] * 10, dtype=torch.int32, device=device)
    temps = torch.tensor([0.5, 1.0, 2.0, 0.0, 0.1, 1.3, -1.0] * 10, device=device)
    x = verify_inputs(device, 70, 9, 3001, seed=1, drawn=mode == "drawn")
    verified(x, 0.0 if mode == "greedy" else temps, counts)


@pytest.mark.parametrize("n", [33, 64])
def test_verification_of_the_largest_trees(device, n):
    verified(verify_inputs(device, 2, n, 5000, seed=n), 1.5)
    x = verify_inputs(device, 2, n, 5000, seed=n, shape="chain")
    x["logits"][:, :-1].scatter_(2, x["tokens"][:, 1:, None], 40.0)  # a chain accepted to its end
    path, kept, _ = verified(x, 0.8, chain=True)
    assert kept.tolist() == [n, n] and path[0].tolist() == list(range(n))


def test_flat_rows_of_a_large_vocabulary(device):
    """Borders between tokens 1e-5 apart: the sums have to be kept in 64 bits to draw the same token every time."""
    for seed in range(4):
        x = verify_inputs(device, 16, 3, 151936, seed=seed, spread=0.01)
        verified(x, 1.0)
        verified(verify_inputs(device, 16, 3, 151936, seed=seed, spread=0.01, drawn=True), 1.0)


def test_numbers_at_the_borders(device):
    x = verify_inputs(device, 8, 4, 999, seed=2, drawn=True)
    for u in (0.0, 1 - 2.0 ** -24, 1.0, 1.5, -0.5, math.nan, math.inf):
        x["uniforms"] = torch.full((8, 4), u, device=device)
        verified(x, 0.9)
        verified(x | dict(draft=None), 0.9)


def test_logits_without_probability(device):
    """Masked tokens (-inf, NaN), the type's lowest value, rows of nothing else, and infinite ones."""
    for dtype in (F32, BF):
        x = verify_inputs(device, 6, 5, 777, seed=3, dtype=dtype)
        x["logits"][:, :, ::3] = -math.inf
        x["logits"][:, :, 1::7] = math.nan
        x["logits"][0] = -math.inf
        x["logits"][1, 0] = math.nan
        x["logits"][2, :, 5] = math.inf
        x["logits"][2, :, 600] = math.inf
        x["logits"][3, :, 2:] = torch.finfo(dtype).min
        x["logits"][4, 0] = torch.finfo(dtype).min
        for t in (0.0, 0.6):
            _, _, following = verified(x, t)
            assert following[0] == -1 and following[1] == -1
        x["draft"] = x["logits"][:, 1:].clone()
        verified(x, 0.6)
        x["draft"] = torch.full_like(x["draft"], -math.inf)
        verified(x, 0.6)


def test_ties_go_to_the_lowest_index(device):
    for vocab in (5, 300, 20_000):
        x = verify_inputs(device, 3, 3, vocab, seed=4, dtype=BF)
        x["logits"].zero_()
        x["logits"][1, :, vocab // 2:] = 1.0
        x["logits"][2, :, vocab - 1] = 2.0
        x["tokens"][:] = torch.tensor([0, 0, vocab // 2], device=device)
        _, _, following = verified(x, 0.0)
        assert following.tolist() == [0, vocab // 2, vocab - 1]


def test_tokens_outside_the_vocabulary_and_twice(device):
    x = verify_inputs(device, 4, 8, 50, seed=5)
    x["parents"][:] = torch.tensor([-1, 0, 0, 0, 0, 0, 0, 0], device=device)
    x["tokens"][0] = torch.tensor([3, -1, 50, 1 << 40, 7, 7, 7, -(1 << 40)], device=device)
    x["tokens"][1] = x["logits"][1, 0].argmax()  # one sibling seven times
    x["uniforms"][1] = 1 - 2.0 ** -24
    verified(x, 1.0)
    verified(x, 0.0)


def test_parents_that_are_not_of_the_tree(device):
    """Nodes below nothing, below later nodes or below themselves are never asked."""
    x = verify_inputs(device, 3, 9, 40, seed=6)
    x["parents"][:] = torch.tensor([5, -1, 2, 0, 3, 7, 99, -8, 4], device=device)
    verified(x, 1.0)
    verified(x, 0.0)


def test_draft_and_target_alike(device):
    """Nothing is left of max(p - q, 0): the whole chain is accepted."""
    x = verify_inputs(device, 4, 5, 2000, seed=7, drawn=True)
    x["draft"] = x["logits"][:, :4].clone()
    _, kept, _ = verified(x, 1.0)
    assert kept.tolist() == [5] * 4


def beside(border):
    """The fp32 numbers next to a border in (0, 1), one step of the nearest to each side: at least 2^-26 of it off, where sums
    and exponentials in 64 bits are off by 10^-11."""
    near = torch.tensor(border, dtype=F32)
    most = torch.tensor(1 - 2.0 ** -24)
    return float(torch.nextafter(near, torch.tensor(0.0))), float(torch.minimum(torch.nextafter(near, torch.tensor(2.0)), most))


def share(row, t):
    return torch.softmax(row.double().cpu() / t, -1)


@pytest.mark.parametrize("vocab", [8, 1000, 5003, 151936])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_numbers_next_to_the_borders_of_acceptance(device, vocab, dtype):
    """Four children of one node, each accepted or rejected by a step of its number, all 16 ways."""
    b, n = 16, 5
    x = verify_inputs(device, b, n, vocab, seed=60 + vocab, dtype=dtype)
    temps = torch.tensor([1.0, 0.5, 1.5, 0.75] * 4, device=device)
    x["parents"][:] = torch.tensor([-1, 0, 0, 0, 0], device=device)
    for i in range(b):
        x["tokens"][i, 1:] = x["logits"][i, 0].float().topk(8).indices[i % 4:i % 4 + 4]
        mass = share(x["logits"][i, 0], float(temps[i]))
        for j in range(1, n):
            t = int(x["tokens"][i, j])
            under, over = beside(float(mass[t] / mass.sum()))
            x["uniforms"][i, j] = over if i >> (j - 1) & 1 else under
            mass[t] = 0.0
    path, kept, _ = verified(x, temps)
    assert kept.tolist() == [2] * 15 + [1] and [int(p) for p in path[:4, 1]] == [1, 2, 1, 3]


@pytest.mark.parametrize("vocab", [8, 1000, 5003, 151936])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_numbers_next_to_the_borders_of_drawn_drafts(device, vocab, dtype):
    """Chains whose token i is rejected by one step of its number, those before it accepted by one."""
    b, n = 6, 6
    x = verify_inputs(device, b, n, vocab, seed=80 + vocab, dtype=dtype, drawn=True)
    temps = torch.tensor([1.0, 0.5, 1.5, 0.75, 1.0, 2.0], device=device)
    for i in range(b):
        for j in range(1, n):
            p, q = share(x["logits"][i, j - 1], float(temps[i])), share(x["draft"][i, j - 1], float(temps[i]))
            t = int((q - p).argmax())
            x["tokens"][i, j] = t
            under, over = beside(float(p[t] / q[t]))
            x["uniforms"][i, j] = over if j == i + 1 else under
    _, kept, _ = verified(x, temps)
    assert kept.tolist() == [1, 2, 3, 4, 5, 6]


@pytest.mark.parametrize("vocab,first,second", [(2, 0, 1), (5000, 7, 4500), (151936, 3, 150_000)])
def test_a_rejected_token_of_nearly_all_probability(device, vocab, first, second):
    """What is left beside it, 10^-5, is a sum of its own: the second child's 0.9995 lies below its whole probability."""
    x = verify_inputs(device, 2, 3, vocab, seed=90)
    x["logits"][:, 0] = -math.inf
    x["logits"][:, 0, first] = 0.0
    x["logits"][:, 0, second] = math.log(1e-5)
    x["parents"][:] = torch.tensor([-1, 0, 0], device=device)
    x["tokens"][:] = torch.tensor([0, first, second], device=device)
    x["uniforms"][:] = torch.tensor([0.5, 0.999995, 0.9995], device=device)
    path, _, following = verified(x, 1.0)
    assert path.tolist() == [[0, 2, -1]] * 2 and (following >= 0).all()


@pytest.mark.parametrize("spread", [0.01, 2.0, 20.0])
@pytest.mark.parametrize("vocab", [3001, 151936])
def test_children_that_hold_all_of_a_rows_probability(device, vocab, spread):
    """At the largest number each but the last with any probability may be rejected, and that one is not."""
    b, m = 64, 7
    x = verify_inputs(device, b, m + 1, vocab, seed=91)
    gen = torch.Generator().manual_seed(92)
    x["parents"][:] = torch.tensor([-1] + [0] * m, device=device)
    x["logits"][:, 0] = -math.inf
    for i in range(b):
        at = torch.randperm(vocab, generator=gen)[:m].to(device)
        x["logits"][i, 0, at] = torch.randn(m, generator=gen).to(device) * spread
        x["tokens"][i, 1:] = at
    x["uniforms"][:, 1:] = 1 - 2.0 ** -24
    _, kept, following = verified(x, 1.0)
    assert (kept == 2).all() and (following >= 0).all()


@pytest.mark.parametrize("vocab", [1000, 151936])
def test_what_is_left_of_rows_that_are_nearly_the_drafts(device, vocab):
    """Two tokens of 3 * 10^-8 apart from a common row: the rejected one more likely in the draft, the other one less, so that a
    third of what is left is the other one's and the rest everyone's, 10^-8 of each."""
    b, n, a, c = 64, 2, 17, 901
    x = verify_inputs(device, b, n, vocab, seed=93)
    rare = x["logits"][:, 0].logsumexp(-1) + math.log(3e-8)
    x["logits"][:, 0, a] = x["logits"][:, 0, c] = rare
    x["draft"] = x["logits"][:, :1].clone()
    x["draft"][:, 0, a] += 1.0
    x["draft"][:, 0, c] -= 1.0
    x["tokens"][:, 1] = a
    x["uniforms"][:, 1] = 0.5
    _, kept, following = verified(x, 1.0)
    assert (kept == 1).all() and 0 < int((following == c).sum()) < b


def test_what_is_left_where_a_32_bit_sum_loses_its_small_terms(device):
    """Beside a weight of 1 those of 2^-24.1 vanish from a 32-bit sum: rows' quotients are off by more than 10^-6."""
    b, vocab = 32, 151936
    x = verify_inputs(device, b, 2, vocab, seed=94)
    small = -24.1 * math.log(2.0)
    x["logits"][:, 0] = small
    x["draft"] = x["logits"][:, :1].clone()
    x["draft"][:, 0, 0] = 0.0
    at = torch.randperm(vocab, generator=torch.Generator().manual_seed(95))[:40].to(device)
    x["logits"][:, 0, at] = torch.linspace(0.0, -3.0, 40, device=device)
    x["tokens"][:, 1] = 0
    x["uniforms"][:, 1] = 0.5
    _, kept, following = verified(x, 1.0)
    assert (kept == 1).all() and len(set(following.tolist())) > 8

def test_logits_of_a_wider_product(device):
    for dtype in (F32, BF):
        x = verify_inputs(device, 3, 4, 1001, seed=8, dtype=dtype, drawn=True)
        for name in ("logits", "draft"):
            b, n, vocab = x[name].shape
            for extra in (1, 7):
                wide = torch.full((b, n, vocab + extra), 1e30, dtype=dtype, device=device)
                wide[..., :vocab] = x[name]
                verified(x | {name: wide[..., :vocab]}, 0.8)
        first = torch.full((3, 9, 1001), 1e30, dtype=dtype, device=device)
        first[:, 0] = x["logits"][:, 0]
        verified(dict(x, logits=first[:, :1], draft=None, tokens=x["tokens"][:, :1].contiguous(),
                      uniforms=x["uniforms"][:, :1].contiguous(), parents=x["parents"][:, :1].contiguous()), 0.8)


@pytest.mark.parametrize("mode", ["tree", "drawn"])
def test_emitted_tokens_are_distributed_as_the_targets(device, mode):
    """40000 sequences of one row and drafts of other distributions: the first token that is emitted has the target's
    probabilities, each within five standard deviations."""
    b, vocab, t = 40_000, 6, 0.8
    gen = torch.Generator(device=device).manual_seed(11)
    row, other = torch.randn(vocab, generator=gen, device=device), torch.randn(vocab, generator=gen, device=device)
    logits = torch.stack([row, torch.zeros_like(row), torch.zeros_like(row)]).expand(b, 3, vocab).contiguous()
    x = dict(logits=logits, uniforms=torch.rand(b, 3, generator=gen, device=device), draft=None,
             parents=torch.tensor([[-1, 0, 0]], dtype=torch.int32, device=device).expand(b, 3).contiguous())
    q = torch.softmax(other / t, -1)
    drawn = torch.multinomial(q.cpu(), b, replacement=True, generator=torch.Generator().manual_seed(12)).to(device)
    second = torch.full_like(drawn, int(row.argmin()))
    x["tokens"] = torch.stack([torch.zeros_like(drawn), drawn, second], 1).contiguous()
    if mode == "drawn":
        x["draft"] = torch.stack([other, row]).expand(b, 2, vocab).contiguous()
    ws = K.tree_verify_workspace(b, 3, vocab, device, drawn=mode == "drawn")
    if mode == "tree":  # a drafted token here is a choice that its draw does not bias
        x["tokens"][:, 1] = int(other.argmax())
    path, kept, following = K.tree_verify(x["logits"], x["tokens"], ws, temperature=t, uniforms=x["uniforms"],
                                          parents=None if mode == "drawn" else x["parents"], draft_logits=x["draft"])
    first = torch.where(kept > 1, torch.gather(x["tokens"], 1, path[:, 1:2].long().clamp(min=0))[:, 0], following)
    p = torch.softmax(row.double() / t, -1).cpu()
    seen = torch.bincount(first.cpu(), minlength=vocab).double() / b
    assert ((seen - p).abs() <= 5 * torch.sqrt(p * (1 - p) / b)).all(), (seen.tolist(), p.tolist())


def test_verification_in_given_tensors_and_one_workspace(device):
    ws = K.tree_verify_workspace(16, 64, 4000, device, drawn=True)
    for seed, (b, n, vocab, drawn) in enumerate([(16, 64, 500, True), (1, 1, 4000, False), (7, 9, 3999, False), (2, 5, 100, True)] * 2):
        out = dict(path=torch.full((b, n), 9, dtype=torch.int32, device=device),
                   kept=torch.full((b,), 9, dtype=torch.int32, device=device),
                   next_token=torch.full((b,), 9, dtype=torch.int64, device=device))
        got = verified(verify_inputs(device, b, n, vocab, seed=seed, drawn=drawn), 1.0, workspace=ws, **out)
        assert all(g is o for g, o in zip(got, out.values()))


def test_a_captured_verification_follows_its_inputs(device):
    for drawn in (False, True):
        x = verify_inputs(device, 3, 6, 30_000, seed=50, drawn=drawn)
        counts = torch.tensor([6, 6, 6], dtype=torch.int32, device=device)
        temps = torch.ones(3, device=device)
        ws = K.tree_verify_workspace(3, 6, 30_000, device, drawn=drawn)

        def call():
            return K.tree_verify(x["logits"], x["tokens"], ws, temperature=temps, uniforms=x["uniforms"], counts=counts,
                                 parents=None if drawn else x["parents"], draft_logits=x["draft"])

        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = call()
        for i in range(4):
            y = verify_inputs(device, 3, 6, 30_000, seed=51 + i, drawn=drawn)
            for name in ("logits", "tokens", "uniforms", "parents", "draft"):
                if x[name] is not None:
                    x[name].copy_(y[name])
            counts.copy_(torch.tensor([6, i, 3], dtype=torch.int32))
            temps.copy_(torch.tensor([0.5 * i, 1.0, 0.7]))
            g.replay()
            torch.cuda.synchronize()
            want = reference(y["logits"], y["tokens"], temps.tolist(), y["uniforms"], None if drawn else y["parents"], counts,
                             y["draft"])
            for a, b in zip(got, want):
                assert torch.equal(a.cpu(), b)


def test_verification_refusals(device):
    x = verify_inputs(device, 2, 4, 100, seed=9, drawn=True)
    ws = K.tree_verify_workspace(2, 4, 100, device, drawn=True)

    def call(**kw):
        a = dict(logits=x["logits"], tokens=x["tokens"], workspace=ws, temperature=1.0, uniforms=x["uniforms"])
        K.tree_verify(**(a | kw))

    ones = torch.ones(2, device=device)
    wrong = [
        (ValueError, dict(logits=x["logits"].cpu())), (TypeError, dict(logits=x["logits"].half())),
        (ValueError, dict(logits=x["logits"][0])), (ValueError, dict(logits=x["logits"].transpose(1, 2))),
        (ValueError, dict(logits=x["logits"][:, ::2])), (TypeError, dict(logits=None)),
        (TypeError, dict(tokens=x["tokens"].int())), (ValueError, dict(tokens=x["tokens"][:, :3])),
        (ValueError, dict(uniforms=None)), (TypeError, dict(uniforms=x["uniforms"].double())),
        (ValueError, dict(uniforms=x["uniforms"][:, :3].contiguous())), (ValueError, dict(temperature=-1.0)),
        (ValueError, dict(temperature=math.nan)), (ValueError, dict(temperature=math.inf)),
        (ValueError, dict(temperature=ones[:1])), (TypeError, dict(temperature=ones.double())),
        (ValueError, dict(temperature=ones.cpu())), (ValueError, dict(temperature=ones, uniforms=None)),
        (ValueError, dict(parents=x["parents"], draft_logits=x["draft"])), (ValueError, dict(draft_logits=x["logits"])),
        (TypeError, dict(draft_logits=x["draft"].to(BF))), (TypeError, dict(parents=x["parents"].long())),
        (ValueError, dict(parents=x["parents"][:1])), (ValueError, dict(counts=x["parents"])),
        (TypeError, dict(path=x["tokens"])), (ValueError, dict(kept=x["parents"])), (TypeError, dict(next_token=ones)),
        (TypeError, dict(workspace=ones)),
    ]
    for error, kw in wrong:
        with pytest.raises(error):
            call(**kw)
    with pytest.raises(RuntimeError):
        call(workspace=ws[:16])
    with pytest.raises(ValueError):
        call(logits=torch.zeros(1, 65, 10, device=device))
    with pytest.raises(ValueError):
        K.tree_verify_workspace(1, 65, 100, device)


# ------------------------------------------------------------------------------------------ keeping a path


def kept_reference(cache, path, kept, lengths):
    ref = cache.clone()
    s_cap, n = cache.shape[2], path.shape[1]
    for i, (line, m, at) in enumerate(zip(path.tolist(), kept.tolist(), lengths.tolist())):
        for j, p in enumerate(line[:max(0, min(m, n))]):
            if at >= 0 and j < p < n and at + p < s_cap:
                ref[:, i, at + j] = cache[:, i, at + p]
    return ref


@pytest.mark.parametrize("layers,n_seq,n,nk,s_cap", [(1, 1, 1, 8, 64), (3, 2, 5, 8, 40), (28, 1, 26, 8, 100), (2, 5, 64, 1, 200),
                                                     (4, 3, 64, 17, 130), (2, 2, 9, 3, 33), (5, 7, 31, 4, 90)])
def test_keeping_a_path(device, layers, n_seq, n, nk, s_cap):
    gen = torch.Generator(device=device).manual_seed(n)
    host = torch.Generator().manual_seed(n)
    for turn in range(3):
        k, v = (torch.randn(layers, n_seq, s_cap, nk, D, generator=gen, device=device).to(BF) for _ in range(2))
        path = torch.full((n_seq, n), -1, dtype=torch.int32)
        kept = torch.randint(1, n + 1, (n_seq,), generator=host).to(torch.int32)
        for i, m in enumerate(kept.tolist()):  # an ascending path from node 0
            path[i, 0] = 0
            path[i, 1:m] = 1 + torch.randperm(n - 1, generator=host)[:m - 1].sort().values.to(torch.int32)
        lengths = torch.randint(0, s_cap - n + 1, (n_seq,), generator=host).to(torch.int32)
        if turn == 1:  # some without a part, some at the cache's end
            lengths[0] = -1
            kept[-1] = 0
            lengths[n_seq // 2] = s_cap - max(1, n // 2)
        if turn == 2:  # entries that are no path
            path = torch.randint(-2, n + 3, (n_seq, n), generator=host).to(torch.int32)
            kept = torch.randint(-1, n + 4, (n_seq,), generator=host).to(torch.int32)
        want = [kept_reference(c, path, kept, lengths) for c in (k, v)]
        K.tree_keep(k, v, path.to(device), kept.to(device), lengths.to(device))
        assert torch.equal(k, want[0]) and torch.equal(v, want[1]), f"turn {turn}"


def test_keeping_a_path_in_strided_caches(device):
    gen = torch.Generator(device=device).manual_seed(1)
    whole_k = torch.randn(3, 6, 50, 8, D, generator=gen, device=device).to(BF)  # sequences first
    whole_v = torch.randn(6, 4, 50, 8, D, generator=gen, device=device).to(BF)
    k, v = whole_k.transpose(0, 1), whole_v[:, :3]
    path = torch.tensor([[0, 2, 5, 6, -1, -1, -1], [0, 1, 2, 3, 4, 5, 6], [0, 3, -1, -1, -1, -1, -1]], dtype=torch.int32, device=device)
    kept = torch.tensor([4, 7, 2], dtype=torch.int32, device=device)
    lengths = torch.tensor([10, 0, 43], dtype=torch.int32, device=device)
    want = [kept_reference(c, path, kept, lengths) for c in (k, v)]
    last = whole_v[:, 3].clone()
    K.tree_keep(k, v, path, kept, lengths)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1]) and torch.equal(whole_v[:, 3], last)


def test_keeping_refusals(device):
    k = torch.zeros(2, 3, 40, 8, D, dtype=BF, device=device)
    i = torch.zeros(3, dtype=torch.int32, device=device)
    path = torch.zeros(3, 5, dtype=torch.int32, device=device)
    K.tree_keep(k, k.clone(), path, i, i)
    wrong = [(k.cpu(), k, path, i, i, ValueError), (k, k[:1], path, i, i, ValueError), (k.float(), k, path, i, i, TypeError),
             (k, k, path[:2], i, i, ValueError), (k, k, path.long(), i, i, TypeError), (k, k, path, i[:2], i, ValueError),
             (k, k, path, i, i.long(), TypeError), (k, k, path, None, i, TypeError), (k[0], k[0], path, i, i, ValueError),
             (k, k, torch.zeros(3, 65, dtype=torch.int32, device=device), i, i, ValueError),
             (k[:1].expand(2, -1, -1, -1, -1), k, path, i, i, ValueError), (k.transpose(2, 3), k.transpose(2, 3), path, i, i, ValueError)]
    for a, b, p, m, at, error in wrong:
        with pytest.raises(error):
            K.tree_keep(a, b, p, m, at)
