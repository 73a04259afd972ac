"""The 8-bit KV cache where values are not finite, lie far apart or belong to no row: against the definition in 64 bits over
what the cache holds (the plain forms and tolerances of test_gpu_kv_q8.py)."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_kv_q8 import (B, BF, D, F64, HALF_BF16, attention, check_out, check_weights, copy_of, filled, inputs, ints,
                                  rows_of)
from torch2vk_amd import kernels as K

pytestmark = pytest.mark.gpu


def chunk_rows(shape, device, seed):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    return torch.randn(shape, generator=gen, device=device).to(BF)


def check_rows(got, q, k, v, last, what):
    """Rows got [t, nh, D] of queries q fp64 that see keys 0 .. last[t]: test_gpu_kv_q8.check_out's tolerance with the largest
    |v| that the row itself sees in the place of the sequence's (2^-37 of it for each key, times the 2^10 of check_out)."""
    ref, _, p, mass_qk = attention(q, k, v, last)
    size = v.abs().repeat_interleave(q.shape[1] // k.shape[0], 0)
    top = size.amax(-1).cummax(-1).values[:, last].T[..., None]
    mass_v = torch.einsum("hts,hsd->thd", p, size) + 2.0 ** -27 * k.shape[1] * top
    tol = HALF_BF16 * 1.01 * ref.abs() + (2.0 ** -10 + 2.0 ** -17 * mass_qk) * mass_v + 1e-38
    bad = ~((got.to(F64) - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}"


# ------------------------------------------------------------------- the unfinished block's values, not finite


@pytest.mark.parametrize("nh,nk,n,end,s_cap", [
    (4, 2, 5, 100, 128), (8, 2, 8, 1030, 1088), (4, 2, 5, 4098, 4160),  # few rows: a tile, two, several units
    (4, 2, 200, 230, 256), (6, 2, 100, 300, 8192), (3, 1, 130, 130, 192)])  # tiles, and their keys split
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_broken_value_of_the_tail_reaches_the_rows_that_see_it(device, nh, nk, n, end, s_cap, value):
    """A NaN or an infinity in the unfinished block's values: its dimension of the rows that see its token is not finite, and
    every other output is what it is without it, rows of earlier blocks and earlier tokens among them."""
    print("tail", nh, nk, n, end, s_cap, value, flush=True)
    length = end - n
    c = filled(1, s_cap, nk, [end], device, 50)
    bad = {(end - 1, 0, 5), (end - 1, nk - 1, 70), (max(length, end // B * B), 0, 127)}
    for token, head, dim in bad:
        c.v_tail[0, head, dim, token % B] = value
    q = chunk_rows((1, n, nh, D), device, 51)
    out = K.flash_attn_prefill_q8(q, c, ints([length], device))[0]
    k, v = rows_of(c, 0, end)
    last = length + torch.arange(n, device=device)
    broken = torch.zeros(n, nh, D, dtype=torch.bool, device=device)
    for token, head, dim in bad:
        broken[token - length:, head * (nh // nk):(head + 1) * (nh // nk), dim] = True
    assert not torch.isfinite(out[broken]).any()
    assert torch.isfinite(out[~broken]).all(), f"{int((~torch.isfinite(out) & ~broken).sum())} outputs that do not see it"
    ref, mass_v, _, mass_qk = attention(q[0].to(F64), k, v.nan_to_num(0.0, 0.0, 0.0), last)
    check_out(torch.where(broken, 0.0, out.float()), torch.where(broken, 0.0, ref), mass_v, mass_qk, "the others")


# -------------------------------------------------------------------------------------- rows past a count


@pytest.mark.parametrize("nh,nk,n,length,count,s_cap", [(4, 2, 5, 100, 3, 192), (8, 2, 8, 200, 1, 256), (4, 2, 6, 5000, 4, 5056),
                                                        (4, 2, 90, 200, 40, 320)])
@pytest.mark.parametrize("part", ["k_scale", "v_scale"])
def test_rows_past_a_count_are_zeros_beside_a_broken_block(device, nh, nk, n, length, count, s_cap, part):
    c = filled(1, s_cap, nk, [length + count], device, 52)
    getattr(c, part)[0, 0, 0] = math.nan
    q = chunk_rows((1, n, nh, D), device, 53)
    out = K.flash_attn_prefill_q8(q, c, ints([length], device), torch.full_like(q, 7.0), counts=ints([count], device))[0]
    group = nh // nk
    assert out[:count, :group].isnan().all() and torch.isfinite(out[:count, group:]).all()
    assert torch.equal(out[count:], torch.zeros_like(out[count:]))


# --------------------------------------------------------------------------- value scales that lie far apart


@pytest.mark.parametrize("low,high", [(-90, 50), (-99, 100), (-60, 0)])
@pytest.mark.parametrize("order", ["low first", "high first", "between"])
@pytest.mark.parametrize("n,s_cap", [(250, 256), (250, 4096)])
def test_chunk_of_value_scales_far_apart(device, low, high, order, n, s_cap):
    """Whole blocks whose value scales are 2^60 to 2^199 apart: every output is finite, rows that see the small ones only are
    as good as among small ones (a tile of 128 tokens holds rows of two blocks), and the weights, which no value has part
    in, are what they are."""
    nh, nk = 2, 2
    c = filled(1, s_cap, nk, [n], device, 54)
    at = {"low first": [low, high, high], "high first": [high, low, low], "between": [low, high, low]}[order]
    for b, e in enumerate(at):
        c.v_scale[0, b] = 2.0 ** e
    c.v_tail.mul_(2.0 ** low)
    q = chunk_rows((1, n, nh, D), device, 55)
    w = torch.rand(1, nk, s_cap, device=device)
    w_out = torch.full_like(w, 0.25)
    out = K.flash_attn_prefill_q8(q, c, ints([0], device), weights=w, weights_out=w_out)[0]
    assert torch.isfinite(out).all() and torch.isfinite(w_out).all()
    k, v = rows_of(c, 0, n)
    last = torch.arange(n, device=device)
    check_rows(out, q[0].to(F64), k, v, last, f"{order} 2^{low} 2^{high}")
    _, _, p, mass_qk = attention(q[0].to(F64), k, v, last)
    check_weights(w_out[0], torch.full_like(w[0], 0.25), p, 0, nh // nk, mass_qk, "weights")


@pytest.mark.parametrize("e_block,e_tail", [(0, 115), (-85, 60), (-85, 115), (100, -90)])
@pytest.mark.parametrize("n", [0, 5, 150])  # a single token's kernel, few rows, tiles
@pytest.mark.parametrize("length", [10, 420])
def test_tail_values_far_from_the_blocks(device, e_block, e_tail, n, length):
    """The unfinished block's values 2^115 to 2^200 over or under those of the blocks, and no blocks."""
    nh, nk, s_cap = 4, 2, 640
    c = filled(1, s_cap, nk, [length + n], device, 56)
    c.v_scale.mul_(2.0 ** e_block)
    c.v_tail.mul_(2.0 ** e_tail)
    if n == 0:
        (q, k_new, v_new), _, _ = inputs(1, nh, nk, device, 57, 1.0)
        out = torch.empty(1, nh, D, dtype=BF, device=device)
        K.attn_decode_q8(q, k_new, v_new * 2.0 ** e_tail, c, out, ints([length], device),
                         K.attn_decode_q8_workspace(1, nh, nk, D, s_cap, device), theta=0.0)
        q, last = q.reshape(1, nh, D), torch.tensor([length], device=device)
        k, v = rows_of(c, 0, length + 1)
    else:
        q = chunk_rows((n, nh, D), device, 58)
        out = K.flash_attn_prefill_q8(q[None], c, ints([length], device))[0]
        last = length + torch.arange(n, device=device)
        k, v = rows_of(c, 0, length + n)
    check_rows(out, q.to(F64), k, v, last, f"blocks 2^{e_block}, tail 2^{e_tail}")


# ------------------------------------------------------------------------------------------ a chunk's weights


@pytest.mark.parametrize("nh,nk,n,length,s_cap", [(4, 2, 200, 0, 256), (4, 2, 200, 70, 320), (4, 2, 5, 300, 320),
                                                  (4, 2, 100, 150, 8192)])
def test_weights_beside_a_block_of_broken_values(device, nh, nk, n, length, s_cap):
    """The weights are the softmax of the scores: a NaN among the values, which makes the outputs that see it NaN, has no part
    in them."""
    end = length + n
    c = filled(1, s_cap, nk, [end], device, 59)
    q = chunk_rows((1, n, nh, D), device, 60)
    w = torch.rand(1, nk, s_cap, device=device)
    want = torch.full_like(w, 0.25)
    K.flash_attn_prefill_q8(q, c, ints([length], device), weights=w, weights_out=want)
    assert torch.isfinite(want).all()
    c.v_scale[0, 1, 0] = math.nan
    got = torch.full_like(w, 0.25)
    out = K.flash_attn_prefill_q8(q, c, ints([length], device), weights=w, weights_out=got)[0]
    sees = length + torch.arange(n, device=device) >= B
    assert out[sees][:, :nh // nk].isnan().all() and torch.isfinite(out[:, nh // nk:]).all()
    assert torch.isfinite(out[~sees]).all()
    k, v = rows_of(c, 0, end)
    assert torch.isfinite(got).all()
    _, _, p, mass_qk = attention(q[0].to(F64), k, torch.zeros_like(v), length + torch.arange(n, device=device))
    prior = torch.full_like(w[0], 0.25)
    prior[:, :length] = w[0, :, :length]
    check_weights(got[0], prior, p, length, nh // nk, mass_qk, "weights")


def test_a_first_query_of_nan_adds_to_what_it_sees(device):
    """A first query of NaN makes the weights of the first token NaN, which it sees, and no others, whatever rows the last
    step of the chunk's queries does not fill."""
    n, s_cap = 200, 256
    c = filled(1, s_cap, 1, [n], device, 61)
    q = chunk_rows((1, n, 1, D), device, 62)
    k, v = rows_of(c, 0, n)
    _, _, p, mass_qk = attention(q[0].to(F64), k, v, torch.arange(n, device=device))
    q[0, 0] = math.nan
    w = torch.full((1, 1, s_cap), 0.25, device=device)
    out = K.flash_attn_prefill_q8(q, c, ints([0], device), weights=w)[0]
    assert out[0].isnan().all() and torch.isfinite(out[1:]).all()
    assert w[0, 0, 0].isnan()
    assert torch.isfinite(w[0, 0, 1:]).all()
    w[0, 0, 0] = p[0, :, 0].sum()
    check_weights(w[0], torch.full_like(w[0], 0.25), p, 0, 1, mass_qk, "weights")


@pytest.mark.parametrize("counts", [None, [0, 0, 0]])
def test_weights_of_a_chunk_without_tokens(device, counts):
    """No new token: weights_out holds the cached tokens' weights as they were."""
    lengths, nk, s_cap = [100, -1, 500], 2, 256
    c = filled(3, s_cap, nk, lengths, device, 63)
    w = torch.rand(3, nk, s_cap, device=device)
    w_out = torch.full_like(w, -7.0)
    q = torch.zeros(3, 0 if counts is None else 4, 4, D, dtype=BF, device=device)
    out = K.flash_attn_prefill_q8(q, c, ints(lengths, device), weights=w, weights_out=w_out,
                                  counts=None if counts is None else ints(counts, device))
    assert not out.any()
    for i, length in enumerate(lengths):
        end = max(0, min(length, s_cap))
        assert torch.equal(w_out[i, :, :end], w[i, :, :end]) and bool((w_out[i, :, end:] == -7).all())


# ----------------------------------------------------------------------- queries of very different elements


@pytest.mark.parametrize("small", [-10, -16, -20])
@pytest.mark.parametrize("n", [0, 3])  # a single token's kernel, few rows
def test_small_elements_of_a_query_keep_their_precision(device, n, small):
    """A query's elements 2^10 to 2^20 under its largest, whose keys are zeros, so that the small ones alone make the scores:
    these are within 2^-18 of sum |q k| all the same."""
    nh, nk, length, s_cap = 4, 2, 400, 448
    c = filled(1, s_cap, nk, [length + n], device, 64, 1.0)
    c.k[..., :D // 2] = 0
    c.k_tail[..., :D // 2] = 0
    c.k_scale.mul_(2.0 ** -small)
    c.k_tail.mul_(2.0 ** -small)
    (q, k_new, v_new), _, _ = inputs(max(1, n), nh, nk, device, 65, 1.0)
    q = q.reshape(-1, nh, D).clone()
    q[..., D // 2:] *= 2.0 ** small
    if n == 0:
        k_new = k_new.reshape(1, nk, D).clone()
        k_new[..., :D // 2] = 0
        out = torch.empty(1, nh, D, dtype=BF, device=device)
        K.attn_decode_q8(q.reshape(1, -1), (k_new * 2.0 ** -small).reshape(1, -1), v_new, c, out, ints([length], device),
                         K.attn_decode_q8_workspace(1, nh, nk, D, s_cap, device), theta=0.0)
        last = torch.tensor([length], device=device)
    else:
        q = q.to(BF)
        out = K.flash_attn_prefill_q8(q[None], c, ints([length], device))[0]
        last = length + torch.arange(n, device=device)
    w = torch.zeros(1, nk, s_cap, device=device)
    k, v = rows_of(c, 0, int(last[-1]) + 1)
    ref, mass_v, p, mass_qk = attention(q.to(F64), k, v, last)
    check_out(out, ref, mass_v, mass_qk, f"2^{small}")
    if n:  # the weights say what the scores are, to check_weights' tolerance
        K.flash_attn_prefill_q8(q[None], c, ints([length], device), weights=w)
        assert torch.isfinite(w).all()
        check_weights(w[0], torch.zeros_like(w[0]), p, length, nh // nk, mass_qk, f"2^{small}")


# ------------------------------------------------------------------------------------------------- eviction


def test_eviction_leaves_a_sequence_that_takes_no_part(device):
    """A negative length: nothing of that sequence in the other cache or the other weights is written."""
    lengths, nk, keep = [300, -1, 130], 2, 2
    c = filled(3, 320, nk, lengths, device, 66)
    w = torch.rand(3, nk, 320, device=device)
    dest = filled(3, 320, nk, [0, 200, 0], device, 67)
    w_out = torch.full_like(w, -7.0)
    before = copy_of(dest)
    _, new = K.kv_cache_q8_evict(c, ints(lengths, device), w, keep, out=dest, weights_out=w_out)
    assert new.tolist() == [128 + 44, -1, 130]
    for name in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail"):
        assert torch.equal(getattr(dest, name)[1].nan_to_num(-3.0), getattr(before, name)[1].nan_to_num(-3.0)), name
    assert bool((w_out[1] == -7).all())


def ranked(w, full, stay, sink, recent):
    """Kept tokens of one head by the definition: the first and the last, then NaN, then by weight, -0 as 0, ties to the
    earliest."""
    def key(t):
        x = w[t]
        if t < sink or t >= full - recent:
            return (0, 0.0, t)
        return (1, 0.0, t) if math.isnan(x) else (2, -x + 0.0, t)

    return sorted(sorted(range(full), key=key)[:stay])


@pytest.mark.parametrize("inside", ["nan", "inf", "positive", "zeros", "negative", "-inf"])
@pytest.mark.parametrize("in_place", [False, True])
def test_eviction_whose_cut_lies_among_special_weights(device, inside, in_place):
    """Weights of six kinds, of which 128 tokens stay: the last that stays is one of the kind named.  NaN ranks above
    infinity, and 0 and -0 are one weight."""
    nk, length, keep, s_cap = 2, 520, 2, 576
    full, sink, recent = 512, 3, 5
    gen = torch.Generator().manual_seed(68)
    kinds = ["nan", "inf", "positive", "zeros", "negative", "-inf"]
    at = kinds.index(inside)
    w = torch.zeros(1, nk, s_cap)
    for h in range(nk):
        # 120 of the sink, recent and all kinds above in sum; the rest of the kind named, and 60 of each below
        counts = [0] * 6
        for i in range(at):
            counts[i] = 110 // at
        for i in range(at + 1, 6):
            counts[i] = 30
        counts[at] = full - sink - recent - sum(counts)
        values = []
        for kind, count in zip(kinds, counts):
            x = torch.rand(count, generator=gen) + 0.5
            values.append({"nan": torch.full((count,), math.nan), "inf": torch.full((count,), math.inf), "positive": x,
                           "zeros": torch.where(x > 1, 0.0, -0.0), "negative": -x, "-inf": torch.full((count,), -math.inf)}[kind])
        x = torch.cat(values)
        w[0, h, sink:full - recent] = x[torch.randperm(len(x), generator=gen)]
    w = w.to(device)
    host = w.cpu()
    c = filled(1, s_cap, nk, [length], device, 69)
    more = {} if in_place else dict(out=K.kv_cache_q8(1, s_cap, nk, D, device), weights_out=torch.zeros_like(w))
    kept, new = K.kv_cache_q8_evict(c, ints([length], device), w, keep, sink=sink, recent=recent, **more)
    assert int(new) == keep * B + length - full
    for h in range(nk):
        row = host[0, h].tolist()
        want = ranked(row, full, keep * B, sink, recent)
        assert kept[0, h].tolist() == want
        rest = set(range(sink, full - recent)) - set(want)
        same = {"nan": math.isnan, "inf": lambda x: x == math.inf, "positive": lambda x: 0 < x < math.inf,
                "zeros": lambda x: x == 0, "negative": lambda x: -math.inf < x < 0, "-inf": lambda x: x == -math.inf}[inside]
        assert any(same(row[t]) for t in want) and any(same(row[t]) for t in rest)  # the cut is inside


# -------------------------------------------------------------------------------------- many wide tiles


def test_many_ragged_tiles_of_a_group_that_does_not_divide_them(device):
    """Over 512 tiles of 256 rows in thread blocks of 8 waves, in rounds of 256 of them of which every other runs from the
    shortest up, a last one that is no multiple of 8 among them; with counts, lengths and a sequence that takes no part."""
    nh, nk, n = 21, 7, 930  # 2790 rows: 11 tiles a head and sequence, 11 * 7 * 11 = 3 * 256 + 79 of them
    lengths = [0, 70, 3, 128, -1, 64, 200, 1, 0, 31, 65]
    counts = [930, 900, 1, 930, 930, 0, 700, 929, 930, 500, 257]
    s_cap = 1024
    c = filled(11, s_cap, nk, [max(0, x) + y if x >= 0 else 0 for x, y in zip(lengths, counts)], device, 70)
    q = chunk_rows((11, n, nh, D), device, 71)
    w = torch.rand(11, nk, s_cap, device=device)
    w_out = torch.full_like(w, 0.25)
    out = K.flash_attn_prefill_q8(q, c, ints(lengths, device), torch.full_like(q, math.nan), counts=ints(counts, device),
                                  weights=w, weights_out=w_out)
    for i, length in enumerate(lengths):
        count = counts[i] if length >= 0 else 0
        assert torch.equal(out[i, count:], torch.zeros_like(out[i, count:]))
        if count == 0:
            continue
        end = min(length + count, s_cap)
        k, v = rows_of(c, i, end)
        last = (length + torch.arange(count, device=device)).clamp(max=end - 1)
        ref, mass_v, p, mass_qk = attention(q[i, :count].to(F64), k, v, last)
        check_out(out[i, :count], ref, mass_v, mass_qk, f"sequence {i}")
        assert torch.isfinite(w_out[i]).all()
        prior = torch.full_like(w[i], 0.25)
        prior[:, :length] = w[i, :, :length]
        check_weights(w_out[i], prior, p, length, nh // nk, mass_qk, f"weights of sequence {i}")


def test_a_broken_tail_in_wide_tiles(device):
    """As in tiles of 4 waves: a NaN and an infinity among the unfinished block's values in thread blocks of 8."""
    nh, nk, n, n_seq, s_cap = 8, 8, 1000, 16, 1088  # 4 tiles of 256 rows a head and sequence, 512 of them
    lengths = [7 * i for i in range(n_seq)]
    ends = [n + x for x in lengths]
    c = filled(n_seq, s_cap, nk, [min(x, s_cap) for x in ends], device, 72)
    q = chunk_rows((n_seq, n, nh, D), device, 73)
    bad = {(3, 2, 11, math.nan), (5, 7, 127, math.inf), (5, 7, 0, -math.inf)}  # sequence, head, dim of its last token
    for i, h, d, value in bad:
        assert ends[i] < s_cap and ends[i] % B
        c.v_tail[i, h, d, (ends[i] - 1) % B] = value
    out = K.flash_attn_prefill_q8(q, c, ints(lengths, device))
    broken = torch.zeros_like(out, dtype=torch.bool)
    for i, h, d, _ in bad:
        broken[i, -1, h, d] = True
    assert torch.equal(~torch.isfinite(out), broken)
    for i in (0, 3, 5, 15):
        end = min(ends[i], s_cap)
        k, v = rows_of(c, i, end)
        last = (lengths[i] + torch.arange(n, device=device)).clamp(max=end - 1)
        ref, mass_v, _, mass_qk = attention(q[i].to(F64), k, v.nan_to_num(0.0, 0.0, 0.0), last)
        keep = ~broken[i]
        check_out(torch.where(keep, out[i].float(), 0.0), torch.where(keep, ref, 0.0), mass_v, mass_qk, f"sequence {i}")


# --------------------------------------------------------------------------------------- behind a full cache


@pytest.mark.parametrize("n", [3, 90])  # few rows, tiles
def test_chunk_behind_a_full_cache(device, n):
    """Lengths at and past the capacity: every query sees all cached tokens, whose weights grow; nothing is written."""
    nh, nk, s_cap, lengths = 4, 2, 256, [256, 300, 255]
    c = filled(3, s_cap, nk, lengths, device, 74)
    (q, k_new, v_new), _, _ = inputs(3 * n, nh, nk, device, 75)
    before = copy_of(c)
    q_out = torch.empty(3, n, nh, D, dtype=BF, device=device)
    K.qk_norm_rope_cache_q8(q, k_new, v_new, q_out, c, ints(lengths, device), theta=1e6)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(c, name)[:2], getattr(before, name)[:2])
    w = torch.rand(3, nk, s_cap, device=device)
    w_out = torch.full_like(w, 0.25)
    out = K.flash_attn_prefill_q8(q_out, c, ints(lengths, device), weights=w, weights_out=w_out)
    for i, length in enumerate(lengths):
        k, v = rows_of(c, i, s_cap)
        last = (length + torch.arange(n, device=device)).clamp(max=s_cap - 1)
        ref, mass_v, p, mass_qk = attention(q_out[i].to(F64), k, v, last)
        check_out(out[i], ref, mass_v, mass_qk, f"sequence {i}")
        assert torch.isfinite(w_out[i]).all()
        prior = w[i].clone()
        prior[:, min(length, s_cap):] = 0.25
        check_weights(w_out[i], prior, p, min(length, s_cap), nh // nk, mass_qk, f"weights of sequence {i}")
