"""The 8-bit KV cache on the GPU: write, single-token and chunk attention, weights, eviction and read back, against the
definition in 64 bits over what the cache holds (include/t2h.h, "8-bit KV cache")."""

from __future__ import annotations

import math

import pytest
import torch

from torch2vk_amd import kernels as K

pytestmark = pytest.mark.gpu

B, D, EPS = 64, 128, 1e-6
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF_BF16 = torch.finfo(BF).eps / 2  # a rounding to bf16, relative to the value
PARTS = ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")


# ------------------------------------------------------------------------------------------- the plain forms


def quantized(x):
    """Codes and scales of blocks [..., 64 * 128], in fp32 as the definition has it."""
    s = x.float().abs().amax((-2, -1)) * (1.0 / 127.0)
    s = torch.where(s < 1e-30, 0.0, s)
    inv = torch.where(s > 0, torch.reciprocal(s), 0.0)
    return torch.round(x.float() * inv[..., None, None]).to(torch.int8), s


def filled(n_seq, s_cap, nk, ends, device, seed, spread=1.0):
    """A cache that holds ends[i] tokens of sequence i; what lies behind them would show as NaN."""
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    c = K.kv_cache_q8(n_seq, s_cap, nk, D, device)
    nb = c.k.shape[1]
    for name, scale, shape in (("k", c.k_scale, (nb, nk, B, D)), ("v", c.v_scale, (nb, nk, D, B))):
        for i in range(n_seq):
            x = torch.randn(shape, generator=gen, device=device) * spread
            x = x * torch.exp2(torch.randint(-3, 4, (nb, nk, 1, 1), generator=gen, device=device).float())
            codes, s = quantized(x.to(BF))
            getattr(c, name)[i] = codes
            scale[i] = s
    c.k_tail.copy_(torch.randn(c.k_tail.shape, generator=gen, device=device) * spread)
    c.v_tail.copy_(torch.randn(c.v_tail.shape, generator=gen, device=device) * spread)
    for i, end in enumerate(ends):
        end = max(0, min(end, s_cap))
        c.k_scale[i, end // B:] = math.nan
        c.v_scale[i, end // B:] = math.nan
        c.k_tail[i, :, end % B:] = math.nan
        c.v_tail[i, :, :, end % B:] = math.nan
    return c


def rows_of(c, i, end):
    """fp64 K and V [nk, end, D] that sequence i's first ``end`` tokens have in the cache."""
    full = end // B
    k = (c.k[i, :full].to(F64) * c.k_scale[i, :full, :, None, None].to(F64)).transpose(0, 1).reshape(c.nk, -1, D)
    v = (c.v[i, :full].to(F64) * c.v_scale[i, :full, :, None, None].to(F64)).permute(1, 0, 3, 2).reshape(c.nk, -1, D)
    r = end - full * B
    return (torch.cat([k, c.k_tail[i, :, :r].to(F64)], 1),
            torch.cat([v, c.v_tail[i, :, :, :r].transpose(1, 2).to(F64)], 1))


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


def attention(q, k, v, last, scale=D ** -0.5):
    """q fp64 [t, nh, D], keys 0 .. last[t] of k, v [nk, s, D] -> out, sum of p |v|, p, and the largest sum of |q k|.
    The sum of p |v| has with it what fp16's least step leaves of a small p: p is held times 2^12 and the ratio of its value
    block's scale to the largest, so the step 2^-24 is rounded to within 2^-25, that is 2^-37 of the largest |v| for each
    key; check_out multiplies by 2^-10, hence 2^-27 here."""
    g = q.shape[1] // k.shape[0]
    k, v = k.repeat_interleave(g, 0), v.repeat_interleave(g, 0)
    score = torch.einsum("thd,hsd->hts", q, k) * scale
    mass = torch.einsum("thd,hsd->hts", q.abs(), k.abs()).amax() * scale
    seen = torch.arange(k.shape[1], device=q.device) <= last[:, None]
    p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
    least = 2.0 ** -27 * k.shape[1] * v.abs().amax()
    return torch.einsum("hts,hsd->thd", p, v), torch.einsum("hts,hsd->thd", p, v.abs()) + least, p, float(mass)


def within(got, ref, tol):
    """Whether got is as near ref as tol everywhere."""
    return bool(((got.to(F64) - ref).abs() <= tol).all())


def check_out(got, ref, mass_v, mass_qk, what):
    """bf16 output: half a step of its own; each p in fp16 (2^-11, and as much again where values are scaled into fp16's
    range), and p's relative error from the scores: fp32 products and sums of 128 terms, at most 2^-18 of sum |q k|."""
    tol = HALF_BF16 * 1.01 * ref.abs() + (2.0 ** -10 + 2.0 ** -17 * mass_qk) * mass_v + 1e-30
    bad = (got.to(F64) - ref).abs() > tol
    assert not bad.any() and torch.isfinite(got).all(), \
        f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.to(F64) - ref).abs() / tol).max()):.2f} x"


def check_weights(got, before, p, length, group, mass_qk, what):
    """fp32 weights of one sequence: p [nh, t, s] summed over a group's heads and the queries, each p to 2^-17 sum |q k| +
    2^-18 (exp, the sum it is divided by, its own sums)."""
    nk, s = got.shape[0], p.shape[-1]
    add = p.reshape(nk, group * p.shape[1], s).sum(1)
    ref = add.clone()
    ref[:, :length] += before[:, :length].to(F64)
    tol = (2.0 ** -17 * mass_qk + 2.0 ** -18) * add + 2.0 ** -23 * ref + 1e-30
    bad = (got[:, :s].to(F64) - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} off, {float(((got[:, :s].to(F64) - ref).abs() / tol).max()):.2f} x"
    assert torch.equal(got[:, s:], before[:, s:]), f"{what}: weights behind the last token changed"


def inputs(rows, nh, nk, device, seed, spread=1.5):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    qkv = torch.randn(rows, (nh + 2 * nk) * D, generator=gen, device=device) * spread
    wq = 1 + 0.3 * torch.randn(D, generator=gen, device=device)
    wk = 1 + 0.3 * torch.randn(D, generator=gen, device=device)
    return qkv.split([nh * D, nk * D, nk * D], 1), wq, wk


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def copy_of(c):
    return K.KVCacheQ8(*(getattr(c, n).clone() for n in PARTS))


def same(a, b):
    return all(torch.equal(getattr(a, n).view(torch.uint8), getattr(b, n).view(torch.uint8)) for n in PARTS)


# --------------------------------------------------------------------------------------------------- write


@pytest.mark.parametrize("n_seq,nk,n,lengths,counts", [
    (1, 2, 1, [0], None), (1, 2, 64, [0], None), (1, 1, 63, [1], None), (2, 3, 130, [0, 5], [130, 7]),
    (3, 2, 65, [63, 64, 127], [65, 0, 1]), (4, 1, 200, [-1, 250, 256, 300], None), (2, 8, 191, [60, 193], [4, 63]),
    (2, 2, 70, [10, 0], [-3, 1000])])
def test_write_holds_the_rounded_rows(device, n_seq, nk, n, lengths, counts):
    """Without norm and RoPE, of bf16 values, codes and scales are those of the definition, bit for bit; nothing else is
    written, whatever lies behind the tokens."""
    print("write", n_seq, nk, n, lengths, counts, flush=True)
    s_cap = 256
    c = filled(n_seq, s_cap, nk, lengths, device, 1)
    (q, k, v), _, _ = inputs(n_seq * n, nk, nk, device, 2)
    k, v = k.to(BF).float(), v.to(BF).float()
    v[:, 3] *= 1e-3
    want = copy_of(c)
    for i, length in enumerate(lengths):
        count = n if counts is None else max(0, min(n, counts[i]))
        if length < 0 or length >= s_cap:
            continue
        end = min(length + count, s_cap)
        kr, vr = k[i * n:(i + 1) * n].reshape(n, nk, D).to(BF), v[i * n:(i + 1) * n].reshape(n, nk, D).to(BF)
        for p in range(length, end):
            want.k_tail[i, :, p % B] = kr[p - length]
            want.v_tail[i, :, :, p % B] = vr[p - length]
            if p % B == B - 1:
                want.k[i, p // B], want.k_scale[i, p // B] = quantized(want.k_tail[i])
                want.v[i, p // B], want.v_scale[i, p // B] = quantized(want.v_tail[i])
        # what the tail holds of a finished block is not looked at
        for got, ref in ((c.k_tail[i], want.k_tail[i]), (c.v_tail[i].transpose(1, 2), want.v_tail[i].transpose(1, 2))):
            if end // B > length // B:
                ref[:, end % B:] = math.nan
    q_out = torch.empty(n_seq * n, nk, D, dtype=BF, device=device)
    K.qk_norm_rope_cache_q8(q, k, v, q_out, c, ints(lengths, device), theta=0.0,
                            counts=None if counts is None else ints(counts, device))
    for i, length in enumerate(lengths):
        end = max(0, length)
        count = n if counts is None else max(0, min(n, counts[i]))
        end = min(s_cap, end + (count if length >= 0 else 0))
        assert torch.equal(c.k[i], want.k[i]) and torch.equal(c.v[i], want.v[i])
        for name in ("k_scale", "v_scale"):
            assert torch.equal(getattr(c, name)[i].nan_to_num(-1), getattr(want, name)[i].nan_to_num(-1))
        assert torch.equal(c.k_tail[i, :, :end % B], want.k_tail[i, :, :end % B])
        assert torch.equal(c.v_tail[i, :, :, :end % B], want.v_tail[i, :, :, :end % B])
        rows = q_out[i * n:(i + 1) * n]
        live = 0 if length < 0 else count
        assert torch.equal(rows[:live], q[i * n:(i + 1) * n].reshape(n, nk, D).to(BF)[:live])
        assert not rows[live:].any()


@pytest.mark.parametrize("nh,nk,offset", [(16, 8, 0), (8, 8, 100000), (10, 2, 7)])
def test_write_norm_and_rope(device, nh, nk, offset):
    """q to half a bf16 step, cached keys to half a code and half a bf16 step, at far positions too (fp32 norm and product:
    2^-20 of the row's largest value)."""
    n, length = 150, 33
    c = filled(1, 256, nk, [length], device, 3)
    (q, k, v), wq, wk = inputs(n, nh, nk, device, 4)
    q_out = torch.empty(n, nh, D, dtype=BF, device=device)
    args = dict(theta=1e6, rope_offsets=ints([offset], device), q_norm_weight=wq, k_norm_weight=wk, eps=EPS)
    K.qk_norm_rope_cache_q8(q, k, v, q_out, c, ints([length], device), **args)
    pos = length + offset + torch.arange(n, device=device)
    ref = norm_rope(q.reshape(n, nh, D), wq, pos, 1e6)
    assert within(q_out, ref, HALF_BF16 * 1.01 * ref.abs() + 2.0 ** -20 * ref.abs().amax(-1, keepdim=True))
    kr, vr = rows_of(c, 0, length + n)
    ref = norm_rope(k.reshape(n, nk, D), wk, pos, 1e6).transpose(0, 1)
    full = (length + n) // B * B
    step = torch.zeros(nk, length + n, 1, dtype=F64, device=device)
    step[:, :full, 0] = c.k_scale[0, :full // B].to(F64).T.repeat_interleave(B, 1)
    tol = HALF_BF16 * 1.01 * ref.abs() + 2.0 ** -20 * ref.abs().amax(-1, keepdim=True) + 0.5001 * step[:, length:]
    assert within(kr[:, length:], ref, tol)
    step[:, :full, 0] = c.v_scale[0, :full // B].to(F64).T.repeat_interleave(B, 1)
    ref = v.reshape(n, nk, D).transpose(0, 1).to(F64)
    assert within(vr[:, length:], ref, HALF_BF16 * 1.01 * ref.abs() + 0.5001 * step[:, length:])


def test_the_cache_does_not_depend_on_the_chunks(device):
    """The same tokens in one chunk, in ragged chunks and one by one in decode steps: the same bits."""
    nh, nk, n = 4, 2, 200
    (q, k, v), wq, wk = inputs(n, nh, nk, device, 5)
    args = dict(theta=1e4, q_norm_weight=wq, k_norm_weight=wk)
    one, many, steps = (K.kv_cache_q8(1, 256, nk, D, device) for _ in range(3))
    out = torch.empty(n, nh, D, dtype=BF, device=device)
    K.qk_norm_rope_cache_q8(q, k, v, out, one, ints([0], device), **args)
    at = 0
    for m in (1, 30, 33, 1, 100, 35):
        K.qk_norm_rope_cache_q8(q[at:at + m], k[at:at + m], v[at:at + m], out[at:at + m], many, ints([at], device), **args)
        at += m
    ws = K.attn_decode_q8_workspace(1, nh, nk, D, 256, device)
    o = torch.empty(1, nh, D, dtype=BF, device=device)
    for t in range(n):
        K.attn_decode_q8(q[t:t + 1], k[t:t + 1], v[t:t + 1], steps, o, ints([t], device), ws, **args)
    for c in (many, steps):
        assert torch.equal(c.k, one.k) and torch.equal(c.v, one.v)
        assert torch.equal(c.k_scale, one.k_scale) and torch.equal(c.v_scale, one.v_scale)
        r = n % B
        assert torch.equal(c.k_tail[:, :, :r], one.k_tail[:, :, :r]) and torch.equal(c.v_tail[..., :r], one.v_tail[..., :r])


def test_blocks_of_zeros_tiny_and_broken_values(device):
    """A block of zeros or of values too small for a scale reads as zeros; one with a NaN or an infinity as NaN, and the
    other head's and the other blocks' values are what they are."""
    nk, n = 2, 256
    (q, k, v), _, _ = inputs(n, nk, nk, device, 6)
    k, v = k.clone(), v.clone()
    k[:64, :D] = 0
    v[64:128, :D] = 1e-33
    k[130, 5] = math.nan
    v[200, D + 5] = math.inf
    c = K.kv_cache_q8(1, 256, nk, D, device)
    out = torch.empty(n, nk, D, dtype=BF, device=device)
    K.qk_norm_rope_cache_q8(q, k, v, out, c, ints([0], device), theta=0.0)
    kd, vd = K.kv_cache_q8_dequantize(c, ints([n], device))
    assert not kd[0, :64, 0].any() and not vd[0, 64:128, 0].any()
    assert kd[0, 128:192, 0].isnan().all() and vd[0, 192:, 1].isnan().all()
    assert torch.isfinite(kd[0, :, 1]).all() and torch.isfinite(vd[0, :, 0]).all()
    assert torch.isfinite(kd[0, 192:, 0]).all() and torch.isfinite(vd[0, :192, 1]).all()


# ---------------------------------------------------------------------------------------------------- decode


@pytest.mark.parametrize("nh,nk,lengths,s_cap,weights", [
    (2, 2, [0], 64, True), (4, 2, [1], 64, False), (16, 8, [63], 128, True), (32, 8, [64], 128, True),
    (8, 1, [62, 63, 64, 65, 127, 128, 190], 192, True), (16, 1, [-1, 5, 192, 500, 191], 192, True),
    (6, 2, [300, 17], 448, True), (5, 1, [1000], 1024, False), (16, 8, [200], 2048, False), (32, 8, [4100], 8192, True),
    (12, 4, [0, 9000, 3, 500, 20000], 20032, True), (8, 8, [700, 64, 1, 129], 768, False),
    (8, 2, list(range(0, 4000, 57)), 4032, True), (20, 4, [70000], 70016, True),
    (4, 2, list(range(3000, -100, -20)), 3008, True)])
def test_decode(device, nh, nk, lengths, s_cap, weights):
    print("decode", nh, nk, lengths[:8], s_cap, weights, flush=True)
    n_seq, group = len(lengths), nh // nk
    c = filled(n_seq, s_cap, nk, lengths, device, 7, 1.0)
    before = copy_of(c)
    (q, k, v), wq, wk = inputs(n_seq, nh, nk, device, 8)
    offsets = [3 * i for i in range(n_seq)]
    w = torch.rand(n_seq, nk, s_cap, device=device) if weights else None
    w_out = torch.full_like(w, 0.25) if weights else None
    ws = K.attn_decode_q8_workspace(n_seq, nh, nk, D, s_cap, device, weights=weights)
    out = torch.full((n_seq, nh, D), math.nan, dtype=BF, device=device)
    K.attn_decode_q8(q, k, v, c, out, ints(lengths, device), ws, theta=1e6, rope_offsets=ints(offsets, device),
                     q_norm_weight=wq, k_norm_weight=wk, eps=EPS, weights=w, weights_out=w_out)
    pos = ints([max(0, x) + o for x, o in zip(lengths, offsets)], device)
    qr, kr = norm_rope(q.reshape(n_seq, nh, D), wq, pos, 1e6), norm_rope(k.reshape(n_seq, nk, D), wk, pos, 1e6)
    for i, length in enumerate(lengths):
        end = 0 if length < 0 else min(length + 1, s_cap)
        if end == 0:
            assert not out[i].any()
            if weights:
                assert torch.equal(w_out[i], torch.full_like(w_out[i], 0.25))
            continue
        kc, vc = rows_of(c, i, end)
        old_k, old_v = rows_of(before, i, min(length, s_cap))
        whole = end // B * B
        keep = min(length, whole if whole <= length else whole - B)  # a block that this token finished is rounded now
        assert torch.equal(kc[:, :keep], old_k[:, :keep]) and torch.equal(vc[:, :keep], old_v[:, :keep])
        if length < s_cap:
            step = c.k_scale[i, length // B].to(F64)[:, None] if end % B == 0 else 0.0
            tol = HALF_BF16 * 1.01 * kr[i].abs() + 2.0 ** -20 * kr[i].abs().amax() + 0.5001 * step
            assert within(kc[:, length], kr[i], tol)
        ref, mass_v, p, mass_qk = attention(qr[i:i + 1], kc, vc, torch.tensor([end - 1], device=device))
        check_out(out[i:i + 1], ref, mass_v, mass_qk, f"sequence {i} of length {length}")
        if weights:
            prior = torch.full_like(w[i], 0.25)
            prior[:, :min(length, s_cap)] = w[i, :, :min(length, s_cap)]
            check_weights(w_out[i], prior, p, min(length, s_cap), group, mass_qk, f"weights of sequence {i}")
        # whole blocks that were there, and those of other sequences, stay as they were
        last = length // B
        assert torch.equal(c.k[i, :last], before.k[i, :last]) and torch.equal(c.v[i, last + 1:], before.v[i, last + 1:])


@pytest.mark.parametrize("scale_k,scale_v", [(30.0, 1.0), (1e-3, 1e-6), (1.0, 1e5)])
def test_decode_of_large_and_small_values(device, scale_k, scale_v):
    """Scores that leave one key only, and values far from 1: nothing overflows or is lost on the way."""
    nh, nk, length = 8, 2, 450
    c = filled(1, 512, nk, [length], device, 9)
    c.k_scale.mul_(scale_k)
    c.k_tail.mul_(scale_k)
    c.v_scale.mul_(scale_v)
    c.v_tail.mul_(scale_v)
    (q, k, v), _, _ = inputs(1, nh, nk, device, 10)
    k, v = k * scale_k, v * scale_v
    out = torch.empty(1, nh, D, dtype=BF, device=device)
    K.attn_decode_q8(q, k, v, c, out, ints([length], device), K.attn_decode_q8_workspace(1, nh, nk, D, 512, device), theta=0.0)
    kc, vc = rows_of(c, 0, length + 1)
    ref, mass_v, _, mass_qk = attention(q.reshape(1, nh, D).to(F64), kc, vc, torch.tensor([length], device=device))
    check_out(out, ref, mass_v, mass_qk, "scaled")


def test_a_broken_block_reaches_its_own_head_only(device):
    nh, nk, length = 4, 2, 500
    c = filled(1, 512, nk, [length], device, 11)
    c.v_scale[0, 2, 1] = math.nan
    (q, k, v), _, _ = inputs(1, nh, nk, device, 12)
    out = torch.empty(1, nh, D, dtype=BF, device=device)
    K.attn_decode_q8(q, k, v, c, out, ints([length], device), K.attn_decode_q8_workspace(1, nh, nk, D, 512, device), theta=0.0)
    assert out[0, 2:].isnan().all()
    kc, vc = rows_of(c, 0, length + 1)
    ref, mass_v, _, mass_qk = attention(q.reshape(1, nh, D).to(F64)[:, :2], kc[:1], vc[:1], torch.tensor([length], device=device))
    check_out(out[:, :2], ref, mass_v, mass_qk, "the other head")


def test_decode_replayed_from_a_graph(device):
    """Steps captured once with their lengths on the device, replayed over a block's end with eager work between, equal
    the eager steps bit for bit; two graphs share a workspace."""
    nh, nk, n_seq, s_cap = 8, 2, 3, 256
    start = [60, 10, 127]
    args = dict(theta=1e6)
    (q, k, v), wq, wk = inputs(n_seq, nh, nk, device, 13)
    args |= dict(q_norm_weight=wq, k_norm_weight=wk)
    ws = K.attn_decode_q8_workspace(n_seq, nh, nk, D, s_cap, device, weights=True)
    runs = []
    for graphed in (False, True):
        c = filled(n_seq, s_cap, nk, start, device, 14)
        w = torch.zeros(n_seq, nk, s_cap, device=device)
        lengths = ints(start, device)
        out = torch.empty(2, n_seq, nh, D, dtype=BF, device=device)

        def step(j):
            K.attn_decode_q8(q, k, v, c, out[j], lengths, ws, weights=w, **args)
            lengths.add_(1)

        outs = []
        if graphed:
            saved, saved_w = copy_of(c), w.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step(0)
            torch.cuda.current_stream().wait_stream(side)
            graphs = []
            for j in range(2):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    step(j)
                graphs.append(g)
            for name in PARTS:
                getattr(c, name).copy_(getattr(saved, name))
            w.copy_(saved_w)
            lengths.copy_(ints(start, device))
        for j in range(8):
            if graphed:
                graphs[j % 2].replay()
                torch.cuda.synchronize()
                (torch.ones(1000, device=device) * 2).sum().item()
            else:
                step(j % 2)
            outs.append(out[j % 2].clone())
        runs.append((torch.stack(outs), w, c))
    assert torch.equal(runs[0][0].view(torch.int16), runs[1][0].view(torch.int16))
    assert torch.equal(runs[0][1], runs[1][1])
    assert torch.equal(runs[0][2].k, runs[1][2].k) and torch.equal(runs[0][2].v, runs[1][2].v)


def test_decode_of_several_shapes_in_one_workspace(device):
    """Calls of different batches, heads and capacities in turn, in one workspace: each as with its own."""
    shapes = [(1, 8, 8, 3000), (40, 8, 1, 2000), (3, 32, 8, 900), (1, 16, 1, 3000), (40, 8, 1, 2000)]
    ws = max((K.attn_decode_q8_workspace(n, nh, nk, D, 3008, device, weights=True) for n, nh, nk, _ in shapes), key=len)
    for rnd, (n, nh, nk, length) in enumerate(shapes):
        lengths = [max(1, length - 61 * i) for i in range(n)]
        c = filled(n, 3008, nk, lengths, device, 30 + rnd)
        (q, k, v), wq, wk = inputs(n, nh, nk, device, 40 + rnd)
        outs = []
        for own in (False, True):
            out = torch.empty(n, nh, D, dtype=BF, device=device)
            w = torch.zeros(n, nk, 3008, device=device)
            K.attn_decode_q8(q, k, v, copy_of(c), out, ints(lengths, device),
                             K.attn_decode_q8_workspace(n, nh, nk, D, 3008, device, weights=True) if own else ws, theta=1e6,
                             q_norm_weight=wq, k_norm_weight=wk, weights=w)
            outs.append((out, w))
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


# ---------------------------------------------------------------------------------------------------- chunks


@pytest.mark.parametrize("nh,nk,n,lengths,counts,s_cap,weights", [
    (2, 2, 1, [0], None, 64, True), (4, 2, 1, [64], None, 128, True), (16, 8, 5, [61, 300], [5, 3], 384, True),
    (8, 1, 64, [0], None, 64, True), (16, 1, 33, [-1, 0, 100], [33, 0, 40], 192, True), (6, 2, 130, [0], None, 192, False),
    (5, 1, 77, [200], None, 320, True), (32, 8, 300, [0, 55], [300, 256], 384, False), (8, 8, 200, [1000, 3], None, 1216, True),
    (16, 8, 512, [700], None, 1280, True), (12, 4, 3, [5000], None, 5056, True), (32, 8, 129, [190], None, 256, False),
    (8, 4, 40, [230, 250], None, 256, True), (4, 4, 700, [0], None, 704, False), (16, 2, 2, [20000], None, 20032, True),
    (3, 3, 1, [8191], None, 8192, False), (8, 2, 1300, [900], None, 2240, True), (32, 8, 5, [3990, 61, 0], [5, 4, 2], 4032, True),
    (8, 8, 32, [100, 33, -1, 160], [28, 32, 5, 32], 192, True), (4, 1, 8, [30000, 120], None, 30016, True),
    (12, 2, 400, [5, -1, 130], [400, 7, 333], 576, True), (16, 1, 256, [0, 100, 60], [256, 1, 0], 384, True),
    (14, 2, 700, [300], [650], 960, True)])
def test_chunk(device, nh, nk, n, lengths, counts, s_cap, weights):
    """A chunk written and attended to, against the definition over what the cache then holds; tokens past the capacity are
    dropped."""
    print("chunk", nh, nk, n, lengths, counts, s_cap, weights, flush=True)
    n_seq, group = len(lengths), nh // nk
    c = filled(n_seq, s_cap, nk, lengths, device, 15)
    (q, k, v), wq, wk = inputs(n_seq * n, nh, nk, device, 16)
    lens = ints(lengths, device)
    cnt = None if counts is None else ints(counts, device)
    q_out = torch.empty(n_seq, n, nh, D, dtype=BF, device=device)
    K.qk_norm_rope_cache_q8(q, k, v, q_out, c, lens, counts=cnt, theta=1e6, q_norm_weight=wq, k_norm_weight=wk)
    w = torch.rand(n_seq, nk, s_cap, device=device) if weights else None
    w_out = torch.full_like(w, 0.25) if weights else None
    out = torch.full_like(q_out, math.nan)
    K.flash_attn_prefill_q8(q_out, c, lens, out, counts=cnt, weights=w, weights_out=w_out)
    for i, length in enumerate(lengths):
        count = n if counts is None else max(0, min(n, counts[i]))
        count = 0 if length < 0 else count
        assert not out[i, count:].any()
        end = min(max(0, length) + count, s_cap)
        if count == 0:
            continue
        kc, vc = rows_of(c, i, end)
        last = (length + torch.arange(count, device=device)).clamp(max=end - 1)
        ref, mass_v, p, mass_qk = attention(q_out[i, :count].to(F64), kc, vc, last)
        check_out(out[i, :count], ref, mass_v, mass_qk, f"sequence {i}")
        if weights:
            prior = torch.full_like(w[i], 0.25)
            prior[:, :length] = w[i, :, :length]
            check_weights(w_out[i], prior, p, length, group, mass_qk, f"weights of sequence {i}")


def test_chunk_scale_and_early_rows_beside_a_broken_block(device):
    """A scale of the caller's; and queries before a block with a NaN do not see it."""
    nh, nk, n = 4, 2, 200
    c = filled(1, 256, nk, [n], device, 17)
    c.v_scale[0, 2, 0] = math.nan
    q = torch.randn(1, n, nh, D, device=device).to(BF)
    out = K.flash_attn_prefill_q8(q, c, ints([0], device), scale=0.05)
    assert out[0, 128:192, :2].isnan().all() and torch.isfinite(out[0, :128]).all() and torch.isfinite(out[0, :, 2:]).all()
    kc, vc = rows_of(c, 0, n)
    last = torch.arange(n, device=device)
    ref, mass_v, _, mass_qk = attention(q[0, :, 2:].to(F64), kc[1:], vc[1:], last, 0.05)
    check_out(out[0, :, 2:], ref, mass_v, mass_qk, "scale")


def test_chunk_values_of_very_different_blocks(device):
    """Blocks whose value scales lie 2^20 apart: rows that see only the small ones keep their precision."""
    nh, nk, n = 4, 1, 256
    c = filled(1, 256, nk, [256], device, 18)
    c.v_scale[0, :3] *= 2.0 ** -20
    q = torch.randn(1, n, nh, D, device=device).to(BF)
    out = K.flash_attn_prefill_q8(q, c, ints([0], device))
    kc, vc = rows_of(c, 0, n)
    ref, mass_v, _, mass_qk = attention(q[0].to(F64), kc, vc, torch.arange(n, device=device))
    check_out(out[0], ref, mass_v, mass_qk, "small blocks")


# -------------------------------------------------------------------------------------------------- eviction


def evicted(c, i, w, length, keep, sink, recent):
    """Kept tokens [nk, stay] of sequence i by the definition."""
    full = length // B * B
    stay = min(full, keep * B)
    kept = []
    for h in range(c.nk):
        x = [math.inf if t < sink or t >= full - recent else (1e300 if math.isnan(v) else v)
             for t, v in enumerate(w[h, :full].tolist())]
        safe = [t < sink or t >= full - recent for t in range(full)]
        order = sorted(range(full), key=lambda t: (not safe[t], -x[t], t))
        kept.append(sorted(order[:stay]))
    return torch.tensor(kept, dtype=torch.long, device=c.k.device).reshape(c.nk, stay), full, stay


@pytest.mark.parametrize("nk,lengths,s_cap,keep,sink,recent,kind", [
    (2, [130], 192, 1, 0, 0, "random"), (1, [64, 63, 0, -1], 128, 1, 0, 0, "random"), (2, [500, 300, 700], 704, 4, 4, 64, "ties"),
    (8, [4100], 4160, 32, 4, 128, "random"), (2, [640], 640, 3, 100, 92, "random"), (1, [5000], 5056, 1, 0, 64, "zeros"),
    (2, [1000], 1024, 7, 1, 30, "special"), (2, [20000, 9000], 20032, 150, 4, 1000, "ties"),
    (1, [70000, 60000], 70016, 300, 4, 500, "special")])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict(device, nk, lengths, s_cap, keep, sink, recent, kind, in_place):
    print("evict", nk, lengths, keep, sink, recent, kind, in_place, flush=True)
    n_seq = len(lengths)
    c = filled(n_seq, s_cap, nk, lengths, device, 19)
    w = torch.rand(n_seq, nk, s_cap, device=device)
    if kind == "ties":
        w = torch.round(w * 8)
    elif kind == "zeros":
        w.zero_()
    elif kind == "special":
        w[:, :, 50::97] = math.nan
        w[:, :, 51::97] = math.inf
        w[:, :, 52::97] = -1.0
        w[:, :, 53::7] = -0.0
        w[:, :, 54::7] = 0.0
    before, w0 = copy_of(c), w.clone()
    lens = ints(lengths, device)
    if in_place:
        dest, w_out = c, w
        kept, new = K.kv_cache_q8_evict(c, lens, w, keep, sink=sink, recent=recent)
    else:
        dest = K.kv_cache_q8(n_seq, (keep + 1) * B, nk, D, device)
        w_out = torch.full((n_seq, nk, dest.s_cap), -7.0, device=device)
        kept, new = K.kv_cache_q8_evict(c, lens, w, keep, sink=sink, recent=recent, out=dest, weights_out=w_out)
        assert same(before, c) and torch.equal(w.view(torch.int32), w0.view(torch.int32))
    assert torch.equal(lens, ints(lengths, device))
    for i, length in enumerate(lengths):
        if length < 0:
            assert int(new[i]) == length and (kept[i] == -1).all()
            continue
        ref, full, stay = evicted(before, i, w0[i], length, keep, sink, recent)
        assert int(new[i]) == stay + length - full
        assert torch.equal(kept[i, :, :stay].long(), ref) and (kept[i, :, stay:] == -1).all()
        got_k, got_v = rows_of(dest, i, int(new[i]))
        old_k, old_v = rows_of(before, i, length)
        tail = torch.arange(full, length, device=device).expand(nk, -1)
        at = torch.cat([ref, tail], 1)
        for got, old, scale in ((got_k, old_k, dest.k_scale), (got_v, old_v, dest.v_scale)):
            want = torch.gather(old, 1, at[..., None].expand(-1, -1, D))
            assert torch.equal(got[:, stay:], want[:, stay:])
            # half a code of the new scale, which is the largest value's 127th
            step = scale[i, :stay // B].to(F64).T
            top = want[:, :stay].abs().reshape(nk, -1, B * D).amax(-1) / 127
            assert within(step, top, 2.0 ** -22 * top)
            half = 0.5001 * step.repeat_interleave(B, 1)[..., None]
            if stay == full:
                half = 0 * half
            assert within(got[:, :stay], want[:, :stay], half)
        want = torch.gather(w0[i], 1, at)
        assert torch.equal(w_out[i, :, :at.shape[1]].view(torch.int32), want.view(torch.int32))
        if not in_place:
            assert (w_out[i, :, at.shape[1]:] == -7).all()


@pytest.mark.parametrize("in_cache,in_weights", [(True, False), (False, True), (True, True)])
def test_evict_half_in_place(device, in_cache, in_weights):
    """The cache's blocks, the weights or both in their own memory: what an eviction into other memory gives, in a captured
    graph too; elements behind what stays are left."""
    lengths, nk, s_cap, keep = [700, 130, 0, -1, 256, 63], 3, 704, 3
    c = filled(len(lengths), s_cap, nk, lengths, device, 33)
    w, lens = torch.rand(len(lengths), nk, s_cap, device=device), ints(lengths, device)
    ref, ref_w = K.kv_cache_q8(len(lengths), s_cap, nk, D, device), torch.full_like(w, -7.0)
    ref_kept, ref_new = K.kv_cache_q8_evict(c, lens, w, keep, sink=2, recent=9, out=ref, weights_out=ref_w)

    def check(dest, w_out, kept, new, old_w):
        assert torch.equal(kept, ref_kept) and torch.equal(new, ref_new)
        for i in range(len(lengths)):
            end = max(0, int(new[i]))
            for name in ("k", "v", "k_scale", "v_scale"):
                assert torch.equal(getattr(dest, name)[i, :end // B], getattr(ref, name)[i, :end // B]), name
            assert torch.equal(dest.k_tail[i].nan_to_num(), ref.k_tail[i].nan_to_num())
            assert torch.equal(dest.v_tail[i].nan_to_num(), ref.v_tail[i].nan_to_num())
            assert torch.equal(w_out[i, :, :end], ref_w[i, :, :end]) and torch.equal(w_out[i, :, end:], old_w[i, :, end:])

    for graph in (False, True):
        mine, w_mine = copy_of(c), w.clone()
        dest = mine if in_cache else K.kv_cache_q8(len(lengths), s_cap, nk, D, device)
        w_out = w_mine if in_weights else torch.full_like(w, -7.0)
        old_w = w_out.clone()
        run = lambda: K.kv_cache_q8_evict(mine, lens, w_mine, keep, sink=2, recent=9, out=dest, weights_out=w_out)  # noqa: E731
        if not graph:
            check(dest, w_out, *run(), old_w)
            continue
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kept, new = run()
        for _ in range(3):
            for name in PARTS:
                getattr(mine, name).copy_(getattr(c, name))
            w_mine.copy_(w)
            g.replay()
            check(dest, w_out, kept, new, old_w)


# ------------------------------------------------------------------------------------------------- read back


@pytest.mark.parametrize("nk,lengths", [(8, [0]), (3, [64, 63, 200, -1, 1000]), (1, [192])])
def test_dequantize(device, nk, lengths):
    c = filled(len(lengths), 192, nk, lengths, device, 20)
    k, v = K.kv_cache_q8_dequantize(c, ints(lengths, device))
    for i, length in enumerate(lengths):
        end = max(0, min(length, 192))
        for got, ref in zip((k, v), rows_of(c, i, end)):
            assert not got[i, end:].any()
            assert torch.equal(got[i, :end], ref.transpose(0, 1).to(BF))


# --------------------------------------------------------------------------------------------- used together


def test_prompt_decode_evict_decode(device):
    """A ragged prompt, steps past a block's end, an eviction in place and more steps, on a stream of its own: every output
    against the definition over the cache, and positions that go on where they were."""
    nh, nk, n_seq, s_cap, n = 8, 2, 2, 512, 330
    counts = [330, 217]
    lengths = ints([0, 0], device)
    offsets = torch.zeros_like(lengths)
    c = K.kv_cache_q8(n_seq, s_cap, nk, D, device)
    w = torch.zeros(n_seq, nk, s_cap, device=device)
    ws = K.attn_decode_q8_workspace(n_seq, nh, nk, D, s_cap, device, weights=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        (q, k, v), wq, wk = inputs(n_seq * n, nh, nk, device, 21)
        norms = dict(theta=1e6, q_norm_weight=wq, k_norm_weight=wk)
        q_out = torch.empty(n_seq, n, nh, D, dtype=BF, device=device)
        K.qk_norm_rope_cache_q8(q, k, v, q_out, c, lengths, counts=ints(counts, device), **norms)
        K.flash_attn_prefill_q8(q_out, c, lengths, counts=ints(counts, device), weights=w)
        lengths += ints(counts, device)
        positions = list(counts)

        def step(seed):
            (q, k, v), _, _ = inputs(n_seq, nh, nk, device, seed)
            out = torch.empty(n_seq, nh, D, dtype=BF, device=device)
            K.attn_decode_q8(q, k, v, c, out, lengths, ws, rope_offsets=offsets, weights=w, **norms)
            qr = norm_rope(q.reshape(n_seq, nh, D), wq, ints(positions, device), 1e6)
            for i in range(n_seq):
                end = int(lengths[i]) + 1
                kc, vc = rows_of(c, i, end)
                ref, mass_v, _, mass_qk = attention(qr[i:i + 1], kc, vc, torch.tensor([end - 1], device=device))
                check_out(out[i:i + 1], ref, mass_v, mass_qk, f"step {seed} sequence {i}")
                positions[i] += 1
            lengths.add_(1)

        for j in range(60):
            step(100 + j)
        total = [x + 60.0 for x in counts]
        for i in range(n_seq):  # every query's weights sum to 1 for each of the group's heads
            got = w[i, :, :int(lengths[i])].sum(-1).to(F64)
            assert within(got, total[i] * (nh // nk), 1e-4 * total[i])
        kept, new = K.kv_cache_q8_evict(c, lengths, w, 3, sink=4, recent=32)
        offsets += lengths - new
        lengths.copy_(new)
        for j in range(70):
            step(200 + j)
    torch.cuda.current_stream().wait_stream(stream)


def test_the_far_end_of_a_large_cache(device):
    """The last of 40 sequences in a cache of 5 GB of codes each for keys and values, past 32 bits: every operator gives it
    what it gives it in a cache of less capacity."""
    nh, nk, n_seq, s_cap, length = 16, 8, 40, 131072, 6000
    lens = ints([-1] * (n_seq - 1) + [length], device)
    low, big = filled(n_seq, 8192, nk, lens.tolist(), device, 31), K.kv_cache_q8(n_seq, s_cap, nk, D, device)
    for name in PARTS:
        part = getattr(low, name)[-1]
        getattr(big, name)[-1, :part.shape[0]] = part
    w_low, w = torch.rand(n_seq, nk, 8192, device=device), torch.zeros(n_seq, nk, s_cap, device=device)
    w[..., :8192] = w_low

    def same(what):
        for name in PARTS:
            part = getattr(low, name)[-1]
            assert torch.equal(getattr(big, name)[-1, :part.shape[0]].nan_to_num(), part.nan_to_num()), f"{what}: {name}"
        assert torch.equal(w[..., :8192], w_low), f"{what}: weights"

    n = 300
    rows, wq, wk = inputs(n_seq * n, nh, nk, device, 32)
    norms = dict(theta=1e6, q_norm_weight=wq, k_norm_weight=wk)
    outs = [torch.empty(n_seq, n, nh, D, dtype=BF, device=device) for _ in range(2)]
    for c, out in zip((low, big), outs):
        K.qk_norm_rope_cache_q8(*rows, out, c, lens, **norms)
    assert torch.equal(*outs) and not outs[1][:-1].any()
    same("chunk write")
    got = K.flash_attn_prefill_q8(outs[1], big, lens, weights=w)
    K.flash_attn_prefill_q8(outs[0], low, lens, weights=w_low)
    kc, vc = rows_of(low, n_seq - 1, length + n)
    ref, mass_v, _, mass_qk = attention(outs[0][-1].to(F64), kc, vc, length + torch.arange(n, device=device))
    check_out(got[-1], ref, mass_v, mass_qk, "chunk")
    assert not got[:-1].any()
    end = length + n
    assert within(w[-1, :, :end], w_low[-1, :, :end], 1e-4 * (1 + w_low[-1, :, :end]))  # other splits, other sums
    w[..., :8192] = w_low
    lens[-1] += n
    few = [K.flash_attn_prefill_q8(outs[0][:, :2].contiguous(), c, lens - 2) for c in (low, big)]
    assert torch.equal(*few), "a few tokens"
    steps = [torch.empty(n_seq, nh, D, dtype=BF, device=device) for _ in range(2)]
    spaces = [K.attn_decode_q8_workspace(n_seq, nh, nk, D, c.s_cap, device, weights=True) for c in (low, big)]
    for j in range(70):  # over a block's end
        q, k, v = (t[j * n_seq:(j + 1) * n_seq] for t in rows)
        for c, step, ws, weights in zip((low, big), steps, spaces, (w_low, w)):
            K.attn_decode_q8(q, k, v, c, step, lens, ws, weights=weights, **norms)
        assert torch.equal(*steps), f"step {j}"
        lens[-1] += 1
    same("steps")
    (kept_low, new_low), (kept, new) = (K.kv_cache_q8_evict(c, lens, x, 30) for c, x in ((low, w_low), (big, w)))
    assert torch.equal(kept, kept_low) and torch.equal(new, new_low) and bool((new[:-1] == -1).all())
    same("eviction")
    for a, b in zip(K.kv_cache_q8_dequantize(big, new), K.kv_cache_q8_dequantize(low, new)):
        assert torch.equal(a[-1, :8192], b[-1]) and not a[-1, 8192:].any() and not a[0].any()


# -------------------------------------------------------------------------------------------------- refusals


def test_refusals(device):
    nh, nk, n_seq, s_cap = 4, 2, 2, 128
    c = K.kv_cache_q8(n_seq, s_cap, nk, D, device)
    (q, k, v), wq, wk = inputs(n_seq, nh, nk, device, 22)
    lens = ints([0, 0], device)
    ws = K.attn_decode_q8_workspace(n_seq, nh, nk, D, s_cap, device)
    out = torch.empty(n_seq, nh, D, dtype=BF, device=device)
    w = torch.zeros(n_seq, nk, s_cap, device=device)

    def decode(q=q, k=k, v=v, cache=c, out=out, lens=lens, ws=ws, **more):
        K.attn_decode_q8(q, k, v, cache, out, lens, ws, **{"theta": 0.0, **more})

    for bad in (dict(q=q.to(BF)), dict(lens=lens.long()), dict(out=out.float()), dict(ws=ws.view(torch.int8))):
        with pytest.raises(TypeError):
            decode(**bad)
    for bad in (dict(q=q[:1]), dict(q=q[:, :D * 3]), dict(k=k[:, :D]), dict(lens=lens[:1]), dict(out=out[:1]), dict(lens=lens.cpu()),
                dict(q_norm_weight=wq), dict(q_norm_weight=wq[:64], k_norm_weight=wk), dict(weights=w[:, :1]),
                dict(weights_out=w), dict(weights=w, weights_out=w[:1]), dict(rope_offsets=lens[:1]),
                dict(q=q[:1].expand(2, -1))):
        with pytest.raises(ValueError):
            decode(**bad)
    from torch2vk_amd._lib import T2HError
    with pytest.raises(T2HError, match="workspace"):
        decode(ws=ws[:16])
    with pytest.raises(TypeError):
        decode(cache=(c.k, c.v))
    with pytest.raises(ValueError):
        K.kv_cache_q8(1, 64, 1, 64, device)
    with pytest.raises(ValueError):
        K.KVCacheQ8(c.k, c.v[:1], c.k_scale, c.v_scale, c.k_tail, c.v_tail)
    with pytest.raises(ValueError):
        K.KVCacheQ8(c.k, c.v.transpose(3, 4), c.k_scale, c.v_scale, c.k_tail, c.v_tail)
    qq = torch.zeros(n_seq, 3, nh, D, dtype=BF, device=device)
    for bad in (qq[:1], qq[:, :, :3], qq.transpose(1, 2), qq[0]):
        with pytest.raises(ValueError):
            K.flash_attn_prefill_q8(bad, c, lens)
    with pytest.raises(ValueError):
        K.flash_attn_prefill_q8(qq, c, lens, qq[:, :2])
    assert K.flash_attn_prefill_q8(qq[:, :0].contiguous(), c, lens).numel() == 0
    for bad in (dict(keep_blocks=0), dict(keep_blocks=1, sink=65), dict(keep_blocks=1, recent=-1), dict(keep_blocks=1, sink=40, recent=40)):
        with pytest.raises(ValueError):
            K.kv_cache_q8_evict(c, lens, w, **bad)
    small = K.kv_cache_q8(n_seq, 64, nk, D, device)
    with pytest.raises(ValueError):
        K.kv_cache_q8_evict(c, lens, w, 1, out=small, weights_out=w[..., :64].contiguous())
    with pytest.raises(ValueError):
        K.kv_cache_q8_dequantize(c, lens, torch.empty(n_seq, 64, nk, D, dtype=BF, device=device))
    assert not c.k.any() and not c.k_tail.any() and not w.any()
