"""What the operators over the 8-bit KV cache are measured on: listed and drawn cases, their plain form, the calls that a
user makes of the framework (``own``), and their definition in 64 bits.

The cache holds 8-bit integers under one fp32 scale for each block of 64 tokens, sequence and KV head, and the tokens of a
sequence's last, unfinished block in bf16 (its tail); a block is rounded once, when its last token arrives.  Values are
transposed within a block.  With x the block's bf16 values: s = max|x| / 127, code = round(x / s), ties to even.

Operators: ``write`` (a chunk's q/k norm and RoPE, and its K and V into the cache), ``decode`` (one token of each sequence:
norm, RoPE, write, attention, and the attention weight that each cached token got), ``chunk`` (causal attention of a chunk's
queries over the cache, with or without those weights), ``evict`` (each head keeps the tokens of most accumulated weight), and
with ``write`` and ``evict`` the cache's values in bf16, as the framework's other paths hold them."""

import math

import torch

own = False

BLOCK, D, EPS, THETA = 64, 128, 1e-6, 1e6
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # one user's short chat: 28 or 36 of these calls in every token, where latency is all that counts
        dict(name="decode_1x200", op="decode", n_seq=1, nh=16, nk=8, lo=200, hi=200, s_cap=2048, weights=False),
        # one user, a few pages of context
        dict(name="decode_1x4096", op="decode", n_seq=1, nh=32, nk=8, lo=4100, hi=4100, s_cap=8192, weights=False),
        # a served batch of ragged lengths that also keeps the weights an eviction goes by
        dict(name="decode_16_ragged_weights", op="decode", n_seq=16, nh=32, nk=8, lo=100, hi=8000, s_cap=8192, weights=True),
        # a full batch of long contexts: as many bytes as a step over a large cache reads
        dict(name="decode_32x16000", op="decode", n_seq=32, nh=32, nk=8, lo=15000, hi=16300, s_cap=16384, weights=False),
        # one prompt chunk of the default size for chunked prompts
        dict(name="write_1x512", op="write", n_seq=1, nh=16, nk=8, n=512, n_lo=512, lo=512, hi=512, s_cap=1088),
        # eight ragged prompts, padded to one length
        dict(name="write_8x2048", op="write", n_seq=8, nh=32, nk=8, n=2048, n_lo=900, lo=0, hi=0, s_cap=2112),
        # a few drafted tokens checked against a context
        dict(name="chunk_2x5_at_4000", op="chunk", n_seq=2, nh=32, nk=8, n=5, n_lo=3, lo=3900, hi=4090, s_cap=4160, weights=False),
        # one prompt of an odd length
        dict(name="chunk_1x1901", op="chunk", n_seq=1, nh=32, nk=8, n=1901, n_lo=1901, lo=0, hi=0, s_cap=1984, weights=False),
        # late chunks of long prompts, with the weights for a later eviction
        dict(name="chunk_4x512_at_7000_weights", op="chunk", n_seq=4, nh=16, nk=8, n=512, n_lo=400, lo=6500, hi=7400, s_cap=8192,
             weights=True),
        # a batch of whole prompts
        dict(name="chunk_8x2048", op="chunk", n_seq=8, nh=32, nk=8, n=2048, n_lo=2048, lo=0, hi=0, s_cap=2112, weights=False),
        # one user's cache halved
        dict(name="evict_1x4096", op="evict", n_seq=1, nh=32, nk=8, lo=4130, hi=4130, s_cap=4160, keep=32, sink=4, recent=128),
        # a served batch brought back to a budget
        dict(name="evict_8x16000", op="evict", n_seq=8, nh=32, nk=8, lo=9000, hi=16300, s_cap=16384, keep=64, sink=4, recent=256),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cap(n):
    return (n + 1 + BLOCK - 1) // BLOCK * BLOCK


def draw(rng):
    op = rng.choice(["decode", "decode", "write", "chunk", "chunk", "evict"])
    nh, nk = rng.choice([(16, 8), (32, 8), (8, 8), (32, 4), (24, 8), (20, 4)])
    if op == "decode":
        n_seq = _spread(rng, 1, 32)
        hi = _spread(rng, 64, min(60000, 400000 // n_seq))
        lo = rng.choice([hi, max(1, hi // 2), 1])
        return dict(op=op, n_seq=n_seq, nh=nh, nk=nk, lo=lo, hi=hi, s_cap=_cap(hi + rng.choice([0, hi])),
                    weights=rng.random() < 0.4)
    if op == "write":
        n_seq = _spread(rng, 1, 8)
        n = _spread(rng, 1, 2048)
        lo = BLOCK * rng.choice([0, 0, 1, 5, 16])
        return dict(op=op, n_seq=n_seq, nh=nh, nk=nk, n=n, n_lo=rng.randint(max(1, n // 2), n), lo=lo, hi=lo,
                    s_cap=_cap(lo + n))
    if op == "chunk":
        n_seq = _spread(rng, 1, 4)
        n = _spread(rng, 1, 2048)
        hi = rng.choice([0, _spread(rng, 1, 16000 // n_seq if n < 500 else 4000 // n_seq)])
        return dict(op=op, n_seq=n_seq, nh=nh, nk=nk, n=n, n_lo=rng.randint(max(1, n // 2), n), lo=rng.choice([hi, hi // 2]),
                    hi=hi, s_cap=_cap(hi + n), weights=rng.random() < 0.4)
    n_seq = _spread(rng, 1, 8)
    hi = _spread(rng, 300, 16000)
    blocks = hi // BLOCK
    keep = rng.randint(max(1, blocks // 4), max(1, 3 * blocks // 4))
    sink = rng.choice([0, 1, 4])
    return dict(op=op, n_seq=n_seq, nh=nh, nk=nk, lo=rng.randint(hi // 2, hi), hi=hi, s_cap=_cap(hi), keep=keep, sink=sink,
                recent=rng.randint(0, keep * BLOCK // 2 - sink))


# ------------------------------------------------------------------------------------------------------ inputs


def _rows(shape, gen, spread=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * spread


def _quantized(x):
    """bf16 values, one block in the last two axes -> (int8 codes, fp32 scales)."""
    x = x.to(F32)
    s = x.abs().amax((-2, -1)) * (1.0 / 127.0)
    s = torch.where(s < 1e-30, 0.0, s)
    inv = torch.where(s > 0, torch.reciprocal(s), 0.0)
    return torch.round(x * inv[..., None, None]).to(torch.int8), s


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    b, nh, nk, s_cap = c["n_seq"], c["nh"], c["nk"], c["s_cap"]
    nb = s_cap // BLOCK
    host = torch.Generator().manual_seed(seed)
    lengths = torch.randint(c["lo"], c["hi"] + 1, (b,), generator=host)
    if b > 1:
        lengths[0] = c["hi"]
    if c["op"] == "decode":  # the tail is returned whole: no sequence finishes a block in these calls
        lengths = torch.where(lengths % BLOCK == BLOCK - 1, lengths - 1, lengths)
    s = dict(case=c, lengths=lengths.to(torch.int32).cuda(), theta=THETA)
    # keys have a few strong channels, as rotary keys do; values none
    channel = 1.0 + 3.0 * (torch.rand(D, generator=gen, device="cuda") < 0.06)
    cache = {"k": torch.empty(b, nb, nk, BLOCK, D, dtype=torch.int8, device="cuda"),
             "v": torch.empty(b, nb, nk, D, BLOCK, dtype=torch.int8, device="cuda"),
             "k_scale": torch.empty(b, nb, nk, device="cuda"), "v_scale": torch.empty(b, nb, nk, device="cuda")}
    for i in range(b):
        cache["k"][i], cache["k_scale"][i] = _quantized((_rows((nb, nk, BLOCK, D), gen) * channel).to(BF))
        cache["v"][i], cache["v_scale"][i] = _quantized(_rows((nb, nk, D, BLOCK), gen).to(BF))
    cache["k_tail"] = (_rows((b, nk, BLOCK, D), gen) * channel).to(BF)
    cache["v_tail"] = _rows((b, nk, D, BLOCK), gen).to(BF)
    s["cache"] = cache
    norms = dict(q_norm_weight=1.0 + 0.3 * _rows((D,), gen), k_norm_weight=channel * (1.0 + 0.1 * _rows((D,), gen)))
    if c["op"] in ("decode", "write"):
        rows = b if c["op"] == "decode" else b * c["n"]
        s["qkv"] = _rows((rows, (nh + 2 * nk) * D), gen, 2.0)  # one product's columns: q, k, v
        s |= norms
        s["rope_offsets"] = torch.randint(0, 20000, (b,), generator=host).to(torch.int32).cuda()
    if c["op"] in ("write", "chunk"):
        counts = torch.randint(c["n_lo"], c["n"] + 1, (b,), generator=host)
        if b > 1:
            counts[0] = c["n"]
        s["counts"] = counts.to(torch.int32).cuda()
    if c["op"] == "chunk":
        s["q"] = _rows((b, c["n"], nh, D), gen, 1.2).to(BF)
    if c.get("weights"):
        s["weights"] = torch.rand(b, nk, s_cap, generator=gen, device="cuda").pow(4) * 8
        s["weights_out"] = torch.zeros_like(s["weights"])
    if c["op"] == "evict":
        s["weights"] = torch.rand(b, nk, s_cap, generator=gen, device="cuda").pow(4) * 8
        # the same weight twice and more, as tokens that no query looked at have
        s["weights"] = torch.where(s["weights"] < 1e-3, 0.0, s["weights"])
        cap = (c["keep"] + 1) * BLOCK
        nbo = cap // BLOCK
        s["out"] = {"k": torch.zeros(b, nbo, nk, BLOCK, D, dtype=torch.int8, device="cuda"),
                    "v": torch.zeros(b, nbo, nk, D, BLOCK, dtype=torch.int8, device="cuda"),
                    "k_scale": torch.zeros(b, nbo, nk, device="cuda"), "v_scale": torch.zeros(b, nbo, nk, device="cuda"),
                    "k_tail": torch.zeros(b, nk, BLOCK, D, dtype=BF, device="cuda"),
                    "v_tail": torch.zeros(b, nk, D, BLOCK, dtype=BF, device="cuda")}
        s["weights_out"] = torch.zeros(b, nk, cap, device="cuda")
    if own:
        from torch2vk_amd import kernels

        s["cache"] = kernels.KVCacheQ8(**s["cache"])
        if "out" in s:
            s["out"] = kernels.KVCacheQ8(**s["out"])
        if c["op"] == "decode":
            s["attn"] = torch.empty(b, nh, D, dtype=BF, device="cuda")
            s["workspace"] = kernels.attn_decode_q8_workspace(b, nh, nk, D, s_cap, "cuda", weights=bool(c["weights"]))
        if c["op"] == "write":
            s["q_out"] = torch.empty(b * c["n"], nh, D, dtype=BF, device="cuda")
    return s


# ----------------------------------------------------------------------------------- the framework's calls


def _own(s):
    from torch2vk_amd import kernels

    c, cache = s["case"], s["cache"]
    nh, nk = c["nh"], c["nk"]
    if c["op"] in ("decode", "write"):
        q, k, v = s["qkv"][:, :nh * D], s["qkv"][:, nh * D:(nh + nk) * D], s["qkv"][:, (nh + nk) * D:]
        args = dict(rope_offsets=s["rope_offsets"], q_norm_weight=s["q_norm_weight"], k_norm_weight=s["k_norm_weight"],
                    theta=s["theta"], eps=EPS)
    if c["op"] == "decode":
        kernels.attn_decode_q8(q, k, v, cache, s["attn"], s["lengths"], s["workspace"], weights=s.get("weights"),
                               weights_out=s.get("weights_out"), **args)
        return dict(out=s["attn"], k_tail=cache.k_tail, v_tail=cache.v_tail, weights=s.get("weights_out"))
    if c["op"] == "write":
        kernels.qk_norm_rope_cache_q8(q, k, v, s["q_out"], cache, s["lengths"], counts=s["counts"], **args)
        keys, values = kernels.kv_cache_q8_dequantize(cache, s["lengths"] + s["counts"])
        return dict(q=s["q_out"], k=keys, v=values)
    if c["op"] == "chunk":
        out = kernels.flash_attn_prefill_q8(s["q"], cache, s["lengths"], counts=s["counts"], weights=s.get("weights"),
                                            weights_out=s.get("weights_out"))
        return dict(out=out, weights=s.get("weights_out"))
    kept, lengths = kernels.kv_cache_q8_evict(cache, s["lengths"], s["weights"], c["keep"], sink=c["sink"],
                                              recent=c["recent"], out=s["out"], weights_out=s["weights_out"])
    keys, values = kernels.kv_cache_q8_dequantize(s["out"], lengths)
    return dict(kept=kept, lengths=lengths, k=keys, v=values, weights=s["weights_out"])


# ------------------------------------------------------------------------------------------- the plain form


def _norm_rope(x, w, pos):
    """Per-head RMS norm and rotate-half RoPE, fp32 [rows, heads, D] at int positions [rows]."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    freq = THETA ** (-torch.arange(D // 2, dtype=F64, device=x.device) / (D // 2))
    angle = (pos.to(F64)[:, None] * freq)[:, None, :]  # 64 bits: a far position has few bits left for its angle
    cos, sin = torch.cos(angle).to(F32), torch.sin(angle).to(F32)
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _heads(s):
    c = s["case"]
    return [x.reshape(len(s["qkv"]), -1, D) for x in s["qkv"].split([c["nh"] * D, c["nk"] * D, c["nk"] * D], 1)]


def _whole(cache, length, s_cap):
    """fp32 K and V [seq, head, token, D] of all s_cap tokens; zeros from the length on."""
    k = cache["k"].to(F32) * cache["k_scale"][..., None, None]
    v = (cache["v"].to(F32) * cache["v_scale"][..., None, None]).transpose(-1, -2)
    tok = torch.arange(s_cap, device="cuda")
    in_tail = ((tok >= (length // BLOCK * BLOCK)[:, None]) & (tok < length[:, None]))[:, None, :, None]
    live = (tok < length[:, None])[:, None, :, None]
    parts = []
    for x, tail in ((k, cache["k_tail"]), (v, cache["v_tail"].transpose(-1, -2))):
        x = x.permute(0, 2, 1, 3, 4).flatten(2, 3)
        x = torch.where(in_tail, tail.to(F32).repeat(1, 1, s_cap // BLOCK, 1), x)
        parts.append(torch.where(live, x, 0.0))
    return parts


def _attention(q, k, v, seen):
    """softmax(q k / sqrt(D)) v over the keys of ``seen``, and its weights; q [seq, head, rows, D], zeros where none is."""
    score = torch.matmul(q, k.transpose(-1, -2)) * D ** -0.5
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(score - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    return torch.matmul(p, v), p


def _add_weights(s, p, length, end):
    """Accumulated weights: a cached token's grow, a new token's begin."""
    tok = torch.arange(p.shape[-1], device="cuda")
    old = (tok < length[:, None])[:, None]
    live = (tok < end[:, None])[:, None]
    return torch.where(live, torch.where(old, s["weights"], 0.0) + p.sum(2), 0.0)


def _plain_decode(s):
    c, cache = s["case"], s["cache"]
    b, nk, s_cap = c["n_seq"], c["nk"], c["s_cap"]
    length = s["lengths"].long()
    pos = length + s["rope_offsets"]
    q, k, v = _heads(s)
    q, k = _norm_rope(q, s["q_norm_weight"], pos), _norm_rope(k, s["k_norm_weight"], pos)
    seq = torch.arange(b, device="cuda")
    cache["k_tail"][seq, :, length % BLOCK] = k.to(BF)
    cache["v_tail"][seq, :, :, length % BLOCK] = v.to(BF)
    keys, values = _whole(cache, length + 1, s_cap)
    seen = (torch.arange(s_cap, device="cuda") <= length[:, None])[:, None, None]
    out, p = _attention(q.reshape(b, nk, -1, D), keys, values, seen)
    weights = _add_weights(s, p, length, length + 1) if c["weights"] else None
    return dict(out=out.reshape(b, c["nh"], D).to(BF), k_tail=cache["k_tail"], v_tail=cache["v_tail"], weights=weights)


def _plain_write(s):
    c, cache = s["case"], s["cache"]
    b, nk, n, nb = c["n_seq"], c["nk"], c["n"], c["s_cap"] // BLOCK
    length, count = s["lengths"].long(), s["counts"].long()
    step = torch.arange(n, device="cuda")
    pos = (length[:, None] + s["rope_offsets"][:, None] + step).reshape(-1)
    q, k, v = _heads(s)
    valid = (step < count[:, None]).reshape(-1, 1, 1)
    q = torch.where(valid, _norm_rope(q, s["q_norm_weight"], pos), 0.0).to(BF)
    k = _norm_rope(k, s["k_norm_weight"], pos)
    tok = torch.arange(c["s_cap"], device="cuda")
    at = (tok - length[:, None]).clamp(0, n - 1)[:, :, None, None].expand(-1, -1, nk, D)
    end = (length + count)[:, None]
    new = ((tok >= length[:, None]) & (tok < end))[:, :, None, None]
    done = (torch.arange(nb, device="cuda") * BLOCK + BLOCK <= end)
    fresh = done & (torch.arange(nb, device="cuda") * BLOCK >= length[:, None] // BLOCK * BLOCK)
    seq, last = torch.arange(b, device="cuda"), ((length + count) // BLOCK).clamp(max=nb - 1)
    for name, x in (("k", k), ("v", v)):
        x = torch.gather(x.reshape(b, n, nk, D).to(BF), 1, at)
        tail = cache["k_tail"] if name == "k" else cache["v_tail"].transpose(-1, -2)
        x = torch.where(new, x, tail.transpose(1, 2).repeat(1, nb, 1, 1))
        x = x.reshape(b, nb, BLOCK, nk, D).transpose(2, 3)
        x = x if name == "k" else x.transpose(-1, -2)
        codes, scale = _quantized(x)
        cache[name] = torch.where(fresh[:, :, None, None, None], codes, cache[name])
        cache[name + "_scale"] = torch.where(fresh[:, :, None], scale, cache[name + "_scale"])
        # no tail is kept for the next pass: the cases begin at whole blocks and read none of the old one's rows
        cache[name + "_tail"] = x[seq, last]
    keys, values = _whole(cache, length + count, c["s_cap"])
    return dict(q=q, k=keys.transpose(1, 2).to(BF), v=values.transpose(1, 2).to(BF))


def _plain_chunk(s):
    c = s["case"]
    b, nh, nk, n, s_cap = c["n_seq"], c["nh"], c["nk"], c["n"], c["s_cap"]
    length, count = s["lengths"].long(), s["counts"].long()
    keys, values = _whole(s["cache"], length + count, s_cap)
    step = torch.arange(n, device="cuda")
    seen = torch.arange(s_cap, device="cuda") <= (length[:, None] + step)[:, :, None]
    seen = (seen & (step < count[:, None])[:, :, None])[:, None, None].expand(-1, -1, nh // nk, -1, -1).flatten(2, 3)
    q = s["q"].to(F32).reshape(b, n, nk, nh // nk, D).permute(0, 2, 3, 1, 4).reshape(b, nk, -1, D)
    out, p = _attention(q, keys, values, seen)
    out = out.reshape(b, nk, nh // nk, n, D).permute(0, 3, 1, 2, 4).reshape(b, n, nh, D)
    weights = _add_weights(s, p, length, length + count) if c["weights"] else None
    return dict(out=out.to(BF), weights=weights)


def _plain_evict(s):
    c = s["case"]
    b, nk, s_cap, most = c["n_seq"], c["nk"], c["s_cap"], c["keep"] * BLOCK
    length = s["lengths"].long()
    full = length // BLOCK * BLOCK
    stay = full.clamp(max=most)
    tok = torch.arange(s_cap, device="cuda")
    safe = (tok < c["sink"]) | (tok >= (full - c["recent"])[:, None])
    rank = torch.where(safe[:, None], math.inf, s["weights"])
    rank = torch.where((tok < full[:, None])[:, None], rank, -1.0)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :most]
    slot = torch.arange(most, device="cuda")
    used = (slot < stay[:, None])[:, None].expand(-1, nk, -1)
    kept = torch.sort(torch.where(used, order, s_cap), -1).values
    lengths = stay + length - full
    keys, values = _whole(s["cache"], length, s_cap)
    # the kept tokens of whole blocks, rounded again under their new blocks' scales; the tail stays as it is
    places = kept.clamp(max=s_cap - 1)
    cap = most + BLOCK
    parts = []
    for x, tail in ((keys, s["cache"]["k_tail"]), (values, s["cache"]["v_tail"].transpose(-1, -2))):
        x = torch.gather(x, 2, places[..., None].expand(-1, -1, -1, D))
        codes, scale = _quantized(torch.where(used[..., None], x, 0.0).reshape(b, nk, -1, BLOCK, D))
        x = torch.cat([(codes.to(F32) * scale[..., None, None]).flatten(2, 3), torch.zeros(b, nk, BLOCK, D, device="cuda")], 2)
        parts.append(_behind(x, tail.to(F32), stay, lengths, cap))
    weights = torch.gather(s["weights"], 2, places)
    weights = torch.cat([torch.where(used, weights, 0.0), torch.zeros(b, nk, BLOCK, device="cuda")], 2)
    last = torch.gather(s["weights"], 2, (full[:, None] + torch.arange(BLOCK, device="cuda")).clamp(max=s_cap - 1)[:, None].expand(-1, nk, -1))
    weights = _behind(weights[..., None], last[..., None], stay, lengths, cap)[..., 0]
    return dict(kept=torch.where(used, kept, -1).to(torch.int32), lengths=lengths.to(torch.int32),
                k=parts[0].transpose(1, 2).to(BF), v=parts[1].transpose(1, 2).to(BF), weights=weights)


def _behind(x, tail, stay, lengths, cap):
    """x [seq, head, cap, .] with the tail's tokens from ``stay`` to ``lengths``."""
    tok = torch.arange(cap, device="cuda")
    here = ((tok >= stay[:, None]) & (tok < lengths[:, None]))[:, None, :, None]
    return torch.where(here, tail.repeat(1, 1, cap // BLOCK, 1), x)


def run(state):
    if own:
        return _own(state)
    return {"decode": _plain_decode, "write": _plain_write, "chunk": _plain_chunk, "evict": _plain_evict}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ the work


def _lengths(case):
    """The mean length and number of new tokens that the inputs have."""
    return (case["lo"] + case["hi"]) / 2, (case.get("n_lo", 1) + case.get("n", 1)) / 2


def work(case):
    c = case
    b, nh, nk = c["n_seq"], c["nh"], c["nk"]
    length, count = _lengths(c)
    token = 2 * nk * D  # bytes of one cached token's K and V
    if c["op"] == "decode":
        moved = b * (length * token + 4 * (nh + 2 * nk) * D + 2 * nh * D + 2 * token)
        if c["weights"]:
            moved += b * 8 * nk * length
        return dict(bytes=moved, flops=b * 4.0 * nh * D * length)
    if c["op"] == "write":  # the values in bf16, as the call gives them, are written too
        moved = b * count * ((nh + 2 * nk) * D * 4 + nh * D * 2 + 2 * token) + b * (length * token + c["s_cap"] * 2 * token)
        return dict(bytes=moved, flops=b * count * 10.0 * (nh + 2 * nk) * D)
    if c["op"] == "chunk":
        moved = b * ((length + count) * token + count * 4 * nh * D) + (b * 8 * nk * (length + count) if c["weights"] else 0)
        return dict(bytes=moved, flops=b * (6.0 if c["weights"] else 4.0) * nh * D * count * (length + count / 2))
    stay = min(length // BLOCK, c["keep"]) * BLOCK
    moved = b * (4 * nk * length + stay * (2 * token + 12 * nk) + stay * token + (stay + BLOCK) * 2 * token)
    return dict(bytes=moved, flops=b * nk * length * 4.0)


# ------------------------------------------------------------------------------------- the definition in 64 bits


def _exact_norm_rope(x, w, pos):
    x = x.to(F64)
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.to(F64)
    half = D // 2
    turn = pos.to(F64)[:, None, None] / torch.pow(torch.tensor(THETA, dtype=F64, device="cuda"),
                                                  torch.arange(half, dtype=F64, device="cuda") / half)
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * turn.cos() - hi * turn.sin(), hi * turn.cos() + lo * turn.sin()], -1)


def _exact_round(x):
    """Token rows [64, D] -> the values that 8 bits under one scale hold."""
    step = x.abs().max() / 127
    return torch.round(x / step) * step if step > 1e-30 else torch.zeros_like(x)


def _exact_rows(cache, i, h, n):
    """fp64 K and V rows [n, D] of one sequence's head."""
    full = n // BLOCK
    k = (cache["k"][i, :full, h].to(F64) * cache["k_scale"][i, :full, h, None, None].to(F64)).reshape(-1, D)
    v = (cache["v"][i, :full, h].to(F64) * cache["v_scale"][i, :full, h, None, None].to(F64)).transpose(1, 2).reshape(-1, D)
    r = n - full * BLOCK
    return torch.cat([k, cache["k_tail"][i, h, :r].to(F64)]), torch.cat([v, cache["v_tail"][i, h, :, :r].T.to(F64)])


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c, cache = case, s["cache"]
    b, nh, nk = c["n_seq"], c["nh"], c["nk"]
    g = nh // nk
    lens = s["lengths"].tolist()
    if c["op"] in ("decode", "chunk"):
        n = c.get("n", 1)
        out = torch.zeros(b, n, nh, D, dtype=F64, device="cuda")
        weights = torch.zeros(b, nk, c["s_cap"], dtype=F64, device="cuda") if c["weights"] else None
        counts = s["counts"].tolist() if c["op"] == "chunk" else [1] * b
        if c["op"] == "decode":
            pos = s["lengths"].long() + s["rope_offsets"].long()
            q, k, v = _heads(s)
            q = _exact_norm_rope(q, s["q_norm_weight"], pos)[:, None]
            k = _exact_norm_rope(k, s["k_norm_weight"], pos)
            for i, at in enumerate(lens):
                cache["k_tail"][i, :, at % BLOCK] = k[i].to(BF)
                cache["v_tail"][i, :, :, at % BLOCK] = v[i].to(BF)
        else:
            q = s["q"].to(F64)
        for i in range(b):
            for h in range(nk):
                keys, values = _exact_rows(cache, i, h, lens[i] + counts[i])
                for j in range(h * g, (h + 1) * g):
                    for t in range(0, counts[i], 512):
                        rows = q[i, t:min(t + 512, counts[i]), j]
                        score = rows @ keys.T / math.sqrt(D)
                        last = lens[i] + t + torch.arange(len(rows), device="cuda")
                        score.masked_fill_(torch.arange(len(keys), device="cuda") > last[:, None], -math.inf)
                        p = torch.softmax(score, -1)
                        out[i, t:t + len(rows), j] = p @ values
                        if weights is not None:
                            weights[i, h, :len(keys)] += p.sum(0)
            if weights is not None:
                weights[i, :, :lens[i]] += s["weights"][i, :, :lens[i]].to(F64)
        if c["op"] == "chunk":
            return dict(out=out, weights=weights)
        return dict(out=out[:, 0], k_tail=None, v_tail=None, weights=weights)
    if c["op"] == "write":
        n, counts = c["n"], s["counts"].tolist()
        q, k, v = _heads(s)
        pos = (s["lengths"].long() + s["rope_offsets"].long())[:, None] + torch.arange(n, device="cuda")
        q = _exact_norm_rope(q, s["q_norm_weight"], pos.reshape(-1)).reshape(b, n, nh, D)
        k = _exact_norm_rope(k, s["k_norm_weight"], pos.reshape(-1)).to(BF).to(F64).reshape(b, n, nk, D)
        v = v.to(BF).to(F64).reshape(b, n, nk, D)
        keys = torch.zeros(b, c["s_cap"], nk, D, dtype=F64, device="cuda")
        values = torch.zeros_like(keys)
        for i in range(b):
            q[i, counts[i]:] = 0
            for h in range(nk):
                old = _exact_rows(cache, i, h, lens[i])
                for to, kept, new in ((keys, old[0], k), (values, old[1], v)):
                    x = torch.cat([kept, new[i, :counts[i], h]])
                    for t in range(lens[i] // BLOCK * BLOCK, len(x) // BLOCK * BLOCK, BLOCK):
                        x[t:t + BLOCK] = _exact_round(x[t:t + BLOCK])
                    to[i, :len(x), h] = x
        return dict(q=q.reshape(b * n, nh, D), k=keys, v=values)
    cap = (c["keep"] + 1) * BLOCK
    keys = torch.zeros(b, cap, nk, D, dtype=F64, device="cuda")
    values = torch.zeros_like(keys)
    weights = torch.zeros(b, nk, cap, dtype=F64, device="cuda")
    kept = torch.full((b, nk, c["keep"] * BLOCK), -1, dtype=torch.int32)
    lengths = torch.zeros(b, dtype=torch.int32)
    for i in range(b):
        full = lens[i] // BLOCK * BLOCK
        stay = min(full, c["keep"] * BLOCK)
        lengths[i] = stay + lens[i] - full
        for h in range(nk):
            w = s["weights"][i, h].to(F64)
            safe = set(range(min(c["sink"], full))) | set(range(max(0, full - c["recent"]), full))
            host = w[:full].tolist()
            order = sorted(range(full), key=lambda t: (t not in safe, -host[t], t))
            mine = sorted(order[:stay])
            kept[i, h, :stay] = torch.tensor(mine, dtype=torch.int32)
            at = torch.tensor(mine + list(range(full, lens[i])), device="cuda", dtype=torch.long)
            weights[i, h, :len(at)] = w[at]
            for to, x in zip((keys, values), _exact_rows(cache, i, h, lens[i])):
                x = x[at]
                for t in range(0, stay, BLOCK):
                    x[t:t + BLOCK] = _exact_round(x[t:t + BLOCK])
                to[i, :len(x), h] = x
    return dict(kept=kept, lengths=lengths, k=keys, v=values, weights=weights)
