"""What the operators for trees of drafted tokens are measured on: listed and drawn cases, their plain form, the calls that a user
makes of the framework (``own``), and their definition in 64 bits.

A step checks up to 64 drafted tokens of a sequence at once.  They are the nodes of a tree: node i hangs on the earlier node
``parents[i]``, or on the cached tokens (-1).  Operators: ``attn`` (the nodes' q/k norm and RoPE at the positions that their depths
give, their K and V into the slots behind the cached tokens, and attention of each node over the cached tokens, its ancestors and
itself), ``verify`` (the walk down the tree that the target's probabilities and given random numbers accept, and the token that
follows it), ``keep`` (the accepted nodes' K and V rows, in all layers, to where the cache goes on)."""

import math

import torch

own = False

D, EPS, THETA = 128, 1e-6, 1e6
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # one user's short chat with a few drafted tokens: 28 of these calls in every step, where latency is all that counts
        dict(name="attn_1x8_at_500", op="attn", n_seq=1, n=8, n_lo=8, nh=16, nk=8, lo=500, hi=500, s_cap=2048, shape="tree"),
        # one user, a bushy tree behind a few pages
        dict(name="attn_1x26_at_4100", op="attn", n_seq=1, n=26, n_lo=26, nh=32, nk=8, lo=4100, hi=4100, s_cap=8192, shape="tree"),
        # a served batch of ragged lengths, short chains of drafts
        dict(name="attn_16x5_ragged", op="attn", n_seq=16, n=5, n_lo=2, nh=32, nk=8, lo=100, hi=8000, s_cap=8192, shape="chain"),
        # the largest trees behind long contexts
        dict(name="attn_4x64_at_15000", op="attn", n_seq=4, n=64, n_lo=50, nh=32, nk=8, lo=14000, hi=15000, s_cap=16384, shape="tree"),
        # a full batch of long contexts: as many bytes as a step over a large cache reads
        dict(name="attn_32x4_at_16000", op="attn", n_seq=32, n=4, n_lo=3, nh=32, nk=8, lo=15000, hi=16300, s_cap=16384, shape="chain"),
        # 8 q heads a KV head, an odd number of nodes and of slots
        dict(name="attn_2x63_at_2000", op="attn", n_seq=2, n=63, n_lo=40, nh=32, nk=4, lo=1800, hi=2001, s_cap=2077, shape="forest"),
        # greedy check of a short chain, latency
        dict(name="verify_greedy_1x8", op="verify", n_seq=1, n=8, n_lo=8, vocab=151936, dtype="f32", mode="greedy", shape="chain",
             temperature=0.0),
        # one user's tree, sampled
        dict(name="verify_tree_1x26", op="verify", n_seq=1, n=26, n_lo=26, vocab=151936, dtype="f32", mode="sample", shape="tree",
             temperature=0.7),
        # a batch whose drafts were drawn from a small model's probabilities
        dict(name="verify_drawn_16x5", op="verify", n_seq=16, n=5, n_lo=2, vocab=151936, dtype="bf16", mode="drawn", shape="chain",
             temperature=0.8),
        # a served batch of trees
        dict(name="verify_tree_32x16", op="verify", n_seq=32, n=16, n_lo=9, vocab=151936, dtype="f32", mode="sample", shape="tree",
             temperature=1.0),
        # one user's accepted path
        dict(name="keep_1x26", op="keep", layers=28, n_seq=1, n=26, nk=8, lo=1500, hi=1500, s_cap=2048, kept_lo=6, kept=6),
        # a served batch's, in the deepest configuration
        dict(name="keep_16x64", op="keep", layers=36, n_seq=16, n=64, nk=8, lo=100, hi=950, s_cap=1024, kept_lo=8, kept=20),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "verify", "verify", "keep"])
    if op == "attn":
        nh, nk = rng.choice([(16, 8), (32, 8), (8, 8), (32, 4), (24, 8), (20, 4), (16, 1)])
        n_seq, n = _spread(rng, 1, 32), _spread(rng, 1, 64)
        most = min(60000, 200000 // n_seq, int(6e10 / (512 * n_seq * n * nh)))
        hi = _spread(rng, 16, max(17, most))
        return dict(op=op, n_seq=n_seq, n=n, n_lo=rng.randint(max(1, n // 2), n), nh=nh, nk=nk, lo=rng.choice([hi, hi // 2, 0]),
                    hi=hi, s_cap=hi + n + rng.choice([0, 1, 37, hi]), shape=rng.choice(["chain", "tree", "forest"]))
    if op == "verify":
        vocab = rng.choice([151936, 151936, _spread(rng, 500, 200000)])
        n_seq = _spread(rng, 1, 64)
        n = _spread(rng, 1, min(64, max(2, 70_000_000 // (n_seq * vocab))))
        mode = rng.choice(["greedy", "sample", "drawn"])
        return dict(op=op, n_seq=n_seq, n=n, n_lo=rng.randint(max(1, n // 2), n), vocab=vocab, dtype=rng.choice(["f32", "bf16"]),
                    mode=mode, shape="chain" if mode == "drawn" else rng.choice(["chain", "tree"]),
                    temperature=0.0 if mode == "greedy" else round(rng.uniform(0.3, 1.5), 2))
    nk, layers = rng.choice([1, 2, 4, 8]), rng.choice([4, 28, 36])
    n_seq, n = _spread(rng, 1, 16), _spread(rng, 4, 64)
    hi = _spread(rng, 16, 900)
    kept = rng.randint(2, max(2, min(20, n // 2)))
    return dict(op=op, layers=layers, n_seq=n_seq, n=n, nk=nk, lo=rng.choice([hi, hi // 2]), hi=hi, s_cap=hi + n + rng.choice([0, 3]),
                kept_lo=max(2, kept // 2), kept=kept)


# ------------------------------------------------------------------------------------------------------ inputs


def _ragged(lo, hi, b, host):
    x = torch.randint(lo, hi + 1, (b,), generator=host)
    x[0] = hi
    return x


def _parents(shape, b, n, host):
    """A chain; a tree whose first nodes have most children; or a forest, some of whose nodes hang on the cached tokens."""
    i = torch.arange(n)
    if shape == "chain":
        return (i - 1).expand(b, n).to(torch.int32)
    up = (torch.rand(b, n, generator=host).pow(1.5) * i).long().clamp(max=(i - 1).clamp(min=0))
    up = torch.where(i > 0, up, -1)
    if shape == "forest":
        up = torch.where(torch.rand(b, n, generator=host) < 0.15, -1, up)
    return up.to(torch.int32)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    b, n = c["n_seq"], c["n"]

    def rows(*shape, spread=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * spread

    s = dict(case=c)
    if c["op"] != "verify":
        s["lengths"] = _ragged(c["lo"], c["hi"], b, host).to(torch.int32).cuda()
    if c["op"] != "keep":
        s["counts"] = _ragged(c["n_lo"], n, b, host).to(torch.int32).cuda()
        s["parents"] = _parents(c["shape"], b, n, host).cuda()
    if c["op"] == "attn":
        nh, nk, s_cap = c["nh"], c["nk"], c["s_cap"]
        # keys have a few strong channels, as rotary keys do; values none
        channel = 1.0 + 3.0 * (torch.rand(D, generator=gen, device="cuda") < 0.06)
        s["k_cache"] = torch.empty(b, s_cap, nk, D, dtype=BF, device="cuda")
        s["v_cache"] = torch.empty(b, s_cap, nk, D, dtype=BF, device="cuda")
        for i in range(b):
            s["k_cache"][i] = rows(s_cap, nk, D) * channel
            s["v_cache"][i] = rows(s_cap, nk, D)
        s["qkv"] = rows(b * n, (nh + 2 * nk) * D, spread=2.0)  # one product's columns: q, k, v
        s["q_norm_weight"] = 1.0 + 0.3 * rows(D)
        s["k_norm_weight"] = channel * (1.0 + 0.1 * rows(D))
        if own:
            from torch2vk_amd import kernels

            s["out"] = torch.empty(b, n, nh, D, dtype=BF, device="cuda")
            s["workspace"] = kernels.attn_tree_workspace(b, n, nh, nk, D, s_cap, "cuda")
        return s
    if c["op"] == "verify":
        vocab, dtype = c["vocab"], F32 if c["dtype"] == "f32" else BF
        logits = rows(b, n, vocab, spread=2.0)
        at = torch.randint(0, vocab, (b, n, 12), generator=gen, device="cuda")  # a few likely tokens after each node
        logits.scatter_add_(2, at, rows(b, n, 12).abs() * 3 + 7)
        s["logits"] = logits.to(dtype)
        s["temperature"] = torch.full((b,), c["temperature"], device="cuda")
        s["uniforms"] = torch.rand(b, n, generator=gen, device="cuda")
        if c["mode"] == "drawn":
            draft = logits[:, :n - 1] * 0.9 + rows(b, n - 1, vocab, spread=0.5)
            s["draft_logits"] = draft.to(dtype)
            race = torch.empty_like(draft).exponential_(generator=gen)
            drawn = (s["draft_logits"].to(F32) / c["temperature"] - race.log()).argmax(-1) if n > 1 else at[:, :0, 0]
            s["tokens"] = torch.cat([at[:, :1, 0], drawn], 1).contiguous()
        else:  # a node's children are its likeliest tokens, in order, now and then one further down
            up = s["parents"].long()
            earlier = (up[:, None] == up[:, :, None]) & (torch.arange(n, device="cuda") < torch.arange(n, device="cuda")[:, None])
            rank = earlier.sum(-1) + (torch.rand(b, n, generator=gen, device="cuda") < 0.2)
            likely = s["logits"].to(F32).topk(min(16, vocab), -1).indices
            of_parent = torch.gather(likely, 1, up.clamp(min=0)[..., None].expand(-1, -1, likely.shape[-1]))
            s["tokens"] = torch.gather(of_parent, 2, (rank % likely.shape[-1])[..., None])[..., 0].contiguous()
        if own:
            from torch2vk_amd import kernels

            s["path"] = torch.empty(b, n, dtype=torch.int32, device="cuda")
            s["kept"] = torch.empty(b, dtype=torch.int32, device="cuda")
            s["next_token"] = torch.empty(b, dtype=torch.int64, device="cuda")
            s["workspace"] = kernels.tree_verify_workspace(b, n, vocab, "cuda", drawn=c["mode"] == "drawn")
        return s
    layers, nk, s_cap = c["layers"], c["nk"], c["s_cap"]
    s["k_cache"] = torch.empty(layers, b, s_cap, nk, D, dtype=BF, device="cuda")
    s["v_cache"] = torch.empty(layers, b, s_cap, nk, D, dtype=BF, device="cuda")
    for i in range(layers):
        s["k_cache"][i] = rows(b, s_cap, nk, D)
        s["v_cache"][i] = rows(b, s_cap, nk, D)
    # accepted nodes behind the slots that they come to, as in a tree laid out level by level: a second pass moves the same rows
    kept = _ragged(c["kept_lo"], c["kept"], b, host)
    path = torch.full((b, n), -1)
    for i, m in enumerate(kept.tolist()):
        path[i, 0] = 0
        path[i, 1:m] = m + torch.randperm(n - m, generator=host)[:m - 1].sort().values
    s["path"], s["kept"] = path.to(torch.int32).cuda(), kept.to(torch.int32).cuda()
    return s


# ----------------------------------------------------------------------------------- the framework's calls


def _own(s):
    from torch2vk_amd import kernels

    c = s["case"]
    if c["op"] == "attn":
        nh, nk = c["nh"], c["nk"]
        q, k, v = s["qkv"][:, :nh * D], s["qkv"][:, nh * D:(nh + nk) * D], s["qkv"][:, (nh + nk) * D:]
        kernels.attn_tree(q, k, v, s["k_cache"], s["v_cache"], s["out"], s["lengths"], s["workspace"], theta=THETA,
                          parents=s["parents"], counts=s["counts"], q_norm_weight=s["q_norm_weight"],
                          k_norm_weight=s["k_norm_weight"], eps=EPS)
        return dict(out=s["out"], k=s["k_cache"], v=s["v_cache"])
    if c["op"] == "verify":
        path, kept, following = kernels.tree_verify(
            s["logits"], s["tokens"], s["workspace"], temperature=s["temperature"], uniforms=s["uniforms"],
            parents=None if c["mode"] == "drawn" else s["parents"], counts=s["counts"], draft_logits=s.get("draft_logits"),
            path=s["path"], kept=s["kept"], next_token=s["next_token"])
        return dict(path=path, kept=kept, next_token=following)
    kernels.tree_keep(s["k_cache"], s["v_cache"], s["path"], s["kept"], s["lengths"])
    return dict(k=s["k_cache"], v=s["v_cache"])


# ------------------------------------------------------------------------------------------- the plain form


def _lineage(parents):
    """[seq, i, j]: node j is i or an ancestor of i."""
    n = parents.shape[1]
    at = torch.arange(n, device="cuda")
    line = ((parents[..., None] == at) | (at[:, None] == at)).to(F32)
    for _ in range(6):  # 64 generations
        line = (torch.matmul(line, line) > 0).to(F32)
    return line > 0


def _norm_rope(x, w, pos):
    """Per-head RMS norm and rotate-half RoPE, fp32 [seq, node, head, D] at int positions [seq, node]."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    freq = THETA ** (-torch.arange(D // 2, dtype=F64, device=x.device) / (D // 2))
    angle = (pos.to(F64)[..., None] * freq)[:, :, None, :]  # 64 bits: a far position has few bits left for its angle
    cos, sin = torch.cos(angle).to(F32), torch.sin(angle).to(F32)
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_attn(s):
    c = s["case"]
    b, n, nh, nk, s_cap = c["n_seq"], c["n"], c["nh"], c["nk"], c["s_cap"]
    length, step = s["lengths"].long(), torch.arange(n, device="cuda")
    line = _lineage(s["parents"])
    valid = step < s["counts"].long()[:, None]
    pos = length[:, None] + line.sum(-1) - 1
    q, k, v = [x.reshape(b, n, -1, D) for x in s["qkv"].split([nh * D, nk * D, nk * D], 1)]
    q, k = _norm_rope(q, s["q_norm_weight"], pos), _norm_rope(k, s["k_norm_weight"], pos)
    seq, slot = torch.arange(b, device="cuda")[:, None], length[:, None] + step
    for cache, new in ((s["k_cache"], k), (s["v_cache"], v)):
        cache[seq, slot] = torch.where(valid[..., None, None], new.to(BF), cache[seq, slot])
    tok = torch.arange(s_cap, device="cuda")
    node = (tok - length[:, None]).clamp(0, n - 1)[:, None, :].expand(-1, n, -1)
    seen = (tok < length[:, None])[:, None] | (torch.gather(line, 2, node) & (tok >= length[:, None])[:, None]
                                               & (tok < (length + s["counts"])[:, None])[:, None])
    seen = (seen & valid[..., None])[:, None, None].expand(-1, -1, nh // nk, -1, -1).reshape(b, 1, -1, s_cap)
    keys, values = (x.to(F32).transpose(1, 2) for x in (s["k_cache"], s["v_cache"]))
    rows = q.reshape(b, n, nk, nh // nk, D).permute(0, 2, 3, 1, 4).reshape(b, nk, -1, D)
    score = torch.where(seen, torch.matmul(rows, keys.transpose(-1, -2)) * D ** -0.5, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e / torch.where(total == 0, 1.0, total), values)
    out = out.reshape(b, nk, nh // nk, n, D).permute(0, 3, 1, 2, 4).reshape(b, n, nh, D)
    return dict(out=out.to(BF), k=s["k_cache"], v=s["v_cache"])


def _softmax_terms(logits, temperature):
    """exp(l / T - max) and the sum, in 64 bits: the borders between a large vocabulary's tokens lie close."""
    x = logits.to(F64) / temperature.to(F64)[:, None, None]
    w = torch.exp(x - x.amax(-1, keepdim=True))
    return w, w.sum(-1)


def _walk(up, accepted, count):
    """The nodes on the accepted path: the accepted child of a node on it that no accepted sibling comes before."""
    b, n = up.shape
    at = torch.arange(n, device="cuda")
    sibling = (up[:, :, None] == up[:, None, :]) & (at < at[:, None])  # [seq, i, j]: j is an earlier child of i's parent
    first = accepted & (at < count[:, None]) & (at > 0) & ~(sibling & accepted[:, None]).any(-1)
    first[:, 0] = count > 0
    on = (~_lineage(up) | first[:, None]).all(-1)
    kept = on.sum(-1)
    path = torch.where(on, at, n).sort(-1).values
    last = torch.gather(path, 1, (kept - 1).clamp(min=0)[:, None])[:, 0]
    return torch.where(path < n, path, -1).to(torch.int32), kept.to(torch.int32), last


def _plain_verify(s):
    c = s["case"]
    b, n, vocab = c["n_seq"], c["n"], c["vocab"]
    up, tokens, count = s["parents"].long(), s["tokens"], s["counts"].long()
    at, seq = torch.arange(n, device="cuda"), torch.arange(b, device="cuda")
    place = (seq[:, None], up.clamp(min=0), tokens)  # a node's token in the row of its parent
    if c["mode"] == "greedy":
        x = s["logits"].to(F32)
        best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(vocab, device="cuda"), vocab).amin(-1)
        path, kept, last = _walk(up, torch.gather(best, 1, up.clamp(min=0)) == tokens, count)
        return dict(path=path, kept=kept, next_token=best[seq, last])
    w, total = _softmax_terms(s["logits"], s["temperature"])
    u = s["uniforms"].to(F64)
    if c["mode"] == "sample":
        earlier = (up[:, :, None] == up[:, None, :]) & (at < at[:, None])
        again = (earlier & (tokens[:, :, None] == tokens[:, None, :])).any(-1)
        mine = torch.where(again, 0.0, w[place])
        rest = torch.gather(total, 1, up.clamp(min=0)) - (earlier * mine[:, None]).sum(-1)
        path, kept, last = _walk(up, u * rest < mine, count)
        out = torch.zeros(b, vocab + 1, dtype=torch.bool, device="cuda")
        gone = (up == last[:, None]) & (at < count[:, None])
        out.scatter_(1, torch.where(gone, tokens, vocab), True)
        mass = torch.where(out[:, :vocab], 0.0, w[seq, last])
    else:
        p = w / total[..., None]
        q, q_total = _softmax_terms(s["draft_logits"], s["temperature"]) if n > 1 else (p, total)
        q = q / q_total[..., None]
        q = torch.cat([q[:, :n - 1], torch.zeros_like(p[:, :1])], 1)
        path, kept, last = _walk(up, u * q[place] < p[place], count)
        mass = torch.where((last == count - 1)[:, None], p[seq, last], (p[seq, last] - q[seq, last]).clamp(min=0))
    run = mass.cumsum(-1)
    following = (run <= u[:, :1] * run[:, -1:]).sum(-1)
    return dict(path=path, kept=kept, next_token=following)


def _plain_keep(s):
    n = s["path"].shape[1]
    step, length = torch.arange(n, device="cuda"), s["lengths"].long()[:, None]
    move = (step < s["kept"].long()[:, None])
    source = length + torch.where(move, s["path"].long(), step)
    seq = torch.arange(len(length), device="cuda")[:, None]
    for cache in (s["k_cache"], s["v_cache"]):
        cache[:, seq, length + step] = cache[:, seq, source]
    return dict(k=s["k_cache"], v=s["v_cache"])


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "verify": _plain_verify, "keep": _plain_keep}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ the work


def work(case):
    """Of the mean lengths and numbers of nodes that the inputs have."""
    c = case
    b = c["n_seq"]
    if c["op"] == "attn":
        nh, nk = c["nh"], c["nk"]
        length, count = ((c["lo"] + c["hi"]) / 2, (c["n_lo"] + c["n"]) / 2) if b > 1 else (c["hi"], c["n"])
        moved = length * 4 * nk * D + count * ((nh + 2 * nk) * 4 * D + 2 * nh * D + 4 * nk * D)
        return dict(bytes=b * moved, flops=b * 4.0 * nh * D * count * length)
    if c["op"] == "verify":
        count = (c["n_lo"] + c["n"]) / 2 if b > 1 else c["n"]
        values = b * (2 * count - 1 if c["mode"] == "drawn" else count) * c["vocab"]
        return dict(bytes=values * (4.0 if c["dtype"] == "f32" else 2.0), flops=values * (1.0 if c["mode"] == "greedy" else 3.0))
    kept = (c["kept_lo"] + c["kept"]) / 2 if b > 1 else c["kept"]
    return dict(bytes=b * (kept - 1) * c["layers"] * c["nk"] * D * 8.0, flops=0.0)


# ------------------------------------------------------------------------------------- the definition in 64 bits


def _exact_norm_rope(x, w, pos):
    x = x.to(F64)
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.to(F64)
    half = D // 2
    turn = pos / torch.pow(torch.tensor(THETA, dtype=F64, device="cuda"), torch.arange(half, dtype=F64, device="cuda") / half)
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * turn.cos() - hi * turn.sin(), hi * turn.cos() + lo * turn.sin()], -1)


def _ancestors(parents, i):
    line = [i]
    while parents[line[-1]] >= 0:
        line.append(parents[line[-1]])
    return line


def _exact_attn(s):
    c = s["case"]
    b, n, nh, nk = c["n_seq"], c["n"], c["nh"], c["nk"]
    g = nh // nk
    out = torch.zeros(b, n, nh, D, dtype=F64, device="cuda")
    k_all, v_all = s["k_cache"].to(F64), s["v_cache"].to(F64)
    lens, counts, parents = s["lengths"].tolist(), s["counts"].tolist(), s["parents"].tolist()
    for i in range(b):
        m, at = counts[i], lens[i]
        lines = [_ancestors(parents[i], t) for t in range(m)]
        rows = s["qkv"][i * n:i * n + m]
        pos = torch.tensor([at + len(x) - 1 for x in lines], dtype=F64, device="cuda")[:, None, None]
        q = _exact_norm_rope(rows[:, :nh * D].reshape(m, nh, D), s["q_norm_weight"], pos)
        k_all[i, at:at + m] = _exact_norm_rope(rows[:, nh * D:(nh + nk) * D].reshape(m, nk, D), s["k_norm_weight"], pos)
        v_all[i, at:at + m] = rows[:, (nh + nk) * D:].reshape(m, nk, D).to(F64)
        hidden = torch.ones(m, at + m, dtype=torch.bool, device="cuda")
        hidden[:, :at] = False
        for t, x in enumerate(lines):
            hidden[t, [at + j for j in x]] = False
        for h in range(nk):  # the cache's rows, rounded to its type
            keys, values = (x[i, :at + m, h].to(BF).to(F64) for x in (k_all, v_all))
            score = torch.einsum("tgd,sd->gts", q[:, h * g:(h + 1) * g], keys) / math.sqrt(D)
            p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            out[i, :m, h * g:(h + 1) * g] = torch.einsum("gts,sd->tgd", p, values)
    return dict(out=out, k=k_all, v=v_all)


def _exact_verify(s):
    c = s["case"]
    b, n, vocab = c["n_seq"], c["n"], c["vocab"]
    path = torch.full((b, n), -1, dtype=torch.int32)
    kept, following = torch.zeros(b, dtype=torch.int32), torch.zeros(b, dtype=torch.int64)
    counts, parents, tokens = s["counts"].tolist(), s["parents"].tolist(), s["tokens"].tolist()
    uniforms = s["uniforms"].to(F64).tolist()
    for i in range(b):
        at, line = 0, [0]
        while True:
            row = s["logits"][i, at].to(F64)
            children = [j for j in range(at + 1, counts[i]) if parents[i][j] == at]
            if c["mode"] == "greedy":
                choice = int((row == row.max()).nonzero()[0, 0])
                step = [j for j in children if tokens[i][j] == choice][:1]
            else:
                t = s["temperature"][i].to(F64)
                mass = torch.softmax(row / t, -1)
                step = []
                for j in children:
                    x = tokens[i][j]
                    if c["mode"] == "sample":
                        if uniforms[i][j] * float(mass.sum()) < float(mass[x]):
                            step = [j]
                            break
                        mass[x] = 0.0
                    else:
                        q = torch.softmax(s["draft_logits"][i, at].to(F64) / t, -1)
                        if uniforms[i][j] * float(q[x]) < float(mass[x]):
                            step = [j]
                            break
                        mass = torch.clamp(mass - q, min=0.0)
            if not step:
                break
            at = step[0]
            line.append(at)
        if c["mode"] != "greedy":
            border = uniforms[i][0] * float(mass.sum())
            choice = int((torch.cumsum(mass, 0) > border).nonzero()[0, 0])
        path[i, :len(line)] = torch.tensor(line, dtype=torch.int32)
        kept[i], following[i] = len(line), choice
    return dict(path=path, kept=kept, next_token=following)


def _exact_keep(s):
    k, v = s["k_cache"].to(F64), s["v_cache"].to(F64)
    for i, (at, m) in enumerate(zip(s["lengths"].tolist(), s["kept"].tolist())):
        places = [at + j for j in s["path"][i, :m].tolist()]
        for x in (k, v):
            x[:, i, at:at + m] = x[:, i, places].clone()
    return dict(k=k, v=v)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"attn": _exact_attn, "verify": _exact_verify, "keep": _exact_keep}[case["op"]](s)
