"""Timed cases of the paged-cache operators: rotary positions, appends to a
paged cache with the rotation on the way, attention over the pages, and
attention for a batch that shares a long prefix.

``own`` false computes each operator in plain form (elementary torch operations
in 32 bits, angles in 64); true makes the calls of kvexp_amd. A case is a dict
of plain values; ``op`` says which operator:

  rope    Context.rope, and its gradient through torch.ops.kvexp.rope
  append  PagedCache.append: keys rotated and written to their pages, values
          copied, queries rotated
  paged   PagedCache.attention
  prefix  PagedCache.attention with a prefix that every sequence shares, kept
          as XKV containers (``xkv``) or as pages of the cache

Keys have a scale 2^U(-6, 4) per channel, as the codec meets them; queries are
scaled so that a score's standard deviation is about 3. Places of the pages
that no token fills hold NaN, as memory that nobody wrote may.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # three axes (frames, rows, columns) over the latents of a video: queries or keys of one layer
        dict(name="rope_video", op="rope", grad=False, tokens=32760, heads=12, dim=128, rotated=128, axes=3,
             interleaved=True, dtype="bf16"),
        # text positions far out, half of the channels rotated, forward and gradient of a training step
        dict(name="rope_train", op="rope", grad=True, tokens=8191, heads=14, dim=64, rotated=32, axes=1,
             interleaved=False, dtype="bf16"),
        # a decode step of 64 sequences: one layer's new keys and values (2 KV heads x 7 queries)
        dict(name="append_step", op="append", seqs=64, new=1, ragged=False, longest=32768, kv=2, group=7, dim=64,
             page=64, axes=1, dtype="bf16"),
        # prompts of up to 4K tokens of eight sequences with image parts (three axes), 8 KV heads x 4 queries
        dict(name="append_prompts", op="append", seqs=8, new=4096, ragged=True, longest=4096, kv=8, group=4, dim=128,
             page=64, axes=3, dtype="bf16"),
        # one sequence, one token: the smallest call, where launches and latency count
        dict(name="paged_one", op="paged", seqs=1, new=1, ragged=False, longest=1021, kv=2, group=7, dim=64, page=64,
             dtype="bf16", lse=True),
        # a decode step over 64 sequences of 1K to 32K tokens in small pages
        dict(name="paged_ragged", op="paged", seqs=64, new=1, ragged=False, longest=32768, kv=2, group=7, dim=64,
             page=16, dtype="bf16", lse=False),
        # long contexts at head_dim 128
        dict(name="paged_64k", op="paged", seqs=4, new=1, ragged=False, longest=65536, kv=8, group=4, dim=128,
             page=128, dtype="bf16", lse=False),
        # draft tokens checked in one call: up to 5 per sequence, head_dim 96, pages of 24 tokens, FP16
        dict(name="paged_drafts", op="paged", seqs=16, new=5, ragged=True, longest=16411, kv=8, group=4, dim=96,
             page=24, dtype="fp16", lse=True),
        # chunks of two prompts over what is cached already
        dict(name="paged_chunk", op="paged", seqs=2, new=2048, ragged=True, longest=16384, kv=8, group=4, dim=128,
             page=64, dtype="bf16", lse=False),
        # four sequences that share a system prompt of 4K tokens, compressed
        dict(name="prefix_4k", op="prefix", seqs=4, new=1, ragged=False, longest=300, prefix=4099, xkv=True, kv=2,
             group=7, dim=64, page=64, dtype="bf16", lse=True),
        # 64 sequences that share 64K compressed tokens (a document), a few hundred of their own each
        dict(name="prefix_64k", op="prefix", seqs=64, new=1, ragged=False, longest=1000, prefix=65536, xkv=True, kv=8,
             group=4, dim=128, page=64, dtype="bf16", lse=False),
        # 256 sequences that share 32K tokens kept in pages
        dict(name="prefix_pages", op="prefix", seqs=256, new=1, ragged=False, longest=512, prefix=32768, xkv=False,
             kv=2, group=7, dim=64, page=64, dtype="bf16", lse=False),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread over their logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "paged", "paged", "paged", "prefix", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256])
    page = rng.choice([16, 64, 64, 128, 24, 1, 100])
    if op == "rope":
        heads, axes = rng.randint(1, 32), rng.choice([1, 2, 3])
        return dict(op="rope", grad=rng.random() < 0.4, tokens=min(_log(rng, 1, 32768), 50_000_000 // (heads * dim)),
                    heads=heads, dim=dim, rotated=rng.choice([dim, dim, dim // 2, dim // 4]), axes=axes,
                    interleaved=rng.random() < 0.4, dtype=dtype)
    kv, group = rng.choice([1, 2, 3, 8]), rng.randint(1, 8)
    per = 4 * kv * dim  # bytes of a token's key and value
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, min(4096, 30_000_000 // (seqs * kv * (group + 2) * dim)))
        return dict(op="append", seqs=seqs, new=new, ragged=rng.random() < 0.5, longest=new + _log(rng, 1, 4096), kv=kv,
                    group=group, dim=dim, page=page, axes=rng.choice([1, 3]), dtype=dtype)
    lse = rng.random() < 0.3
    if op == "paged":
        seqs = _log(rng, 1, 64)
        longest = min(_log(rng, 1, 65536), 300_000_000 // (per * seqs))
        new = 1 if rng.random() < 0.6 else min(longest, _log(rng, 2, 512))
        new = max(1, min(new, 150_000_000 // (longest * seqs * kv * group)))
        return dict(op="paged", seqs=seqs, new=new, ragged=rng.random() < 0.5, longest=longest, kv=kv, group=group,
                    dim=dim, page=page, dtype=dtype, lse=lse)
    xkv = rng.random() < 0.6
    seqs = _log(rng, 2, 256)
    prefix = min(_log(rng, 100, 65536), 200_000_000 // per, 500_000_000 // (seqs * kv * group))
    longest = min(_log(rng, 1, 2000), 100_000_000 // (per * seqs))
    return dict(op="prefix", seqs=seqs, new=rng.choice([1, 1, 1, min(3, longest)]), ragged=False, longest=longest,
                prefix=prefix, xkv=xkv, kv=kv, group=group, dim=dim, page=page, dtype="bf16" if xkv else dtype, lse=lse)


# ------------------------------------------------------------------ inputs --
def lengths(case):
    """Tokens of each sequence, the new ones among them: the longest, the others spread over [1/32, 1] of it (the same
    for every seed)."""
    r = random.Random(case["seqs"] * 1000003 + case["longest"])
    n = case["longest"]
    return [n] + [max(1, _log(r, max(1, n // 32), n)) for _ in range(case["seqs"] - 1)]


def new_tokens(case):
    """New (query) tokens of each sequence: alike, or spread over [1, new]; no more than the sequence holds."""
    r = random.Random(case["seqs"] * 7919 + case["new"])
    most = [case["new"]] + [r.randint(1, case["new"]) if case["ragged"] else case["new"]
                            for _ in range(case["seqs"] - 1)]
    return [min(m, n) for m, n in zip(most, lengths(case))]


def _generator(seed, pos):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + pos) % (1 << 62))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _frequencies(rotated, axes):
    """Rotation frequencies and the axis of each: the axes take turns, as images and video interleave them."""
    n = rotated // 2
    freq = (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).to(torch.float32).cuda()
    return freq, (torch.arange(n) % axes).to(torch.uint8).cuda()


def _positions(g, tokens, axes):
    """Positions [axes, tokens]: far ones on one axis; frame, row and column on several."""
    if axes == 1:
        return (torch.arange(tokens, device="cuda") + torch.randint(0, 1 << 20, (1,), generator=g, device="cuda"))[None]
    return torch.randint(0, 1 << 10, (axes, tokens), generator=g, device="cuda")


def _pages(g, case, extra):
    """Page pools [pages, kv, page, dim] of keys and values, a table [seqs, width] of pages in random order, the
    lengths, and `extra` more pages; the keys' scales [kv, dim]."""
    ns, pt, kv, dim = lengths(case), case["page"], case["kv"], case["dim"]
    need = [(n + pt - 1) // pt for n in ns]
    width, pages = max(need), sum(need) + extra + 3
    scale = torch.exp2(torch.rand(kv, dim, generator=g, device="cuda") * 10 - 6)
    dtype = TYPES[case["dtype"]]
    k = (_normal(g, pages, kv, pt, dim) * scale[:, None]).to(dtype)
    v = (_normal(g, pages, kv, pt, dim) * 0.5).to(dtype)
    order = torch.randperm(pages, generator=g, device="cuda")
    at = torch.tensor([sum(need[:b]) for b in range(len(ns))], device="cuda")
    col = torch.arange(width, device="cuda")[None]
    held = col < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(held, order[torch.where(held, at[:, None] + col, 0)], -1).to(torch.int32)
    lens = torch.tensor(ns, dtype=torch.int32, device="cuda")
    # places past each sequence's end
    last = table.gather(1, (torch.tensor(need, device="cuda") - 1)[:, None])[:, 0].long()
    past = torch.arange(pt, device="cuda")[None] >= (lens - (torch.tensor(need, device="cuda") - 1) * pt)[:, None]
    where = torch.zeros(pages, pt, dtype=torch.bool, device="cuda")
    where[last] = past
    k.masked_fill_(where[:, None, :, None], math.nan)
    v.masked_fill_(where[:, None, :, None], math.nan)
    return k, v, table, lens, order[sum(need):sum(need) + extra].to(torch.int32), scale


def prepare(case, seed):
    s = dict(case=case)
    g = _generator(seed, 1)
    dtype = TYPES[case["dtype"]]
    if case["op"] == "rope":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        s["x"] = _normal(g, t, h, d).to(dtype).requires_grad_(case["grad"])
        s["dy"] = _normal(g, t, h, d).to(dtype) if case["grad"] else None
        s["freq"], s["axis"] = _frequencies(case["rotated"], case["axes"])
        s["pos"] = _positions(g, t, case["axes"])
        if own:
            kvexp = _kvexp()
            s["rope"] = kvexp.Rope(s["freq"], s["axis"], interleaved=case["interleaved"])
        return s
    dim, kv, heads = case["dim"], case["kv"], case["kv"] * case["group"]
    prefix = case.get("prefix", 0)
    paged = prefix and not case["xkv"]
    extra = (prefix + case["page"] - 1) // case["page"] if paged else 0
    s["k"], s["v"], s["table"], s["lens"], s["prefix_table"], scale = _pages(g, case, extra)
    ns = new_tokens(case)
    total = sum(ns)
    s["new"], s["most"] = ns, max(ns)
    starts = [sum(ns[:b]) for b in range(len(ns) + 1)]
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if min(ns) != max(ns) else None
    if case["op"] == "append":
        qkv = _normal(g, total, heads + 2 * kv, dim).to(dtype)  # one product gives all three
        s["q"], s["new_k"], s["new_v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        s["freq"], s["axis"] = _frequencies(dim, case["axes"])
        s["pos"] = _positions(g, total, case["axes"])
    else:
        norm = scale.square().sum(1).sqrt().repeat_interleave(case["group"])
        s["scale"] = 1.0 / math.sqrt(dim)
        s["q"] = (_normal(g, total, heads, dim) * (3 / norm / s["scale"])[:, None]).to(dtype)
        if prefix and case["xkv"]:
            s["prefix_k"] = (_normal(g, kv, prefix, dim) * scale[:, None]).to(dtype)
            x = _normal(g, kv, prefix, dim) * 0.5
            s["prefix_v"] = torch.where(torch.rand(kv, prefix, dim, generator=g, device="cuda") < 0.003, x * 2.0**-20,
                                        x).to(dtype)
    if own:
        kvexp, ctx = _kvexp(), _context()
        s["cache"] = kvexp.PagedCache(ctx, kv, dim, s["k"].shape[0], case["page"], dtype, k=s["k"], v=s["v"])
        if case["op"] == "append":
            s["rope"] = kvexp.Rope(s["freq"], s["axis"])
        if prefix and case["xkv"]:
            coded = [[ctx.encode(x[h], prefix, dim) for h in range(kv)] for x in (s["prefix_k"], s["prefix_v"])]
            s["prefix"] = ctx.prefix(coded[0], coded[1])
        elif prefix:
            s["prefix"] = s["cache"].prefix(s["prefix_table"], prefix)
    return s


# ------------------------------------------------------------- the framework --
_ctx = None


def _kvexp():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "compressed-kv-attention_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import kvexp_amd

    return kvexp_amd


def _context():
    global _ctx
    if _ctx is None:
        _ctx = _kvexp().Context(0)
    return _ctx


def _run_own(s):
    case = s["case"]
    if case["op"] == "rope":
        if not case["grad"]:
            return [_context().rope(s["x"], s["pos"], s["rope"])]
        import kvexp_amd.torch_ops  # noqa: F401  (registers the operator)

        y = torch.ops.kvexp.rope(s["x"], s["pos"], s["freq"], s["axis"], case["interleaved"])
        return [y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]]
    batch = _kvexp().Batch(s["table"], s["lens"], s["starts"], max_new=s["most"])
    if case["op"] == "append":
        q = s["cache"].append(s["new_k"], s["new_v"], batch, rope=s["rope"], positions=s["pos"], q=s["q"])
        return [s["k"], s["v"], q]
    return _outputs(case, s["cache"].attention(s["q"], batch, scale=s["scale"], prefix=s.get("prefix"),
                                               return_lse=case["lse"]))


def _outputs(case, r):
    return list(r) if case["lse"] else [r]


# ----------------------------------------------------------------- plain form --
def _rotate(x, pos, freq, axis, interleaved):
    """x [tokens, heads, dim] with its first 2 n channels rotated, in 32 bits; angles in 64."""
    n = freq.numel()
    angle = pos.double()[axis.long()].T * freq.double()
    c, si = angle.cos().float()[:, None], angle.sin().float()[:, None]
    f = x.float()
    a, b = (f[..., 0:2 * n:2], f[..., 1:2 * n:2]) if interleaved else (f[..., :n], f[..., n:2 * n])
    y1, y2 = a * c - b * si, b * c + a * si
    y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([y, f[..., 2 * n:]], -1).to(x.dtype)


def _token_places(s):
    """Sequence and place among its new tokens of every new token."""
    new = torch.tensor(s["new"], device="cuda")
    b = torch.repeat_interleave(torch.arange(len(s["new"]), device="cuda"), new, output_size=sum(s["new"]))
    start = new.cumsum(0) - new
    return b, torch.arange(b.numel(), device="cuda") - start[b], new


def _gather(pages, table):
    """The tokens [seqs, kv, width * page, dim] that a table of pages names, in 32 bits."""
    x = pages[table.long().clamp(min=0)]
    b, w, h, p, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, w * p, d).float()


def _run_plain(s):
    case = s["case"]
    if case["op"] == "rope":
        y = _rotate(s["x"], s["pos"], s["freq"], s["axis"], case["interleaved"])
        return [y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]] if case["grad"] else [y]
    b, i, new = _token_places(s)
    if case["op"] == "append":
        at = s["lens"].long()[b] - new[b] + i
        page = s["table"].long()[b, at // case["page"]]
        s["k"][page, :, at % case["page"]] = _rotate(s["new_k"], s["pos"], s["freq"], s["axis"], False)
        s["v"][page, :, at % case["page"]] = s["new_v"]
        return [s["k"], s["v"], _rotate(s["q"], s["pos"], s["freq"], s["axis"], False)]
    seqs, most, kv, group, dim = case["seqs"], s["most"], case["kv"], case["group"], case["dim"]
    # queries [seqs, kv, most * group, dim]; the places past a sequence's new tokens see nothing
    q = torch.zeros(seqs, most, kv, group, dim, device="cuda")
    q[b, i] = s["q"].float().view(-1, kv, group, dim) * s["scale"]
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs, kv, most * group, dim)
    seen = s["lens"].long()[:, None] - new[:, None] + torch.arange(most, device="cuda") + 1
    seen = torch.where(torch.arange(most, device="cuda") < new[:, None], seen, 0).repeat_interleave(group, 1)
    k, v = _gather(s["k"], s["table"]), _gather(s["v"], s["table"])
    at = torch.arange(k.shape[2], device="cuda")
    v = torch.where((at < s["lens"][:, None])[:, None, :, None], v, 0.0)
    x = torch.matmul(q, k.transpose(2, 3).contiguous())
    x = torch.where(at < seen[:, None, :, None], x, -math.inf)
    m = x.amax(3)
    if "prefix" in case:
        if case["xkv"]:
            pk, pv = s["prefix_k"].float(), s["prefix_v"].float()
        else:
            pk, pv = (_gather(p, s["prefix_table"][None])[0, :, :case["prefix"]] for p in (s["k"], s["v"]))
        pq = q.transpose(0, 1).reshape(kv, seqs * most * group, dim)
        px = torch.matmul(pq, pk.transpose(1, 2).contiguous())
        m = torch.maximum(m, px.amax(2).view(kv, seqs, most * group).transpose(0, 1))
    m = torch.where(torch.isinf(m), 0.0, m)
    e = torch.exp(x - m[..., None])
    total, out = e.sum(3), torch.matmul(e, v)
    if "prefix" in case:
        pe = torch.exp(px - m.transpose(0, 1).reshape(kv, -1, 1))
        total = total + pe.sum(2).view(kv, seqs, most * group).transpose(0, 1)
        out = out + torch.matmul(pe, pv).view(kv, seqs, most * group, dim).transpose(0, 1)
    out = torch.where(total[..., None] > 0, out / total[..., None], 0.0)
    out = out.view(seqs, kv, most, group, dim).permute(0, 2, 1, 3, 4)[b, i].reshape(-1, kv * group, dim).to(s["q"].dtype)
    lse = (m + torch.log(total)).view(seqs, kv, most, group).permute(0, 2, 1, 3)[b, i].reshape(-1, kv * group)
    return [out, lse] if case["lse"] else [out]


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ----------------------------------------------------------------------- work --
def _coded(tokens, dim):
    """Bytes of a container of this many tokens in 128-token blocks, all 4-bit, without escapes."""
    return (tokens + 127) // 128 * (8 + dim) + tokens * dim * 3 // 2


def work(case):
    dim = case["dim"]
    if case["op"] == "rope":
        x = case["tokens"] * case["heads"] * dim * 2
        turns = 2 if case["grad"] else 1
        return dict(bytes=turns * (2 * x + 8 * case["axes"] * case["tokens"]),
                    flops=turns * 3 * case["tokens"] * case["heads"] * case["rotated"])
    ns, new = lengths(case), new_tokens(case)
    kv, heads = case["kv"], case["kv"] * case["group"]
    if case["op"] == "append":
        return dict(bytes=sum(new) * (4 * (heads + 2 * kv) * dim + 8 * case["axes"]), flops=3 * sum(new) * (heads + kv) * dim)
    seen = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(ns, new))
    bytes_ = 4 * sum(ns) * kv * dim + sum(new) * heads * (4 * dim + (4 if case["lse"] else 0))
    if "prefix" in case:
        seen += sum(new) * case["prefix"]
        bytes_ += kv * (2 * _coded(case["prefix"], dim) if case["xkv"] else 4 * case["prefix"] * dim)
    return dict(bytes=bytes_, flops=4 * dim * heads * seen)


# ---------------------------------------------------------------------- exact --
def _turned(x, pos, freq, axis, interleaved, back=False):
    """The rotation as a product of complex numbers, in 64 bits."""
    n = freq.numel()
    w = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"),
                    (pos.double()[axis.long()] * freq.double()[:, None]).T)[:, None]
    y = x.detach().double().clone()
    z = torch.complex(y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else torch.complex(y[..., :n], y[..., n:2 * n])
    z = z * (w.conj() if back else w)
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = z.real, z.imag
    else:
        y[..., :n], y[..., n:2 * n] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        at = s["pos"], s["freq"], s["axis"], case["interleaved"]
        return [_turned(s["x"], *at)] + ([_turned(s["dy"], *at, back=True)] if case["grad"] else [])
    pt, kv, group, dim = case["page"], case["kv"], case["group"], case["dim"]
    ns, table = s["lens"].tolist(), s["table"].tolist()
    if case["op"] == "append":
        at = s["pos"], s["freq"], s["axis"], False
        k, v, rows = s["k"].double(), s["v"].double(), _turned(s["new_k"], *at)
        t = 0
        for b, m in enumerate(s["new"]):
            p = torch.arange(ns[b] - m, ns[b], device="cuda")
            page = torch.tensor(table[b], device="cuda")[p // pt]
            k[page, :, p % pt], v[page, :, p % pt] = rows[t:t + m], s["new_v"][t:t + m].double()
            t += m
        return [k, v, _turned(s["q"], *at)]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    p = case.get("prefix", 0)
    for h in range(kv):
        if p and case["xkv"]:
            front = s["prefix_k"][h].double(), s["prefix_v"][h].double()
        elif p:
            front = tuple(x[s["prefix_table"].long(), h].reshape(-1, dim)[:p].double() for x in (s["k"], s["v"]))
        t = 0
        for b, m in enumerate(s["new"]):
            pages = torch.tensor(table[b][:(ns[b] + pt - 1) // pt], device="cuda")
            k, v = (x[pages, h].reshape(-1, dim)[:ns[b]].double() for x in (s["k"], s["v"]))
            if p:
                k, v = torch.cat([front[0], k]), torch.cat([front[1], v])
            q = s["q"][t:t + m, h * group:(h + 1) * group].double().reshape(-1, dim)
            x = (q @ k.T) * s["scale"]
            x = x.view(m, group, -1)
            last = p + ns[b] - m + torch.arange(m, device="cuda") + 1
            x = x.masked_fill(torch.arange(k.shape[0], device="cuda") >= last[:, None, None], -math.inf)
            z = torch.logsumexp(x, 2)
            out[t:t + m, h * group:(h + 1) * group] = torch.exp(x - z[..., None]) @ v
            lse[t:t + m, h * group:(h + 1) * group] = z
            t += m
    return [out, lse] if case["lse"] else [out]
