"""Attention of a batch behind a prefix that it shares (XKV containers or pages), the operators run together, and their
streams, graphs and torch operators; against plain implementations in 64 bits (paged_ref.py)."""
import math

import pytest

torch = pytest.importorskip("torch")

import paged_ref as ref
from conftest import say
from test_gpu_paged import BF, FP, freqs, gen

pytestmark = pytest.mark.gpu


def prefix_kv(g, n_kv, tokens, dim, kind):
    """K and V [n_kv, tokens, dim] whose blocks take the wanted modes."""
    k, v = (torch.randn(n_kv, tokens, dim, generator=g) for _ in range(2))
    if kind == "mixed":  # raw blocks (exponents all over), 4-bit ones, 2-bit ones
        at = torch.arange(tokens) // 50 % 3
        wide = torch.exp2(torch.randint(-30, 3, k.shape, generator=g).float())
        narrow = torch.rand(k.shape, generator=g) * 1.75 + 0.25
        k = torch.where((at == 0)[None, :, None], k * wide, torch.where((at == 1)[None, :, None], narrow, k))
        v = torch.where((at == 2)[None, :, None], v * wide, torch.where((at == 0)[None, :, None], narrow, v))
    if kind == "escapes":
        v = torch.where(torch.rand(v.shape, generator=g) < 0.02, v * 2.0**-20, v)
        k = torch.where(torch.rand(k.shape, generator=g) < 0.02, k * 2.0**-24, k)
    return k.to(BF).cuda(), v.to(BF).cuda()


def encode(ctx, x, block):
    return [ctx.encode(x[h].contiguous(), x.shape[1], x.shape[2], block) for h in range(x.shape[0])]


CASES = [
    # lens, new, page, kv heads, group, dim, prefix tokens, block, kind
    ([40, 3], [1, 1], 16, 2, 7, 64, 300, 128, "plain"),
    ([1], [1], 64, 1, 1, 64, 1, 128, "plain"),
    ([40, 0, 17], [1, 1, 1], 24, 2, 4, 128, 1000, 128, "escapes"),
    ([65, 64], [3, 3], 64, 1, 5, 96, 777, 64, "mixed"),
    ([90, 9], [1, 1], 64, 2, 3, 32, 515, 255, "mixed"),
    ([33], [40], 16, 1, 4, 64, 129, 100, "escapes"),   # fewer tokens than it brings: the prefix alone for the first
    ([20, 30], [1, 1], 16, 1, 2, 256, 400, 128, "escapes"),
    ([20, 30], [2, 2], 16, 2, 2, 192, 333, 7, "plain"),
    ([50] * 40, [1] * 40, 16, 1, 8, 80, 640, 1, "plain"),   # many rows: several row tiles
    ([70] * 3, [60] * 3, 64, 1, 2, 40, 64, 128, "escapes"),
]


@pytest.mark.parametrize("i", range(len(CASES)))
@pytest.mark.parametrize("modes", ["reference", "3bit"])
def test_container_prefix(ctx, i, modes):
    import kvexp_amd as kv

    lens, new, page, n_kv, group, dim, tokens, block, kind = CASES[i]
    g = gen(300 + i)
    c = ref.make_batch(g, lens, new, page, n_kv, dim, BF)
    pk, pv = prefix_kv(g, n_kv, tokens, dim, kind)
    q = (torch.randn(sum(new), n_kv * group, dim, generator=g) * 2).to(BF).cuda()
    cache = kv.PagedCache(ctx, n_kv, dim, c["k"].shape[0], page, BF, k=c["k"], v=c["v"])
    ctx.set_encoder_modes(kv.MODES_REFERENCE | (kv.MODE_3BIT if modes == "3bit" else 0))
    try:
        ks, vs = encode(ctx, pk, block), encode(ctx, pv, block)
    finally:
        ctx.set_encoder_modes(kv.MODES_REFERENCE)
    prefix = ctx.prefix(ks, vs)
    say("prefix", modes, CASES[i])
    batch = kv.Batch(c["table"], c["lens"])
    out, lse = cache.attention(q, batch, prefix=prefix, return_lse=True, check_errors=True)
    both = tuple(x.double().cpu().transpose(0, 1) for x in (pk, pv))
    want = ref.batch_reference(c, lens, new, q, 1 / math.sqrt(dim), both)
    ref.check_attention(out, lse, want, BF, False)
    assert torch.equal(out, cache.attention(q, batch, prefix=prefix))
    prefix.close()
    with pytest.raises(ValueError, match="closed"):
        cache.attention(q, batch, prefix=prefix)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("page,tokens,seqs,new,group,dim", [(16, 333, 2, 1, 4, 64), (24, 1000, 9, 1, 8, 128),
                                                            (64, 64, 3, 2, 2, 256), (1, 70, 1, 1, 3, 32),
                                                            (100, 1, 40, 1, 7, 96)])
def test_page_prefix(ctx, dtype, page, tokens, seqs, new, group, dim):
    import kvexp_amd as kv

    g = gen(page + tokens)
    n_pages = (tokens + page - 1) // page
    lens = [1 + 37 * b % 90 for b in range(seqs)]
    c = ref.make_batch(g, lens, [new] * seqs, page, 2, dim, dtype, spare=n_pages + 1)
    table = c["spare"][:n_pages].int().cuda()
    if tokens % page:
        c["k"][table[-1].long(), :, tokens % page:] = math.nan
        c["v"][table[-1].long(), :, tokens % page:] = math.nan
    q = torch.randn(seqs * new, 2 * group, dim, generator=g).to(dtype).cuda()
    cache = kv.PagedCache(ctx, 2, dim, c["k"].shape[0], page, dtype, k=c["k"], v=c["v"])
    say("page prefix", dtype, page, tokens, seqs, new, group, dim)
    out, lse = cache.attention(q, kv.Batch(c["table"], c["lens"]), prefix=cache.prefix(table, tokens), return_lse=True,
                               check_errors=True)
    both = tuple(ref.tokens_of(c[x], table.tolist(), tokens) for x in ("k", "v"))
    want = ref.batch_reference(c, lens, [new] * seqs, q, 1 / math.sqrt(dim), both)
    ref.check_attention(out, lse, want, dtype, split_p=False)


def test_damaged_prefixes_are_refused(ctx):
    import kvexp_amd as kv

    g = gen(41)
    pk, pv = prefix_kv(g, 1, 300, 64, "escapes")
    k, v = encode(ctx, pk, 128)[0], encode(ctx, pv, 128)[0]

    def copy(e, **kw):
        return kv.Encoded(**{**dict(blob=e.blob.clone(), nbytes=e.nbytes, offsets=e.offsets.clone(),
                                    first=e.first.clone(), seq=e.seq, dim=e.dim, block=e.block), **kw})

    bad = copy(k)
    bad.blob[0] = 1
    with pytest.raises(kv.KvexpHipError, match="unknown xkv block mode"):
        ctx.prefix([bad], [v])
    with pytest.raises(kv.KvexpHipError, match="truncated coded xkv block"):
        ctx.prefix([copy(k, nbytes=k.nbytes - 3)], [v])
    with pytest.raises(kv.KvexpHipError, match="ran out of tokens"):
        ctx.prefix([copy(k, seq=301)], [copy(v, seq=301)])
    shifted = copy(k)
    shifted.first += 1
    with pytest.raises(kv.KvexpHipError, match="index does not match"):
        ctx.prefix([shifted], [v])
    with pytest.raises(ValueError, match="one length"):
        ctx.prefix([k], [copy(v, seq=299)])


def test_generation_loop(ctx):
    """The operators as a serving program runs them: a compressed prefix, prompts appended in one call and attended
    in chunks, then decode steps, each against the whole sequence in 64 bits."""
    import kvexp_amd as kv

    g = gen(42)
    P, page, n_kv, group, dim, steps = 200, 16, 2, 4, 64, 5
    prompts = [30, 7, 65]
    total = [p + steps for p in prompts]
    heads = n_kv * group
    freq = freqs(dim // 2)
    rope = kv.Rope(freq)
    raw_k, raw_v = (torch.randn(P, n_kv, dim, generator=g).to(BF).cuda() for _ in range(2))
    turned = ctx.rope(raw_k, None, rope)
    enc = [[ctx.encode(x[:, h].contiguous(), P, dim) for h in range(n_kv)] for x in (turned, raw_v)]
    prefix = ctx.prefix(*enc)
    need = [(n + page - 1) // page for n in total]
    order = torch.randperm(sum(need) + 2, generator=g)
    table = torch.full((3, max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n].int()
    cache = ctx.paged_cache(n_kv, dim, sum(need) + 2, page)
    cache.k.fill_(math.nan), cache.v.fill_(math.nan)
    table = table.cuda()
    keep = [[torch.zeros(0, n_kv, dim, dtype=torch.double), torch.zeros(0, n_kv, dim, dtype=torch.double)] for _ in prompts]
    lens = [0, 0, 0]
    for step in range(steps + 1):
        new = prompts if step == 0 else [1, 1, 1]
        lens = [a + b for a, b in zip(lens, new)]
        qkv = torch.randn(sum(new), heads + 2 * n_kv, dim, generator=g).to(BF).cuda()
        starts = torch.tensor([0, new[0], new[0] + new[1], sum(new)], dtype=torch.int32).cuda()
        batch = kv.Batch(table, torch.tensor(lens, dtype=torch.int32).cuda(), starts if step == 0 else None,
                         max_new=max(new))
        say("generation", step)
        q = cache.append(qkv[:, heads:heads + n_kv], qkv[:, heads + n_kv:], batch, rope=rope, offset=P,
                         q=qkv[:, :heads])
        out, lse = cache.attention(q, batch, prefix=prefix, return_lse=True, check_errors=True)
        pos = torch.cat([torch.arange(P + n - m, P + n) for n, m in zip(lens, new)])[None]
        ref.check_rotated(q, *ref.rotate(qkv[:, :heads], pos, freq))
        t = 0
        for b, m in enumerate(new):
            rows = ref.tokens_of(cache.k, table[b].tolist(), lens[b])[-m:]
            want, size = ref.rotate(qkv[t:t + m, heads:heads + n_kv], pos[:, t:t + m], freq)
            ref.check_rotated(rows.to(BF), want, size)
            keep[b][0] = torch.cat([keep[b][0], rows])
            keep[b][1] = torch.cat([keep[b][1], qkv[t:t + m, heads + n_kv:].double().cpu()])
            ks = torch.cat([turned.double().cpu(), keep[b][0]])
            vs = torch.cat([raw_v.double().cpu(), keep[b][1]])
            want = ref.attention(q[t:t + m].double().cpu(), ks, vs, [P + lens[b] - m + i + 1 for i in range(m)],
                                 1 / math.sqrt(dim))
            ref.check_attention(out[t:t + m], lse[t:t + m], want, BF, False)
            t += m


def test_graph_replays_follow_lengths_and_tables(ctx):
    """A step captured once (append, attention behind a prefix) and replayed over new tokens, lengths and pages, with
    eager calls and synchronisation between; two graphs of the same cache replayed on two streams."""
    import kvexp_amd as kv

    g = gen(43)
    page, n_kv, group, dim, seqs = 16, 2, 4, 64, 3
    heads = n_kv * group
    pk, pv = prefix_kv(g, n_kv, 500, dim, "escapes")
    prefix = ctx.prefix(encode(ctx, pk, 128), encode(ctx, pv, 128))
    cache = ctx.paged_cache(n_kv, dim, 40, page)
    cache.k.normal_(), cache.v.normal_()
    table = torch.randperm(40, generator=g)[:36].view(seqs, 12).int().cuda()
    lens = torch.tensor([5, 100, 64], dtype=torch.int32).cuda()
    rope = kv.Rope(freqs(32))
    qkv = torch.randn(seqs, heads + 2 * n_kv, dim, generator=g).to(BF).cuda()

    def step(x):
        batch = kv.Batch(table, lens)
        q = cache.append(x[:, heads:heads + n_kv], x[:, heads + n_kv:], batch, rope=rope, offset=500, q=x[:, :heads])
        return cache.attention(q, batch, prefix=prefix), cache.attention(q, batch)

    side = torch.cuda.Stream()
    graphs = []
    static = [qkv.clone(), qkv.clone()]
    for x in static:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(x)
        graphs.append((graph, outs))
    for i in range(4):
        x = torch.randn(qkv.shape, generator=g).to(BF).cuda()
        lens += 1 if i else 0
        table.copy_(table[:, torch.randperm(12, generator=g).cuda()])
        static[0].copy_(x)
        say("replay", i)
        graphs[0][0].replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in graphs[0][1]]
        want = step(x)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        cache.status()
    # the same tokens from both graphs at once, each on its own stream: the appends write the same values
    static[1].copy_(static[0])
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    graphs[0][0].replay()
    with torch.cuda.stream(other):
        graphs[1][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], want))
    assert all(torch.equal(a, b) for a, b in zip(graphs[1][1], want))


def test_other_streams_and_calls_at_once(ctx):
    """Calls queued on a stream of their own, by argument and by torch's current stream, and two calls at once."""
    import kvexp_amd as kv

    g = gen(44)
    lens = [3000, 700]
    c = ref.make_batch(g, lens, [1, 1], 64, 2, 128, BF)
    cache = kv.PagedCache(ctx, 2, 128, c["k"].shape[0], 64, BF, k=c["k"], v=c["v"])
    batch = kv.Batch(c["table"], c["lens"])
    q = [torch.randn(2, 8, 128, generator=g).to(BF).cuda() for _ in range(2)]
    want = [cache.attention(x, batch) for x in q]
    torch.cuda.synchronize()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    a = cache.attention(q[0], batch, stream=s[0])
    with torch.cuda.stream(s[1]):
        b = cache.attention(q[1], batch)
    torch.cuda.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    x = torch.randn(9, 2, 64, generator=g).to(BF).cuda()
    r = kv.Rope(freqs(32))
    y = ctx.rope(x, None, r)
    torch.cuda.synchronize()
    z = ctx.rope(x, None, r, stream=s[0])
    s[0].synchronize()
    assert torch.equal(y, z)


def test_torch_operators(ctx):
    import kvexp_amd as kv
    from kvexp_amd import torch_ops

    g = gen(45)
    lens = [100, 33]
    c = ref.make_batch(g, lens, [1, 1], 16, 2, 64, BF)
    q = torch.randn(2, 8, 64, generator=g).to(BF).cuda()
    k, v = (torch.randn(2, 2, 64, generator=g).to(BF).cuda() for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    mine = kv.PagedCache(ctx, 2, 64, c["k"].shape[0], 16, BF, k=c["k"].clone(), v=c["v"].clone())
    batch = kv.Batch(c["table"], c["lens"])
    freq = freqs(32)
    turned = torch.ops.kvexp.paged_append(c["k"], c["v"], status, k, v, c["table"], c["lens"], None, q, freq)
    assert torch.equal(turned, mine.append(k, v, batch, rope=kv.Rope(freq), q=q))
    for a, b in ((c["k"], mine.k), (c["v"], mine.v)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    out, lse = torch.ops.kvexp.paged_attention(c["k"], c["v"], status, turned, c["table"], c["lens"], None, 0.125)
    want, want_lse = mine.attention(turned, batch, 0.125, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    pk, pv = prefix_kv(g, 2, 150, 64, "plain")
    ks, vs = encode(ctx, pk, 128), encode(ctx, pv, 128)
    h = torch_ops.register_prefix(ks, vs)
    out, lse = torch.ops.kvexp.prefix_attention(c["k"], c["v"], status, turned, c["table"], c["lens"], None, h, 0.125)
    want, want_lse = mine.attention(turned, batch, 0.125, prefix=ctx.prefix(ks, vs), return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    torch_ops.unregister_prefix(h)
    table = c["spare"][:2].int().cuda()
    out, _ = torch.ops.kvexp.paged_attention(c["k"], c["v"], status, turned, c["table"], c["lens"], None, 0.125, 0, 0,
                                             table, 30)
    assert torch.equal(out, mine.attention(turned, batch, 0.125, prefix=mine.prefix(table, 30)))
    assert int(status) == 0
    with pytest.raises(ValueError, match="unknown handle"):
        torch.ops.kvexp.prefix_attention(c["k"], c["v"], status, turned, c["table"], c["lens"], None, h, 0.125)


def test_no_float_is_read_past_the_pools(ctx):
    """Pools that end with the last token of the last page, and far pages: offsets past 32 bits."""
    import kvexp_amd as kv

    g = gen(46)
    page, dim, n_kv = 64, 128, 8
    n = 2**32 // (page * dim * n_kv) + 3  # the last pages start past 2^32 elements
    k = torch.zeros(n, n_kv, page, dim, dtype=BF, device="cuda")
    v = torch.zeros(n, n_kv, page, dim, dtype=BF, device="cuda")
    far = torch.tensor([[n - 1, 0, n - 2]], dtype=torch.int32).cuda()
    lens = [180]
    for p in (n - 1, 0, n - 2):
        k[p] = torch.randn(n_kv, page, dim, generator=g).to(BF)
        v[p] = torch.randn(n_kv, page, dim, generator=g).to(BF)
    cache = kv.PagedCache(ctx, n_kv, dim, n, page, BF, k=k, v=v)
    new_k, new_v = (torch.randn(3, n_kv, dim, generator=g).to(BF).cuda() for _ in range(2))
    batch = kv.Batch(far, torch.tensor(lens, dtype=torch.int32).cuda())
    say("far pages")
    cache.append(new_k, new_v, batch, check_errors=True)
    assert torch.equal(k[n - 2, :, 49:52].transpose(0, 1), new_k)
    for rows, group in ((3, 2), (3, 8)):
        q = torch.randn(rows, n_kv * group, dim, generator=g).to(BF).cuda()
        out, lse = cache.attention(q, batch, return_lse=True, check_errors=True)
        want = ref.batch_reference(dict(k=k, v=v, table=far), lens, [3], q, 1 / math.sqrt(dim))
        ref.check_attention(out, lse, want, BF, rows * group <= 16)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-44])
def test_container_prefix_scales(ctx, scale):
    import kvexp_amd as kv

    g = gen(47)
    lens, tokens, dim = [30, 0], 500, 64
    c = ref.make_batch(g, lens, [1, 1], 16, 2, dim, BF)
    pk, pv = prefix_kv(g, 2, tokens, dim, "escapes")
    prefix = ctx.prefix(encode(ctx, pk, 100), encode(ctx, pv, 100))
    cache = kv.PagedCache(ctx, 2, dim, c["k"].shape[0], 16, BF, k=c["k"], v=c["v"])
    q = torch.randn(2, 6, dim, generator=g).to(BF).cuda()
    say("prefix scale", scale)
    out, lse = cache.attention(q, kv.Batch(c["table"], c["lens"]), scale, prefix=prefix, return_lse=True)
    both = tuple(x.double().cpu().transpose(0, 1) for x in (pk, pv))
    ref.check_attention(out, lse, ref.batch_reference(c, lens, [1, 1], q, scale, both), BF, False)
