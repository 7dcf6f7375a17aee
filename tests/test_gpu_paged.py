"""Rotary positions, appends to a paged cache and attention over its pages
against plain implementations in 64 bits (paged_ref.py, which derives the
bounds)."""
import math

import pytest

torch = pytest.importorskip("torch")

import paged_ref as ref
from conftest import say

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def freqs(n, base=10000.0):
    return (base ** (-torch.arange(n, dtype=torch.float64) / n)).float().cuda()


# ------------------------------------------------------------------- rope --
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,n,axes", [(1, 1, 8, 4, 1), (3, 5, 64, 32, 1), (77, 14, 64, 16, 3),
                                                     (130, 3, 80, 40, 2), (19, 2, 96, 5, 3), (5, 1, 256, 128, 1),
                                                     (2100, 2, 128, 64, 3), (33, 7, 40, 1, 1), (4200, 1, 24, 6, 2)])
def test_rope(ctx, dtype, interleaved, tokens, heads, dim, n, axes):
    import kvexp_amd as kv

    g = gen(tokens + dim + n)
    x = torch.randn(tokens, heads, dim, generator=g).to(dtype).cuda()
    freq = freqs(n)
    axis = None if axes == 1 else torch.randint(0, axes, (n,), generator=g).to(torch.uint8).cuda()
    pos = torch.randint(0, 1 << 20, (axes, tokens), generator=g).cuda()
    say("rope", dtype, interleaved, tokens, heads, dim, n, axes)
    r = kv.Rope(freq, axis, interleaved, scale=1.25)
    y = ctx.rope(x, pos, r)
    want, size = ref.rotate(x, pos, freq, axis, interleaved, 1.25)
    ref.check_rotated(y, want, size, 1.25)
    back = ctx.rope(x, pos.to(torch.int32), r, inverse=True)
    ref.check_rotated(back, *ref.rotate(x, pos, freq, axis, interleaved, 1.25, inverse=True), 1.25)
    inplace = x.clone()
    assert ctx.rope(inplace, pos, r, out=inplace) is inplace
    assert torch.equal(inplace.view(torch.int16), y.view(torch.int16))


def test_rope_strides_positions_and_far_angles(ctx):
    import kvexp_amd as kv

    g = gen(5)
    qkv = torch.randn(50, 24, 64, generator=g).to(BF).cuda()
    freq = freqs(32)
    r = kv.Rope(freq)
    for x in (qkv[:, 3:9], qkv.transpose(0, 1)[:20].transpose(0, 1), qkv[::3], qkv[:, :, 8:48], qkv[:, 2:3, 4:60]):
        rr = kv.Rope(freq[: x.shape[2] // 2].contiguous())
        pos = torch.arange(x.shape[0]).cuda()
        say("rope strides", tuple(x.shape), x.stride())
        y = ctx.rope(x, None, rr)
        assert torch.equal(y, ctx.rope(x, pos, rr)) and torch.equal(y, ctx.rope(x.contiguous(), pos, rr))
        ref.check_rotated(y, *ref.rotate(x, pos[None], rr.inv_freq))
    x = qkv[:8]
    far = torch.tensor([0, 1, -1, 2**24 + 1, 2**31 - 1, -(2**31), 2**31 + 5, 2**33 + 3]).cuda()
    # the angle in 64 bits: pos * freq is off by pos 2^-53 itself, far below the bound
    ref.check_rotated(ctx.rope(x, far, r), *ref.rotate(x, far[None], freq))
    assert ctx.rope(qkv[:0], None, r).shape == (0, 24, 64)


def test_rope_gradient(ctx):
    """Against the formula, and against differences: the rotation is linear, so a difference over a step of 1 from 0
    gives its column (rounded once, as the gradient is)."""
    import kvexp_amd.torch_ops  # noqa: F401

    g = gen(6)
    x = torch.randn(21, 3, 64, generator=g).to(BF).cuda().requires_grad_()
    dy = torch.randn(21, 3, 64, generator=g).to(BF).cuda()
    freq, pos = freqs(24), torch.randint(0, 5000, (1, 21), generator=g).cuda()
    y = torch.ops.kvexp.rope(x, pos, freq)
    (dx,) = torch.autograd.grad(y, x, dy)
    want, size = ref.rotate(dy, pos, freq, inverse=True)
    ref.check_rotated(dx, want, size)
    for ch in (0, 5, 23, 24, 47, 50):
        e = torch.zeros(21, 3, 64, dtype=BF, device="cuda")
        e[:, :, ch] = 1
        col = torch.ops.kvexp.rope(e, pos, freq).double().cpu()
        d = (col * dy.double().cpu()).sum(2)
        # dx is rounded once (2^-8 of it), each of the column's two values once
        tol = 2.0**-8 * d.abs() + 2.0**-8 * (col * dy.double().cpu()).abs().sum(2) * 2 + 1e-6
        assert bool(((dx.double().cpu()[:, :, ch] - d).abs() <= tol).all())


# ----------------------------------------------------------------- append --
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("page", [1, 16, 24, 64, 100])
@pytest.mark.parametrize("dim,n,axes", [(64, 32, 1), (96, 20, 3), (128, 64, 1), (40, 3, 2)])
def test_append(ctx, dtype, page, dim, n, axes):
    import kvexp_amd as kv

    g = gen(page * 1000 + dim)
    new = [1, 0, 7, 30, 3, 2]
    lens = [1, 9, 7, 131, 200, 1]  # the last holds fewer tokens than it brings
    c = ref.make_batch(g, lens, new, page, 2, dim, dtype, unused=5.0)
    total = sum(new)
    qkv = torch.randn(total + 2, 6 + 4, dim, generator=g).to(dtype).cuda()  # two rows behind the last sequence
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    freq = freqs(n)
    axis = None if axes == 1 else (torch.arange(n) % axes).to(torch.uint8).cuda()
    pos = torch.randint(0, 100000, (axes, total + 2), generator=g).cuda()
    cache = kv.PagedCache(ctx, 2, dim, c["k"].shape[0], page, dtype, k=c["k"].clone(), v=c["v"].clone())
    q_out = torch.full_like(q, 7.0)
    batch = kv.Batch(c["table"], c["lens"], c["starts"])
    say("append", dtype, page, dim, n, axes)
    cache.append(k, v, batch, rope=kv.Rope(freq, axis), positions=pos, q=q, q_out=q_out, check_errors=True)
    want_k, size = ref.rotate(k, pos, freq, axis)
    expect_k, expect_v = c["k"].clone(), c["v"].clone()
    got_k = torch.zeros(total, 2, dim, dtype=dtype)
    written, t = [], 0
    for b, m in enumerate(new):
        for i in range(m):
            at = lens[b] - m + i
            if at >= 0:
                p, o = int(c["table"][b, at // page]), at % page
                got_k[t] = cache.k[p, :, o].cpu()
                expect_k[p, :, o], expect_v[p, :, o] = cache.k[p, :, o], v[t]
                written.append(t)
            t += 1
    ref.check_rotated(got_k[written], want_k[written], size[written])
    # every other place of the pools as it was
    assert torch.equal(cache.k.view(torch.int16), expect_k.view(torch.int16))
    assert torch.equal(cache.v.view(torch.int16), expect_v.view(torch.int16))
    ref.check_rotated(q_out[:total], *[x[:total] for x in ref.rotate(q, pos, freq, axis)])
    assert bool((q_out[total:] == 7).all())


def test_append_places_offsets_and_layouts(ctx):
    """Positions from the places (plus an offset), no rotation, a pool with tokens ahead of heads, uniform counts."""
    import kvexp_amd as kv

    g = gen(9)
    lens, new, page, dim = [5, 70, 33], [2, 2, 2], 16, 64
    c = ref.make_batch(g, lens, new, page, 3, dim, BF, unused=0.0)
    k, v = (torch.randn(6, 3, dim, generator=g).to(BF).cuda() for _ in range(2))
    batch = kv.Batch(c["table"], c["lens"])
    freq = freqs(32)
    n = c["k"].shape[0]
    caches = []
    for layout in range(2):
        pools = []
        for _ in range(2):
            x = torch.zeros(n, page, 3, dim, dtype=BF, device="cuda") if layout else \
                torch.zeros(n, 3, page, dim, dtype=BF, device="cuda")
            pools.append(x.transpose(1, 2) if layout else x)
        cache = kv.PagedCache(ctx, 3, dim, n, page, BF, k=pools[0], v=pools[1])
        say("append layout", layout)
        assert cache.append(k, v, batch, rope=kv.Rope(freq), offset=1000, check_errors=True) is None
        caches.append(cache)
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    pos = torch.tensor([[1000 + n - 2 + i for n in lens for i in range(2)]])
    want, size = ref.rotate(k, pos, freq)
    got = torch.stack([caches[0].k[int(c["table"][b, (lens[b] - 2 + i) // page]), :, (lens[b] - 2 + i) % page]
                       for b in range(3) for i in range(2)])
    ref.check_rotated(got, want, size)
    plain = kv.PagedCache(ctx, 3, dim, n, page, BF, k=torch.zeros_like(caches[0].k), v=torch.zeros_like(caches[0].v))
    plain.append(k, v, batch, check_errors=True)
    got = torch.stack([plain.k[int(c["table"][b, (lens[b] - 2 + i) // page]), :, (lens[b] - 2 + i) % page]
                       for b in range(3) for i in range(2)])
    assert torch.equal(got, k) and torch.equal(plain.v, caches[0].v)


def test_bad_pages_and_lengths_are_reported(ctx):
    import kvexp_amd as kv

    g = gen(10)
    lens, new = [40, 40], [1, 1]
    c = ref.make_batch(g, lens, new, 16, 1, 64, BF, unused=0.0)
    cache = kv.PagedCache(ctx, 1, 64, c["k"].shape[0], 16, BF, k=c["k"], v=c["v"])
    k = torch.randn(2, 1, 64, generator=g).to(BF).cuda()
    q = torch.randn(2, 4, 64, generator=g).to(BF).cuda()
    good = cache.attention(q, kv.Batch(c["table"], c["lens"]), check_errors=True)
    before = cache.k.clone()
    for page in (-1, c["k"].shape[0], 2**31 - 1):
        table = c["table"].clone()
        table[1, 2] = page
        batch = kv.Batch(table, c["lens"])
        say("bad page", page)
        out = cache.attention(q, batch)
        with pytest.raises(kv.KvexpHipError, match="outside the pool"):
            cache.status()
        cache.status()  # cleared
        assert torch.equal(out[0], good[0])
        other = kv.PagedCache(ctx, 1, 64, c["k"].shape[0], 16, BF, k=before.clone(), v=c["v"].clone())
        with pytest.raises(kv.KvexpHipError, match="outside the pool"):
            other.append(k, k, batch, check_errors=True)
        at = int(c["table"][0, 2]), 0, 39 % 16
        assert torch.equal(other.k[at], k[0, 0])  # the good sequence's token, and nothing else
        other.k[at] = before[at]
        assert torch.equal(other.k, before)
    long = c["lens"].clone()
    long[1] = 16 * c["table"].shape[1] + 1
    table = c["table"].clamp(min=0)
    with pytest.raises(kv.KvexpHipError, match="past its page table"):
        cache.attention(q, kv.Batch(table, long), check_errors=True)
    with pytest.raises(kv.KvexpHipError, match="past its page table"):
        other.append(k, k, kv.Batch(table, long), check_errors=True)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    cache.attention(q, kv.Batch(c["table"], c["lens"], starts, max_new=1), check_errors=True)
    wide = torch.tensor([0, 0, 2], dtype=torch.int32).cuda()
    with pytest.raises(kv.KvexpHipError, match="max_new"):
        cache.attention(q, kv.Batch(c["table"], c["lens"], wide, max_new=1), check_errors=True)


# -------------------------------------------------------------- attention --
CASES = [
    # lens, new tokens, page, kv heads, group, dim
    ([1], [1], 16, 1, 1, 64),
    ([37], [1], 16, 2, 7, 64),
    ([64, 1, 0, 33], [1, 1, 1, 1], 64, 2, 7, 64),
    ([513, 1200, 31], [1, 1, 1], 24, 2, 4, 96),
    ([4097, 64, 300, 1023], [1, 1, 1, 1], 128, 1, 8, 128),
    ([700, 65], [1, 1], 1, 2, 3, 32),
    ([260, 97], [1, 1], 100, 1, 16, 256),
    ([300, 2], [1, 1], 16, 3, 5, 80),
    ([190], [1], 64, 1, 2, 8),
    ([190, 77], [1, 1], 64, 2, 2, 200),
    ([511, 129], [4, 2], 64, 2, 3, 64),    # few rows with a causal end
    ([300, 129, 6], [5, 0, 6], 24, 2, 4, 96),   # many rows, ragged, one without new tokens
    ([700, 40, 333], [70, 40, 1], 64, 2, 4, 128),
    ([150], [150], 16, 1, 3, 64),          # a whole prompt
    ([300, 9], [40, 12], 64, 1, 2, 192),   # the second holds fewer tokens than it brings
    ([333, 80], [33, 17], 16, 1, 8, 256),
    ([100, 65], [17, 33], 1, 1, 1, 24),
    ([600], [9], 100, 2, 11, 112),
]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention(ctx, dtype, i):
    import kvexp_amd as kv

    lens, new, page, n_kv, group, dim = CASES[i]
    g = gen(100 + i)
    c = ref.make_batch(g, lens, new, page, n_kv, dim, dtype)
    q = (torch.randn(sum(new), n_kv * group, dim, generator=g) * 3).to(dtype).cuda()
    cache = kv.PagedCache(ctx, n_kv, dim, c["k"].shape[0], page, dtype, k=c["k"], v=c["v"])
    same = len(set(new)) == 1
    batch = kv.Batch(c["table"], c["lens"], None if same else c["starts"], max_new=max(new))
    say("attention", dtype, CASES[i])
    out, lse = cache.attention(q, batch, return_lse=True, check_errors=True)
    want = ref.batch_reference(c, lens, new, q, 1 / math.sqrt(dim))
    ref.check_attention(out, lse, want, dtype, split_p=max(new) * group <= 16)
    assert torch.equal(out, cache.attention(q, batch))  # the same bits every time
    again = cache.attention(q, kv.Batch(c["table"], c["lens"], c["starts"]))  # (max_new unknown: another cut)
    ref.check_attention(again, None, want, dtype, split_p=sum(new) * group <= 16)


@pytest.mark.parametrize("new,group", [(1, 4), (3, 4), (20, 4)])
def test_masked_places_stay_out(ctx, new, group):
    """Infinities and NaN in places that a row does not see: behind the length, in other sequences' pages, and (rows
    of several new tokens) in the later new tokens themselves."""
    import kvexp_amd as kv

    g = gen(new)
    lens, page, dim = [77, 300], 16, 64
    c = ref.make_batch(g, lens, [new] * 2, page, 1, dim, BF, unused=math.inf)
    q = torch.randn(2 * new, group, dim, generator=g).to(BF).cuda()
    cache = kv.PagedCache(ctx, 1, dim, c["k"].shape[0], page, BF, k=c["k"], v=c["v"])
    batch = kv.Batch(c["table"], c["lens"])
    if new > 1:
        for b, value in ((0, math.nan), (1, -math.inf)):  # the last token's key and value
            at = lens[b] - 1
            c["k"][int(c["table"][b, at // page]), :, at % page] = value
            c["v"][int(c["table"][b, at // page]), :, at % page] = value
    say("masked", new)
    out, lse = cache.attention(q, batch, return_lse=True, check_errors=True)
    rows = [b * new + i for b in range(2) for i in range(new - 1 if new > 1 else 1)]
    want = ref.batch_reference(c, lens, [new] * 2, q, 1 / 8)
    want = [w[rows] for w in want]
    ref.check_attention(out[rows], lse[rows], want, BF, split_p=new * group <= 16)
    if new > 1:
        assert bool(torch.isnan(out[new - 1]).all()) and not bool(torch.isfinite(out[-1]).all())


def test_many_splits_and_bounds(ctx):
    """Any max_len gives the same attention; splits joined by the merge."""
    import kvexp_amd as kv

    g = gen(77)
    lens, page, dim = [9000, 17, 4500], 64, 64
    c = ref.make_batch(g, lens, [1] * 3, page, 2, dim, BF)
    q = torch.randn(3, 8, dim, generator=g).to(BF).cuda()
    cache = kv.PagedCache(ctx, 2, dim, c["k"].shape[0], page, BF, k=c["k"], v=c["v"])
    want = ref.batch_reference(c, lens, [1] * 3, q, 0.2)
    for max_len in (None, 1, 100, 5000, 9000, 2**31 - 1):
        say("max_len", max_len)
        out, lse = cache.attention(q, kv.Batch(c["table"], c["lens"], max_len=max_len), 0.2, return_lse=True,
                                   check_errors=True)
        ref.check_attention(out, lse, want, BF, True)


def test_strided_queries_outputs_and_empty_calls(ctx):
    import kvexp_amd as kv

    g = gen(78)
    lens, page, dim = [200, 90], 64, 64
    c = ref.make_batch(g, lens, [3, 3], page, 2, dim, BF)
    cache = kv.PagedCache(ctx, 2, dim, c["k"].shape[0], page, BF, k=c["k"], v=c["v"])
    batch = kv.Batch(c["table"], c["lens"])
    qkv = torch.randn(6, 12, dim, generator=g).to(BF).cuda()
    want, lse = cache.attention(qkv[:, :8].contiguous(), batch, return_lse=True)
    big = torch.full((8, 6, dim), 3.0, dtype=BF, device="cuda").transpose(0, 1)
    lse2 = torch.zeros_like(lse)
    assert cache.attention(qkv[:, :8], batch, out=big, lse=lse2) is big
    assert torch.equal(big, want) and torch.equal(lse, lse2)
    odd = torch.randn(6, 8, dim + 1, generator=g).to(BF).cuda()[:, :, 1:]
    assert torch.equal(cache.attention(odd, batch), cache.attention(odd.contiguous(), batch))
    none = kv.Batch(c["table"][:0], c["lens"][:0])
    assert cache.attention(qkv[:0, :8], none).shape == (0, 8, dim)
    assert cache.attention(qkv[:0, :8], batch).shape == (0, 8, dim)
    assert cache.append(qkv[:0, 8:10], qkv[:0, 10:], batch, q=qkv[:0, :8], rope=kv.Rope(freqs(32))).shape == (0, 8, dim)


def test_rows_behind_the_last_sequence(ctx):
    """A padded batch: rows behind starts[-1] and sequences without new tokens leave the outputs alone."""
    import kvexp_amd as kv

    g = gen(79)
    lens, new, page, dim = [50, 20, 0], [2, 1, 0], 16, 64
    c = ref.make_batch(g, lens, new, page, 1, dim, BF)
    q = torch.randn(6, 4, dim, generator=g).to(BF).cuda()
    cache = kv.PagedCache(ctx, 1, dim, c["k"].shape[0], page, BF, k=c["k"], v=c["v"])
    out = torch.full_like(q, 9.0)
    cache.attention(q, kv.Batch(c["table"], c["lens"], c["starts"]), out=out, check_errors=True)
    assert bool((out[3:] == 9).all())
    ref.check_attention(out[:3], None, ref.batch_reference(c, lens, new, q[:3], 1 / 8), BF, False)


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.2, 1e-30, 1e-44])
@pytest.mark.parametrize("new,group,dim", [(1, 4, 64), (5, 4, 64), (20, 4, 64), (70, 4, 128), (9, 4, 256)])
def test_scales(ctx, scale, new, group, dim):
    """Scales of 0, below float's normal numbers and below 0, over masked places."""
    import kvexp_amd as kv

    g = gen(new + dim)
    lens, page = [77, 300], 16
    c = ref.make_batch(g, lens, [new] * 2, page, 1, dim, BF)
    q = torch.randn(2 * new, group, dim, generator=g).to(BF).cuda()
    cache = kv.PagedCache(ctx, 1, dim, c["k"].shape[0], page, BF, k=c["k"], v=c["v"])
    say("scale", scale, new, group, dim)
    out, lse = cache.attention(q, kv.Batch(c["table"], c["lens"]), scale, return_lse=True, check_errors=True)
    ref.check_attention(out, lse, ref.batch_reference(c, lens, [new] * 2, q, scale), BF, split_p=new * group <= 16)


@pytest.mark.parametrize("seqs", [64, 65, 130, 300])
def test_many_ragged_sequences(ctx, seqs):
    """Counts of sequences about the merge's 64 starts at a time, some without new tokens, over several splits."""
    import kvexp_amd as kv

    g = gen(seqs)
    new = torch.randint(0, 3, (seqs,), generator=g).tolist()
    lens = [(37 * b) % 90 + n for b, n in enumerate(new)]
    lens[seqs // 2] = 2500
    new[seqs // 2] = 2
    page, dim = 64, 32
    c = ref.make_batch(g, lens, new, page, 1, dim, BF)
    q = torch.randn(sum(new) + 3, 2, dim, generator=g).to(BF).cuda()
    cache = kv.PagedCache(ctx, 1, dim, c["k"].shape[0], page, BF, k=c["k"], v=c["v"])
    want = ref.batch_reference(c, lens, new, q[:-3], 0.3)
    for max_new in (2, None):
        out = torch.full_like(q, 9.0)
        say("ragged", seqs, max_new)
        cache.attention(q, kv.Batch(c["table"], c["lens"], c["starts"], max_new), 0.3, out=out, check_errors=True)
        ref.check_attention(out[:-3], None, want, BF, False)
        assert bool((out[-3:] == 9).all())


def test_outputs_whose_rows_overlap_are_refused(ctx):
    import kvexp_amd as kv

    x = torch.randn(3, 4, 64).to(BF).cuda()
    with pytest.raises(ValueError, match="on one another"):
        ctx.rope(x, None, kv.Rope(freqs(32)), out=torch.zeros(1, 4, 64, dtype=BF, device="cuda").expand(3, 4, 64))
    with pytest.raises(ValueError, match="on one another"):
        ctx.rope(x, None, kv.Rope(freqs(32)), out=torch.zeros(3, 1, 64, dtype=BF, device="cuda").expand(3, 4, 64))


def test_rope_traced_and_captured(ctx):
    """Forward and gradient through a trace of both, twice differentiated, and captured into a graph and replayed."""
    import kvexp_amd.torch_ops  # noqa: F401

    g = gen(8)
    x = torch.randn(33, 3, 64, generator=g).to(BF).cuda().requires_grad_()
    dy = torch.randn(33, 3, 64, generator=g).to(BF).cuda().requires_grad_()
    freq, pos = freqs(32), torch.randint(0, 5000, (33,), generator=g).cuda()

    def both(x, dy):
        y = torch.ops.kvexp.rope(x, pos, freq)
        return y, torch.autograd.grad(y, x, dy, create_graph=True)[0]

    y, dx = both(x, dy)
    (ddy,) = torch.autograd.grad(dx, dy, x.detach())  # the gradient of the gradient's is the rotation
    assert torch.equal(ddy, y.detach())
    y, dx = y.detach(), dx.detach()
    say("trace")
    fn = torch.compile(lambda x: torch.ops.kvexp.rope(x, pos, freq) * 2, backend="aot_eager", fullgraph=True)
    z = fn(x)
    assert torch.equal(z, 2 * y)
    assert torch.equal(torch.autograd.grad(z, x, dy.detach() / 2)[0], dx)

    say("capture")
    xs, ds = x.detach().clone().requires_grad_(), dy.detach().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(torch.ops.kvexp.rope(xs, pos, freq), xs, ds)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.ops.kvexp.rope(xs, pos, freq)
        (grad,) = torch.autograd.grad(out, xs, ds)
    for i in range(3):
        with torch.no_grad():
            xs.copy_(torch.randn(33, 3, 64, generator=g)), ds.copy_(torch.randn(33, 3, 64, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        e = xs.detach().clone().requires_grad_()
        want = torch.ops.kvexp.rope(e, pos, freq)
        assert torch.equal(out, want) and torch.equal(grad, torch.autograd.grad(want, e, ds)[0])
        torch.cuda.synchronize()


@pytest.mark.parametrize("new,longest,dim", [(1, 40, 64), (1, 3000, 64), (6, 700, 128), (70, 80, 64), (70, 3000, 128)])
def test_outputs_over_the_queries(ctx, new, longest, dim):
    """out may be q: one split and several, few rows and many."""
    import kvexp_amd as kv

    g = gen(new + longest)
    lens, page = [longest, 75], 64
    c = ref.make_batch(g, lens, [new] * 2, page, 2, dim, BF)
    q = torch.randn(2 * new, 8, dim, generator=g).to(BF).cuda()
    cache = kv.PagedCache(ctx, 2, dim, c["k"].shape[0], page, BF, k=c["k"], v=c["v"])
    batch = kv.Batch(c["table"], c["lens"])
    say("out over q", new, longest, dim)
    want = cache.attention(q, batch)
    assert cache.attention(q, batch, out=q) is q and torch.equal(q, want)


def test_tables_of_other_layouts(ctx):
    """A table in columns, one that every sequence shares by a stride of 0, and a slice of a wider one."""
    import kvexp_amd as kv

    g = gen(90)
    lens, page, dim = [150, 90, 33], 64, 64
    c = ref.make_batch(g, lens, [1] * 3, page, 1, dim, BF)
    q = torch.randn(3, 4, dim, generator=g).to(BF).cuda()
    cache = kv.PagedCache(ctx, 1, dim, c["k"].shape[0], page, BF, k=c["k"], v=c["v"])
    want = cache.attention(q, kv.Batch(c["table"], c["lens"]))
    wide = torch.full((3, 20), -1, dtype=torch.int32).cuda()
    wide[:, 5:5 + c["table"].shape[1]] = c["table"]
    for t in (c["table"].t().contiguous().t(), wide[:, 5:5 + c["table"].shape[1]]):
        assert torch.equal(want, cache.attention(q, kv.Batch(t, c["lens"])))
    same = c["table"][:1].expand(3, -1)
    lens = torch.tensor([150, 90, 33], dtype=torch.int32).cuda()
    assert torch.equal(cache.attention(q, kv.Batch(same, lens)), cache.attention(q, kv.Batch(same.contiguous(), lens)))
