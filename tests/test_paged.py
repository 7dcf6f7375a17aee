"""CPU checks of the paged cache: what its C entries and its Python calls refuse (argument checks run before a device
is touched), the workspace's size, and shape inference of its torch operators."""
import ctypes as C
import math
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")
kv = pytest.importorskip("kvexp_amd")

from kvexp_amd import paged

BF, FP = torch.bfloat16, torch.float16
PTR = 1 << 20  # an aligned address that nothing reads


def pages(**kw):
    d = dict(k=PTR, v=PTR, k_page=8192, k_head=4096, k_token=64, v_page=8192, v_head=4096, v_token=64, dtype=0,
             n_pages=10, page_tokens=64, n_heads=2, dim=64)
    return paged._Pages(**{**d, **kw})


def batch(**kw):
    d = dict(table=PTR, lens=PTR, starts=None, table_stride=5, table_width=5, n_seqs=3, n_tokens=3)
    return paged._Batch(**{**d, **kw})


def rows(**kw):
    return paged._Rows(**{**dict(data=PTR, token=256, head=64), **kw})


def rope(**kw):
    return paged._Rope(**{**dict(inv_freq=PTR, axes=None, n_freq=32, n_axes=1, interleaved=0, scale=1.0), **kw})


def positions(**kw):
    return paged._Positions(**{**dict(data=PTR, axis_stride=0, offset=0, wide=0), **kw})


def refused(rc, match):
    assert rc != 0
    msg = kv.lib().kvexp_hip_last_error().decode()
    assert match in msg, msg
    return rc


@pytest.mark.parametrize("change,match", [
    (dict(rope=None), "without frequencies"),
    (dict(rope=rope(inv_freq=None)), "without frequencies"),
    (dict(rope=rope(n_freq=0)), "without frequencies"),
    (dict(rope=rope(n_freq=33)), "more rotated channels"),
    (dict(rope=rope(n_freq=2**30 + 1)), "more rotated channels"),
    (dict(rope=rope(n_axes=0)), "without axes"),
    (dict(positions=positions(data=PTR + 2)), "unaligned positions"),
    (dict(positions=positions(data=PTR + 4, wide=1)), "unaligned positions"),
    (dict(rope=rope(n_axes=3), positions=positions(axis_stride=4)), "axes of the positions overlap"),
    (dict(x=None), "null x"),
    (dict(x=rows(data=None)), "null x"),
    (dict(x=rows(data=PTR + 8)), "16-byte aligned"),
    (dict(x=rows(token=100)), "multiples of 8"),
    (dict(out=rows(head=12)), "multiples of 8"),
    (dict(out=None), "null out"),
    (dict(dim=60), "multiple of 8"),
    (dict(dim=264), "at most 256"),
    (dict(dim=0), "multiple of 8"),
    (dict(dtype=2), "BF16 or FP16"),
    (dict(n=-1), "empty rows"),
    (dict(heads=0), "empty rows"),
    (dict(n=2**27 + 1), "more tokens or heads"),
    (dict(heads=2**20 + 1), "more tokens or heads"),
    (dict(), "null context"),
])
def test_rope_entry_refuses(change, match):
    a = dict(rope=rope(), positions=positions(), x=rows(), out=rows(), n=5, heads=4, dim=64, dtype=0)
    a.update(change)
    refused(kv.lib().kvexp_hip_rope_rows(None, a["rope"], a["positions"], a["x"], a["out"], a["n"], a["heads"], a["dim"],
                                         a["dtype"], 0, None), match)


PAGES_AND_BATCHES = [
    (dict(pages=None), "null pages"),
    (dict(pages=pages(k=None)), "null pages"),
    (dict(pages=pages(dtype=7)), "BF16 or FP16"),
    (dict(pages=pages(dim=12)), "multiple of 8"),
    (dict(pages=pages(n_pages=0)), "empty pages"),
    (dict(pages=pages(page_tokens=0)), "empty pages"),
    (dict(pages=pages(v_token=65)), "strides of pages"),
    (dict(pages=pages(v=PTR + 8)), "16-byte aligned"),
    (dict(batch=None), "null batch"),
    (dict(batch=batch(n_seqs=-1)), "negative size"),
    (dict(batch=batch(n_seqs=0)), "tokens of no sequence"),
    (dict(batch=batch(lens=None)), "null table or lens"),
    (dict(batch=batch(table=None)), "null table or lens"),
    (dict(batch=batch(table_stride=4)), "overlap"),
    (dict(batch=batch(table_width=2**25, table_stride=2**25)), "2^30 tokens"),
    (dict(batch=batch(n_tokens=4)), "n_tokens / n_seqs"),
    (dict(batch=batch(n_tokens=6, max_new=1)), "max_new below"),
]


@pytest.mark.parametrize("change,match", PAGES_AND_BATCHES + [
    (dict(q=rows()), "q and q_out go together"),
    (dict(q=rows(), q_out=rows(), rope=None), "queries without a rotation"),
    (dict(q=rows(), q_out=rows(), heads=0), "no query heads"),
    (dict(q=rows(token=4), q_out=rows()), "q must be"),
    (dict(q=rows(), q_out=rows(data=PTR + 2)), "q_out must be"),
    (dict(status=None), "null status"),
    (dict(k=None), "null k"),
    (dict(v=rows(head=4)), "v must be"),
    (dict(q=rows(), q_out=rows(), heads=2**30), "more tokens or heads"),
    (dict(), "null context"),
])
def test_append_entry_refuses(change, match):
    a = dict(pages=pages(), batch=batch(), k=rows(), v=rows(), rope=rope(), positions=None, q=None, q_out=None, heads=4,
             status=PTR)
    a.update(change)
    refused(kv.lib().kvexp_hip_paged_append(None, a["pages"], a["batch"], a["k"], a["v"], a["rope"], a["positions"],
                                            a["q"], a["q_out"], a["heads"], a["status"], None), match)


@pytest.mark.parametrize("change,match", PAGES_AND_BATCHES + [
    (dict(heads=0), "multiple of the cache's heads"),
    (dict(heads=3), "multiple of the cache's heads"),
    (dict(scale=math.nan), "not finite"),
    (dict(scale=-math.inf), "not finite"),
    (dict(scale=3e38), "past float's range"),
    (dict(status=None), "null status"),
    (dict(q=rows(token=12)), "q must be"),
    (dict(out=None), "null out"),
    (dict(shared=paged._Shared(None, None, 3, 100)), "containers or pages"),
    (dict(shared=paged._Shared(None, PTR, 3, 0)), "empty shared prefix"),
    (dict(shared=paged._Shared(None, PTR, 3, 193)), "shorter than its tokens"),
    (dict(shared=paged._Shared(None, PTR, 2**25, 2**30 + 1)), "2^30 tokens"),
    (dict(), "null context"),
])
def test_attention_entry_refuses(change, match):
    L = kv.lib()
    a = dict(pages=pages(), batch=batch(), shared=None, q=rows(), heads=4, scale=0.125, out=rows(), status=PTR)
    a.update(change)
    refused(L.kvexp_hip_paged_attention(None, a["pages"], a["batch"], a["shared"], a["q"], a["heads"], a["scale"],
                                        a["out"], None, None, 0, a["status"], None), match)
    if not set(change) & {"scale", "status", "q", "out"}:
        assert L.kvexp_hip_paged_attention_workspace(None, a["pages"], a["batch"], a["shared"], a["heads"]) == -1


def test_empty_calls_need_nothing():
    L = kv.lib()
    none = batch(n_tokens=0, lens=None, table=None, table_width=0)
    assert L.kvexp_hip_paged_attention_workspace(None, pages(), none, None, 4) == 0
    assert L.kvexp_hip_paged_attention(None, pages(), none, None, None, 4, 0.1, None, None, None, 0, PTR, None) == 0
    assert L.kvexp_hip_paged_append(None, pages(), none, None, None, None, None, None, None, 0, PTR, None) == 0
    assert L.kvexp_hip_rope_rows(None, rope(), None, None, None, 0, 4, 64, 0, 0, None) == 0


def test_prefix_entry_refuses():
    L, out = kv.lib(), C.c_void_p()
    head = kv._Head()
    refused(L.kvexp_hip_prefix_create(None, None, 1, 64, None, C.byref(out)), "bad argument")
    refused(L.kvexp_hip_prefix_create(None, None, 1, 64, None, None), "null output")
    refused(L.kvexp_hip_prefix_create(None, head, 1, 60, None, C.byref(out)), "multiple of 8")
    refused(L.kvexp_hip_prefix_create(None, head, 1, 64, None, C.byref(out)), "empty shared prefix")
    head.seq = 5
    refused(L.kvexp_hip_prefix_create(None, head, 1, 64, None, C.byref(out)), "block indexes")
    head.seq = 2**30 + 1
    refused(L.kvexp_hip_prefix_create(None, head, 1, 64, None, C.byref(out)), "2^30 tokens")
    assert L.kvexp_hip_prefix_destroy(None) == 0
    refused(L.kvexp_hip_paged_status(None, PTR, None), "null argument")


# ----------------------------------------------------------------- Python --
CTX = SimpleNamespace(device=0, h=None)


def test_rope_refuses():
    x = torch.zeros(3, 2, 64, dtype=BF)
    f = torch.zeros(32)
    for bad, match in ((torch.zeros(3, 2, 64), "bfloat16 or float16"), (x[0], "head_dim"), (x[:, :, :60], "multiple of 8"),
                       (torch.zeros(3, 2, 264, dtype=FP), "at most 256"), (x, "must be on cuda:0")):
        with pytest.raises(ValueError, match=match):
            paged.rope(CTX, bad, None, kv.Rope(f))
    with pytest.raises(ValueError, match="must be torch.bfloat16"):
        paged.rope(CTX, x, None, kv.Rope(f), out=x.half())
    with pytest.raises(ValueError, match=r"must be \[3, 2, 64\]"):
        paged.rope(CTX, x, None, kv.Rope(f), out=x[:2])
    for args, match in (((f.double(),), "float32"), ((f[:0],), "float32"), ((f[None],), "float32"),
                        ((f, f.int()), "uint8"), ((f, f[:3].to(torch.uint8)), "uint8"),
                        ((f, None, False, math.inf), "not finite")):
        with pytest.raises(ValueError, match=match):
            kv.Rope(*args)


def test_batches_refuse():
    t, n = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for args, match in (((t.long(), n), "table must be int32"), ((t[0], n), "2 dimensions"), ((t, n.long()), "lens must"),
                        ((t, n[:2]), "one row per sequence"), ((t, n, n), "one more"), ((t, n, n.float()), "starts must")):
        with pytest.raises(ValueError, match=match):
            kv.Batch(*args)


def test_caches_refuse():
    k = torch.zeros(5, 2, 16, 64, dtype=BF)
    for args, kw, match in (((2, 60, 5), {}, "multiple of 8"), ((0, 64, 5), {}, "empty pages"),
                            ((2, 64, 5, 16, torch.float32), {}, "bfloat16 or float16"),
                            ((2, 64, 5, 16, BF), dict(k=k), "go together"),
                            ((2, 64, 5, 16, FP), dict(k=k, v=k), "must be torch.float16"),
                            ((2, 64, 4, 16, BF), dict(k=k, v=k), "must be"),
                            ((2, 64, 5, 16, BF), dict(k=k, v=k.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
                            ((2, 64, 5, 16, BF), dict(k=k, v=k), "on cuda:0"),
                            ((2, 64, 5, 16, BF), dict(status=torch.zeros(2, dtype=torch.int32)), "one int32 word")):
        with pytest.raises(ValueError, match=match):
            kv.PagedCache(CTX, *args, **kw)


def test_what_was_checked_stays():
    """Tensors that a call reads cannot be exchanged for others that nothing has checked."""
    b = kv.Batch(torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    r = kv.Rope(torch.zeros(32), torch.zeros(32, dtype=torch.uint8))
    for o, names in ((b, ("table", "lens", "starts", "n_seqs")), (r, ("inv_freq", "axes"))):
        for n in names:
            with pytest.raises(AttributeError):
                setattr(o, n, getattr(o, n))
    for n in ("k", "v", "status_word"):
        with pytest.raises(AttributeError):
            setattr(object.__new__(kv.PagedCache), n, None)


@pytest.fixture
def cache():
    c = object.__new__(kv.PagedCache)  # (no device to hold its pages)
    c.ctx, c.dtype, c.n_pages, c.n_heads, c.page_tokens, c.dim = CTX, BF, 5, 2, 16, 64
    return c


def test_calls_refuse(cache):
    t, n = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    b = kv.Batch(t, n)
    k, q = torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, 8, 64, dtype=BF)
    r = kv.Rope(torch.zeros(32))
    for args, kw, match in (((k[0], k, b), {}, "k must be"), ((k, k[:2], b), {}, "v must be"), ((k.half(), k, b), {}, "k must be"),
                            ((k, k[:, :1], b), {}, "v must be"), ((k, k, b), dict(q=q), "queries without a rotation"),
                            ((k, k, b, r), dict(q=q[:2]), "q must be"), ((k, k, b, r), dict(q_out=q), "go together"),
                            ((k, k, b, r), dict(q=q, q_out=q[:, :4]), "q_out must be"), ((k, k, b, r), {}, "on cuda:0"),
                            ((torch.zeros((), dtype=BF), k, b), {}, "k must be")):
        with pytest.raises(ValueError, match=match):
            cache.append(*args, **kw)
    lse = torch.zeros(3, 8)
    for args, kw, match in (((q[:, :7], b), {}, "7 query heads over 2"), ((q[:, :0], b), {}, "0 query heads"),
                            ((q[..., :32], b), {}, "q must be"), ((q.half(), b), {}, "q must be"),
                            ((q, b), dict(out=q.half()), "out must be"), ((q, b), dict(out=q[:2]), "out must be"),
                            ((q, b), dict(lse=lse.double()), "lse must be"), ((q, b), dict(lse=lse[:, :4]), "lse must be"),
                            ((q, b), dict(lse=torch.zeros(8, 3).t()), "lse must be"),
                            ((q, b, math.nan), {}, "not finite"), ((q, b), {}, "on cuda:0")):
        with pytest.raises(ValueError, match=match):
            cache.attention(*args, **kw)
    for table, seq, match in ((t, 5, r"int32 \[pages\]"), (t[0].long(), 5, r"int32 \[pages\]"), (t[0], 0, "0 tokens"),
                              (t[0], 65, "65 tokens in 4 pages")):
        with pytest.raises(ValueError, match=match):
            cache.prefix(table, seq)
    with pytest.raises(ValueError, match="one K and one V"):
        kv.Prefix(CTX, [], [])


# -------------------------------------------------------- torch operators --
def test_operators_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import kvexp_amd.torch_ops  # noqa: F401

    ops = torch.ops.kvexp
    with FakeTensorMode():
        pool = torch.empty(9, 2, 16, 64, dtype=BF)
        status, lens = torch.empty(1, dtype=torch.int32), torch.empty(3, dtype=torch.int32)
        table = torch.empty(3, 4, dtype=torch.int32)
        kvs, q, f = torch.empty(6, 2, 64, dtype=BF), torch.empty(6, 8, 64, dtype=BF), torch.empty(32)
        x = torch.empty(6, 8, 64, dtype=FP, requires_grad=True)
        y = ops.rope(x, None, f)
        assert y.shape == x.shape and y.dtype == FP and y.requires_grad
        assert torch.autograd.grad(y, x, torch.empty_like(y))[0].shape == x.shape
        assert ops.paged_append(pool, pool, status, kvs, kvs, table, lens, None, q, f).shape == q.shape
        out, lse = ops.paged_attention(pool, pool, status, q, table, lens, None, 0.1)
        assert out.shape == q.shape and out.dtype == BF and lse.shape == (6, 8) and lse.dtype == torch.float32
        out, lse = ops.prefix_attention(pool, pool, status, q, table, lens, None, 1, 0.1)
        assert out.shape == q.shape and lse.shape == (6, 8)


def test_operators_refuse_cpu_tensors():
    import kvexp_amd.torch_ops  # noqa: F401

    x = torch.zeros(3, 2, 64, dtype=BF, requires_grad=True)
    with pytest.raises(ValueError, match="ROCm device tensor"):
        torch.ops.kvexp.rope(x, None, torch.zeros(32))
    pool, i32 = torch.zeros(4, 2, 16, 64, dtype=BF), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm device tensors"):
        torch.ops.kvexp.paged_attention(pool, pool, i32[:1], x.detach(), i32[:, None], i32, None, 0.1)


@pytest.mark.parametrize("d", [1, 2, 3, 7, 24, 48, 100, 641, 2**20 + 1, 2**30 - 1, 2**30 + 1])
def test_division_of_tokens_into_pages(d):
    """The quotient that the kernels form by a product, as the host sets it up, for every kind of divisor."""
    shift = (d - 1).bit_length()
    magic = 2 ** (31 + shift) // d + 1
    assert magic < 2**32 or d & (d - 1) == 0
    ts = {0, 1, d - 1, d, d + 1, 2**31 - 1, 2**31 - 2}
    ts |= {x for k in range(1, 2**31 // d + 1, max(1, 2**31 // d // 500)) for x in (k * d - 1, k * d)}
    for t in ts:
        if 0 <= t < 2**31 and d & (d - 1):
            assert t * magic >> (31 + shift) == t // d
