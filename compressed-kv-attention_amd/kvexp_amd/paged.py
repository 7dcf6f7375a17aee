"""A cache of plain keys and values in pages, for batches of sequences: rotary
positions, the append with the rotation on the way, and attention over the
pages and over a prefix that the batch shares (include/kvexp_hip.h, "paged
cache").

    cache = ctx.paged_cache(n_kv_heads, dim, n_pages, page_tokens=64)
    rope = kvexp_amd.Rope(inv_freq)                      # axes= for several position axes
    batch = kvexp_amd.Batch(table, lens)                 # lens count the new tokens
    q = cache.append(k, v, batch, rope=rope, q=q)        # keys rotated into their pages, queries rotated
    out = cache.attention(q, batch)                      # or attention(q, batch, prefix=prefix)

Tensors are torch tensors on the context's device; calls run on torch's current
stream (or ``stream=``) and read tables, lengths and positions there, so they
may be captured in a graph. Each attention call takes its workspace from torch's
allocator, so calls may overlap. The elements are bfloat16 or float16.
"""
from __future__ import annotations

import ctypes as C
import math

DTYPES = ("bfloat16", "float16")


class _Pages(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p),
                ("k_page", C.c_int64), ("k_head", C.c_int64), ("k_token", C.c_int64),
                ("v_page", C.c_int64), ("v_head", C.c_int64), ("v_token", C.c_int64),
                ("dtype", C.c_int32), ("n_pages", C.c_int32), ("page_tokens", C.c_int32), ("n_heads", C.c_int32),
                ("dim", C.c_int32), ("reserved", C.c_int32)]


class _Batch(C.Structure):
    _fields_ = [("table", C.c_void_p), ("lens", C.c_void_p), ("starts", C.c_void_p), ("table_stride", C.c_int64),
                ("table_width", C.c_int32), ("n_seqs", C.c_int32), ("n_tokens", C.c_int32), ("max_new", C.c_int32),
                ("max_len", C.c_int32), ("reserved", C.c_int32)]


class _Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("token", C.c_int64), ("head", C.c_int64)]


class _Rope(C.Structure):
    _fields_ = [("inv_freq", C.c_void_p), ("axes", C.c_void_p), ("n_freq", C.c_int32), ("n_axes", C.c_int32),
                ("interleaved", C.c_int32), ("scale", C.c_float)]


class _Positions(C.Structure):
    _fields_ = [("data", C.c_void_p), ("axis_stride", C.c_int64), ("offset", C.c_int64), ("wide", C.c_int32),
                ("reserved", C.c_int32)]


class _Shared(C.Structure):
    _fields_ = [("xkv", C.c_void_p), ("table", C.c_void_p), ("table_width", C.c_int32), ("n_tokens", C.c_int32)]


def declare(L, head) -> None:
    """Argument types of the paged entries of the library L."""
    vp, i32, P = C.c_void_p, C.c_int, C.POINTER
    L.kvexp_hip_rope_rows.argtypes = [vp, P(_Rope), P(_Positions), P(_Rows), P(_Rows), i32, i32, i32, i32, i32, vp]
    L.kvexp_hip_paged_append.argtypes = [vp, P(_Pages), P(_Batch), P(_Rows), P(_Rows), P(_Rope), P(_Positions),
                                         P(_Rows), P(_Rows), i32, vp, vp]
    L.kvexp_hip_prefix_create.argtypes = [vp, P(head), i32, i32, vp, P(vp)]
    L.kvexp_hip_prefix_destroy.argtypes = [vp]
    L.kvexp_hip_paged_attention_workspace.restype = C.c_int64
    L.kvexp_hip_paged_attention_workspace.argtypes = [vp, P(_Pages), P(_Batch), P(_Shared), i32]
    L.kvexp_hip_paged_attention.argtypes = [vp, P(_Pages), P(_Batch), P(_Shared), P(_Rows), i32, C.c_float, P(_Rows),
                                            vp, vp, C.c_size_t, vp, vp]
    L.kvexp_hip_paged_status.argtypes = [vp, vp, vp]


def _kv():
    import kvexp_amd

    return kvexp_amd


def _dtype_code(who: str, dtype) -> int:
    name = str(dtype).replace("torch.", "")
    if name not in DTYPES:
        raise ValueError(f"{who}: elements are bfloat16 or float16, not {name}")
    return DTYPES.index(name)


def _check_rows(who: str, name: str, t, dtype, n=None, heads=None, dim=None) -> None:
    if t.dim() != 3:
        raise ValueError(f"{who}: {name} must be [tokens, heads, head_dim]")
    if t.dtype != dtype:
        raise ValueError(f"{who}: {name} must be {dtype}, not {t.dtype}")
    want = (n, heads, dim)
    if any(w is not None and int(s) != w for s, w in zip(t.shape, want)):
        raise ValueError(f"{who}: {name} must be {list(want)}, not {list(t.shape)}")


def _check_device(who: str, device: int, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (t.device.type != "cuda" or t.device.index != device):
            raise ValueError(f"{who}: {name} must be on cuda:{device}, not {t.device}")


def _fits(t) -> bool:
    return (t.stride(2) == 1 or t.shape[2] == 1) and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 \
        and t.data_ptr() % 16 == 0


def _rows(t) -> _Rows:
    return _Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _readable(t):
    """t, or a copy of it where its layout is not one the kernels read."""
    import torch

    return t if t.numel() == 0 or _fits(t) else t.clone(memory_format=torch.contiguous_format)


class _on:
    """torch's current stream set to `stream` for the allocations inside (None: as it is)."""

    def __init__(self, stream):
        import torch

        if stream is not None and not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream))
        self.stream = stream
        self.guard = None if stream is None else torch.cuda.stream(stream)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


def _raw_stream(device: int):
    import torch

    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


class Rope:
    """A rotation of the first 2 n channels of a row.

    inv_freq  float32 [n] on the device: the angle of pair i is its position times inv_freq[i]
    axes      uint8 [n] on the device: the position axis of each pair (None: one axis)
    interleaved  pairs are channels (2 i, 2 i + 1) instead of (i, i + n)
    scale     factor of the rotated channels
    """

    def __init__(self, inv_freq, axes=None, interleaved: bool = False, scale: float = 1.0):
        if inv_freq.dim() != 1 or str(inv_freq.dtype) != "torch.float32" or inv_freq.numel() == 0:
            raise ValueError("kvexp.Rope: inv_freq must be float32 [n]")
        if axes is not None and (str(axes.dtype) != "torch.uint8" or axes.shape != inv_freq.shape):
            raise ValueError("kvexp.Rope: axes must be uint8, one per frequency")
        if not math.isfinite(scale):
            raise ValueError("kvexp.Rope: the scale is not finite")
        self.inv_freq, self.axes = inv_freq.contiguous(), None if axes is None else axes.contiguous()
        self.interleaved, self.scale = bool(interleaved), float(scale)

    def _struct(self, who: str, device: int, dim: int, n_axes: int) -> _Rope:
        _check_device(who, device, inv_freq=self.inv_freq, axes=self.axes)
        n = int(self.inv_freq.numel())
        if 2 * n > dim:
            raise ValueError(f"{who}: {2 * n} rotated channels, head_dim {dim}")
        return _Rope(self.inv_freq.data_ptr(), None if self.axes is None else self.axes.data_ptr(), n, n_axes,
                     int(self.interleaved), self.scale)


def _positions(who: str, device: int, positions, offset: int, n: int):
    """(_Positions, axes, what it points at)."""
    if positions is None:
        return _Positions(None, 0, int(offset), 0, 0), 1, None
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dim() != 2 or positions.shape[1] != n or positions.shape[0] == 0:
        raise ValueError(f"{who}: positions must be [tokens] or [axes, tokens] with {n} tokens")
    wide = str(positions.dtype) == "torch.int64"
    if not wide and str(positions.dtype) != "torch.int32":
        raise ValueError(f"{who}: positions must be int32 or int64")
    _check_device(who, device, positions=positions)
    if positions.stride(1) != 1 or (positions.shape[0] > 1 and positions.stride(0) < n):
        positions = positions.contiguous()
    return (_Positions(positions.data_ptr(), positions.stride(0), 0, int(wide), 0), int(positions.shape[0]),
            positions)


def rope(ctx, x, positions, rope: Rope, out=None, inverse: bool = False, stream=None):
    """x [tokens, heads, head_dim] rotated by `rope` at `positions` ([tokens], [axes, tokens], or None for 0, 1, 2, ..),
    into out (which may be x) or a new tensor; inverse: rotated back."""
    import torch

    kv, who = _kv(), "kvexp.rope"
    code = _dtype_code(who, x.dtype)
    _check_rows(who, "x", x, x.dtype)
    n, heads, dim = (int(s) for s in x.shape)
    if out is not None:
        _check_rows(who, "out", out, x.dtype, n, heads, dim)
        if not _fits(out):
            raise ValueError(f"{who}: out must have contiguous channels, strides of multiples of 8, 16-byte alignment")
    _check_device(who, ctx.device, x=x, out=out)
    with _on(stream):
        x = x.detach()
        at, axes, keep = _positions(who, ctx.device, positions, 0, n)
        r = rope._struct(who, ctx.device, dim, axes)
        src = _readable(x)
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if x.numel():
            kv.check(kv.lib().kvexp_hip_rope_rows(ctx.h, r, at, _rows(src), _rows(out), n, heads, dim, code,
                                                  int(inverse), _raw_stream(ctx.device)))
    del keep
    return out


class Batch:
    """Sequences over a paged cache, and the new tokens that a call brings.

    table     int32 [seqs, width]: the pages of each sequence; entries past its length are not read
    lens      int32 [seqs]: tokens of each sequence, the new ones included
    starts    int32 [seqs + 1]: rows [starts[b], starts[b + 1]) of the call's tensors are sequence b's new tokens
              (None: the same number each)
    max_new   the most new tokens of a sequence (with starts; None: all of the call's)
    max_len   a bound on lens that the number of splits follows (None: the table's)
    """

    def __init__(self, table, lens, starts=None, max_new: int | None = None, max_len: int | None = None):
        who = "kvexp.Batch"
        for name, t, d in (("table", table, 2), ("lens", lens, 1), ("starts", starts, 1)):
            if t is not None and (t.dim() != d or str(t.dtype) != "torch.int32"):
                raise ValueError(f"{who}: {name} must be int32 with {d} dimension{'s' if d > 1 else ''}")
        n = int(lens.shape[0])
        if int(table.shape[0]) != n or (starts is not None and int(starts.shape[0]) != n + 1):
            raise ValueError(f"{who}: table and lens have one row per sequence, starts one more")
        self.table = table if table.stride(1) == 1 or table.shape[1] <= 1 else table.contiguous()
        self.lens, self.starts = lens.contiguous(), None if starts is None else starts.contiguous()
        self.max_new, self.max_len = max_new, max_len

    @property
    def n_seqs(self) -> int:
        return int(self.lens.shape[0])

    def _struct(self, who: str, device: int, n_tokens: int) -> _Batch:
        _check_device(who, device, table=self.table, lens=self.lens, starts=self.starts)
        if self.starts is None and (n_tokens % self.n_seqs if self.n_seqs else n_tokens):
            raise ValueError(f"{who}: {n_tokens} tokens of {self.n_seqs} sequences without starts")
        return _Batch(self.table.data_ptr(), self.lens.data_ptr(),
                      None if self.starts is None else self.starts.data_ptr(), self.table.stride(0),
                      int(self.table.shape[1]), self.n_seqs, n_tokens, int(self.max_new or 0), int(self.max_len or 0), 0)


class Prefix:
    """A prefix that a batch shares, kept as XKV containers: one K and one V
    container (Encoded, or Cache.view()) per KV head, all of the same tokens."""

    def __init__(self, ctx, ks, vs, stream=None):
        kv, who = _kv(), "kvexp.Prefix"
        if len(ks) != len(vs) or not ks:
            raise ValueError(f"{who}: one K and one V container per head")
        seq, dim = int(ks[0].seq), int(ks[0].dim)
        if any(int(e.seq) != seq or int(e.dim) != dim for e in list(ks) + list(vs)):
            raise ValueError(f"{who}: containers of one length and head_dim")
        arr, self._keep = kv._heads_array([dict(kx=k, vx=v, seq=seq) for k, v in zip(ks, vs)])
        h = C.c_void_p()
        kv.check(kv.lib().kvexp_hip_prefix_create(ctx.h, arr, len(ks), dim, kv._stream(stream), C.byref(h)))
        self.ctx, self.h, self.n_heads, self.dim, self.seq = ctx, h, len(ks), dim, seq

    def _struct(self, who: str, cache) -> _Shared:
        if not self.h:
            raise ValueError(f"{who}: the prefix is closed")
        return _Shared(self.h, None, 0, self.seq)

    def close(self) -> None:
        """Frees the tables (the caller's calls that use them must be over)."""
        if getattr(self, "h", None):
            _kv().lib().kvexp_hip_prefix_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagePrefix:
    """A prefix that a batch shares, kept in pages of the cache (int32 [pages])."""

    def __init__(self, cache, table, seq: int):
        who = "kvexp.PagePrefix"
        if table.dim() != 1 or str(table.dtype) != "torch.int32":
            raise ValueError(f"{who}: table must be int32 [pages]")
        if seq <= 0 or int(table.shape[0]) * cache.page_tokens < seq:
            raise ValueError(f"{who}: {int(seq)} tokens in {int(table.shape[0])} pages of {cache.page_tokens}")
        self.cache, self.table, self.seq = cache, table.contiguous(), int(seq)

    def _struct(self, who: str, cache) -> _Shared:
        if cache is not self.cache:
            raise ValueError(f"{who}: the prefix is in pages of another cache")
        _check_device(who, cache.ctx.device, prefix=self.table)
        return _Shared(None, self.table.data_ptr(), int(self.table.shape[0]), self.seq)


class PagedCache:
    """Pages of keys and values: k and v [n_pages, n_heads, page_tokens, head_dim] (given, in any strides that are
    multiples of 8 elements with contiguous channels, or made here)."""

    def __init__(self, ctx, n_heads: int, dim: int, n_pages: int, page_tokens: int = 64, dtype=None, k=None, v=None):
        import torch

        who = "kvexp.PagedCache"
        dtype = torch.bfloat16 if dtype is None else dtype
        self._code = _dtype_code(who, dtype)
        if dim <= 0 or dim % 8 or dim > 256:
            raise ValueError(f"{who}: head_dim must be a multiple of 8 and at most 256")
        if min(n_heads, n_pages, page_tokens) <= 0:
            raise ValueError(f"{who}: empty pages")
        shape = (int(n_pages), int(n_heads), int(page_tokens), int(dim))
        if (k is None) != (v is None):
            raise ValueError(f"{who}: k and v go together")
        for name, t in (("k", k), ("v", v)):
            if t is None:
                continue
            if tuple(t.shape) != shape or t.dtype != dtype:
                raise ValueError(f"{who}: {name} must be {dtype} {list(shape)}")
            if t.stride(3) != 1 or any(t.stride(i) % 8 for i in range(3)) or t.data_ptr() % 16:
                raise ValueError(f"{who}: {name} must have contiguous channels, strides of multiples of 8 elements and "
                                 "16-byte alignment")
        _check_device(who, ctx.device, k=k, v=v)
        dev = torch.device("cuda", ctx.device)
        self.ctx, self.dtype = ctx, dtype
        self.n_pages, self.n_heads, self.page_tokens, self.dim = shape
        self.k = torch.empty(shape, dtype=dtype, device=dev) if k is None else k
        self.v = torch.empty(shape, dtype=dtype, device=dev) if v is None else v
        self.status_word = torch.zeros(1, dtype=torch.int32, device=dev)
        sk, sv = self.k.stride(), self.v.stride()
        self._struct = _Pages(self.k.data_ptr(), self.v.data_ptr(), sk[0], sk[1], sk[2], sv[0], sv[1], sv[2],
                              self._code, shape[0], shape[2], shape[1], shape[3], 0)

    def prefix(self, table, seq: int) -> PagePrefix:
        """The first `seq` tokens of the pages `table` (int32 [pages]) as a prefix that batches share."""
        return PagePrefix(self, table, seq)

    def append(self, k, v, batch: Batch, rope: Rope | None = None, positions=None, offset: int = 0, q=None, q_out=None,
               check_errors: bool = False, stream=None):
        """Writes the batch's new keys (rotated by `rope`) and values [tokens, n_heads, head_dim] to their pages;
        returns q [tokens, query heads, head_dim] rotated (into q_out, which may be q), or None. positions: [tokens] or
        [axes, tokens]; None: each token's index in its sequence plus `offset` (the tokens of a shared prefix)."""
        import torch

        kv, who = _kv(), "kvexp.paged_append"
        n = int(k.shape[0])
        _check_rows(who, "k", k, self.dtype, n, self.n_heads, self.dim)
        _check_rows(who, "v", v, self.dtype, n, self.n_heads, self.dim)
        if q is not None:
            _check_rows(who, "q", q, self.dtype, n, None, self.dim)
            if rope is None:
                raise ValueError(f"{who}: queries without a rotation")
        if q_out is not None:
            if q is None:
                raise ValueError(f"{who}: q and q_out go together")
            _check_rows(who, "q_out", q_out, self.dtype, *q.shape)
            if not _fits(q_out):
                raise ValueError(f"{who}: q_out must have contiguous channels, strides of multiples of 8, 16-byte "
                                 "alignment")
        _check_device(who, self.ctx.device, k=k, v=v, q=q, q_out=q_out)
        with _on(stream):
            at, axes, keep = _positions(who, self.ctx.device, positions, offset, n)
            r = None if rope is None else rope._struct(who, self.ctx.device, self.dim, axes)
            b = batch._struct(who, self.ctx.device, n)
            if q is not None and q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            if n and (q is None or q.shape[1]):
                k, v, src = _readable(k), _readable(v), None if q is None else _readable(q)
                kv.check(kv.lib().kvexp_hip_paged_append(
                    self.ctx.h, self._struct, b, _rows(k), _rows(v), r, at, None if src is None else _rows(src),
                    None if src is None else _rows(q_out), 0 if src is None else int(src.shape[1]),
                    self.status_word.data_ptr(), _raw_stream(self.ctx.device)))
            if check_errors:
                self.status()
        del keep
        return q_out

    def attention(self, q, batch: Batch, scale: float | None = None, prefix=None, out=None, lse=None,
                  return_lse: bool = False, check_errors: bool = False, stream=None):
        """Attention of the new tokens' queries q [tokens, query heads, head_dim] over the pages (and `prefix`, a Prefix
        or PagePrefix that every sequence shares): token i of a sequence's n new ones sees the first len - n + i + 1
        tokens of it. scale: of the scores (None: 1 / sqrt(head_dim)). Returns out, or (out, lse [tokens, query
        heads] float32) with return_lse; a token that sees nothing gives 0 and -inf."""
        import torch

        kv, who = _kv(), "kvexp.paged_attention"
        _check_rows(who, "q", q, self.dtype, None, None, self.dim)
        n, heads = int(q.shape[0]), int(q.shape[1])
        if heads == 0 or heads % self.n_heads:
            raise ValueError(f"{who}: {heads} query heads over {self.n_heads} heads")
        if out is not None:
            _check_rows(who, "out", out, self.dtype, n, heads, self.dim)
            if not _fits(out):
                raise ValueError(f"{who}: out must have contiguous channels, strides of multiples of 8, 16-byte "
                                 "alignment")
        if lse is not None and (tuple(lse.shape) != (n, heads) or lse.dtype != torch.float32
                                or not lse.is_contiguous()):
            raise ValueError(f"{who}: lse must be contiguous float32 [{n}, {heads}]")
        scale = 1.0 / math.sqrt(self.dim) if scale is None else float(scale)
        if not math.isfinite(scale):
            raise ValueError(f"{who}: the scale is not finite")
        _check_device(who, self.ctx.device, q=q, out=out, lse=lse)
        with _on(stream):
            b = batch._struct(who, self.ctx.device, n)
            sh = None if prefix is None else prefix._struct(who, self)
            src = _readable(q.detach())
            if out is None:
                out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            if lse is None and return_lse:
                lse = torch.empty((n, heads), dtype=torch.float32, device=q.device)
            L = kv.lib()
            size = L.kvexp_hip_paged_attention_workspace(self.ctx.h, self._struct, b, sh, heads)
            if size < 0:
                raise kv.KvexpHipError(1, L.kvexp_hip_last_error().decode())
            ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
            if n:
                kv.check(L.kvexp_hip_paged_attention(
                    self.ctx.h, self._struct, b, sh, _rows(src), heads, scale, _rows(out),
                    None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), size,
                    self.status_word.data_ptr(), _raw_stream(self.ctx.device)))
            if check_errors:
                self.status()
        return (out, lse) if return_lse else out

    def status(self, stream=None) -> None:
        """Raises what the cache's calls found wrong on the device since the last check (synchronises)."""
        kv = _kv()
        kv.check(kv.lib().kvexp_hip_paged_status(self.ctx.h, self.status_word.data_ptr(), kv._stream(stream)))
