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


_torch = _lib = None


def _load():
    """torch and the library, once (importing this module loads neither)."""
    global _torch, _lib
    if _lib is None:
        import torch

        import kvexp_amd

        _torch, _lib = torch, kvexp_amd.lib()
    return _torch, _lib


def _kv():
    import kvexp_amd

    return kvexp_amd


def _check(rc: int) -> None:
    if rc:
        _kv().check(rc)


def _dtype_code(who: str, dtype) -> int:
    torch = _torch_module()
    if dtype is torch.bfloat16:
        return 0
    if dtype is torch.float16:
        return 1
    raise ValueError(f"{who}: elements are bfloat16 or float16, not {dtype}")


def _torch_module():
    if _torch is not None:
        return _torch
    import torch

    return torch


def _check_rows(who: str, name: str, t, dtype, n=None, heads=None, dim=None) -> None:
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{who}: {name} must be [tokens, heads, head_dim]")
    if t.dtype is not dtype:
        raise ValueError(f"{who}: {name} must be {dtype}, not {t.dtype}")
    if (n is not None and shape[0] != n) or (heads is not None and shape[1] != heads) or \
            (dim is not None and shape[2] != dim):
        raise ValueError(f"{who}: {name} must be {[n, heads, dim]}, not {list(shape)}")


def _check_device(who: str, device: int, *tensors, names) -> None:
    for t in tensors:
        if t is not None and t.get_device() != device:  # (-1: not on a GPU)
            name = next(n for n, x in zip(names, tensors) if x is t)
            raise ValueError(f"{who}: {name} must be on cuda:{device}, not {t.device}")


def _rows(t) -> _Rows | None:
    """t as the kernels read it; None where its layout is not one they do."""
    token, head, channel = t.stride()
    p = t.data_ptr()
    if (channel != 1 and t.shape[2] != 1) or (token | head) % 8 or p % 16:
        return None
    return _Rows(p, token, head)


def _readable(t):
    """(rows, what they point at): t, or a copy of it where its layout is not one the kernels read."""
    r = _rows(t)
    if r is None:
        t = t.clone(memory_format=_torch_module().contiguous_format)
        r = _rows(t)
    return r, t


def _writable(who: str, name: str, t) -> _Rows:
    r = _rows(t)
    if r is None:
        raise ValueError(f"{who}: {name} must have contiguous channels, strides of multiples of 8 and 16-byte alignment")
    if (r.token == 0 and t.shape[0] > 1) or (r.head == 0 and t.shape[1] > 1):
        raise ValueError(f"{who}: rows of {name} lie on one another")
    return r


class _on:
    """torch's current stream set to `stream` for what is inside (None: as it is)."""

    def __init__(self, stream):
        self.guard = None
        if stream is not None:
            torch = _torch_module()
            if not isinstance(stream, torch.cuda.Stream):
                stream = torch.cuda.ExternalStream(int(stream))
            self.guard = torch.cuda.stream(stream)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


def _raw_stream(device: int) -> int:
    return _torch_module()._C._cuda_getCurrentRawStream(device)


def _read_only(name: str):
    """A property without a setter: what was checked when the object was made stays what the calls use."""
    return property(lambda self: getattr(self, name))


class Rope:
    """A rotation of the first 2 n channels of a row.

    inv_freq  float32 [n] on the device: the angle of pair i is its position times inv_freq[i]
    axes      uint8 [n] on the device: the position axis of each pair (None: one axis)
    interleaved  pairs are channels (2 i, 2 i + 1) instead of (i, i + n)
    scale     factor of the rotated channels
    """

    def __init__(self, inv_freq, axes=None, interleaved: bool = False, scale: float = 1.0):
        torch = _torch_module()
        if inv_freq.dim() != 1 or inv_freq.dtype is not torch.float32 or inv_freq.numel() == 0:
            raise ValueError("kvexp.Rope: inv_freq must be float32 [n]")
        if axes is not None and (axes.dtype is not torch.uint8 or axes.shape != inv_freq.shape):
            raise ValueError("kvexp.Rope: axes must be uint8, one per frequency")
        if not math.isfinite(scale):
            raise ValueError("kvexp.Rope: the scale is not finite")
        self._inv_freq, self._axes = inv_freq.contiguous(), None if axes is None else axes.contiguous()
        self.interleaved, self.scale = bool(interleaved), float(scale)

    inv_freq, axes = _read_only("_inv_freq"), _read_only("_axes")

    def _struct(self, who: str, device: int, dim: int, n_axes: int) -> _Rope:
        inv_freq, axes = self._inv_freq, self._axes
        _check_device(who, device, inv_freq, axes, names=("inv_freq", "axes"))
        n = inv_freq.numel()
        if 2 * n > dim:
            raise ValueError(f"{who}: {2 * n} rotated channels, head_dim {dim}")
        return _Rope(inv_freq.data_ptr(), None if axes is None else axes.data_ptr(), n, n_axes, int(self.interleaved),
                     self.scale)


def _positions(who: str, device: int, positions, offset: int, n: int):
    """(_Positions, axes, what it points at)."""
    if positions is None:
        return _Positions(None, 0, int(offset), 0, 0), 1, None
    torch = _torch_module()
    shape = positions.shape
    if len(shape) not in (1, 2) or shape[-1] != n or shape[0] == 0:
        raise ValueError(f"{who}: positions must be [tokens] or [axes, tokens] with {n} tokens")
    wide = positions.dtype is torch.int64
    if not wide and positions.dtype is not torch.int32:
        raise ValueError(f"{who}: positions must be int32 or int64")
    _check_device(who, device, positions, names=("positions",))
    axes = 1 if len(shape) == 1 else int(shape[0])
    if positions.stride(-1) != 1 or (axes > 1 and positions.stride(0) < n):
        positions = positions.contiguous()
    return _Positions(positions.data_ptr(), positions.stride(0) if axes > 1 else 0, 0, int(wide), 0), axes, positions


def rope(ctx, x, positions, rope: Rope, out=None, inverse: bool = False, stream=None):
    """x [tokens, heads, head_dim] rotated by `rope` at `positions` ([tokens], [axes, tokens], or None for 0, 1, 2, ..),
    into out (which may be x) or a new tensor; inverse: rotated back."""
    who = "kvexp.rope"
    code = _dtype_code(who, x.dtype)
    _check_rows(who, "x", x, x.dtype)
    n, heads, dim = x.shape
    if dim == 0 or dim % 8 or dim > 256:
        raise ValueError(f"{who}: head_dim must be a multiple of 8 and at most 256")
    if out is not None:
        _check_rows(who, "out", out, x.dtype, n, heads, dim)
    _check_device(who, ctx.device, x, out, names=("x", "out"))
    if stream is not None:
        with _on(stream):
            return globals()["rope"](ctx, x, positions, rope, out, inverse)
    torch, L = _load()
    at, axes, keep = _positions(who, ctx.device, positions, 0, n)
    r = rope._struct(who, ctx.device, dim, axes)
    if out is None:
        out = x.new_empty(x.shape)
    to = _writable(who, "out", out)
    if n and heads:
        src, x = _readable(x)
        _check(L.kvexp_hip_rope_rows(ctx.h, r, at, src, to, n, heads, dim, code, int(inverse), _raw_stream(ctx.device)))
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
        who, i32 = "kvexp.Batch", _torch_module().int32
        for name, t, d in (("table", table, 2), ("lens", lens, 1), ("starts", starts, 1)):
            if t is not None and (t.dtype is not i32 or t.dim() != d):
                raise ValueError(f"{who}: {name} must be int32 with {d} dimension{'s' if d > 1 else ''}")
        n, (rows, width) = lens.shape[0], table.shape
        if rows != n or (starts is not None and starts.shape[0] != n + 1):
            raise ValueError(f"{who}: table and lens have one row per sequence, starts one more")
        rs, cs = table.stride()
        self._table = table if (width <= 1 or cs == 1) and (n <= 1 or rs >= width) else table.contiguous()
        self._lens, self._starts, self._n_seqs = lens.contiguous(), None if starts is None else starts.contiguous(), n
        self.max_new, self.max_len = max_new, max_len

    table, lens, starts, n_seqs = (_read_only(x) for x in ("_table", "_lens", "_starts", "_n_seqs"))

    def _struct(self, who: str, device: int, n_tokens: int) -> _Batch:
        table, lens, starts, n = self._table, self._lens, self._starts, self._n_seqs
        _check_device(who, device, table, lens, starts, names=("table", "lens", "starts"))
        if starts is None and (n_tokens % n if n else n_tokens):
            raise ValueError(f"{who}: {n_tokens} tokens of {n} sequences without starts")
        return _Batch(table.data_ptr(), lens.data_ptr(), None if starts is None else starts.data_ptr(), table.stride(0),
                      table.shape[1], n, n_tokens, int(self.max_new or 0), int(self.max_len or 0))


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
        if table.dim() != 1 or table.dtype is not _torch_module().int32:
            raise ValueError(f"{who}: table must be int32 [pages]")
        if seq <= 0 or int(table.shape[0]) * cache.page_tokens < seq:
            raise ValueError(f"{who}: {int(seq)} tokens in {int(table.shape[0])} pages of {cache.page_tokens}")
        self.cache, self.table, self.seq = cache, table.contiguous(), int(seq)

    def _struct(self, who: str, cache) -> _Shared:
        if cache is not self.cache:
            raise ValueError(f"{who}: the prefix is in pages of another cache")
        _check_device(who, cache.ctx.device, self.table, names=("prefix",))
        return _Shared(None, self.table.data_ptr(), int(self.table.shape[0]), self.seq)


class PagedCache:
    """Pages of keys and values: k and v [n_pages, n_heads, page_tokens, head_dim] (given, in any strides that are
    multiples of 8 elements with contiguous channels, or made here). status: an int32 word on the device for the errors
    that only the device can see (None: one of its own)."""

    def __init__(self, ctx, n_heads: int, dim: int, n_pages: int, page_tokens: int = 64, dtype=None, k=None, v=None,
                 status=None):
        torch = _torch_module()
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
        if status is not None and (status.dtype is not torch.int32 or status.numel() != 1):
            raise ValueError(f"{who}: status must be one int32 word")
        _check_device(who, ctx.device, k, v, status, names=("k", "v", "status"))
        dev = torch.device("cuda", ctx.device)
        self.ctx, self.dtype = ctx, dtype
        self.n_pages, self.n_heads, self.page_tokens, self.dim = shape
        self._k = torch.empty(shape, dtype=dtype, device=dev) if k is None else k
        self._v = torch.empty(shape, dtype=dtype, device=dev) if v is None else v
        self._status = torch.zeros(1, dtype=torch.int32, device=dev) if status is None else status
        self._sizes = {}
        sk, sv = self.k.stride(), self.v.stride()
        self._struct = _Pages(self.k.data_ptr(), self.v.data_ptr(), sk[0], sk[1], sk[2], sv[0], sv[1], sv[2],
                              self._code, shape[0], shape[2], shape[1], shape[3], 0)

    k, v, status_word = _read_only("_k"), _read_only("_v"), _read_only("_status")

    def prefix(self, table, seq: int) -> PagePrefix:
        """The first `seq` tokens of the pages `table` (int32 [pages]) as a prefix that batches share."""
        return PagePrefix(self, table, seq)

    def append(self, k, v, batch: Batch, rope: Rope | None = None, positions=None, offset: int = 0, q=None, q_out=None,
               check_errors: bool = False, stream=None):
        """Writes the batch's new keys (rotated by `rope`) and values [tokens, n_heads, head_dim] to their pages;
        returns q [tokens, query heads, head_dim] rotated (into q_out, which may be q), or None. positions: [tokens] or
        [axes, tokens]; None: each token's index in its sequence plus `offset` (the tokens of a shared prefix)."""
        who = "kvexp.paged_append"
        n = int(k.shape[0]) if k.dim() else 0
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
        _check_device(who, self.ctx.device, k, v, q, q_out, names=("k", "v", "q", "q_out"))
        if stream is not None:
            with _on(stream):
                return self.append(k, v, batch, rope, positions, offset, q, q_out, check_errors)
        torch, L = _load()
        at, axes, keep = _positions(who, self.ctx.device, positions, offset, n)
        r = None if rope is None else rope._struct(who, self.ctx.device, self.dim, axes)
        b = batch._struct(who, self.ctx.device, n)
        if q is not None and q_out is None:
            q_out = q.new_empty(q.shape)
        to = None if q is None else _writable(who, "q_out", q_out)
        if n:
            (kr, k), (vr, v) = _readable(k), _readable(v)
            qr, heads = None, 0
            if q is not None and q.shape[1]:
                (qr, q), heads = _readable(q), int(q.shape[1])
            _check(L.kvexp_hip_paged_append(self.ctx.h, self._struct, b, kr, vr, r, at, qr, to if heads else None, heads,
                                            self._status.data_ptr(), _raw_stream(self.ctx.device)))
        if check_errors:
            self.status()
        return q_out

    def attention(self, q, batch: Batch, scale: float | None = None, prefix=None, out=None, lse=None,
                  return_lse: bool = False, check_errors: bool = False, stream=None):
        """Attention of the new tokens' queries q [tokens, query heads, head_dim] over the pages (and `prefix`, a Prefix
        or PagePrefix that every sequence shares): token i of a sequence's n new ones sees the first len - n + i + 1
        tokens of it. scale: of the scores (None: 1 / sqrt(head_dim)). Returns out, or (out, lse [tokens, query
        heads] float32) with return_lse; a token that sees nothing gives 0 and -inf."""
        who = "kvexp.paged_attention"
        _check_rows(who, "q", q, self.dtype, None, None, self.dim)
        n, heads, _ = q.shape
        if heads == 0 or heads % self.n_heads:
            raise ValueError(f"{who}: {heads} query heads over {self.n_heads} heads")
        if out is not None:
            _check_rows(who, "out", out, self.dtype, n, heads, self.dim)
        if lse is not None and (tuple(lse.shape) != (n, heads) or lse.dtype is not _torch_module().float32
                                or not lse.is_contiguous()):
            raise ValueError(f"{who}: lse must be contiguous float32 [{n}, {heads}]")
        scale = 1.0 / math.sqrt(self.dim) if scale is None else float(scale)
        if not math.isfinite(scale):
            raise ValueError(f"{who}: the scale is not finite")
        _check_device(who, self.ctx.device, q, out, lse, names=("q", "out", "lse"))
        if stream is not None:
            with _on(stream):
                return self.attention(q, batch, scale, prefix, out, lse, return_lse, check_errors)
        torch, L = _load()
        b = batch._struct(who, self.ctx.device, n)
        sh = None if prefix is None else prefix._struct(who, self)
        if out is None:
            out = q.new_empty(q.shape)
        to = _writable(who, "out", out)
        if lse is None and return_lse:
            lse = torch.empty((n, heads), dtype=torch.float32, device=q.device)
        # the workspace follows the sizes of the call
        key = (n, heads, b.n_seqs, b.table_width, batch._starts is None, batch.max_new, batch.max_len,
               None if sh is None else (sh.xkv is None, sh.n_tokens))
        size = self._sizes.get(key)
        if size is None:
            size = L.kvexp_hip_paged_attention_workspace(self.ctx.h, self._struct, b, sh, heads)
            if size < 0:
                raise _kv().KvexpHipError(1, L.kvexp_hip_last_error().decode())
            if len(self._sizes) >= 1024:
                self._sizes.clear()
            self._sizes[key] = size
        if n:
            ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
            src, q = _readable(q)
            _check(L.kvexp_hip_paged_attention(
                self.ctx.h, self._struct, b, sh, src, heads, scale, to, None if lse is None else lse.data_ptr(),
                None if ws is None else ws.data_ptr(), size, self._status.data_ptr(), _raw_stream(self.ctx.device)))
        if check_errors:
            self.status()
        return (out, lse) if return_lse else out

    def status(self, stream=None) -> None:
        """Raises what the cache's calls found wrong on the device since the last check (synchronises)."""
        kv = _kv()
        kv.check(kv.lib().kvexp_hip_paged_status(self.ctx.h, self._status.data_ptr(), kv._stream(stream)))
