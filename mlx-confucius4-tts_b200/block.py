"""The decoder block's operators over torch CUDA tensors: the paged key-value
cache, the attention of one new token per sequence over it, and the linear
layer with its epilogue. BlockOps holds the calls (SamplingContext has them),
KVCache describes a cache's tensors. The C ABI in include/c4s_sampling.h
defines each operator.

Arguments are checked here (ValueError, TypeError) before the C call, whose own
refusals raise C4SError. Calls are ordered on the current torch stream of the
context's device, or on `stream`; with `stream` the outputs that a call
allocates belong to that stream.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math

BF16, FP16, FP32 = 0, 1, 2
HEAD_DIMS = (64, 96, 128)
ACTIVATIONS = {"none": 0, "gelu": 1, "gelu_erf": 2, "silu": 3, "relu": 4}


class _CacheStruct(C.Structure):
    """c4s_kv_cache."""
    _fields_ = ([(n, C.c_void_p) for n in ("k", "v", "k_sb", "v_sb")] +
                [(n, C.c_int64) for n in ("page_stride", "head_stride", "token_stride", "sb_page_stride",
                                          "sb_head_stride", "sb_token_stride")] +
                [(n, C.c_int32) for n in ("num_pages", "page_size", "kv_heads", "head_dim", "bits", "dtype", "group")])


def signatures():
    """ctypes argument types of the block's entry points."""
    vp, i32, i64, f32 = C.c_void_p, C.c_int32, C.c_int64, C.c_float
    kv = [vp, C.POINTER(_CacheStruct), vp, i64, i32, i32, vp, vp, i32, i64, i64, i64, vp, vp, vp]
    return {
        "c4s_linear": ([vp, vp, i32, i32, i32, i64, vp, vp, f32, vp, vp, i32, i64, vp, i32, vp, i64, vp, i32, i64, vp],
                       C.c_int),
        "c4s_kv_write": (kv, C.c_int),
        "c4s_kv_read": (kv, C.c_int),
        "c4s_attention_workspace": ([vp, i32, i32, i32], C.c_int64),
        "c4s_paged_attention": ([vp, C.POINTER(_CacheStruct), vp, i64, i32, i32, vp, i32, i32, i64, i64, vp, vp, f32,
                                 vp, i64, i64, vp, i64, vp], C.c_int),
    }


def _torch():
    import torch
    return torch


def _type(t, what: str, fp32: bool = False) -> int:
    """c4s_dtype of a tensor; int16 / uint16 tensors hold bf16 bit patterns."""
    torch = _torch()
    kinds = {torch.bfloat16: BF16, torch.float16: FP16, torch.int16: BF16, torch.uint16: BF16}
    if fp32:
        kinds[torch.float32] = FP32
    if t.dtype not in kinds:
        raise TypeError(f"{what}: {t.dtype} is not supported")
    return kinds[t.dtype]


def _ints(t, what: str, dtype, shape):
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}")
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous, of shape {tuple(shape)}")


def _on(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the context on {device}")


class KVCache:
    """A layer's paged key-value cache: views of its tensors.

    k, v        16-bit: bf16 or fp16 [pages, kv_heads, page_size, head_dim];
                codes (bits 8 or 4): uint8 [pages, kv_heads, page_size,
                head_dim * bits / 8]. Any strides with contiguous rows: pass
                pool.transpose(1, 2) of a [pages, page_size, kv_heads, ...] pool.
    k_sb, v_sb  codes: fp32 [pages, kv_heads, page_size, head_dim / group, 2],
                the (scale, bias) pair of each group.
    """

    def __init__(self, k, v, k_sb=None, v_sb=None, bits: int = 16):
        torch = _torch()
        if bits not in (16, 8, 4):
            raise ValueError("bits must be 16, 8 or 4")
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError("k and v must be alike, [pages, kv_heads, page_size, row]")
        if k.stride(3) != 1:
            raise ValueError("cache rows must be contiguous")
        self.k, self.v, self.k_sb, self.v_sb, self.bits = k, v, k_sb, v_sb, bits
        s = self.struct = _CacheStruct()
        s.num_pages, s.kv_heads, s.page_size = k.shape[0], k.shape[1], k.shape[2]
        s.bits = bits
        if bits == 16:
            if k_sb is not None or v_sb is not None:
                raise ValueError("a 16-bit cache has no scales")
            s.dtype = _type(k, "cache")
            s.head_dim, s.group = k.shape[3], 0
        else:
            if k.dtype != torch.uint8:
                raise TypeError("codes are uint8")
            if k_sb is None or v_sb is None:
                raise ValueError("codes need k_sb and v_sb")
            s.dtype = BF16
            s.head_dim = k.shape[3] * 8 // bits
            if (k_sb.dtype != torch.float32 or k_sb.dim() != 5 or k_sb.shape[:3] != k.shape[:3] or k_sb.shape[4] != 2
                    or k_sb.shape != v_sb.shape or v_sb.dtype != torch.float32 or k_sb.stride() != v_sb.stride()):
                raise ValueError("k_sb and v_sb must be alike, fp32 [pages, kv_heads, page_size, head_dim / group, 2]")
            if k_sb.shape[3] < 1 or s.head_dim % k_sb.shape[3] or k_sb.stride(4) != 1 or \
                    (k_sb.shape[3] > 1 and k_sb.stride(3) != 2):
                raise ValueError("the pairs of a row must be contiguous, one for each group of head_dim")
            s.group = s.head_dim // k_sb.shape[3]
            if s.group not in (32, 64):
                raise ValueError("groups are of 32 or 64 elements")
            s.k_sb, s.v_sb = k_sb.data_ptr(), v_sb.data_ptr()
            s.sb_page_stride, s.sb_head_stride, s.sb_token_stride = (4 * x for x in k_sb.stride()[:3])
        if s.head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
        s.k, s.v = k.data_ptr(), v.data_ptr()
        s.page_stride, s.head_stride, s.token_stride = (k.element_size() * x for x in k.stride()[:3])

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=None, bits: int = 16,
              group: int = 64, token_major: bool = False, device=None):
        """A new cache, its tensors zeroed: dtype (bf16 by default) rows, or codes."""
        torch = _torch()

        def pool(tail, dt):
            mid = (page_size, kv_heads) if token_major else (kv_heads, page_size)
            x = torch.zeros((num_pages, *mid, *tail), dtype=dt, device=device)
            return x.transpose(1, 2) if token_major else x
        if bits == 16:
            dt = torch.bfloat16 if dtype is None else dtype
            return cls(pool((head_dim,), dt), pool((head_dim,), dt))
        if group not in (32, 64) or head_dim % group:
            raise ValueError("groups are of 32 or 64 elements and divide head_dim")
        row, sb = (head_dim * bits // 8,), (head_dim // group, 2)
        return cls(pool(row, torch.uint8), pool(row, torch.uint8), pool(sb, torch.float32), pool(sb, torch.float32),
                   bits=bits)

    @property
    def kv_heads(self):
        return self.struct.kv_heads

    @property
    def head_dim(self):
        return self.struct.head_dim

    @property
    def page_size(self):
        return self.struct.page_size

    def _check_table(self, table):
        torch = _torch()
        if table.dtype != torch.int32:
            raise TypeError("page_table must be int32")
        if table.dim() != 2 or table.shape[1] < 1 or (table.shape[1] > 1 and table.stride(1) != 1) or \
                (table.shape[0] > 1 and table.stride(0) < table.shape[1]):
            raise ValueError("page_table must be [sequences, pages] with contiguous rows")


def _rows(t, what: str, heads: int, dim: int):
    """Checks a [n, heads, dim] tensor with contiguous rows."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim:
        raise ValueError(f"{what} must be [n, {heads}, {dim}]")
    if t.stride(2) != 1 or t.stride(0) < 0 or t.stride(1) < 0:
        raise ValueError(f"{what}: rows must be contiguous")


def check_kv(cache: KVCache, page_table, k, v, pos, tok_off, write: bool):
    """Refuses what c4s_kv_write / c4s_kv_read cannot take; returns (B, T, c4s_dtype)."""
    torch = _torch()
    cache._check_table(page_table)
    B, T = page_table.shape[0], k.shape[0]
    _rows(k, "k", cache.kv_heads, cache.head_dim)
    if k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
        raise ValueError("k and v must be alike")
    kind = _type(k, "k", fp32=not write)
    if write and cache.bits == 16 and kind != cache.struct.dtype:
        raise TypeError("k and v must be of the cache's type")
    if not write and (k.stride(1) < cache.head_dim or (T > 1 and k.stride(0) < cache.head_dim)) and cache.kv_heads > 1:
        raise ValueError("the rows of k and v must not overlap")
    _ints(pos, "pos", torch.int32, (B,))
    if tok_off is None:
        if T != B:
            raise ValueError("without tok_off there is one token per sequence")
    else:
        _ints(tok_off, "tok_off", torch.int64, (B + 1,))
    return B, T, kind


def check_attention(q, cache: KVCache, page_table, lens, start, out):
    """Refuses what c4s_paged_attention cannot take; returns (B, q_heads, c4s_dtype)."""
    torch = _torch()
    cache._check_table(page_table)
    B = page_table.shape[0]
    if q.dim() != 3 or q.shape[0] != B or q.shape[1] < 1 or q.shape[1] % cache.kv_heads:
        raise ValueError("q must be [sequences, q_heads, head_dim], q_heads a multiple of the cache's heads")
    _rows(q, "q", q.shape[1], cache.head_dim)
    kind = _type(q, "q")
    if cache.bits == 16 and kind != cache.struct.dtype:
        raise TypeError("q must be of the cache's type")
    _ints(lens, "lens", torch.int32, (B,))
    if start is not None:
        _ints(start, "start", torch.int32, (B,))
    if out is not None:
        _rows(out, "out", q.shape[1], cache.head_dim)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out must be like q")
        if (B > 1 and out.stride(0) < cache.head_dim) or (q.shape[1] > 1 and out.stride(1) < cache.head_dim):
            raise ValueError("the rows of out must not overlap")
    return B, q.shape[1], kind


def _matrix(t, what: str, shape):
    if t.dim() != 2 or tuple(t.shape) != tuple(shape) or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{what} must be {tuple(shape)} with contiguous rows")


def check_linear(x, weight, bias, act, residual, gamma, beta, out, out_dtype):
    """Refuses what c4s_linear cannot take; returns (M, K, N, c4s_dtype of x, of out, torch type of out)."""
    torch = _torch()
    if x.dim() != 2 or weight.dim() != 2:
        raise ValueError("x must be [M, K] and weight [N, K]")
    M, K = x.shape
    N = weight.shape[0]
    _matrix(x, "x", (M, K))
    _matrix(weight, "weight", (N, K))
    kind = _type(x, "x")
    if _type(weight, "weight") != kind:
        raise TypeError("x and weight must be of one type")
    if act not in ACTIVATIONS:
        raise ValueError(f"act must be one of {tuple(ACTIVATIONS)}")
    if out_dtype is None:
        out_dtype = x.dtype if out is None else out.dtype
    okind = FP32 if out_dtype == torch.float32 else kind
    if out_dtype != torch.float32 and out_dtype != x.dtype:
        raise TypeError("out is of x's type or fp32")
    for name, t, n in (("bias", bias, N), ("gamma", gamma, K), ("beta", beta, K)):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (n,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous fp32 [{n}]")
    for name, t in (("residual", residual), ("out", out)):
        if t is not None:
            if t.dtype != out_dtype:
                raise TypeError(f"{name} must be {out_dtype}")
            _matrix(t, name, (M, N))
    if M > 1 and out is not None and out.stride(0) < N:
        raise ValueError("the rows of out must not overlap")
    return M, K, N, kind, okind, out_dtype


class BlockOps:
    """The block's operators of a context (SamplingContext)."""

    def _allocating(self, stream):
        """New tensors belong to the stream that the call runs on."""
        return contextlib.nullcontext() if stream is None else _torch().cuda.stream(stream)

    def kv_write(self, cache: KVCache, page_table, k, v, pos, tok_off=None, stream=None):
        """Writes new tokens' k, v [T, kv_heads, head_dim] into the cache
        (c4s_kv_write). page_table int32 [B, pages]; pos int32 [B], the position
        of each sequence's first new token (< 0: skip it); tok_off int64 [B+1],
        the sequences' tokens, or None for one token per sequence."""
        B, T, kind = check_kv(cache, page_table, k, v, pos, tok_off, True)
        _on(self.device, k=k, v=v, page_table=page_table, pos=pos, tok_off=tok_off, cache=cache.k)
        rc = self.lib.c4s_kv_write(
            self._h, C.byref(cache.struct), page_table.data_ptr(), page_table.stride(0), page_table.shape[1], B,
            k.data_ptr(), v.data_ptr(), kind, k.stride(0), k.stride(1), T,
            None if tok_off is None else tok_off.data_ptr(), pos.data_ptr(), self._stream(stream))
        self._check(rc, "c4s_kv_write")

    def kv_read(self, cache: KVCache, page_table, pos, tok_off=None, total: int | None = None, dtype=None, k_out=None,
                v_out=None, stream=None):
        """Reads positions back (c4s_kv_read): (k, v) [total, kv_heads,
        head_dim] of `dtype` (the cache's type, or bf16 for codes), total =
        tok_off[B] (the sequences, without tok_off)."""
        torch = _torch()
        if (k_out is None) != (v_out is None):
            raise ValueError("k_out and v_out go together")
        if k_out is None:
            if total is None:
                if tok_off is not None:
                    raise ValueError("total is needed with tok_off")
                total = page_table.shape[0]
            if dtype is None:
                dtype = torch.float16 if cache.bits == 16 and cache.struct.dtype == FP16 else torch.bfloat16
            with self._allocating(stream):
                k_out, v_out = (torch.empty((total, cache.kv_heads, cache.head_dim), dtype=dtype, device=self.device)
                                for _ in "kv")
        B, T, kind = check_kv(cache, page_table, k_out, v_out, pos, tok_off, False)
        _on(self.device, k_out=k_out, v_out=v_out, page_table=page_table, pos=pos, tok_off=tok_off, cache=cache.k)
        rc = self.lib.c4s_kv_read(
            self._h, C.byref(cache.struct), page_table.data_ptr(), page_table.stride(0), page_table.shape[1], B,
            k_out.data_ptr(), v_out.data_ptr(), kind, k_out.stride(0), k_out.stride(1), T,
            None if tok_off is None else tok_off.data_ptr(), pos.data_ptr(), self._stream(stream))
        self._check(rc, "c4s_kv_read")
        return k_out, v_out

    def attention_workspace(self, batch: int, q_heads: int, head_dim: int, stream=None):
        """A zeroed workspace for paged_attention. Keep one per stream (or captured graph)."""
        n = self.lib.c4s_attention_workspace(self._h, batch, q_heads, head_dim)
        if n < 0:
            self._check(int(n), "c4s_attention_workspace")
        with self._allocating(stream):
            return _torch().zeros(n, dtype=_torch().uint8, device=self.device)

    def paged_attention(self, q, cache: KVCache, page_table, lens, start=None, scale: float | None = None, out=None,
                        work=None, stream=None):
        """Attention of one new token per sequence over its cached positions
        [start, lens) (c4s_paged_attention): q [B, q_heads, head_dim] -> out,
        like q. lens, start int32 [B]; scale 1 / sqrt(head_dim) by default;
        work: attention_workspace() (None: one for this call)."""
        torch = _torch()
        B, heads, kind = check_attention(q, cache, page_table, lens, start, out)
        _on(self.device, q=q, page_table=page_table, lens=lens, start=start, out=out, work=work, cache=cache.k)
        if out is None:
            with self._allocating(stream):
                out = torch.empty((B, heads, cache.head_dim), dtype=q.dtype, device=self.device)
        if work is None:
            work = self.attention_workspace(B, heads, cache.head_dim, stream)
        if scale is None:
            scale = 1.0 / math.sqrt(cache.head_dim)
        rc = self.lib.c4s_paged_attention(
            self._h, C.byref(cache.struct), page_table.data_ptr(), page_table.stride(0), page_table.shape[1], B,
            q.data_ptr(), kind, heads, q.stride(0), q.stride(1), lens.data_ptr(),
            None if start is None else start.data_ptr(), scale, out.data_ptr(), out.stride(0), out.stride(1),
            work.data_ptr(), work.numel() * work.element_size(), self._stream(stream))
        self._check(rc, "c4s_paged_attention")
        return out

    def linear(self, x, weight, bias=None, act: str = "none", residual=None, layer_norm: bool = False, gamma=None,
               beta=None, eps: float = 1e-5, norm_out=None, out=None, out_dtype=None, stream=None):
        """act(LN(x) weight^T + bias) + residual (c4s_linear): x [M, K] and
        weight [N, K] bf16 or fp16 -> out [M, N] of x's type or fp32. bias,
        gamma, beta fp32; act one of ACTIVATIONS; residual of out's type (it may
        be out); layer_norm=False skips the LayerNorm; norm_out: [M, K] workspace
        of the normalised rows."""
        torch = _torch()
        M, K, N, kind, okind, out_dtype = check_linear(x, weight, bias, act, residual, gamma, beta, out, out_dtype)
        _on(self.device, x=x, weight=weight, bias=bias, residual=residual, gamma=gamma, beta=beta, out=out,
            norm_out=norm_out)
        if norm_out is not None:
            _matrix(norm_out, "norm_out", (M, K))
            if norm_out.dtype != x.dtype or not norm_out.is_contiguous():
                raise ValueError("norm_out must be contiguous, of x's type")
        with self._allocating(stream):
            if out is None:
                out = torch.empty((M, N), dtype=out_dtype, device=self.device)
            if layer_norm and norm_out is None:
                norm_out = torch.empty((M, K), dtype=x.dtype, device=self.device)
        rc = self.lib.c4s_linear(
            self._h, x.data_ptr(), kind, M, K, x.stride(0), None if gamma is None else gamma.data_ptr(),
            None if beta is None else beta.data_ptr(), eps, norm_out.data_ptr() if layer_norm else None,
            weight.data_ptr(), N, weight.stride(0), None if bias is None else bias.data_ptr(), ACTIVATIONS[act],
            None if residual is None else residual.data_ptr(), 0 if residual is None else residual.stride(0),
            out.data_ptr(), okind, out.stride(0), self._stream(stream))
        self._check(rc, "c4s_linear")
        return out
