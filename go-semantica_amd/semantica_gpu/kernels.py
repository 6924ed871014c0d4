"""Kernel-seam wrappers: the reference's internal/kernels entry points over
device tensors (torch is used only to hold HIP device memory and streams).

  quantize_symmetric_int8   <- QuantizeSymmetricINT8Into  internal/kernels/quantize.go:29
  Q8Weight + matmul_q8_0    <- MatMulQ8_0INT8             internal/kernels/quantize.go:346
  block_sums                <- the int32 block dots of matmulInnerLoop* (simd_amd64.s:241-304)
  rmsnorm                   <- RMSNorm                    internal/kernels/norm.go:8
  qknorm_rope               <- QK-norm + ApplyRoPECachedParallel (model_int8.go:371-452)
  attention                 <- MultiHeadAttentionChunked  internal/kernels/attention.go:88
  gelu_quick_mul            <- GELUQuickSIMD + VecMulF32  activation.go:47, matmul.go:238
  pool_l2                   <- MeanPoolingPartial + l2Normalize (attention.go:423, model.go:808)

and the layer operators of sibling models, which have no counterpart there:

  attention_masked, block_norm, AdapterBank + adapters_apply
  KVCache + kv_cache_write, kv_cache_read, attention_shared
  Q4Weight + matmul_q4

They take row-strided 2-D tensors of float32, float16 or bfloat16 and the CSR
offsets as an int32 device tensor, run asynchronously on the current stream of the
tensors' device (or `stream`), and allocate nothing but the default workspaces of
adapters_apply and attention_shared.
"""
from __future__ import annotations

import collections
import ctypes

import numpy as np

from . import _lib


def _vp(t):
    return ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    if stream is None:
        import torch
        return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    return ctypes.c_void_p(stream)


def _off(offsets):
    a = np.ascontiguousarray(offsets, np.int32)
    return a, ctypes.c_void_p(a.ctypes.data)


def _check_dev(*ts):
    for t in ts:
        if not t.is_cuda or not t.is_contiguous():
            raise ValueError("kernel-seam wrappers take contiguous device tensors")


class Q8Weight:
    """A raw Q8_0 matrix [out_dim][in_dim/32][34 B] repacked on the device."""

    def __init__(self, ctx, raw_q8: np.ndarray, out_dim: int, in_dim: int):
        self.ctx, self.lib = ctx, ctx.lib
        raw = np.ascontiguousarray(raw_q8, np.uint8)
        if raw.size != out_dim * (in_dim // 32) * 34:
            raise ValueError("raw Q8_0 size does not match out_dim x in_dim")
        h = ctypes.c_void_p()
        _lib.check(self.lib.sg_q8_weight_create(ctx.handle, ctypes.c_void_p(raw.ctypes.data), out_dim, in_dim,
                                                ctypes.byref(h)))
        self.handle, self.out_dim, self.in_dim = h, out_dim, in_dim

    def close(self):
        if self.handle:
            self.lib.sg_q8_weight_free(self.handle)
            self.handle = None


def quantize_symmetric_int8(ctx, x, offsets, q_out, scale_out, stream=None):
    _check_dev(x, q_out, scale_out)
    rows, cols = x.shape
    off, offp = _off(offsets)
    _lib.check(ctx.lib.sg_quantize_act(ctx.handle, _vp(x), rows, cols, offp, len(off) - 1, _vp(q_out),
                                       _vp(scale_out), _stream(stream)))


def matmul_q8_0(ctx, dst, w: Q8Weight, x, row_scale, stream=None):
    _check_dev(dst, x, row_scale)
    _lib.check(ctx.lib.sg_matmul_q8_0_int8(ctx.handle, _vp(dst), w.handle, _vp(x), _vp(row_scale), x.shape[0],
                                           _stream(stream)))


def matmul_q8_0_noalloc(ctx, dst, w: Q8Weight, x, row_scale, stream=None):
    """matmul_q8_0 with the operand relayout in the library's fixed per-device
    scratch (sg_matmul_q8_0_int8_noalloc): no device allocation."""
    _check_dev(dst, x, row_scale)
    _lib.check(ctx.lib.sg_matmul_q8_0_int8_noalloc(ctx.handle, _vp(dst), w.handle, _vp(x), _vp(row_scale),
                                                   x.shape[0], _stream(stream)))


def matmul_q8_0_kernel_us(ctx, dst, w: Q8Weight, x, row_scale, reps: int, stream=None) -> float:
    """Average time of the GEMM kernel alone over `reps` back-to-back launches
    (sg_matmul_q8_0_int8_bench; the operand relayout runs once, untimed)."""
    _check_dev(dst, x, row_scale)
    us = ctypes.c_float()
    _lib.check(ctx.lib.sg_matmul_q8_0_int8_bench(ctx.handle, _vp(dst), w.handle, _vp(x), _vp(row_scale), x.shape[0],
                                                 reps, _stream(stream), ctypes.byref(us)))
    return float(us.value)


def ffn_gate_up(ctx, dst, w_gate: Q8Weight, w_up: Q8Weight, x, row_scale, stream=None):
    """geluquick(x @ w_gate) * (x @ w_up) in one GEMM (model_int8.go:520-535)."""
    _check_dev(dst, x, row_scale)
    _lib.check(ctx.lib.sg_ffn_gate_up(ctx.handle, _vp(dst), w_gate.handle, w_up.handle, _vp(x), _vp(row_scale),
                                      x.shape[0], _stream(stream)))


def block_sums(ctx, out, w: Q8Weight, x, stream=None):
    _check_dev(out, x)
    _lib.check(ctx.lib.sg_q8_block_sums(ctx.handle, _vp(out), w.handle, _vp(x), x.shape[0], _stream(stream)))


def rmsnorm(ctx, dst, src, weight, eps, stream=None):
    _check_dev(dst, src, weight)
    rows, n = src.shape
    _lib.check(ctx.lib.sg_rmsnorm(ctx.handle, _vp(dst), _vp(src), _vp(weight), rows, n, ctypes.c_float(eps),
                                  _stream(stream)))


def qknorm_rope(ctx, q, k, q_norm, k_norm, n_heads, n_kv_heads, head_dim, eps, rope_base, max_seq_len, offsets,
                stream=None):
    _check_dev(q, k)
    off, offp = _off(offsets)
    _lib.check(ctx.lib.sg_qknorm_rope(ctx.handle, _vp(q), q.shape[1], _vp(k), k.shape[1],
                                      _vp(q_norm) if q_norm is not None else None,
                                      _vp(k_norm) if k_norm is not None else None, n_heads, n_kv_heads, head_dim,
                                      ctypes.c_float(eps), ctypes.c_float(rope_base), max_seq_len, offp, len(off) - 1,
                                      _stream(stream)))


def attention(ctx, out, q, k, v, n_heads, n_kv_heads, head_dim, offsets, stream=None):
    _check_dev(out, q, k, v)
    off, offp = _off(offsets)
    _lib.check(ctx.lib.sg_attention(ctx.handle, _vp(out), _vp(q), q.shape[1], _vp(k), _vp(v), k.shape[1], n_heads,
                                    n_kv_heads, head_dim, offp, len(off) - 1, _stream(stream)))


def attention_exact(ctx, out, q, k, v, n_heads, n_kv_heads, head_dim, offsets, stream=None):
    """attention() in the reference's float32 order (sg_attention_exact): bit-identical to it."""
    _check_dev(out, q, k, v)
    off, offp = _off(offsets)
    _lib.check(ctx.lib.sg_attention_exact(ctx.handle, _vp(out), _vp(q), q.shape[1], _vp(k), _vp(v), k.shape[1],
                                          n_heads, n_kv_heads, head_dim, offp, len(off) - 1, _stream(stream)))


def hbm_probe_us(ctx, kind: int, a, b, c, reps: int, stream=None) -> float:
    """sg_hbm_probe: average microseconds per launch of the streaming yardstick
    (kind 0: c = a + b fp32; kind 1: c = int8 codes of a)."""
    _check_dev(a, c)
    us = ctypes.c_float()
    _lib.check(ctx.lib.sg_hbm_probe(ctx.handle, kind, _vp(a), _vp(b) if b is not None else None, _vp(c),
                                    a.numel(), reps, _stream(stream), ctypes.byref(us)))
    return us.value


def issue_probe(ctx, kind: int, waves_per_simd: int, iters: int = 20000, stream=None):
    """sg_issue_probe: SIMD cycles per 32x32 subtile and K-block of the GEMM's
    arithmetic with no memory traffic (kind 0: MFMA + block-serial update;
    1: the VALU part; 2: the MFMA), and the shader clock in GHz."""
    cyc, ghz = ctypes.c_float(), ctypes.c_float()
    _lib.check(ctx.lib.sg_issue_probe(ctx.handle, kind, waves_per_simd, iters, _stream(stream), ctypes.byref(cyc),
                                      ctypes.byref(ghz)))
    return cyc.value, ghz.value


def gelu_quick_mul(ctx, dst, gate, up, stream=None):
    _check_dev(dst, gate, up)
    rows, cols = gate.shape
    _lib.check(ctx.lib.sg_gelu_quick_mul(ctx.handle, _vp(dst), dst.shape[1], _vp(gate), gate.shape[1], _vp(up),
                                         up.shape[1], rows, cols, _stream(stream)))


def embed_tokens(model, dst, tokens, stream=None):
    _check_dev(dst, tokens)
    _lib.check(model.lib.sg_embed_tokens(model.handle, _vp(dst), _vp(tokens), tokens.shape[0], _stream(stream)))


def pool_l2(ctx, out, x, out_dim, offsets, stream=None):
    _check_dev(out, x)
    off, offp = _off(offsets)
    _lib.check(ctx.lib.sg_pool_l2(ctx.handle, _vp(out), _vp(x), x.shape[1], out_dim, offp, len(off) - 1,
                                  _stream(stream)))


# The checks below are on the path of every call, which for a short query takes the
# GPU no longer than it takes Python: they read each property once and tell what is
# wrong only when something is.
_TORCH = None
_DTYPES = {}


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch
        _DTYPES.update({torch.float32: _lib.SG_F32, torch.float16: _lib.SG_F16, torch.bfloat16: _lib.SG_BF16})
        _TORCH = torch
    return _TORCH


def _dtype(t):
    _torch()
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"{t.dtype}: float32, float16 or bfloat16 is needed")
    return d


def _rows_of(ctx, name, t, rows, cols, dtype):
    """The pointer and row stride of a [rows][cols] tensor whose rows are contiguous."""
    if t.get_device() != ctx.device:
        raise ValueError(f"{name} must lie on the context's device")
    if t.dtype != dtype:
        raise ValueError(f"{name}: {t.dtype} beside {dtype}")
    if t.shape != (rows, cols):
        raise ValueError(f"{name}: shape {tuple(t.shape)} where ({rows}, {cols}) is needed")
    ld, inner = t.stride()
    if inner != 1 and cols > 1:
        raise ValueError(f"{name}: its rows must be contiguous")
    if rows <= 1:  # a single row's stride means nothing: whole 16 bytes
        size = t.element_size()
        ld = -(-cols * size // 16) * 16 // size
    return t.data_ptr(), ld


def _vec(ctx, name, t, n, dtype):
    """The pointer of an optional contiguous array of n values; n None: any number."""
    if t is None:
        return None
    if t.get_device() != ctx.device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous on the context's device")
    if t.dtype != dtype or (n is not None and t.numel() != n):
        raise ValueError(f"{name}: {n if n is not None else 'any number of'} values of {dtype} are needed")
    return t.data_ptr()


_MOST = 2**31 - 1  # what the C ABI's counts hold; ctypes would drop the bits above


def _too_many(what, n):
    raise ValueError(f"{what}: {n} are more than a call takes")


def _offsets(ctx, t):
    """The pointer of the CSR offsets and the number of sequences."""
    if t.numel() > _MOST:
        _too_many("offsets", t.numel())
    return _vec(ctx, "offsets", t, None, _torch().int32), t.numel() - 1


def _stream_of(ctx, stream):
    if stream is not None:
        return stream
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # current_stream() builds an object: 1 us
    return raw(ctx.device) if raw else torch.cuda.current_stream(ctx.device).cuda_stream


def attention_masked(ctx, out, q, k, v, n_heads, n_kv_heads, offsets, *, scale=0.0, softcap=0.0, slopes=None,
                     doc_ids=None, causal=False, prefix=None, window=0, stream=None):
    """Attention of every sequence with itself, scores capped, biased or masked (sg_attention_masked).

    q, out [rows, n_heads * hd], k, v [rows, n_kv_heads * hd]; offsets int32 [n_seq + 1];
    slopes float32 [n_heads]; doc_ids int32 [rows]; prefix int32 [n_seq]."""
    torch = _torch()
    rows, qd = q.shape
    if rows > _MOST or qd > _MOST:
        _too_many("rows or columns of q", max(rows, qd))
    hd = qd // max(n_heads, 1)
    if hd * n_heads != qd:
        raise ValueError(f"q: {qd} columns for {n_heads} heads")
    dtype = q.dtype
    qp, ldq = _rows_of(ctx, "q", q, rows, qd, dtype)
    o, ldo = _rows_of(ctx, "out", out, rows, qd, dtype)
    kp, ldk = _rows_of(ctx, "k", k, rows, n_kv_heads * hd, dtype)
    vp, ldv = _rows_of(ctx, "v", v, rows, n_kv_heads * hd, dtype)
    off, n_seq = _offsets(ctx, offsets)
    mask = _lib.AttnMask(scale, softcap, _vec(ctx, "slopes", slopes, n_heads, torch.float32),
                         _vec(ctx, "doc_ids", doc_ids, rows, torch.int32),
                         _vec(ctx, "prefix", prefix, n_seq, torch.int32), causal, max(-1, min(window, _MOST)))
    _lib.check(ctx.lib.sg_attention_masked(ctx.handle, o, ldo, qp, ldq, kp, ldk, vp, ldv, _dtype(q), n_heads, n_kv_heads,
                                           hd, rows, off, n_seq, mask, _stream_of(ctx, stream)))


def block_norm(ctx, xn, sum, x, h, w_post, w_pre, eps, *, gate=None, scale=1.0, offsets=None, stream=None):
    """Post-norm of x, gate and scale, residual addition to h, next pre-norm (sg_block_norm).

    sum, xn, x, h [rows, cols]; w_post (or None), w_pre (None with xn None), float32 [cols];
    gate float32 [cols], or [n_seq, cols] with offsets."""
    f32 = _torch().float32
    rows, cols = x.shape
    if rows > _MOST or cols > _MOST:
        _too_many("rows or columns of x", max(rows, cols))
    dtype = x.dtype
    xp, ldx = _rows_of(ctx, "x", x, rows, cols, dtype)
    hp, ldh = _rows_of(ctx, "h", h, rows, cols, dtype)
    s, lds = _rows_of(ctx, "sum", sum, rows, cols, dtype)
    n, ldn = _rows_of(ctx, "xn", xn, rows, cols, dtype) if xn is not None else (None, 0)
    off, n_seq = _offsets(ctx, offsets) if offsets is not None else (None, 0)
    _lib.check(ctx.lib.sg_block_norm(ctx.handle, n, ldn, s, lds, xp, ldx, hp, ldh, _dtype(x), rows, cols,
                                     _vec(ctx, "w_post", w_post, cols, f32), _vec(ctx, "w_pre", w_pre, cols, f32), eps,
                                     _vec(ctx, "gate", gate, cols if offsets is None else cols * n_seq, f32), scale, off,
                                     n_seq, _stream_of(ctx, stream)))


_COLLECTED = collections.deque()  # handles of banks, caches, and how they are freed


def _free_collected():
    while _COLLECTED:
        try:
            free, handle = _COLLECTED.popleft()
        except IndexError:  # another thread's
            return
        free(handle)


class AdapterBank:
    """Low-rank adapters of one projection (sg_adapter_bank_create): a [n, rank, in_dim]
    and b [n, out_dim, rank] device tensors, scales float32 [n].

    Making and closing a bank wait for the device and are not for a time when any thread
    captures a graph.  A bank that is dropped may be collected at such a time, so its memory
    is kept until the next one is made or closed; close() frees it at once."""

    def __init__(self, ctx, a, b, scales, stream=None):
        self.handle = None
        n, rank, in_dim = a.shape
        if b.dim() != 3 or b.shape[0] != n or b.shape[2] != rank:
            raise ValueError(f"b: shape {tuple(b.shape)} beside a's {tuple(a.shape)}")
        if max(*a.shape, *b.shape) > _MOST:
            _too_many("a or b", max(*a.shape, *b.shape))
        self.ctx, self.lib, self.dtype = ctx, ctx.lib, a.dtype
        self.n, self.rank, self.in_dim, self.out_dim = n, rank, in_dim, b.shape[1]
        _free_collected()
        h = ctypes.c_void_p()
        _lib.check(self.lib.sg_adapter_bank_create(
            ctx.handle, _vec(ctx, "a", a, None, a.dtype), _vec(ctx, "b", b, None, a.dtype),
            _vec(ctx, "scales", scales, n, _torch().float32), _dtype(a), n, rank, in_dim, self.out_dim,
            _stream_of(ctx, stream), ctypes.byref(h)))
        self.handle = h

    def work_bytes(self, rows):
        """Bytes of `work` that adapters_apply needs for `rows` rows or fewer."""
        if rows > _MOST:
            _too_many("rows", rows)
        size = ctypes.c_size_t()
        _lib.check(self.lib.sg_adapters_work_bytes(self.handle, rows, ctypes.byref(size)))
        return size.value

    def close(self):
        _free_collected()
        if self.handle:
            self.lib.sg_adapter_bank_free(self.handle)
            self.handle = None

    def __del__(self):
        if self.handle and _COLLECTED is not None:  # (None: the interpreter ends)
            _COLLECTED.append((self.lib.sg_adapter_bank_free, self.handle))


def _workspace(size, like, stream):
    """`size` bytes from torch's allocator, of the stream that will use them."""
    torch = _torch()
    if stream is None:
        return torch.empty(size, dtype=torch.uint8, device=like.device)
    # Of that stream: what the current one gave back, its work may still write.
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=like.device)):
        return torch.empty(size, dtype=torch.uint8, device=like.device)


def adapters_apply(ctx, dst, base, bank: AdapterBank, x, offsets, adapter_ids, *, work=None, stream=None):
    """dst = base + each row's adapter applied to x (sg_adapters_apply).

    x [rows, in_dim], base and dst [rows, out_dim] (dst may be base); adapter_ids int32
    [n_seq], -1 for none.  work: a uint8 device tensor of bank.work_bytes(rows) at least,
    not shared by calls that may run at the same time; None: one from torch's allocator."""
    torch = _torch()
    rows = x.shape[0]
    if rows > _MOST:
        _too_many("rows of x", rows)
    xp, ldx = _rows_of(ctx, "x", x, rows, bank.in_dim, bank.dtype)
    d, ldd = _rows_of(ctx, "dst", dst, rows, bank.out_dim, bank.dtype)
    b, ldb = _rows_of(ctx, "base", base, rows, bank.out_dim, bank.dtype)
    off, n_seq = _offsets(ctx, offsets)
    if work is None:
        work = _workspace(max(bank.work_bytes(rows), 16), x, stream)
    _lib.check(ctx.lib.sg_adapters_apply(ctx.handle, d, ldd, b, ldb, bank.handle, xp, ldx, rows, off, n_seq,
                                         _vec(ctx, "adapter_ids", adapter_ids, n_seq, torch.int32),
                                         _vec(ctx, "work", work, None, torch.uint8), work.numel(),
                                         _stream_of(ctx, stream)))


class KVCache:
    """Keys and values of `slots` tokens kept on the GPU (sg_kv_cache_create), n_kv_heads heads
    of head_dim; dtype: of rows in and out and of queries.  bits 8: codes and a scale for each
    token and head; bits 0: the values themselves.

    Made and closed as an AdapterBank is: neither is for a time when any thread captures a graph."""

    def __init__(self, ctx, slots, n_kv_heads, head_dim, dtype, bits=8, stream=None):
        self.handle = None
        _torch()
        if dtype not in _DTYPES:
            raise ValueError(f"{dtype}: float32, float16 or bfloat16 is needed")
        if max(slots, n_kv_heads, head_dim) > _MOST:
            _too_many("slots, heads or dims", max(slots, n_kv_heads, head_dim))
        self.ctx, self.lib, self.dtype, self.bits = ctx, ctx.lib, dtype, bits
        self.slots, self.n_kv_heads, self.head_dim = slots, n_kv_heads, head_dim
        _free_collected()
        h = ctypes.c_void_p()
        _lib.check(self.lib.sg_kv_cache_create(ctx.handle, slots, n_kv_heads, head_dim, _DTYPES[dtype], bits,
                                               _stream_of(ctx, stream), ctypes.byref(h)))
        self.handle = h

    @property
    def nbytes(self):
        """Bytes of device memory that it holds."""
        size = ctypes.c_size_t()
        _lib.check(self.lib.sg_kv_cache_bytes(self.handle, ctypes.byref(size)))
        return size.value

    def work_bytes(self, n_heads, rows, n_seq, n_prefix):
        """Bytes of `work` that attention_shared needs for so many rows, sequences and prefixes or fewer."""
        if max(n_heads, rows, n_seq, n_prefix) > _MOST:
            _too_many("heads, rows, sequences or prefixes", max(n_heads, rows, n_seq, n_prefix))
        size = ctypes.c_size_t()
        _lib.check(self.lib.sg_attention_shared_work_bytes(self.handle, n_heads, rows, n_seq, n_prefix,
                                                           ctypes.byref(size)))
        return size.value

    def close(self):
        _free_collected()
        if self.handle:
            self.lib.sg_kv_cache_free(self.handle)
            self.handle = None

    def __del__(self):
        if self.handle and _COLLECTED is not None:  # (None: the interpreter ends)
            _COLLECTED.append((self.lib.sg_kv_cache_free, self.handle))


def _kv_rows(call, ctx, cache, k, v, offsets, starts, stream):
    rows, cols = k.shape[0], cache.n_kv_heads * cache.head_dim
    if rows > _MOST:
        _too_many("rows of k", rows)
    kp, ldk = _rows_of(ctx, "k", k, rows, cols, cache.dtype)
    vp, ldv = _rows_of(ctx, "v", v, rows, cols, cache.dtype)
    off, n_seq = _offsets(ctx, offsets)
    st = _vec(ctx, "starts", starts, n_seq, _torch().int32)
    _lib.check(call(ctx.handle, cache.handle, kp, ldk, vp, ldv, rows, off, n_seq, st, _stream_of(ctx, stream)))


def kv_cache_write(ctx, cache: KVCache, k, v, offsets, starts, *, stream=None):
    """Rows of k and v [rows, n_kv_heads * head_dim] into the cache (sg_kv_cache_write): those of
    sequence i, offsets[i] .. offsets[i + 1], go to the slots from starts[i] (int32 [n_seq]) on."""
    _kv_rows(ctx.lib.sg_kv_cache_write, ctx, cache, k, v, offsets, starts, stream)


def kv_cache_read(ctx, k, v, cache: KVCache, offsets, starts, *, stream=None):
    """The cache's rows back into k and v (sg_kv_cache_read), as kv_cache_write places them."""
    _kv_rows(ctx.lib.sg_kv_cache_read, ctx, cache, k, v, offsets, starts, stream)


def attention_shared(ctx, out, q, cache: KVCache, n_heads, offsets, starts, lengths, shared=None, prefix_starts=None,
                     prefix_lengths=None, *, scale=0.0, softcap=0.0, causal=True, window=0, work=None, stream=None):
    """Attention of a batch's queries over kept keys, long prefixes read once for all the
    sequences that share them (sg_attention_shared).

    q, out [rows, n_heads * head_dim]; offsets int32 [n_seq + 1].  Sequence i's own keys, its
    queries' tokens last, are slots starts[i] .. starts[i] + lengths[i]; sequences shared[p] ..
    shared[p + 1] stand behind prefix p, slots prefix_starts[p] .. prefix_starts[p] +
    prefix_lengths[p] (all int32 device tensors; shared None: no prefixes).  work: a uint8
    device tensor of cache.work_bytes(...) at least, not shared by calls that may run at the
    same time; None: one from torch's allocator."""
    torch = _torch()
    i32 = torch.int32
    rows, cols = q.shape[0], n_heads * cache.head_dim
    if rows > _MOST or n_heads > _MOST:
        _too_many("rows or heads of q", max(rows, n_heads))
    qp, ldq = _rows_of(ctx, "q", q, rows, cols, cache.dtype)
    o, ldo = _rows_of(ctx, "out", out, rows, cols, cache.dtype)
    off, n_seq = _offsets(ctx, offsets)
    n_prefix = 0
    if shared is not None:
        if shared.numel() > _MOST:
            _too_many("shared", shared.numel())
        n_prefix = shared.numel() - 1
        if n_prefix < 0 or prefix_starts is None or prefix_lengths is None:
            raise ValueError("shared: [n_prefix + 1] offsets, with prefix_starts and prefix_lengths")
    keys = _lib.SharedKeys(_vec(ctx, "starts", starts, n_seq, i32), _vec(ctx, "lengths", lengths, n_seq, i32),
                           _vec(ctx, "shared", shared, None, i32), _vec(ctx, "prefix_starts", prefix_starts, n_prefix, i32),
                           _vec(ctx, "prefix_lengths", prefix_lengths, n_prefix, i32), n_prefix, scale, softcap, causal,
                           max(-1, min(window, _MOST)))
    if work is None:
        work = _workspace(max(cache.work_bytes(n_heads, rows, max(n_seq, 0), n_prefix), 16), q, stream)
    _lib.check(ctx.lib.sg_attention_shared(ctx.handle, o, ldo, qp, ldq, cache.handle, n_heads, rows, off, n_seq, keys,
                                           _vec(ctx, "work", work, None, torch.uint8), work.numel(),
                                           _stream_of(ctx, stream)))


class Q4Weight:
    """A matrix of 4-bit weights with group scales (sg_q4_weight_create): w = scale * (code - zero).

    codes uint8 [out_dim, in_dim / 2], the even input in a byte's lower four bits; scales
    [out_dim, in_dim / group] float16 (kept so) or float32 or bfloat16 (kept as float32); zeros
    uint8 [out_dim, in_dim / group] or None for 8; device tensors.  group: 32, 64 or 128.

    Made and closed as an AdapterBank is: neither is for a time when any thread captures a graph."""

    def __init__(self, ctx, codes, scales, zeros=None, stream=None):
        self.handle = None
        torch = _torch()
        out_dim, half = codes.shape
        groups = scales.shape[1] if scales.dim() == 2 else 0
        if groups <= 0 or 2 * half % groups:
            raise ValueError(f"scales: shape {tuple(scales.shape)} beside codes {tuple(codes.shape)}")
        if max(out_dim, 2 * half) > _MOST:
            _too_many("rows or columns of codes", max(out_dim, 2 * half))
        h = ctypes.c_void_p()
        args = (_vec(ctx, "codes", codes, None, torch.uint8), _vec(ctx, "scales", scales, out_dim * groups, scales.dtype),
                _dtype(scales), _vec(ctx, "zeros", zeros, out_dim * groups, torch.uint8))
        _free_collected()
        _lib.check(ctx.lib.sg_q4_weight_create(ctx.handle, *args, out_dim, 2 * half, 2 * half // groups,
                                               _stream_of(ctx, stream), ctypes.byref(h)))
        self.ctx, self.lib, self.handle = ctx, ctx.lib, h
        self.out_dim, self.in_dim, self.group = out_dim, 2 * half, 2 * half // groups

    @classmethod
    def from_q4_0(cls, ctx, raw_q4: np.ndarray, out_dim: int, in_dim: int):
        """From GGUF's raw Q4_0 blocks [out_dim][in_dim/32][18 B] (sg_q4_weight_create_q4_0)."""
        raw = np.ascontiguousarray(raw_q4, np.uint8)
        if raw.size != out_dim * (in_dim // 32) * 18:
            raise ValueError("raw Q4_0 size does not match out_dim x in_dim")
        self = cls.__new__(cls)
        self.handle = None
        h = ctypes.c_void_p()
        _free_collected()
        _lib.check(ctx.lib.sg_q4_weight_create_q4_0(ctx.handle, ctypes.c_void_p(raw.ctypes.data), out_dim, in_dim,
                                                    ctypes.byref(h)))
        self.ctx, self.lib, self.handle = ctx, ctx.lib, h
        self.out_dim, self.in_dim, self.group = out_dim, in_dim, 32
        return self

    def close(self):
        _free_collected()
        if self.handle:
            self.lib.sg_q4_weight_free(self.handle)
            self.handle = None

    def __del__(self):
        if self.handle and _COLLECTED is not None:  # (None: the interpreter ends)
            _COLLECTED.append((self.lib.sg_q4_weight_free, self.handle))


def matmul_q4(ctx, dst, w: Q4Weight, x, *, stream=None):
    """dst = x @ w^T for a few rows (sg_matmul_q4): x [rows, in_dim], dst [rows, out_dim]."""
    rows = x.shape[0]
    if rows > _MOST:
        _too_many("rows of x", rows)
    xp, ldx = _rows_of(ctx, "x", x, rows, w.in_dim, x.dtype)
    d, ldd = _rows_of(ctx, "dst", dst, rows, w.out_dim, x.dtype)
    _lib.check(ctx.lib.sg_matmul_q4(ctx.handle, d, ldd, w.handle, xp, ldx, _dtype(x), rows, _stream_of(ctx, stream)))
