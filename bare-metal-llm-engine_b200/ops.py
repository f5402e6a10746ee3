"""Torch-tensor front end of the hot path.

Tensors supply device memory and the current CUDA stream; every computation is
a call into libengine_b200.so.  Inputs must be contiguous CUDA tensors of the
stated dtype (checked here, loudly); outputs are allocated when not given.
"""
from __future__ import annotations

import ctypes

import torch

from . import KvPages as _KvPages
from . import cuda as _c


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _req(t: torch.Tensor, dtype: torch.dtype, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the library has no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous (row-major)")
    return t


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def matmul_f32(A, B, out=None, variant: str = "register_tiled"):
    """C = A @ B, FP32 [M,K] x [K,N] (engine::cuda::matmul_<variant>)."""
    _req(A, torch.float32, "A")
    _req(B, torch.float32, "B")
    M, K = A.shape
    N = B.shape[1]
    C = out if out is not None else torch.empty(M, N, device=A.device, dtype=torch.float32)
    fn = {"naive": _c.matmul_naive, "tiled": _c.matmul_tiled,
          "register_tiled": _c.matmul_register_tiled}[variant]
    fn(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, _stream())
    return C


def matmul(A, B, out=None):
    """C = A @ B with FP16 or BF16 A[M,K], B[K,N] on tcgen05 tensor cores."""
    bf16 = A.dtype == torch.bfloat16
    dt = torch.bfloat16 if bf16 else torch.float16
    _req(A, dt, "A")
    _req(B, dt, "B")
    M, K = A.shape
    N = B.shape[1]
    C = out if out is not None else torch.empty(M, N, device=A.device, dtype=dt)
    (_c.matmul_bf16 if bf16 else _c.matmul_f16)(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K,
                                                _stream())
    return C


def linear(X, W, residual=None, out=None):
    """Y = X @ W^T (+ residual) with W stored [N,K]; FP16 or BF16."""
    bf16 = X.dtype == torch.bfloat16
    dt = torch.bfloat16 if bf16 else torch.float16
    _req(X, dt, "X")
    _req(W, dt, "W")
    if residual is not None:
        _req(residual, dt, "residual")
    M, K = X.shape
    N = W.shape[0]
    Y = out if out is not None else torch.empty(M, N, device=X.device, dtype=dt)
    (_c.linear_bf16 if bf16 else _c.linear_f16)(X.data_ptr(), W.data_ptr(), _ptr(residual),
                                                Y.data_ptr(), M, N, K, _stream())
    return Y


def gemv(W, x, residual=None, out=None):
    """y = W[N,K] @ x[K] (+ residual), FP16 decode GEMV."""
    _req(W, torch.float16, "W")
    _req(x, torch.float16, "x")
    N, K = W.shape
    y = out if out is not None else torch.empty(N, device=W.device, dtype=torch.float16)
    _c.gemv_f16_nk(W.data_ptr(), x.data_ptr(), _ptr(residual), y.data_ptr(), N, K, _stream())
    return y


def rmsnorm_linear(x, gamma, W, eps: float = 1e-5, residual=None, out=None):
    """Y = rmsnorm(x; gamma, eps) @ W^T (+ residual), FP16, W stored [N,K]."""
    _req(x, torch.float16, "x")
    _req(W, torch.float16, "W")
    if gamma is not None:
        _req(gamma, torch.float16, "gamma")
    if residual is not None:
        _req(residual, torch.float16, "residual")
    M, K = x.shape
    N = W.shape[0]
    Y = out if out is not None else torch.empty(M, N, device=x.device, dtype=torch.float16)
    _c.rmsnorm_linear_f16(x.data_ptr(), _ptr(gamma), W.data_ptr(), _ptr(residual), Y.data_ptr(),
                          M, N, K, eps, _stream())
    return Y


def rmsnorm_linear_kv(x, gamma, W, eps, k_cache, v_cache, kv_row0: int, pos: int, out=None):
    """Batch-1 rmsnorm_linear (x [1, K]) whose output rows [kv_row0, kv_row0 + H_kv*d)
    and the next H_kv*d rows (the token's K and V) are also stored at position pos
    of the head-major caches [H_kv, max_len, d], in the same kernel."""
    _req(x, torch.float16, "x")
    _req(W, torch.float16, "W")
    if gamma is not None:
        _req(gamma, torch.float16, "gamma")
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous():
            raise TypeError(f"{n} must be a contiguous CUDA float16 tensor [H_kv, max_len, d]")
    M, K = x.shape
    if M != 1:
        raise ValueError("rmsnorm_linear_kv: one token (x [1, K])")
    N = W.shape[0]
    hk, max_len, d = k_cache.shape
    Y = out if out is not None else torch.empty(1, N, device=x.device, dtype=torch.float16)
    _c.rmsnorm_linear_kv_f16(x.data_ptr(), _ptr(gamma), W.data_ptr(), 0, Y.data_ptr(), N, K, eps,
                             k_cache.data_ptr(), v_cache.data_ptr(), kv_row0, hk, d, max_len, pos,
                             _stream())
    return Y


def rmsnorm_linear_swiglu(x, gamma, W_gu, eps: float = 1e-5, out=None):
    """swiglu(g, u) with [g | u] = rmsnorm(x; gamma, eps) @ W_gu^T, W_gu [2F,K] = gate
    rows then up rows; FP16.  Same result as rmsnorm_linear followed by swiglu."""
    _req(x, torch.float16, "x")
    _req(W_gu, torch.float16, "W_gu")
    if gamma is not None:
        _req(gamma, torch.float16, "gamma")
    M, K = x.shape
    F = W_gu.shape[0] // 2
    Y = out if out is not None else torch.empty(M, F, device=x.device, dtype=torch.float16)
    _c.rmsnorm_linear_swiglu_f16(x.data_ptr(), _ptr(gamma), W_gu.data_ptr(), Y.data_ptr(), M, F,
                                 K, eps, _stream())
    return Y


def quant_repack(qtype, blocks, N, K):
    """Packed GGUF blocks (uint8 CUDA tensor) -> (payload, scales) in the layout
    gemv_q streams: payload [N, K] int8 (Q8_0) or [N, K/2] uint8 (Q4_0, each
    block's 16 nibble bytes in GGUF order), scales [N, K/32] FP16."""
    _req(blocks, torch.uint8, "blocks")
    pay = K if qtype == _c.Q8_0 else K // 2
    q = torch.empty(N, pay, device=blocks.device, dtype=torch.uint8)
    d = torch.empty(N, K // 32, device=blocks.device, dtype=torch.float16)
    _c.quant_repack(qtype, blocks.data_ptr(), q.data_ptr(), d.data_ptr(), N, K, _stream())
    return q, d


def gemv_q(qtype, q, scales, x, residual=None, out=None):
    """y = W x (+ residual) for W given by quant_repack's (payload, scales)."""
    _req(q, torch.uint8, "q")
    _req(scales, torch.float16, "scales")
    _req(x, torch.float16, "x")
    N, K = scales.shape[0], x.numel()
    y = out if out is not None else torch.empty(N, device=x.device, dtype=torch.float16)
    _c.gemv_q_nk(qtype, q.data_ptr(), scales.data_ptr(), x.data_ptr(), _ptr(residual),
                 y.data_ptr(), N, K, _stream())
    return y


def residual_rmsnorm(x, residual, weight=None, eps: float = 1e-5):
    """(norm_out, sum_out): sum_out = x + residual, norm_out = rmsnorm(sum_out) *
    weight, FP32 [rows, cols] (engine::cuda::residual_rmsnorm)."""
    _req(x, torch.float32, "x")
    _req(residual, torch.float32, "residual")
    if weight is not None:
        _req(weight, torch.float32, "weight")
    rows, cols = x.shape
    norm = torch.empty_like(x)
    sm = torch.empty_like(x)
    _c.residual_rmsnorm(x.data_ptr(), residual.data_ptr(), _ptr(weight), norm.data_ptr(),
                        sm.data_ptr(), rows, cols, eps, _stream())
    return norm, sm


def attention(q, k, v, scale=None, q_pos_offset: int = 0, is_causal: bool = True,
              want_lse: bool = False):
    """out [s_q, H, d] (FP16) of q [s_q, H, d] over k / v [H_kv, s_kv, d]
    (engine::cuda::attention_prefill); with want_lse also lse [s_q, H] (FP32)."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _req(t, torch.float16, n)
    s_q, H, d = q.shape
    H_kv, s_kv, _ = k.shape
    scale = d ** -0.5 if scale is None else scale
    out = torch.empty_like(q)
    lse = torch.empty(s_q, H, device=q.device, dtype=torch.float32) if want_lse else None
    _c.attention_prefill(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), s_q, s_kv, H,
                         H_kv, d, s_kv * d, scale, q_pos_offset, is_causal, _ptr(lse), _stream())
    return (out, lse) if want_lse else out


def attention_decode(q, k, v, scale=None, split_kv: int = 0):
    """out [H, d] of one query row q [H, d] over all kv_len keys of k / v
    [H_kv, kv_len, d] (engine::cuda::attention_decode, split-KV)."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _req(t, torch.float16, n)
    H, d = q.shape
    H_kv, kv_len, _ = k.shape
    scale = d ** -0.5 if scale is None else scale
    out = torch.empty_like(q)
    _c.attention_decode(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), kv_len, H, H_kv,
                        d, kv_len * d, scale, split_kv, _stream())
    return out


def kv_cache_write(k_rows, v_rows, k_cache, v_cache, pos: int, n_seq: int = 1):
    """Scatters K / V rows into head-major caches [n_seq * H_kv, max_len, d] at
    positions pos.. (engine::cuda::detail::kv_cache_write, batched over n_seq
    sequences).  k_rows / v_rows are [n_seq * s_new, H_kv * d] views whose rows
    may be strided (e.g. the K and V columns of a fused Q/K/V projection)."""
    for t, n in ((k_rows, "k_rows"), (v_rows, "v_rows"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dtype != torch.float16 or not t.is_cuda:
            raise TypeError(f"{n} must be a CUDA float16 tensor")
    if k_rows.stride(1) != 1 or v_rows.stride(1) != 1 or k_rows.stride(0) != v_rows.stride(0):
        raise ValueError("k_rows / v_rows: rows must be contiguous and share one pitch")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("caches must be contiguous [n_seq * H_kv, max_len, d]")
    hk, max_len, d = k_cache.shape
    H_kv = hk // n_seq
    s_new = k_rows.shape[0] // n_seq
    if k_rows.shape[1] != H_kv * d:
        raise ValueError("k_rows: width != H_kv * d")
    _c.kv_cache_write_rows(k_rows.data_ptr(), v_rows.data_ptr(), k_rows.stride(0), k_cache.data_ptr(),
                           v_cache.data_ptr(), n_seq, s_new, H_kv, d, pos, max_len, _stream())


def attention_cached(q, k_cache, v_cache, kv_len: int, q_pos_offset: int, is_causal: bool = True,
                     scale=None, out=None):
    """attention_prefill of q [s_q, H, d] over the first kv_len positions of the
    caches [H_kv, max_len, d] (kv_head_stride = max_len * d)."""
    _req(q, torch.float16, "q")
    s_q, H, d = q.shape
    H_kv, max_len, _ = k_cache.shape
    scale = d ** -0.5 if scale is None else scale
    o = out if out is not None else torch.empty_like(q)
    _c.attention_prefill(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(), s_q,
                         kv_len, H, H_kv, d, max_len * d, scale, q_pos_offset, is_causal, 0,
                         _stream())
    return o


def attention_decode_cached(q, k_cache, v_cache, kv_len: int, scale=None, out=None):
    """attention_decode of one query row per head, q [H, d], over the first
    kv_len positions of the caches [H_kv, max_len, d]; a batch of equal-length
    sequences is q [B * H, d] over caches [B * H_kv, max_len, d]."""
    _req(q, torch.float16, "q")
    H, d = q.shape
    H_kv, max_len, _ = k_cache.shape
    scale = d ** -0.5 if scale is None else scale
    o = out if out is not None else torch.empty_like(q)
    _c.attention_decode(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(), kv_len,
                        H, H_kv, d, max_len * d, scale, 0, _stream())
    return o


class PagedKV:
    """An 8-bit paged KV cache (engine_kv_pages_t): the tensors, and the handle that
    the kv_pages_* and attention_paged_* calls take.

    k, v              [n_layers, n_pages, H_kv, page, d] int8 or float8_e4m3fn codes
    k_scale, v_scale  [n_layers, n_pages, H_kv] float32; value = scale * code
    table             [n_slots, max_pages] int32, a slot's pages by position (-1: none)
    length            [n_slots] int32, tokens of each slot
    ref               [n_pages] int32, slots that use a page (0: free)

    The tensors stay the caller's and may be read at any time; the kernels keep
    table, length and ref, so they are not to be replaced by others afterwards."""

    def __init__(self, k, v, k_scale, v_scale, table, length, ref):
        if k.dtype not in (torch.int8, torch.float8_e4m3fn):
            raise TypeError(f"k must be int8 or float8_e4m3fn, got {k.dtype}")
        if k.dim() != 5 or v.shape != k.shape:
            raise ValueError("k and v must be [n_layers, n_pages, H_kv, page, d], of one shape")
        n_layers, n_pages, hk, page, d = k.shape
        for t, dt, shape, n in ((k, k.dtype, k.shape, "k"), (v, k.dtype, k.shape, "v"),
                                (k_scale, torch.float32, k.shape[:3], "k_scale"),
                                (v_scale, torch.float32, k.shape[:3], "v_scale"),
                                (table, torch.int32, None, "table"),
                                (length, torch.int32, table.shape[:1], "length"),
                                (ref, torch.int32, k.shape[1:2], "ref")):
            _req(t, dt, n)
            if shape is not None and t.shape != shape:
                raise ValueError(f"{n} must be {tuple(shape)}, got {tuple(t.shape)}")
            if t.device != k.device:
                raise ValueError(f"{n} must be on {k.device}")
        if table.dim() != 2:
            raise ValueError("table must be [n_slots, max_pages]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.table, self.length, self.ref = table, length, ref
        self.n_slots, self.max_pages = table.shape
        self.n_kv_heads, self.head_dim, self.n_pages = hk, d, n_pages
        self.width = hk * d
        self.device_index = k.device.index
        self.desc = _KvPages(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                             table.data_ptr(), length.data_ptr(), ref.data_ptr(), n_layers, n_pages,
                             hk, page, d, self.n_slots, self.max_pages,
                             _c.KV_I8 if k.dtype == torch.int8 else _c.KV_E4M3)
        self.handle = ctypes.addressof(self.desc)

    @classmethod
    def empty(cls, n_layers, n_pages, n_kv_heads, page_size, head_dim, n_slots, max_pages,
              dtype=torch.int8, device="cuda"):
        """A new cache without sequences."""
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        z = dict(device=device, dtype=torch.int32)
        return cls(torch.empty(shape, device=device, dtype=dtype),
                   torch.empty(shape, device=device, dtype=dtype),
                   torch.zeros(shape[:3], device=device), torch.zeros(shape[:3], device=device),
                   torch.full((n_slots, max_pages), -1, **z), torch.zeros(n_slots, **z),
                   torch.zeros(n_pages, **z))


def _kv_stream(kv) -> int:
    """The current stream of the cache's device, which has to be the current device.  (The raw
    handle: torch.cuda.current_stream() builds an object, 3 us, as long as a small call.)"""
    if kv.device_index != torch._C._cuda_getDevice():
        raise ValueError(f"the cache is on cuda:{kv.device_index}, which is not the current device")
    return torch._C._cuda_getCurrentRawStream(kv.device_index)


def _kv_i32(kv, t, name: str) -> int:
    """Address of an int32 tensor on the cache's device."""
    if type(t) is not torch.Tensor or t.dtype is not torch.int32 or t.get_device() != kv.device_index \
            or not t.is_contiguous():
        _req(t, torch.int32, name)
        if t.get_device() != kv.device_index:
            raise ValueError(f"{name} must be on the cache's device")
    return t.data_ptr()


def _kv_slots(kv, slots, n) -> int:
    """Address of the slots of a call over n entries (None: slots 0 .. n - 1)."""
    if slots is None:
        return 0
    if slots.numel() != n:
        raise ValueError(f"slots must have {n} entries, got {slots.numel()}")
    return _kv_i32(kv, slots, "slots")


def kv_pages_extend(kv, slots, n_new):
    """Adds n_new[i] tokens to slot slots[i] (int32 tensors; slots None: 0, 1, ...),
    taking the pages they need, lowest free id first.  Returns status [1] int32:
    0, or the number of missing pages, or -1 for a bad argument; unless 0, nothing
    changed.  Nothing is synchronised: read the status when it is wanted."""
    st = _kv_stream(kv)
    n = n_new.numel()
    add = _kv_i32(kv, n_new, "n_new")
    status = torch.empty(1, device=n_new.device, dtype=torch.int32)
    _c.kv_pages_extend(kv.handle, _kv_slots(kv, slots, n), add, status.data_ptr(), n, st)
    return status


def kv_pages_fork(kv, parents, children):
    """Makes the empty slots children[i] copies of parents[i]: full pages shared, the
    partly filled one copied in all layers.  Returns status as kv_pages_extend."""
    st = _kv_stream(kv)
    par, chi = _kv_i32(kv, parents, "parents"), _kv_i32(kv, children, "children")
    n = parents.numel()
    if n != children.numel():
        raise ValueError("parents and children must have as many entries")
    status = torch.empty(1, device=parents.device, dtype=torch.int32)
    _c.kv_pages_fork(kv.handle, par, chi, status.data_ptr(), n, st)
    return status


def kv_pages_free(kv, slots):
    """Empties the slots; pages without a user left are free again."""
    st = _kv_stream(kv)
    _c.kv_pages_free(kv.handle, _kv_i32(kv, slots, "slots"), slots.numel(), st)


def kv_pages_compact(kv):
    """Moves the pages in use to the lowest ids, in all layers; tables and ref follow.
    Returns remap [n_pages] int32: the new id of each page, -1 if it was free."""
    st = _kv_stream(kv)
    remap = torch.empty(kv.n_pages, device=kv.ref.device, dtype=torch.int32)
    _c.kv_pages_compact(kv.handle, remap.data_ptr(), st)
    return remap


def _kv_f16(kv, t, name):
    if t.dtype is not torch.float16 or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA float16 tensor")
    if t.get_device() != kv.device_index:
        raise ValueError(f"{name} must be on the cache's device")


def kv_pages_write(kv, layer: int, k_rows, v_rows, slots=None, cu_new=None, status=None):
    """Stores K / V rows [n_tokens, H_kv * d] (FP16, rows may be strided views, e.g. the
    columns of a fused Q/K/V projection) as the LAST positions of the slots: rows
    [cu_new[i], cu_new[i+1]) of slot slots[i], or one row each where cu_new is None.
    Call kv_pages_extend first: it counts them.  With its `status` given, nothing is written
    unless that is 0 (behind an extend that was refused, the last positions are those of earlier
    rows); a step that does not read it on the host, a captured one, passes it on."""
    st = _kv_stream(kv)
    _kv_f16(kv, k_rows, "k_rows")
    _kv_f16(kv, v_rows, "v_rows")
    shape, stride = k_rows.shape, k_rows.stride()
    if len(shape) != 2 or shape[1] != kv.width:
        raise ValueError("k_rows must be [n_tokens, H_kv * d]")
    n_tokens = shape[0]
    if v_rows.shape != shape or stride[1] != 1 or v_rows.stride(1) != 1 or (n_tokens > 1 and v_rows.stride(0) != stride[0]):
        raise ValueError("k_rows / v_rows: rows must be contiguous, as many, and share one pitch")
    n_seq, cu = n_tokens, 0
    if cu_new is not None:
        n_seq, cu = cu_new.numel() - 1, _kv_i32(kv, cu_new, "cu_new")
    if status is not None and status.numel() != 1:
        raise ValueError("status must be the one word of kv_pages_extend")
    _c.kv_pages_write(kv.handle, layer, k_rows.data_ptr(), v_rows.data_ptr(),
                      stride[0] if n_tokens > 1 else kv.width,
                      _kv_slots(kv, slots, n_seq), cu, n_seq, n_tokens, st,
                      0 if status is None else _kv_i32(kv, status, "status"))


def _paged_q(kv, q, out):
    """Checks q [n, H, d] (heads contiguous, rows may be strided) and out; (n, H, pitch, out)."""
    _kv_f16(kv, q, "q")
    shape, stride = q.shape, q.stride()
    if len(shape) != 3 or shape[2] != kv.head_dim:
        raise ValueError("q must be [n, H, d]")
    n, H, d = shape
    if stride[2] != 1 or (H > 1 and stride[1] != d):
        raise ValueError("q: the heads of a row must be contiguous")
    if out is None:
        out = torch.empty(shape, device=q.device, dtype=torch.float16)
    else:
        _req(out, torch.float16, "out")
        if out.shape != shape or out.get_device() != kv.device_index:
            raise ValueError("out must have q's shape and device")
    return n, H, (stride[0] if n > 1 else H * d), out


def attention_paged_decode(kv, layer: int, q, slots=None, scale=None, out=None,
                           want_lse: bool = False):
    """out [B, H, d] of one query row per sequence, q [B, H, d], over all positions of
    the slots (None: slots 0 .. B - 1); with want_lse also lse [B, H] (FP32)."""
    st = _kv_stream(kv)
    B, H, pitch, o = _paged_q(kv, q, out)
    lse = torch.empty(B, H, device=q.device, dtype=torch.float32) if want_lse else None
    _c.attention_paged_decode(kv.handle, layer, q.data_ptr(), pitch, _kv_slots(kv, slots, B),
                              o.data_ptr(), _ptr(lse), B, H,
                              kv.head_dim ** -0.5 if scale is None else scale, st)
    return (o, lse) if want_lse else o


def attention_paged_prefill(kv, layer: int, q, slots, cu_q, scale=None, out=None,
                            is_causal: bool = True, want_lse: bool = False):
    """out [T, H, d] of the query rows [cu_q[i], cu_q[i+1]) of q [T, H, d], the LAST
    positions of slot slots[i] (None: slot i), over the slot's positions up to their
    own (all of them unless is_causal).  Rows past cu_q[-1] are left as they were in
    `out`.  With want_lse also lse [T, H] (FP32).  Prompts and single rows are faster in two
    calls: the kernel is chosen by the average number of rows."""
    st = _kv_stream(kv)
    T, H, pitch, o = _paged_q(kv, q, out)
    n_seq, cu = cu_q.numel() - 1, _kv_i32(kv, cu_q, "cu_q")
    lse = torch.empty(T, H, device=q.device, dtype=torch.float32) if want_lse else None
    _c.attention_paged_prefill(kv.handle, layer, q.data_ptr(), pitch, _kv_slots(kv, slots, n_seq),
                               cu, o.data_ptr(), _ptr(lse), n_seq, T, H,
                               kv.head_dim ** -0.5 if scale is None else scale, is_causal, st)
    return (o, lse) if want_lse else o


def swiglu(gate, up, out=None):
    _req(gate, torch.float16, "gate")
    _req(up, torch.float16, "up")
    o = out if out is not None else torch.empty_like(gate)
    _c.swiglu_fp16(gate.data_ptr(), up.data_ptr(), o.data_ptr(), gate.numel(), _stream())
    return o


def embedding(table, ids, out=None):
    _req(table, torch.float16, "table")
    _req(ids, torch.int32, "ids")
    V, D = table.shape
    T = ids.numel()
    o = out if out is not None else torch.empty(T, D, device=table.device, dtype=torch.float16)
    _c.embedding_fp16(table.data_ptr(), ids.data_ptr(), o.data_ptr(), T, D, V, _stream())
    return o
