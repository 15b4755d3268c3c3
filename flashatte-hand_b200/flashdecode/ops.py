"""Torch-facing host API of the paged-KV GQA decode operator.

``run_kernel`` mirrors the reference binding ``run_kernel_torch``
(scripts/evaluate_flashattn_submission.py:46-78): same argument names and
order, tensors in, pointers forwarded to the C ABI, nothing returned, and
arguments the operator rejects are ignored silently exactly as the reference
does (``last_error()`` tells why).

``flash_decode`` is the extended call with the ``flash_attn_with_kvcache``
argument vocabulary the reference's evaluator uses for its oracle
(evaluate_flashattn_submission.py:232-247): q, k_cache, v_cache,
cache_seqlens, block_table, softmax_scale, return_softmax_lse.  It runs on
the tensors' device and current stream and raises on any error.
"""
from __future__ import annotations

import contextlib
import math

import torch

from ._lib import (FD_DTYPE_BF16, FD_DTYPE_E2M1, FD_DTYPE_E4M3, FD_DTYPE_FP16, FD_DTYPE_FP32,
                   FlashDecodeError, check, load_library)

_DTYPES = {torch.bfloat16: FD_DTYPE_BF16, torch.float16: FD_DTYPE_FP16}
# the codes' type of 4-bit caches, where torch has it: calls over other caches
# do not need it
_FP4 = getattr(torch, "float4_e2m1fn_x2", None)
_CACHE_DTYPES = {torch.bfloat16: FD_DTYPE_BF16, torch.float16: FD_DTYPE_FP16,
                 torch.float8_e4m3fn: FD_DTYPE_E4M3}
if _FP4 is not None:
    _CACHE_DTYPES[_FP4] = FD_DTYPE_E2M1
_INT32 = torch.int32
_OUT_DTYPES = {torch.bfloat16: FD_DTYPE_BF16, torch.float16: FD_DTYPE_FP16, torch.float32: FD_DTYPE_FP32}


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_handle(stream, dev: torch.device) -> int:
    """cudaStream_t of `stream`, or of the current stream of `dev` (read
    without building a Stream object when torch offers that)."""
    if stream is not None:
        return stream.cuda_stream
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    if _raw_stream is not None:
        return _raw_stream(idx)
    return torch.cuda.current_stream(idx).cuda_stream


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_NO_SWITCH = contextlib.nullcontext()


def _on_device(dev: torch.device):
    """Context that makes `dev` current, or nothing when it already is (the
    device switch costs more than the rest of a small call)."""
    if dev.index is None or dev.index == _current_device():
        return _NO_SWITCH
    return torch.cuda.device(dev)


def _launch(fn, dev: torch.device, stream, args) -> None:
    """fn(*args, stream handle) with `dev` current; raises on a bad status."""
    handle = _stream_handle(stream, dev)
    if dev.index == _current_device():
        status = fn(*args, handle)
    else:
        with torch.cuda.device(dev):
            status = fn(*args, handle)
    if status:
        check(status)


def _new(shape, dtype: torch.dtype, dev: torch.device, stream=None) -> torch.Tensor:
    """An output tensor.  One that a kernel on `stream` writes is allocated
    there: a block of the current stream's pool may still be read by work
    queued on that stream for its last owner.  The current stream, where the
    caller may use and drop it, is recorded."""
    if stream is None or stream.cuda_stream == _stream_handle(None, dev):
        return torch.empty(shape, dtype=dtype, device=dev)
    with _on_stream(stream, dev):
        t = torch.empty(shape, dtype=dtype, device=dev)
    t.record_stream(torch.cuda.current_stream(dev))
    return t


def _on_stream(stream, dev: torch.device):
    """Context that makes `stream` current: torch's, or any object that names a
    stream of `dev` by its cuda_stream."""
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(stream.cuda_stream, device=dev)
    return torch.cuda.stream(stream)


def _require_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("flashdecode runs on CUDA tensors only (no CPU path)")


def _require_device(first, *tensors) -> None:
    """Every tensor of a call (None: not given) lies on one CUDA device: a
    kernel that followed a pointer of another one would fault."""
    index = first.get_device()
    if index < 0:
        raise ValueError("flashdecode runs on CUDA tensors only (no CPU path)")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError("the tensors of a call must lie on one device")


def run_kernel(q, k_cache_paged, v_cache_paged, output, cache_seqlens, block_table, batch_size,
               seqlen_k, seqlen_q, num_heads, num_heads_k, headdim, page_block_size, num_blocks,
               causal) -> None:
    """Reference operator surface: bf16, scale 1/sqrt(headdim), default stream."""
    lib = load_library()
    lib.run_kernel(_ptr(q), _ptr(k_cache_paged), _ptr(v_cache_paged), _ptr(output),
                   _ptr(cache_seqlens), _ptr(block_table), int(batch_size), int(seqlen_k),
                   int(seqlen_q), int(num_heads), int(num_heads_k), int(headdim),
                   int(page_block_size), int(num_blocks), int(causal))


def last_error() -> tuple[int, str]:
    """(status, message) of the last C-ABI call on this thread."""
    lib = load_library()
    return int(lib.fd_last_error()), lib.fd_last_error_message().decode()


def device_status() -> int:
    """Read and clear the device error word of the library-owned workspace."""
    return int(load_library().fd_device_status())


def workspace_size(batch_size: int, num_heads: int, num_heads_k: int, headdim: int = 128,
                   seqlen_q: int = 1, kv_dtype: torch.dtype | None = None) -> int:
    """Bytes of workspace that flash_decode needs (kv_dtype: that of the
    caches, to be given for float4_e2m1fn_x2)."""
    lib = load_library()
    size = lib.fd_decode_workspace_size_fp4 if kv_dtype is not None and kv_dtype == _FP4 \
        else lib.fd_decode_workspace_size_mq
    return int(size(batch_size, seqlen_q, num_heads, num_heads_k, headdim))


def flash_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                 softmax_scale: float | None = None, return_softmax_lse: bool = False,
                 out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                 max_seqlen_k: int | None = None, workspace: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None, lse: torch.Tensor | None = None,
                 causal: bool = False, k: torch.Tensor | None = None,
                 v: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, k_block_scale: torch.Tensor | None = None,
                 v_block_scale: torch.Tensor | None = None):
    """Paged decode attention for seqlen_q >= 1 query tokens per sequence.

    q [B, sq, Hq, D]; k_cache/v_cache [num_blocks, page, Hkv, D];
    cache_seqlens [B] int32; block_table [B, max_blocks] int32.
    Returns out [B, sq, Hq, D] (and lse fp32 natural log: [B, Hq] for sq = 1,
    else [B, Hq, sq]).  causal: query token i sits at position L - sq + i
    (L = attended keys) and sees keys up to it.  `out` and `lse` may be
    given as preallocated contiguous buffers; passing `lse` implies
    return_softmax_lse.

    k / v [B, seqlen_new, Hkv, D] (optional, together): as in
    flash_attn_with_kvcache, they are first written into the cache at
    positions cache_seqlens[b] .. cache_seqlens[b] + seqlen_new - 1, then
    attention runs over L = cache_seqlens[b] + seqlen_new keys;
    cache_seqlens itself is left unchanged.

    FP8 cache: k_cache / v_cache of dtype torch.float8_e4m3fn with k_scale /
    v_scale fp32 [Hkv] (the attended key is k_cache * k_scale[h]); q stays
    bf16 or fp16 and k / v, when given, are 16-bit rows quantised into the
    cache.  Head dim 128, seqlen_q * (Hq / Hkv) <= 16, pages of a multiple
    of 16 tokens.

    4-bit cache: k_cache / v_cache of dtype torch.float4_e2m1fn_x2
    [num_blocks, page, Hkv, D / 2] with block scales k_block_scale /
    v_block_scale torch.float8_e4m3fn [num_blocks, Hkv, page, D / 16] (one
    for 16 consecutive values) and k_scale / v_scale fp32 [Hkv]: the attended
    key is e2m1 * block scale * k_scale[h].  Otherwise as the FP8 cache, with
    head dim 64, 128 or 256 and any number of query rows.
    """
    call = _prepare(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale,
                    return_softmax_lse, out, out_dtype, max_seqlen_k, workspace, lse, causal, k, v,
                    k_scale, v_scale, k_block_scale, v_block_scale, stream)
    with _on_device(q.device):
        check(call.fn(*call.args, _stream_handle(stream, q.device)))
    return (call.out, call.lse) if call.return_lse else call.out


class _Call:
    """One validated C call: entry point, its arguments up to the stream, and
    the output tensors it writes."""

    __slots__ = ("fn", "args", "out", "lse", "return_lse")

    def __init__(self, fn, args, out, lse, return_lse):
        self.fn, self.args, self.out, self.lse, self.return_lse = fn, args, out, lse, return_lse


def _prepare(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, return_softmax_lse,
             out, out_dtype, max_seqlen_k, workspace, lse, causal, k, v, k_scale, v_scale,
             k_block_scale=None, v_block_scale=None, stream=None) -> _Call:
    """Check the arguments of flash_decode, allocate the outputs it was not
    given (for a kernel on `stream`) and bind the C entry point that serves
    them."""
    lib = load_library()
    _require_cuda(q, k_cache, v_cache, cache_seqlens, block_table)
    if q.dim() != 4:
        raise ValueError(f"q must be [B, seqlen_q, Hq, D], got {tuple(q.shape)}")
    kv8 = k_cache.dtype == torch.float8_e4m3fn
    kv4 = k_cache.dtype == _FP4
    if q.dtype not in _DTYPES or v_cache.dtype != k_cache.dtype \
            or not (kv8 or kv4 or k_cache.dtype == q.dtype):
        raise ValueError("q, k_cache, v_cache must share dtype bf16 or fp16 (or e4m3 or e2m1 caches)")
    if kv8 or kv4:
        _check_scales(k_scale, v_scale, k_cache.shape[2])
    elif k_scale is not None or v_scale is not None:
        raise ValueError("k_scale / v_scale apply to float8_e4m3fn and float4_e2m1fn_x2 caches only")
    _check_block_scales(k_block_scale, v_block_scale, k_cache)
    if cache_seqlens.dtype != torch.int32 or block_table.dtype != torch.int32:
        raise ValueError("cache_seqlens and block_table must be int32")
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache),
                    ("cache_seqlens", cache_seqlens), ("block_table", block_table)):
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    B, sq, Hq, D = q.shape
    num_blocks, page, Hkv, Dk = k_cache.shape
    if tuple(v_cache.shape) != tuple(k_cache.shape) or (2 * Dk if kv4 else Dk) != D:
        raise ValueError("k_cache/v_cache shape mismatch")
    if block_table.dim() != 2 or block_table.shape[0] != B or cache_seqlens.shape != (B,):
        raise ValueError("block_table must be [B, max_blocks] and cache_seqlens [B]")
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    odt = q.dtype if out_dtype is None else out_dtype
    if out is None:
        out = _new((B, sq, Hq, D), odt, q.device, stream)
    elif out.dtype != odt or tuple(out.shape) != (B, sq, Hq, D) or not out.is_contiguous():
        raise ValueError("out has the wrong shape, dtype or layout")
    lse_shape = (B, Hq) if sq == 1 else (B, Hq, sq)
    if lse is not None:
        if lse.dtype != torch.float32 or lse.numel() != B * Hq * sq or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous fp32 {lse_shape} tensor")
        return_softmax_lse = True
    elif return_softmax_lse:
        lse = _new(lse_shape, torch.float32, q.device, stream)
    ws_ptr, ws_bytes = None, 0
    if workspace is not None:
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    if (k is None) != (v is None):
        raise ValueError("k and v must be given together")
    causal_i = 1 if causal else 0
    max_len = int(max_seqlen_k or 0)
    if kv4:
        if k is not None:
            _check_new_kv(k, v, k_cache, B, q.dtype)
        _require_device(q, k_cache, v_cache, k_block_scale, v_block_scale, k_scale, v_scale,
                        k, v, out, lse, cache_seqlens, block_table, workspace)
        args = (_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_block_scale), _ptr(v_block_scale),
                _ptr(k_scale), _ptr(v_scale), _ptr(k), _ptr(v), 0 if k is None else k.shape[1],
                _ptr(out), _ptr(lse), _ptr(cache_seqlens), _ptr(block_table),
                int(block_table.shape[1]), B, sq, Hq, Hkv, D, page, num_blocks, _DTYPES[q.dtype],
                _OUT_DTYPES[odt], scale, causal_i, max_len, ws_ptr, ws_bytes)
        return _Call(lib.fd_decode_paged_fp4, args, out, lse, return_softmax_lse)
    if kv8:
        if k is not None:
            _check_new_kv(k, v, k_cache, B, q.dtype)
        args = (_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(k),
                _ptr(v), 0 if k is None else k.shape[1], _ptr(out), _ptr(lse), _ptr(cache_seqlens),
                _ptr(block_table), int(block_table.shape[1]), B, sq, Hq, Hkv, D, page, num_blocks,
                _DTYPES[q.dtype], _OUT_DTYPES[odt], scale, causal_i, max_len, ws_ptr, ws_bytes)
        return _Call(lib.fd_decode_paged_fp8, args, out, lse, return_softmax_lse)
    if k is not None:
        _check_new_kv(k, v, k_cache, B)
        args = (_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k), _ptr(v), _ptr(out), _ptr(lse),
                _ptr(cache_seqlens), _ptr(block_table), int(block_table.shape[1]), B, sq,
                k.shape[1], Hq, Hkv, D, page, num_blocks, _DTYPES[q.dtype], _OUT_DTYPES[odt],
                scale, causal_i, max_len, ws_ptr, ws_bytes)
        return _Call(lib.fd_decode_paged_kvappend, args, out, lse, return_softmax_lse)
    args = (_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), _ptr(lse), _ptr(cache_seqlens),
            _ptr(block_table), int(block_table.shape[1]), B, sq, Hq, Hkv, D, page, num_blocks,
            _DTYPES[q.dtype], _OUT_DTYPES[odt], scale, causal_i, max_len, ws_ptr, ws_bytes)
    return _Call(lib.fd_decode_paged_mq, args, out, lse, return_softmax_lse)


class DecodePlan:
    """flash_decode bound to fixed tensors and checked once.

    A serving loop writes each step's query, lengths and page table into the
    same buffers; binding them once leaves a single C call per step (no
    argument checks, no output allocation: about a third of flash_decode's
    host time).  Takes flash_decode's arguments; the outputs are allocated
    once (or given) and overwritten by every call.  The bound tensors must
    stay alive and keep their storage, as for a captured CUDA graph: build a
    new plan when one of them is reallocated.

        plan = DecodePlan(q, k_cache, v_cache, cache_seqlens, block_table,
                          return_softmax_lse=True)
        out, lse = plan()          # on the current stream, or plan(stream)
    """

    def __init__(self, q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale=None,
                 return_softmax_lse=False, out=None, out_dtype=None, max_seqlen_k=None,
                 workspace=None, lse=None, causal=False, k=None, v=None, k_scale=None,
                 v_scale=None, k_block_scale=None, v_block_scale=None):
        self._call = _prepare(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale,
                              return_softmax_lse, out, out_dtype, max_seqlen_k, workspace, lse,
                              causal, k, v, k_scale, v_scale, k_block_scale, v_block_scale)
        self._device = q.device
        self._keep = (q, k_cache, v_cache, cache_seqlens, block_table, workspace, k, v, k_scale,
                      v_scale, k_block_scale, v_block_scale)

    @property
    def out(self) -> torch.Tensor:
        return self._call.out

    @property
    def lse(self) -> torch.Tensor | None:
        return self._call.lse

    def __call__(self, stream: torch.cuda.Stream | None = None):
        c = self._call
        with _on_device(self._device):
            check(c.fn(*c.args, _stream_handle(stream, self._device)))
        return (c.out, c.lse) if c.return_lse else c.out


def _check_scales(k_scale, v_scale, Hkv: int) -> None:
    for name, sc in (("k_scale", k_scale), ("v_scale", v_scale)):
        if sc is None:
            raise ValueError(f"{name} [Hkv] fp32 is required with a float8_e4m3fn or "
                             "float4_e2m1fn_x2 cache")
        _require_cuda(sc)
        if sc.dtype != torch.float32 or sc.shape != (Hkv,) or not sc.is_contiguous():
            raise ValueError(f"{name} must be a contiguous fp32 [{Hkv}] tensor")


def _check_block_scales(k_block_scale, v_block_scale, k_cache: torch.Tensor) -> None:
    """Block scales are given exactly with a 4-bit cache, in its shape."""
    if k_cache.dtype != _FP4:
        if k_block_scale is not None or v_block_scale is not None:
            raise ValueError("k_block_scale / v_block_scale apply to float4_e2m1fn_x2 caches only")
        return
    shape = k_cache.shape
    if len(shape) != 4 or shape[3] % 8 != 0:
        raise ValueError("a float4_e2m1fn_x2 cache is [num_blocks, page, Hkv, D / 2] with D a "
                         "multiple of 16")
    num_blocks, page, Hkv, half = shape
    want = (num_blocks, Hkv, page, half // 8)
    for name, sc in (("k_block_scale", k_block_scale), ("v_block_scale", v_block_scale)):
        if sc is None:
            raise ValueError(f"{name} is required with a float4_e2m1fn_x2 cache")
        if sc.dtype != torch.float8_e4m3fn or sc.shape != want or not sc.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float8_e4m3fn {want} tensor")


def _check_new_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, B: int,
                  new_dtype: torch.dtype | None = None) -> None:
    _require_cuda(k, v)
    if k.dim() != 4 or tuple(v.shape) != tuple(k.shape):
        raise ValueError("k and v must both be [B, seqlen_new, Hkv, D]")
    D = k_cache.shape[3] * (2 if k_cache.dtype == _FP4 else 1)
    if k.shape[0] != B or k.shape[2] != k_cache.shape[2] or k.shape[3] != D:
        raise ValueError("k / v shape does not match the batch and cache heads")
    want = k_cache.dtype if new_dtype is None else new_dtype
    if k.dtype != want or v.dtype != want:
        raise ValueError(f"k / v must be {want}")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("k and v must be contiguous")


def append_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              cache_seqlens: torch.Tensor, block_table: torch.Tensor,
              stream: torch.cuda.Stream | None = None, k_scale: torch.Tensor | None = None,
              v_scale: torch.Tensor | None = None, k_block_scale: torch.Tensor | None = None,
              v_block_scale: torch.Tensor | None = None) -> None:
    """Write k / v [B, seqlen_new, Hkv, D] into the paged cache at positions
    cache_seqlens[b] + t (the cache update of flash_attn_with_kvcache).  For
    float8_e4m3fn caches k / v are 16-bit and stored as e4m3(x / scale[h])
    with the fp32 [Hkv] k_scale / v_scale; float4_e2m1fn_x2 caches also take
    the block scales to write (see flash_decode)."""
    lib = load_library()
    _require_cuda(k_cache, v_cache, cache_seqlens, block_table)
    if cache_seqlens.dtype != torch.int32 or block_table.dtype != torch.int32:
        raise ValueError("cache_seqlens and block_table must be int32")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and block_table.is_contiguous()):
        raise ValueError("caches and block_table must be contiguous")
    kv8 = k_cache.dtype == torch.float8_e4m3fn
    if k_cache.dtype not in _CACHE_DTYPES or v_cache.dtype != k_cache.dtype \
            or tuple(v_cache.shape) != tuple(k_cache.shape):
        raise ValueError("k_cache/v_cache must be bf16, fp16, float8_e4m3fn or float4_e2m1fn_x2 "
                         "with equal shapes")
    B = block_table.shape[0]
    num_blocks, page, Hkv, D = k_cache.shape
    _check_block_scales(k_block_scale, v_block_scale, k_cache)
    st = stream if stream is not None else torch.cuda.current_stream(k.device)
    if k_cache.dtype == _FP4:
        _check_scales(k_scale, v_scale, Hkv)
        if k.dtype not in _DTYPES:
            raise ValueError("k / v must be bf16 or fp16")
        _check_new_kv(k, v, k_cache, B, k.dtype)
        if cache_seqlens.shape != (B,) or not cache_seqlens.is_contiguous():
            raise ValueError("cache_seqlens must be a contiguous [B] tensor")
        _require_device(k, v, k_cache, v_cache, k_block_scale, v_block_scale, k_scale,
                        v_scale, cache_seqlens, block_table)
        with torch.cuda.device(k.device):
            status = lib.fd_append_kv_paged_fp4(
                _ptr(k), _ptr(v), _ptr(k_cache), _ptr(v_cache), _ptr(k_block_scale),
                _ptr(v_block_scale), _ptr(k_scale), _ptr(v_scale), _ptr(cache_seqlens),
                _ptr(block_table), int(block_table.shape[1]), B, k.shape[1], Hkv, 2 * D, page,
                num_blocks, _DTYPES[k.dtype], st.cuda_stream)
        check(status)
        return
    if kv8:
        _check_scales(k_scale, v_scale, Hkv)
        if k.dtype not in _DTYPES:
            raise ValueError("k / v must be bf16 or fp16")
        _check_new_kv(k, v, k_cache, B, k.dtype)
        with torch.cuda.device(k.device):
            status = lib.fd_append_kv_paged_fp8(
                _ptr(k), _ptr(v), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
                _ptr(cache_seqlens), _ptr(block_table), int(block_table.shape[1]), B, k.shape[1],
                Hkv, D, page, num_blocks, _DTYPES[k.dtype], st.cuda_stream)
        check(status)
        return
    _check_new_kv(k, v, k_cache, B)
    with torch.cuda.device(k.device):
        status = lib.fd_append_kv_paged(
            _ptr(k), _ptr(v), _ptr(k_cache), _ptr(v_cache), _ptr(cache_seqlens), _ptr(block_table),
            int(block_table.shape[1]), B, k.shape[1], Hkv, D, page, num_blocks, _DTYPES[k.dtype],
            st.cuda_stream)
    check(status)


def _check_slot_cache(k_cache, v_cache, slot_map, k_scale, v_scale, k_block_scale, v_block_scale):
    """Checks that append_kv_slots and gather_kv share, but for the device of
    the tensors; returns (T, page, Hkv, D, num_blocks) of the call."""
    dtype, shape = k_cache.dtype, k_cache.shape
    if dtype not in _CACHE_DTYPES or v_cache.dtype != dtype or len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("k_cache/v_cache must be bf16, fp16, float8_e4m3fn or float4_e2m1fn_x2 "
                         "[num_blocks, page, Hkv, D] tensors with equal shapes")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    slots = slot_map.shape
    if slot_map.dtype != torch.int64 or len(slots) != 1 or not slot_map.is_contiguous():
        raise ValueError("slot_map must be a contiguous int64 [T] tensor")
    num_blocks, page, Hkv, D = shape
    if dtype in _DTYPES:
        if k_scale is not None or v_scale is not None:
            raise ValueError("k_scale / v_scale apply to float8_e4m3fn and float4_e2m1fn_x2 caches only")
    else:
        _check_scales(k_scale, v_scale, Hkv)
    _check_block_scales(k_block_scale, v_block_scale, k_cache)
    return slots[0], page, Hkv, 2 * D if dtype == _FP4 else D, num_blocks


def append_kv_slots(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    slot_map: torch.Tensor, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None, k_block_scale: torch.Tensor | None = None,
                    v_block_scale: torch.Tensor | None = None,
                    stream: torch.cuda.Stream | None = None) -> None:
    """Write packed rows k / v [T, Hkv, D] (bf16 or fp16) into the paged cache
    at slot_map [T] int64: slot = page id * page + row in the page, as
    assign_pages gives them; negative slots are skipped.  The rows may have
    any stride from token to token (a slice of a fused projection); the cache
    is of any kind flash_decode reads, and quantised ones take their scales.
    The slots should be distinct."""
    lib = load_library()
    _require_device(k_cache, v_cache, slot_map, k, v, k_scale, v_scale, k_block_scale, v_block_scale)
    T, page, Hkv, D, num_blocks = _check_slot_cache(k_cache, v_cache, slot_map, k_scale, v_scale,
                                                    k_block_scale, v_block_scale)
    src, dst = _DTYPES.get(k.dtype), _CACHE_DTYPES[k_cache.dtype]
    if src is None or v.dtype != k.dtype:
        raise ValueError("k / v must be bf16 or fp16")
    if k_cache.dtype in _DTYPES and src != dst:
        raise ValueError(f"k / v must be {k_cache.dtype}")
    want = (T, Hkv, D)
    row = Hkv * D
    token = []
    for name, x in (("k", k), ("v", v)):
        if x.shape != want:
            raise ValueError(f"{name} must be [T, Hkv, D] = {want}, got {tuple(x.shape)}")
        st, sh, sd = x.stride()
        if T > 0 and ((D > 1 and sd != 1) or (Hkv > 1 and sh != D) or (T > 1 and st < row)):
            raise ValueError(f"the heads of a token of {name} must be contiguous")
        token.append(st if T > 1 else row)
    dev = k_cache.device
    _launch(lib.fd_append_kv_slots, dev, stream, (
        k.data_ptr(), token[0], v.data_ptr(), token[1], k_cache.data_ptr(), v_cache.data_ptr(),
        _ptr(k_block_scale), _ptr(v_block_scale), _ptr(k_scale), _ptr(v_scale), slot_map.data_ptr(),
        T, Hkv, D, page, num_blocks, src, dst))


def gather_kv(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_map: torch.Tensor,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
              k_block_scale: torch.Tensor | None = None, v_block_scale: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None, k_out: torch.Tensor | None = None,
              v_out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None):
    """The cache rows at slot_map [T] int64 as values: k, v [T, Hkv, D] of
    out_dtype (default: the cache's type, bf16 for quantised caches), zeros at
    negative slots.  The inverse of append_kv_slots."""
    lib = load_library()
    _require_device(k_cache, v_cache, slot_map, k_scale, v_scale, k_block_scale, v_block_scale, k_out, v_out)
    T, page, Hkv, D, num_blocks = _check_slot_cache(k_cache, v_cache, slot_map, k_scale, v_scale,
                                                    k_block_scale, v_block_scale)
    if out_dtype is None:
        out_dtype = k_out.dtype if k_out is not None else \
            k_cache.dtype if k_cache.dtype in _DTYPES else torch.bfloat16
    odt = _OUT_DTYPES.get(out_dtype)
    if odt is None:
        raise ValueError("out_dtype must be bf16, fp16 or fp32")
    dev = k_cache.device
    want = (T, Hkv, D)
    for name, x in (("k_out", k_out), ("v_out", v_out)):
        if x is not None and (x.dtype != out_dtype or x.shape != want or not x.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {out_dtype} {want} CUDA tensor")
    if k_out is None:
        k_out = _new(want, out_dtype, dev, stream)
    if v_out is None:
        v_out = _new(want, out_dtype, dev, stream)
    _launch(lib.fd_gather_kv_slots, dev, stream, (
        k_cache.data_ptr(), v_cache.data_ptr(), _ptr(k_block_scale), _ptr(v_block_scale),
        _ptr(k_scale), _ptr(v_scale), slot_map.data_ptr(), T, k_out.data_ptr(), v_out.data_ptr(),
        Hkv, D, page, num_blocks, _CACHE_DTYPES[k_cache.dtype], odt))
    return k_out, v_out


def _check_int32(name: str, t: torch.Tensor, shape) -> None:
    if t.dtype is not _INT32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)}")


def _check_pool(block_table, free_pages, free_count) -> tuple[int, int, int]:
    """Checks that assign_pages and release_pages share; returns (B, width of
    the table, pages of the pool)."""
    table, pool = block_table.shape, free_pages.shape
    if len(table) != 2:
        raise ValueError("block_table must be [B, max_blocks]")
    if len(pool) != 1:
        raise ValueError("free_pages must be [num_blocks]")
    _check_int32("block_table", block_table, table)
    _check_int32("free_pages", free_pages, pool)
    _check_int32("free_count", free_count, (2,))
    return table[0], table[1], pool[0]


def assign_pages(block_table: torch.Tensor, cache_seqlens: torch.Tensor, new_lens: torch.Tensor,
                 free_pages: torch.Tensor, free_count: torch.Tensor, page_block_size: int,
                 slot_map: torch.Tensor | None = None, num_slots: int | None = None,
                 cu_new_lens: torch.Tensor | None = None, seqlens_out: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None):
    """Pages and cache slots for a step's new tokens, on the device.

    Request b holds cache_seqlens[b] tokens in the pages of its block_table
    row and gets new_lens[b] more.  Pages come off the top of the stack
    free_pages [num_blocks] int32 (its size is the cache's number of pages),
    of which free_count[0] entries are free, in the order of the requests, and
    are entered in block_table; free_count [2] int32 starts as (free, 0) and
    its second word belongs to the library.

    Returns (slot_map, cu_new_lens, seqlens_out): the slot of each packed new
    token (int64; give a slot_map buffer of fixed size, e.g. for a CUDA graph,
    or num_slots = the step's tokens; -1 behind the last token), the prefix
    sums of new_lens [B + 1], and the lengths afterwards (a buffer may be
    given; cache_seqlens itself updates them in place).  A request that does
    not fit gets nothing (slots -1, length unchanged) and device_status()
    reports FD_ERR_NO_PAGES; requests are served in order.
    """
    lib = load_library()
    _require_device(block_table, cache_seqlens, new_lens, free_pages, free_count, slot_map, cu_new_lens,
                    seqlens_out)
    B, width, num_blocks = _check_pool(block_table, free_pages, free_count)
    _check_int32("cache_seqlens", cache_seqlens, (B,))
    _check_int32("new_lens", new_lens, (B,))
    dev = block_table.device
    if slot_map is None:
        if num_slots is None:
            raise ValueError("give slot_map or num_slots")
        num_slots = int(num_slots)
        slot_map = _new(num_slots, torch.int64, dev, stream)
    else:
        slots = slot_map.shape
        if slot_map.dtype != torch.int64 or len(slots) != 1 or not slot_map.is_contiguous():
            raise ValueError("slot_map must be a contiguous int64 [num_slots] CUDA tensor")
        num_slots = slots[0]
    if cu_new_lens is None:
        cu_new_lens = _new(B + 1, _INT32, dev, stream)
    else:
        _check_int32("cu_new_lens", cu_new_lens, (B + 1,))
    if seqlens_out is None:
        seqlens_out = _new(B, _INT32, dev, stream)
    else:
        _check_int32("seqlens_out", seqlens_out, (B,))
    _launch(lib.fd_assign_pages, dev, stream, (
        block_table.data_ptr(), width, cache_seqlens.data_ptr(), new_lens.data_ptr(),
        free_pages.data_ptr(), free_count.data_ptr(), B, int(page_block_size), num_blocks,
        seqlens_out.data_ptr(), cu_new_lens.data_ptr(), slot_map.data_ptr(), num_slots))
    return slot_map, cu_new_lens, seqlens_out


def release_pages(block_table: torch.Tensor, cache_seqlens: torch.Tensor, keep_lens: torch.Tensor,
                  free_pages: torch.Tensor, free_count: torch.Tensor, page_block_size: int,
                  stream: torch.cuda.Stream | None = None) -> None:
    """Give back the pages of cache_seqlens[b] tokens that keep_lens[b] tokens
    do not need (0: the request is finished).  Their block_table entries
    become -1; the lengths are not changed.  Releasing what the last
    assign_pages took leaves the stack as it was."""
    lib = load_library()
    _require_device(block_table, cache_seqlens, keep_lens, free_pages, free_count)
    B, width, num_blocks = _check_pool(block_table, free_pages, free_count)
    _check_int32("cache_seqlens", cache_seqlens, (B,))
    _check_int32("keep_lens", keep_lens, (B,))
    dev = block_table.device
    _launch(lib.fd_release_pages, dev, stream, (
        block_table.data_ptr(), width, cache_seqlens.data_ptr(), keep_lens.data_ptr(),
        free_pages.data_ptr(), free_count.data_ptr(), B, int(page_block_size), num_blocks))


def combine_lse(part_o: torch.Tensor, part_lse: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
                return_lse: bool = False, stream: torch.cuda.Stream | None = None):
    """Merge partial results over disjoint KV ranges.

    part_o [n, rows, D] fp32 (normalised), part_lse [n, rows] fp32 natural log.
    Each part must be contiguous; the parts themselves may be strided (views
    into one gathered buffer of per-part [O | LSE] blocks).
    Returns out [rows, D] (and lse [rows]).
    """
    lib = load_library()
    _require_cuda(part_o, part_lse)
    if part_o.dtype != torch.float32 or part_lse.dtype != torch.float32:
        raise ValueError("partials must be fp32")
    n, rows, D = part_o.shape
    st = stream if stream is not None else torch.cuda.current_stream(part_o.device)
    with _on_stream(st, part_o.device):  # copies are read by the kernel on this stream
        if part_o.stride()[1:] != (D, 1):
            part_o = part_o.contiguous()
        if part_lse.stride(1) != 1:
            part_lse = part_lse.contiguous()
    out = _new((rows, D), out_dtype, part_o.device, stream)
    lse = _new((rows,), torch.float32, part_o.device, stream) if return_lse else None
    with torch.cuda.device(part_o.device):
        status = lib.fd_combine_lse(_ptr(part_o), part_o.stride(0), _ptr(part_lse), part_lse.stride(0),
                                    n, rows, D, _ptr(out), _OUT_DTYPES[out_dtype], _ptr(lse),
                                    st.cuda_stream)
    check(status)
    return (out, lse) if return_lse else out


__all__ = ["run_kernel", "flash_decode", "DecodePlan", "append_kv", "append_kv_slots", "gather_kv",
           "assign_pages", "release_pages", "combine_lse", "last_error", "device_status",
           "workspace_size", "FlashDecodeError"]
