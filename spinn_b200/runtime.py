"""Host-side API mirroring SPINN's operator and runtime interfaces.

* Operator level -- :func:`conv2d`, :func:`gemm`, :func:`matmul` call the C-ABI drop-in
  kernels with the reference's argument conventions (``SpinnTensor`` records, ENNF
  parameter blocks; ``SPINN/run_time/ops/conv/conv2d.c``, ``ops/mm/gemm.c``,
  ``ops/mm/matmul.c``).  Arrays may be NumPy (host memory, like the reference arena) or
  CUDA torch tensors (device memory).
* Decoder serving -- :func:`linear`, :func:`cache_append`, :func:`paged_attention`, :func:`cache_evict` work on
  CUDA torch tensors, on torch's current stream of their device; :func:`stream_sync`
  reports what only the device could see (a bad page number, a length beyond its table).
* Model level -- :class:`Model` wraps ``spinn_cuda_load / _plan / _run / _free``, the
  device-resident counterpart of ``spinn_load / spinn_plan / spinn_run / spinn_free``
  (``SPINN/run_time/spinn_runtime.h:107-133``).
"""
from __future__ import annotations

import ctypes
import struct
from typing import List, Optional, Sequence

import numpy as np

from . import lib as _L
from .lib import SpinnTensor, check, lib

CONV_PARAMS_FMT = "<4H4H8H4HHBB"   # ENNF_ConvParams (SPINN/ennf_op_params.h:23-31)
GEMM_PARAMS_FMT = "<ffBB2x"        # ENNF_GemmParams (SPINN/ennf_op_params.h:134-140)


def conv_params(kernel=(0, 0), strides=(1, 1), pads=(0, 0, 0, 0), dilations=(1, 1), group=1,
                auto_pad=0, fused_act=0) -> bytes:
    """Packs an ``ENNF_ConvParams`` block; ``fused_act`` goes into ``reserved``."""
    def pad(v, n):
        v = list(v)[:n]
        return v + [0] * (n - len(v))
    return struct.pack(CONV_PARAMS_FMT, *pad(kernel, 4), *pad(strides, 4), *pad(pads, 8),
                       *pad(dilations, 4), group, auto_pad, fused_act)


def gemm_params(alpha=1.0, beta=1.0, trans_a=0, trans_b=0) -> bytes:
    return struct.pack(GEMM_PARAMS_FMT, alpha, beta, trans_a, trans_b)


class _Arg:
    """A SpinnTensor record over a NumPy array (host) or a CUDA torch tensor (device)."""

    def __init__(self, arr, is_weight: bool = False, tid: int = 0):
        self.arr = arr
        t = SpinnTensor()
        shape = tuple(arr.shape)
        if len(shape) > 8:
            raise ValueError("at most 8 dimensions")
        t.id = tid
        t.dtype = 1
        t.ndim = len(shape)
        for i, d in enumerate(shape):
            t.dims[i] = int(d)
        n = int(np.prod(shape)) if shape else 1
        t.elem_count = n
        t.is_weight = 1 if is_weight else 0
        t.size = n * 4
        if isinstance(arr, np.ndarray):
            if arr.dtype != np.float32 or not arr.flags["C_CONTIGUOUS"]:
                raise TypeError("host arrays must be C-contiguous float32")
            t.data = arr.ctypes.data
        else:  # torch tensor
            import torch
            if arr.dtype != torch.float32 or not arr.is_contiguous():
                raise TypeError("torch tensors must be contiguous float32")
            t.data = arr.data_ptr()
        self.rec = t


def _call(fn_name: str, ins: Sequence[_Arg], outs: Sequence[_Arg], params: bytes) -> None:
    n_in, n_out = len(ins), len(outs)
    in_arr = (ctypes.POINTER(SpinnTensor) * n_in)(*[ctypes.pointer(a.rec) for a in ins])
    out_arr = (ctypes.POINTER(SpinnTensor) * n_out)(*[ctypes.pointer(a.rec) for a in outs])
    pbuf = ctypes.create_string_buffer(params, len(params)) if params else None
    rc = getattr(lib(), fn_name)(ctypes.cast(in_arr, ctypes.c_void_p), n_in,
                                 ctypes.cast(pbuf, ctypes.c_void_p) if pbuf else None, len(params),
                                 ctypes.cast(out_arr, ctypes.c_void_p), n_out)
    check(rc, fn_name)


def init(device: int = 0, scratch_bytes: int = 0) -> None:
    check(lib().spinn_cuda_init(device, scratch_bytes), "spinn_cuda_init")


def sync() -> None:
    check(lib().spinn_cuda_sync(), "spinn_cuda_sync")


def shutdown() -> None:
    lib().spinn_cuda_shutdown()


def conv2d(x, w, y, bias=None, residual=None, params: bytes = b"") -> None:
    """``op_conv2d`` semantics: inputs [X, W, (B), (R)], residual last when the fused act is 4/5."""
    ins = [_Arg(x), _Arg(w, True)]
    if bias is not None:
        ins.append(_Arg(bias, True))
    if residual is not None:
        ins.append(_Arg(residual))
    _call("spinn_cuda_conv2d", ins, [_Arg(y)], params or conv_params())


def gemm(a, b, y, c=None, params: bytes = b"", b_is_weight: bool = True) -> None:
    ins = [_Arg(a), _Arg(b, b_is_weight)]
    if c is not None:
        ins.append(_Arg(c, True))
    _call("spinn_cuda_gemm", ins, [_Arg(y)], params or gemm_params())


def matmul(a, b, y) -> None:
    _call("spinn_cuda_matmul", [_Arg(a), _Arg(b)], [_Arg(y)], b"")


# ------------------------------------------------------------------ decoder serving
_CACHE = struct.Struct("<QQqqqiiiiii")         # SpinnCudaCache
_TABLE = struct.Struct("<QQqii")               # SpinnCudaPageTable
_APPEND = struct.Struct("<QQqqqqQii")          # SpinnCudaAppend
_ATTENTION = struct.Struct("<QQqqqqQQqqqqiifi")  # SpinnCudaAttention
_EVICT = struct.Struct("<QQqqqqQqiiQQii")      # SpinnCudaEvict
_LINEAR = struct.Struct("<QQQQQqqqqiiiiii")    # SpinnCudaLinear
_ACTS = {"none": 0, "relu": 1, "silu": 3, "gelu": 6, "gelu_tanh": 7}
_torch = None
_dtype_codes: dict = {}


def _torch_module():
    global _torch
    if _torch is None:
        import torch
        _dtype_codes.update({torch.float32: _L.FP32, torch.float16: _L.FP16, torch.bfloat16: _L.BF16})
        _torch = torch
    return _torch


def _on_device(name, *tensors) -> int:
    """The one CUDA device of the tensors (None among them is skipped)."""
    dev = tensors[0].get_device()
    if dev < 0:
        raise TypeError(f"{name}: CUDA tensors are required")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name}: tensors on different devices")
    return dev


def _queue(dev: int, call) -> None:
    """``call(stream)`` with `dev` as the current device and torch's current stream of it."""
    torch = _torch
    if torch.cuda.current_device() == dev:
        call(torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            call(torch.cuda.current_stream(dev).cuda_stream)


def _cache_desc(name, k, v) -> bytes:
    if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
        raise ValueError(f"{name}: k_cache and v_cache must be [pages, page_size, heads, dim] of one shape, "
                         "layout and type")
    code = _dtype_codes.get(k.dtype)
    if code is None:
        raise TypeError(f"{name}: caches of {k.dtype} are not supported (float32, float16, bfloat16)")
    pages, page, heads, dim = k.shape
    ps, ts, hs, es = k.stride()
    if es != 1 and dim != 1:
        raise ValueError(f"{name}: the cache's last dimension must be contiguous")
    return _CACHE.pack(k.data_ptr(), v.data_ptr(), ps, ts, hs, code, pages, page, heads, dim, 0)


def _table_desc(name, table, lens) -> bytes:
    i32 = _torch.int32
    if table.dtype != i32 or lens.dtype != i32:
        raise TypeError(f"{name}: page_table and lens must be int32")
    if table.dim() != 2 or lens.dim() != 1 or lens.shape[0] != table.shape[0] or not lens.is_contiguous() or \
            (table.stride(1) != 1 and table.shape[1] != 1):
        raise ValueError(f"{name}: page_table must be [seqs, max_pages] with contiguous rows, lens [seqs]")
    return _TABLE.pack(table.data_ptr(), lens.data_ptr(), table.stride(0), table.shape[0], table.shape[1])


def _rows(name, what, t, cache, shape):
    """(pointer, stride, stride) of a [n, heads, dim] tensor of the cache's type."""
    if t.dtype != cache.dtype:
        raise TypeError(f"{name}: {what} must have the cache's type {cache.dtype}, not {t.dtype}")
    if tuple(t.shape) != shape or (t.stride(2) != 1 and shape[2] != 1):
        raise ValueError(f"{name}: {what} must be {shape} with contiguous rows, not {tuple(t.shape)}")
    return t.data_ptr(), t.stride(0), t.stride(1)


def _weights(name, what, t, seqs, heads):
    if t is None:
        return 0, 0, 0
    if t.dtype != _torch.float32:
        raise TypeError(f"{name}: {what} must be float32")
    if t.dim() != 3 or t.shape[0] != seqs or t.shape[1] != heads or (t.stride(2) != 1 and t.shape[2] != 1):
        raise ValueError(f"{name}: {what} must be [{seqs}, {heads}, length] with contiguous rows")
    return t.data_ptr(), t.stride(0), t.stride(1)


def stream_sync(device: Optional[int] = None) -> None:
    """Waits for torch's current stream and raises the deferred error of the operators below, if
    any (``spinn_cuda_stream_sync``).  Not during graph capture."""
    torch = _torch_module()
    _queue(torch.cuda.current_device() if device is None else device,
           lambda st: check(lib().spinn_cuda_stream_sync(st), "spinn_cuda_stream_sync"))


def linear(x, w, y, bias=None, residual=None, act: str = "none") -> None:
    """``y = act(x @ w.T + bias) + residual`` in fp16 or bf16 (fp32: :func:`gemm`), accumulated in fp32
    and rounded once.

    ``x`` is ``[m, k]``, ``w`` ``[n, k]``, ``y`` and ``residual`` ``[m, n]``, with contiguous rows of any
    stride, ``bias`` ``[n]``; ``act`` is "none", "relu", "silu", "gelu" (by erf) or "gelu_tanh".  ``y``
    may be ``residual`` itself.  Rows of ``x`` and ``w`` that start on 16-byte boundaries are read in
    place; others are copied first when ``x`` has more than 16 rows."""
    torch = _torch_module()
    name = "linear"
    dev = _on_device(name, x, w, y, bias, residual)
    code = _dtype_codes.get(x.dtype)
    if x.dtype != w.dtype or x.dtype != y.dtype or code not in (_L.FP16, _L.BF16):
        raise TypeError(f"{name}: x, w and y must all be float16 or all bfloat16")
    if x.dim() != 2 or w.dim() != 2 or y.dim() != 2:
        raise ValueError(f"{name}: x, w and y must be 2-D")
    (m, k), (n, k2) = x.shape, w.shape
    if k != k2 or y.shape[0] != m or y.shape[1] != n:
        raise ValueError(f"{name}: shapes {tuple(x.shape)}, {tuple(w.shape)} and {tuple(y.shape)} do not match")
    xs, ws, ys, rs = x.stride(), w.stride(), y.stride(), (n, 1)
    bp = rp = 0
    if bias is not None:
        if bias.dtype != x.dtype or tuple(bias.shape) != (n,) or (bias.stride(0) != 1 and n != 1):
            raise ValueError(f"{name}: bias must be a contiguous [{n}] of {x.dtype}")
        bp = bias.data_ptr()
    if residual is not None:
        if residual.dtype != x.dtype or residual.shape != y.shape:
            raise ValueError(f"{name}: residual must be {tuple(y.shape)} of {x.dtype}")
        rs = residual.stride()
        rp = residual.data_ptr()
    if act not in _ACTS:
        raise ValueError(f"{name}: act must be one of {', '.join(_ACTS)}")
    if (xs[1] != 1 and k != 1) or (ws[1] != 1 and k != 1) or (n != 1 and (ys[1] != 1 or rs[1] != 1)):
        raise ValueError(f"{name}: rows must be contiguous")
    if m == 0:
        return
    # the stride of a single row means nothing
    desc = _LINEAR.pack(x.data_ptr(), w.data_ptr(), bp, rp, y.data_ptr(), xs[0] if m > 1 else k, ws[0] if n > 1 else k,
                        rs[0] if m > 1 else n, ys[0] if m > 1 else n, m, n, k, code, _ACTS[act], 0)

    def call(st):
        L = lib()
        size = L.spinn_cuda_linear_workspace(desc)
        space = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        check(L.spinn_cuda_linear(desc, space.data_ptr() if size else None, size, st), "spinn_cuda_linear")

    _queue(dev, call)


def cache_append(k, v, k_cache, v_cache, page_table, lens, starts=None) -> None:
    """Writes new tokens' rows ``k`` and ``v`` ``[tokens, kv_heads, head_dim]`` into the paged cache.

    Rows ``starts[s] .. starts[s + 1] - 1`` (int32, ``[seqs + 1]``) become tokens ``lens[s]``,
    ``lens[s] + 1``, ... of sequence ``s``; without ``starts`` there is one row per sequence.
    ``lens`` (the lengths before) is not changed.  Caches are ``[pages, page_size, kv_heads,
    head_dim]`` in fp32, fp16 or bf16 with any strides but a contiguous last dimension,
    ``page_table`` is int32 ``[seqs, max_pages]``."""
    torch = _torch_module()
    name = "cache_append"
    dev = _on_device(name, k_cache, v_cache, k, v, page_table, lens, starts)
    cache, table = _cache_desc(name, k_cache, v_cache), _table_desc(name, page_table, lens)
    tokens = k.shape[0]
    shape = (tokens, k_cache.shape[2], k_cache.shape[3])
    kp, kt, kh = _rows(name, "k", k, k_cache, shape)
    vp, vt, vh = _rows(name, "v", v, k_cache, shape)
    sp = 0
    if starts is not None:
        if starts.dtype != torch.int32:
            raise TypeError(f"{name}: starts must be int32")
        if starts.dim() != 1 or starts.shape[0] != lens.shape[0] + 1 or not starts.is_contiguous():
            raise ValueError(f"{name}: starts must be [seqs + 1]")
        sp = starts.data_ptr()
    elif tokens != lens.shape[0]:
        raise ValueError(f"{name}: {tokens} rows for {lens.shape[0]} sequences without starts")
    if tokens == 0:
        return
    rows = _APPEND.pack(kp, vp, kt, kh, vt, vh, sp, tokens, 0)
    _queue(dev, lambda st: check(lib().spinn_cuda_cache_append(cache, table, rows, st), "spinn_cuda_cache_append"))


def paged_attention(q, k_cache, v_cache, page_table, lens, y, scale=None, weights=None, weights_out=None) -> None:
    """Attention of one new token per sequence over its cached tokens, into ``y``.

    ``q`` and ``y`` are ``[seqs, q_heads, head_dim]`` of the cache's type; head ``h`` reads key head
    ``h // (q_heads // kv_heads)``.  ``scale`` defaults to ``head_dim ** -0.5``.  A sequence of
    length 0 gets zeros.  With ``weights_out`` (fp32 ``[seqs, kv_heads, length]``) the probabilities
    of each key head's queries are summed and added to ``weights`` (zeros when None; may be
    ``weights_out`` itself); entries past a sequence's length are left as they were."""
    torch = _torch_module()
    name = "paged_attention"
    if lens.numel() == 0:
        return
    dev = _on_device(name, k_cache, v_cache, q, page_table, lens, y, weights, weights_out)
    cache, table = _cache_desc(name, k_cache, v_cache), _table_desc(name, page_table, lens)
    seqs, heads, dim = lens.shape[0], k_cache.shape[2], k_cache.shape[3]
    if q.dim() != 3:
        raise ValueError(f"{name}: q must be [seqs, q_heads, head_dim]")
    q_heads = q.shape[1]
    qp, qs, qh = _rows(name, "q", q, k_cache, (seqs, q_heads, dim))
    yp, ys, yh = _rows(name, "y", y, k_cache, (seqs, q_heads, dim))
    wp, ws, wh = _weights(name, "weights", weights, seqs, heads)
    op, os_, oh = _weights(name, "weights_out", weights_out, seqs, heads)
    capacity = 0
    if weights_out is not None:
        capacity = weights_out.shape[2]
        if weights is not None:
            capacity = min(capacity, weights.shape[2])
    elif weights is not None:
        raise ValueError(f"{name}: weights without weights_out")
    desc = _ATTENTION.pack(qp, yp, qs, qh, ys, yh, wp, op, ws, wh, os_, oh, capacity, q_heads,
                           dim ** -0.5 if scale is None else scale, 0)

    def call(st):
        L = lib()
        size = L.spinn_cuda_paged_attention_workspace(cache, table, desc)
        space = torch.empty(size, dtype=torch.uint8, device=q.device)
        check(L.spinn_cuda_paged_attention(cache, table, desc, space.data_ptr(), size, st), "spinn_cuda_paged_attention")

    _queue(dev, call)


def cache_evict(k_cache, v_cache, page_table, lens, weights, weights_out, out_table, new_lens, kept, budget,
                recent=0) -> None:
    """Cuts every sequence back to ``budget`` tokens, for each key head by itself: the last ``recent``
    tokens stay, and of the others those with the largest accumulated ``weights`` (fp32 ``[seqs,
    kv_heads, length]``; ties: the earlier token, NaN lowest), in their order.

    Their rows move to the first tokens of the pages in ``out_table`` -- ``page_table`` itself for a
    cut in place (no page may then belong to two sequences), or a table of pages that no sequence
    reads.  ``new_lens`` (int32 ``[seqs]``) gets the new lengths, ``kept`` (int32 ``[seqs, kv_heads,
    budget]``) the slots that were kept (-1 past the new length), ``weights_out`` their weights and
    zeros from there to the old length; it may be ``weights`` itself."""
    torch = _torch_module()
    name = "cache_evict"
    if lens.numel() == 0:
        return
    dev = _on_device(name, k_cache, v_cache, page_table, lens, weights, weights_out, out_table, new_lens, kept)
    cache, table = _cache_desc(name, k_cache, v_cache), _table_desc(name, page_table, lens)
    seqs, heads = lens.shape[0], k_cache.shape[2]
    i32 = torch.int32
    if out_table.dtype != i32 or new_lens.dtype != i32 or kept.dtype != i32:
        raise TypeError(f"{name}: out_table, new_lens and kept must be int32")
    if out_table.dim() != 2 or out_table.shape[0] != seqs or (out_table.stride(1) != 1 and out_table.shape[1] != 1):
        raise ValueError(f"{name}: out_table must be [seqs, max_pages] with contiguous rows")
    if new_lens.shape != lens.shape or not new_lens.is_contiguous():
        raise ValueError(f"{name}: new_lens must be [seqs]")
    if tuple(kept.shape) != (seqs, heads, budget) or not kept.is_contiguous():
        raise ValueError(f"{name}: kept must be [{seqs}, {heads}, {budget}], contiguous")
    wp, ws, wh = _weights(name, "weights", weights, seqs, heads)
    op, os_, oh = _weights(name, "weights_out", weights_out, seqs, heads)
    desc = _EVICT.pack(wp, op, ws, wh, os_, oh, out_table.data_ptr(), out_table.stride(0), out_table.shape[1],
                       min(weights.shape[2], weights_out.shape[2]), new_lens.data_ptr(), kept.data_ptr(), budget,
                       recent)
    _queue(dev, lambda st: check(lib().spinn_cuda_cache_evict(cache, table, desc, st), "spinn_cuda_cache_evict"))


class Model:
    """A ``.ennf`` model planned on one GPU (load -> plan -> run)."""

    def __init__(self, source, device: int = 0, max_arena_bytes: int = 0, flags: int = 0):
        L = lib()
        if isinstance(source, (bytes, bytearray, memoryview)):
            buf = bytes(source)
            self._h = L.spinn_cuda_load_buffer(buf, len(buf))
        else:
            self._h = L.spinn_cuda_load(str(source).encode())
        if not self._h:
            raise _L.SpinnCudaError(_L.EFORMAT, "spinn_cuda_load", _L.last_error())
        self.device = device
        self.flags = flags
        try:
            check(L.spinn_cuda_plan(self._h, device, max_arena_bytes, flags), "spinn_cuda_plan")
        except Exception:
            L.spinn_cuda_free(self._h)
            self._h = None
            raise

    def close(self) -> None:
        if getattr(self, "_h", None):
            lib().spinn_cuda_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def io_dims(self, is_output: bool, index: int = 0) -> List[int]:
        dims = (ctypes.c_uint32 * 8)()
        nd = check(lib().spinn_cuda_io_dims(self._h, int(is_output), index, dims), "spinn_cuda_io_dims")
        return [int(dims[i]) for i in range(nd)]

    def io_count(self, is_output: bool) -> int:
        return check(lib().spinn_cuda_io_count(self._h, int(is_output)), "spinn_cuda_io_count")

    def io_ptr(self, is_output: bool, index: int = 0):
        n = ctypes.c_size_t(0)
        p = lib().spinn_cuda_io_ptr(self._h, int(is_output), index, ctypes.byref(n))
        if not p:
            raise _L.SpinnCudaError(_L.ESTATE, "spinn_cuda_io_ptr", "no such buffer")
        return p, n.value

    def output(self, index: int) -> np.ndarray:
        """Graph output `index` of the last run, copied to host (fp32 or int64)."""
        dt = np.int64 if check(lib().spinn_cuda_io_dtype(self._h, 1, index), "spinn_cuda_io_dtype") == 7 \
            else np.float32
        out = np.empty(self.io_dims(True, index), dt)
        check(lib().spinn_cuda_copy_output(self._h, index, out.ctypes.data, out.nbytes), "spinn_cuda_copy_output")
        return out

    def tensor(self, tensor_id: int, dims: Sequence[int], first: int = 0, count: Optional[int] = None,
               dtype=np.float32) -> np.ndarray:
        """Items ``first .. first+count-1`` (dim 0) of ENNF tensor `tensor_id` after a run, in the
        .ennf layout (``dims`` as the .ennf declares them; ``spinn_cuda_copy_tensor``).  Any
        activation when planned with ``PLAN_KEEP``, otherwise graph outputs only."""
        count = int(dims[0]) - first if count is None else count
        out = np.empty((count,) + tuple(int(d) for d in dims[1:]), dtype)
        check(lib().spinn_cuda_copy_tensor(self._h, int(tensor_id), int(first), int(count), out.ctypes.data,
                                           out.nbytes), "spinn_cuda_copy_tensor")
        return out

    def run(self, x: np.ndarray, out: Optional[np.ndarray] = None) -> np.ndarray:
        """Host input -> host output 0 (``spinn_run``)."""
        x = np.ascontiguousarray(x, dtype=np.float32)
        if out is None:
            out = np.empty(self.io_dims(True, 0), np.float32)
        check(lib().spinn_cuda_run(self._h, x.ctypes.data, out.ctypes.data), "spinn_cuda_run")
        return out

    def run_ptr(self, host_in: int, host_out: int) -> None:
        check(lib().spinn_cuda_run(self._h, host_in, host_out), "spinn_cuda_run")

    def submit_ptr(self, host_in: int, host_out: int) -> None:
        """Queues one run (``spinn_cuda_submit``): host buffers by address, pinned for overlap;
        they must stay untouched until :meth:`wait` returns."""
        check(lib().spinn_cuda_submit(self._h, host_in or None, host_out or None), "spinn_cuda_submit")

    def wait(self) -> None:
        """Waits for every submitted run (``spinn_cuda_wait``)."""
        check(lib().spinn_cuda_wait(self._h), "spinn_cuda_wait")

    def run_device(self, stream: int = 0) -> None:
        check(lib().spinn_cuda_run_device(self._h, stream or None), "spinn_cuda_run_device")

    def run_profiled(self, stream: int = 0) -> None:
        """One run with per-step device timing (plan with PLAN_PROFILE); synchronous."""
        check(lib().spinn_cuda_run_profiled(self._h, stream or None), "spinn_cuda_run_profiled")

    def plan_info(self) -> dict:
        a, w = ctypes.c_uint64(0), ctypes.c_uint64(0)
        s, k = ctypes.c_int(0), ctypes.c_int(0)
        check(lib().spinn_cuda_plan_info(self._h, ctypes.byref(a), ctypes.byref(w), ctypes.byref(s),
                                         ctypes.byref(k)), "spinn_cuda_plan_info")
        return {"arena_bytes": a.value, "weight_bytes": w.value, "steps": s.value, "kernels": k.value}

    def step_kinds(self) -> List[int]:
        n = self.plan_info()["steps"]
        return [lib().spinn_cuda_step_kind(self._h, i) for i in range(n)]

    def profile(self):
        """(op_type, ms, flops) per step of the last run; plan with PLAN_PROFILE."""
        n = self.plan_info()["steps"]
        ops = (ctypes.c_int * n)()
        ms = (ctypes.c_float * n)()
        fl = (ctypes.c_double * n)()
        k = check(lib().spinn_cuda_profile(self._h, ops, ms, fl, n), "spinn_cuda_profile")
        return [(ops[i], ms[i], fl[i]) for i in range(k)]
