"""Host-side mirror of the reference's kernel bindings, backed by CUDA.

The reference binds its Rust/WASM kernels in
packages/engine/src/runner/wasm/wasm-kernels.ts; this module offers the same
operations with the same argument meaning and the same error behaviour
(assertWasmOk, wasm-kernels.ts:1882-1896 -> assert_cuda_ok), but every call
runs on the GPU through libheliocuda.so:

    reference (wasm-kernels.ts)             here
    ------------------------------------    ---------------------------------------
    matMulQuantizedWasm           :416      mat_mul_quantized
    createWasmQuantizedWeightHandle :520    create_quantized_weight_handle
    releaseWasmQuantizedWeightHandle :576   release_quantized_weight_handle
    matMulQuantizedWasmResident   :593      mat_mul_quantized_resident
    matMulQuantizedWasmResidentMulti :648   mat_mul_quantized_resident_multi
    matMulDequantizedWasm         :468      mat_mul_dequantized
    quantizedTypeId               :1908     quantized_type_id

Activations and outputs are torch CUDA tensors (float32); numpy arrays are
accepted too and are copied to the device and back (the host round trip is
then part of the call, as it is for the WASM linear-memory copies).
"""
from __future__ import annotations

import ctypes as C
import functools
import warnings
from dataclasses import dataclass, field

import numpy as np
import torch

from . import _lib

OK, ERR_SHAPE, ERR_HEADS, ERR_TYPE, ERR_CUDA, ERR_TIMEOUT, ERR_NCCL, ERR_ARG = range(8)

_TYPE_IDS = {"Q4_K": 1, "Q5_K": 2, "Q6_K": 3, "IQ4_XS": 4, "Q8_0": 5, "Q4_0": 6}
_TYPE_NAMES = {v: k for k, v in _TYPE_IDS.items()}


class CudaKernelError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(message)
        self.code = code


def quantized_type_id(type_name: str) -> int:
    """wasm-kernels.ts:1908-1923."""
    try:
        return _TYPE_IDS[type_name]
    except KeyError:
        raise CudaKernelError(ERR_TYPE, f"unsupported quantized type {type_name}") from None


def assert_cuda_ok(code: int, kernel_name: str) -> None:
    """wasm-kernels.ts:1882-1896, with the GPU codes added."""
    if code == OK:
        return
    detail = _lib.last_error()
    if code == ERR_SHAPE:
        raise CudaKernelError(code, f"{kernel_name} cuda shape mismatch ({detail})")
    if code == ERR_HEADS:
        raise CudaKernelError(code, f"{kernel_name} cuda head count mismatch ({detail})")
    if code == ERR_TYPE:
        raise CudaKernelError(code, f"{kernel_name} cuda unsupported type ({detail})")
    raise CudaKernelError(code, f"{kernel_name} cuda failed with code {code}: {detail}")


def init_device(device: int | None = None) -> int:
    dev = torch.cuda.current_device() if device is None else int(device)
    torch.cuda.set_device(dev)
    assert_cuda_ok(_lib.lib().hpc_device_init(dev), "deviceInit")
    return dev


def _stream() -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _as_device_f32(x) -> tuple[torch.Tensor, bool]:
    """Returns (contiguous cuda float32 tensor, came_from_host)."""
    if isinstance(x, torch.Tensor):
        if not x.is_cuda:
            return x.to(device="cuda", dtype=torch.float32).contiguous(), True
        if x.dtype != torch.float32:
            raise TypeError("activations must be float32")
        return x.contiguous(), False
    arr = np.ascontiguousarray(x, dtype=np.float32)
    return torch.from_numpy(arr).to("cuda"), True


def _ptr(t: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(t.data_ptr())


@dataclass
class CudaQuantizedWeightHandle:
    """Resident weight in HBM (wasm-kernels.ts:387-397 WasmQuantizedWeightHandle)."""
    type: str
    row_count: int
    input_size: int
    device: int
    device_bytes: int
    _h: C.c_void_p = field(repr=False)
    released: bool = False

    @property
    def handle(self) -> C.c_void_p:
        if self.released:
            raise CudaKernelError(ERR_ARG, "weight handle already released")
        return self._h


def create_quantized_weight_handle(type_name: str, weight_bytes, input_size: int,
                                   row_count: int) -> CudaQuantizedWeightHandle:
    """Upload + repack once (wasm-kernels.ts:520-574).  weight_bytes: host
    bytes/np.uint8, or a uint8 CUDA tensor already on the device."""
    if input_size <= 0 or row_count <= 0:
        raise CudaKernelError(ERR_SHAPE,
                              f"Resident quantized weight shape mismatch: inputSize={input_size} rowCount={row_count}")
    tid = quantized_type_id(type_name)
    h = C.c_void_p()
    if isinstance(weight_bytes, torch.Tensor) and weight_bytes.is_cuda:
        wb = weight_bytes.contiguous()
        code = _lib.lib().hpc_weight_upload_device(tid, _ptr(wb), wb.numel(), input_size, row_count, _stream(),
                                                    C.byref(h))
    else:
        if isinstance(weight_bytes, torch.Tensor):
            weight_bytes = weight_bytes.numpy()
        wb = np.ascontiguousarray(np.frombuffer(weight_bytes, dtype=np.uint8)
                                  if isinstance(weight_bytes, (bytes, bytearray, memoryview)) else weight_bytes,
                                  dtype=np.uint8)
        code = _lib.lib().hpc_weight_upload(tid, wb.ctypes.data_as(C.c_void_p), wb.size, input_size, row_count,
                                            C.byref(h))
    assert_cuda_ok(code, "createQuantizedWeightHandle")
    nbytes = C.c_size_t()
    _lib.lib().hpc_weight_info(h, None, None, None, C.byref(nbytes))
    return CudaQuantizedWeightHandle(type_name, row_count, input_size, torch.cuda.current_device(), nbytes.value, h)


def release_quantized_weight_handle(handle: CudaQuantizedWeightHandle) -> None:
    """wasm-kernels.ts:576-584."""
    if handle.released:
        return
    assert_cuda_ok(_lib.lib().hpc_weight_release(handle.handle), "releaseQuantizedWeightHandle")
    handle.released = True


def dequantize_resident(handle: CudaQuantizedWeightHandle) -> torch.Tensor:
    """f32 [row_count, input_size], bit-exact to lib.rs dequantize_q4_k/q6_k."""
    out = torch.empty((handle.row_count, handle.input_size), dtype=torch.float32, device="cuda")
    assert_cuda_ok(_lib.lib().hpc_weight_dequantize(handle.handle, _ptr(out), out.numel(), _stream()),
                   "dequantizeResident")
    return out


def quantize_q8_k(x: torch.Tensor, input_size: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Q8_K of each column, bit-exact to lib.rs:1774-1811: (d, qs, bsums32)."""
    x, _ = _as_device_f32(x)
    cols = x.numel() // input_size if input_size else 0
    d = torch.empty(cols * (input_size // 256), dtype=torch.float32, device="cuda")
    qs = torch.empty(cols * input_size, dtype=torch.int8, device="cuda")
    bs = torch.empty(cols * (input_size // 32), dtype=torch.int16, device="cuda")
    assert_cuda_ok(_lib.lib().hpc_quantize_q8_k(_ptr(x), x.numel(), input_size, cols, _ptr(d), _ptr(qs), _ptr(bs),
                                                _stream()), "quantizeQ8K")
    return d, qs, bs


def mat_mul_quantized_resident(handle: CudaQuantizedWeightHandle, input_columns, input_size: int, row_count: int,
                               column_count: int):
    """wasm-kernels.ts:593-646 -> hp_matmul_quantized_prepared_f32 (lib.rs:225)."""
    if handle.input_size != input_size or handle.row_count != row_count:
        raise CudaKernelError(ERR_SHAPE, f"Resident quantized matmul handle shape mismatch: "
                                         f"{handle.input_size}x{handle.row_count}")
    x, from_host = _as_device_f32(input_columns)
    if x.numel() != input_size * column_count:
        raise CudaKernelError(ERR_SHAPE, f"Resident quantized matmul input shape mismatch: {x.numel()}")
    out = torch.empty(row_count * column_count, dtype=torch.float32, device="cuda")
    code = _lib.lib().hpc_matmul_quantized_prepared_f32(handle.handle, _ptr(x), x.numel(), input_size, row_count,
                                                        column_count, _ptr(out), out.numel(), _stream())
    assert_cuda_ok(code, "matMulQuantizedResident")
    return out.cpu().numpy() if from_host else out


def mat_mul_quantized_resident_multi(handles, input_columns, input_size: int, column_count: int):
    """wasm-kernels.ts:648-749 -> hp_matmul_quantized_prepared_multi_f32
    (lib.rs:302); one launch for up to 8 weights (the reference takes 2-4)."""
    handles = list(handles)
    if not 1 <= len(handles) <= 8:
        return None
    for h in handles:
        if h.input_size != input_size:
            raise CudaKernelError(ERR_SHAPE, f"Resident quantized multi matmul handle shape mismatch: {h.input_size}")
    x, from_host = _as_device_f32(input_columns)
    if x.numel() != input_size * column_count:
        raise CudaKernelError(ERR_SHAPE, f"Resident quantized multi matmul input shape mismatch: {x.numel()}")
    outs = [torch.empty(h.row_count * column_count, dtype=torch.float32, device="cuda") for h in handles]
    n = len(handles)
    hs = (C.c_void_p * n)(*[h.handle for h in handles])
    os_ = (C.c_void_p * n)(*[o.data_ptr() for o in outs])
    ls = (C.c_size_t * n)(*[o.numel() for o in outs])
    code = _lib.lib().hpc_matmul_quantized_prepared_multi_f32(n, _ptr(x), x.numel(), input_size, column_count, hs, os_,
                                                              ls, _stream())
    assert_cuda_ok(code, "MatMulQuantizedResidentMulti")
    return [o.cpu().numpy() for o in outs] if from_host else outs


def set_wide_matmul_kind(kind: int) -> None:
    """Tensor-core kind of the >= 16-column Q4_K matmul: 0 = mma.sync
    (default), 1 = tcgen05 (hpc_set_wide_matmul_kind)."""
    assert_cuda_ok(_lib.lib().hpc_set_wide_matmul_kind(int(kind)), "setWideMatmulKind")


def mat_mul_rmsnorm(handles, x, w_pre, column_count: int, *, y=None, w_post=None, eps: float = 1e-6):
    """The decode step's norm-fused projection (hpc_matmul_rmsnorm_f32):
    h = x + rmsNorm(y) * w_post (or x when y is None), then every weight
    times Q8_K(rmsNorm(h) * w_pre) -- wasm/layers.ts:161-247's rmsNorm,
    quantize_q8_k and hp_matmul_quantized_prepared_multi_f32 in one launch.
    Device tensors in; returns (outputs, h or None)."""
    handles = list(handles)
    n = len(handles)
    if not 1 <= n <= 8:
        raise CudaKernelError(ERR_SHAPE, f"matMulRmsNorm: {n} weights")
    d = int(handles[0].input_size)
    for t in (x, w_pre) + ((y, w_post) if y is not None else ()):
        if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
            raise CudaKernelError(ERR_ARG, "matMulRmsNorm: contiguous f32 device tensors")
    nbytes = C.c_size_t()
    assert_cuda_ok(_lib.lib().hpc_q8_workspace_bytes(d, column_count, C.byref(nbytes)), "q8 workspace")
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device="cuda")
    outs = [torch.empty(h.row_count * column_count, dtype=torch.float32, device="cuda") for h in handles]
    x_out = torch.empty_like(x) if y is not None else None
    hs = (C.c_void_p * n)(*[h.handle for h in handles])
    os_ = (C.c_void_p * n)(*[o.data_ptr() for o in outs])
    ls = (C.c_size_t * n)(*[o.numel() for o in outs])
    code = _lib.lib().hpc_matmul_rmsnorm_f32(n, hs, _ptr(ws), nbytes.value, d, column_count, _ptr(x),
                                             _ptr(y) if y is not None else None,
                                             _ptr(w_post) if w_post is not None else None, _ptr(w_pre),
                                             float(eps), _ptr(x_out) if x_out is not None else None, os_, ls,
                                             _stream())
    assert_cuda_ok(code, "matMulRmsNorm")
    return outs, x_out


def mat_mul_quantized(type_name: str, weight_bytes, input_columns, input_size: int, row_count: int,
                      column_count: int) -> np.ndarray:
    """wasm-kernels.ts:416-466 -> hp_matmul_quantized_f32 (lib.rs:41): host
    buffers in and out, nothing stays resident."""
    tid = quantized_type_id(type_name)
    w = np.ascontiguousarray(np.frombuffer(weight_bytes, dtype=np.uint8)
                             if isinstance(weight_bytes, (bytes, bytearray, memoryview)) else weight_bytes,
                             dtype=np.uint8)
    x = np.ascontiguousarray(input_columns, dtype=np.float32)
    if x.size != input_size * column_count:
        raise CudaKernelError(ERR_SHAPE, f"Quantized matmul input shape mismatch: {x.size}")
    out = np.empty(row_count * column_count, np.float32)
    code = _lib.lib().hpc_matmul_quantized_f32(tid, w.ctypes.data_as(C.c_void_p), w.size,
                                               x.ctypes.data_as(C.c_void_p), x.size, input_size, row_count,
                                               column_count, out.ctypes.data_as(C.c_void_p), out.size)
    assert_cuda_ok(code, "matMulQuantized")
    return out


def mat_mul_dequantized(type_name: str, weight_bytes, input_columns, input_size: int, row_count: int,
                        column_count: int) -> np.ndarray:
    """wasm-kernels.ts:468-520 matMulDequantizedWasm -> hp_matmul_dequantized_f32
    (lib.rs:103-154): bit-exact dequantized rows times the input columns with
    the reference's sequential f32 sum; host buffers in and out."""
    tid = quantized_type_id(type_name)
    w = np.ascontiguousarray(np.frombuffer(weight_bytes, dtype=np.uint8)
                             if isinstance(weight_bytes, (bytes, bytearray, memoryview)) else weight_bytes,
                             dtype=np.uint8)
    x = np.ascontiguousarray(input_columns, dtype=np.float32)
    if x.size != input_size * column_count:
        raise CudaKernelError(ERR_SHAPE, f"Dequantized matmul input shape mismatch: {x.size}")
    out = np.empty(row_count * column_count, np.float32)
    code = _lib.lib().hpc_matmul_dequantized_f32(tid, w.ctypes.data_as(C.c_void_p), w.size,
                                                 x.ctypes.data_as(C.c_void_p), x.size, input_size, row_count,
                                                 column_count, out.ctypes.data_as(C.c_void_p), out.size)
    assert_cuda_ok(code, "matMulDequantized")
    return out


def mat_mul_dequantized_resident(handle: CudaQuantizedWeightHandle, input_columns, input_size: int, row_count: int,
                                 column_count: int):
    """The same arithmetic on a resident weight (hpc_matmul_dequantized_prepared_f32)."""
    x, from_host = _as_device_f32(input_columns)
    out = torch.empty(row_count * column_count, dtype=torch.float32, device="cuda")
    code = _lib.lib().hpc_matmul_dequantized_prepared_f32(handle.handle, _ptr(x), x.numel(), input_size, row_count,
                                                          column_count, _ptr(out), out.numel(), _stream())
    assert_cuda_ok(code, "matMulDequantizedResident")
    return out.cpu().numpy() if from_host else out


def lm_head_topk(handle: CudaQuantizedWeightHandle, hidden, column_count: int, k: int, *, softcap: float = 0.0,
                 id_offset: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Fused LM head + top-k on normed hidden columns: (ids, values), each
    [column_count, k], ordered by value descending then id ascending
    (runtime.ts:514-527).  softcap > 0 applies fround(tanh(v/c)*c) after
    selection (mergeTopCandidates, webgpu/segment-runner.ts:3773-3794)."""
    x, from_host = _as_device_f32(hidden)
    if x.numel() != handle.input_size * column_count:
        raise CudaKernelError(ERR_SHAPE, f"LM head hidden shape mismatch: {x.numel()}")
    ids = torch.empty((column_count, k), dtype=torch.int32, device="cuda")
    vals = torch.empty((column_count, k), dtype=torch.float32, device="cuda")
    code = _lib.lib().hpc_lm_head_topk(handle.handle, _ptr(x), x.numel(), handle.input_size, column_count, k,
                                       id_offset, softcap, _ptr(ids), _ptr(vals), _stream())
    assert_cuda_ok(code, "lmHeadTopK")
    if from_host:
        return ids.cpu(), vals.cpu()
    return ids, vals


def sample_candidates(ids: torch.Tensor, vals: torch.Tensor, *, top_k: int, top_p: float, temperature: float,
                      greedy: bool, rng_state: int, token_out: torch.Tensor, table: torch.Tensor | None = None,
                      scale: float = 1.0, row_out: torch.Tensor | None = None) -> None:
    """The sampler's token draw on the device (hpc_sample_candidates): ids /
    vals a sorted candidate list (device int32 / f32), token_out a device
    int32 slot; with `table` ([rows][hidden] f32) the chosen row * scale goes
    to row_out.  Nothing is read back (no synchronization)."""
    if ids.dtype != torch.int32 or vals.dtype != torch.float32 or not ids.is_cuda or not vals.is_cuda:
        raise CudaKernelError(ERR_TYPE, "sample: candidates must be device int32 ids and f32 values")
    n = ids.numel()
    rows, hidden = (table.shape[0], table.shape[1]) if table is not None else (0, 0)
    if table is not None and (row_out is None or row_out.numel() < hidden or table.dtype != torch.float32
                              or not table.is_contiguous()):
        raise CudaKernelError(ERR_SHAPE, "sample: the table must be contiguous f32 and row_out hold a row")
    code = _lib.lib().hpc_sample_candidates(_ptr(ids), _ptr(vals), n, max(1, int(top_k)), float(top_p),
                                            float(temperature), 1 if greedy else 0, int(rng_state) & 0xFFFFFFFF,
                                            _ptr(token_out), _ptr(table) if table is not None else None, rows,
                                            hidden, float(scale), _ptr(row_out) if row_out is not None else None,
                                            _stream())
    assert_cuda_ok(code, "sampleCandidates")


def set_matmul_order(exact: bool) -> None:
    """Reference f32 order (default) or the reordered kernels for the matmul
    and LM-head calls (hpc_set_matmul_order)."""
    assert_cuda_ok(_lib.lib().hpc_set_matmul_order(int(bool(exact))), "setMatmulOrder")


def device_error() -> None:
    """Raises CudaKernelError: ERR_TIMEOUT if a kernel's bounded wait gave up,
    ERR_SHAPE if a paged batch pointed outside its buffers."""
    assert_cuda_ok(_lib.lib().hpc_device_error(), "deviceStatus")


# ---- serving many sequences: paged KV cache and its attention ---------------------

# csrc/hc_host.cpp: the four calls below in their plain case, at a third of
# the host time.  Its functions answer NotImplemented for everything else, which
# then goes the whole way here.
_host = None


class _NoHost:
    """In the host module's place where it does not load: every call goes the
    whole way here, to the same kernels."""

    @staticmethod
    def append(*args):
        return NotImplemented

    paged = prompt = logits = append


def _load_host():
    global _host
    lib = _lib.lib()
    try:
        from . import _host as module
        built_for = getattr(module, "built_for", "another version")
        if built_for != _lib.host_built_for():
            raise ImportError(f"it was built for {built_for}")
    except ImportError as e:
        warnings.warn(f"heliopause_b200._host does not load ({e}): serving calls take some 10 us longer on the host; run "
                      "`python -m heliopause_b200.build`", RuntimeWarning, stacklevel=3)
        _host = _NoHost
        return _host
    module.bind(*(C.cast(getattr(lib, "hpc_" + name), C.c_void_p).value for name in (
        "paged_kv_append", "attention_workspace_bytes", "paged_attention", "prompt_attention",
        "logits_topk_workspace_bytes", "logits_topk")))
    _host = module
    return module

_DTYPE_IDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _raw_stream(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)


def _check_i32(name: str, dev: int, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous():
            raise CudaKernelError(ERR_ARG, f"{name}: starts, lengths and page tables are contiguous int32 tensors on "
                                           f"cuda:{dev}")


def _rows3(name: str, t: torch.Tensor, dev: int, shape: tuple) -> tuple[torch.Tensor, int]:
    """[rows][heads][dim] on the device, heads and elements contiguous within a row; and its row stride."""
    if t.shape != shape or t.get_device() != dev:
        raise CudaKernelError(ERR_SHAPE, f"{name}: {shape} on cuda:{dev}, not {tuple(t.shape)} on {t.device}")
    rows, heads, dim = shape
    st = t.stride()
    if st[2] != 1 or (st[1] != dim and heads > 1) or st[0] % 8 or st[0] < heads * dim or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format), heads * dim
    return t, st[0]


def _check_cache(name: str, key_cache: torch.Tensor, value_cache: torch.Tensor) -> None:
    if key_cache.dim() != 4 or key_cache.shape != value_cache.shape or key_cache.dtype != value_cache.dtype:
        raise CudaKernelError(ERR_SHAPE, f"{name}: key and value caches are [pages][page_size][kv_heads][head_dim]")
    if not (key_cache.is_cuda and key_cache.get_device() == value_cache.get_device() and key_cache.is_contiguous()
            and value_cache.is_contiguous()):
        raise CudaKernelError(ERR_ARG, f"{name}: the caches are contiguous tensors on one device")


def _check_batch(name: str, dev: int, page_table: torch.Tensor, query_starts: torch.Tensor,
                 kv_lens: torch.Tensor) -> tuple[int, int]:
    """Sequences and the page table's width."""
    _check_i32(name, dev, page_table, query_starts, kv_lens)
    seqs, table = kv_lens.numel(), page_table.shape
    if len(table) != 2 or table[0] != seqs or query_starts.numel() != seqs + 1:
        raise CudaKernelError(ERR_SHAPE, f"{name}: {seqs} sequences, a table of {tuple(table)}, "
                                         f"{query_starts.numel()} starts")
    return seqs, table[1]


def paged_kv_append(k: torch.Tensor, v: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                    page_table: torch.Tensor, query_starts: torch.Tensor, kv_lens: torch.Tensor, *,
                    q: torch.Tensor | None = None, inv_freq: torch.Tensor | None = None,
                    q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, norm_v: bool = False,
                    eps: float = 1e-6, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """New tokens into a paged KV cache (hpc_paged_kv_append): per-head RMS
    norms, the NeoX rotation by position * inv_freq (f64) and the write into
    each token's page, in place; returns the queries normed and rotated in
    the cache's type (q_out, or a new tensor), or None without q.

    k, v, q: [rows][heads][head_dim], f32 or the cache's type, views with a
    row stride allowed.  key_cache, value_cache: [pages][page_size][kv_heads]
    [head_dim].  Sequence s owns rows query_starts[s] .. query_starts[s+1];
    kv_lens[s] is its length with them; its token j lies in page
    page_table[s][j // page_size].  Rows behind the last sequence are left."""
    done = (_host or _load_host()).append(k, v, key_cache, value_cache, page_table, query_starts, kv_lens, q, inv_freq,
                                          q_norm, k_norm, norm_v, eps, q_out)
    if done is not NotImplemented:
        return done
    name = "pagedKvAppend"
    _check_cache(name, key_cache, value_cache)
    dev, dt = key_cache.get_device(), key_cache.dtype
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return paged_kv_append(k, v, key_cache, value_cache, page_table, query_starts, kv_lens, q=q,
                                   inv_freq=inv_freq, q_norm=q_norm, k_norm=k_norm, norm_v=norm_v, eps=eps, q_out=q_out)
    pages, page_size, kv_heads, dim = key_cache.shape
    seqs, width = _check_batch(name, dev, page_table, query_starts, kv_lens)
    xt = k.dtype
    if k.dim() != 3 or v.shape != k.shape or v.dtype != xt:
        raise CudaKernelError(ERR_SHAPE, f"{name}: keys of {tuple(k.shape)} {xt}, values of {tuple(v.shape)} {v.dtype}")
    if dt not in _DTYPE_IDS or xt not in _DTYPE_IDS:
        raise CudaKernelError(ERR_TYPE, f"{name}: {xt} into a cache of {dt}")
    rows, heads = k.shape[0], kv_heads
    shape = (rows, kv_heads, dim)
    k, ks = _rows3(name, k, dev, shape)
    v, vs = _rows3(name, v, dev, shape)
    qp = op = None
    qs = 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != rows or q.dtype != xt:
            raise CudaKernelError(ERR_SHAPE, f"{name}: queries and keys differ in rows or type")
        heads = q.shape[1]
        shape = (rows, heads, dim)
        q, qs = _rows3(name, q, dev, shape)
        if q_out is None:
            q_out = key_cache.new_empty(shape)
        elif q_out.shape != shape or q_out.dtype != dt or q_out.get_device() != dev or not q_out.is_contiguous():
            raise CudaKernelError(ERR_SHAPE, f"{name}: q_out is contiguous {shape} of {dt}")
        qp, op = q.data_ptr(), q_out.data_ptr()
    fp, half = None, 0
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float64 or inv_freq.get_device() != dev or not inv_freq.is_contiguous():
            raise CudaKernelError(ERR_ARG, f"{name}: inv_freq is a contiguous float64 tensor on cuda:{dev}")
        half = inv_freq.numel()
        fp = inv_freq.data_ptr() if half else None
    norms = [None, None]
    for i, w in enumerate((q_norm, k_norm)):
        if w is not None:
            if w.dtype is not torch.float32 or w.numel() != dim or w.get_device() != dev or not w.is_contiguous():
                raise CudaKernelError(ERR_ARG, f"{name}: norm weights are {dim} contiguous float32 values on cuda:{dev}")
            norms[i] = w.data_ptr()
    code = _lib.lib().hpc_paged_kv_append(
        k.data_ptr(), ks, v.data_ptr(), vs, qp, qs, _DTYPE_IDS[xt], rows, heads, kv_heads, dim, fp, half, norms[0],
        norms[1], norm_v, eps, key_cache.data_ptr(), value_cache.data_ptr(), _DTYPE_IDS[dt], pages, page_size,
        page_table.data_ptr(), width, query_starts.data_ptr(), kv_lens.data_ptr(), seqs, op, _raw_stream(dev))
    if code:
        assert_cuda_ok(code, name)
    return q_out if q is not None else None


class _workspace:
    """Device memory for the length of one call on the current stream: the
    allocator hands a freed block on in stream order, as with a tensor, at a
    third of a tensor's cost (0.5 us against 1.5)."""
    __slots__ = ("ptr",)

    def __init__(self, nbytes: int, stream: int):
        self.ptr = torch._C._cuda_cudaCachingAllocator_raw_alloc(nbytes, stream)

    def __enter__(self) -> int:
        return self.ptr

    def __exit__(self, *exc):
        torch._C._cuda_cudaCachingAllocator_raw_delete(self.ptr)


@functools.lru_cache(maxsize=None)
def _attention_workspace(heads: int, kv_heads: int, dim: int) -> int:
    n = C.c_size_t()
    assert_cuda_ok(_lib.lib().hpc_attention_workspace_bytes(heads, kv_heads, dim, C.byref(n)), "attentionWorkspace")
    return n.value


def _attention_out(name: str, dev: int, shape: tuple, q: torch.Tensor, out, out_dtype, return_lse):
    dt = out.dtype if out is not None else out_dtype or q.dtype
    if dt not in _DTYPE_IDS:
        raise CudaKernelError(ERR_TYPE, f"{name}: output of {dt}")
    if out is None:
        out = q.new_empty(shape) if dt is q.dtype else q.new_empty(shape, dtype=dt)
    elif out.shape != shape or out.get_device() != dev or not out.is_contiguous():
        raise CudaKernelError(ERR_SHAPE, f"{name}: out is contiguous {shape} on cuda:{dev}")
    lse = torch.full(shape[:2], -torch.inf, dtype=torch.float32, device=q.device) if return_lse else None
    return out, lse


def paged_attention(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, page_table: torch.Tensor,
                    query_starts: torch.Tensor, kv_lens: torch.Tensor, *, max_query_len: int, scale: float,
                    window: int = 0, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                    return_lse: bool = False):
    """Causal attention of every sequence's newest rows over its pages
    (hpc_paged_attention): decode (one row each), verify, or chunks of
    prompts.  Arguments as paged_kv_append's; window > 0: a row sees that
    many keys, itself included.  max_query_len: the most rows of a sequence.
    out may be a contiguous q itself, and lies over no other input.
    Returns [rows][heads][head_dim] (and the log-sum-exp [rows][heads] with
    return_lse)."""
    if not return_lse:
        done = (_host or _load_host()).paged(q, key_cache, value_cache, page_table, query_starts, kv_lens, max_query_len,
                                             scale, window, out, out_dtype)
        if done is not NotImplemented:
            return done
    name = "pagedAttention"
    _check_cache(name, key_cache, value_cache)
    dev, dt = key_cache.get_device(), key_cache.dtype
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return paged_attention(q, key_cache, value_cache, page_table, query_starts, kv_lens,
                                   max_query_len=max_query_len, scale=scale, window=window, out=out,
                                   out_dtype=out_dtype, return_lse=return_lse)
    pages, page_size, kv_heads, dim = key_cache.shape
    seqs, width = _check_batch(name, dev, page_table, query_starts, kv_lens)
    if q.dim() != 3 or q.dtype != dt:
        raise CudaKernelError(ERR_TYPE, f"{name}: queries of {q.dtype} over a cache of {dt}")
    rows, heads, _ = q.shape
    shape = (rows, heads, dim)
    q, qs = _rows3(name, q, dev, shape)
    if max_query_len < 0 or window < 0:
        raise CudaKernelError(ERR_SHAPE, f"{name}: max_query_len {max_query_len}, window {window}")
    out, lse = _attention_out(name, dev, shape, q, out, out_dtype, return_lse)
    nbytes, stream = _attention_workspace(heads, kv_heads, dim), _raw_stream(dev)
    with _workspace(nbytes, stream) as ws:
        code = _lib.lib().hpc_paged_attention(
            q.data_ptr(), qs, key_cache.data_ptr(), value_cache.data_ptr(), _DTYPE_IDS.get(dt, -1), pages, page_size,
            page_table.data_ptr(), width, query_starts.data_ptr(), kv_lens.data_ptr(), seqs, rows, heads, kv_heads, dim,
            max_query_len, scale, window, ws, nbytes, out.data_ptr(), _DTYPE_IDS[out.dtype],
            lse.data_ptr() if return_lse else None, stream)
    if code:
        assert_cuda_ok(code, name)
    return (out, lse) if return_lse else out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, query_starts: torch.Tensor, *,
                     max_query_len: int, scale: float, window: int = 0, out: torch.Tensor | None = None,
                     out_dtype: torch.dtype | None = None, return_lse: bool = False):
    """Causal attention over whole prompts packed row behind row
    (hpc_prompt_attention): q [rows][heads][head_dim], k and v
    [rows][kv_heads][head_dim] (f16 or bf16; views with a row stride allowed),
    sequence s = rows query_starts[s] .. query_starts[s+1]."""
    if not return_lse:
        done = (_host or _load_host()).prompt(q, k, v, query_starts, max_query_len, scale, window, out, out_dtype)
        if done is not NotImplemented:
            return done
    name = "promptAttention"
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or not q.is_cuda:
        raise CudaKernelError(ERR_SHAPE, f"{name}: q, k and v are [rows][heads][head_dim] device tensors")
    dev, dt = q.get_device(), q.dtype
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return prompt_attention(q, k, v, query_starts, max_query_len=max_query_len, scale=scale, window=window,
                                    out=out, out_dtype=out_dtype, return_lse=return_lse)
    if k.dtype != dt or v.dtype != dt:
        raise CudaKernelError(ERR_TYPE, f"{name}: queries of {dt}, keys of {k.dtype}, values of {v.dtype}")
    shape = rows, heads, dim = q.shape
    kv_rows, kv_heads, _ = k.shape
    if kv_rows != rows:
        raise CudaKernelError(ERR_SHAPE, f"{name}: {rows} query rows, {kv_rows} key rows")
    _check_i32(name, dev, query_starts)
    seqs = query_starts.numel() - 1
    if seqs < 0:
        raise CudaKernelError(ERR_SHAPE, f"{name}: query_starts is empty")
    q, qs = _rows3(name, q, dev, shape)
    k, ks = _rows3(name, k, dev, (rows, kv_heads, dim))
    v, vs = _rows3(name, v, dev, (rows, kv_heads, dim))
    if max_query_len < 0 or window < 0:
        raise CudaKernelError(ERR_SHAPE, f"{name}: max_query_len {max_query_len}, window {window}")
    out, lse = _attention_out(name, dev, shape, q, out, out_dtype, return_lse)
    nbytes, stream = _attention_workspace(heads, kv_heads, dim), _raw_stream(dev)
    with _workspace(nbytes, stream) as ws:
        code = _lib.lib().hpc_prompt_attention(
            q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, _DTYPE_IDS.get(dt, -1), query_starts.data_ptr(), seqs,
            rows, heads, kv_heads, dim, max_query_len, scale, window, ws, nbytes, out.data_ptr(), _DTYPE_IDS[out.dtype],
            lse.data_ptr() if return_lse else None, stream)
    if code:
        assert_cuda_ok(code, name)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=256)
def _logits_workspace(rows: int, vocab: int, k: int) -> int:
    n = C.c_size_t()
    assert_cuda_ok(_lib.lib().hpc_logits_topk_workspace_bytes(rows, vocab, k, C.byref(n)), "logitsTopK")
    return n.value


def logits_topk(logits: torch.Tensor, k: int, *, history: torch.Tensor | None = None,
                history_starts: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                presence: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                bias_values: torch.Tensor | None = None, bias_starts: torch.Tensor | None = None,
                allowed: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Penalties for repeated tokens, biases and a grammar mask on logits
    [rows][vocab] (f32), and the k best of every row (hpc_logits_topk): ids
    (int32) and values, [rows][k], in the order sample_candidates takes;
    (-1, -inf) where a row has fewer than k tokens left.

    history: the rows' tokens one behind the other, row r's at
    history_starts[r] .. [r+1], its first prompt_lens[r] of the prompt;
    repetition, frequency, presence: one f32 per row; bias_ids / bias_values:
    the same for biases with bias_starts; allowed: int32 words of 32 tokens,
    [rows][>= ceil(vocab / 32)].  Logits and their history entries stay as
    they are."""
    done = (_host or _load_host()).logits(logits, k, history, history_starts, prompt_lens, repetition, frequency, presence,
                                          bias_ids, bias_values, bias_starts, allowed)
    if done is not NotImplemented:
        return done
    name = "logitsTopK"
    if logits.dim() != 2 or logits.dtype is not torch.float32 or not logits.is_cuda:
        raise CudaKernelError(ERR_TYPE, f"{name}: logits are [rows][vocab] float32 on a device")
    dev = logits.get_device()
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return logits_topk(logits, k, history=history, history_starts=history_starts, prompt_lens=prompt_lens,
                               repetition=repetition, frequency=frequency, presence=presence, bias_ids=bias_ids,
                               bias_values=bias_values, bias_starts=bias_starts, allowed=allowed)
    rows, vocab = logits.shape
    stride, one = logits.stride()
    if one != 1 or stride < vocab:
        logits = logits.contiguous()
        stride = vocab
    if rows <= 1:
        stride = max(vocab, 1)

    def ptr(t, dtype, count, what):
        if t is None:
            return None
        if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous() or (count >= 0 and t.numel() != count):
            raise CudaKernelError(ERR_SHAPE, f"{name}: {what} is contiguous {dtype} on cuda:{dev}"
                                             + ("" if count < 0 else f" with {count} values"))
        return t.data_ptr() or None

    if (history is None) != (history_starts is None):
        raise CudaKernelError(ERR_ARG, f"{name}: history and history_starts go together")
    if (bias_ids is None) != (bias_starts is None) or (bias_ids is None) != (bias_values is None):
        raise CudaKernelError(ERR_ARG, f"{name}: bias_ids, bias_values and bias_starts go together")
    i32, f32 = torch.int32, torch.float32
    astride = 0
    if allowed is not None:
        if allowed.dim() != 2 or allowed.shape[0] != rows:
            raise CudaKernelError(ERR_SHAPE, f"{name}: allowed is [rows][words]")
        astride = allowed.shape[1]
    hist_n = history.numel() if history is not None else 0
    bias_n = bias_ids.numel() if bias_ids is not None else 0
    args = (ptr(history, i32, -1, "history"), hist_n, ptr(history_starts, i32, rows + 1, "history_starts"),
            ptr(prompt_lens, i32, rows, "prompt_lens"), ptr(repetition, f32, rows, "repetition"),
            ptr(frequency, f32, rows, "frequency"), ptr(presence, f32, rows, "presence"),
            ptr(bias_ids, i32, -1, "bias_ids"), ptr(bias_values, f32, bias_n, "bias_values"), bias_n,
            ptr(bias_starts, i32, rows + 1, "bias_starts"), ptr(allowed, i32, -1, "allowed"), astride)
    nbytes, stream = _logits_workspace(rows, vocab, k), _raw_stream(dev)
    vals = logits.new_empty((rows, k))
    ids = torch.empty_like(vals, dtype=i32)
    with _workspace(nbytes, stream) as ws:
        code = _lib.lib().hpc_logits_topk(logits.data_ptr(), stride, rows, vocab, k, *args, ws, nbytes, ids.data_ptr(),
                                          vals.data_ptr(), stream)
    if code:
        assert_cuda_ok(code, name)
    return ids, vals
