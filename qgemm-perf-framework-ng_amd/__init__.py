"""qgemm-perf-framework-ng_amd — MI355X (gfx950) backend for the quantized GGML GEMM path.

Python binding of the C-ABI in include/pfng_hip.h (libpfng_hip.so, built
in-tree by the Makefile beside this file). The library operates on device
memory; this module passes torch tensors' device pointers and the current HIP
stream. Block buffers are uint8 tensors holding the GGML block bytes
(include/pfng_blocks.h), shaped (rows, blocks_per_row * block_bytes).

There is no CPU fallback: every call goes to the HIP library, and loading
fails loudly when libpfng_hip.so is missing.
"""
from __future__ import annotations

import ctypes
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libpfng_hip.so")

# pfng_quantization_type (include/pfng_blocks.h), numbered as the reference's QuantizationType
Q4_0, Q4_K, IQ2_XXS = 0, 1, 2
TYPE_NAMES = {Q4_0: "q4_0", Q4_K: "q4_K", IQ2_XXS: "iq2_xxs"}
# pfng_path
PATH_AUTO, PATH_GEMV, PATH_MFMA, PATH_NAIVE = 0, 1, 2, 3
PATH_NAMES = {PATH_AUTO: "auto", PATH_GEMV: "gemv", PATH_MFMA: "mfma", PATH_NAIVE: "naive"}
# pfng_status
OK, ERR_INVALID_ARGUMENT, ERR_UNSUPPORTED, ERR_HIP, ERR_DEVICE = 0, 1, 2, 3, 4

QK = {Q4_0: 32, Q4_K: 256, IQ2_XXS: 256}
WEIGHT_BLOCK_BYTES = {Q4_0: 18, Q4_K: 144, IQ2_XXS: 66}
ACT_BLOCK_BYTES = {Q4_0: 34, Q4_K: 292, IQ2_XXS: 292}


class PfngError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"pfng status {status}: {message}")
        self.status = status


def build(jobs: int = 8) -> None:
    """Compile libpfng_hip.so for gfx950 (hipcc cross-compiles without a GPU)."""
    subprocess.run(["make", "-s", "-C", HERE, f"-j{jobs}"], check=True)


_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `make -C {HERE}` (no CPU fallback exists)")
        # torch carries its own HIP runtime (torch/lib/libamdhip64.so, soname
        # libamdhip64.so.7, which torch's libraries name without the version).
        # Loaded first, it satisfies the library's libamdhip64.so.7 and both
        # share one runtime; loaded after the library, it would come in as a
        # second runtime beside ROCm's, and the library's runtime then fails on
        # the device torch holds. The tensors and streams this binding passes
        # belong to torch's runtime, so load torch first.
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        L = ctypes.CDLL(LIB_PATH)
        vp, i64, sz, ci = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t, ctypes.c_int
        L.pfng_hip_last_error.restype = ctypes.c_char_p
        L.pfng_hip_version.restype = ctypes.c_char_p
        L.pfng_hip_device_check.argtypes = [ctypes.c_char_p, sz, ctypes.POINTER(ctypes.c_int)]
        for name in ("pfng_hip_quantize_q8_0", "pfng_hip_quantize_q8_K", "pfng_hip_quantize_q4_0",
                     "pfng_hip_quantize_q4_K"):
            getattr(L, name).argtypes = [vp, vp, i64, i64, vp]
        for name in ("pfng_hip_mul_mat_q4_0_q8_0", "pfng_hip_mul_mat_q4_K_q8_K", "pfng_hip_mul_mat_iq2_xxs_q8_K"):
            getattr(L, name).argtypes = [vp, vp, vp, i64, i64, i64, ci, vp]
        L.pfng_hip_mul_mat.argtypes = [ci, vp, vp, vp, i64, i64, i64, ci, vp]
        L.pfng_hip_auto_path.argtypes = [ci, i64, i64, i64]
        L.pfng_hip_compute_workspace_size.restype = sz
        L.pfng_hip_compute_workspace_size.argtypes = [ci, i64, i64]
        L.pfng_hip_compute.argtypes = [ci, vp, vp, vp, i64, i64, i64, vp, sz, ci, vp]
        L.pfng_hip_compute_noalloc.argtypes = [ci, vp, vp, vp, i64, i64, i64, ci, vp]
        L.pfng_hip_block_isums.argtypes = [ci, vp, vp, vp, i64, i64, i64, vp]
        f32 = ctypes.c_float
        L.pfng_hip_kv4_page_bytes.restype = i64
        L.pfng_hip_kv4_page_bytes.argtypes = [ci, ci]
        L.pfng_hip_kv_block_tables.argtypes = [vp, vp, ci, vp, i64, ci, vp, i64, ci, i64, vp, vp, vp, vp, vp, vp]
        L.pfng_hip_qk_norm_rope.argtypes = [vp, i64, vp, i64, ci, vp, i64, vp, i64, ci, vp, vp, f32, vp, i64, ci, ci,
                                            vp, i64, ci, ci, ci, vp]
        L.pfng_hip_kv4_store.argtypes = [vp, i64, vp, i64, ci, vp, i64, vp, i64, ci, ci, ci, vp]
        L.pfng_hip_kv4_read.argtypes = [vp, i64, ci, ci, ci, vp, i64, vp, vp, ci, vp]
        L.pfng_hip_attention_kv4_workspace_size.restype = i64
        L.pfng_hip_attention_kv4_workspace_size.argtypes = [ci, i64, i64, ci, ci, ci, ci, i64, i64]
        L.pfng_hip_attention_kv4.argtypes = [vp, i64, vp, i64, ci, vp, vp, i64, i64, ci, vp, i64, ci, vp, i64, ci, ci,
                                             ci, f32, ci, i64, i64, i64, vp, i64, vp]
        L.pfng_host_create_input.argtypes = [ci, ci, ctypes.c_uint32, sz, sz, sz, vp, vp]
        L.pfng_host_quantize_weights.argtypes = [ci, vp, vp, sz, sz]
        L.pfng_host_compute.argtypes = [ci, vp, vp, vp, sz, sz, sz, sz]
        L.pfng_host_fp32_to_fp16.restype = ctypes.c_uint16
        L.pfng_host_fp32_to_fp16.argtypes = [ctypes.c_float]
        L.pfng_host_fp16_to_fp32.restype = ctypes.c_float
        L.pfng_host_fp16_to_fp32.argtypes = [ctypes.c_uint16]
        L.pfng_host_checksum.restype = ctypes.c_double
        L.pfng_host_checksum.argtypes = [vp, sz]
        _lib = L
    return _lib


# C-ABI symbols declared in include/pfng_hip.h
EXPORTED_SYMBOLS = (
    "pfng_hip_last_error", "pfng_hip_version", "pfng_hip_device_check",
    "pfng_hip_quantize_q8_0", "pfng_hip_quantize_q8_K", "pfng_hip_quantize_q4_0", "pfng_hip_quantize_q4_K",
    "pfng_hip_mul_mat_q4_0_q8_0", "pfng_hip_mul_mat_q4_K_q8_K", "pfng_hip_mul_mat_iq2_xxs_q8_K",
    "pfng_hip_mul_mat", "pfng_hip_auto_path", "pfng_hip_compute_workspace_size", "pfng_hip_compute",
    "pfng_hip_compute_noalloc", "pfng_hip_block_isums", "pfng_hip_kv4_page_bytes", "pfng_hip_kv_block_tables",
    "pfng_hip_qk_norm_rope", "pfng_hip_kv4_store", "pfng_hip_kv4_read", "pfng_hip_attention_kv4_workspace_size",
    "pfng_hip_attention_kv4",
)
# host-side C-ABI declared in include/pfng_host.h
HOST_SYMBOLS = (
    "pfng_host_create_input", "pfng_host_quantize_weights", "pfng_host_compute", "pfng_host_fp32_to_fp16",
    "pfng_host_fp16_to_fp32", "pfng_host_checksum",
)
INPUT_REFERENCE, INPUT_BASELINE = 0, 1


def last_error() -> str:
    return lib().pfng_hip_last_error().decode()


def check(status: int) -> None:
    if status:
        raise PfngError(status, last_error())


def version() -> str:
    return lib().pfng_hip_version().decode()


def device_check() -> tuple[str, int]:
    arch = ctypes.create_string_buffer(64)
    cus = ctypes.c_int(0)
    check(lib().pfng_hip_device_check(arch, 64, ctypes.byref(cus)))
    return arch.value.decode(), cus.value


# ---------------------------------------------------------------------------
# host-side input generation (bench/framework/benchmark.cpp:29-94)
# ---------------------------------------------------------------------------

def create_input(qtype: int, m: int, n: int, k: int, seed: int = 1, variant: int = INPUT_BASELINE):
    """Synthetic inputs as the reference harness makes them: returns (activation
    float32 (m, k), weight uint8 (n, k/QK * block_bytes)) as numpy arrays."""
    import numpy as np
    act = np.empty((m, k), np.float32)
    w = np.empty((n, (k // QK[qtype]) * WEIGHT_BLOCK_BYTES[qtype]), np.uint8)
    rc = lib().pfng_host_create_input(qtype, variant, seed, m, n, k, act.ctypes.data, w.ctypes.data)
    if rc != 0:
        raise ValueError(f"pfng_host_create_input({TYPE_NAMES.get(qtype, qtype)}, m={m}, n={n}, k={k}) failed: {rc}")
    return act, w


def quantize_weights(qtype: int, x):
    """Host weight quantizer of the reference (q4_0 or q4_K): float32 (rows, k)
    -> uint8 (rows, k/QK * block_bytes)."""
    import numpy as np
    x = np.ascontiguousarray(x, dtype=np.float32)
    rows, k = x.shape
    y = np.empty((rows, (k // QK[qtype]) * WEIGHT_BLOCK_BYTES[qtype]), np.uint8)
    rc = lib().pfng_host_quantize_weights(qtype, x.ctypes.data, y.ctypes.data, rows, k)
    if rc != 0:
        raise ValueError(f"pfng_host_quantize_weights({TYPE_NAMES.get(qtype, qtype)}, k={k}) failed: {rc}")
    return y


def host_compute(qtype: int, activation, weight, n: int, threads: int = 1):
    """llama_reference::compute on the host (the harness's verification
    reference): float32 (m, k) activations and uint8 weight blocks -> float32 (m, n)."""
    import numpy as np
    act = np.ascontiguousarray(activation, dtype=np.float32)
    w = np.ascontiguousarray(weight, dtype=np.uint8)
    m, k = act.shape
    out = np.empty((m, n), np.float32)
    if qtype in QK and k % QK[qtype] == 0 and w.nbytes < n * (k // QK[qtype]) * WEIGHT_BLOCK_BYTES[qtype]:
        raise ValueError("weight buffer is smaller than n rows of k/QK blocks")
    rc = lib().pfng_host_compute(qtype, act.ctypes.data, w.ctypes.data, out.ctypes.data, m, n, k, threads)
    if rc != 0:
        raise ValueError(f"pfng_host_compute({TYPE_NAMES.get(qtype, qtype)}, m={m}, n={n}, k={k}) failed: {rc}")
    return out


def checksum(out) -> float:
    """Sum of every 257th output (kernels/common/adapter_common.cpp:18-23)."""
    import numpy as np
    out = np.ascontiguousarray(out, dtype=np.float32)
    return float(lib().pfng_host_checksum(out.ctypes.data, out.size))


# ---------------------------------------------------------------------------
# torch-level helpers (torch is plumbing: device memory and streams)
# ---------------------------------------------------------------------------

# A single-token product takes about 4 us on the GPU, so a call's time is this
# binding's own: pointers and streams go to ctypes as plain integers (the argtypes
# convert them), the current stream comes from torch without a Stream object, and
# a tensor that fits passes its check in one expression. compute() at m = 1,
# 4096 x 4096, out and workspace given: 9.5 -> 5.5 us a call, mul_mat 8.4 -> 5.1.
_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


_raw_stream = None


def _stream(stream=None) -> int:
    """The hipStream_t of `stream`, or of the current device's current stream."""
    if stream is not None:
        return stream.cuda_stream
    global _raw_stream
    if _raw_stream is None:
        torch = _torch()
        raw, device = (getattr(torch._C, name, None) for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"))
        if raw is None:
            return torch.cuda.current_stream().cuda_stream
        torch.cuda.init()
        _raw_stream = lambda: raw((device or torch.cuda.current_device)())
    return _raw_stream()


def _p(t) -> int:
    return t.data_ptr()


def _need(t, nbytes: int, name: str) -> None:
    """The C-ABI takes bare device pointers: check here that a tensor is a
    contiguous device tensor holding at least `nbytes` bytes."""
    if t.is_cuda and t.is_contiguous() and t.nbytes >= nbytes:
        return
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    raise ValueError(f"{name} holds {t.nbytes} bytes, {nbytes} needed")


def _blocks(qtype: int, rows: int, k: int, weight: bool) -> int:
    per = WEIGHT_BLOCK_BYTES[qtype] if weight else ACT_BLOCK_BYTES[qtype]
    return rows * (k // QK[qtype]) * per


def quantize_q8_0(x, out=None, stream=None):
    """x: (rows, k) float32 CUDA tensor -> (rows, k/32*34) uint8 block_q8_0 bytes."""
    torch = _torch()
    rows, k = x.shape
    if out is None:
        out = torch.empty((rows, (k // 32) * 34), dtype=torch.uint8, device=x.device)
    _need(x, rows * k * 4, "x")
    _need(out, _blocks(Q4_0, rows, k, False), "out")
    check(lib().pfng_hip_quantize_q8_0(_p(x), _p(out), rows, k, _stream(stream)))
    return out


def quantize_weights_gpu(qtype: int, x, out=None, stream=None):
    """Reference weight quantizer on the device: x (rows, k) float32 CUDA tensor
    -> (rows, k/QK * block_bytes) uint8 block bytes (q4_0 or q4_K)."""
    torch = _torch()
    rows, k = x.shape
    if out is None:
        out = torch.empty((rows, (k // QK[qtype]) * WEIGHT_BLOCK_BYTES[qtype]), dtype=torch.uint8, device=x.device)
    fn = {Q4_0: lib().pfng_hip_quantize_q4_0, Q4_K: lib().pfng_hip_quantize_q4_K}[qtype]
    _need(x, rows * k * 4, "x")
    _need(out, _blocks(qtype, rows, k, True), "out")
    check(fn(_p(x), _p(out), rows, k, _stream(stream)))
    return out


def quantize_q8_K(x, out=None, stream=None):
    """x: (rows, k) float32 CUDA tensor -> (rows, k/256*292) uint8 block_q8_K bytes."""
    torch = _torch()
    rows, k = x.shape
    if out is None:
        out = torch.empty((rows, (k // 256) * 292), dtype=torch.uint8, device=x.device)
    _need(x, rows * k * 4, "x")
    _need(out, _blocks(Q4_K, rows, k, False), "out")
    check(lib().pfng_hip_quantize_q8_K(_p(x), _p(out), rows, k, _stream(stream)))
    return out


def quantize_activation(qtype: int, x, out=None, stream=None):
    return quantize_q8_0(x, out, stream) if qtype == Q4_0 else quantize_q8_K(x, out, stream)


def mul_mat(qtype: int, weight, act_q, m: int, n: int, k: int, path: int = PATH_AUTO, out=None, stream=None):
    """C (m, n) float32 = W (n x k, quantized) . A (m x k, q8)^T on the GPU."""
    torch = _torch()
    if out is None:
        out = torch.empty((m, n), dtype=torch.float32, device=weight.device)
    if qtype in QK and m > 0 and n > 0 and k > 0 and k % QK[qtype] == 0:  # other shapes: the library reports the error
        _need(weight, _blocks(qtype, n, k, True), "weight")
        _need(act_q, _blocks(qtype, m, k, False), "act_q")
        _need(out, m * n * 4, "out")
    check(lib().pfng_hip_mul_mat(qtype, _p(weight), _p(act_q), _p(out), m, n, k, path, _stream(stream)))
    return out


def auto_path(qtype: int, m: int, n: int, k: int) -> int:
    """The path PATH_AUTO takes for this shape (aligned operands): PATH_GEMV or
    PATH_MFMA, PATH_AUTO for an empty product, or -1 when PATH_AUTO declines it
    (only PATH_NAIVE runs such a shape). Touches no device."""
    return lib().pfng_hip_auto_path(qtype, m, n, k)


def compute(qtype: int, activation, weight, n: int, path: int = PATH_AUTO, out=None, workspace=None, stream=None):
    """llama_reference::compute on the GPU: quantize fp32 activations, then the product."""
    m, k = activation.shape
    known = qtype in QK and m > 0 and k > 0
    need = _blocks(qtype, m, k, False) if known else lib().pfng_hip_compute_workspace_size(qtype, m, k)
    if workspace is None:
        torch = _torch()
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=activation.device)
    if out is None:
        torch = _torch()
        out = torch.empty((m, n), dtype=torch.float32, device=activation.device)
    if known and n > 0 and k % QK[qtype] == 0:
        _need(activation, m * k * 4, "activation")
        _need(weight, _blocks(qtype, n, k, True), "weight")
        _need(out, m * n * 4, "out")
        _need(workspace, need, "workspace")
    check(lib().pfng_hip_compute(qtype, activation.data_ptr(), weight.data_ptr(), out.data_ptr(), m, n, k,
                                 workspace.data_ptr(), workspace.numel(), path, _stream(stream)))
    return out


def compute_noalloc(qtype: int, activation, weight, n: int, path: int = PATH_AUTO, out=None, stream=None):
    """compute() without a workspace: the library's static per-device scratch
    holds the quantized activations (at most 16 MiB of them)."""
    torch = _torch()
    m, k = activation.shape
    if out is None:
        out = torch.empty((m, n), dtype=torch.float32, device=activation.device)
    if qtype in QK and m > 0 and n > 0 and k > 0 and k % QK[qtype] == 0:
        _need(activation, m * k * 4, "activation")
        _need(weight, _blocks(qtype, n, k, True), "weight")
        _need(out, m * n * 4, "out")
    check(lib().pfng_hip_compute_noalloc(qtype, _p(activation), _p(weight), _p(out), m, n, k, path, _stream(stream)))
    return out


def block_isums(qtype: int, weight, act_q, m: int, n: int, k: int, stream=None):
    """Exact integer parts of every block dot (diagnostic; see include/pfng_hip.h)."""
    torch = _torch()
    nb = k // QK[qtype]
    shape = (m, n, nb, 2) if qtype == Q4_K else (m, n, nb)
    out = torch.empty(shape, dtype=torch.int32, device=weight.device)
    if qtype in QK and m > 0 and n > 0 and k > 0 and k % QK[qtype] == 0:
        _need(weight, _blocks(qtype, n, k, True), "weight")
        _need(act_q, _blocks(qtype, m, k, False), "act_q")
    check(lib().pfng_hip_block_isums(qtype, _p(weight), _p(act_q), _p(out), m, n, k, _stream(stream)))
    return out


# ---------------------------------------------------------------------------
# serving: a paged 4-bit cache of keys and values
# ---------------------------------------------------------------------------

# As for the products, a small call's time is this binding's own: a tensor that fits passes its checks in one
# expression, and what does not fit is told apart only then. Nothing here takes part in autograd: results have no
# gradient, whatever the inputs.

# pfng_element_type
F32, BF16, F16 = 0, 1, 2
_element_types = {}  # by torch dtype
_float32 = _int32 = None


def _types() -> None:
    global _float32, _int32
    torch = _torch()
    _float32, _int32 = torch.float32, torch.int32
    _element_types.update({torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16})


def _element_type(dtype, name: str) -> int:
    if not _element_types:
        _types()
    kind = _element_types.get(dtype)
    if kind is None:
        raise ValueError(f"{name} has the type {dtype}: float32, bfloat16 and float16 are supported")
    return kind


def _new(shape, dtype, device, stream):
    """A tensor that a call on `stream` writes: allocated for that stream, so that the allocator hands its memory
    out again only behind the call."""
    torch = _torch()
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _new_like(t, dtype, stream):
    """_new() of t's shape."""
    torch = _torch()
    if stream is None:
        return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)
    with torch.cuda.stream(stream):
        return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _token_stride(t, name: str) -> int:
    """Elements from token to token of a device tensor (tokens, heads, head_dim) whose heads are contiguous."""
    if t.is_cuda:
        tokens, heads, dim = t.shape
        if t.is_contiguous():
            return heads * dim
        stride, head_stride, step = t.stride()
        if step == 1 and (head_stride == dim or heads <= 1):
            return stride if tokens > 1 else max(stride, heads * dim)
        raise ValueError(f"{name}: the heads of a token must be contiguous (strides {tuple(t.stride())})")
    raise ValueError(f"{name} must be a device tensor")


def _three(t, name: str):
    if t.dim() != 3:
        raise ValueError(f"{name} must have the shape (tokens, heads, head_dim), not {tuple(t.shape)}")
    return t.shape


def _ints(t, count: int, name: str) -> int:
    """Pointer of a contiguous int32 device tensor of at least `count` numbers."""
    if t.dtype is _int32 and t.is_cuda and t.is_contiguous() and t.numel() >= count:
        return t.data_ptr()
    if _int32 is None:
        _types()
        return _ints(t, count, name)
    if t.is_cuda and t.dtype is _int32 and t.is_contiguous():
        raise ValueError(f"{name} holds {t.numel()} numbers, {count} needed")
    raise ValueError(f"{name} must be a contiguous int32 device tensor")


def _floats(t, count: int, name: str) -> int:
    """Pointer of a contiguous float32 device tensor of at least `count` numbers."""
    if t.dtype is _float32 and t.is_cuda and t.is_contiguous() and t.numel() >= count:
        return t.data_ptr()
    if _float32 is None:
        _types()
        return _floats(t, count, name)
    raise ValueError(f"{name} must be a contiguous float32 device tensor of {count} numbers")


def _table(t, requests: int, name: str = "block_table"):
    """(pointer, row stride, columns) of an int32 (requests, max_pages) device tensor."""
    if _int32 is None:
        _types()
    if not (t.is_cuda and t.dim() == 2 and t.dtype is _int32 and t.shape[0] >= requests):
        raise ValueError(f"{name} must be an int32 device tensor with {requests} rows")
    columns = t.shape[1]
    if t.is_contiguous():
        return t.data_ptr(), columns, columns
    stride, step = t.stride()
    if columns > 1 and step != 1:
        raise ValueError(f"{name}: the entries of a row must be contiguous")
    if stride < columns and t.shape[0] > 1:
        raise ValueError(f"{name}: the rows must not overlap (strides {tuple(t.stride())})")
    return t.data_ptr(), max(stride, columns), columns


def _cache_shape(cache, head_dim: int):
    """(pages, kv_heads, page_size) of a cache as kv4_cache() makes it."""
    if not (cache.is_cuda and cache.dim() == 4 and cache.element_size() == 1 and cache.is_contiguous() and
            cache.shape[1] == 2):
        raise ValueError("cache must be a contiguous uint8 device tensor (pages, 2, kv_heads, page bytes)")
    pages, _, kv_heads, page_bytes = cache.shape
    per_token = head_dim // 2 + head_dim // 16
    if per_token == 0 or page_bytes % per_token:
        raise ValueError(f"cache: pages of {page_bytes} bytes do not hold heads of {head_dim}")
    return pages, kv_heads, page_bytes // per_token


def kv4_cache(pages: int, kv_heads: int, head_dim: int, page_size: int, device="cuda"):
    """An empty cache: uint8 (pages, 2, kv_heads, bytes of a head's page), the layout of include/pfng_hip.h."""
    page_bytes = lib().pfng_hip_kv4_page_bytes(page_size, head_dim)
    if not page_bytes or pages <= 0 or kv_heads <= 0:
        raise ValueError(f"no cache of {pages} pages of {page_size} tokens for {kv_heads} heads of {head_dim}: pages "
                         "hold a power of two of tokens from 16 to 1024, heads 64, 128 or 256 elements")
    return _torch().zeros((pages, 2, kv_heads, page_bytes), dtype=_torch().uint8, device=device)


def kv_block_tables(cached, added, free_pages, page_size: int, block_table, tokens: int, stream=None):
    """The tables of one step of len(cached) requests (int32 device tensors): each request's new pages, taken from
    free_pages in order, go into block_table (requests, max_pages) in place. Returns (starts, lengths, positions,
    slots, used): int32 of requests + 1, requests, tokens, tokens and 1 numbers. `tokens` is how many positions and
    slots are wanted (those past the last new token are 0 and -1); used[0] counts the pages taken, more than
    free_pages has where it is too short (then those tokens' slots are -1)."""
    requests = cached.numel()
    table, stride, columns = _table(block_table, requests)
    have = _ints(cached, requests, "cached")
    count = 2 * requests + 2 * tokens + 2
    whole = cached.new_empty(count) if stream is None else _new((count,), cached.dtype, cached.device, stream)
    p = whole.data_ptr()
    at = p + 4 * (requests + 1)
    status = lib().pfng_hip_kv_block_tables(
        have, _ints(added, requests, "added"), requests, _ints(free_pages, 0, "free_pages"), free_pages.numel(), page_size,
        table, stride, columns, tokens, p, at, at + 4 * requests, at + 4 * (requests + tokens),
        at + 4 * (requests + 2 * tokens), _stream(stream))
    if status:
        check(status)
    return whole.split_with_sizes((requests + 1, requests, tokens, tokens, 1))


def qk_norm_rope(q, k, positions, cos_sin, q_weight=None, k_weight=None, eps: float = 1e-6, adjacent: bool = False,
                 out_dtype=None, q_out=None, k_out=None, stream=None):
    """Root-mean-square norms of every head of q (tokens, q_heads, head_dim) and k (tokens, kv_heads, head_dim) with
    fp32 weights (None: no norm), and the rotation by row positions[t] of the fp32 table cos_sin (positions, rot_dim:
    cosines, then sines), in one pass; pairs (i, i + rot_dim / 2), or (2i, 2i + 1) if adjacent. Tokens may be strided,
    as parts of one projection are. Returns (q_out, k_out) of out_dtype (default: q's type)."""
    tokens, q_heads, dim = _three(q, "q")
    k_tokens, kv_heads, k_dim = _three(k, "k")
    in_type = _element_type(q.dtype, "q")
    if k_tokens != tokens or k_dim != dim or k.dtype is not q.dtype:
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} do not belong together")
    q_stride, k_stride = _token_stride(q, "q"), _token_stride(k, "k")
    if q_out is None and k_out is None:
        dtype = out_dtype or q.dtype
        out_type = _element_type(dtype, "out_dtype")
        q_out, k_out = _new_like(q, dtype, stream), _new_like(k, dtype, stream)
        q_out_stride, k_out_stride = q_heads * dim, kv_heads * dim
    else:
        if q_out is None:
            q_out = _new_like(q, out_dtype or k_out.dtype, stream)
        if k_out is None:
            k_out = _new_like(k, q_out.dtype, stream)
        out_type = _element_type(q_out.dtype, "q_out")
        if q_out.shape != q.shape or k_out.shape != k.shape or q_out.dtype != k_out.dtype:
            raise ValueError("q_out and k_out must have the shapes of q and k and one type")
        q_out_stride, k_out_stride = _token_stride(q_out, "q_out"), _token_stride(k_out, "k_out")
    q_w = 0 if q_weight is None else _floats(q_weight, dim, "q_weight")
    k_w = 0 if k_weight is None else _floats(k_weight, dim, "k_weight")
    rows, rot = (0, 0) if cos_sin is None else cos_sin.shape
    status = lib().pfng_hip_qk_norm_rope(
        q.data_ptr(), q_stride, k.data_ptr(), k_stride, in_type, q_out.data_ptr(), q_out_stride, k_out.data_ptr(),
        k_out_stride, out_type, q_w, k_w, eps, _floats(cos_sin, rows * rot, "cos_sin") if rot else 0, rows, rot, adjacent,
        _ints(positions, tokens, "positions") if rot else 0, tokens, q_heads, kv_heads, dim, _stream(stream))
    if status:
        check(status)
    return q_out, k_out


def kv4_store(k, v, slots, cache, stream=None):
    """Stores k and v (tokens, kv_heads, head_dim) at int32 slots (tokens) of the cache, as q4_0 blocks."""
    tokens, heads, dim = _three(k, "k")
    pages, kv_heads, page_size = _cache_shape(cache, dim)
    if v.shape != k.shape or v.dtype is not k.dtype or heads != kv_heads:
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} do not fit a cache of {kv_heads} heads")
    status = lib().pfng_hip_kv4_store(k.data_ptr(), _token_stride(k, "k"), v.data_ptr(), _token_stride(v, "v"),
                                      _element_type(k.dtype, "k"), _ints(slots, tokens, "slots"), tokens, cache.data_ptr(),
                                      pages, kv_heads, dim, page_size, _stream(stream))
    if status:
        check(status)


def kv4_read(cache, slots, head_dim: int, dtype=None, stream=None):
    """(k, v), each (len(slots), kv_heads, head_dim) of dtype (default float32): what the cache holds at the slots."""
    dtype = dtype or _torch().float32
    element = _element_type(dtype, "dtype")
    pages, kv_heads, page_size = _cache_shape(cache, head_dim)
    tokens = slots.numel()
    both = _new((2, tokens, kv_heads, head_dim), dtype, cache.device, stream)
    k = both.data_ptr()
    check(lib().pfng_hip_kv4_read(cache.data_ptr(), pages, kv_heads, head_dim, page_size, _ints(slots, tokens, "slots"),
                                  tokens, k, k + both.nbytes // 2, element, _stream(stream)))
    return both.unbind(0)


def attention_kv4_workspace(dtype, tokens: int, requests: int, q_heads: int, kv_heads: int, head_dim: int,
                            max_added: int, max_length: int, causal: bool = True) -> int:
    """Bytes of workspace attention_kv4 needs for queries of dtype and these sizes on the current device. They do not
    grow with the sizes (it goes by how the keys are split): ask for the sizes of each call."""
    size = lib().pfng_hip_attention_kv4_workspace_size(_element_type(dtype, "dtype"), tokens, requests, q_heads, kv_heads,
                                                       head_dim, causal, max_added, max_length)
    if size < 0:
        raise PfngError(ERR_INVALID_ARGUMENT, last_error())
    return size


def attention_kv4(q, cache, block_table, lengths, starts=None, max_added: int = 1, max_length=None, scale=None,
                  causal: bool = True, window: int = 0, out=None, workspace=None, stream=None):
    """Attention of q (tokens, q_heads, head_dim) over the cache -> out of q's shape and type.

    Request r has lengths[r] keys in the pages block_table[r]; its tokens starts[r] .. starts[r + 1] - 1 are the last
    of them (starts None: one token each). A query sees the keys up to its own position (causal False: all of the
    request's) and, with a window, only the last `window` of them; one that sees none gets zeros. max_added and
    max_length, the most tokens and keys of one request, choose the launch; the default max_length is what the table
    holds. With a window far shorter than the requests a max_length of window + max_added chooses a faster one.
    scale: head_dim ** -0.5 by default."""
    tokens, q_heads, dim = _three(q, "q")
    kind = _element_type(q.dtype, "q")
    pages, kv_heads, page_size = _cache_shape(cache, dim)
    requests = lengths.numel()
    table, table_stride, max_pages = _table(block_table, requests)
    if out is None:
        out = _new_like(q, q.dtype, stream)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have the shape and type of q")
    if max_length is None:
        max_length = max_pages * page_size
    L = lib()
    size = 0
    if workspace is None:
        size = L.pfng_hip_attention_kv4_workspace_size(kind, tokens, requests, q_heads, kv_heads, dim, causal, max_added,
                                                       max_length)
        if size < 0:
            raise PfngError(ERR_INVALID_ARGUMENT, last_error())
        if size:
            workspace = _new((size,), _torch().uint8, q.device, stream)
    else:
        size = workspace.nbytes
        _need(workspace, size, "workspace")
    check(L.pfng_hip_attention_kv4(
        q.data_ptr(), _token_stride(q, "q"), out.data_ptr(), _token_stride(out, "out"), kind,
        0 if starts is None else _ints(starts, requests + 1, "starts"), _ints(lengths, requests, "lengths"), requests,
        tokens, q_heads, table, table_stride, max_pages, cache.data_ptr(), pages, kv_heads, dim, page_size,
        dim ** -0.5 if scale is None else scale, causal, window, max_added, max_length,
        workspace.data_ptr() if size else 0, size, _stream(stream)))
    return out
