"""Python bindings of libb200_sampler.so (the C-ABI in include/b200_sampler.h).

The package directory is named ``llama2.cu_b200``; load it with
``load_package()`` from ``__graft_entry__`` / tests (the dot in the name keeps
it out of the normal import path).  Everything here is a thin ctypes layer:
the sampling itself runs in the library's sm_100a kernels, and every call
fails loudly (``SamplerError``) when the library or a GPU is missing.
"""
import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libb200_sampler.so")

SAMPLER_FLAG_PROBS_IN = 1
SAMPLER_FLAG_GREEDY_BELOW_1E6 = 2
SAMPLER_FLAG_NAN_TOKEN1 = 4
MODE_DO_SAMPLE = SAMPLER_FLAG_GREEDY_BELOW_1E6
MODE_SAMPLE_DEBUG = SAMPLER_FLAG_GREEDY_BELOW_1E6 | SAMPLER_FLAG_NAN_TOKEN1
ROW_NAN, ROW_NO_CANDIDATE, ROW_SLOW_PATH, ROW_SERIAL, ROW_TIMEOUT = 1, 2, 4, 8, 16
MAX_VOCAB = 32768
DTYPE_F32, DTYPE_BF16, DTYPE_F16 = 0, 1, 2
FILTERED_MAX_VOCAB = 1048576

# Every symbol the header declares (the CPU tests check the library exports them).
EXPORTED_SYMBOLS = [
    "build_sampler", "free_sampler", "random_u32", "random_f32", "sample_argmax", "sample_mult",
    "sample_topp", "sample", "sample_debug", "do_sample", "sampler_workspace_bytes", "sampler_batched", "sampler_batched_host",
    "sampler_seed_states", "sampler_last_launch_count", "sampler_last_error", "sampler_shard_rows",
    "sampler_nccl_get_unique_id", "sampler_nccl_comm_init", "sampler_nccl_allgather_ids",
    "sampler_nccl_comm_destroy", "sampler_batched_noalloc", "classifier_sample_fused",
    "classifier_logits", "rmsnorm_bf16", "classifier_rmsnorm_sample_fused", "sampler_gather_rows",
    "sampler_selftest_wait_timeout", "sampler_filtered", "quantize_fp8", "rmsnorm_fp8", "classifier_logits_fp8",
    "classifier_fp8_workspace_bytes", "classifier_fp8_sample_filtered", "classifier_fp8_selftest_wait_timeout",
]


class SamplerError(RuntimeError):
    pass


class ProbIndex(ctypes.Structure):
    _fields_ = [("prob", ctypes.c_float), ("index", ctypes.c_int)]


class Sampler(ctypes.Structure):
    """Same layout as llama2.c's Sampler (llama2.c:973-979)."""
    _fields_ = [("vocab_size", ctypes.c_int), ("probindex", ctypes.POINTER(ProbIndex)),
                ("temperature", ctypes.c_float), ("topp", ctypes.c_float),
                ("rng_state", ctypes.c_ulonglong)]


class SamplerBatchConfig(ctypes.Structure):
    _fields_ = [("vocab_size", ctypes.c_int), ("temperature", ctypes.c_float),
                ("topp", ctypes.c_float), ("flags", ctypes.c_int)]


class SamplerFilterConfig(ctypes.Structure):
    _fields_ = [("vocab_size", ctypes.c_int), ("logits_dtype", ctypes.c_int), ("temperature", ctypes.c_float),
                ("topk", ctypes.c_int), ("topp", ctypes.c_float), ("minp", ctypes.c_float)]


_lib = None


def library_path():
    return LIB_PATH


def lib():
    """Loads the library (RTLD_LOCAL) and declares the prototypes."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise SamplerError(f"{LIB_PATH} is missing: build it with llama2.cu_b200/build.py")
    L = ctypes.CDLL(LIB_PATH)
    P, c_int, c_float, c_ull, c_size = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_ulonglong, ctypes.c_size_t
    fp = ctypes.POINTER(c_float)
    L.build_sampler.argtypes = [ctypes.POINTER(Sampler), c_int, c_float, c_float, c_ull]
    L.build_sampler.restype = None
    L.free_sampler.argtypes = [ctypes.POINTER(Sampler)]
    L.free_sampler.restype = None
    L.random_u32.argtypes = [ctypes.POINTER(c_ull)]
    L.random_u32.restype = ctypes.c_uint
    L.random_f32.argtypes = [ctypes.POINTER(c_ull)]
    L.random_f32.restype = c_float
    L.sample_argmax.argtypes = [fp, c_int]
    L.sample_argmax.restype = c_int
    L.sample_mult.argtypes = [fp, c_int, c_float]
    L.sample_mult.restype = c_int
    L.sample_topp.argtypes = [fp, c_int, c_float, ctypes.POINTER(ProbIndex), c_float]
    L.sample_topp.restype = c_int
    L.sample.argtypes = [ctypes.POINTER(Sampler), fp]
    L.sample.restype = c_int
    L.sample_debug.argtypes = [ctypes.POINTER(Sampler), fp]
    L.sample_debug.restype = c_int
    L.do_sample.argtypes = [ctypes.POINTER(Sampler), fp]
    L.do_sample.restype = c_int
    L.sampler_workspace_bytes.argtypes = [c_int, c_int]
    L.sampler_workspace_bytes.restype = c_size
    L.sampler_batched.argtypes = [ctypes.POINTER(SamplerBatchConfig), P, c_int, ctypes.c_longlong, P, P, P,
                                  P, P, P, P, P, c_size, P]
    L.sampler_batched.restype = c_int
    L.sampler_batched_host.argtypes = [ctypes.POINTER(SamplerBatchConfig), P, c_int, ctypes.c_longlong, P, P, P]
    L.sampler_batched_host.restype = c_int
    L.sampler_seed_states.argtypes = [P, c_int, c_ull, ctypes.c_longlong, P]
    L.sampler_seed_states.restype = c_int
    L.sampler_last_launch_count.argtypes = []
    L.sampler_last_launch_count.restype = c_int
    L.sampler_last_error.argtypes = []
    L.sampler_last_error.restype = ctypes.c_char_p
    L.sampler_shard_rows.argtypes = [c_int, c_int, c_int, ctypes.POINTER(c_int), ctypes.POINTER(c_int)]
    L.sampler_shard_rows.restype = c_int
    L.sampler_nccl_get_unique_id.argtypes = [P]
    L.sampler_nccl_get_unique_id.restype = c_int
    L.sampler_nccl_comm_init.argtypes = [ctypes.POINTER(P), c_int, P, c_int]
    L.sampler_nccl_comm_init.restype = c_int
    L.sampler_nccl_allgather_ids.argtypes = [P, P, c_int, P, P]
    L.sampler_nccl_allgather_ids.restype = c_int
    L.sampler_nccl_comm_destroy.argtypes = [P]
    L.sampler_nccl_comm_destroy.restype = c_int
    L.classifier_sample_fused.argtypes = [ctypes.POINTER(SamplerBatchConfig), P, P, c_int, c_int, P, P, P, P, P, P,
                                          P, P]
    L.classifier_sample_fused.restype = c_int
    L.classifier_logits.argtypes = [P, P, c_int, c_int, c_int, P, P]
    L.classifier_logits.restype = c_int
    L.rmsnorm_bf16.argtypes = [P, P, c_int, c_int, P, P]
    L.rmsnorm_bf16.restype = c_int
    L.classifier_rmsnorm_sample_fused.argtypes = [ctypes.POINTER(SamplerBatchConfig), P, P, P, c_int, c_int, P, P,
                                                  P, P, P, P, P, P]
    L.classifier_rmsnorm_sample_fused.restype = c_int
    L.sampler_gather_rows.argtypes = [P, c_int, c_int, P, c_int, P, P]
    L.sampler_gather_rows.restype = c_int
    L.sampler_selftest_wait_timeout.argtypes = [ctypes.c_uint, ctypes.POINTER(c_int)]
    L.sampler_selftest_wait_timeout.restype = c_int
    L.classifier_fp8_selftest_wait_timeout.argtypes = [ctypes.c_uint, ctypes.POINTER(c_int)]
    L.classifier_fp8_selftest_wait_timeout.restype = c_int
    c_ll = ctypes.c_longlong
    L.sampler_filtered.argtypes = [ctypes.POINTER(SamplerFilterConfig), P, c_int, c_ll, P, P, P, P, P, P, P, P, P, P, P]
    L.sampler_filtered.restype = c_int
    L.quantize_fp8.argtypes = [P, c_int, c_int, c_int, c_ll, c_int, P, P, P]
    L.quantize_fp8.restype = c_int
    L.rmsnorm_fp8.argtypes = [P, c_int, P, c_int, c_int, c_ll, P, P, P]
    L.rmsnorm_fp8.restype = c_int
    L.classifier_logits_fp8.argtypes = [P, P, P, P, c_int, c_int, c_int, P, c_int, c_ll, P]
    L.classifier_logits_fp8.restype = c_int
    L.classifier_fp8_workspace_bytes.argtypes = [c_int, c_int, c_int, c_int]
    L.classifier_fp8_workspace_bytes.restype = c_size
    L.classifier_fp8_sample_filtered.argtypes = [ctypes.POINTER(SamplerFilterConfig), P, c_int, P, P, P, c_int, c_int,
                                                 P, P, P, P, P, P, P, P, P, P, P, P, c_size, P]
    L.classifier_fp8_sample_filtered.restype = c_int
    _lib = L
    return L


def _check(rc, what):
    if rc != 0:
        raise SamplerError(f"{what} failed ({rc}): {lib().sampler_last_error().decode()}")


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise SamplerError("device entry point given a CPU tensor")


def shard_rows(batch, world, rank):
    b, c = ctypes.c_int(), ctypes.c_int()
    _check(lib().sampler_shard_rows(batch, world, rank, ctypes.byref(b), ctypes.byref(c)), "sampler_shard_rows")
    return b.value, c.value


def seed_states(states, seed, row_offset=0, stream=None):
    """states: int64 CUDA tensor [B] (bit pattern of the uint64 states)."""
    _require_cuda(states)
    _check(lib().sampler_seed_states(_ptr(states), states.numel(), ctypes.c_ulonglong(seed), row_offset,
                                     _stream_ptr(stream)), "sampler_seed_states")


def _stream_ptr(stream):
    if stream is None:
        import torch
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def sample_batched(logits, temperature, topp, rng_state=None, *, temperature_rows=None, topp_rows=None,
                   coins=None, out_ids=None, probs_out=None, row_flags=None, probs_in=False,
                   workspace=None, stream=None, mode=0):
    """Batched device sampling over the rows of a CUDA fp32 tensor [B, ld].

    rng_state: int64 CUDA tensor [B] advanced in place (uint64 bit patterns).
    mode: 0 (sample()'s rules), MODE_SAMPLE_DEBUG or MODE_DO_SAMPLE.
    Returns out_ids (int32 CUDA tensor [B]).  Asynchronous on `stream`.
    """
    import torch
    _require_cuda(logits, rng_state, temperature_rows, topp_rows, coins, probs_out, row_flags, workspace)
    if logits.dtype != torch.float32 or logits.dim() != 2 or logits.stride(1) != 1:
        raise SamplerError("logits must be a row-major float32 [B, ld] tensor")
    B, V = logits.shape
    if out_ids is None:
        out_ids = torch.empty(B, dtype=torch.int32, device=logits.device)
    cfg = SamplerBatchConfig(V, float(temperature), float(topp), (SAMPLER_FLAG_PROBS_IN if probs_in else 0) | mode)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    rc = lib().sampler_batched(ctypes.byref(cfg), _ptr(logits), B, logits.stride(0), _ptr(temperature_rows),
                               _ptr(topp_rows), _ptr(coins), _ptr(rng_state), _ptr(out_ids), _ptr(probs_out),
                               _ptr(row_flags), _ptr(workspace), ws_bytes, _stream_ptr(stream))
    _check(rc, "sampler_batched")
    return out_ids


def classifier_sample_fused(hidden, wcls, temperature, topp, rng_state=None, *, temperature_rows=None,
                            topp_rows=None, coins=None, out_ids=None, logits_out=None, row_flags=None, stream=None):
    """Fused classifier + sampling: hidden bf16 CUDA [B, D], wcls bf16 CUDA
    [V, D]; logits = hidden . wcls^T (fp32, optionally returned in
    logits_out [B, V]) sampled per row as sample_batched() does.
    Returns out_ids (int32 CUDA tensor [B]).  Asynchronous on `stream`."""
    import torch
    _require_cuda(hidden, wcls, rng_state, temperature_rows, topp_rows, coins, logits_out, row_flags)
    for t in (hidden, wcls):
        if t.dtype != torch.bfloat16 or t.dim() != 2 or not t.is_contiguous():
            raise SamplerError("hidden and wcls must be contiguous bfloat16 matrices")
    B, D = hidden.shape
    V = wcls.shape[0]
    if wcls.shape[1] != D:
        raise SamplerError("hidden and wcls disagree on the model dimension")
    if logits_out is not None and (logits_out.dtype != torch.float32 or tuple(logits_out.shape) != (B, V)
                                   or not logits_out.is_contiguous()):
        raise SamplerError("logits_out must be a contiguous float32 [B, V] tensor")
    if out_ids is None:
        out_ids = torch.empty(B, dtype=torch.int32, device=hidden.device)
    cfg = SamplerBatchConfig(V, float(temperature), float(topp), 0)
    rc = lib().classifier_sample_fused(ctypes.byref(cfg), _ptr(hidden), _ptr(wcls), B, D, _ptr(temperature_rows),
                                       _ptr(topp_rows), _ptr(coins), _ptr(rng_state), _ptr(out_ids),
                                       _ptr(logits_out), _ptr(row_flags), _stream_ptr(stream))
    _check(rc, "classifier_sample_fused")
    return out_ids


def classifier_logits(hidden, wcls, logits_out=None, stream=None):
    """logits = hidden . wcls^T (bf16 in, fp32 out): tensor cores from three rows,
    a CUDA-core GEMV streaming wcls for one or two."""
    import torch
    _require_cuda(hidden, wcls, logits_out)
    B, D = hidden.shape
    V = wcls.shape[0]
    if logits_out is None:
        logits_out = torch.empty(B, V, dtype=torch.float32, device=hidden.device)
    rc = lib().classifier_logits(_ptr(hidden), _ptr(wcls), B, D, V, _ptr(logits_out), _stream_ptr(stream))
    _check(rc, "classifier_logits")
    return logits_out


def rmsnorm_bf16(x, norm_weight, out=None, stream=None):
    """bf16(norm_weight * x / rms(x)) per row of a float32 CUDA tensor [B, D]."""
    import torch
    _require_cuda(x, norm_weight, out)
    B, D = x.shape
    if out is None:
        out = torch.empty(B, D, dtype=torch.bfloat16, device=x.device)
    _check(lib().rmsnorm_bf16(_ptr(x), _ptr(norm_weight), B, D, _ptr(out), _stream_ptr(stream)), "rmsnorm_bf16")
    return out


def classifier_rmsnorm_sample_fused(x, norm_weight, wcls, temperature, topp, rng_state=None, *,
                                    temperature_rows=None, topp_rows=None, coins=None, out_ids=None,
                                    logits_out=None, row_flags=None, stream=None):
    """Decode step from fp32 hidden states [B, D]: final RMSNorm, classifier
    GEMM, sampling.  Returns out_ids (int32 CUDA tensor [B])."""
    import torch
    _require_cuda(x, norm_weight, wcls, rng_state, temperature_rows, topp_rows, coins, logits_out, row_flags)
    if x.dtype != torch.float32 or not x.is_contiguous() or wcls.dtype != torch.bfloat16:
        raise SamplerError("x must be contiguous float32 [B, D] and wcls bfloat16 [V, D]")
    B, D = x.shape
    V = wcls.shape[0]
    if out_ids is None:
        out_ids = torch.empty(B, dtype=torch.int32, device=x.device)
    cfg = SamplerBatchConfig(V, float(temperature), float(topp), 0)
    rc = lib().classifier_rmsnorm_sample_fused(ctypes.byref(cfg), _ptr(x), _ptr(norm_weight), _ptr(wcls), B, D,
                                               _ptr(temperature_rows), _ptr(topp_rows), _ptr(coins),
                                               _ptr(rng_state), _ptr(out_ids), _ptr(logits_out), _ptr(row_flags),
                                               _stream_ptr(stream))
    _check(rc, "classifier_rmsnorm_sample_fused")
    return out_ids


def gather_rows(table, ids, out=None, stream=None):
    """out[b] = table[ids[b]] on the device (float32 table [R, D], int32 ids [B])."""
    import torch
    _require_cuda(table, ids, out)
    R, D = table.shape
    B = ids.numel()
    if out is None:
        out = torch.empty(B, D, dtype=torch.float32, device=table.device)
    _check(lib().sampler_gather_rows(_ptr(table), R, D, _ptr(ids), B, _ptr(out), _stream_ptr(stream)),
           "sampler_gather_rows")
    return out


def sample_batched_host(logits_np, temperature, topp, states_np, topp_rows_np=None, probs_in=False):
    """Host-buffer entry point: numpy float32 [B, V] in, int32 ids out; the
    uint64 states array is advanced in place."""
    import numpy as np
    B, V = logits_np.shape
    assert logits_np.dtype == np.float32 and logits_np.flags.c_contiguous
    ids = np.empty(B, dtype=np.int32)
    cfg = SamplerBatchConfig(V, float(temperature), float(topp), SAMPLER_FLAG_PROBS_IN if probs_in else 0)
    tp = None if topp_rows_np is None else topp_rows_np.ctypes.data_as(ctypes.c_void_p)
    st = None if states_np is None else states_np.ctypes.data_as(ctypes.c_void_p)
    rc = lib().sampler_batched_host(ctypes.byref(cfg), logits_np.ctypes.data_as(ctypes.c_void_p), B, V, tp, st,
                                    ids.ctypes.data_as(ctypes.c_void_p))
    _check(rc, "sampler_batched_host")
    return ids


# ---- filtered sampling and the 8-bit classifier ----
# These calls take microseconds on the device, so what they do on the host counts:
# torch is looked up once, addresses go to ctypes as integers, and the current
# device and stream are read without building objects for them.
class _Torch:
    """torch and what the calls below need of it, filled on first use."""
    codes = {}

    @classmethod
    def load(cls):
        import torch
        cls.torch, cls.empty, cls.f32, cls.i32, cls.i64 = torch, torch.empty, torch.float32, torch.int32, torch.int64
        cls.f8, cls.u8 = torch.float8_e4m3fn, torch.uint8
        cls.codes = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16}
        cls.device = staticmethod(torch._C._cuda_getDevice)
        cls.stream = staticmethod(torch._C._cuda_getCurrentRawStream)
        return cls


def _matrix(t, what):
    """dtype code, rows, columns, row stride and device of a row-major CUDA matrix (any stride that keeps rows apart)."""
    code = (_Torch.codes or _Torch.load().codes).get(t.dtype)
    if code is None:
        raise SamplerError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    if not t.is_cuda or t.dim() != 2:
        raise SamplerError(f"{what} must be a CUDA matrix")
    rows, cols = t.shape
    ld, step = t.stride()
    if cols > 1 and step != 1:
        raise SamplerError(f"{what} must be row-major")
    if rows <= 1:
        ld = cols
    elif ld < cols:
        raise SamplerError(f"{what} has overlapping rows")
    return code, rows, cols, ld, t.device


def _vector(t, what, n, dtype, device):
    """Address of a contiguous vector of n elements on `device`; None passes."""
    if t is None:
        return None
    if t.dtype != dtype or t.numel() != n or t.device != device or not t.is_contiguous():
        raise SamplerError(f"{what} must be a contiguous {dtype} tensor of {n} elements on {device}")
    return t.data_ptr()


def _block_matrix(t, what, rows, cols, dtype, device):
    """Address of a contiguous matrix of the given shape."""
    if t.dtype != dtype or t.shape != (rows, cols) or t.device != device or not t.is_contiguous():
        raise SamplerError(f"{what} must be a contiguous {dtype} tensor [{rows}, {cols}] on {device}")
    return t.data_ptr()


def _alloc(shape, dtype, device, stream):
    """torch.empty in the order of the stream that will use it (a block of another
    stream's could still be in use there)."""
    if stream is None:
        return _Torch.empty(shape, dtype=dtype, device=device)
    with _Torch.torch.cuda.stream(stream):
        return _Torch.empty(shape, dtype=dtype, device=device)


def _on_device(device, rows, stream, name, *args):
    """Calls entry point `name` with the operands' device current, on `stream`
    (default: that device's current one); nothing for an empty batch, whose
    tensors have no address."""
    if rows == 0:
        return
    if _Torch.device() != device.index:
        with _Torch.torch.cuda.device(device):
            return _on_device(device, rows, stream, name, *args)
    if stream is None:
        handle = _Torch.stream(device.index)
    elif stream.device != device:
        raise SamplerError(f"the stream is on {stream.device}, the operands on {device}")
    else:
        handle = stream.cuda_stream
    rc = getattr(_lib or lib(), name)(*args, handle)
    if rc != 0:
        _check(rc, name)


def sample_filtered(logits, temperature, topk, topp, minp, rng_state=None, *, temperature_rows=None, topk_rows=None,
                    topp_rows=None, minp_rows=None, coins=None, out_ids=None, logprobs_out=None, kept_out=None,
                    row_flags=None, stream=None):
    """Token ids of the rows of a CUDA float32, bfloat16 or float16 matrix
    [B, V] (any row stride, V up to FILTERED_MAX_VOCAB) by temperature, top-k,
    top-p and min-p, each for every row or per row (*_rows; top-k int32), from
    given coins or one draw of rng_state per row.  topk <= 0, topp outside
    (0, 1) and minp <= 0 are off; a row with T < 1e-6 takes its first largest
    logit.  logprobs_out float32, kept_out and row_flags int32 (each [B])
    receive ln(p) of the id among the kept entries, their count, and the row's
    ROW_* bits.  Returns out_ids (int32 CUDA tensor [B]).  Asynchronous on
    `stream`."""
    code, B, V, ld, dev = _matrix(logits, "logits")
    f32, i32 = _Torch.f32, _Torch.i32
    if out_ids is None:
        out_ids = _alloc(B, i32, dev, stream)
    cfg = SamplerFilterConfig(V, code, temperature, min(max(topk, 0), V), topp, minp)
    _on_device(dev, B, stream, "sampler_filtered", cfg, logits.data_ptr(), B, ld,
               _vector(temperature_rows, "temperature_rows", B, f32, dev),
               _vector(topk_rows, "topk_rows", B, i32, dev), _vector(topp_rows, "topp_rows", B, f32, dev),
               _vector(minp_rows, "minp_rows", B, f32, dev), _vector(coins, "coins", B, f32, dev),
               _vector(rng_state, "rng_state", B, _Torch.i64, dev), _vector(out_ids, "out_ids", B, i32, dev),
               _vector(logprobs_out, "logprobs_out", B, f32, dev), _vector(kept_out, "kept_out", B, i32, dev),
               _vector(row_flags, "row_flags", B, i32, dev))
    return out_ids


def _fp8_outputs(R, D, block_rows, dev, out, scales_out, stream):
    rows, cols = -(-R // block_rows), (D + 127) // 128
    if out is None:
        out = _alloc((R, D), _Torch.f8, dev, stream)
        qp = out.data_ptr()
    else:
        qp = _block_matrix(out, "out", R, D, _Torch.f8, dev)
    if scales_out is None:
        scales_out = _alloc((rows, cols), _Torch.f32, dev, stream)
        sp = scales_out.data_ptr()
    else:
        sp = _block_matrix(scales_out, "scales_out", rows, cols, _Torch.f32, dev)
    return out, scales_out, qp, sp


def quantize_fp8(x, block_rows=1, *, out=None, scales_out=None, stream=None):
    """x (float32, bfloat16 or float16 CUDA matrix [R, D], any row stride) as
    float8_e4m3fn [R, D] with one float32 scale per block of block_rows (1 for
    activations, 128 for weights) by 128 columns.  Returns (values, scales)."""
    code, R, D, ld, dev = _matrix(x, "x")
    if block_rows != 1 and block_rows != 128:
        raise SamplerError("block_rows must be 1 or 128")
    out, scales_out, qp, sp = _fp8_outputs(R, D, block_rows, dev, out, scales_out, stream)
    _on_device(dev, R, stream, "quantize_fp8", x.data_ptr(), code, R, D, ld, block_rows, qp, sp)
    return out, scales_out


def rmsnorm_fp8(x, norm_weight, *, out=None, scales_out=None, stream=None):
    """quantize_fp8(norm_weight * x / rms(x)) with block_rows 1 in one pass: x
    float32, bfloat16 or float16 [B, D], norm_weight float32 [D]."""
    code, B, D, ld, dev = _matrix(x, "x")
    out, scales_out, qp, sp = _fp8_outputs(B, D, 1, dev, out, scales_out, stream)
    _on_device(dev, B, stream, "rmsnorm_fp8", x.data_ptr(), code,
               _vector(norm_weight, "norm_weight", D, _Torch.f32, dev), B, D, ld, qp, sp)
    return out, scales_out


def _fp8_weights(wcls, wcls_scales, D, dev):
    if wcls.dim() != 2 or wcls.shape[1] != D:
        raise SamplerError(f"wcls must be [V, {D}]")
    V = wcls.shape[0]
    return (V, _block_matrix(wcls, "wcls", V, D, _Torch.f8, dev),
            _block_matrix(wcls_scales, "wcls_scales", (V + 127) // 128, (D + 127) // 128, _Torch.f32, dev))


def classifier_logits_fp8(hidden, hidden_scales, wcls, wcls_scales, logits_out=None, stream=None):
    """logits = (hidden * hidden_scales) . (wcls * wcls_scales)^T with fp32
    accumulation, from quantize_fp8's operands (hidden at block_rows 1 or
    rmsnorm_fp8's, wcls at 128).  logits_out: float32 (default) or bfloat16
    [B, V], any row stride."""
    if hidden.dim() != 2 or not hidden.is_cuda:
        raise SamplerError("hidden must be a CUDA matrix")
    B, D = hidden.shape
    dev = hidden.device
    if not _Torch.codes:
        _Torch.load()
    hp = _block_matrix(hidden, "hidden", B, D, _Torch.f8, dev)
    hsp = _block_matrix(hidden_scales, "hidden_scales", B, (D + 127) // 128, _Torch.f32, dev)
    V, wp, wsp = _fp8_weights(wcls, wcls_scales, D, dev)
    if logits_out is None:
        logits_out = _alloc((B, V), _Torch.f32, dev, stream)
    code, rows, cols, ld, out_dev = _matrix(logits_out, "logits_out")
    if rows != B or cols != V or out_dev != dev:
        raise SamplerError(f"logits_out must be [{B}, {V}] on {dev}")
    _on_device(dev, B, stream, "classifier_logits_fp8", hp, hsp, wp, wsp, B, D, V, logits_out.data_ptr(), code, ld)
    return logits_out


def classifier_fp8_sample_filtered(x, norm_weight, wcls, wcls_scales, temperature, topk, topp, minp, rng_state=None,
                                   *, temperature_rows=None, topk_rows=None, topp_rows=None, minp_rows=None,
                                   coins=None, out_ids=None, logprobs_out=None, kept_out=None, logits_out=None,
                                   row_flags=None, stream=None):
    """Decode step on 8-bit weights from hidden states x [B, D] (contiguous
    float32, bfloat16 or float16): rmsnorm_fp8 (quantize_fp8 when norm_weight
    is None), classifier_logits_fp8, sample_filtered.  logits_out: contiguous
    float32 or bfloat16 [B, V] that receives the logits (float32 otherwise).
    Returns out_ids."""
    x_code, B, D, ld, dev = _matrix(x, "x")
    if ld != D:
        raise SamplerError("x must be contiguous")
    V, wp, wsp = _fp8_weights(wcls, wcls_scales, D, dev)
    f32, i32 = _Torch.f32, _Torch.i32
    code, lp = DTYPE_F32, None
    if logits_out is not None:
        code = _Torch.codes.get(logits_out.dtype)
        if code is None:
            raise SamplerError("logits_out must be float32 or bfloat16")
        lp = _block_matrix(logits_out, "logits_out", B, V, logits_out.dtype, dev)
    n = lib().classifier_fp8_workspace_bytes(B, D, V, code if lp is None else -1)
    ws = _alloc(n, _Torch.u8, dev, stream)  # from torch's allocator: inside a capture, the graph's own
    if out_ids is None:
        out_ids = _alloc(B, i32, dev, stream)
    cfg = SamplerFilterConfig(V, code, temperature, min(max(topk, 0), V), topp, minp)
    _on_device(dev, B, stream, "classifier_fp8_sample_filtered", cfg, x.data_ptr(), x_code,
               _vector(norm_weight, "norm_weight", D, f32, dev), wp, wsp, B, D,
               _vector(temperature_rows, "temperature_rows", B, f32, dev),
               _vector(topk_rows, "topk_rows", B, i32, dev), _vector(topp_rows, "topp_rows", B, f32, dev),
               _vector(minp_rows, "minp_rows", B, f32, dev), _vector(coins, "coins", B, f32, dev),
               _vector(rng_state, "rng_state", B, _Torch.i64, dev), _vector(out_ids, "out_ids", B, i32, dev),
               _vector(logprobs_out, "logprobs_out", B, f32, dev), _vector(kept_out, "kept_out", B, i32, dev), lp,
               _vector(row_flags, "row_flags", B, i32, dev), ws.data_ptr(), n)
    return out_ids


def last_launch_count():
    return lib().sampler_last_launch_count()


# ---- llama2.c surface, for tests that read like the reference's call sites ----
def build_sampler(vocab_size, temperature, topp, rng_seed):
    s = Sampler()
    lib().build_sampler(ctypes.byref(s), vocab_size, temperature, topp, ctypes.c_ulonglong(rng_seed))
    return s


def free_sampler(s):
    lib().free_sampler(ctypes.byref(s))


def sample(s, logits_np, entry="sample"):
    """llama2.c sample(): logits_np (float32, writable) is overwritten with the
    probabilities when temperature != 0.  entry="sample_debug" / "do_sample"
    calls the variants of the reference's CUDA translation units instead."""
    fp = logits_np.ctypes.data_as(ctypes.POINTER(ctypes.c_float))
    r = getattr(lib(), entry)(ctypes.byref(s), fp)
    if r < 0:
        raise SamplerError(f"{entry} failed: " + lib().sampler_last_error().decode())
    return r
