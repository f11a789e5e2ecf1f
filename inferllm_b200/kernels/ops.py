"""Single kernels of the library called from Python, for the tests of each kernel alone and for
the kernel benchmarks (`bench.py --kernels`); the engine does not go through this module.

Every function takes CUDA tensors, allocates the outputs and scratch with torch, launches one
kernel entry point of `csrc/` on torch's current stream and returns without synchronising.  A size
that a kernel cannot take is refused with a `KernelError` that names it.  Which kernel the engine
picks for which sizes is decided in the C++ core (`kernels/ops.h`): `linear`, `linear_gated` and the
policy functions here ask it, so the choices tested are the ones that run.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools

import torch

from .. import binding as _b
from ..binding import KernelError   # noqa: F401


def load():
    return _b.lib()

_DT = {torch.float32: 0, torch.bfloat16: 1}
MAX_HEAD_DIM_GENERIC = 256
MAX_SAMPLE_WORDS = 8 * 45056
MAX_NORM_WIDTH = 200 * 1024 // 4


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    """The current CUDA stream's handle (asked for at every launch: the short way, since a prompt
    step of a few hundred tokens is bound by what the host spends per launch)."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


_HERE = contextlib.nullcontext()


def _on(device):
    """For tensors of another device than the current one: kernels are launched on theirs, on its current stream."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


P_, I_, F_, LL_ = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong
_KERNEL_SIGNATURES = {
    "illm_embedding": [P_, P_, I_, P_, I_, I_, I_, P_, P_],
    "illm_add_rmsnorm": [P_, P_, P_, I_, P_, I_, P_, I_, I_, F_, I_, P_],
    "illm_residual_add": [P_, P_, I_, LL_, P_],
    "illm_swiglu": [P_, P_, I_, I_, I_, P_],
    "illm_rope_kv_write": [P_, P_, P_, P_, P_, I_, P_, P_, I_, I_, I_, I_, I_, I_, I_, I_, I_, P_, P_],
    "illm_attention_generic_ex": [P_, I_, P_, P_, P_, I_, P_, P_, P_, I_, I_, I_, I_, I_, I_, I_, F_, I_, P_, P_, I_, I_, F_, I_, P_],
    "illm_attention_generic": [P_, I_, P_, P_, P_, I_, P_, P_, P_, I_, I_, I_, I_, I_, I_, I_, F_, I_, P_, P_, I_, P_],
    "illm_attention_decode": [P_, I_, P_, P_, P_, I_, P_, P_, P_, P_, P_, I_, I_, I_, I_, I_, I_, F_, I_, P_],
    "illm_attention_decode_supported": [I_, I_, I_],
    "illm_attention_decode_gqa": [P_, I_, P_, P_, P_, I_, P_, P_, P_, P_, P_, I_, I_, I_, I_, I_, I_, F_, I_, P_],
    "illm_attention_decode_ring": [P_, I_, P_, P_, LL_, P_, I_, P_, P_, P_, P_, P_, I_, I_, I_, I_, I_, I_, F_, I_, P_, P_],
    "illm_attention_decode_ring_rope": [P_, P_, I_, LL_, P_, I_, I_, I_, P_, P_, LL_, P_, I_, P_, P_, P_, P_, P_, I_, I_, I_, I_, I_, I_,
                                        F_, I_, P_, P_, P_],
    "illm_kv_write_int8": [P_, P_, I_, LL_, P_, P_, P_, P_, P_, I_, LL_, P_, P_, P_, P_, I_, I_, I_, I_, I_, I_, I_, I_, I_, P_, P_],
    "illm_kv_read_int8": [P_, P_, P_, P_, P_, P_, P_, I_, LL_, P_, P_, I_, LL_, I_, I_, I_, P_],
    "illm_attention_int8": [P_, I_, P_, P_, P_, P_, P_, I_, LL_, P_, P_, P_, I_, I_, I_, I_, I_, I_, I_, F_, P_, P_],
    "illm_attention_pages": [P_, I_, P_, P_, P_, P_, LL_, P_, I_, P_, P_, P_, P_, P_, I_, I_, P_, P_, P_, I_, I_, I_, I_, I_, I_, F_, I_, I_, P_, P_],
    "illm_attention_tiles_int8": [P_, I_, P_, P_, P_, P_, LL_, P_, I_, P_, P_, P_, I_, I_, I_, I_, I_, I_, I_, F_, I_, P_, P_],
    "illm_attention_tiles_cluster": [I_],
    "illm_attention_tiles_prefix": [P_, I_, P_, P_, P_, P_, LL_, P_, I_, P_, P_, P_, I_, P_, P_, I_, I_, I_, I_, F_, I_, I_, I_, P_, P_],
    "illm_attention_prefill": [P_, I_, P_, P_, P_, I_, P_, P_, P_, I_, I_, I_, I_, I_, I_, I_, F_, P_],
    "illm_gemm_bf16_tc": [P_, P_, P_, I_, I_, I_, I_, P_, I_, P_, P_, I_],
    "illm_splitk_reduce": [P_, P_, I_, LL_, I_, P_],
    "illm_add_rmsnorm_partials": [P_, P_, I_, LL_, P_, I_, P_, I_, P_, I_, I_, F_, I_, P_],
    "illm_rope_kv_write_partials": [P_, P_, I_, LL_, P_, P_, P_, P_, I_, P_, P_, I_, I_, I_, I_, I_, I_, I_, I_, I_, P_, P_],
    "illm_gemm_bf16_tc2": [P_, P_, P_, I_, I_, I_, I_, I_, P_, P_],
    "illm_swiglu_partials": [P_, I_, LL_, P_, I_, I_, P_],
    "illm_gemm_bf16_tc_gated": [P_, P_, P_, I_, I_, I_, I_, P_, P_],
    "illm_attention_prefill_tc": [P_, I_, I_, P_, P_, LL_, P_, I_, P_, P_, P_, I_, I_, I_, I_, I_, I_, I_, F_, P_, P_],
    "illm_gemm_f32_nt": [P_, P_, P_, I_, I_, I_, I_, I_, I_, P_, P_],
    "illm_argmax": [P_, I_, I_, I_, P_, P_, P_, P_],
    "illm_sample": [P_, I_, I_, I_, P_, P_, I_, F_, F_, I_, F_, P_, P_, P_, P_],
    "illm_sample_scratch_elems": [I_, I_, I_, F_],
    "illm_linear_adapters_ws": [I_, I_, I_, I_, I_, I_, I_, I_],
    "illm_linear_adapters": [P_, P_, I_, I_, I_, I_, P_, P_, P_, I_, I_, P_, I_, I_, I_, P_, I_, P_, I_, P_, P_],
    "illm_sample_rows": [P_, I_, I_, I_, LL_, P_, P_, P_, P_, P_, P_, P_],
    "illm_fill_random": [P_, I_, LL_, ctypes.c_ulonglong, F_, F_, P_],
    "illm_poison_pages": [P_, P_, LL_, I_, LL_, P_, I_, P_],
    "illm_selftest_wait_timeout": [P_, P_, LL_, I_, P_],
}
_declared = False


def _declare():
    """Argument types of the kernels' own entry points (declared on first use)."""
    global _declared
    if _declared:
        return
    h = _b.lib()
    for name, args in _KERNEL_SIGNATURES.items():
        fn = getattr(h, name)
        fn.argtypes = args
        fn.restype = LL_ if name in ("illm_sample_scratch_elems", "illm_linear_adapters_ws") else I_
    _declared = True


_plain_load = load


def load():   # noqa: F811
    _declare()
    return _plain_load()


_replayed = 0


def launch_count() -> int:
    """How many kernels of this package have been launched: the library counts every kernel it
    launches (a launch into a stream capture once), replays of captured graphs are added by
    `count_launches`.  Library products (cuBLAS) are not counted."""
    return int(_b.lib().illm_launch_count_total()) + _replayed


def count_launches(n: int) -> None:
    """Account for kernels launched by replaying a captured graph."""
    global _replayed
    _replayed += n


def _check(code, what):
    if code != 0:
        if code == 10001:
            raise KernelError(f"{what}: the kernel refused its arguments")
        raise KernelError(f"{what}: CUDA error {code}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(t, name, dtype=None, dim=None):
    if not t.is_cuda:
        raise KernelError(f"{name} must be a CUDA tensor: inferllm_b200 has no CPU path")
    if not t.is_contiguous():
        raise KernelError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise KernelError(f"{name} must be {dtype}, found {t.dtype}")
    if dim is not None and t.dim() != dim:
        raise KernelError(f"{name} must have {dim} dimensions, found shape {tuple(t.shape)}")
    # rows of a multiple of 16 bytes are read 16 bytes at a time (the address is looked at first: it
    # is almost always aligned, and these checks run a few hundred times per step)
    if t.data_ptr() & 15 and t.dtype.is_floating_point and t.numel() and (t.shape[-1] * t.element_size()) % 16 == 0:
        raise KernelError(f"{name} must start on a 16-byte boundary")


def act_code(dtype):
    if dtype not in _DT:
        raise KernelError(f"unsupported dtype {dtype}: the kernels take float32 and bfloat16")
    return _DT[dtype]


# The library chooses a kernel for every new shape of a product, which costs a prompt step whose
# token count it has not seen before about 4.5 ms (7B size: 9.5 to 10 ms for a prompt of a never
# seen length of 200 to 300 tokens, 5.2 ms for one seen before), and prompts come in every length.
# Activations of prompt steps are therefore allocated with their rows rounded up to a multiple of
# 64, of which the caller sees the first M; `linear` hands the library the whole buffer and gives
# back the first M rows of the result, so the library only ever sees multiples of 64.  The rows
# beyond M are never initialised and never read back: a row of a product depends on its own row
# of the input only.
LIBRARY_ROW_BUCKET = 64


def _rows(M, cols, dtype, device):
    """An uninitialised [M, cols] activation; for prompt-sized M the head of a buffer of whole buckets."""
    if dtype == torch.bfloat16 and M > LIBRARY_ROW_BUCKET and M % LIBRARY_ROW_BUCKET:
        padded = -(-M // LIBRARY_ROW_BUCKET) * LIBRARY_ROW_BUCKET
        return torch.empty((padded, cols), dtype=dtype, device=device)[:M]
    return torch.empty((M, cols), dtype=dtype, device=device)


def _whole_buckets(x):
    """The buffer of whole buckets behind an activation made by `_rows`, or None."""
    M, K = x.shape
    if M > LIBRARY_ROW_BUCKET and M % LIBRARY_ROW_BUCKET and x.storage_offset() == 0:
        padded = -(-M // LIBRARY_ROW_BUCKET) * LIBRARY_ROW_BUCKET
        if x.untyped_storage().nbytes() >= padded * K * x.element_size():
            return x.as_strided((padded, K), (K, 1))
    return None


def embedding(ids, table, err):
    """ids int32 [T], table [V, H] (float32 or bfloat16) -> float32 [T, H]."""
    _need(ids, "ids", torch.int32, 1)
    _need(table, "table", None, 2)
    T, (V, H) = ids.numel(), table.shape
    out = torch.empty((T, H), dtype=torch.float32, device=ids.device)
    _check(load().illm_embedding(_ptr(ids), _ptr(table), act_code(table.dtype), _ptr(out), T, H, V,
                                 _ptr(err), _stream()), "embedding")
    return out


def add_rmsnorm(resid, delta, weight, eps, out_dtype, rows=None, write_resid=True):
    """y = rmsnorm(resid (+ delta)) * weight; resid is updated in place when `write_resid`.
    `rows` (int32 [K]) gathers: only those rows are normed and y is [K, H]."""
    _need(resid, "resid", torch.float32, 2)
    H = resid.shape[1]
    if H > MAX_NORM_WIDTH:
        raise KernelError(f"rmsnorm: width {H} exceeds the {MAX_NORM_WIDTH} that one block's "
                          "shared memory holds")
    partials = None
    if isinstance(delta, SplitKPartials):
        if out_dtype == torch.bfloat16 and H % 8 == 0 and H <= 16384 and tuple(delta.shape) == tuple(resid.shape):
            partials, delta = delta, None
        else:
            delta = delta.materialize(out_dtype)
    if delta is not None:
        _need(delta, "delta", out_dtype, 2)
        if delta.shape != resid.shape:
            raise KernelError(f"delta {tuple(delta.shape)} does not match resid {tuple(resid.shape)}")
    _need(weight, "norm weight", None, 1)
    if weight.numel() != H:
        raise KernelError(f"norm weight has {weight.numel()} elements, the rows have {H}")
    n = resid.shape[0] if rows is None else rows.numel()
    if rows is not None:
        _need(rows, "rows", torch.int32, 1)
    y = _rows(n, H, out_dtype, resid.device)
    if partials is not None:
        _check(load().illm_add_rmsnorm_partials(
            _ptr(resid), _ptr(partials.ws), partials.splits, partials.rows * partials.cols, _ptr(weight),
            act_code(weight.dtype), _ptr(y), act_code(out_dtype), _ptr(rows), n, H, float(eps),
            1 if write_resid else 0, _stream()), "add_rmsnorm_partials")
        return y
    _check(load().illm_add_rmsnorm(_ptr(resid), _ptr(delta), _ptr(weight), act_code(weight.dtype),
                                   _ptr(y), act_code(out_dtype), _ptr(rows), n, H, float(eps),
                                   1 if write_resid else 0, _stream()), "add_rmsnorm")
    return y


def residual_add(resid, delta):
    if isinstance(delta, SplitKPartials):
        delta = delta.materialize(torch.bfloat16)
    _need(resid, "resid", torch.float32)
    _need(delta, "delta")
    if delta.shape != resid.shape:
        raise KernelError("residual_add: shapes differ")
    _check(load().illm_residual_add(_ptr(resid), _ptr(delta), act_code(delta.dtype), resid.numel(),
                                    _stream()), "residual_add")


def swiglu(gu):
    """silu(gate) * up of a packed projection [T, 2I] whose columns 2i, 2i + 1 are gate and up of
    output i -> [T, I].  `gu` may be `SplitKPartials` (bfloat16 result)."""
    if isinstance(gu, SplitKPartials):
        T, I2 = gu.shape
        if I2 % 16 == 0:
            out = _rows(T, I2 // 2, torch.bfloat16, gu.device)
            _check(load().illm_swiglu_partials(_ptr(gu.ws), gu.splits, gu.rows * gu.cols, _ptr(out), T, I2 // 2,
                                               _stream()), "swiglu_partials")
            return out
        gu = gu.materialize(torch.bfloat16)
    _need(gu, "gu", None, 2)
    T, I2 = gu.shape
    if I2 % 2:
        raise KernelError("swiglu: the packed projection must have an even number of columns")
    out = _rows(T, I2 // 2, gu.dtype, gu.device)
    _check(load().illm_swiglu(_ptr(gu), _ptr(out), act_code(gu.dtype), T, I2 // 2, _stream()), "swiglu")
    return out


def _test_device():
    """The library's device context for calls outside an engine, on torch's current stream."""
    dev = ctypes.c_void_p()
    _b.check(_b.lib().illm_test_device(ctypes.c_void_p(_stream() or 1), ctypes.byref(dev)))    # 1: cudaStreamLegacy (0 would mean "none")
    return dev


_info_dev = None


def _info_device():
    """One device context whose error word and figures serve every call of this module outside an
    engine, whatever torch's current stream is (a context of its own per stream would be created,
    with an allocation, inside a stream capture)."""
    global _info_dev
    if _info_dev is None:
        _info_dev = ctypes.c_void_p()
        _b.check(_b.lib().illm_test_device(ctypes.c_void_p(1), ctypes.byref(_info_dev)))
    return _info_dev


def _take(dev, ptr, shape, dtype, device):
    out = torch.empty(shape, dtype=dtype, device=device)
    if out.numel():
        _b.check(_b.lib().illm_copy_device(dev, out.data_ptr(), ptr, out.numel() * out.element_size()))
    return out


def linear_gated(x, w, backend=None):
    """silu(gate) * up of x [M, K] . w [2I, K]^T, where w's rows 2i, 2i + 1 are the gate and the up
    row of output i -> [M, I], by the kernel the engine picks for these sizes (`ops::linear_gated`)."""
    _need(x, "x", None, 2)
    _need(w, "w", x.dtype, 2)
    dev = _test_device()
    _b.check(_b.lib().illm_test_device_rewind(dev))
    out = ctypes.c_void_p()
    _b.check(_b.lib().illm_op_linear_gated(dev, (backend or _GEMM_BACKEND).encode(), x.data_ptr(), x.shape[0], x.shape[1],
                                           w.data_ptr(), w.shape[0], act_code(x.dtype), ctypes.byref(out)))
    return _take(dev, out, (x.shape[0], w.shape[0] // 2), x.dtype, x.device)


def rope_kv_write(qkv, cos_sin, rot_dim, token_pos, token_seq, block_table, k_cache, v_cache,
                  n_heads, n_kv_heads, head_dim, page_size, write_kv, err):
    """Rotate Q (and K) of the packed projection in place and store K, V in the cache pages.
    `cos_sin` float32 [positions, rot_dim/2, 2] or None with rot_dim 0.  Returns the tensor whose
    first n_heads*head_dim columns hold the rotated queries: `qkv` itself, or, if `qkv` came as
    `SplitKPartials`, a new tensor (the slices are added up on the way)."""
    partials = None
    if isinstance(qkv, SplitKPartials):
        if head_dim % 8 == 0 and rot_dim % 16 == 0 and k_cache is not None and k_cache.dtype == torch.bfloat16:
            partials = qkv
            qkv = torch.empty(partials.shape, dtype=torch.bfloat16, device=partials.device)
        else:
            qkv = qkv.materialize(torch.bfloat16)
    _need(qkv, "qkv", None, 2)
    T = qkv.shape[0]
    if qkv.shape[1] != (n_heads + 2 * n_kv_heads) * head_dim:
        raise KernelError(f"qkv width {qkv.shape[1]} is not (heads + 2 kv heads) * head_dim")
    for name, t in (("token_pos", token_pos), ("token_seq", token_seq)):
        _need(t, name, torch.int32, 1)
    _need(block_table, "block_table", torch.int32, 2)
    if write_kv:
        _need(k_cache, "k_cache", qkv.dtype, 4)
        _need(v_cache, "v_cache", qkv.dtype, 4)
        if tuple(k_cache.shape[1:]) != (n_kv_heads, page_size, head_dim):
            raise KernelError(f"cache pages {tuple(k_cache.shape)} do not match "
                              f"[pages, {n_kv_heads}, {page_size}, {head_dim}]")
    n_pos = 0
    if rot_dim:
        _need(cos_sin, "cos_sin", torch.float32, 3)
        if cos_sin.shape[1] != rot_dim // 2:
            raise KernelError("cos_sin table does not match rot_dim")
        n_pos = cos_sin.shape[0]
    if partials is not None:
        _check(load().illm_rope_kv_write_partials(
            _ptr(qkv), _ptr(partials.ws), partials.splits, partials.rows * partials.cols,
            _ptr(cos_sin) if rot_dim else None, _ptr(token_pos), _ptr(token_seq), _ptr(block_table),
            block_table.shape[1], _ptr(k_cache) if write_kv else None, _ptr(v_cache) if write_kv else None,
            act_code(qkv.dtype), T, n_heads, n_kv_heads, head_dim, rot_dim, page_size, 1 if write_kv else 0,
            n_pos, _ptr(err), _stream()), "rope_kv_write_partials")
        return qkv
    _check(load().illm_rope_kv_write(
        _ptr(qkv), _ptr(cos_sin) if rot_dim else None, _ptr(token_pos), _ptr(token_seq),
        _ptr(block_table), block_table.shape[1], _ptr(k_cache) if write_kv else None,
        _ptr(v_cache) if write_kv else None, act_code(qkv.dtype), T, n_heads, n_kv_heads, head_dim,
        rot_dim, page_size, 1 if write_kv else 0, n_pos, _ptr(err), _stream()), "rope_kv_write")
    return qkv


def attention_generic(qkv, k_cache, v_cache, block_table, token_pos, token_seq, n_heads,
                      n_kv_heads, head_dim, page_size, window, scale, prompts=0):
    """Attention of each token (query heads in the first n_heads*head_dim columns of `qkv`)
    over its sequence's cache pages; returns [T, n_heads*head_dim].  `window` may be negative: chunks of that many
    positions.  `prompts`: 1 takes the tokens by eights, 2 those that are worth it (other kernels, the same result)."""
    if head_dim % 8 or head_dim > MAX_HEAD_DIM_GENERIC:
        raise KernelError(f"attention: head size {head_dim} is not supported (multiples of 8 up to "
                          f"{MAX_HEAD_DIM_GENERIC})")
    if n_heads % n_kv_heads:
        raise KernelError("attention: heads must be a multiple of kv heads")
    _need(qkv, "qkv", None, 2)
    _need(k_cache, "k_cache", qkv.dtype, 4)
    _need(v_cache, "v_cache", qkv.dtype, 4)
    T = qkv.shape[0]
    out = _rows(T, n_heads * head_dim, qkv.dtype, qkv.device)
    _check(load().illm_attention_generic_ex(
        _ptr(qkv), qkv.shape[1], _ptr(k_cache), _ptr(v_cache), _ptr(block_table),
        block_table.shape[1], _ptr(token_pos), _ptr(token_seq), _ptr(out), act_code(qkv.dtype), T,
        n_heads, n_kv_heads, head_dim, page_size, int(window or 0), float(scale), head_dim, None, None, 0,
        0, 0.0, int(prompts), _stream()),
        "attention_generic")
    return out


DECODE_CHUNK = 256


def attention_decode_supported(dtype, n_heads, n_kv_heads, head_dim, page_size) -> bool:
    return dtype == torch.bfloat16 and n_heads % n_kv_heads == 0 and bool(
        load().illm_attention_decode_supported(head_dim, n_heads // n_kv_heads, page_size))


def attention_decode(qkv, k_cache, v_cache, block_table, token_pos, token_seq, n_heads, n_kv_heads,
                     head_dim, page_size, window, scale, max_len):
    """bfloat16 attention of single tokens, split over chunks of 256 keys and merged in a fixed
    order.  `max_len` bounds the sequence lengths of the launch (it sizes the grid and the
    scratch, not the result)."""
    _need(qkv, "qkv", torch.bfloat16, 2)
    _need(k_cache, "k_cache", torch.bfloat16, 4)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    T = qkv.shape[0]
    n_chunks = max(1, -(-int(max_len) // DECODE_CHUNK))
    part_acc = torch.empty((T, n_heads, n_chunks, head_dim), dtype=torch.float32, device=qkv.device)
    part_ml = torch.empty((T, n_heads, n_chunks, 2), dtype=torch.float32, device=qkv.device)
    out = _rows(T, n_heads * head_dim, torch.bfloat16, qkv.device)
    for t0 in range(0, T, 65535):
        t1 = min(T, t0 + 65535)
        _check(load().illm_attention_decode(
            _ptr(qkv[t0:t1]), qkv.shape[1], _ptr(k_cache), _ptr(v_cache), _ptr(block_table),
            block_table.shape[1], _ptr(token_pos[t0:t1]), _ptr(token_seq[t0:t1]), _ptr(part_acc[t0:t1]),
            _ptr(part_ml[t0:t1]), _ptr(out[t0:t1]), t1 - t0, n_heads, n_kv_heads, head_dim, page_size,
            int(window or 0), float(scale), n_chunks, _stream()), "attention_decode")
    return out


GQA_DECODE_CHUNK = 128
GQA_DECODE_MIN_GROUP = 4        # from this many query heads per KV head on, the MMA kernel is the faster one


def attention_decode_gqa_supported(dtype, n_heads, n_kv_heads, head_dim) -> bool:
    return (dtype == torch.bfloat16 and head_dim in (64, 128) and n_heads % n_kv_heads == 0
            and 2 <= n_heads // n_kv_heads <= 16)


def attention_decode_gqa(qkv, k_cache, v_cache, block_table, token_pos, token_seq, n_heads, n_kv_heads,
                         head_dim, page_size, window, scale, max_len):
    """bfloat16 attention of single tokens with grouped heads on warp-level MMAs (the query heads
    of a KV head are the rows of one tile), split over chunks of 128 keys and merged in a fixed
    order.  Any page size, group sizes 2..16, head size 64 or 128."""
    _need(qkv, "qkv", torch.bfloat16, 2)
    _need(k_cache, "k_cache", torch.bfloat16, 4)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    T = qkv.shape[0]
    n_chunks = max(1, -(-int(max_len) // GQA_DECODE_CHUNK))
    part_acc = torch.empty((T, n_heads, n_chunks, head_dim), dtype=torch.float32, device=qkv.device)
    part_ml = torch.empty((T, n_heads, n_chunks, 2), dtype=torch.float32, device=qkv.device)
    out = _rows(T, n_heads * head_dim, torch.bfloat16, qkv.device)
    for t0 in range(0, T, 65535):
        t1 = min(T, t0 + 65535)
        _check(load().illm_attention_decode_gqa(
            _ptr(qkv[t0:t1]), qkv.shape[1], _ptr(k_cache), _ptr(v_cache), _ptr(block_table),
            block_table.shape[1], _ptr(token_pos[t0:t1]), _ptr(token_seq[t0:t1]), _ptr(part_acc[t0:t1]),
            _ptr(part_ml[t0:t1]), _ptr(out[t0:t1]), t1 - t0, n_heads, n_kv_heads, head_dim, page_size,
            int(window or 0), float(scale), n_chunks, _stream()), "attention_decode_gqa")
    return out


RING_DECODE_MAX_SPLITS = 32


def attention_decode_ring_supported(dtype, n_heads, n_kv_heads, head_dim, page_size) -> bool:
    return (dtype == torch.bfloat16 and head_dim in (64, 128) and n_heads % n_kv_heads == 0
            and n_heads // n_kv_heads <= 16 and page_size % 64 == 0)


def attention_decode_ring_splits(T, n_kv_heads, max_len, head_dim=128, n_sms=None) -> int:
    """Blocks per (token, kv head) of the ring decode attention: the engine's policy
    (`ops::attention_decode_ring_splits`), for the SM count of the current device unless given."""
    return int(_b.lib().illm_policy_ring_splits(int(T), int(n_kv_heads), int(max_len), int(head_dim), int(n_sms or n_sms_of_device())))


def attention_diff_splits(T, head_groups, max_seq_len, n_sms=None) -> int:
    """Blocks per (token, group of query heads) of the single-token kernel of differential attention: the engine's
    policy (`ops::attention_diff_splits`), for the SM count of the current device unless given."""
    return int(_b.lib().illm_policy_attention_diff_splits(int(T), int(head_groups), int(max_seq_len), int(n_sms or n_sms_of_device())))


def attention_generic_form(q_lens, n_heads, n_sms=None):
    """How the engine's policy has `attention_generic` take a step whose sequences bring `q_lens` tokens (0 one by one, 1 by eights, 2 by
    eights where that is worth it), and the step's dense and sparse tiles of eight tokens."""
    lens, tiles = (ctypes.c_int * len(q_lens))(*q_lens), (ctypes.c_int * 2)()
    return int(_b.lib().illm_policy_attention_generic(lens, len(q_lens), int(n_heads), int(n_sms or n_sms_of_device()), tiles)), tiles[0], tiles[1]


def scan_form(kind, T, B, max_q, n_heads, head_dim, v_head_dim):
    """Who takes the tokens of a recurrence's step in the bfloat16 mode: 0 token by token, 1 chunks of eight (chunk_scan.cu), 2 the delta
    rule's own chunks.  kind: 0 linear attention, 1 the delta rule with a decay per channel, 2 with one per head."""
    return int(_b.lib().illm_policy_scan_form(int(kind), int(T), int(B), int(max_q), int(n_heads), int(head_dim), int(v_head_dim)))


def attention_decode_ring(qkv, k_cache, v_cache, block_table, token_pos, token_seq, n_heads, n_kv_heads,
                          head_dim, page_size, window, scale, max_len, splits=None, rope=None):
    """bfloat16 attention of single tokens as a stream: K/V tiles of 64 keys by TMA through a ring
    of shared-memory stages, the query heads of a KV head as rows of warp-level MMAs, the tiles
    of a token dealt round-robin to `splits` blocks and merged in a fixed order.  Group sizes
    1..16, head size 64 or 128, pages of a multiple of 64 positions.

    `rope` = (cos_sin table or None, rot_dim, write_kv, step error word): the kernel also does what
    `rope_kv_write` does (rotation of Q and of the new K row, K and V into the cache pages); `qkv`
    is then the unrotated packed projection, as a bfloat16 tensor or as `SplitKPartials`."""
    partials = None
    if isinstance(qkv, SplitKPartials):
        if rope is None:
            raise KernelError("attention_decode_ring: unreduced slices need the fused position encoding")
        partials = qkv
        T = partials.rows
        width = partials.cols
    else:
        _need(qkv, "qkv", torch.bfloat16, 2)
        T, width = qkv.shape
    _need(k_cache, "k_cache", torch.bfloat16, 4)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    if rope is not None and width != (n_heads + 2 * n_kv_heads) * head_dim:
        raise KernelError(f"qkv width {width} is not (heads + 2 kv heads) * head_dim")
    out = torch.empty((T, n_heads * head_dim), dtype=torch.bfloat16, device=k_cache.device)
    for t0 in range(0, T, 65535):
        t1 = min(T, t0 + 65535)
        n = attention_decode_ring_splits(t1 - t0, n_kv_heads, max_len, head_dim) if splits is None else int(splits)
        part_acc = part_ml = None
        if n > 1:
            part_acc = torch.empty((t1 - t0, n_heads, n, head_dim), dtype=torch.float32, device=out.device)
            part_ml = torch.empty((t1 - t0, n_heads, n, 2), dtype=torch.float32, device=out.device)
        if rope is None:
            _check(load().illm_attention_decode_ring(
                _ptr(qkv[t0:t1]), width, _ptr(k_cache), _ptr(v_cache), k_cache.shape[0], _ptr(block_table),
                block_table.shape[1], _ptr(token_pos[t0:t1]), _ptr(token_seq[t0:t1]), _ptr(part_acc), _ptr(part_ml),
                _ptr(out[t0:t1]), t1 - t0, n_heads, n_kv_heads, head_dim, page_size, int(window or 0), float(scale),
                n, _ptr(tc_error_word(out.device)), _stream()), "attention_decode_ring")
            continue
        table, rot_dim, write_kv, step_err = rope
        n_pos = 0
        if rot_dim:
            _need(table, "cos_sin", torch.float32, 3)
            if table.shape[1] != rot_dim // 2:
                raise KernelError("cos_sin table does not match rot_dim")
            n_pos = table.shape[0]
        if T > 65535:
            raise KernelError("attention_decode_ring with the position encoding inside takes at most 65535 tokens")
        _check(load().illm_attention_decode_ring_rope(
            None if partials is not None else _ptr(qkv),
            _ptr(partials.ws) if partials is not None else None,
            partials.splits if partials is not None else 0,
            T * width if partials is not None else 0,
            _ptr(table) if rot_dim else None, int(rot_dim), n_pos, 1 if write_kv else 0, _ptr(k_cache), _ptr(v_cache),
            k_cache.shape[0], _ptr(block_table), block_table.shape[1], _ptr(token_pos[t0:t1]), _ptr(token_seq[t0:t1]),
            _ptr(part_acc), _ptr(part_ml), _ptr(out[t0:t1]), t1 - t0, n_heads, n_kv_heads, head_dim, page_size,
            int(window or 0), float(scale), n, _ptr(tc_error_word(out.device)), _ptr(step_err), _stream()),
            "attention_decode_ring_rope")
    return out


def attention_prefill_supported(dtype, n_heads, n_kv_heads, head_dim) -> bool:
    return dtype == torch.bfloat16 and head_dim in (64, 128) and n_heads % n_kv_heads == 0


def attention_prefill(qkv, k_cache, v_cache, block_table, cu_q, seq_lens, max_q, n_heads, n_kv_heads,
                      head_dim, page_size, window, scale):
    """bfloat16 tensor-core attention of whole prompts (or chunks that continue a sequence).
    `cu_q` int32 [B+1]: token offsets of the sequences in the step; `seq_lens` int32 [B]: their
    lengths after the step; `max_q`: the most tokens one sequence brings."""
    _need(qkv, "qkv", torch.bfloat16, 2)
    _need(k_cache, "k_cache", torch.bfloat16, 4)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    T, B = qkv.shape[0], seq_lens.numel()
    out = _rows(T, n_heads * head_dim, torch.bfloat16, qkv.device)
    _check(load().illm_attention_prefill(
        _ptr(qkv), qkv.shape[1], _ptr(k_cache), _ptr(v_cache), _ptr(block_table), block_table.shape[1],
        _ptr(cu_q), _ptr(seq_lens), _ptr(out), B, int(max_q), n_heads, n_kv_heads, head_dim, page_size,
        int(window or 0), float(scale), _stream()), "attention_prefill")
    return out


def attention_prefill_tc_supported(dtype, n_heads, n_kv_heads, head_dim, page_size) -> bool:
    return (dtype == torch.bfloat16 and head_dim in (64, 128) and n_heads % n_kv_heads == 0
            and page_size % 64 == 0)


def attention_prefill_tc(qkv, k_cache, v_cache, block_table, cu_q, seq_lens, max_q, n_heads, n_kv_heads,
                         head_dim, page_size, window, scale):
    """The tcgen05 / TMA version of `attention_prefill` (head size 64 or 128, pages of a
    multiple of 64 positions)."""
    _need(qkv, "qkv", torch.bfloat16, 2)
    _need(k_cache, "k_cache", torch.bfloat16, 4)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    T, B = qkv.shape[0], seq_lens.numel()
    out = _rows(T, n_heads * head_dim, torch.bfloat16, qkv.device)
    _check(load().illm_attention_prefill_tc(
        _ptr(qkv), qkv.shape[1], T, _ptr(k_cache), _ptr(v_cache), k_cache.shape[0], _ptr(block_table),
        block_table.shape[1], _ptr(cu_q), _ptr(seq_lens), _ptr(out), B, int(max_q), n_heads, n_kv_heads,
        head_dim, page_size, int(window or 0), float(scale), _ptr(tc_error_word(qkv.device)), _stream()),
        "attention_prefill_tc")
    return out


def attention(qkv, kv, ctx, n_heads, n_kv_heads, head_dim, window, scale):
    """Attention of the step's tokens over the cache entry `kv` (a KVView): picks the kernel
    for the dtype, head size and kind of step."""
    group = n_heads // n_kv_heads if n_kv_heads else 0
    # grids and scratch of the decode kernels are sized for the longest sequence the cache allows,
    # so that the launch is the same at every step
    if ctx.is_decode and attention_decode_ring_supported(qkv.dtype, n_heads, n_kv_heads, head_dim, kv.page_size):
        return attention_decode_ring(qkv, kv.k, kv.v, kv.block_table, ctx.token_pos, ctx.token_seq,
                                     n_heads, n_kv_heads, head_dim, kv.page_size, window, scale,
                                     ctx.max_seq_len)
    if ctx.is_decode and (group >= GQA_DECODE_MIN_GROUP or not attention_decode_supported(
            qkv.dtype, n_heads, n_kv_heads, head_dim, kv.page_size)) and attention_decode_gqa_supported(
            qkv.dtype, n_heads, n_kv_heads, head_dim):
        return attention_decode_gqa(qkv, kv.k, kv.v, kv.block_table, ctx.token_pos, ctx.token_seq,
                                    n_heads, n_kv_heads, head_dim, kv.page_size, window, scale,
                                    ctx.max_seq_len)
    if ctx.is_decode and attention_decode_supported(qkv.dtype, n_heads, n_kv_heads, head_dim, kv.page_size):
        return attention_decode(qkv, kv.k, kv.v, kv.block_table, ctx.token_pos, ctx.token_seq,
                                n_heads, n_kv_heads, head_dim, kv.page_size, window, scale,
                                ctx.max_seq_len)
    if not ctx.is_decode and attention_prefill_tc_supported(qkv.dtype, n_heads, n_kv_heads, head_dim,
                                                            kv.page_size):
        return attention_prefill_tc(qkv, kv.k, kv.v, kv.block_table, ctx.cu_q, ctx.seq_lens, ctx.max_q,
                                    n_heads, n_kv_heads, head_dim, kv.page_size, window, scale)
    if not ctx.is_decode and attention_prefill_supported(qkv.dtype, n_heads, n_kv_heads, head_dim):
        return attention_prefill(qkv, kv.k, kv.v, kv.block_table, ctx.cu_q, ctx.seq_lens, ctx.max_q,
                                 n_heads, n_kv_heads, head_dim, kv.page_size, window, scale)
    return attention_generic(qkv, kv.k, kv.v, kv.block_table, ctx.token_pos, ctx.token_seq,
                             n_heads, n_kv_heads, head_dim, kv.page_size, window, scale)


def gemm_f32(x, w):
    """float32 x [M, K] . w [N, K]^T -> [M, N] with float32 FMA accumulation."""
    _need(x, "x", torch.float32, 2)
    _need(w, "w", torch.float32, 2)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise KernelError(f"gemm: x is [{M}, {K}] but w is {tuple(w.shape)}")
    out = torch.empty((M, N), dtype=torch.float32, device=x.device)
    for m0 in range(0, M, 65535 * 64):
        m1 = min(M, m0 + 65535 * 64)
        _check(load().illm_gemm_f32_nt(_ptr(x[m0:m1]), _ptr(w), _ptr(out[m0:m1]), m1 - m0, N, K, K, K,
                                       N, _ptr(tc_error_word(x.device)), _stream()), "gemm_f32")
    return out


def n_sms_of_device() -> int:
    """Multiprocessors of the current device (148 without one: what the CPU tests of the policies use)."""
    if not torch.cuda.is_available():
        return 148
    n, tc, st = ctypes.c_int(), ctypes.c_void_p(), ctypes.c_void_p()
    _b.lib().illm_test_device_info(_info_device(), ctypes.byref(n), ctypes.byref(tc), ctypes.byref(st))
    return n.value


def tc_error_word(device=None):
    """The error word of the tensor-core kernels' bounded waits, of the library's device context for
    calls outside an engine: an int32 tensor [1] that views it."""
    from ..engine import device_view
    n, tc, st = ctypes.c_int(), ctypes.c_void_p(), ctypes.c_void_p()
    _b.lib().illm_test_device_info(_info_device(), ctypes.byref(n), ctypes.byref(tc), ctypes.byref(st))
    return device_view(tc.value, (1,), torch.int32, torch.cuda.current_device())


class SplitKPartials:
    """The K slices of a split matrix product that have not been added up yet: float32
    [splits, M, N].  `add_rmsnorm` and `rope_kv_write` take it in place of the finished tensor
    and do the addition themselves (ascending order of the slice, as the stand-alone reduction
    does), which saves a kernel per product in a decode step; `materialize` is for everyone else."""

    def __init__(self, ws: torch.Tensor):
        self.ws = ws
        self.splits, self.rows, self.cols = ws.shape
        self.shape = (self.rows, self.cols)
        self.device = ws.device

    def materialize(self, dtype=torch.bfloat16) -> torch.Tensor:
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        _check(load().illm_splitk_reduce(_ptr(self.ws), _ptr(out), act_code(dtype), self.rows * self.cols,
                                         self.splits, _stream()), "splitk_reduce")
        return out


def gemm_tc_splits(M, N, K, n_sms=None):
    """How many slices of K a decode-sized product (M <= 64) is cut into: the engine's policy
    (`ops::gemm_tc_splits`)."""
    return int(_b.lib().illm_policy_gemm_tc_splits(int(M), int(N), int(K), int(n_sms or n_sms_of_device())))


def gemm_bf16_tc(x, w, out_dtype=torch.bfloat16, splits=None, defer_reduce=False):
    """bfloat16 x [M, K] . w [N, K]^T on tcgen05 tensor cores, float32 accumulation.
    `defer_reduce`: if the product is split over K, return its slices as `SplitKPartials`
    instead of adding them up."""
    _need(x, "x", torch.bfloat16, 2)
    _need(w, "w", torch.bfloat16, 2)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise KernelError(f"gemm: x is [{M}, {K}] but w is {tuple(w.shape)}")
    if K % 8 or x.data_ptr() % 16 or w.data_ptr() % 16:
        raise KernelError(f"gemm_bf16_tc: K = {K} must be a multiple of 8 and the operands 16-byte aligned")
    out = torch.empty((M, N), dtype=out_dtype, device=x.device)
    if splits is None:
        splits = gemm_tc_splits(M, N, K)
    else:
        k_iters = -(-K // 64)
        splits = max(1, min(int(splits), k_iters))
        splits = -(-k_iters // -(-k_iters // splits))
    if M > 64:
        splits = 1
    ws = torch.empty((splits, M, N), dtype=torch.float32, device=x.device) if splits > 1 else None
    defer = bool(defer_reduce and splits > 1)
    _check(load().illm_gemm_bf16_tc(_ptr(x), _ptr(w), _ptr(out), act_code(out_dtype), M, N, K, _ptr(ws),
                                    splits, _ptr(tc_error_word(x.device)), _stream(), 1 if defer else 0),
           "gemm_bf16_tc")
    return SplitKPartials(ws) if defer else out


def gemm_bf16_tc_gated(x, w):
    """silu(gate) * up of bfloat16 x [M <= 64, K] . w [2I, K]^T (rows 2i, 2i + 1: gate and up of output
    i) -> [M, I] bfloat16, the activation applied to the accumulators (no split of K)."""
    _need(x, "x", torch.bfloat16, 2)
    _need(w, "w", torch.bfloat16, 2)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K or N % 2 or M > 64 or K % 8:
        raise KernelError(f"gemm_bf16_tc_gated: x {tuple(x.shape)}, w {tuple(w.shape)}: at most 64 rows, K a multiple of 8, "
                          "an even number of weight rows")
    out = torch.empty((M, N // 2), dtype=torch.bfloat16, device=x.device)
    _check(load().illm_gemm_bf16_tc_gated(_ptr(x), _ptr(w), _ptr(out), M, N, K, 1, _ptr(tc_error_word(x.device)), _stream()),
           "gemm_bf16_tc_gated")
    return out


def set_pdl(on: bool) -> None:
    """Programmatic dependent launch of the package's kernels (on by default)."""
    _b.lib().illm_set_pdl_enabled(1 if on else 0)


def gemm_bf16_tc2(x, w, out_dtype=torch.bfloat16, gated=False):
    """bfloat16 x [M, K] . w [N, K]^T on pairs of SMs (tcgen05 cta_group::2), for prompts.
    `gated`: w's rows 2i, 2i + 1 are the gate and the up row of output i and the result is
    silu(gate) * up, [M, N / 2]."""
    _need(x, "x", torch.bfloat16, 2)
    _need(w, "w", torch.bfloat16, 2)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise KernelError(f"gemm: x is [{M}, {K}] but w is {tuple(w.shape)}")
    if K % 8 or x.data_ptr() % 16 or w.data_ptr() % 16 or (gated and N % 2):
        raise KernelError(f"gemm_bf16_tc2: K = {K} must be a multiple of 8, the operands 16-byte aligned"
                          " and a gated weight an even number of rows")
    out = _rows(M, N // 2 if gated else N, out_dtype, x.device)
    _check(load().illm_gemm_bf16_tc2(_ptr(x), _ptr(w), _ptr(out), act_code(out_dtype), 1 if gated else 0, M, N, K,
                                     _ptr(tc_error_word(x.device)), _stream()), "gemm_bf16_tc2")
    return out


_GEMM_BACKEND = "auto"


def gemm_backend() -> str:
    return _GEMM_BACKEND


def set_gemm_backend(name: str) -> None:
    """Which kernels `linear` and `linear_gated` of this module ask for when no `backend` is given:
    "auto" | "tc" | "library" (see `ops::GemmBackend`; an engine has its own setting)."""
    global _GEMM_BACKEND
    if name not in ("tc", "library", "auto"):
        raise ValueError("gemm backend must be 'tc', 'library' or 'auto'")
    _GEMM_BACKEND = name


def linear(x, w, out_dtype=None, defer_reduce=False, backend=None):
    """x [M, K] . w [N, K]^T by the kernel the engine picks for these sizes (`ops::linear`).
    `defer_reduce=True` allows the result to come back as `SplitKPartials`."""
    _need(x, "x", None, 2)
    _need(w, "w", x.dtype, 2)
    out_dtype = out_dtype or x.dtype
    dev = _test_device()
    _b.check(_b.lib().illm_test_device_rewind(dev))
    out, ws, splits = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_int()
    M, N = x.shape[0], w.shape[0]
    _b.check(_b.lib().illm_op_linear(dev, (backend or _GEMM_BACKEND).encode(), x.data_ptr(), M, x.shape[1], w.data_ptr(), N,
                                     act_code(x.dtype), act_code(out_dtype), 1 if defer_reduce else 0, ctypes.byref(out),
                                     ctypes.byref(ws), ctypes.byref(splits)))
    if ws.value:
        return SplitKPartials(_take(dev, ws, (splits.value, M, N), torch.float32, x.device))
    return _take(dev, out, (M, N), out_dtype, x.device)


_error_words = {}


def _error_word(device):
    """The address of the tensor-core kernels' error word on this device (outside an engine)."""
    at = _error_words.get(device.index)
    if at is None:
        dev, n, tc, st = ctypes.c_void_p(), ctypes.c_int(), ctypes.c_void_p(), ctypes.c_void_p()
        with _on(device):
            _b.check(_b.lib().illm_test_device(ctypes.c_void_p(1), ctypes.byref(dev)))
            _b.lib().illm_test_device_info(dev, ctypes.byref(n), ctypes.byref(tc), ctypes.byref(st))
        at = _error_words[device.index] = tc.value
    return at


ADAPTER_GROUP, MAX_ADAPTER_RANK = 16, 256


class Adapters:
    """Room for `count` low-rank adapters of one projection W [n_out, n_in], each of a rank up to `rank` (at most 256):
    y += scale * (x A^T) B^T with A [r, n_in] and B [n_out, r].  They are laid out once, as the kernels read them: `a`
    [count, R, n_in] and `b` [count, R / 16, n_out, 16] with R the rank rounded up to 16.  An adapter that was never put has
    rank 0 and adds nothing."""

    def __init__(self, count, rank, n_out, n_in, dtype=torch.bfloat16, device=None):
        if count < 1 or not 1 <= rank <= MAX_ADAPTER_RANK or n_out < 1 or n_in < 1:
            raise KernelError(f"adapters: {count} adapters of rank {rank} for [{n_out}, {n_in}]: at least one, ranks of 1 to {MAX_ADAPTER_RANK}")
        act_code(dtype)
        if dtype == torch.bfloat16 and n_in % 8:
            raise KernelError(f"adapters: the inner size {n_in} must be a multiple of 8 in bfloat16")
        self.count, self.rank, self.n_out, self.n_in, self.dtype = count, rank, n_out, n_in, dtype
        self.R = -(-rank // ADAPTER_GROUP) * ADAPTER_GROUP
        if count * self.R * (n_out // ADAPTER_GROUP + 1) >= 2 ** 31:
            raise KernelError(f"adapters: {count} adapters of {n_out} outputs and rank {self.R} have more than 2^31 rows")
        self.device = torch.empty(0, device="cuda" if device is None else device).device
        if self.device.type != "cuda":
            raise KernelError("adapters live on a CUDA device: inferllm_b200 has no CPU path")
        self.a = torch.zeros((count, self.R, n_in), dtype=dtype, device=self.device)
        self.b = torch.zeros((count, self.R // ADAPTER_GROUP, n_out, ADAPTER_GROUP), dtype=dtype, device=self.device)
        self.scales = torch.zeros((count,), dtype=torch.float32, device=self.device)
        self.ranks = [0] * count
        self.changes = 0        # how often a rank has changed
        self.pointers = self.a.data_ptr(), self.b.data_ptr(), self.scales.data_ptr()
        _error_word(self.device)    # (made here: a call that is captured first of all could not)

    def put(self, i, a, b, scale=1.0):
        """Adapter i becomes scale * b a (a [r, n_in], b [n_out, r], any float type); what it was is gone.  Works on torch's
        current stream, like any torch operation, and looks at the numbers, which have to be finite in the adapters' type.  A plan
        made before an adapter got a larger rank is refused; a captured call keeps the plan, and with it the ranks, that it was
        captured with."""
        if not 0 <= i < self.count:
            raise KernelError(f"adapters: there is no adapter {i} among {self.count}")
        if a.dim() != 2 or b.dim() != 2 or a.shape[1] != self.n_in or b.shape[0] != self.n_out or a.shape[0] != b.shape[1]:
            raise KernelError(f"adapters: factors {tuple(a.shape)} and {tuple(b.shape)} do not fit [r, {self.n_in}] and [{self.n_out}, r]")
        r = a.shape[0]
        if r > self.rank:
            raise KernelError(f"adapters: rank {r} exceeds the {self.rank} there is room for")
        if not (a.is_floating_point() and b.is_floating_point()):
            raise KernelError("adapters: the factors must be floating-point tensors")
        scale = float(scale)
        finite = abs(scale) <= torch.finfo(torch.float32).max
        a, b = (f.detach().to(self.device, self.dtype) for f in (a, b))
        if r > 0:
            # (the prompt product multiplies an adapter's b with the zeros of its neighbours' tokens; NaN is its own least and largest)
            finite = finite and bool(torch.stack(torch.aminmax(a) + torch.aminmax(b)).isfinite().all())
        if not finite:
            raise KernelError(f"adapters: adapter {i} is not finite in {self.dtype}")
        own = self.a.untyped_storage().data_ptr(), self.b.untyped_storage().data_ptr()
        a, b = (f.clone() if f.untyped_storage().data_ptr() in own else f for f in (a, b))      # (an adapter's factors, put again)
        self.a[i, :r] = a
        self.a[i, r:].zero_()
        whole, rest = divmod(r, ADAPTER_GROUP)
        to = self.b[i]
        if whole:
            to[:whole] = b[:, :r - rest].unflatten(1, (whole, ADAPTER_GROUP)).transpose(0, 1)
        to[whole:].zero_()
        if rest:
            to[whole, :, :rest] = b[:, r - rest:]
        self.scales[i] = scale
        if self.ranks[i] != r:
            self.ranks[i] = r
            self.changes += 1

    def remove(self, i):
        """Adapter i adds nothing any more."""
        self.put(i, self.a.new_zeros((0, self.n_in)), self.b.new_zeros((self.n_out, 0)), 0.0)


class AdapterRows:
    """Which adapter each token of a step has: `index` [T] of whole numbers on the host, -1 for none.  Made once per step and
    used for every projection whose adapters have these ranks (or smaller ones)."""

    def __init__(self, index, ranks, device=None):
        index = index.tolist() if hasattr(index, "tolist") else list(index)
        self.T, self.ranks = len(index), list(ranks)
        self.named = sorted({a for a in index if a >= 0})
        self.device = torch.empty(0, device="cuda" if device is None else device).device
        sizes, total, c_index, c_ranks = (ctypes.c_int * 4)(), ctypes.c_int(), _b.ints(index), _b.ints(self.ranks)
        _b.check(_b.lib().illm_adapter_plan(c_index, self.T, c_ranks, len(self.ranks), sizes, ctypes.byref(total), None))
        host = torch.zeros(total.value, dtype=torch.int32)
        _b.check(_b.lib().illm_adapter_plan(c_index, self.T, c_ranks, len(self.ranks), sizes, ctypes.byref(total),
                                            ctypes.cast(host.data_ptr(), _b.PI)))
        self.slots, self.groups, self.chunks = sizes[1], sizes[2], sizes[3]
        self.plan = host.to(self.device)
        self.plan_ptr = self.plan.data_ptr()
        self._fitted, self._ws = None, {}
        self.most_groups = max((-(-self.ranks[a] // ADAPTER_GROUP) for a in self.named), default=0)

    def ws_bytes(self, code, N, K, R):
        """The workspace of a product by this plan."""
        n = self._ws.get((code, N, K, R))
        if n is None:
            n = self._ws[code, N, K, R] = load().illm_linear_adapters_ws(code, self.T, N, K, R, self.slots, self.groups, self.chunks)
        return n

    def fits(self, adapters):
        """Whether the plan covers these adapters' ranks."""
        if self._fitted is not None and self._fitted[0] is adapters and self._fitted[1] == adapters.changes:
            return True
        have, need = self.ranks, adapters.ranks
        ok = all(a < len(need) and -(-need[a] // ADAPTER_GROUP) <= -(-have[a] // ADAPTER_GROUP) for a in self.named) and self.most_groups * ADAPTER_GROUP <= adapters.R
        if ok:
            self._fitted = adapters, adapters.changes
        return ok


def linear_adapters(x, w, adapters, rows, out_dtype=None):
    """y[t] = x[t] . W^T + scale_a (x[t] . A_a^T) . B_a^T, a the adapter that `rows` gives token t (none: the product alone).
    x [T, K], w [N, K] float32 or bfloat16, `adapters` an `Adapters` of [N, K], `rows` an `AdapterRows` of T tokens; sums in
    float32, rounded once to `out_dtype` (default x's; float32 is the other choice)."""
    if x.dim() != 2 or w.dim() != 2 or not (x.is_contiguous() and w.is_contiguous()):
        raise KernelError(f"linear_adapters: x and w must be contiguous matrices, found {tuple(x.shape)} and {tuple(w.shape)}")
    (T, K), (N, wk) = x.shape, w.shape
    device, dtype, out_dtype = x.device, x.dtype, out_dtype or x.dtype
    if adapters.device != device or w.device != device or rows.device != device:
        raise KernelError(f"linear_adapters: x is on {device}, w on {w.device}, the adapters on {adapters.device} and the plan on {rows.device}: one CUDA device is needed")
    if wk != K or adapters.n_in != K or adapters.n_out != N or adapters.dtype != dtype or w.dtype != dtype:
        raise KernelError(f"linear_adapters: x is {dtype} [{T}, {K}], w {w.dtype} [{N}, {wk}] and the adapters are {adapters.dtype} for [{adapters.n_out}, {adapters.n_in}]")
    if rows.T != T:
        raise KernelError(f"linear_adapters: the plan is of {rows.T} tokens, x has {T}")
    if not rows.fits(adapters):
        raise KernelError("linear_adapters: the plan was made for other ranks than the adapters have: make a new one")
    if out_dtype not in _DT or (dtype == torch.float32 and out_dtype != dtype):
        raise KernelError(f"linear_adapters: a result in {out_dtype} of {dtype} operands (float32, or the operands' type)")
    px, pw = x.data_ptr(), w.data_ptr()
    if (px | pw) & 15 and (dtype == torch.bfloat16 or K % 4 == 0):
        raise KernelError("linear_adapters: x and w must start on a 16-byte boundary")
    # (new_empty with plain arguments: half the host's time of torch.empty, and a call of few tokens is bound by the host)
    out = x.new_empty(T, N) if out_dtype is dtype else x.new_empty(T, N, dtype=out_dtype)
    if T == 0:
        return out
    lib, code = load(), _DT[dtype]
    a, b, scales = adapters.pointers
    with _on(device):
        ws = x.new_empty(rows.ws_bytes(code, N, K, adapters.R), dtype=torch.uint8)
        _check(lib.illm_linear_adapters(px, pw, code, T, N, K, a, b, scales, adapters.count, adapters.R, rows.plan_ptr, rows.slots, rows.groups, rows.chunks,
                                        out.data_ptr(), _DT[out_dtype], ws.data_ptr(), 0, _error_word(device), _stream()), "linear_adapters")
    return out


# ---- a cache of eight-bit rows, and positions that sequences hold in common

def _stream_on(device):
    """The current stream of the current device, where that is known: one question less."""
    return _raw_stream(device.index) if _raw_stream is not None else _stream()


def _rows_beside(x, M, cols, dtype):
    """`_rows` on the device of x (1.3 us of the host's time instead of 2.4)."""
    if M > LIBRARY_ROW_BUCKET:
        return _rows(M, cols, dtype, x.device)
    return x.new_empty(M, cols) if x.dtype is dtype else x.new_empty(M, cols, dtype=dtype)


class _Fixed:
    """What a call takes from it (sizes, addresses) is looked up once, so it stays as it was made: to have other tensors make another."""

    def __setattr__(self, name, value):
        raise AttributeError(f"{type(self).__name__}.{name} is not changed: make another")

    def __delattr__(self, name):
        raise AttributeError(f"{type(self).__name__}.{name} is not taken away")


class CacheInt8(_Fixed):
    """Keys and values of one cache entry in eight bits: `k`, `v` uint8 [pages, kv heads, page_size, head_dim] and `k_scale`,
    `v_scale` float32 [pages, kv heads, page_size].  A row (the values of one position and kv head) stands for
    (u - 128) * scale; `kv_write_int8` makes it with scale = max|x| / 127.  The tensors are held and written in place; none can be put in
    another's place."""

    def __init__(self, k, v, k_scale, v_scale):
        for name, t in (("k", k), ("v", v)):
            _need(t, name, torch.uint8, 4)
            if t.shape != k.shape or t.device != k.device:
                raise KernelError(f"cache: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            _need(t, name, torch.float32, 3)
            if t.shape != k.shape[:3] or t.device != k.device:
                raise KernelError(f"cache: {name} {tuple(t.shape)} does not fit pages {tuple(k.shape)}")
        if any(t.data_ptr() & 15 for t in (k, v, k_scale, v_scale)):
            raise KernelError("cache: pages and scales must start on 16-byte boundaries")
        pages, n_kv_heads, page_size, head_dim = k.shape
        if min(k.shape) < 1 or head_dim % 8 or head_dim > MAX_HEAD_DIM_GENERIC:
            raise KernelError(f"cache: pages {tuple(k.shape)}: head sizes are multiples of 8 up to {MAX_HEAD_DIM_GENERIC}")
        if k.numel() // head_dim >= 2 ** 31:
            raise KernelError(f"cache: pages {tuple(k.shape)} have more than 2^31 rows")
        # (tensors of its own over the same memory: one that a user points elsewhere leaves these, and the addresses, as they are)
        k, v, k_scale, v_scale = (t.detach() for t in (k, v, k_scale, v_scale))
        self.__dict__.update(k=k, v=v, k_scale=k_scale, v_scale=v_scale, pages=pages, n_kv_heads=n_kv_heads, page_size=page_size, head_dim=head_dim, device=k.device,
                             pointers=(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()))
        _error_word(k.device)       # (made here: a call that is captured first of all could not)

    @classmethod
    def empty(cls, pages, n_kv_heads, page_size, head_dim, device="cuda"):
        """Room for so many pages; what lies in them is nobody's."""
        def rows(dtype, *more):
            return torch.empty((pages, n_kv_heads, page_size) + more, dtype=dtype, device=device)
        return cls(rows(torch.uint8, head_dim), rows(torch.uint8, head_dim), rows(torch.float32), rows(torch.float32))


def _page_entry(cache):
    """Of a cache entry (CacheInt8 or a bfloat16 pair (k, v)): its device, pages, kv heads, page size, head size and pointers."""
    if isinstance(cache, CacheInt8):
        return cache.device, cache.pages, cache.n_kv_heads, cache.page_size, cache.head_dim, cache.pointers
    k, v = cache
    _need(k, "k", torch.bfloat16, 4)
    _need(v, "v", torch.bfloat16, 4)
    if k.shape != v.shape or k.device != v.device or min(k.shape) < 1:
        raise KernelError(f"cache: k {tuple(k.shape)} and v {tuple(v.shape)} must be alike and not empty")
    return (k.device,) + tuple(k.shape) + ((k.data_ptr(), v.data_ptr(), None, None),)


def _step_array(t, name, T, device):
    # (these run before every small kernel: one look at what is almost always right, the words only where it is not)
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != T or t.device != device or not t.is_contiguous():
        raise KernelError(f"{name} must be int32 [{T}] on {device}, found {t.dtype} {tuple(t.shape)} on {t.device}")


def _block_table(t, device):
    if t.dtype is not torch.int32 or t.dim() != 2 or t.shape[1] < 1 or t.device != device or not t.is_contiguous():
        raise KernelError(f"block_table must be int32 [sequences, pages] with at least one page, on {device}, found {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.shape[1]


def _query_rows(q, device, n_heads, n_kv_heads, head_dim):
    """The query heads in the first n_heads * head_dim columns of q (rows may lie further apart): rows and their distance."""
    if q.dim() != 2 or q.device != device:
        raise KernelError(f"q must be a matrix on {device}, found shape {tuple(q.shape)} on {q.device}")
    act_code(q.dtype)
    if n_heads < 1 or n_heads % n_kv_heads:
        raise KernelError(f"attention: {n_heads} heads are no multiple of {n_kv_heads} kv heads")
    (T, width), (apart, side) = q.shape, q.stride()
    if width < n_heads * head_dim:
        raise KernelError(f"q has {width} columns, {n_heads} heads of {head_dim} need {n_heads * head_dim}")
    if T and (side != 1 or (T > 1 and not width <= apart < 2 ** 31)):
        raise KernelError("q: a row's elements must lie side by side, and rows apart, by less than 2^31")
    if T and (q.data_ptr() & 15 or (T > 1 and apart * q.element_size() & 15)):
        raise KernelError("q: rows must start on 16-byte boundaries")
    return T, apart if T > 1 else -(-width // 8) * 8


def kv_write_int8(qkv, cos_sin, rot_dim, token_pos, token_seq, block_table, cache, n_heads, err):
    """Rotate the queries and keys of the packed projection [T, (heads + 2 kv heads) * head_dim] and write keys and values into
    the pages of `cache` (CacheInt8) in eight bits.
    `cos_sin` float32 [positions, rot_dim/2, 2] or None with rot_dim 0.  Returns the rotated queries [T, heads * head_dim], a
    new tensor; `qkv` may be `SplitKPartials`.  `err` (int32 [1]): 2 for a position without a page, 3 for one beyond the table;
    such a token's rows are not written.  Two tokens of one call must not name the same position."""
    if not isinstance(cache, CacheInt8):
        raise KernelError("kv_write_int8 writes a CacheInt8")
    device, d, nkv = cache.device, cache.head_dim, cache.n_kv_heads
    if isinstance(qkv, SplitKPartials):
        dtype, at, parts, splits, apart = torch.bfloat16, None, qkv.ws.data_ptr(), qkv.splits, qkv.rows * qkv.cols
    else:
        _need(qkv, "qkv", None, 2)
        dtype, at, parts, splits, apart = qkv.dtype, qkv.data_ptr(), None, 0, 0
    code = act_code(dtype)
    T, columns = qkv.shape
    if columns != (n_heads + 2 * nkv) * d or n_heads < 1:
        raise KernelError(f"qkv width {columns} is not (heads + 2 kv heads) * head_dim")
    if qkv.device != device or err.device != device:
        raise KernelError("qkv, err and the cache must be on one device")
    _need(err, "err", torch.int32)
    width = _block_table(block_table, device)
    _step_array(token_pos, "token_pos", T, device)
    _step_array(token_seq, "token_seq", T, device)
    if rot_dim < 0 or rot_dim > d or rot_dim % 2:
        raise KernelError(f"rot_dim {rot_dim} must be even and at most the head size {d}")
    n_pos, turns = 0, None
    if rot_dim:
        if cos_sin is None:
            raise KernelError("a rotation needs its cos/sin table")
        _need(cos_sin, "cos_sin", torch.float32, 3)
        n_pos, half, two = cos_sin.shape
        if half != rot_dim // 2 or two != 2 or cos_sin.device != device:
            raise KernelError("cos_sin table does not match rot_dim")
        turns = cos_sin.data_ptr()
        if turns & 15:
            raise KernelError("cos_sin must start on a 16-byte boundary")
    with _on(device):
        q = _rows_beside(err, T, n_heads * d, dtype)
        _check(load().illm_kv_write_int8(
            at, parts, splits, apart, q.data_ptr(), turns, token_pos.data_ptr(), token_seq.data_ptr(), block_table.data_ptr(), width, cache.pages, *cache.pointers, code, T,
            n_heads, nkv, d, rot_dim, cache.page_size, 1, n_pos, err.data_ptr(), _stream_on(device)), "kv_write_int8")
    return q


def kv_read_int8(cache, token_pos, token_seq, block_table, dtype=torch.bfloat16):
    """What the rows of given positions stand for: keys and values [n, kv heads, head_dim] of `dtype`.  A position without a page reads as
    NaN."""
    if not isinstance(cache, CacheInt8):
        raise KernelError("kv_read_int8 reads a CacheInt8")
    n, code, width = token_pos.numel(), act_code(dtype), _block_table(block_table, cache.device)
    _step_array(token_pos, "token_pos", n, cache.device)
    _step_array(token_seq, "token_seq", n, cache.device)
    with _on(cache.device):
        k = cache.k_scale.new_empty(n, cache.n_kv_heads, cache.head_dim, dtype=dtype)
        v = torch.empty_like(k)
        _check(load().illm_kv_read_int8(*cache.pointers, token_pos.data_ptr(), token_seq.data_ptr(), block_table.data_ptr(), width, cache.pages, k.data_ptr(), v.data_ptr(), code, n, cache.n_kv_heads, cache.head_dim, cache.page_size, _stream_on(cache.device)), "kv_read_int8")
    return k, v


def attention_int8_tc_supported(dtype, n_heads, n_kv_heads, head_dim, page_size, decode) -> bool:
    """Whether the tensor-core kernels take these sizes (the engine's rule); the others go to the plain kernel."""
    return (dtype == torch.bfloat16 and n_heads % n_kv_heads == 0 and head_dim in (64, 128) and page_size % 64 == 0
            and (not decode or n_heads // n_kv_heads <= 16))


def _attention_int8_plain(q, stride, cache, block_table, token_pos, token_seq, n_heads, span, scale):
    T = q.shape[0]
    out = _rows_beside(q, T, n_heads * cache.head_dim, q.dtype)
    _check(load().illm_attention_int8(_ptr(q), stride, *cache.pointers, _ptr(block_table), block_table.shape[1], cache.pages, _ptr(token_pos), _ptr(token_seq), _ptr(out),
                                      act_code(q.dtype), T, n_heads, cache.n_kv_heads, cache.head_dim, cache.page_size, span, float(scale),
                                      _error_word(cache.device), _stream_on(cache.device)), "attention_int8")
    return out


_sms = {}


def _splits(pairs, keys, wide, device) -> int:
    n_sms = _sms.get(device.index)
    if n_sms is None:
        n_sms = _sms[device.index] = torch.cuda.get_device_properties(device).multi_processor_count
    return pages_splits(pairs, keys, wide, n_sms)


@functools.lru_cache(maxsize=4096)
def pages_splits(pairs, keys, wide, n_sms) -> int:
    """Blocks per (token, kv head) of `attention_decode_int8`, or (`wide`) parts of a common prefix that 256 rows walk together: the engine's policies
    (`ops::attention_pages_splits`, `ops::attention_prefix_splits`)."""
    return int(_b.lib().illm_policy_pages_splits(int(pairs), int(keys), int(wide), int(n_sms)))


@functools.lru_cache(maxsize=4096)
def _in_cluster(pairs, splits, n_sms):
    """Whether the blocks of a (token, kv head) join their shares as a cluster (`ops::attention_pages_in_cluster`)."""
    return bool(_b.lib().illm_policy_pages_in_cluster(pairs, splits, n_sms))


def _shares(q, T, n_heads, slots, d):
    """Scratch of attention_pages beside q and where its two parts begin."""
    cut = T * n_heads * slots * d
    ws = q.new_empty(cut + T * n_heads * slots * 2, dtype=torch.float32)
    at = ws.data_ptr()
    return ws, at, at + 4 * cut


def attention_decode_int8(q, cache, block_table, token_pos, token_seq, n_heads, window, scale, max_len, splits=None):
    """Attention of single tokens over a cache of eight-bit rows: q [T, >= heads * head_dim] (rotated query heads first), the token's own position
    included.  `window` as elsewhere (0 all, negative: chunks).  `max_len` bounds the sequences' lengths (it sizes the grid, not the result).
    Returns [T, heads * head_dim].  bfloat16 with head sizes 64 and 128 and pages of a multiple of 64 positions runs on tensor cores, everything else
    (float32 among it) on a plain kernel."""
    if not isinstance(cache, CacheInt8):
        raise KernelError("attention_decode_int8 reads a CacheInt8")
    device, d, nkv, span = cache.device, cache.head_dim, cache.n_kv_heads, int(window or 0)
    T, stride = _query_rows(q, device, n_heads, nkv, d)
    width = _block_table(block_table, device)
    _step_array(token_pos, "token_pos", T, device)
    _step_array(token_seq, "token_seq", T, device)
    max_len = int(max_len)
    if max_len < 1:
        raise KernelError(f"max_len must be positive, found {max_len}")
    with _on(device):
        if not attention_int8_tc_supported(q.dtype, n_heads, nkv, d, cache.page_size, True):
            return _attention_int8_plain(q, stride, cache, block_table, token_pos, token_seq, n_heads, span, scale)
        out = q.new_empty(T, n_heads * d)
        run, keys, err, stream = load().illm_attention_pages, min(max_len, abs(span)) if span else max_len, _error_word(device), _stream_on(device)
        for t0 in range(0, T, 65535):
            n = min(T - t0, 65535)
            s = _splits(n * nkv, keys, False, device)
            s = s if splits is None else int(splits)
            ws, acc, ml = (None, None, None) if s == 1 or _in_cluster(n * nkv, s, _sms[device.index]) else _shares(q, n, n_heads, s, d)
            _check(run(q.data_ptr() + t0 * stride * 2, stride, *cache.pointers, cache.pages, block_table.data_ptr(), width, token_pos.data_ptr() + 4 * t0,
                       token_seq.data_ptr() + 4 * t0, None, None, None, 0, 0, acc, ml, out.data_ptr() + t0 * n_heads * d * 2, n, n_heads, nkv, d, cache.page_size, span,
                       float(scale), s, 0, err, stream), "attention_decode_int8")
    return out


def attention_prompts_int8(q, cache, block_table, cu_q, seq_lens, max_q, n_heads, window, scale, tile_rows=None):
    """Attention of whole prompts (or chunks that continue a sequence) over a cache of eight-bit rows, the step's own rows written already.
    `cu_q` int32 [B + 1], `seq_lens` int32 [B] (after the step) and `max_q` as for `attention_prefill_tc` (at least the most new tokens of a sequence: rows
    behind it are not written, nor are those behind the last sequence).  Returns [T, heads * head_dim].  bfloat16 with head
    sizes 64 and 128 and pages of a multiple of 64 positions."""
    if not isinstance(cache, CacheInt8):
        raise KernelError("attention_prompts_int8 reads a CacheInt8")
    device, d, nkv, B, max_q = cache.device, cache.head_dim, cache.n_kv_heads, seq_lens.numel(), int(max_q)
    T, stride = _query_rows(q, device, n_heads, nkv, d)
    width = _block_table(block_table, device)
    _step_array(seq_lens, "seq_lens", B, device)
    _step_array(cu_q, "cu_q", B + 1, device)
    if max_q < 0 or max_q > T:
        raise KernelError(f"max_q {max_q} is outside the step's {T} tokens")
    if not attention_int8_tc_supported(q.dtype, n_heads, nkv, d, cache.page_size, False):
        raise KernelError(f"attention_prompts_int8 takes bfloat16, head sizes 64 and 128 and pages of a multiple of 64 positions, found {q.dtype}, {d} and "
                          f"{cache.page_size} (attention_decode_int8 takes prompts of other sizes token by token)")
    with _on(device):
        out = _rows_beside(q, T, n_heads * d, torch.bfloat16)
        if T and B:
            _check(load().illm_attention_tiles_int8(q.data_ptr(), stride, *cache.pointers, cache.pages, block_table.data_ptr(), width, cu_q.data_ptr(), seq_lens.data_ptr(),
                                                    out.data_ptr(), B, max_q, n_heads, nkv, d, cache.page_size, int(window or 0), float(scale), int(tile_rows or 0),
                                                    _error_word(device), _stream_on(device)), "attention_prompts_int8")
    return out


class SharedPrefixes(_Fixed):
    """Which tokens of a step (one per sequence) see their first positions in common: `groups` of (positions, [tokens]), whose block tables name
    the same pages for those positions; `lens` [T] on the host: the positions that each token sees, its own included; `group_heads`: query heads per kv
    head (at most 16).  Made once per step and used for every layer.  Tokens in no group are served too."""

    def __init__(self, groups, lens, group_heads, device=None):
        groups = [(int(p), [int(t) for t in m]) for p, m in groups]
        lens = lens.tolist() if hasattr(lens, "tolist") else list(lens)
        T, group_heads = len(lens), int(group_heads)
        device = torch.empty(0, device="cuda" if device is None else device).device
        sizes, total = (ctypes.c_int * 7)(), ctypes.c_int()
        args = (len(groups), _b.ints(p for p, _ in groups), _b.ints(len(m) for _, m in groups), _b.ints(t for _, m in groups for t in m), _b.ints(lens), T, group_heads, sizes,
                ctypes.byref(total))
        _b.check(_b.lib().illm_prefix_plan(*args, None))
        host = torch.zeros(max(1, total.value), dtype=torch.int32)
        _b.check(_b.lib().illm_prefix_plan(*args, ctypes.cast(host.data_ptr(), _b.PI)))
        plan = host.to(device)
        at = plan.data_ptr()
        self.__dict__.update(T=T, group_heads=group_heads, device=device, tiles=sizes[0], wide=bool(sizes[1]), longest_prefix=sizes[2], longest_rest=sizes[3], per_tile=sizes[6],
                             longest=max(lens), host=host, plan=plan, pointers=(at + 4 * sizes[4], at, at + 4 * sizes[5]))         # start, tiles, members
        _error_word(device)         # (as in CacheInt8)


def attention_decode_shared(q, cache, block_table, token_pos, token_seq, plan, n_heads, scale, max_len, own_splits=None, pre_splits=None):
    """Attention of single tokens whose sequences hold first positions in common (`plan`, SharedPrefixes): a group's common keys are read once for all of
    its tokens.  `cache`: CacheInt8 or a bfloat16 pair (k, v) of pages [pages, kv heads, page_size, head_dim]; all positions are visible (no window).
    `token_pos` must be those that the plan was made for, `max_len` at least the longest.  bfloat16 queries, head sizes 64 and 128, pages of a multiple of 64
    positions, at most 16 query heads per kv head; others are refused."""
    device, pages, nkv, page_size, d, pointers = _page_entry(cache)
    T, stride = _query_rows(q, device, n_heads, nkv, d)
    width = _block_table(block_table, device)
    _step_array(token_pos, "token_pos", T, device)
    _step_array(token_seq, "token_seq", T, device)
    if not attention_int8_tc_supported(q.dtype, n_heads, nkv, d, page_size, True):
        raise KernelError(f"attention_decode_shared takes bfloat16, head sizes 64 and 128, pages of a multiple of 64 positions and up to 16 query heads per kv head, "
                          f"found {q.dtype}, {d}, {page_size} and {n_heads} over {nkv}")
    if plan.T != T or plan.device != device or plan.group_heads != n_heads // nkv:
        raise KernelError(f"attention_decode_shared: the plan is for {plan.T} tokens with {plan.group_heads} query heads per kv head on {plan.device}")
    if not float(scale) >= 0.0:
        raise KernelError(f"attention_decode_shared: the scale {scale} must not be negative")
    if int(max_len) < plan.longest:
        raise KernelError(f"attention_decode_shared: max_len {max_len} is below the plan's longest sequence {plan.longest}")
    with _on(device):
        out = q.new_empty(T, n_heads * d)
        common = plan.tiles > 0
        own = _splits(T * nkv, max(1, plan.longest_rest), False, device) if own_splits is None else int(own_splits)
        pre = (_splits(plan.tiles * nkv, plan.longest_prefix, plan.wide, device) if pre_splits is None else int(pre_splits)) if common else 0
        kept = pre // load().illm_attention_tiles_cluster(pre) if plan.wide and pre > 0 else pre           # shares of the prefixes that are left in memory
        ws, acc, ml = _shares(q, T, n_heads, own + kept, d) if common or own > 1 else (None, None, None)
        start, tiles, members = plan.pointers if common else (None, None, None)
        h, err, stream = load(), _error_word(device), _stream_on(device)
        at, table, pos, seq = q.data_ptr(), block_table.data_ptr(), token_pos.data_ptr(), token_seq.data_ptr()
        if common and plan.wide:
            _check(h.illm_attention_tiles_prefix(at, stride, *pointers, pages, table, width, seq, tiles, members, plan.tiles, acc, ml, n_heads, nkv, d, page_size,
                                                 float(scale), own + kept, own, pre, err, stream), "attention_decode_shared")
        _check(h.illm_attention_pages(at, stride, *pointers, pages, table, width, pos, seq, start, tiles, members, 0 if plan.wide else plan.tiles, plan.per_tile, acc, ml,
                                      out.data_ptr(), T, n_heads, nkv, d, page_size, 0, float(scale), own, kept, err, stream), "attention_decode_shared")
    return out


def argmax(logits):
    """float32 [B, V] -> int32 [B], the lowest id among equal maxima (two passes: chunks of 2048
    elements, then the chunks' results)."""
    _need(logits, "logits", torch.float32, 2)
    B, V = logits.shape
    out = torch.empty((B,), dtype=torch.int32, device=logits.device)
    n_chunks = -(-V // 2048)
    for b0 in range(0, B, 65535):
        b1 = min(B, b0 + 65535)
        sv = torch.empty((b1 - b0, n_chunks), dtype=torch.float32, device=logits.device)
        si = torch.empty((b1 - b0, n_chunks), dtype=torch.int32, device=logits.device)
        _check(load().illm_argmax(_ptr(logits[b0:b1]), b1 - b0, V, V, _ptr(out[b0:b1]), _ptr(sv), _ptr(si),
                                  _stream()), "argmax")
    return out


def sample(logits, uniforms, temp, top_k=0, top_p=1.0, repeat_penalty=1.0, last_tokens=None):
    """Temperature / repetition penalty / top-k / top-p sampling, one draw per row.
    `uniforms` float32 [B] in [0, 1); `last_tokens` int32 [B, n] (-1 pads) or None."""
    _need(logits, "logits", torch.float32, 2)
    _need(uniforms, "uniforms", torch.float32, 1)
    B, V = logits.shape
    if uniforms.numel() != B:
        raise KernelError("sample: one uniform number per row is needed")
    n_last = 0
    if last_tokens is not None:
        _need(last_tokens, "last_tokens", torch.int32, 2)
        n_last = last_tokens.shape[1]
    z = torch.empty((B, V), dtype=torch.float32, device=logits.device)
    out = torch.empty((B,), dtype=torch.int32, device=logits.device)
    for b0 in range(0, B, 65535):
        b1 = min(B, b0 + 65535)
        # temperature alone and top_k <= 64 run in two passes over chunks of the row and need scratch
        n_scratch = int(load().illm_sample_scratch_elems(b1 - b0, V, int(top_k), float(top_p)))
        scratch = torch.empty((n_scratch,), dtype=torch.int32, device=logits.device) if n_scratch else None
        _check(load().illm_sample(_ptr(logits[b0:b1]), b1 - b0, V, V, _ptr(z[b0:b1]),
                                  _ptr(last_tokens[b0:b1]) if last_tokens is not None else None, n_last, float(temp),
                                  float(repeat_penalty), int(top_k), float(top_p), _ptr(uniforms[b0:b1]),
                                  _ptr(out[b0:b1]), _ptr(scratch), _stream()), "sample")
    return out


def _per_row(t, name, dtype, B, device):
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != (B,) or not t.is_contiguous() or t.device != device:
        raise KernelError(f"sample_rows: {name} must be a contiguous {dtype} tensor [{B}] on {device}, found {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def sample_rows(logits, uniforms, temp=None, top_k=None, top_p=None, min_p=None):
    """The next token of every row by settings of its own -> int32 [B].

    logits [B, V] float32 or bfloat16 (rows may be further apart than V); uniforms float32 [B] in [0, 1); temp, top_p and
    min_p float32 [B], top_k int32 [B], each None for "off" in every row (temperature 1).  With w = exp((l - max l) / temp) and
    the words in descending order of their logit (equal ones in ascending order of their id), a row keeps the first top_k
    (<= 0: all), of these the shortest prefix whose weight reaches top_p of theirs (>= 1: all, <= 0: the first), of these the
    words with w >= min_p (<= 0: all, above 1 counts as 1), and takes the first of them, ids ascending, at which the sum of the weights
    exceeds u times their whole sum.  temp <= 0 or NaN: the lowest id of the largest.  Words at -inf or NaN never come; a row
    without any other gives -1.  Weights are made in float64 and summed as integers: the result does not depend on the
    order of a sum."""
    if not logits.is_cuda:
        raise KernelError("logits must be a CUDA tensor: inferllm_b200 has no CPU path")
    if logits.dim() != 2 or logits.dtype not in _DT:
        raise KernelError(f"sample_rows: logits must be float32 or bfloat16 [B, V], found {logits.dtype} {tuple(logits.shape)}")
    B, V = logits.shape
    device = logits.device
    if V == 0 or (V > 1 and logits.stride(1) != 1) or (B > 1 and logits.stride(0) < V):
        raise KernelError(f"sample_rows: rows of at least one word, each contiguous and none within another, found {tuple(logits.shape)} with strides {logits.stride()}")
    if V > MAX_SAMPLE_WORDS:
        raise KernelError(f"sample_rows: rows of {V} words exceed the {MAX_SAMPLE_WORDS} that a cluster's shared memory holds")
    if uniforms is None:
        raise KernelError("sample_rows: one uniform number per row is needed")
    u = _per_row(uniforms, "uniforms", torch.float32, B, device)
    settings = (_per_row(temp, "temp", torch.float32, B, device), _per_row(top_k, "top_k", torch.int32, B, device),
                _per_row(top_p, "top_p", torch.float32, B, device), _per_row(min_p, "min_p", torch.float32, B, device))
    out = logits.new_empty(B, dtype=torch.int32)
    with _on(device):
        _check(load().illm_sample_rows(logits.data_ptr(), _DT[logits.dtype], B, V, logits.stride(0) if B > 1 else V, u, *settings, out.data_ptr(),
                                       _stream()), "sample_rows")
    return out


def fill_random(out, key: int, std: float, mean: float = 0.0):
    """out[i] = mean + std * z_i, z_i value i of the stream `key` (`weights.random_init.random_key`);
    float32 or bfloat16, in place."""
    _need(out, "out")
    _check(load().illm_fill_random(_ptr(out), act_code(out.dtype), out.numel(), int(key), float(std), float(mean),
                                   _stream()), "fill_random")
    return out


def poison_pages(k, v, pages):
    """Fill the given pages (int32 tensor on the device) of the cache tensors k, v
    [entries, pages, kv heads, page_size, head_dim] with NaN, in every entry."""
    _need(k, "k", None, 5)
    _need(v, "v", k.dtype, 5)
    _need(pages, "pages", torch.int32, 1)
    page_bytes = k.shape[2] * k.shape[3] * k.shape[4] * k.element_size()
    _check(load().illm_poison_pages(_ptr(k), _ptr(v), k.shape[1] * page_bytes, k.shape[0], page_bytes, _ptr(pages),
                                    pages.numel(), _stream()), "poison_pages")


def selftest_wait_timeout(err=None, limit_clocks: int = 1 << 20, code: int = 4):
    """Runs the bounded mbarrier wait of the tensor-core kernels on a barrier nobody arrives at, with
    a short limit.  `err`: the int32 error word to raise (a tensor [1]; default the word of this
    module's own device context; `Engine.info()["tc_error_word"]` is an engine's).  Returns (error word,
    1 if the wait reported its time-out, clocks waited); the word is left set."""
    if err is None:
        err = tc_error_word()
    result = torch.zeros(2, dtype=torch.int64, device=err.device)
    _check(load().illm_selftest_wait_timeout(_ptr(err), _ptr(result), int(limit_clocks), int(code), _stream()),
           "selftest_wait_timeout")
    r = result.tolist()
    return int(err.item()), int(r[0]), int(r[1])

