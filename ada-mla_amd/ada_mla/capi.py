"""ctypes binding of the C ABI in include/mla_mi355x.h (libmla_mi355x.so).

This is the binding a Python caller without the torch extension would add;
the parity tests call the kernels through it. torch is used only for device
memory and the current stream: tensors are passed as raw device pointers.
"""
from __future__ import annotations

import ctypes
import os
import re

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmla_mi355x.so")
HEADER_PATH = os.path.join(os.path.dirname(os.path.dirname(_HERE)), "include", "mla_mi355x.h")

HEAD_DIM_K = 576
HEAD_DIM_V = 512
STATUS_SUCCESS = 0
STATUS_INVALID_VALUE = 1
STATUS_MISALIGNED = 2
STATUS_WORKSPACE_TOO_SMALL = 3
STATUS_HIP_ERROR = 4
STATUS_SCRATCH_EXCEEDED = 5
NOALLOC_SCRATCH_BYTES = 32 << 20
FLAG_SCALAR_TRANSPOSE = 1
FLAG_FP32_PARTIALS = 4
FLAG_FP8_CACHE = 16  # plan queries: the fp8-cache entries' plan
FLAG_TWO_LAUNCHES = 8
FLAG_ROPE_HALVES = 32  # append_kv: pairs i, i + 32

_vp, _i, _u, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_uint, ctypes.c_size_t
_f, _ll = ctypes.c_float, ctypes.c_longlong
_SIGNATURES = {
    "mla_abi_version": (_i, []),
    "mla_status_string": (ctypes.c_char_p, [_i]),
    "mla_last_hip_error": (_i, []),
    "mla_decode_split_num_splits": (_i, [_i, _i, _i, _u]),
    "mla_decode_split_head_tile": (_i, [_i, _i, _i, _u]),
    "mla_decode_split_launches": (_i, [_i, _i, _i, _u]),
    "mla_decode_split_workspace_size": (_sz, [_i, _i, _i]),
    "mla_decode_split_fp16": (_i, [_vp, _vp, _vp, _vp, _sz, _i, _i, _i, _vp]),
    "mla_decode_split_fp16_ex": (_i, [_vp, _vp, _vp, _vp, _sz, _i, _i, _i, _u, _vp]),
    "mla_decode_split_fp16_noalloc": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "mla_decode_split_fp16_partials": (_i, [_vp, _vp, _vp, _sz, _i, _i, _i, _u, _vp]),
    "mla_decode_split_fp16_combine": (_i, [_vp, _sz, _vp, _i, _i, _i, _u, _vp]),
    "mla_decode_fused_workspace_size": (_sz, [_i, _i, _i]),
    "mla_decode_fused_fp32": (_i, [_vp, _vp, _vp, _vp, _sz, _i, _i, _i, _i, _vp]),
    "mla_decode_split_batched_workspace_size": (_sz, [_i, _i, _i, _i]),
    "mla_decode_split_batched_fp16": (_i, [_vp, _vp, _vp, _vp, _vp, _sz, _i, _i, _i, _i, _vp]),
    "mla_decode_split_batched_fp16_partials": (_i, [_vp, _vp, _vp, _vp, _sz, _i, _i, _i, _i, _vp]),
    "mla_decode_split_batched_fp16_combine": (_i, [_vp, _sz, _vp, _vp, _i, _i, _i, _i, _vp]),
    "mla_decode_split_bf16": (_i, [_vp, _vp, _vp, _vp, _sz, _i, _i, _i, _vp]),
    "mla_decode_split_batched_bf16": (_i, [_vp, _vp, _vp, _vp, _vp, _sz, _i, _i, _i, _i, _vp]),
    "mla_decode_paged_workspace_size": (_sz, [_i, _i, _i, _i]),
    "mla_project_output_workspace_size": (_sz, [_i, _i, _i]),
    "mla_decode_split_fp8_workspace_size": (_sz, [_i, _i, _i, _i]),
    "mla_decode_split_fp8": (_i, [_vp, _vp, ctypes.c_float, _vp, _vp, _sz, _i, _i, _i, _vp]),
    "mla_decode_split_batched_fp8": (_i, [_vp, _vp, ctypes.c_float, _vp, _vp, _vp, _sz, _i, _i, _i, _i, _vp]),
    "mla_absorb_query_fp16": (_i, [_vp, _vp, _vp, _vp, _i, _i, _vp]),
    "mla_absorb_query_bf16": (_i, [_vp, _vp, _vp, _vp, _i, _i, _vp]),
    "mla_project_output_fp16": (_i, [_vp, _vp, _vp, _vp, _vp, _sz, _i, _i, _i, _vp]),
    "mla_project_output_bf16": (_i, [_vp, _vp, _vp, _vp, _vp, _sz, _i, _i, _i, _vp]),
    "mla_decode_paged_fp16": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _sz, _i, _i, _i, _i, _i, _i, _i, _vp]),
    "mla_decode_paged_bf16": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _sz, _i, _i, _i, _i, _i, _i, _i, _vp]),
    "mla_decode_paged_fp8_workspace_size": (_sz, [_i, _i, _i, _i]),
    "mla_decode_paged_fp8_fp16": (_i, [_vp, _vp, _f] + [_vp] * 4 + [_sz] + [_i] * 7 + [_vp]),
    "mla_decode_paged_fp8_bf16": (_i, [_vp, _vp, _f] + [_vp] * 4 + [_sz] + [_i] * 7 + [_vp]),
    "mla_paged_tables": (_i, [_vp] * 10 + [_i] * 5 + [_vp]),
    "mla_quantize_fp8_fp16": (_i, [_vp] * 3 + [_i, _i, _ll, _vp]),
    "mla_quantize_fp8_bf16": (_i, [_vp] * 3 + [_i, _i, _ll, _vp]),
    "mla_linear_fp8_workspace_size": (_sz, [_i] * 3),
    "mla_linear_fp8_plan": (_i, [_i] * 4 + [_vp] * 4),
    "mla_linear_fp8_fp16": (_i, [_vp] * 5 + [_sz] + [_i] * 3 + [_ll, _ll, _vp]),
    "mla_linear_fp8_bf16": (_i, [_vp] * 5 + [_sz] + [_i] * 3 + [_ll, _ll, _vp]),
    "mla_linear_fp8_quantized_fp16": (_i, [_vp] * 6 + [_sz] + [_i] * 3 + [_ll] * 4 + [_vp]),
    "mla_linear_fp8_quantized_bf16": (_i, [_vp] * 6 + [_sz] + [_i] * 3 + [_ll] * 4 + [_vp]),
    "mla_page_tables_workspace_size": (_sz, [_i]),
    "mla_fork_tables": (_i, [_vp] * 12 + [_sz] + [_i] * 6 + [_vp]),
    "mla_compact_tables": (_i, [_vp] * 9 + [_sz] + [_i] * 5 + [_vp]),
    "mla_copy_pages": (_i, [_vp, _vp] + [_i] * 5 + [_vp]),
    "mla_append_kv_fp16": (_i, [_vp] * 8 + [_f, _f, _i, _i, _i, _ll, _ll, _ll, _ll, _u, _vp]),
    "mla_append_kv_bf16": (_i, [_vp] * 8 + [_f, _f, _i, _i, _i, _ll, _ll, _ll, _ll, _u, _vp]),
    "mla_decode_tree_workspace_size": (_sz, [_i] * 5),
    "mla_decode_tree_fp16": (_i, [_vp] * 8 + [_sz] + [_i] * 8 + [_vp]),
    "mla_decode_tree_bf16": (_i, [_vp] * 8 + [_sz] + [_i] * 8 + [_vp]),
    "mla_prefill_workspace_size": (_sz, [_i] * 4),
    "mla_prefill_fp16": (_i, [_vp] * 10 + [_sz] + [_i] * 7 + [_vp]),
    "mla_prefill_bf16": (_i, [_vp] * 10 + [_sz] + [_i] * 7 + [_vp]),
}

_lib = None


class MlaError(RuntimeError):
    def __init__(self, fn: str, status: int):
        lib = load()
        msg = lib.mla_status_string(status).decode()
        if status == STATUS_HIP_ERROR:
            msg += f" (hipError_t {lib.mla_last_hip_error()})"
        super().__init__(f"{fn}: {msg}")
        self.status = status


def load():
    """Load libmla_mi355x.so (after torch, so that the library binds to the
    HIP runtime torch already loaded). Raises if the library is not built."""
    global _lib
    if _lib is None:
        import torch  # noqa: F401
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is not built (run python ada-mla_amd/build.py)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            f = getattr(lib, name)
            f.restype = res
            f.argtypes = args
        _lib = lib
    return _lib


def declared_functions() -> list[str]:
    """Function names declared in include/mla_mi355x.h."""
    text = open(HEADER_PATH).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(mla_[a-z0-9_]+)\s*\(", text)))


def _stream(t):
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _check(fn: str, st: int):
    if st != STATUS_SUCCESS:
        raise MlaError(fn, st)


def decode_split_fp16(q, c, num_splits: int = 0, flags: int = 0, out=None):
    """fp16 decode through mla_decode_split_fp16_ex: q [n_h, 576], c [N, 576]."""
    import torch
    lib = load()
    assert q.dtype == torch.float16 and c.dtype == torch.float16
    assert q.is_contiguous() and c.is_contiguous() and q.shape[1] == HEAD_DIM_K and c.shape[1] == HEAD_DIM_K
    n_h, n = q.shape[0], c.shape[0]
    if out is None:
        out = torch.empty((n_h, HEAD_DIM_V), dtype=torch.float16, device=q.device)
    ws_bytes = lib.mla_decode_split_workspace_size(n_h, n, num_splits)
    if ws_bytes == 0:
        raise MlaError("mla_decode_split_workspace_size", STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _check("mla_decode_split_fp16_ex",
           lib.mla_decode_split_fp16_ex(q.data_ptr(), c.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                        ws_bytes, n_h, n, num_splits, flags, _stream(q)))
    return out


def decode_fused_fp32(q, c, num_splits: int = 0, out=None):
    """fp32 decode through mla_decode_fused_fp32."""
    import torch
    lib = load()
    assert q.dtype == torch.float32 and c.dtype == torch.float32
    assert q.is_contiguous() and c.is_contiguous()
    n_h, n = q.shape[0], c.shape[0]
    if out is None:
        out = torch.empty((n_h, HEAD_DIM_V), dtype=torch.float32, device=q.device)
    ws_bytes = lib.mla_decode_fused_workspace_size(n_h, n, num_splits)
    if ws_bytes == 0:
        raise MlaError("mla_decode_fused_workspace_size", STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _check("mla_decode_fused_fp32",
           lib.mla_decode_fused_fp32(q.data_ptr(), c.data_ptr(), out.data_ptr(), ws.data_ptr(), ws_bytes,
                                     n_h, q.shape[1], n, num_splits, _stream(q)))
    return out


def decode_split_bf16(q, c, num_splits: int = 0, out=None):
    """bf16 decode through mla_decode_split_bf16: q [n_h, 576], c [N, 576]."""
    import torch
    lib = load()
    assert q.dtype == torch.bfloat16 and c.dtype == torch.bfloat16
    assert q.is_contiguous() and c.is_contiguous() and q.shape[1] == HEAD_DIM_K and c.shape[1] == HEAD_DIM_K
    n_h, n = q.shape[0], c.shape[0]
    if out is None:
        out = torch.empty((n_h, HEAD_DIM_V), dtype=torch.bfloat16, device=q.device)
    ws_bytes = lib.mla_decode_split_workspace_size(n_h, n, num_splits)
    if ws_bytes == 0:
        raise MlaError("mla_decode_split_workspace_size", STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _check("mla_decode_split_bf16",
           lib.mla_decode_split_bf16(q.data_ptr(), c.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                     ws_bytes, n_h, n, num_splits, _stream(q)))
    return out


def decode_split_batched_bf16(q, c, cu_seqlens, num_splits: int = 0, out=None):
    """Batched bf16 decode (mla_decode_split_batched_bf16); shapes as decode_split_batched_fp16."""
    return _decode_batched(q, c, cu_seqlens, num_splits, out, "mla_decode_split_batched_bf16")


def decode_split_batched_fp16(q, c, cu_seqlens, num_splits: int = 0, out=None):
    """Batched fp16 decode: q [B, n_h, 576], c [sum N, 576], cu_seqlens [B+1] int32 (device)."""
    return _decode_batched(q, c, cu_seqlens, num_splits, out, "mla_decode_split_batched_fp16")


def _decode_batched(q, c, cu_seqlens, num_splits, out, fn):
    import torch
    lib = load()
    dt = torch.bfloat16 if fn.endswith("bf16") else torch.float16
    assert q.dtype == dt and c.dtype == dt and cu_seqlens.dtype == torch.int32
    assert q.is_contiguous() and c.is_contiguous() and cu_seqlens.is_contiguous()
    b, n_h = q.shape[0], q.shape[1]
    total = c.shape[0]
    if out is None:
        out = torch.empty((b, n_h, HEAD_DIM_V), dtype=dt, device=q.device)
    ws_bytes = lib.mla_decode_split_batched_workspace_size(b, n_h, total, num_splits)
    if ws_bytes == 0:
        raise MlaError("mla_decode_split_batched_workspace_size", STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _check(fn, getattr(lib, fn)(q.data_ptr(), c.data_ptr() if total else None, cu_seqlens.data_ptr(),
                                out.data_ptr(), ws.data_ptr(), ws_bytes, b, n_h, total, num_splits,
                                _stream(q)))
    return out


def decode_paged(q, kv_cache, block_table, cu_seqlens, total_tokens: int, num_splits: int = 0, out=None,
                 cache_scale: float = 1.0):
    """Paged-KV decode (mla_decode_paged_fp16 / _bf16 by q's dtype, mla_decode_paged_fp8_* for a
    float8_e4m3fn cache holding C / cache_scale): q [B, n_h, 576],
    kv_cache [num_pages, page_size, 576], block_table [B, max_pages] int32,
    cu_seqlens [B+1] int32 (device), total_tokens = cu_seqlens[B] (host)."""
    import torch
    lib = load()
    fp8 = kv_cache.dtype == torch.float8_e4m3fn
    assert q.dtype in (torch.float16, torch.bfloat16) and (fp8 or (kv_cache.dtype == q.dtype and cache_scale == 1.0))
    assert block_table.dtype == torch.int32 and cu_seqlens.dtype == torch.int32
    assert q.is_contiguous() and kv_cache.is_contiguous() and block_table.is_contiguous()
    b, n_h = q.shape[0], q.shape[1]
    num_pages, page_size = kv_cache.shape[0], kv_cache.shape[1]
    if out is None:
        out = torch.empty((b, n_h, HEAD_DIM_V), dtype=q.dtype, device=q.device)
    size = "mla_decode_paged_fp8_workspace_size" if fp8 else "mla_decode_paged_workspace_size"
    ws_bytes = getattr(lib, size)(b, n_h, total_tokens, num_splits)
    if ws_bytes == 0:
        raise MlaError(size, STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    fn = ("mla_decode_paged_fp8_" if fp8 else "mla_decode_paged_") + _suffix(q)
    scale = (float(cache_scale),) if fp8 else ()
    _check(fn, getattr(lib, fn)(q.data_ptr(), kv_cache.data_ptr(), *scale, block_table.data_ptr(), cu_seqlens.data_ptr(),
                                out.data_ptr(), ws.data_ptr(), ws_bytes, b, n_h, total_tokens, page_size,
                                num_pages, block_table.shape[1], num_splits, _stream(q)))
    return out


def _suffix(t):
    import torch
    return {torch.float16: "fp16", torch.bfloat16: "bf16"}[t.dtype]


def absorb_query(q_nope, q_rope, w_uk, out=None):
    """Q* [B, n_h, 576] = [q_nope W_UK[h], q_rope] (mla_absorb_query_*): q_nope [B, n_h, 128],
    q_rope [B, n_h, 64], w_uk [n_h, 128, 512]."""
    import torch
    lib = load()
    b, n_h = q_nope.shape[0], q_nope.shape[1]
    assert q_nope.shape == (b, n_h, 128) and q_rope.shape == (b, n_h, 64) and w_uk.shape == (n_h, 128, 512)
    assert q_rope.dtype == q_nope.dtype == w_uk.dtype
    assert q_nope.is_contiguous() and q_rope.is_contiguous() and w_uk.is_contiguous()
    if out is None:
        out = torch.empty((b, n_h, HEAD_DIM_K), dtype=q_nope.dtype, device=q_nope.device)
    fn = "mla_absorb_query_" + _suffix(q_nope)
    _check(fn, getattr(lib, fn)(q_nope.data_ptr(), q_rope.data_ptr(), w_uk.data_ptr(), out.data_ptr(), b, n_h,
                                _stream(q_nope)))
    return out


def project_output(o_star, w_uv, w_o, out=None):
    """out [B, d_model] = concat_h(O*[:, h] W_UV[h]^T) W_O^T (mla_project_output_*): o_star
    [B, n_h, 512], w_uv [n_h, 128, 512], w_o [d_model, n_h * 128]."""
    import torch
    lib = load()
    b, n_h = o_star.shape[0], o_star.shape[1]
    d_model = w_o.shape[0]
    assert o_star.shape == (b, n_h, 512) and w_uv.shape == (n_h, 128, 512) and w_o.shape == (d_model, n_h * 128)
    assert o_star.dtype == w_uv.dtype == w_o.dtype
    assert o_star.is_contiguous() and w_uv.is_contiguous() and w_o.is_contiguous()
    if out is None:
        out = torch.empty((b, d_model), dtype=o_star.dtype, device=o_star.device)
    ws_bytes = lib.mla_project_output_workspace_size(b, n_h, d_model)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=o_star.device)
    fn = "mla_project_output_" + _suffix(o_star)
    _check(fn, getattr(lib, fn)(o_star.data_ptr(), w_uv.data_ptr(), w_o.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                ws_bytes, b, n_h, d_model, _stream(o_star)))
    return out


def decode_split_fp8(q, c_fp8, c_scale: float, num_splits: int = 0, out=None):
    """fp8-cache decode (mla_decode_split_fp8): q [n_h, 576] fp16, c_fp8 [N, 576] torch.float8_e4m3fn
    (or uint8 bytes) holding C / c_scale -> [n_h, 512] fp16."""
    import torch
    lib = load()
    assert q.dtype == torch.float16 and c_fp8.element_size() == 1
    assert q.is_contiguous() and c_fp8.is_contiguous() and q.shape[1] == HEAD_DIM_K and c_fp8.shape[1] == HEAD_DIM_K
    n_h, n = q.shape[0], c_fp8.shape[0]
    if out is None:
        out = torch.empty((n_h, HEAD_DIM_V), dtype=torch.float16, device=q.device)
    ws_bytes = lib.mla_decode_split_fp8_workspace_size(1, n_h, n, num_splits)
    if ws_bytes == 0:
        raise MlaError("mla_decode_split_fp8_workspace_size", STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _check("mla_decode_split_fp8", lib.mla_decode_split_fp8(q.data_ptr(), c_fp8.data_ptr(), float(c_scale), out.data_ptr(),
                                                            ws.data_ptr(), ws_bytes, n_h, n, num_splits, _stream(q)))
    return out


def decode_split_batched_fp8(q, c_fp8, c_scale: float, cu_seqlens, num_splits: int = 0, out=None):
    """Batched fp8-cache decode (mla_decode_split_batched_fp8); shapes as decode_split_batched_fp16."""
    import torch
    lib = load()
    assert q.dtype == torch.float16 and c_fp8.element_size() == 1 and cu_seqlens.dtype == torch.int32
    b, n_h, total = q.shape[0], q.shape[1], c_fp8.shape[0]
    if out is None:
        out = torch.empty((b, n_h, HEAD_DIM_V), dtype=torch.float16, device=q.device)
    ws_bytes = lib.mla_decode_split_fp8_workspace_size(b, n_h, total, num_splits)
    if ws_bytes == 0:
        raise MlaError("mla_decode_split_fp8_workspace_size", STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _check("mla_decode_split_batched_fp8",
           lib.mla_decode_split_batched_fp8(q.data_ptr(), c_fp8.data_ptr() if total else None, float(c_scale),
                                            cu_seqlens.data_ptr(), out.data_ptr(), ws.data_ptr(), ws_bytes, b, n_h,
                                            total, num_splits, _stream(q)))
    return out


def _ptr(t):
    return None if t is None else t.data_ptr()


def paged_tables(context_lens, new_lens, block_table, free_pages, free_start, page_size: int, total_new: int):
    """mla_paged_tables: int32 device tensors context_lens, new_lens [B], block_table [B, max_pages] (new
    pages written in place), free_pages [F], free_start [1] -> (cu_seqlens [B+1], cu_new [B+1], slots
    [total_new] int64, positions [total_new], free_next [1])."""
    import torch
    lib = load()
    for t in (context_lens, new_lens, block_table, free_pages, free_start):
        assert t.dtype == torch.int32 and t.is_contiguous()
    b = context_lens.shape[0]
    i32 = dict(dtype=torch.int32, device=context_lens.device)
    cu_seqlens, cu_new = torch.empty(b + 1, **i32), torch.empty(b + 1, **i32)
    slots = torch.empty(total_new, dtype=torch.int64, device=context_lens.device)
    positions, free_next = torch.empty(total_new, **i32), torch.empty(1, **i32)
    _check("mla_paged_tables",
           lib.mla_paged_tables(_ptr(context_lens), _ptr(new_lens), _ptr(free_pages), _ptr(free_start),
                                _ptr(block_table), _ptr(cu_seqlens), _ptr(cu_new), _ptr(slots), _ptr(positions),
                                _ptr(free_next), b, total_new, free_pages.shape[0], page_size, block_table.shape[1],
                                _stream(context_lens)))
    return cu_seqlens, cu_new, slots, positions, free_next


def fork_tables(block_table, lens, parents, free_pages, free_start, page_size: int, num_pages: int, kept_lens=None,
                pinned=None, workspace=None):
    """mla_fork_tables: int32 device tensors block_table [R, max_pages], lens [R], parents [B], free_pages [F]
    (written in place), free_start [1], kept_lens [B] or None, pinned [num_pages] or None -> (block_table
    [B, max_pages], lens [B], copies [B, 3], free_next [1])."""
    import torch
    lib = load()
    for t in (block_table, lens, parents, free_pages, free_start, kept_lens, pinned):
        assert t is None or (t.dtype == torch.int32 and t.is_contiguous())
    (rows, width), b = block_table.shape, parents.shape[0]
    assert lens.shape == (rows,) and free_start.shape == (1,) and (kept_lens is None or kept_lens.shape == (b,))
    assert pinned is None or pinned.shape == (num_pages,)
    i32 = dict(dtype=torch.int32, device=block_table.device)
    table, new_lens, copies, nxt = (torch.empty(s, **i32) for s in ((b, width), (b,), (b, 3), (1,)))
    ws_bytes = lib.mla_page_tables_workspace_size(num_pages)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=block_table.device) if workspace is None else workspace
    _check("mla_fork_tables",
           lib.mla_fork_tables(_ptr(block_table), _ptr(lens), _ptr(parents), _ptr(kept_lens), _ptr(pinned),
                               _ptr(free_pages), _ptr(free_start), _ptr(table), _ptr(new_lens), _ptr(copies), _ptr(nxt),
                               _ptr(ws), ws.numel(), rows, b, num_pages, free_pages.shape[0], page_size, width,
                               _stream(block_table)))
    return table, new_lens, copies, nxt


def compact_tables(block_table, lens, free_pages, free_start, page_size: int, num_pages: int, pinned=None,
                   workspace=None):
    """mla_compact_tables: int32 device tensors as for fork_tables -> (block_table, copies [min(F, num_pages // 2), 3],
    free_pages)."""
    import torch
    lib = load()
    for t in (block_table, lens, free_pages, free_start, pinned):
        assert t is None or (t.dtype == torch.int32 and t.is_contiguous())
    rows, width = block_table.shape
    assert lens.shape == (rows,) and free_start.shape == (1,) and (pinned is None or pinned.shape == (num_pages,))
    table, new_free = torch.empty_like(block_table), torch.empty_like(free_pages)
    copies = torch.empty((min(free_pages.shape[0], num_pages // 2), 3), dtype=torch.int32, device=block_table.device)
    ws_bytes = lib.mla_page_tables_workspace_size(num_pages)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=block_table.device) if workspace is None else workspace
    _check("mla_compact_tables",
           lib.mla_compact_tables(_ptr(block_table), _ptr(lens), _ptr(pinned), _ptr(free_pages), _ptr(free_start),
                                  _ptr(table), _ptr(copies), _ptr(new_free), _ptr(ws), ws.numel(), rows, num_pages,
                                  free_pages.shape[0], page_size, width, _stream(block_table)))
    return table, copies, new_free


def copy_pages(kv_cache, copies):
    """mla_copy_pages: kv_cache [num_pages, page_size, 576] or [layers, num_pages, page_size, 576], written in place;
    copies [n, 3] int32 (page, page, rows)."""
    import torch
    lib = load()
    assert kv_cache.is_contiguous() and kv_cache.shape[-1] == HEAD_DIM_K and kv_cache.dim() in (3, 4)
    assert copies.dtype == torch.int32 and copies.is_contiguous() and copies.shape[1] == 3
    layers = kv_cache.shape[0] if kv_cache.dim() == 4 else 1
    _check("mla_copy_pages", lib.mla_copy_pages(_ptr(kv_cache), _ptr(copies), copies.shape[0], layers, kv_cache.shape[-3],
                                                kv_cache.shape[-2], kv_cache.element_size(), _stream(kv_cache)))


def quantize_fp8(x):
    """mla_quantize_fp8_*: x [M, K] (last dimension contiguous) -> (float8_e4m3fn [M, K], scales [M, ceil(K / 128)],
    a view of what the call writes block by block)."""
    import torch
    lib = load()
    m, k = x.shape
    assert x.stride(1) == 1
    q = torch.empty((m, k), dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((-(-k // 128), m), dtype=torch.float32, device=x.device)
    fn = "mla_quantize_fp8_" + _suffix(x)
    _check(fn, getattr(lib, fn)(_ptr(x), _ptr(q), _ptr(scales), m, k, x.stride(0), _stream(x)))
    return q, scales.t()


def linear_fp8_plan(rows: int, inputs: int, outputs: int, quantized: bool = False):
    """mla_linear_fp8_plan -> (outputs and rows of a workgroup's tile, splits of the inputs, launches)."""
    out = [ctypes.c_int() for _ in range(4)]
    _check("mla_linear_fp8_plan", load().mla_linear_fp8_plan(rows, inputs, outputs, int(quantized), *map(ctypes.byref, out)))
    return tuple(v.value for v in out)


def linear_fp8(x, w, w_scale, x_scale=None, dtype=None, out=None, workspace=None):
    """mla_linear_fp8_*: x [M, K] 16-bit, or float8_e4m3fn with x_scale [M, ceil(K / 128)]; w [N, K] float8_e4m3fn with
    w_scale [ceil(N / 128), ceil(K / 128)] -> [M, N]."""
    import torch
    lib = load()
    (m, k), n = x.shape, w.shape[0]
    assert w.shape == (n, k) and x.stride(1) == 1 and w.stride(1) == 1 and w_scale.is_contiguous()
    assert w_scale.shape == (-(-n // 128), -(-k // 128)) and w_scale.dtype == torch.float32
    if out is None:
        out = torch.empty((m, n), dtype=x.dtype if x_scale is None else dtype or torch.bfloat16, device=x.device)
    ws_bytes = lib.mla_linear_fp8_workspace_size(m, k, n)
    if ws_bytes == 0:
        raise MlaError("mla_linear_fp8_workspace_size", STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if workspace is None else workspace
    if x_scale is None:
        fn, scale, strides = "mla_linear_fp8_" + _suffix(x), (), ()
    else:
        assert x_scale.shape == (m, -(-k // 128)) and x_scale.dtype == torch.float32
        fn, scale, strides = "mla_linear_fp8_quantized_" + _suffix(out), (_ptr(x_scale),), x_scale.stride()
    _check(fn, getattr(lib, fn)(_ptr(x), *scale, _ptr(w), _ptr(w_scale), _ptr(out), _ptr(ws), ws.numel(), m, k, n,
                                x.stride(0), w.stride(0), *strides, _stream(x)))
    return out


def append_kv(kv, norm_weight, cos_sin, positions, slots, kv_cache, q_rope=None, eps: float = 1e-6,
              cache_scale: float = 1.0, interleaved: bool = True, out=None):
    """mla_append_kv_*: kv [T, 576] and q_rope [T, n_h, 64] (last dimension contiguous, other strides
    multiples of 8), kv_cache [..., 576] contiguous, of kv's type or float8_e4m3fn -> rotated q_rope or None."""
    import torch
    lib = load()
    tokens = kv.shape[0]
    assert kv.shape == (tokens, HEAD_DIM_K) and kv.stride(1) == 1 and kv_cache.is_contiguous()
    assert norm_weight.dtype == kv.dtype and cos_sin.dtype == torch.float32 and cos_sin.shape[1] == 64
    assert positions.dtype == torch.int32 and slots.dtype == torch.int64
    n_h = 0 if q_rope is None else q_rope.shape[1]
    if q_rope is not None:
        assert q_rope.dtype == kv.dtype and q_rope.stride(2) == 1 and q_rope.shape == (tokens, n_h, 64)
        if out is None:
            out = torch.empty((tokens, n_h, 64), dtype=kv.dtype, device=kv.device)
    flags = (FLAG_FP8_CACHE if kv_cache.dtype == torch.float8_e4m3fn else 0) | (0 if interleaved else FLAG_ROPE_HALVES)
    fn = "mla_append_kv_" + _suffix(kv)
    _check(fn, getattr(lib, fn)(_ptr(kv), _ptr(norm_weight), _ptr(cos_sin), _ptr(positions), _ptr(slots), _ptr(q_rope),
                                _ptr(kv_cache), _ptr(out), eps, cache_scale, tokens, n_h, cos_sin.shape[0],
                                kv_cache.numel() // HEAD_DIM_K, kv.stride(0), q_rope.stride(0) if n_h else 0,
                                q_rope.stride(1) if n_h else 0, flags, _stream(kv)))
    return out


def decode_tree(q, kv_cache, block_table, cu_seqlens, tree_mask, total_tokens: int, draft_lens=None,
                num_splits: int = 0, out=None, workspace=None):
    """mla_decode_tree_*: q [B, drafts, n_h, 576], kv_cache [num_pages, page_size, 576], block_table
    [B, max_pages] int32, cu_seqlens [B+1] int32, tree_mask [B, drafts] int64, draft_lens [B] int32 or None."""
    import torch
    lib = load()
    b, drafts, n_h, _ = q.shape
    assert kv_cache.dtype == q.dtype and block_table.dtype == torch.int32 and cu_seqlens.dtype == torch.int32
    assert tree_mask.dtype == torch.int64 and tree_mask.shape == (b, drafts)
    assert q.is_contiguous() and kv_cache.is_contiguous() and block_table.is_contiguous() and tree_mask.is_contiguous()
    if out is None:
        out = torch.empty((b, drafts, n_h, HEAD_DIM_V), dtype=q.dtype, device=q.device)
    ws_bytes = lib.mla_decode_tree_workspace_size(b, drafts, n_h, total_tokens, num_splits)
    if ws_bytes == 0:
        raise MlaError("mla_decode_tree_workspace_size", STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if workspace is None else workspace
    fn = "mla_decode_tree_" + _suffix(q)
    _check(fn, getattr(lib, fn)(_ptr(q), _ptr(kv_cache), _ptr(block_table), _ptr(cu_seqlens), _ptr(tree_mask),
                                _ptr(draft_lens), _ptr(out), _ptr(ws), ws.numel(), b, drafts, n_h, total_tokens,
                                kv_cache.shape[1], kv_cache.shape[0], block_table.shape[1], num_splits, _stream(q)))
    return out


def prefill(q_nope, q_rope, w_uk, w_uv, kv_cache, cu_q, cu_seqlens, total_tokens: int, block_table=None, out=None,
            workspace=None):
    """mla_prefill_*: q_nope [T, n_h, 128], q_rope [T, n_h, 64], w_uk / w_uv [n_h, 128, 512], kv_cache
    [total_tokens, 576] or, with block_table [B, max_pages] int32, [num_pages, page_size, 576]."""
    import torch
    lib = load()
    queries, n_h, _ = q_nope.shape
    b = cu_q.shape[0] - 1
    assert q_nope.dtype == q_rope.dtype == w_uk.dtype == w_uv.dtype == kv_cache.dtype
    for t in (q_nope, q_rope, w_uk, w_uv, kv_cache, cu_q, cu_seqlens):
        assert t.is_contiguous()
    if out is None:
        out = torch.empty((queries, n_h, 128), dtype=q_nope.dtype, device=q_nope.device)
    ws_bytes = lib.mla_prefill_workspace_size(b, n_h, queries, total_tokens)
    if ws_bytes == 0:
        raise MlaError("mla_prefill_workspace_size", STATUS_INVALID_VALUE)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q_nope.device) if workspace is None else workspace
    paged = block_table is not None
    fn = "mla_prefill_" + _suffix(q_nope)
    _check(fn, getattr(lib, fn)(_ptr(q_nope), _ptr(q_rope), _ptr(w_uk), _ptr(w_uv), _ptr(kv_cache), _ptr(block_table),
                                _ptr(cu_q), _ptr(cu_seqlens), _ptr(out), _ptr(ws), ws.numel(), b, n_h, queries,
                                total_tokens, kv_cache.shape[1] if paged else 0, kv_cache.shape[0] if paged else 0,
                                block_table.shape[1] if paged else 0, _stream(q_nope)))
    return out
