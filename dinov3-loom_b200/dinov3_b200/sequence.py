"""Attention over packed sequences and over a paged key-value cache, on CUDA tensors: the Python
face of dv3k_attention_packed, dv3k_rope_append and dv3k_attention_paged
(include/dinov3_kernels.h), whose text has the formulas and the rules on strides.

    q, k, v = ...                                    # [rows, heads, dim], float16 or bfloat16
    out = attention_packed(q, k, v, cu)              # sequences packed one behind the other
    q = rope_append(q, k, v, k_cache, v_cache, page_table, lens, cos, sin, cu_new=cu)
    out = attention_paged(q, k_cache, v_cache, page_table, lens)   # one new token per sequence

The calls are asynchronous on torch's current stream of the tensors' device, can be captured into a
CUDA graph, and allocate only what they return (and attention_paged its scratch, unless it is
given) through torch's allocator. They compute no gradients: a tensor that wants one is refused.
`status` is an optional int32 CUDA tensor of two words, cleared and read by the caller, that
collects what only the device sees (bad pages and positions).
"""
from __future__ import annotations

import struct

import torch

from . import _lib

# The argument structs of dinov3_kernels.h: pointers and 8-byte integers first, then 4-byte ones.
_PACKED = struct.Struct("8Q8q8IfI")
_APPEND = struct.Struct("12Q11q12I")
_PAGED = struct.Struct("9Q7qQ9If")

_TYPES = {torch.float16: 0, torch.bfloat16: 1}


def _refuse(message: str):
    from . import INVALID_ARGUMENT, DINOv3Error

    raise DINOv3Error(INVALID_ARGUMENT, message)


def _check_rows(name, t, like):
    """A tensor [rows, heads, dim] of the call's type on its device."""
    if t.dtype != like.dtype or t.device != like.device:
        _refuse(f"{name} must have the type and device of q: {t.dtype} on {t.device}")
    if t.dim() != 3 or t.stride(2) != 1 and t.shape[2] > 1:
        _refuse(f"{name} must be [rows, heads, dim] with a contiguous dim: {tuple(t.shape)}, strides {t.stride()}")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} requires a gradient, which this operator does not compute")


def _check_ints(name, t, like, dims):
    if t.dtype != torch.int32 or t.device != like.device or t.dim() != dims:
        _refuse(f"{name} must be int32 with {dims} dimension(s) on {like.device}: {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        _refuse(f"{name} must be contiguous")


def _check_first(q):
    if q.dtype not in _TYPES or not q.is_cuda:
        _refuse(f"expected a float16 or bfloat16 CUDA tensor, got {q.dtype} on {q.device}")


def _check_cache(k_cache, v_cache, like, kv_heads, dim):
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dtype != like.dtype or t.device != like.device:
            _refuse(f"{name} must have the type and device of the rows: {t.dtype} on {t.device}")
        if t.dim() != 4 or t.shape[1] != kv_heads or t.shape[3] != dim or t.shape != k_cache.shape:
            _refuse(f"{name} must be [pages, {kv_heads}, page_size, {dim}]: {tuple(t.shape)}")
        if t.stride()[1:] != (t.shape[2] * dim, dim, 1) and t.numel() and not t[0].is_contiguous():
            _refuse(f"{name} must be contiguous within a page")
        if t.requires_grad and torch.is_grad_enabled():
            _refuse(f"{name} requires a gradient, which this operator does not compute")


def _optional(name, t, like, dtype, shape):
    """Address of an optional contiguous tensor, 0 for None."""
    if t is None:
        return 0
    if t.dtype != dtype or t.device != like.device or not t.is_contiguous() or (shape and tuple(t.shape) != shape):
        _refuse(f"{name} must be a contiguous {dtype} tensor of shape {shape or 'any'} on {like.device}")
    return t.data_ptr()


def _status(t, like):
    if t is None:
        return 0
    if t.numel() < 2:
        _refuse("status must hold two words")
    return _optional("status", t, like, torch.int32, None)


def _output(name, out, like, shape):
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    _check_rows(name, out, like)
    if tuple(out.shape) != tuple(shape):
        _refuse(f"{name} must have shape {tuple(shape)}: {tuple(out.shape)}")
    return out


def _launch(function, args, device):
    """Call on the current stream of `device`, made current for the call where it is not."""
    if torch.cuda.current_device() == device.index:
        rc = function(args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = function(args, torch.cuda.current_stream().cuda_stream)
    if rc:
        from . import _check

        _check(rc)


def attention_packed(q, k, v, cu_q, cu_k=None, *, causal=False, scale=None, out=None, lse=None, status=None):
    """Attention of packed sequences (dv3k_attention_packed) -> out [total_q, q_heads, dim].

    q [total_q, q_heads, dim]; k, v [total_k, kv_heads, dim]; cu_q, cu_k int32 [n_seq + 1] (cu_k None:
    cu_q). scale defaults to dim ** -0.5. `out` may be given; rows outside the sequences are left as
    they were. `lse`, float32 [total_q, q_heads], is filled where given."""
    _check_first(q)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_rows(name, t, q)
    if cu_k is None:
        cu_k = cu_q
    _check_ints("cu_q", cu_q, q, 1)
    _check_ints("cu_k", cu_k, q, 1)
    total_q, q_heads, dim = q.shape
    total_k, kv_heads, _ = k.shape
    if k.shape[2] != dim or v.shape != k.shape:
        _refuse(f"k and v must be [rows, kv_heads, {dim}] alike: {tuple(k.shape)}, {tuple(v.shape)}")
    n_seq = cu_q.shape[0] - 1
    if n_seq < 0 or cu_k.shape[0] != n_seq + 1:
        _refuse("cu_q and cu_k must have the same n_seq + 1 entries")
    out = _output("out", out, q, q.shape)
    args = _PACKED.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _optional("lse", lse, q, torch.float32, (total_q, q_heads)),
        cu_q.data_ptr(), cu_k.data_ptr(), _status(status, q),
        q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), out.stride(0), out.stride(1),
        n_seq, total_q, total_k, q_heads, kv_heads, dim, _TYPES[q.dtype], 1 if causal else 0,
        dim ** -0.5 if scale is None else scale, 0)
    _launch(_lib.load().dv3k_attention_packed, args, q.device)
    return out


def rope_append(q, k, v, k_cache, v_cache, page_table, lens, cos=None, sin=None, *, cu_new=None, q_out=None, status=None):
    """Rotate q and k by their positions and append k and v to the cache (dv3k_rope_append)
    -> the rotated q [total, q_heads, dim] (None where q is None).

    k, v [total, kv_heads, dim]; caches [pages, kv_heads, page_size, dim]; page_table int32 [n_seq,
    max_pages]; lens int32 [n_seq], the lengths with the new rows; cu_new int32 [n_seq + 1], or None
    for one row per sequence; cos, sin float32 [positions, rot_dim / 2], or None for no rotation.
    `q_out` may be q itself."""
    _check_first(k)
    for name, t in (("k", k), ("v", v)):
        _check_rows(name, t, k)
    total, kv_heads, dim = k.shape
    if v.shape != k.shape:
        _refuse(f"k and v must have the same shape: {tuple(k.shape)}, {tuple(v.shape)}")
    _check_cache(k_cache, v_cache, k, kv_heads, dim)
    _check_ints("page_table", page_table, k, 2)
    _check_ints("lens", lens, k, 1)
    n_seq, max_pages = page_table.shape
    if lens.shape[0] != n_seq:
        _refuse("lens must have one entry for each row of page_table")
    if cu_new is not None:
        _check_ints("cu_new", cu_new, k, 1)
        if cu_new.shape[0] != n_seq + 1:
            _refuse("cu_new must have n_seq + 1 entries")
    if (cos is None) != (sin is None):
        _refuse("cos and sin go together")
    positions = rot_dim = 0
    if cos is not None:
        if cos.dim() != 2:
            _refuse("cos must be [positions, rot_dim / 2]")
        positions, rot_dim = cos.shape[0], 2 * cos.shape[1]
    if q is None:
        q_heads, q_args, q_strides = 0, (0, 0), (0, 0, 0, 0)
    else:
        _check_rows("q", q, k)
        if q.shape[0] != total or q.shape[2] != dim:
            _refuse(f"q must be [{total}, q_heads, {dim}]: {tuple(q.shape)}")
        q_heads = q.shape[1]
        q_out = _output("q_out", q_out, q, q.shape)
        q_args = (q.data_ptr(), q_out.data_ptr())
        q_strides = (q.stride(0), q.stride(1), q_out.stride(0), q_out.stride(1))
    args = _APPEND.pack(
        q_args[0], k.data_ptr(), v.data_ptr(), q_args[1], k_cache.data_ptr(), v_cache.data_ptr(),
        0 if cu_new is None else cu_new.data_ptr(), lens.data_ptr(), page_table.data_ptr(),
        _optional("cos", cos, k, torch.float32, None), _optional("sin", sin, k, torch.float32, None if cos is None else tuple(cos.shape)),
        _status(status, k),
        q_strides[0], q_strides[1], k.stride(0), k.stride(1), v.stride(0), v.stride(1), q_strides[2], q_strides[3],
        k_cache.stride(0), v_cache.stride(0), page_table.stride(0),
        n_seq, total, max_pages, k_cache.shape[0], k_cache.shape[2], positions, rot_dim, q_heads, kv_heads, dim, _TYPES[k.dtype], 0)
    _launch(_lib.load().dv3k_rope_append, args, k.device)
    return q_out if q is not None else None


def attention_paged(q, k_cache, v_cache, page_table, lens, *, max_len=None, scale=None, out=None, lse=None, workspace=None, status=None):
    """Attention of one new token per sequence over the paged cache (dv3k_attention_paged)
    -> out [n_seq, q_heads, dim].

    q [n_seq, q_heads, dim]; caches [pages, kv_heads, page_size, dim]; page_table int32 [n_seq,
    max_pages]; lens int32 [n_seq]. max_len bounds lens (default: what page_table holds) and decides
    how far sequences are split. `lse`, float32 [n_seq, q_heads], is filled where given. `workspace`:
    a byte tensor of attention_paged_workspace's size to use instead of a new one."""
    _check_first(q)
    _check_rows("q", q, q)
    n_seq, q_heads, dim = q.shape
    kv_heads = k_cache.shape[1] if k_cache.dim() == 4 else 0
    _check_cache(k_cache, v_cache, q, kv_heads, dim)
    _check_ints("page_table", page_table, q, 2)
    _check_ints("lens", lens, q, 1)
    max_pages, page_size = page_table.shape[1], k_cache.shape[2]
    if page_table.shape[0] != n_seq or lens.shape[0] != n_seq:
        _refuse("page_table and lens must have one entry for each row of q")
    room = max_pages * page_size
    if max_len is None or max_len > room:
        max_len = room
    elif max_len < 0:
        _refuse("max_len must not be negative")
    out = _output("out", out, q, q.shape)
    lse_at = _optional("lse", lse, q, torch.float32, (n_seq, q_heads))

    def pack(at, size):
        return _PAGED.pack(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), lse_at, lens.data_ptr(), page_table.data_ptr(), at,
            _status(status, q),
            q.stride(0), q.stride(1), out.stride(0), out.stride(1), k_cache.stride(0), v_cache.stride(0), page_table.stride(0),
            size, n_seq, max_len, max_pages, k_cache.shape[0], page_size, q_heads, kv_heads, dim, _TYPES[q.dtype],
            dim ** -0.5 if scale is None else scale)

    lib = _lib.load()
    if workspace is None:
        need = lib.dv3k_attention_paged_workspace(pack(0, 0))
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    at = _optional("workspace", workspace, q, torch.uint8, None)
    _launch(lib.dv3k_attention_paged, pack(at, workspace.numel() if at else 0), q.device)
    return out
