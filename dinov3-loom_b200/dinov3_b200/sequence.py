"""Attention over packed sequences and over a paged key-value cache, on CUDA tensors: the Python
face of dv3k_attention_packed, dv3k_rope_append and dv3k_attention_paged
(include/dinov3_kernels.h), whose text has the formulas and the rules on strides.

    q, k, v = ...                                    # [rows, heads, dim], float16 or bfloat16
    out = attention_packed(q, k, v, cu)              # sequences packed one behind the other
    q = rope_append(q, k, v, k_cache, v_cache, page_table, lens, cos, sin, cu_new=cu)
    out = attention_paged(q, k_cache, v_cache, page_table, lens)   # one new token per sequence

The calls are asynchronous on torch's current stream of the tensors' device (which need not be the
current device), can be captured into a CUDA graph, and allocate only what they return (and the
attentions their scratch, unless it is given) through torch's allocator. They compute no
gradients: a tensor that wants one, or carries a forward-mode tangent, is refused. What does not fit raises DINOv3Error
(INVALID_ARGUMENT) before anything is launched, outputs that share memory with another tensor among
it. `status` is an optional int32 CUDA tensor of two words, cleared and read by the caller, that collects
what only the device sees: bad pages and positions, and a launch that gave up a wait and left its
outputs incomplete. Without it nothing tells of these.
"""
from __future__ import annotations

import ctypes

import torch  # noqa: F401  (its libraries, before the binding that is linked against them)

from . import INVALID_ARGUMENT, DINOv3Error, _check, _lib

try:
    from . import _sequence
except ImportError as e:
    raise _lib.LibraryMissing(f"the tensor binding is not built; run `python dinov3-loom_b200/build.py` ({e})") from e


def _refuse(message: str):
    raise DINOv3Error(INVALID_ARGUMENT, message)


_names = ("dv3k_attention_packed", "dv3k_attention_packed_workspace", "dv3k_rope_append", "dv3k_attention_paged",
          "dv3k_attention_paged_workspace")
_sequence.bind(*(ctypes.cast(getattr(_lib.load(), n), ctypes.c_void_p).value for n in _names), _refuse, _check)


def attention_packed(q, k, v, cu_q, cu_k=None, *, causal=False, scale=None, out=None, lse=None, workspace=None, status=None):
    """Attention of packed sequences (dv3k_attention_packed) -> out [total_q, q_heads, dim].

    q [total_q, q_heads, dim]; k, v [total_k, kv_heads, dim]; cu_q, cu_k int32 [n_seq + 1] (cu_k None:
    cu_q). scale defaults to dim ** -0.5. `out` may be given; rows outside the sequences are left as
    they were (in a new one: whatever the memory held). `lse`, float32 [total_q, q_heads], is filled where given. `workspace`: a uint8 tensor of
    attention_packed_workspace(dim) bytes to use instead of a new one."""
    return _sequence.attention_packed(q, k, v, cu_q, cu_k, causal, scale, out, lse, workspace, status)


def attention_packed_workspace(dim, device=None) -> int:
    """Bytes of a workspace that every attention_packed with that head dim can use on the device (None:
    the current one). Calls that may overlap on the GPU (two streams, two graphs) need one each."""
    with torch.cuda.device(device):
        return _size(_lib.load().dv3k_attention_packed_workspace_bound(dim), "no call has head dim", dim)


def attention_paged_workspace(n_seq, q_heads, kv_heads, dim, device=None) -> int:
    """Bytes of a workspace that every attention_paged with these heads and up to n_seq sequences of any
    length can use on the device (None: the current one). Calls that may overlap need one each."""
    with torch.cuda.device(device):
        return _size(_lib.load().dv3k_attention_paged_workspace_bound(n_seq, q_heads, kv_heads, dim), "no call has n_seq, q_heads, kv_heads, dim",
                     n_seq, q_heads, kv_heads, dim)


def _size(n, refusal, *what):
    if n == 0:
        _refuse(f"{refusal} {', '.join(map(str, what))}")
    return n


def rope_append(q, k, v, k_cache, v_cache, page_table, lens, cos=None, sin=None, *, cu_new=None, q_out=None, status=None):
    """Rotate q and k by their positions and append k and v to the cache (dv3k_rope_append)
    -> the rotated q [total, q_heads, dim] (None where q is None).

    k, v [total, kv_heads, dim]; caches [pages, kv_heads, page_size, dim]; page_table int32 [n_seq,
    max_pages]; lens int32 [n_seq], the lengths with the new rows; cu_new int32 [n_seq + 1], or None
    for one row per sequence; cos, sin float32 [positions, rot_dim / 2], or None for no rotation.
    `q_out` may be q itself; rows outside the sequences are left as they were."""
    return _sequence.rope_append(q, k, v, k_cache, v_cache, page_table, lens, cos, sin, cu_new, q_out, status)


def attention_paged(q, k_cache, v_cache, page_table, lens, *, max_len=None, scale=None, out=None, lse=None, workspace=None, status=None):
    """Attention of one new token per sequence over the paged cache (dv3k_attention_paged)
    -> out [n_seq, q_heads, dim].

    q [n_seq, q_heads, dim]; caches [pages, kv_heads, page_size, dim]; page_table int32 [n_seq,
    max_pages]; lens int32 [n_seq]. max_len bounds lens (default: what page_table holds) and decides
    how far sequences are split. `lse`, float32 [n_seq, q_heads], is filled where given. `workspace`:
    a uint8 tensor of attention_paged_workspace(...) bytes to use instead of a new one."""
    return _sequence.attention_paged(q, k_cache, v_cache, page_table, lens, max_len, scale, out, lse, workspace, status)
