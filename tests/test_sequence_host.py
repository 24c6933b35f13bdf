"""Argument checks of the packed and paged entry points, which launch nothing and need no GPU."""
import ctypes
import os
import struct
import subprocess

import pytest

import dinov3_b200 as dv
from dinov3_b200 import _lib

from conftest import ROOT

BUF = ctypes.create_string_buffer(4096)
BASE = (ctypes.addressof(BUF) + 63) & ~63

# The argument structs of dinov3_kernels.h: pointers and 8-byte integers first, then 4-byte ones.
PACKED_STRUCT, APPEND_STRUCT, PAGED_STRUCT = struct.Struct("9Q8qQ8IfI"), struct.Struct("12Q11q12I"), struct.Struct("9Q7qQ9If")

PACKED = ["q", "k", "v", "out", "lse", "cu_q", "cu_k", "workspace", "status", "q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "out_token",
          "out_head", "workspace_bytes", "n_seq", "total_q", "total_k", "q_heads", "kv_heads", "head_dim", "dtype", "causal", "scale", "reserved"]
APPEND = ["q", "k", "v", "q_out", "k_cache", "v_cache", "cu_new", "lens", "page_table", "cos", "sin", "status", "q_token", "q_head", "k_token",
          "k_head", "v_token", "v_head", "q_out_token", "q_out_head", "k_page", "v_page", "table_stride", "n_seq", "total", "max_pages", "n_pages",
          "page_size", "positions", "rot_dim", "q_heads", "kv_heads", "head_dim", "dtype", "reserved"]
PAGED = ["q", "k_cache", "v_cache", "out", "lse", "lens", "page_table", "workspace", "status", "q_seq", "q_head", "out_seq", "out_head", "k_page",
         "v_page", "table_stride", "workspace_bytes", "n_seq", "max_len", "max_pages", "n_pages", "page_size", "q_heads", "kv_heads", "head_dim",
         "dtype", "scale"]

packed_ok = dict(dict.fromkeys(PACKED, 0), q=BASE, k=BASE, v=BASE, out=BASE, cu_q=BASE, cu_k=BASE, q_token=256, q_head=64, k_token=256, k_head=64,
                 v_token=256, v_head=64, out_token=256, out_head=64, n_seq=1, total_q=4, total_k=4, q_heads=4, kv_heads=2, head_dim=64, scale=0.125)
append_ok = dict(dict.fromkeys(APPEND, 0), q=BASE, k=BASE, v=BASE, q_out=BASE, k_cache=BASE, v_cache=BASE, cu_new=BASE, lens=BASE, page_table=BASE,
                 cos=BASE, sin=BASE, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, q_out_token=256, q_out_head=64,
                 k_page=2048, v_page=2048, table_stride=4, n_seq=2, total=4, max_pages=4, n_pages=8, page_size=16, positions=64, rot_dim=64, q_heads=4,
                 kv_heads=2, head_dim=64)
paged_ok = dict(dict.fromkeys(PAGED, 0), q=BASE, k_cache=BASE, v_cache=BASE, out=BASE, lens=BASE, page_table=BASE, q_seq=256, q_head=64, out_seq=256,
                out_head=64, k_page=2048, v_page=2048, table_stride=4, n_seq=2, max_len=64, max_pages=4, n_pages=8, page_size=16, q_heads=4,
                kv_heads=2, head_dim=64, scale=0.125)


def call(name, pack, fields, values):
    rc = getattr(_lib.load(), name)(pack.pack(*(values[f] for f in fields)), None)
    return rc, _lib.last_error()


def refused(name, pack, fields, ok, text, **changes):
    rc, message = call(name, pack, fields, dict(ok, **changes))
    assert rc == dv.INVALID_ARGUMENT and text in message, (changes, message)


HEADS = [("dtype", dict(dtype=2)), ("head_dim", dict(head_dim=80)), ("kv_heads", dict(kv_heads=0)), ("multiple", dict(q_heads=5)),
         ("multiple", dict(q_heads=258))]


@pytest.mark.parametrize("text,changes", HEADS + [
    ("q_heads", dict(q_heads=0)), ("causal", dict(causal=2)), ("reserved", dict(reserved=1)), ("scale", dict(scale=0.0)), ("scale", dict(scale=-1.0)),
    ("scale", dict(scale=float("nan"))), ("scale", dict(scale=float("inf"))), ("strides", dict(q_token=0)), ("strides", dict(k_head=4)),
    ("strides", dict(v_token=-128)), ("strides", dict(out_head=1 << 40)), ("overlap", dict(out_token=64)), ("overlap", dict(out_head=8)),
    ("overlap", dict(out_token=128, out_head=200)), ("null", dict(q=0)), ("null", dict(cu_k=0)), ("null", dict(v=0)), ("aligned", dict(k=BASE + 2)),
    ("aligned", dict(out=BASE + 8)), ("too many", dict(total_q=1 << 31)),
    ("workspace", dict(total_k=4096)), ("workspace", dict(total_k=4096, workspace=BASE, workspace_bytes=1000)), ("aligned", dict(workspace=BASE + 8)),
    ("4-byte", dict(lse=BASE + 2)), ("4-byte", dict(cu_q=BASE + 1)), ("4-byte", dict(status=BASE + 2)), ("out overlaps", dict(out=BASE)),
    ("out overlaps", dict(q=BASE + 1024, k=BASE + 2048)),
])
def test_packed_refusals(text, changes):
    refused("dv3k_attention_packed", PACKED_STRUCT, PACKED, packed_ok, text, **changes)


CACHE = [("page_size", dict(page_size=0)), ("page_size", dict(page_size=1 << 17)), ("2^31", dict(max_pages=1 << 30)), ("n_pages", dict(n_pages=1 << 31)),
         ("cache", dict(k_cache=0)), ("overlap", dict(v_page=2040)), ("overlap", dict(k_page=2052)), ("page_table", dict(page_table=0)),
         ("page_table", dict(page_table=BASE + 2)), ("table_stride", dict(table_stride=3)), ("aligned", dict(v_cache=BASE + 4))]


@pytest.mark.parametrize("text,changes", HEADS + CACHE + [
    ("reserved", dict(reserved=3)), ("go together", dict(q=0)), ("go together", dict(q_heads=0)), ("rot_dim", dict(rot_dim=24)),
    ("rot_dim", dict(rot_dim=80)), ("total", dict(cu_new=0)), ("strides", dict(k_token=4)), ("strides", dict(q_head=0)), ("overlap", dict(q_out_token=64)),
    ("null", dict(k=0)), ("null", dict(lens=0)), ("null", dict(q_out=0)), ("null", dict(sin=0)), ("aligned", dict(cos=BASE + 4)),
    ("4-byte", dict(lens=BASE + 2)), ("4-byte", dict(cu_new=BASE + 3)), ("q_out overlaps", dict(q_out_token=512)), ("q_out overlaps", dict(q_head=8)),
])
def test_append_refusals(text, changes):
    refused("dv3k_rope_append", APPEND_STRUCT, APPEND, append_ok, text, **changes)


@pytest.mark.parametrize("text,changes", HEADS + CACHE + [
    ("q_heads", dict(q_heads=0)), ("too many", dict(n_seq=1 << 29)), ("scale", dict(scale=float("nan"))), ("strides", dict(q_seq=12)), ("overlap", dict(out_seq=128)),
    ("null", dict(out=0)), ("null", dict(lens=0)), ("aligned", dict(q=BASE + 8)), ("aligned", dict(workspace=BASE + 8)),
    ("workspace", dict(max_pages=4096, table_stride=4096, max_len=65536)), ("4-byte", dict(lens=BASE + 2)), ("4-byte", dict(status=BASE + 1)),
    ("out overlaps", dict(out=BASE)),
])
def test_paged_refusals(text, changes):
    refused("dv3k_attention_paged", PAGED_STRUCT, PAGED, paged_ok, text, **changes)


def test_null_arguments_and_nothing_to_do():
    lib = _lib.load()
    for name in ("dv3k_attention_packed", "dv3k_rope_append", "dv3k_attention_paged"):
        assert getattr(lib, name)(None, None) == dv.INVALID_ARGUMENT and "null" in _lib.last_error()
    assert lib.dv3k_attention_paged_workspace(None) == 0 and lib.dv3k_attention_packed_workspace(None) == 0
    few = dict(packed_ok, total_k=1024)
    assert lib.dv3k_attention_packed_workspace(PACKED_STRUCT.pack(*(few[f] for f in PACKED))) == 0  # nothing long to cut
    for changes in (dict(n_seq=0), dict(total_q=0, q=0, out=0), dict(total_q=0, q_head=0, out_token=0)):
        assert call("dv3k_attention_packed", PACKED_STRUCT, PACKED, dict(packed_ok, **changes))[0] == 0
    for changes in (dict(n_seq=0), dict(total=0, q=0, k=0), dict(total=0, q_head=0, q_out_head=0, k_token=0)):
        assert call("dv3k_rope_append", APPEND_STRUCT, APPEND, dict(append_ok, **changes))[0] == 0
    assert call("dv3k_attention_paged", PAGED_STRUCT, PAGED, dict(paged_ok, n_seq=0, q=0))[0] == 0
    assert call("dv3k_attention_paged", PAGED_STRUCT, PAGED, dict(paged_ok, n_seq=0, q_head=0, out_head=0))[0] == 0


def test_structs_match_the_header(tmp_path):
    """Field order and size of the argument structs used here, as the C compiler lays them out."""
    lines = []
    for struct, fields in (("dv3k_packed_attention", PACKED), ("dv3k_rope_append_args", APPEND), ("dv3k_paged_attention", PAGED)):
        lines += [f'printf("%zu ", offsetof({struct}, {f}));' for f in fields] + [f'printf("%zu\\n", sizeof({struct}));']
    source = tmp_path / "layout.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "dinov3_kernels.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-std=c11", "-I" + os.path.join(ROOT, "include"), str(source), "-o", str(tmp_path / "layout")], check=True)
    rows = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines()
    for row, pack, fields in zip(rows, (PACKED_STRUCT, APPEND_STRUCT, PAGED_STRUCT), (PACKED, APPEND, PAGED)):
        offsets = [int(x) for x in row.split()]
        assert offsets[-1] == pack.size and len(offsets) == len(fields) + 1
        for i, f in enumerate(fields):
            values = [0] * len(fields)
            values[i] = 1
            at = next(j for j, b in enumerate(pack.pack(*values)) if b)
            assert offsets[i] <= at < offsets[i] + 8 and at < offsets[i + 1], f


def test_tensor_binding_is_built_and_refuses_what_is_no_cuda_tensor():
    torch = pytest.importorskip("torch")
    q, cu = torch.zeros(4, 4, 64, dtype=torch.float16), torch.tensor([0, 4], dtype=torch.int32)
    cache, n = torch.zeros(2, 4, 8, 64, dtype=torch.float16), torch.tensor([4], dtype=torch.int32)
    for call in (lambda: dv.attention_packed(q, q, q, cu), lambda: dv.attention_packed(q, None, q, cu), lambda: dv.rope_append(q, q, q, cache, cache, n[None], n),
                 lambda: dv.attention_paged(q[:1], cache, cache, n[None], n)):
        with pytest.raises(dv.DINOv3Error) as e:
            call()
        assert e.value.code == dv.INVALID_ARGUMENT and ("CUDA tensor" in str(e.value) or "must be a tensor" in str(e.value))
