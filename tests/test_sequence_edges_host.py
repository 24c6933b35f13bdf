"""What the packed and paged operators' host side and package do at their edges, without a GPU."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "dinov3-loom_b200", "csrc")

PARTS = r"""
#include <cstdio>
#include <cstring>
#include <vector>
#include "packed_parts.h"
template <int kDim> int check(uint32_t n) {
  using P = dv3::Parts<kDim>;
  std::vector<uint64_t> buffer(P::bytes(n) / 8 + 1, ~0ull);  // what an allocator may hand out
  const P p = P::of(buffer.data(), n);
  const char *base = reinterpret_cast<const char *>(buffer.data());
  auto at = [&](const void *x) { return static_cast<size_t>(static_cast<const char *>(x) - base); };
  const uint32_t ctas = P::ctas(n);
  // the pieces lie one behind the other, aligned for their loads, inside the buffer
  if (at(p.done) < 4 || at(p.what) < at(p.done) + 4 * ctas || at(p.ml) < at(p.what) + n * sizeof(dv3::Part)) return 1;
  if (at(p.o) < at(p.ml) + size_t{n} * 2048 || at(p.o) + size_t{n} * 1024 * kDim > P::bytes(n)) return 2;
  if (at(p.what) % 16 || at(p.ml) % 16 || at(p.o) % 16) return 3;
  // nothing written, one CTA that gave up, a count that came through all the same: never joined
  *p.count = n;
  if (p.finished(n, 0, 1)) return 4;
  for (uint32_t i = 0; i < ctas; ++i) p.done[i] = P::kDone;
  if (!p.finished(n, 0, 1)) return 5;
  for (uint32_t bad = 0; bad < ctas; ++bad) {
    for (const uint32_t word : {P::kGaveUp, ~0u, 1u}) {
      p.done[bad] = word;
      bool all = true;
      for (uint32_t thread = 0; thread < 256; ++thread) all = all && p.finished(n, thread, 256);
      if (all || p.finished(n, 0, 1)) return 6;
    }
    p.done[bad] = P::kDone;
  }
  return 0;
}
int main() {
  for (uint32_t n : {2u, 10u, 264u, 296u, 1024u})
    if (int e = check<64>(n) ? check<64>(n) : check<128>(n)) return printf("%u: %d\n", n, e), 1;
  puts("ok");
}
"""


def test_the_join_waits_for_every_block_of_the_launch_before(tmp_path):
    """Parts that a block never described hold whatever the workspace held: the join's check of them."""
    source = tmp_path / "parts.cpp"
    source.write_text(PARTS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I" + CSRC, str(source), "-o", str(tmp_path / "parts")], check=True)
    got = subprocess.run([str(tmp_path / "parts")], capture_output=True, text=True)
    assert got.stdout == "ok\n", got.stdout


SIZES = """
import sys
sys.path[:0] = sys.argv[1:]
from dinov3_b200 import _lib
from test_sequence_host import PACKED, PACKED_STRUCT, PAGED, PAGED_STRUCT, packed_ok, paged_ok
lib = _lib.load()
packed = lambda **c: lib.dv3k_attention_packed_workspace(PACKED_STRUCT.pack(*(dict(packed_ok, **c)[f] for f in PACKED)))
paged = lambda **c: lib.dv3k_attention_paged_workspace(PAGED_STRUCT.pack(*(dict(paged_ok, **c)[f] for f in PAGED)))
long = dict(max_pages=4096, max_len=65536)
assert packed(total_k=4096) > 0 and paged(**long) > 0
for c in (dict(page_size=0), dict(page_size=65537), dict(page_size=2**32 - 1), dict(max_pages=2**31), dict(n_seq=0), dict(n_seq=2**29), dict(n_seq=2**32 - 1),
          dict(q_heads=0), dict(q_heads=5), dict(kv_heads=0), dict(head_dim=0), dict(q_heads=258)):
    assert paged(**dict(long, **c)) == 0, c
    assert paged(**c) == 0, c
for c in (dict(n_seq=0), dict(n_seq=2**32 - 1), dict(total_q=0), dict(total_q=2**32 - 1), dict(total_k=2**32 - 1), dict(q_heads=0), dict(q_heads=5),
          dict(kv_heads=0), dict(head_dim=80), dict(q_heads=258)):
    assert packed(**dict(dict(total_k=4096), **c)) == 0, c
print("ok")
"""


def test_size_calls_of_what_the_launch_refuses():
    """No workspace, and no crash, for arguments that no call accepts."""
    got = subprocess.run([sys.executable, "-c", SIZES, os.path.join(ROOT, "dinov3-loom_b200"), os.path.join(ROOT, "tests")], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout == "ok\n", (got.returncode, got.stderr[-1500:])


REGIONS = r"""
#include <cstdio>
#include <random>
#include <set>
#include "regions.h"
using dv3::Region;
static std::set<uintptr_t> bytes_of(const Region &r) {
  std::set<uintptr_t> s;
  for (uint32_t i = 0; i < r.n_outer; ++i)
    for (uint32_t j = 0; j < r.n_inner; ++j)
      for (int64_t b = 0; b < r.bytes; ++b) s.insert(reinterpret_cast<uintptr_t>(r.base) + i * r.outer + j * r.inner + b);
  return s;
}
static bool share(const Region &a, const Region &b) {
  const auto x = bytes_of(a), y = bytes_of(b);
  for (uintptr_t i : x)
    if (y.count(i)) return true;
  return false;
}
static const void *at(int64_t x) { return reinterpret_cast<const void *>(x); }
int main() {
  std::mt19937 rng(5);
  auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % (hi - lo + 1)); };
  int apart = 0, views = 0;
  for (int n = 0; n < 20000; ++n) {
    Region r[2];
    for (Region &x : r) x = {at(pick(100, 160)), pick(1, 24), pick(1, 24), static_cast<uint32_t>(pick(0, 4)), static_cast<uint32_t>(pick(0, 4)), pick(0, 9)};
    if (n % 2) r[1].outer = r[0].outer, r[1].inner = r[0].inner;
    if (dv3::apart(r[0], r[1]) != dv3::apart(r[1], r[0])) return puts("not symmetric"), 1;
    if (!dv3::apart(r[0], r[1])) continue;
    ++apart;
    if (share(r[0], r[1])) return puts("shares"), 1;
  }
  // columns of one buffer [rows][columns][8 bytes], and slices of its vectors: told apart exactly
  for (int n = 0; n < 20000; ++n) {
    const int rows = pick(1, 4), columns = pick(1, 5), width = pick(1, 8);
    Region r[2];
    for (Region &x : r) {
      const int c0 = pick(0, columns - 1), w0 = pick(0, width - 1);
      x = {at(1000 + c0 * width + w0), columns * width, width, static_cast<uint32_t>(rows), static_cast<uint32_t>(pick(1, columns - c0)), pick(1, width - w0)};
      if (pick(0, 1)) std::swap(x.outer, x.inner), std::swap(x.n_outer, x.n_inner);
    }
    ++views;
    if (dv3::apart(r[0], r[1]) == share(r[0], r[1])) return puts("views"), 1;
  }
  // nothing, and strides whose product passes 64 bits
  if (!dv3::apart({nullptr, 1, 1, 1, 1, 1}, {at(5), 1, 1, 1, 1, 1})) return puts("null"), 1;
  const Region far = {at(1 << 20), int64_t{1} << 38, int64_t{1} << 38, 0x7fffffffu, 0x7fffffffu, 256};
  if (dv3::apart(far, {at((1 << 20) + (int64_t{1} << 39)), 256, 256, 1, 1, 256}) || !dv3::apart(far, {at(1 << 19), 256, 256, 4, 4, 256})) return puts("far"), 1;
  printf("ok %d\n", apart > 3000);
}
"""


def test_regions_are_told_apart(tmp_path):
    source = tmp_path / "regions.cpp"
    source.write_text(REGIONS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I" + CSRC, str(source), "-o", str(tmp_path / "regions")], check=True)
    got = subprocess.run([str(tmp_path / "regions")], capture_output=True, text=True)
    assert got.stdout == "ok 1\n", got.stdout


from test_sequence_host import (APPEND, APPEND_STRUCT, BASE, PACKED, PACKED_STRUCT, PAGED, PAGED_STRUCT, append_ok, packed_ok,  # noqa: E402
                                paged_ok, refused)

FAR = {name: BASE + (i + 1) * (1 << 24) for i, name in enumerate("q k v out lse cu_q cu_k status q_out k_cache v_cache cu_new lens page_table cos sin".split())}


def moved(ok):
    """The arguments with every tensor far from the others: addresses that nothing reads."""
    return {f: FAR[f] if f in FAR and v else v for f, v in ok.items()}


# q is [4][4][64], 2048 bytes; k, v [4][2][64] in rows of 256 elements; caches [8][2][16][64]
@pytest.mark.parametrize("changes", [
    dict(out=FAR["q"] + 128), dict(out=FAR["q"] - 16), dict(out=FAR["q"] + 2032), dict(out=FAR["k"] - 128), dict(out=FAR["v"] + 16), dict(out=FAR["cu_q"] - 2032),
    dict(out=FAR["cu_k"]), dict(lse=FAR["q"] + 4), dict(lse=FAR["v"]), dict(lse=FAR["out"] + 2044), dict(status=FAR["out"]), dict(lse=FAR["cu_q"]),
    dict(out=FAR["q"], out_token=512), dict(out=FAR["q"] + 64 * 2, q_token=512, out_token=512),
])
def test_packed_outputs_that_overlap(changes):
    refused("dv3k_attention_packed", PACKED_STRUCT, PACKED, moved(packed_ok), "overlap", **changes)


@pytest.mark.parametrize("changes", [
    dict(q_out=FAR["q"] + 128), dict(q_out=FAR["q"] - 2032), dict(q_out=FAR["k"]), dict(q_out=FAR["v"] + 64), dict(q_out=FAR["k_cache"] + 4096),
    dict(q_out=FAR["cos"]), dict(k_cache=FAR["v_cache"]), dict(k_cache=FAR["v_cache"] + 4096), dict(v_cache=FAR["k_cache"] + 2048), dict(k_cache=FAR["k"]),
    dict(v_cache=FAR["q"] - 4096), dict(k_cache=FAR["page_table"]), dict(v_cache=FAR["lens"]), dict(k_cache=FAR["sin"]), dict(q_out=FAR["cu_new"]),
    dict(status=FAR["k_cache"] + 8),
])
def test_append_outputs_that_overlap(changes):
    refused("dv3k_rope_append", APPEND_STRUCT, APPEND, moved(append_ok), "overlap", **changes)


@pytest.mark.parametrize("changes", [
    dict(out=FAR["q"] + 128), dict(out=FAR["k_cache"] + 4096), dict(out=FAR["v_cache"]), dict(out=FAR["page_table"]), dict(out=FAR["lens"] - 1008), dict(lse=FAR["out"]),
    dict(lse=FAR["q"] + 8), dict(lse=FAR["k_cache"]), dict(status=FAR["out"] + 8),
])
def test_paged_outputs_that_overlap(changes):
    refused("dv3k_attention_paged", PAGED_STRUCT, PAGED, moved(paged_ok), "overlap", **changes)


STAR = """
import sys
sys.path.insert(0, sys.argv[1])
sys.modules["torch"] = None  # an import of it raises
from dinov3_b200 import *
import dinov3_b200
assert DINOv3 is dinov3_b200.DINOv3 and "attention_packed" not in globals()
assert not any(m == "torch" or m.startswith("torch.") for m in sys.modules if sys.modules[m])
try:
    dinov3_b200.attention_packed
except ImportError as e:
    print("ok")
"""


def test_a_star_import_needs_no_torch():
    """What every name of the package but the sequence operators' needs."""
    got = subprocess.run([sys.executable, "-c", STAR, os.path.join(ROOT, "dinov3-loom_b200")], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout == "ok\n", got.stderr[-1500:]


STUB = """#!/bin/sh
# in nvcc's place: notes the call, makes the output
while [ $# -gt 0 ]; do case "$1" in
  -ltorch_cuda) binding=1;;
  -o) shift; out="$1";;
esac; shift; done
echo "$out" >> "$(dirname "$0")/calls"
if [ "$binding" ] && [ -e "$(dirname "$0")/broken" ]; then echo "no such header"; exit 1; fi
: > "$out"
"""


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """build.py with a stub for nvcc, its outputs in a folder of their own, and a torch of a few files."""
    import importlib.util

    spec = importlib.util.spec_from_file_location("dv3_build_under_test", os.path.join(ROOT, "dinov3-loom_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(STUB)
    nvcc.chmod(0o755)
    torch = tmp_path / "torch"
    (torch / "lib").mkdir(parents=True)
    (torch / "version.py").write_text("__version__ = '1'\n")
    (torch / "lib" / "libtorch_cuda.so").write_text("")
    for name, to in (("NVCC", nvcc), ("BUILD", tmp_path / "objects"), ("LIB", tmp_path / "libdinov3.so"), ("BINDING_LIB", tmp_path / "_sequence.so")):
        monkeypatch.setattr(mod, name, str(to))
    found = type("Spec", (), {"submodule_search_locations": [str(torch)]})()
    monkeypatch.setattr(mod.importlib.util, "find_spec", lambda name: found)

    def calls():
        log = tmp_path / "calls"
        got = log.read_text().split() if log.exists() else []
        log.write_text("")
        return got

    mod.tmp, mod.torch, mod.calls = tmp_path, torch, calls
    return mod


def test_the_library_builds_whatever_torch_is(builder, capfd, monkeypatch):
    (builder.torch / "lib" / "libtorch_cuda.so").unlink()
    builder.build()
    assert os.path.exists(builder.LIB) and not os.path.exists(builder.BINDING_LIB) and "CUDA" in capfd.readouterr().err
    (builder.torch / "lib" / "libtorch_cuda.so").write_text("")
    (builder.tmp / "broken").write_text("")
    os.unlink(builder.LIB)
    builder.build()
    assert os.path.exists(builder.LIB) and not os.path.exists(builder.BINDING_LIB) and "no such header" in capfd.readouterr().err
    (builder.tmp / "broken").unlink()
    builder.build()
    assert os.path.exists(builder.BINDING_LIB) and capfd.readouterr().err == ""
    monkeypatch.setattr(builder.importlib.util, "find_spec", lambda name: None)
    builder.build(force=True)
    assert capfd.readouterr().err == ""


def test_the_binding_follows_torch_and_python(builder, monkeypatch):
    binding = [builder.BINDING_LIB]
    builder.build()
    assert builder.calls().count(binding[0]) == 1
    builder.build()
    assert builder.calls() == []
    (builder.torch / "version.py").write_text("__version__ = '2'\n")
    builder.build()
    assert builder.calls() == binding
    builder.build()
    assert builder.calls() == []
    soabi = builder.sysconfig.get_config_var
    monkeypatch.setattr(builder.sysconfig, "get_config_var", lambda name: "cpython-399" if name == "SOABI" else soabi(name))
    builder.build()
    assert builder.calls() == binding
    # one that was built for another torch and cannot be built for this one goes: it might not load, or crash
    (builder.torch / "version.py").write_text("__version__ = '3'\n")
    (builder.tmp / "broken").write_text("")
    builder.build()
    assert not os.path.exists(builder.BINDING_LIB)


def test_one_workspace_for_every_call():
    """The sizes of single calls go up and down with their arguments; the bounds cover all of them."""
    import random

    from dinov3_b200 import _lib
    lib, rng = _lib.load(), random.Random(3)
    needs = set()
    for _ in range(3000):
        kv, group, dim = rng.choice([1, 2, 3, 8, 40]), rng.choice([1, 2, 4, 7, 16, 17, 33, 128]), rng.choice([64, 128])
        n = int(2 ** rng.uniform(0, 12))
        heads = dict(q_heads=kv * group, kv_heads=kv, head_dim=dim)
        page = rng.choice([1, 16, 67])
        c = dict(paged_ok, n_seq=n, max_len=int(2 ** rng.uniform(0, 22)), page_size=page, max_pages=(1 << 22) // page, **heads)
        need = lib.dv3k_attention_paged_workspace(PAGED_STRUCT.pack(*(c[f] for f in PAGED)))
        needs.add(need > 0)
        for more in (n, n + 1, 2 * n + 5):
            assert need <= lib.dv3k_attention_paged_workspace_bound(more, kv * group, kv, dim)
        c = dict(packed_ok, n_seq=n, total_q=int(2 ** rng.uniform(0, 20)), total_k=int(2 ** rng.uniform(0, 24)), **heads)
        need = lib.dv3k_attention_packed_workspace(PACKED_STRUCT.pack(*(c[f] for f in PACKED)))
        needs.add(need > 0)
        assert need <= lib.dv3k_attention_packed_workspace_bound(dim)
    assert needs == {False, True}
    # not far above what a call may need: the largest of one long sequence
    one = dict(paged_ok, n_seq=1, max_len=1 << 22, max_pages=1 << 18, q_heads=32, kv_heads=8, head_dim=128)
    assert lib.dv3k_attention_paged_workspace_bound(1, 32, 8, 128) <= 1.01 * lib.dv3k_attention_paged_workspace(PAGED_STRUCT.pack(*(one[f] for f in PAGED)))
    for refused_heads in ((0, 4, 4, 64), (2**30, 4, 4, 64), (4, 5, 4, 64), (4, 4, 0, 64), (4, 4, 4, 80)):
        assert lib.dv3k_attention_paged_workspace_bound(*refused_heads) == 0
    assert lib.dv3k_attention_packed_workspace_bound(96) == 0


def test_more_sequences_than_a_search_may_walk():
    refused("dv3k_attention_packed", PACKED_STRUCT, PACKED, packed_ok, "too many", n_seq=(1 << 24) + 1)
    refused("dv3k_attention_packed", PACKED_STRUCT, PACKED, packed_ok, "overlap", n_seq=1 << 24)  # not for their number
