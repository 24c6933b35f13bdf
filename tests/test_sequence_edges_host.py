"""What the packed and paged operators' host side and package do at their edges, without a GPU."""
import os
import subprocess
import sys

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
