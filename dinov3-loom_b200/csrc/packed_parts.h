// packed_parts.h - the workspace in which packed attention's cut items leave their partial results
// for the joining launch, and the check that they are all there. Plain C++ on host and device.
//
// A CTA describes a part when it takes it up. A CTA that gave up (an expired wait) leaves the parts
// it did not take up undescribed: whatever the workspace held before, which the join must not take for
// rows and places. So every CTA writes at its end whether it did all of its work, and the join does
// nothing unless all did.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#define DV3_HOST_DEVICE __host__ __device__
#else
#define DV3_HOST_DEVICE
#endif

namespace dv3 {

struct Part {
  int32_t q_row, q_count, head, index, parts;
  int32_t unused[3];
};

// For up to `n` parts: their number, a word of each CTA (one for every two parts), then for each part what
// it is, (max, sum) of its 2 x 128 rows, and their outputs, four channels of 128 rows after another.
template <int kDim>
struct Parts {
  static constexpr uint32_t kDone = 0x646f6e65u, kGaveUp = 0;
  uint32_t *count;
  uint32_t *done;  // [ctas]
  Part *what;
  float *ml;  // pairs [part][2][128]
  float *o;   // fours [part][2][kDim / 4][128]

  DV3_HOST_DEVICE static uint32_t ctas(uint32_t n) { return n / 2; }
  DV3_HOST_DEVICE static size_t head_bytes(uint32_t n) { return (16 + size_t{4} * ctas(n) + 15) / 16 * 16; }
  DV3_HOST_DEVICE static size_t bytes(uint32_t n) {
    return head_bytes(n) + static_cast<size_t>(n) * (sizeof(Part) + 256 * 2 * sizeof(float) + 256 * kDim * sizeof(float));
  }
  DV3_HOST_DEVICE static Parts of(void *workspace, uint32_t n) {
    Parts p;
    uint8_t *at = static_cast<uint8_t *>(workspace);
    p.count = reinterpret_cast<uint32_t *>(at);
    p.done = reinterpret_cast<uint32_t *>(at + 16);
    p.what = reinterpret_cast<Part *>(at + head_bytes(n));
    p.ml = reinterpret_cast<float *>(p.what + n);
    p.o = p.ml + static_cast<size_t>(n) * 512;
    return p;
  }
  // Whether CTAs `from`, `from` + `step`, ... did all of their work.
  DV3_HOST_DEVICE bool finished(uint32_t n, uint32_t from, uint32_t step) const {
    for (uint32_t i = from; i < ctas(n); i += step)
      if (done[i] != kDone) return false;
    return true;
  }
};

}  // namespace dv3
