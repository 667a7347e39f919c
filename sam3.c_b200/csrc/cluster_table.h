// cluster_table.h - how many clusters of a kernel run at once, by device and
// cluster size, asked once for each.
#pragma once
#include <atomic>

namespace s3 {

// A kernel's own table: devices differ in what fits.
struct ClusterTable {
  static constexpr int kDevices = 64, kMost = 16;
  std::atomic<int> known[kDevices][kMost + 1] = {};  // what fits, plus one; 0: not asked yet

  // ask(&fit) is 0 where the question was answered; a failed one is not kept,
  // counts as nothing fits this time, and is asked again.
  template <class Ask>
  int fit(int device, int n, Ask ask) {
    const bool keep = device >= 0 && device < kDevices;
    if (const int k = keep ? known[device][n].load() : 0) return k - 1;
    int f = 0;
    if (ask(&f) != 0 || f < 0) return 0;
    if (keep) known[device][n].store(f + 1);
    return f;
  }
};

}  // namespace s3
