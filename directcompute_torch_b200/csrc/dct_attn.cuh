// What the attention kernels share: which keys a row sees, and where its data lies.
//
// A key head's rows are r = i * group + g: position i of the group's query head g, so
// neighbouring rows see (almost) the same keys and one load of a key serves the group.
#pragma once
#include "dct_common.cuh"
#include "kernels.h"

namespace dct {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnSpan {
  int m, n;                    // valid queries and keys of the batch entry
  DCT_DEV AttnSpan(const AttnArgs& a, int b) {
    m = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
    n = a.kv_lens ? min(max(a.kv_lens[b], 0), a.kv_len) : a.kv_len;
  }
  // keys [lo, hi) of query i
  DCT_DEV int lo(const AttnArgs& a, int i) const { return a.window ? max(0, i + n - m - a.window + 1) : 0; }
  DCT_DEV int hi(const AttnArgs& a, int i) const {
    if (i >= m) return 0;
    const int p = i + n - m;
    return a.causal ? min(n, p + 1) : a.window ? min(n, p + a.window) : n;
  }
  // queries [first, last) that may see key j
  DCT_DEV int first(const AttnArgs& a, int j) const {
    const int p = j - (n - m);
    return max(0, a.causal ? p : a.window ? p - a.window + 1 : 0);
  }
  DCT_DEV int last(const AttnArgs& a, int j) const {
    if (j >= n) return 0;
    return a.window ? min(m, j - (n - m) + a.window) : m;
  }
};

}  // namespace dct
