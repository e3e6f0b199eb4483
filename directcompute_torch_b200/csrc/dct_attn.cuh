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
    return a.window ? max(0, min(m, j - (n - m) + a.window)) : m;     // not negative: rows are `group` times as many
  }
};

struct RowAt {                 // a row's query position and head
  int i, h;
  DCT_DEV RowAt(const AttnArgs& a, int hk, int r) : i(r / a.group), h(hk * a.group + r % a.group) {}
};

// the offset of (b, t, h) in a strided tensor
DCT_DEV int64_t at(const int64_t* s, int b, int t, int h) { return b * s[0] + t * s[1] + h * s[2]; }

// ---------------------------------------------------------------------------
// what the tensor-core kernels know about their operands (q, k, v, dout)
// ---------------------------------------------------------------------------
// A tile of 128 rows is held as 2^e x = hi + lo in float16 with its largest magnitude in
// [2^14, 2^15); an element is then off by 2^-23 of itself or 2^-40 of that largest one.
struct AttnTile {
  int32_t e;
};
// Of a key head: magnitudes as float bits, which order like integers, so that they meet by
// atomic maximum from 0 (the same in any order).
struct AttnStats {
  uint32_t top_q, top_k;       // the largest |q|, |k|
  uint32_t bad;                // some tile cannot be split
  uint32_t top_v, low_v;       // the largest |v| of a tile, and ~ the smallest that is not 0
  uint32_t pad[3];
};
// Tiles of infinities or NaN, of sizes whose scaling could leave float32, or with rows so far
// apart that the small ones would lose their own accuracy to the common scale (2^-14 of it
// leaves 26 bits), cannot be split.  `low` is the smallest row maximum that is not 0.  Neither
// can those whose features are as far apart, where they make a result's features.
constexpr int kApart = 14;
DCT_DEV bool tile_splits(uint32_t top, uint32_t low) {
  const int t = (int)(top >> 23) - 127, l = (int)(low >> 23) - 127;
  return top == 0 || (t >= -60 && t <= 44 && l >= t - kApart);
}
// Whether a head takes the tensor cores: scores beyond 2^18 would amplify a tile's 2^-40 past
// float32's own error; tiles of v further than 2^60 apart could overflow the running outputs,
// which carry the scale of the tile added last.
DCT_DEV bool head_splits(const AttnStats& st, float scale, int dim) {
  if (st.low_v && (int)(st.top_v >> 23) - (int)(~st.low_v >> 23) > 60) return false;
  return !st.bad && fabsf(scale) * dim * __uint_as_float(st.top_q) * __uint_as_float(st.top_k) < 262144.f;
}

}  // namespace dct
