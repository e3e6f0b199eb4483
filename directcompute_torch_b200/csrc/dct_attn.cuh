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

struct RowAt {                 // a row's query position and head
  int i, h;
  DCT_DEV RowAt(const AttnArgs& a, int hk, int r) : i(r / a.group), h(hk * a.group + r % a.group) {}
};

// the offset of (b, t, h) in a strided tensor
DCT_DEV int64_t at(const int64_t* s, int b, int t, int h) { return b * s[0] + t * s[1] + h * s[2]; }

// ---------------------------------------------------------------------------
// what the tensor-core kernels know about a key head's operands (q, k, v, dout)
// ---------------------------------------------------------------------------
// Magnitudes over the valid rows as float bits, which order like integers, so that they
// meet by atomic maximum from 0 (the same in any order).
struct AttnStats {
  uint32_t top[4];             // the largest |x|; from 0x7f800000 on: infinity or NaN
  uint32_t low[4];             // ~ the smallest row maximum that is not 0
  uint32_t norm[4];            // the largest row norm
};
// Each operand is held as 2^e x = hi + lo in float16 with its largest magnitude in
// [2^14, 2^15); an element is then off by 2^-23 of itself or 2^-40 of that largest one.
// dS is scaled by 2^eds, from |dS / (P scale)| <= 2 max|dout row| max|v row|.
struct AttnScales {
  int e[4], eds;
  bool split;                  // false: the head goes to the float32 kernels
};
DCT_DEV AttnScales scales_of(const AttnStats& st, float scale, int dim, bool backward) {
  AttnScales s;
  s.split = true;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (t == 3 && !backward) { s.e[t] = 0; break; }
    const int top = (int)(st.top[t] >> 23) - 127, low = st.low[t] ? (int)(~st.low[t] >> 23) - 127 : top;
    s.e[t] = st.top[t] ? 14 - top : 0;
    // infinities and NaN; sizes whose scaling leaves float32; rows so far apart that the
    // small ones would lose their own accuracy to the common scale
    if (st.top[t] && (top < -100 || top > 100 || low < top - 14)) s.split = false;
  }
  // scores beyond 2^18 amplify the common scale's 2^-40 past float32's own error
  const float most = __uint_as_float(st.top[0]) * __uint_as_float(st.top[1]);
  if (!(fabsf(scale) * dim * most < 262144.f)) s.split = false;
  s.eds = 0;
  if (backward) {
    const float n = __uint_as_float(st.norm[2]) * __uint_as_float(st.norm[3]);
    if (!(n < 1e30f)) s.split = false;
    else if (n > 0.f) s.eds = 13 - ((int)(__float_as_uint(n) >> 23) - 127);
    if (n > 0.f && n < 1e-30f) s.split = false;
  }
  return s;
}

}  // namespace dct
