// Rotary positions: each pair of features turns by position * frequency.
//
// Memory bound: 8 bytes per feature (one read, one write) and 3 flops a pair side.  A
// block takes whole tokens (about 4096 features: one token of a wide projection, several
// of a narrow one), so the angles of a token are formed once for all its heads: the turn
// position * f / 2pi is reduced to [-1/2, 1/2] and its sine and cosine are taken in
// float64 (a far position times a float32 frequency would lose its angle: at position
// 2^20 half an ulp of the product is 0.03 rad), then rounded once to float32.  The
// block's first loads are issued before that work, so it hides behind them.
#include "dct_common.cuh"
#include "kernels.h"

namespace dct {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;                 // units in flight per thread

struct RotaryGeom {
  const float* x;
  const int32_t* positions;
  float* y;
  int64_t xs[3], ys[3];
  uint32_t length, heads, half;           // half: pairs per head
  uint32_t tokens, per_block;             // batch * length, tokens per block
  int32_t start;
  FastDiv by_length, by_units, by_heads;  // unit index -> (token, head, unit)
  uint32_t units;                         // units per head
  float magnitude;
  bool inverse;
};

struct Unit {                             // the features of one unit
  const float* x;
  float* y;
  uint32_t u, token;                      // unit within the head, token within the block
};

template <int V>
struct Vec;
template <>
struct Vec<4> {
  using T = float4;
  static DCT_DEV T load(const float* p) { return ld_stream4(p); }
  static DCT_DEV void store(float* p, T v) { st_stream4(p, v); }
};
template <>
struct Vec<1> {
  using T = float;
  static DCT_DEV T load(const float* p) { return ld_stream(p); }
  static DCT_DEV void store(float* p, T v) { st_stream(p, v); }
};

DCT_DEV float2 turn(float a, float b, float2 cs) {
  return make_float2(fmaf(a, cs.x, -(b * cs.y)), fmaf(b, cs.x, a * cs.y));
}

// V = 4: a unit is 4 neighbouring features (INTER: two pairs; else the first halves of
// four pairs, whose second halves lie half a rotation away) or 4 copied features.
// V = 1: a unit is one pair or one copied feature.
template <int V, bool INTER>
__global__ void __launch_bounds__(kThreads) k_rotary(const __grid_constant__ RotaryGeom g,
                                                     const __grid_constant__ RotaryTurns f) {
  extern __shared__ float2 table[];       // [token][half] (cos, sin) * magnitude
  using L = Vec<V>;
  using T = typename L::T;
  const uint32_t t0 = blockIdx.x * g.per_block;
  const uint32_t tokens = min(g.per_block, g.tokens - t0);
  const uint32_t total = tokens * g.heads * g.units;
  const uint32_t pair_units = INTER ? (V == 4 ? g.half / 2 : g.half) : g.half / V;

  Unit un[kAhead];
  T a[kAhead], b[kAhead];
  auto fetch = [&](uint32_t first) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint32_t i = first + k * kThreads;
      if (i >= total) continue;
      const uint32_t th = g.by_units.div(i), u = i - th * g.units;
      const uint32_t token = g.by_heads.div(th), h = th - token * g.heads;
      const uint32_t bt = t0 + token, bb = g.by_length.div(bt), t = bt - bb * g.length;
      // first feature of the unit
      const uint32_t at = u < pair_units ? (INTER ? (V == 4 ? 4 * u : 2 * u) : V * u)
                                         : 2 * g.half + V * (u - pair_units);
      un[k].u = u;
      un[k].token = token;
      un[k].x = g.x + bb * g.xs[0] + t * g.xs[1] + h * g.xs[2] + at;
      un[k].y = g.y + bb * g.ys[0] + t * g.ys[1] + h * g.ys[2] + at;
      a[k] = L::load(un[k].x);
      if (u < pair_units) {
        if constexpr (!INTER) b[k] = L::load(un[k].x + g.half);
        else if constexpr (V == 1) b[k] = L::load(un[k].x + 1);
      }
    }
  };
  auto finish = [&](uint32_t first) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (first + k * kThreads >= total) continue;
      const Unit& n = un[k];
      if (n.u >= pair_units) {
        L::store(n.y, a[k]);
        continue;
      }
      const float2* cs = table + n.token * g.half;
      if constexpr (V == 1) {
        const float2 r = turn(a[k], b[k], cs[n.u]);
        n.y[0] = r.x;
        n.y[INTER ? 1 : g.half] = r.y;
      } else if constexpr (INTER) {
        const float2 p = turn(a[k].x, a[k].y, cs[2 * n.u]), q = turn(a[k].z, a[k].w, cs[2 * n.u + 1]);
        L::store(n.y, make_float4(p.x, p.y, q.x, q.y));
      } else {
        const float2* c = cs + 4 * n.u;
        const float2 p = turn(a[k].x, b[k].x, c[0]), q = turn(a[k].y, b[k].y, c[1]);
        const float2 r = turn(a[k].z, b[k].z, c[2]), s = turn(a[k].w, b[k].w, c[3]);
        L::store(n.y, make_float4(p.x, q.x, r.x, s.x));
        L::store(n.y + g.half, make_float4(p.y, q.y, r.y, s.y));
      }
    }
  };

  fetch(threadIdx.x);
  for (uint32_t i = threadIdx.x; i < tokens * g.half; i += kThreads) {
    const uint32_t token = i / g.half, j = i - token * g.half;
    const uint32_t bt = t0 + token;
    const int64_t pos = g.positions ? (int64_t)g.positions[bt]
                                    : (int64_t)g.start + (bt - g.by_length.div(bt) * g.length);
    double s, c, n = (double)pos * f.turns[j];
    n -= rint(n);
    sincospi(2.0 * n, &s, &c);
    table[i] = make_float2((float)(g.magnitude * c), (float)((g.inverse ? -g.magnitude : g.magnitude) * s));
  }
  __syncthreads();
  for (uint32_t first = threadIdx.x; first < total; first += kAhead * kThreads) {
    finish(first);
    fetch(first + kAhead * kThreads);
  }
}

}  // namespace

cudaError_t launch_rotary(const RotaryArgs& a, const RotaryTurns& f, cudaStream_t st) {
  if (!a.batch || !a.length || !a.heads) return cudaSuccess;
  RotaryGeom g;
  g.x = a.x; g.positions = a.positions; g.y = a.y;
  bool vec = aligned16_h(a.x) && aligned16_h(a.y) && a.head_dim % 4 == 0 &&
             (a.interleaved ? a.rotated % 4 == 0 : a.rotated % 8 == 0);
  for (int i = 0; i < 3; ++i) {
    g.xs[i] = a.xs[i];
    g.ys[i] = a.ys[i];
    vec = vec && a.xs[i] % 4 == 0 && a.ys[i] % 4 == 0;
  }
  g.length = a.length; g.heads = a.heads; g.half = a.rotated / 2;
  g.tokens = a.batch * a.length;
  g.start = a.start;
  g.magnitude = a.magnitude;
  g.inverse = a.inverse;
  const uint32_t copied = a.in_place ? 0 : a.head_dim - a.rotated;   // in place, the rest is there already
  g.units = vec ? (a.interleaved ? a.rotated / 4 : a.rotated / 8) + copied / 4 : g.half + copied;
  if (!g.units) return cudaSuccess;
  const uint32_t width = a.heads * a.head_dim;
  g.per_block = width >= 4096 ? 1 : 4096 / width;
  if (g.per_block > g.tokens) g.per_block = g.tokens;
  // a table of at most 16 KB: 4096 features hold at most 2048 pairs, a wider token's heads at most 128
  g.by_length = FastDiv(g.length); g.by_units = FastDiv(g.units); g.by_heads = FastDiv(g.heads);
  const uint32_t blocks = (g.tokens + g.per_block - 1) / g.per_block;
  const size_t smem = sizeof(float2) * g.per_block * g.half;
  if (vec && a.interleaved) k_rotary<4, true><<<blocks, kThreads, smem, st>>>(g, f);
  else if (vec) k_rotary<4, false><<<blocks, kThreads, smem, st>>>(g, f);
  else if (a.interleaved) k_rotary<1, true><<<blocks, kThreads, smem, st>>>(g, f);
  else k_rotary<1, false><<<blocks, kThreads, smem, st>>>(g, f);
  return cudaGetLastError();
}

}  // namespace dct
