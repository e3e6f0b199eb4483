// Attention on the CUDA cores: float32 products and sums of any input.
//
// Eight lanes share a key (or, for the key gradients, a row), each holding a float4 of
// every 32 features, so a warp reads four rows of memory at a time in full sectors and a
// dot product is finished by three shuffles.  A block of 4 warps walks 16 keys at a time
// for R rows of one key head, which share each load; every octet keeps its own running
// maximum, sum and output, joined at the end in a fixed order.
//
// It is bound by the bytes of K and V when there are few rows (one new token per
// sequence), where the keys are split over blocks so that every SM reads, and the
// splits' records are joined by a second kernel.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "dct_attn.cuh"

namespace dct {
namespace {

constexpr int kWarps = 4, kOctets = 4 * kWarps;
constexpr unsigned kFull = 0xffffffffu;
constexpr int kMostSplits = 64;
constexpr int kAhead = 3;                // steps of the key ring

// 16 bytes (or zeros, for `bytes` 0) into shared memory, behind the thread's back
DCT_DEV void copy_async(void* to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from),
               "r"(bytes)
               : "memory");
}
DCT_DEV void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
DCT_DEV void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// feature of element e of chunk c for lane l of an octet
template <int NV, bool VEC>
DCT_DEV void load_row(float (&x)[4 * NV], const float* p, int lane, int dim) {
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int f = (c * 8 + lane) * 4;
    if constexpr (VEC) {
      const float4 v = f < dim ? *reinterpret_cast<const float4*>(p + f) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[4 * c] = v.x; x[4 * c + 1] = v.y; x[4 * c + 2] = v.z; x[4 * c + 3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * c + e] = f + e < dim ? p[f + e] : 0.f;
    }
  }
}

template <int N>
DCT_DEV float dot(const float (&x)[N], const float (&y)[N]) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    s0 = fmaf(x[e], y[e], s0);
    s1 = fmaf(x[e + 1], y[e + 1], s1);
  }
  return s0 + s1;
}

DCT_DEV float octet_sum(float s) {
  s += __shfl_xor_sync(kFull, s, 1);
  s += __shfl_xor_sync(kFull, s, 2);
  s += __shfl_xor_sync(kFull, s, 4);
  return s;
}

// 2^(x - top), with 0 for a place whose running maximum is still -inf
DCT_DEV float weight(float x, float top) { return exp2f(x - (top == -INFINITY ? 0.f : top)); }

// record of a split: [dim] outputs, then the maximum (base 2) and the sum
DCT_DEV float* record(float* part, const AttnArgs& a, int64_t row, int splits, int split) {
  return part + (row * splits + split) * (a.dim + 2);
}

DCT_DEV void store_row(const AttnArgs& a, int b, const RowAt& w, int f, float acc, float top, float sum) {
  a.out[at(a.os, b, w.i, w.h) + f] = sum == 0.f ? 0.f : acc / sum;
  if (f == 0 && a.lse)
    a.lse[((int64_t)b * a.q_heads + w.h) * a.q_len + w.i] = sum == 0.f ? -INFINITY : fmaf(top, kLn2, logf(sum));
}

template <int NV, bool VEC, int R>
DCT_DEV void rows_forward(const AttnArgs& a, int item, int groups, int splits, float* part,
                          float (&sh)[kWarps][R][32 * NV + 2]) {
  constexpr int F = 4 * NV;
  const int lane = threadIdx.x & 7, oct = threadIdx.x >> 3, warp = threadIdx.x >> 5;
  const int split = item % splits, gi = (item / splits) % groups, bh = item / splits / groups;
  const int b = bh / a.kv_heads, hk = bh % a.kv_heads, rows = a.q_len * a.group;
  if (a.stats && head_splits(a.stats[bh], a.scale, a.dim)) return;
  const AttnSpan span(a, b);
  const float scale = a.scale * kLog2e;

  float q[R][F], acc[R][F], top[R], sum[R];
  int lo[R], hi[R], k0 = INT_MAX, k1 = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = gi * R + r;
    const RowAt w(a, hk, row);
    lo[r] = hi[r] = 0;
    if (row < rows && w.i < span.m) {
      lo[r] = span.lo(a, w.i);
      hi[r] = span.hi(a, w.i);
      if (lo[r] < hi[r]) {
        k0 = min(k0, lo[r]);
        k1 = max(k1, hi[r]);
      }
      load_row<NV, VEC>(q[r], a.q + at(a.qs, b, w.i, w.h), lane, a.dim);
    } else {
#pragma unroll
      for (int e = 0; e < F; ++e) q[r][e] = 0.f;
    }
    top[r] = -INFINITY;
    sum[r] = 0.f;
#pragma unroll
    for (int e = 0; e < F; ++e) acc[r][e] = 0.f;
  }
  if (k0 < k1 && splits > 1) {
    const int per = ((k1 - k0 + splits - 1) / splits + kOctets - 1) / kOctets * kOctets;
    const int64_t from = k0 + (int64_t)split * per;
    k1 = (int)min((int64_t)k1, from + per);
    k0 = (int)min((int64_t)k1, from);
  }
  const float* kp = a.k + at(a.ks, b, 0, hk);
  const float* vp = a.v + at(a.vs, b, 0, hk);
  auto add = [&](int j, const float (&x)[R], const float (&v)[F]) {      // key j, its scores and value
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (j >= lo[r] && j < hi[r] && j < k1) {            // uniform in the octet
        if (x[r] > top[r]) {
          const float c = weight(top[r], x[r]);
          sum[r] *= c;
#pragma unroll
          for (int e = 0; e < F; ++e) acc[r][e] *= c;
          top[r] = x[r];
        }
        const float p = weight(x[r], top[r]);
        sum[r] += p;
#pragma unroll
        for (int e = 0; e < F; ++e) acc[r][e] = fmaf(p, v[e], acc[r][e]);
      }
  };
  if constexpr (VEC) {
    // Two keys an octet at a time, two such steps ahead of their use in shared memory.  A
    // thread copies just what it reads itself, so nothing but its own copies is waited for.
    extern __shared__ float4 ring[];
    auto place = [&](int step, int u, int value) {
      return ring + ((step % kAhead * 2 + u) * 2 + value) * NV * (32 * kWarps) + threadIdx.x;
    };
    auto fetch = [&](int step) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t j = min(k0 + (step * 2 + u) * kOctets + oct, k1 - 1);
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          const int f = (c * 8 + lane) * 4, bytes = f < a.dim ? 16 : 0;    // 0: zeros are written
          copy_async(place(step, u, 0) + c * 32 * kWarps, kp + j * a.ks[1] + (bytes ? f : 0), bytes);
          copy_async(place(step, u, 1) + c * 32 * kWarps, vp + j * a.vs[1] + (bytes ? f : 0), bytes);
        }
      }
    };
    auto read = [&](float (&x)[F], const float4* from) {
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const float4 v = from[c * 32 * kWarps];
        x[4 * c] = v.x; x[4 * c + 1] = v.y; x[4 * c + 2] = v.z; x[4 * c + 3] = v.w;
      }
    };
    const int steps = k0 < k1 ? (k1 - k0 + 2 * kOctets - 1) / (2 * kOctets) : 0;
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i) {
      if (i < steps) fetch(i);
      copy_commit();
    }
    for (int i = 0; i < steps; ++i) {
      if (i + kAhead - 1 < steps) fetch(i + kAhead - 1);
      copy_commit();
      copy_wait<kAhead - 1>();
      float x[2][R], k[F];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        read(k, place(i, u, 0));
#pragma unroll
        for (int r = 0; r < R; ++r) x[u][r] = octet_sum(dot(q[r], k)) * scale;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        read(k, place(i, u, 1));
        add(k0 + (i * 2 + u) * kOctets + oct, x[u], k);
      }
    }
  } else {
    for (int base = k0; base < k1; base += kOctets) {
      const int j = min(base + oct, k1 - 1);
      float k[F], v[F], x[R];
      load_row<NV, VEC>(k, kp + (int64_t)j * a.ks[1], lane, a.dim);
      load_row<NV, VEC>(v, vp + (int64_t)j * a.vs[1], lane, a.dim);
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = octet_sum(dot(q[r], k)) * scale;
      add(base + oct, x, v);
    }
  }
  // join the octets of a warp, then the warps
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {
      const float t = __shfl_xor_sync(kFull, top[r], o), both = fmaxf(top[r], t);
      const float mine = weight(top[r], both), other = weight(t, both);
      sum[r] = sum[r] * mine + __shfl_xor_sync(kFull, sum[r], o) * other;
#pragma unroll
      for (int e = 0; e < F; ++e) acc[r][e] = acc[r][e] * mine + __shfl_xor_sync(kFull, acc[r][e], o) * other;
      top[r] = both;
    }
    if ((threadIdx.x & 31) < 8) {
#pragma unroll
      for (int e = 0; e < F; ++e) sh[warp][r][((e >> 2) * 8 + lane) * 4 + (e & 3)] = acc[r][e];
      sh[warp][r][32 * NV] = top[r];
      sh[warp][r][32 * NV + 1] = sum[r];
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < R * a.dim; t += 32 * kWarps) {
    const int r = t / a.dim, f = t - r * a.dim, row = gi * R + r;
    if (row >= rows) continue;
    float best = -INFINITY, s = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) best = fmaxf(best, sh[w][r][32 * NV]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float c = weight(sh[w][r][32 * NV], best);
      s += sh[w][r][32 * NV + 1] * c;
      o += sh[w][r][f] * c;
    }
    if (splits == 1) {
      store_row(a, b, RowAt(a, hk, row), f, o, best, s);
    } else {
      float* rec = record(part, a, (int64_t)bh * rows + row, splits, split);
      rec[f] = o;
      if (f == 0) {
        rec[a.dim] = best;
        rec[a.dim + 1] = s;
      }
    }
  }
}

// A block takes one item, or with `stats` items in turn: most heads then belong to the
// tensor cores, and passing over them is cheaper than a block for each.
template <int NV, bool VEC, int R>
__global__ void __launch_bounds__(32 * kWarps) k_attn_rows(const __grid_constant__ AttnArgs a, int groups, int splits,
                                                           float* part, int items) {
  __shared__ float sh[kWarps][R][32 * NV + 2];
  pdl_entry();
  if (a.any && !*a.any) return;
  for (int i = blockIdx.x; i < items; i += gridDim.x) {
    rows_forward<NV, VEC, R>(a, i, groups, splits, part, sh);
    __syncthreads();
  }
}

// joins a row's splits in order, a block per row
__global__ void __launch_bounds__(128) k_attn_join(const __grid_constant__ AttnArgs a, int splits, float* part,
                                                   bool tensor) {
  __shared__ float share[kMostSplits], best, sum;
  pdl_entry();
  const int rows = a.q_len * a.group;
  const int64_t row = blockIdx.x;
  const int bh = (int)(row / rows);
  if (a.stats && head_splits(a.stats[bh], a.scale, a.dim) != tensor) return;
  const float* rec = record(part, a, row, splits, 0);
  const int step = a.dim + 2;
  if (threadIdx.x < 32) {
    float t[kMostSplits / 32], m = -INFINITY, s = 0.f;
#pragma unroll
    for (int u = 0; u < kMostSplits / 32; ++u) {
      const int i = threadIdx.x + 32 * u;
      t[u] = i < splits ? rec[i * step + a.dim] : -INFINITY;
      m = fmaxf(m, t[u]);
    }
    m = warp_max_f(m);
#pragma unroll
    for (int u = 0; u < kMostSplits / 32; ++u) {
      const int i = threadIdx.x + 32 * u;
      if (i >= splits) continue;
      share[i] = weight(t[u], m);
      s = fmaf(rec[i * step + a.dim + 1], share[i], s);
    }
    s = warp_sum_f(s);
    if (threadIdx.x == 0) {
      best = m;
      sum = s;
    }
  }
  __syncthreads();
  const int f = threadIdx.x;
  if (f >= a.dim) return;
  float o = 0.f;
#pragma unroll 8
  for (int i = 0; i < splits; ++i) o = fmaf(rec[i * step + f], share[i], o);
  store_row(a, bh / a.kv_heads, RowAt(a, bh % a.kv_heads, (int)(row % rows)), f, o, best, sum);
}

// delta = sum_d dout out, an octet per (batch, head, position).  The products are summed as the
// gradients sum dout v: a row that sees one key, whose out is that key's v, gets
// dP - delta = 0 and gradients of exactly 0.
template <int NV, bool VEC>
__global__ void __launch_bounds__(128) k_attn_delta(const __grid_constant__ AttnArgs a) {
  const int64_t rows = (int64_t)a.batch * a.q_heads * a.q_len, row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 3);
  const int64_t r = min(row, rows - 1);
  const int lane = threadIdx.x & 7;
  const int i = (int)(r % a.q_len), b = (int)(r / a.q_len / a.q_heads), h = (int)(r / a.q_len % a.q_heads);
  const bool in = row < rows && i < AttnSpan(a, b).m;
  float go[4 * NV] = {}, o[4 * NV] = {};
  if (in) {
    load_row<NV, VEC>(go, a.dout + at(a.os, b, i, h), lane, a.dim);
    load_row<NV, VEC>(o, a.out + at(a.os, b, i, h), lane, a.dim);
  }
  const float s = octet_sum(dot(go, o));
  if (row < rows && lane == 0)
    a.delta[((int64_t)b * a.kv_heads + h / a.group) * padded_rows(a) + (int64_t)i * a.group + h % a.group] = s;
}

// sums x over the octets of a block into sh, then calls store(feature, total)
template <int NV, typename Store>
DCT_DEV void join_sums(float (&x)[4 * NV], float (&sh)[kWarps][32 * NV], int dim, Store store) {
  const int lane = threadIdx.x & 7, warp = threadIdx.x >> 5;
#pragma unroll
  for (int e = 0; e < 4 * NV; ++e) {
    x[e] += __shfl_xor_sync(kFull, x[e], 8);
    x[e] += __shfl_xor_sync(kFull, x[e], 16);
  }
  __syncthreads();
  if ((threadIdx.x & 31) < 8) {
#pragma unroll
    for (int e = 0; e < 4 * NV; ++e) sh[warp][((e >> 2) * 8 + lane) * 4 + (e & 3)] = x[e];
  }
  __syncthreads();
  for (int f = threadIdx.x; f < dim; f += 32 * kWarps) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += sh[w][f];
    store(f, s);
  }
}

// dq of R rows: an octet per key
template <int NV, bool VEC, int R>
DCT_DEV void rows_dq(const AttnArgs& a, int item, int groups, float (&sh)[kWarps][32 * NV]) {
  constexpr int F = 4 * NV;
  const int lane = threadIdx.x & 7, oct = threadIdx.x >> 3;
  const int gi = item % groups, bh = item / groups;
  const int b = bh / a.kv_heads, hk = bh % a.kv_heads, rows = a.q_len * a.group;
  if (a.stats && head_splits(a.stats[bh], a.scale, a.dim)) return;
  const AttnSpan span(a, b);
  const float scale = a.scale * kLog2e;
  float q[R][F], go[R][F], dq[R][F], lse[R], delta[R];
  int lo[R], hi[R], k0 = INT_MAX, k1 = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = gi * R + r;
    const RowAt w(a, hk, row);
    lo[r] = hi[r] = 0;
#pragma unroll
    for (int e = 0; e < F; ++e) q[r][e] = go[r][e] = dq[r][e] = 0.f;
    if (row < rows && w.i < span.m) {
      const int64_t s = ((int64_t)b * a.q_heads + w.h) * a.q_len + w.i;
      lse[r] = a.lse[s] * kLog2e;
      delta[r] = a.delta[(int64_t)bh * padded_rows(a) + row];
      if (lse[r] == -INFINITY) continue;                    // the row sees nothing
      lo[r] = span.lo(a, w.i);
      hi[r] = span.hi(a, w.i);
      if (lo[r] < hi[r]) {
        k0 = min(k0, lo[r]);
        k1 = max(k1, hi[r]);
      }
      load_row<NV, VEC>(q[r], a.q + at(a.qs, b, w.i, w.h), lane, a.dim);
      load_row<NV, VEC>(go[r], a.dout + at(a.os, b, w.i, w.h), lane, a.dim);
    }
  }
  const float* kp = a.k + at(a.ks, b, 0, hk);
  const float* vp = a.v + at(a.vs, b, 0, hk);
  for (int base = k0; base < k1; base += kOctets) {
    const int j = base + oct, jj = min(j, k1 - 1);
    float k[F], v[F];
    load_row<NV, VEC>(k, kp + (int64_t)jj * a.ks[1], lane, a.dim);
    load_row<NV, VEC>(v, vp + (int64_t)jj * a.vs[1], lane, a.dim);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float x = octet_sum(dot(q[r], k)) * scale, dp = octet_sum(dot(go[r], v));
      if (j >= lo[r] && j < hi[r]) {
        const float ds = exp2f(x - lse[r]) * (dp - delta[r]) * a.scale;
#pragma unroll
        for (int e = 0; e < F; ++e) dq[r][e] = fmaf(ds, k[e], dq[r][e]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = gi * R + r;
    const RowAt w(a, hk, row);
    const int64_t o = at(a.dqs, b, w.i, w.h);
    join_sums<NV>(dq[r], sh, a.dim, [&](int f, float s) {
      if (row < rows) a.dq[o + f] = s;
    });
  }
}

// dk and dv of R keys: an octet per row
template <int NV, bool VEC, int R>
DCT_DEV void rows_dkv(const AttnArgs& a, int item, int groups, float (&sh)[kWarps][32 * NV]) {
  constexpr int F = 4 * NV;
  const int lane = threadIdx.x & 7, oct = threadIdx.x >> 3;
  const int gi = item % groups, bh = item / groups;
  const int b = bh / a.kv_heads, hk = bh % a.kv_heads;
  if (a.stats && head_splits(a.stats[bh], a.scale, a.dim)) return;
  const AttnSpan span(a, b);
  const float scale = a.scale * kLog2e;
  float k[R][F], v[R][F], dk[R][F], dv[R][F];
  int lo[R], hi[R], r0 = INT_MAX, r1 = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = gi * R + r;
    lo[r] = hi[r] = 0;
#pragma unroll
    for (int e = 0; e < F; ++e) k[r][e] = v[r][e] = dk[r][e] = dv[r][e] = 0.f;
    if (j < span.n) {
      lo[r] = span.first(a, j) * a.group;
      hi[r] = span.last(a, j) * a.group;
      if (lo[r] < hi[r]) {
        r0 = min(r0, lo[r]);
        r1 = max(r1, hi[r]);
      }
      load_row<NV, VEC>(k[r], a.k + at(a.ks, b, j, hk), lane, a.dim);
      load_row<NV, VEC>(v[r], a.v + at(a.vs, b, j, hk), lane, a.dim);
    }
  }
  for (int base = r0; base < r1; base += kOctets) {
    const int row = base + oct;
    const RowAt w(a, hk, min(row, r1 - 1));
    const int64_t s = ((int64_t)b * a.q_heads + w.h) * a.q_len + w.i;
    const float lse = a.lse[s] * kLog2e, delta = a.delta[(int64_t)bh * padded_rows(a) + min(row, r1 - 1)];
    float q[F], go[F];
    load_row<NV, VEC>(q, a.q + at(a.qs, b, w.i, w.h), lane, a.dim);
    load_row<NV, VEC>(go, a.dout + at(a.os, b, w.i, w.h), lane, a.dim);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float x = octet_sum(dot(q, k[r])) * scale, dp = octet_sum(dot(go, v[r]));
      if (row >= lo[r] && row < hi[r] && lse != -INFINITY) {
        const float p = exp2f(x - lse), ds = p * (dp - delta) * a.scale;
#pragma unroll
        for (int e = 0; e < F; ++e) {
          dv[r][e] = fmaf(p, go[e], dv[r][e]);
          dk[r][e] = fmaf(ds, q[e], dk[r][e]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = gi * R + r;
    const int64_t ok = at(a.dks, b, j, hk), ov = at(a.dvs, b, j, hk);
    join_sums<NV>(dk[r], sh, a.dim, [&](int f, float s) {
      if (j < a.kv_len) a.dk[ok + f] = s;
    });
    join_sums<NV>(dv[r], sh, a.dim, [&](int f, float s) {
      if (j < a.kv_len) a.dv[ov + f] = s;
    });
  }
}

template <int NV, bool VEC, int R>
__global__ void __launch_bounds__(32 * kWarps) k_attn_rows_backward(const __grid_constant__ AttnArgs a, int groups_q,
                                                                    int items_q, int groups_k, int items_k) {
  __shared__ float sh[kWarps][32 * NV];
  pdl_entry();
  if (a.any && !*a.any) return;
  for (int64_t i = blockIdx.x; i < (int64_t)items_q + items_k; i += gridDim.x) {
    if (i < items_q) rows_dq<NV, VEC, R>(a, (int)i, groups_q, sh);
    else rows_dkv<NV, VEC, R>(a, (int)(i - items_q), groups_k, sh);
    __syncthreads();
  }
}

unsigned blocks_for(const AttnArgs& a, int64_t items) {
  return (unsigned)(a.stats ? std::min<int64_t>(items, 8ll * dev_info().sm_count) : std::min<int64_t>(items, INT_MAX));
}

bool aligned(const float* p, const int64_t* s) {
  return aligned16_h(p) && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
}

// calls f(NV, VEC) as compile-time constants
template <typename F>
cudaError_t by_width(int dim, bool vec, F f) {
  const int nv = (dim + 31) / 32;
#define DCT_NV(n)                                                                                     \
  case n:                                                                                             \
    return vec ? f(std::integral_constant<int, n>{}, std::true_type{})                                \
               : f(std::integral_constant<int, n>{}, std::false_type{});
  switch (nv) { DCT_NV(1) DCT_NV(2) DCT_NV(3) DCT_NV(4) }
#undef DCT_NV
  return cudaErrorInvalidValue;
}

int rows_per_block(const AttnArgs& a) {
  const int64_t rows = (int64_t)a.q_len * a.group;
  return rows >= 4 ? 4 : rows >= 2 ? 2 : 1;
}

// splits of the keys: about eight blocks an SM, none shorter than 128 keys
int rows_splits(const AttnArgs& a) {
  const int R = rows_per_block(a);
  const int64_t blocks = (int64_t)a.batch * a.kv_heads * (((int64_t)a.q_len * a.group + R - 1) / R);
  if (!blocks) return 1;
  const int64_t want = (8ll * dev_info().sm_count + blocks - 1) / blocks, most = (a.kv_len + 127) / 128;
  return (int)std::max<int64_t>(1, std::min<int64_t>(kMostSplits, std::min(want, most)));
}

}  // namespace

size_t attn_rows_ws_bytes(const AttnArgs& a) {
  const int splits = rows_splits(a);
  return splits == 1 ? 0 : sizeof(float) * (size_t)a.batch * a.q_heads * a.q_len * splits * (a.dim + 2);
}

cudaError_t launch_attn_rows_forward(const AttnArgs& a, void* ws, cudaStream_t st) {
  const int R = rows_per_block(a), splits = rows_splits(a);
  const int64_t rows = (int64_t)a.q_len * a.group, groups = (rows + R - 1) / R;
  const int64_t blocks = groups * splits * a.batch * a.kv_heads;
  if (!blocks) return cudaSuccess;
  if (blocks > INT_MAX) return cudaErrorInvalidConfiguration;
  const bool vec = a.dim % 4 == 0 && aligned(a.q, a.qs) && aligned(a.k, a.ks) && aligned(a.v, a.vs);
  float* part = static_cast<float*>(ws);
  cudaError_t e = by_width(a.dim, vec, [&](auto nv, auto v) {
    constexpr int NV = decltype(nv)::value;
    constexpr bool V = decltype(v)::value;
    const unsigned n = blocks_for(a, blocks);
    const int items = (int)blocks, g = (int)groups;
    const auto kernel = R == 4 ? k_attn_rows<NV, V, 4> : R == 2 ? k_attn_rows<NV, V, 2> : k_attn_rows<NV, V, 1>;
    const size_t smem = V ? sizeof(float4) * kAhead * 4 * NV * 32 * kWarps : 0;      // 96 KB at 128 features
    const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (set != cudaSuccess) return set;
    return launch_pdl(kernel, dim3(n), dim3(32 * kWarps), smem, st, a, g, splits, part, items);
  });
  if (e != cudaSuccess || splits == 1) return e;
  return launch_attn_join(a, splits, part, false, st);
}

cudaError_t launch_attn_join(const AttnArgs& a, int splits, float* part, bool tensor, cudaStream_t st) {
  return launch_pdl(k_attn_join, dim3((unsigned)((int64_t)a.batch * a.q_heads * a.q_len)), dim3(128), 0, st, a, splits,
                    part, tensor);
}

cudaError_t launch_attn_delta(const AttnArgs& a, cudaStream_t st) {
  const int64_t rows = (int64_t)a.batch * a.q_heads * a.q_len;
  if (!rows) return cudaSuccess;
  return by_width(a.dim, a.dim % 4 == 0 && aligned(a.dout, a.os) && aligned(a.out, a.os), [&](auto nv, auto v) {
    k_attn_delta<decltype(nv)::value, decltype(v)::value><<<(unsigned)((rows + 15) / 16), 128, 0, st>>>(a);
    return cudaGetLastError();
  });
}

cudaError_t launch_attn_rows_backward(const AttnArgs& a, cudaStream_t st) {
  constexpr int R = 2;
  const bool vec = a.dim % 4 == 0 && aligned(a.q, a.qs) && aligned(a.k, a.ks) && aligned(a.v, a.vs) &&
                   aligned(a.dout, a.os);
  const int64_t gq = ((int64_t)a.q_len * a.group + R - 1) / R, gk = ((int64_t)a.kv_len + R - 1) / R;
  const int64_t heads = (int64_t)a.batch * a.kv_heads;
  if (gq * heads > INT_MAX || gk * heads > INT_MAX) return cudaErrorInvalidConfiguration;
  return by_width(a.dim, vec, [&](auto nv, auto v) {
    constexpr int NV = decltype(nv)::value;
    constexpr bool V = decltype(v)::value;
    const int nq = (int)(gq * heads), nk = (int)(gk * heads);
    if (!(nq + (int64_t)nk)) return cudaSuccess;
    return launch_pdl(k_attn_rows_backward<NV, V, R>, dim3(blocks_for(a, nq + (int64_t)nk)), dim3(32 * kWarps), 0, st,
                      a, (int)gq, nq, (int)gk, nk);
  });
}

}  // namespace dct
