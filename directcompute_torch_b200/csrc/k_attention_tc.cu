// Attention on the fifth-generation tensor cores at float32 accuracy.
//
// A pass over the operands writes them as split float16 tiles of 128 rows, each with a power
// of two of its own (k_attn_split; arithmetic and layout in dct_umma.cuh), and the products
// run on those: three matrix instructions for each product of float32 numbers, so the bound
// is a third of the float16 rate, about 540 TFLOP/s.
//
// A tile is [64 features][hi, lo][128 rows][64 float16], 32 KB for every 64 features, so
// one bulk copy brings it and it serves as either operand: with its features as the
// contraction (scores) or with its rows (the products with P, dS).
//
// Heads that the split cannot hold (infinities, NaN, rows or features of very different size)
// take the kernels of k_attention.cu, which pick them by the same test on the device.
#include <limits.h>

#include <algorithm>

#include "dct_attn.cuh"
#include "dct_umma.cuh"

namespace dct {
namespace {

constexpr int kTile = 128;
constexpr uint32_t kBlockBytes = 2 * kTile * 128;      // 64 features of a tile, hi and lo

// 2^x by the hardware (2 ulp; results below 2^-126 are 0)
DCT_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^e for -126 <= e <= 127, clamped to that.  A tile's exponent is -30 to 74 and the sum of two
// up to 148: harmless for scores (2^-126 of a number below 2^37 is as good as nothing in an
// exponent), but dP and delta stay in units of dout's tile, and sums are scaled back in two steps.
DCT_DEV float pow2(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }
DCT_DEV uint32_t lane_bits(int warp) { return (uint32_t)(warp & 3) * 32u << 16; }

struct Tiles {
  uint8_t* p[4];               // q, k, v, dout
  AttnTile* info[4];           // [heads][tiles]
  AttnStats* stats;            // [heads]
  uint32_t* any;               // set where a head does not take the tensor cores
  float *lse2, *delta;         // [heads][padded rows], backward: log-sums in log2 units, sum dout out in
                               // units of dout's tile
  int64_t tiles[4];            // of a head
};

// the rows of operand t of a head that are valid, and one of them
DCT_DEV int rows_of(const AttnArgs& a, const AttnSpan& s, int t) { return t == 1 || t == 2 ? s.n : s.m * a.group; }
DCT_DEV const float* row_of(const AttnArgs& a, int t, int b, int hk, int r) {
  if (t == 1) return a.k + at(a.ks, b, r, hk);
  if (t == 2) return a.v + at(a.vs, b, r, hk);
  const RowAt w(a, hk, r);
  return t == 0 ? a.q + at(a.qs, b, w.i, w.h) : a.dout + at(a.os, b, w.i, w.h);
}

// features [first, first + N) of a row, as far as it has them
template <int N>
DCT_DEV void store_features(float* row, int first, int dim, bool vec, const float (&x)[N]) {
  if (vec) {
#pragma unroll
    for (int e = 0; e < N; e += 4)
      if (first + e < dim)
        *reinterpret_cast<float4*>(row + first + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (first + e < dim) row[first + e] = x[e];
  }
}

// ---------------------------------------------------------------------------
// splitting
// ---------------------------------------------------------------------------
// blocks [tensor][head][tile] of 512 threads; a thread takes 8 features of every 32nd (64th)
// row and holds them while the block finds the tile's magnitude, so each operand is read
// once.  With dout come delta = sum dout out and the log-sums.  Bound by memory: 8 bytes a
// feature (12 for dout).  Three blocks an SM for 64 features: training with a window 196 us with
// two, 191.5 with three.
template <int BLOCKS>
__global__ void __launch_bounds__(512, BLOCKS == 1 ? 3 : 2) k_attn_split(const __grid_constant__ AttnArgs a,
                                                                         const __grid_constant__ Tiles w, int tq,
                                                                         int tk, bool vec) {
  constexpr int kGroups = 8 * BLOCKS, kStep = 512 / kGroups, kPasses = kTile / kStep;
  __shared__ uint32_t sh[2];
  __shared__ uint2 sizes[16][kGroups];             // exponents of 8 features' largest |x|, a warp's rows
  touch(a);
  touch(w);
  pdl_entry();
  const int heads = a.batch * a.kv_heads;
  int x = blockIdx.x, t = 0;
  for (; t < 3; ++t) {                             // q, k, v, dout in turn
    const int n = heads * (t == 0 ? tq : tk);
    if (x < n) break;
    x -= n;
  }
  const int per = t == 1 || t == 2 ? tk : tq, bh = x / per, tile = x - bh * per;
  const int g = threadIdx.x % kGroups, row0 = threadIdx.x / kGroups, b = bh / a.kv_heads, hk = bh % a.kv_heads;
  const AttnSpan span(a, b);
  const int rows = rows_of(a, span, t);
  if (tile * kTile >= rows && t != 3) return;      // nothing reads it (dout's log-sums are read by whole tiles)
  // operands whose features are a result's: v in out, q in dk, k in dq, dout in dv
  const bool by_feature = a.dout ? t != 2 : t == 2;
  if (threadIdx.x < 2) sh[threadIdx.x] = 0;
  __syncthreads();
  float v[kPasses][8], delta[kPasses];
  uint32_t top = 0, low = 0;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int r = tile * kTile + row0 + p * kStep;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[p][e] = 0.f;
    if (r >= rows) continue;
    const float* src = row_of(a, t, b, hk, r) + g * 8;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      if (vec) {
        if (g * 8 + e < a.dim) *reinterpret_cast<float4*>(v[p] + e) = *reinterpret_cast<const float4*>(src + e);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (g * 8 + e + q < a.dim) v[p][e + q] = src[e + q];
      }
    }
  }
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[p][e]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < kGroups; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    top = max(top, m);
    if (m) low = max(low, ~m);
    if (t == 3) {
      float d = 0.f;
      const int r = tile * kTile + row0 + p * kStep;
      if (r < rows) {
        const RowAt q(a, hk, r);
        const float* o = a.out + at(a.os, b, q.i, q.h) + g * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (g * 8 + e < a.dim) d = fmaf(v[p][e], o[e], d);
      }
#pragma unroll
      for (int o = 1; o < kGroups; o <<= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
      if (g == 0) {
        const int64_t at_row = (int64_t)bh * padded_rows(a) + r;
        float l = INFINITY;                        // a row that sees nothing: P = 2^(s - inf) = 0
        if (r < rows) {
          const RowAt q(a, hk, r);
          l = a.lse[((int64_t)b * a.q_heads + q.h) * a.q_len + q.i] * kLog2e;
          if (l == -INFINITY) l = INFINITY;
        }
        w.lse2[at_row] = l;
        a.delta[at_row] = delta[p] = d;
      }
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (by_feature) {
    uint32_t c[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t m = 0;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) m = max(m, __float_as_uint(v[p][e]) & 0x7fffffffu);
      c[e >> 2] |= max(m >> 23, min(m, 1u)) << 8 * (e & 3);                // 0: nothing but zeros
    }
#pragma unroll
    for (int o = kGroups; o < 32; o <<= 1) {
      c[0] = __vmaxu4(c[0], __shfl_xor_sync(0xffffffffu, c[0], o));
      c[1] = __vmaxu4(c[1], __shfl_xor_sync(0xffffffffu, c[1], o));
    }
    if (lane < kGroups) sizes[warp][lane] = make_uint2(c[0], c[1]);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_max_sync(0xffffffffu, low);
  if (lane == 0) {
    atomicMax(&sh[0], top);
    atomicMax(&sh[1], low);
  }
  __syncthreads();
  top = sh[0];
  const bool splits = tile_splits(top, ~sh[1]);
  const int e = top && splits ? 14 - ((int)(top >> 23) - 127) : 0;
  if (threadIdx.x == 0) {
    w.info[t][bh * w.tiles[t] + tile] = AttnTile{e};
    if (t == 0) atomicMax(&w.stats[bh].top_q, top);
    if (t == 1) atomicMax(&w.stats[bh].top_k, top);
    if (t == 2 && top) {
      atomicMax(&w.stats[bh].top_v, top);
      atomicMax(&w.stats[bh].low_v, ~top);
    }
    if (!splits) w.stats[bh].bad = 1;
  }
  if (by_feature && warp == 1 && lane < 2 * kGroups) {     // 4 features a lane
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) c = __vmaxu4(c, lane & 1 ? sizes[i][lane >> 1].y : sizes[i][lane >> 1].x);
#pragma unroll
    for (int e = 0; e < 32; e += 8)
      if ((c >> e & 255) && (c >> e & 255) + kApart < top >> 23) w.stats[bh].bad = 1;
  }
  if (!splits) return;
  const float f = pow2(e);
  if (t == 3 && g == 0) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
      w.delta[(int64_t)bh * padded_rows(a) + tile * kTile + row0 + p * kStep] = delta[p] * f;
  }
  if (g >= (a.dim + 15) / 16 * 2) return;          // features that no product reads
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) split2(v[p][2 * q] * f, v[p][2 * q + 1] * f, h[q], l[q]);
    uint8_t* o = w.p[t] + ((bh * w.tiles[t] + tile) * BLOCKS + g / 8) * (int64_t)kBlockBytes +
                 chunk_at(row0 + p * kStep, g % 8);
    *reinterpret_cast<uint4*>(o) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(o + kBlockBytes / 2) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// ---------------------------------------------------------------------------
// what the three kernels share
// ---------------------------------------------------------------------------
// 16 warps compute, four threads a row of 128 (warp w holds rows 32 (w & 3) .. and quarter
// w >> 2 of the columns); warp 17 issues the matrix instructions, warps 16 and 18 load, each
// its own ring of slots: the two inner operands are used up in different orders, and in one
// ring each would wait for the other's slots.  Four warps a scheduler hide the latencies
// that one phase after the other has.  The operand that rests lies in tensor memory where
// there is room; the inner side comes in half tiles of 64 rows where there is not enough
// shared memory for whole ones (a matrix instruction 64 columns wide takes 45 or 48 cycles,
// one of 128 takes 64: measured).
constexpr int kSoft = 16;
constexpr int kThreads = 32 * (kSoft + 4);
constexpr int kHalf = 64;

// Registers move from the four helping warps (one idle) to the computing ones: 640 threads
// start with 96 each, 61440 in all, of which 60416 are taken.  (Inside the roles' branches,
// where the compiler sees which code has how many.)
constexpr int kUpRegs = 104, kDownRegs = 56;
constexpr int kRegs = 32 * (kSoft * kUpRegs + 4 * kDownRegs);
DCT_DEV void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kUpRegs)); }
DCT_DEV void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kDownRegs)); }

template <int BLOCKS>
struct Sizes {
  static constexpr int kD = 64 * BLOCKS, kF = kD / 4;              // features, of them a thread's
  static constexpr uint32_t kTileBytes = BLOCKS * kBlockBytes, kSlotBytes = kTileBytes / 2;
};

// half tile `h` (64 rows) of operand t: [64 features][hi, lo][64 rows][64 float16]
template <int BLOCKS>
DCT_DEV void load_half(const Tiles& w, int bh, int t, int64_t h, uint8_t* to, uint64_t* bar) {
  const uint8_t* from = w.p[t] + (bh * w.tiles[t] + h / 2) * (int64_t)(BLOCKS * kBlockBytes) + (h & 1) * kChunkBytes;
#pragma unroll
  for (int i = 0; i < 2 * BLOCKS; ++i) bulk_load(to + i * kChunkBytes, from + i * 2 * kChunkBytes, kChunkBytes, bar);
}
// a whole tile as it lies
template <int BLOCKS>
DCT_DEV void load_tile(const Tiles& w, int bh, int t, int64_t tile, uint8_t* to, uint64_t* bar) {
  const uint8_t* from = w.p[t] + (bh * w.tiles[t] + tile) * (int64_t)(BLOCKS * kBlockBytes);
#pragma unroll
  for (uint32_t o = 0; o < BLOCKS * kBlockBytes; o += kBlockBytes / 2)
    bulk_load(to + o, from + o, kBlockBytes / 2, bar);
}

// A thread's quarter of its row of a whole tile into tensor memory as an operand: columns of
// hi, then of lo.
template <int BLOCKS>
DCT_DEV void tile_to_tmem(const uint8_t* tile, uint32_t addr, int warp, int row) {
  constexpr int kGroups = 2 * BLOCKS;              // of 8 features, a thread's
  const int g0 = (warp >> 2) * kGroups;
#pragma unroll
  for (int low = 0; low < 2; ++low) {
    uint32_t r[4 * kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int f = g0 + g;
      const uint4 v = *reinterpret_cast<const uint4*>(tile + (f >> 3) * kBlockBytes + low * (kBlockBytes / 2) +
                                                      chunk_at(row, f & 7));
      r[4 * g] = v.x; r[4 * g + 1] = v.y; r[4 * g + 2] = v.z; r[4 * g + 3] = v.w;
    }
    tmem_store(addr + lane_bits(warp) + low * 32 * BLOCKS + g0 * 4, r);
  }
}

// A ring of slots: loads fill them in turn, matrix instructions empty them.
template <int N>
struct Ring {
  uint64_t full[N], empty[N];
  DCT_DEV void init() {
    for (int s = 0; s < N; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
  }
  // fills `count` slots: load(number, slot, barrier)
  template <typename Wait, typename Load>
  DCT_DEV void fill(int count, uint32_t bytes, Wait& wait, Load load) {
    int it = 0;
    for (; it < count; ++it) {
      if (!wait(&empty[it % N], (it / N) ^ 1)) break;
      mbar_arrive_expect_tx(&full[it % N], bytes);
      load(it, it % N, &full[it % N]);
    }
    // every copy has landed before the block ends
    for (int u = max(0, it - N); u < it; ++u) mbar_wait(&full[u % N], (u / N) & 1, wait.err);
  }
  template <typename Wait>
  DCT_DEV bool ready(int it, Wait& wait) { return wait(&full[it % N], it / N); }
  DCT_DEV void release(int it) { umma_commit(&empty[it % N]); }
};

// D = A B^T over the features: A a whole tile in shared memory, B a half tile.  The small
// products come first: every matrix instruction rounds its sum toward zero.
// `steps`: 16 features each; what lies behind is neither written nor read.  (FULL: a constant
// number of them, 3% faster at 128 features than asking for each step.)
template <int BLOCKS>
DCT_DEV void mma_features_ss(uint32_t d, uint64_t a, uint64_t b, int steps) {
  constexpr uint32_t id = umma_idesc(kTile, kHalf, false, false);
  constexpr uint64_t lo_a = kBlockBytes / 32, lo_b = kChunkBytes / 16;
  auto sa = [](int c) { return (uint64_t)((c >> 2) * (kBlockBytes / 16) + (c & 3) * 2); };
  auto sb = [](int c) { return (uint64_t)((c >> 2) * (2 * kChunkBytes / 16) + (c & 3) * 2); };
#pragma unroll
  for (int c = 0; c < 4 * BLOCKS; ++c) {
    if (c >= steps) break;
    umma(d, a + lo_a + sa(c), b + sb(c), id, c != 0);
    umma(d, a + sa(c), b + lo_b + sb(c), id, true);
  }
#pragma unroll
  for (int c = 0; c < 4 * BLOCKS; ++c)
    if (c < steps) umma(d, a + sa(c), b + sb(c), id, true);
}
// the same with A in tensor memory, B a tile of ROWS rows
template <int BLOCKS, int ROWS>
DCT_DEV void mma_features_ts(uint32_t d, uint32_t a, uint64_t b, int steps) {
  constexpr uint32_t id = umma_idesc(kTile, ROWS, false, false);
  constexpr uint64_t lo_b = ROWS * 128 / 16;
  auto sb = [](int c) { return (uint64_t)((c >> 2) * (2 * ROWS * 128 / 16) + (c & 3) * 2); };
#pragma unroll
  for (int c = 0; c < 4 * BLOCKS; ++c) {
    if (c >= steps) break;
    umma_ts(d, a + 32 * BLOCKS + 8 * c, b + sb(c), id, c != 0);
    umma_ts(d, a + 8 * c, b + lo_b + sb(c), id, true);
  }
#pragma unroll
  for (int c = 0; c < 4 * BLOCKS; ++c)
    if (c < steps) umma_ts(d, a + 8 * c, b + sb(c), id, true);
}
// D (+)= A B over 64 rows: A in tensor memory, for each Q rows Q/2 columns of hi and Q/2 of
// lo (store_operand); B a half tile with its rows as the contraction
template <int BLOCKS, int Q>
DCT_DEV void mma_rows(uint32_t d, uint32_t a, uint64_t b, bool add, int steps) {
  const uint32_t id = umma_idesc(kTile, 16 * steps, false, true);
  constexpr uint64_t lo_b = kChunkBytes / 16;
  auto sa = [](int c) { return (uint32_t)(16 * c / Q * Q + 16 * c % Q / 2); };
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    umma_ts(d, a + Q / 2 + sa(c), b + c * 128, id, add || c != 0);
    umma_ts(d, a + sa(c), b + lo_b + c * 128, id, true);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) umma_ts(d, a + sa(c), b + c * 128, id, true);
}

// Q values as an operand's columns
template <int Q>
DCT_DEV void store_operand(uint32_t addr, const float (&x)[Q]) {
  uint32_t h[Q / 2], l[Q / 2];
#pragma unroll
  for (int e = 0; e < Q / 2; ++e) split2(x[2 * e], x[2 * e + 1], h[e], l[e]);
  tmem_store(addr, h);
  tmem_store(addr + Q / 2, l);
}

// a warp's arrival after its accesses to tensor memory
DCT_DEV void arrive_warp(uint64_t* bar) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Bounded waits of one warp or thread.  After one has run out the others are passed over, and
// the loops go on to their ends: whoever still counts on meeting this one must not wait.
struct Waits {
  uint32_t* err;
  bool ok = true;
  DCT_DEV bool operator()(uint64_t* bar, int phase) {
    ok = ok && mbar_wait(bar, phase & 1, err);
    tc_fence_after();
    return ok;
  }
};

// shared memory: tiles first (1024-byte aligned), then the kernel's barriers and vectors
DCT_DEV bool misaligned(const uint8_t* sm, uint32_t* err) {
  if ((smem_addr(sm) & 1023) == 0) return false;
  if (err && threadIdx.x == 0) atomicOr(err, DCT_DEVERR_WAIT_TIMEOUT);
  return true;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// P is held as 2^15 P: a weight is at most 1 (and what a score's rounding adds: 2^0.02 at 2^18),
// and hi + lo reach 2^-40 of its row's largest one so far.  That is a choice: a row whose result
// is made of weights below 2^-17 of its largest has them in fewer bits than float32.
constexpr float kUp = 15.f;

template <int BLOCKS>
struct Forward : Sizes<BLOCKS> {
  static constexpr int kKeys = BLOCKS == 1 ? 3 : 2, kValues = BLOCKS == 1 ? 6 : 3;   // tiles of K, halves of V
  struct Control {
    Ring<kKeys> k;
    Ring<kValues> v;
    uint64_t q_full, s_full[2], p_full[2], o_full, o_empty;
    uint32_t tmem;
    float exch[4][kTile];
  };
  static constexpr uint32_t kV = kKeys * Sizes<BLOCKS>::kTileBytes;          // where the halves of V begin
  static constexpr uint32_t kEnd = kV + kValues * Sizes<BLOCKS>::kSlotBytes;
  static constexpr size_t kSmem = kEnd + sizeof(Control);
};

DCT_DEV void rows_sync(int warp) {                 // the four warps that share rows
  asm volatile("bar.sync %0, 128;" ::"r"(1 + (warp & 3)) : "memory");
}

// One tile of 128 rows of a key head against its keys, 128 at a time: softmax(Q K^T) V with
// the running maximum and sum.  The next scores are formed while the warps work on these;
// each tile's P V is drained into registers, where the outputs are scaled when the maximum
// moves, so no accumulator lives longer than one tile and the tensor cores' rounding toward
// zero does not build up.  P goes back into the scores' place as the product's operand.
template <int BLOCKS, bool FULL>
__global__ void __launch_bounds__(kThreads, 1) k_attn_forward(const __grid_constant__ AttnArgs a,
                                                              const __grid_constant__ Tiles w, int row_tiles,
                                                              int splits, float* part, bool vec_out, uint32_t* err) {
  using S = Forward<BLOCKS>;
  extern __shared__ __align__(1024) uint8_t sm[];
  auto& ctl = *reinterpret_cast<typename S::Control*>(sm + S::kEnd);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (misaligned(sm, err)) return;
  if (threadIdx.x == 0) {
    ctl.k.init();
    ctl.v.init();
    mbar_init(&ctl.q_full, kSoft);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctl.s_full[s], 1);
      mbar_init(&ctl.p_full[s], kSoft);
    }
    mbar_init(&ctl.o_full, 1);
    mbar_init(&ctl.o_empty, kSoft);
    mbar_fence_init();
  }
  if (warp == kSoft + 1) tmem_alloc(&ctl.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // S twice, P V, the operand Q
  const uint32_t tm_s = ctl.tmem, tm_o = tm_s + 256, tm_q = tm_s + 384;
  const int heads = a.batch * a.kv_heads, bh = blockIdx.x % heads, rest = blockIdx.x / heads;
  const int split = rest % splits, tile = row_tiles - 1 - rest / splits;                     // long rows first
  const int b = bh / a.kv_heads, hk = bh % a.kv_heads;
  const int rows = a.q_len * a.group, r0 = tile * kTile;
  const int i0 = r0 / a.group, i_end = (min(r0 + kTile, rows) - 1) / a.group;    // positions of the tile's rows
  touch(a);
  touch(w);
  pdl_entry();
  const AttnStats stats = w.stats[bh];
  const AttnSpan span(a, b);
  const bool splits_head = head_splits(stats, a.scale, a.dim);
  if (!splits_head && threadIdx.x == 0) *w.any = 1;          // work for the float32 kernels
  const int i1 = min(i_end, span.m - 1);
  int t0 = 0, n = 0;
  if (splits_head && i0 < span.m) {
    const int k0 = span.lo(a, i0), k1 = span.hi(a, i1);
    t0 = k0 / kTile;
    int t1 = k1 > k0 ? (k1 + kTile - 1) / kTile : t0;
    if (splits > 1) {
      const int per = (t1 - t0 + splits - 1) / splits;
      const int from = min(t1, t0 + split * per);
      t1 = min(t1, from + per);
      t0 = from;
    }
    n = t1 - t0;
  }
  Waits wait{err};
  const int steps = FULL ? 4 * BLOCKS : (a.dim + 15) / 16;

  if (warp >= kSoft) {
    registers_down();
    if (warp == kSoft) {
      if (elect_one())
        ctl.k.fill(n, S::kTileBytes, wait, [&](int it, int s, uint64_t* bar) {
          load_tile<BLOCKS>(w, bh, 1, t0 + it, sm + s * S::kTileBytes, bar);
        });
    } else if (warp == kSoft + 2) {
      if (elect_one())
        ctl.v.fill(2 * n, S::kSlotBytes, wait, [&](int it, int s, uint64_t* bar) {
          load_half<BLOCKS>(w, bh, 2, 2 * t0 + it, sm + S::kV + s * S::kSlotBytes, bar);
        });
    } else if (warp == kSoft + 1) {
      if (n && elect_one()) {
        wait(&ctl.q_full, 0);
        auto key = [&](int j) { return smem_addr(sm + j % S::kKeys * S::kTileBytes); };
        auto value = [&](int it) { return smem_addr(sm + S::kV + it % S::kValues * S::kSlotBytes); };
        auto scores = [&](int j) {                 // S(j) = Q K(j)^T
          if (!ctl.k.ready(j, wait)) return;
          mma_features_ts<BLOCKS, kTile>(tm_s + (j & 1) * kTile, tm_q, umma_desc(key(j), kChunkBytes, 1024), steps);
          ctl.k.release(j);
          umma_commit(&ctl.s_full[j & 1]);
        };
        scores(0);
        for (int j = 0; j < n && wait.ok; ++j) {
          if (j + 1 < n) scores(j + 1);
          wait(&ctl.p_full[j & 1], j >> 1);
          wait(&ctl.o_empty, j ^ 1);
          for (int h = 0; h < 2; ++h) {
            const int it = 2 * j + h;
            if (!ctl.v.ready(it, wait)) break;
            mma_rows<BLOCKS, 32>(tm_o, tm_s + (j & 1) * kTile + h * kHalf, umma_desc(value(it), 2 * kChunkBytes, 1024),
                                 h, steps);
            ctl.v.release(it);
          }
          umma_commit(&ctl.o_full);
        }
      }
    }
  } else if (splits_head) {
    registers_up();
    const int quarter = warp >> 2, row = (warp & 3) * 32 + lane, r = r0 + row;
    const RowAt at_row(a, hk, min(r, rows - 1));
    const bool in = r < rows && at_row.i < span.m;
    const int lo = in ? span.lo(a, at_row.i) : 0, hi = in ? span.hi(a, at_row.i) : 0;
    const AttnTile *ki = w.info[1] + bh * w.tiles[1] + t0, *vi = w.info[2] + bh * w.tiles[2] + t0;
    const int eq = w.info[0][bh * w.tiles[0] + tile].e;
    const float scale = a.scale * kLog2e, hidden = scale < 0.f ? INFINITY : -INFINITY;
    int ek = n ? ki[0].e : 0, ev = n ? vi[0].e : 0, ev_last = ev;    // of the tile at hand, of the one before
    float o[S::kF], top = -INFINITY, sum = 0.f, scale_o = 1.f;
#pragma unroll
    for (int e = 0; e < S::kF; ++e) o[e] = 0.f;
    if (n) {
      tile_to_tmem<BLOCKS>(w.p[0] + (bh * w.tiles[0] + tile) * (int64_t)S::kTileBytes, tm_q, warp, row);
      tmem_wait_st();
      arrive_warp(&ctl.q_full);
    }
    auto take = [&](int j) {                       // adds P V of tile j
      wait(&ctl.o_full, j);
      uint32_t v[S::kF];
      tmem_load(tm_o + lane_bits(warp) + quarter * S::kF, v);
      tmem_wait_ld();
      arrive_warp(&ctl.o_empty);
#pragma unroll
      for (int e = 0; e < S::kF; ++e) o[e] = fmaf(o[e], scale_o, __uint_as_float(v[e]));
    };
    for (int j = 0; j < n; ++j) {
      const int key = (t0 + j) * kTile + quarter * 32;
      // (f is not 0: a masked score is infinite, and times 0 it would not be)
      const float f = copysignf(fmaxf(fabsf(scale * pow2(-eq - ek)), 1e-36f), scale);
      const int ek_next = j + 1 < n ? ki[j + 1].e : 0, ev_next = j + 1 < n ? vi[j + 1].e : 0;
      wait(&ctl.s_full[j & 1], j >> 1);
      const uint32_t addr = tm_s + lane_bits(warp) + (j & 1) * kTile + quarter * 32;
      uint32_t x[32];
      tmem_load32(addr, x);
      tmem_wait_ld();
      if (__any_sync(0xffffffffu, key < lo || key + 32 > hi)) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (key + e < lo || key + e >= hi) x[e] = __float_as_uint(hidden);
      }
      // the largest of f x: a negative scale turns the order
      float best = __uint_as_float(x[0]);
      if (f >= 0.f) {
#pragma unroll
        for (int e = 1; e < 32; ++e) best = fmaxf(best, __uint_as_float(x[e]));
      } else {
#pragma unroll
        for (int e = 1; e < 32; ++e) best = fminf(best, __uint_as_float(x[e]));
      }
      ctl.exch[quarter][row] = best * f;
      rows_sync(warp);
      float next = fmaxf(fmaxf(ctl.exch[0][row], ctl.exch[1][row]), fmaxf(ctl.exch[2][row], ctl.exch[3][row]));
      rows_sync(warp);
      next = fmaxf(top, next);
      const float base = next == -INFINITY ? 0.f : next;       // nothing seen yet: every weight is 0
      const float move = ex2(top - base), up = kUp - base;
      top = next;
      float p[32], s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        p[e] = ex2(fmaf(__uint_as_float(x[e]), f, up));
        p[e + 1] = ex2(fmaf(__uint_as_float(x[e + 1]), f, up));
        s0 += p[e];
        s1 += p[e + 1];
      }
      store_operand<32>(addr, p);
      sum = fmaf(sum, move, s0 + s1);
      tmem_wait_st();
      arrive_warp(&ctl.p_full[j & 1]);
      if (j) take(j - 1);
      // the outputs are held as 2^ev of the tile that was added last
      scale_o = move * pow2(ev - ev_last);
      ev_last = ev;
      ek = ek_next;
      ev = ev_next;
    }
    if (n) take(n - 1);
    // the four quarters of a row meet
    ctl.exch[quarter][row] = sum;
    rows_sync(warp);
    sum = (ctl.exch[0][row] + ctl.exch[1][row]) + (ctl.exch[2][row] + ctl.exch[3][row]);
    if (wait.ok && r < rows) {
      float back = pow2(-ev_last);
      const float down = exp2f(-kUp);
      if (splits > 1) {
        float* rec = part + (((int64_t)bh * rows + r) * splits + split) * (a.dim + 2);
        back *= down;
#pragma unroll
        for (int e = 0; e < S::kF; ++e)
          if (quarter * S::kF + e < a.dim) rec[quarter * S::kF + e] = o[e] * back;
        if (quarter == 0) {
          rec[a.dim] = top;
          rec[a.dim + 1] = sum * down;
        }
      } else {
        const float inv = sum == 0.f ? 0.f : back / sum;
#pragma unroll
        for (int e = 0; e < S::kF; ++e) o[e] *= inv;
        store_features<S::kF>(a.out + at(a.os, b, at_row.i, at_row.h), quarter * S::kF, a.dim, vec_out, o);
        if (quarter == 0 && a.lse)
          a.lse[((int64_t)b * a.q_heads + at_row.h) * a.q_len + at_row.i] =
              sum == 0.f ? -INFINITY : fmaf(top, kLn2, logf(sum * down));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kSoft + 1) tmem_free(tm_s, 512);
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// Two kinds of blocks that each form the scores and dP = dout V^T again, for dq (a tile of rows
// against its keys) and for dk and dv (a tile of keys against the rows that see them): seven
// products instead of five, but every gradient has one owner, no atomics and one order.
// The accumulators carry scales of their half tile, so they are drained after each.
template <int N>
DCT_DEV void drain(uint32_t addr, float f, float (&acc)[N]) {
#pragma unroll
  for (int c = 0; c < N; c += 16) {                // by 16: registers are short
    uint32_t v[16];
    tmem_load16(addr + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[c + e] = fmaf(__uint_as_float(v[e]), f, acc[c + e]);
  }
}
template <int N>
DCT_DEV void drain(uint32_t addr, float2 f, float (&acc)[N]) {
#pragma unroll
  for (int c = 0; c < N; c += 16) {
    uint32_t v[16];
    tmem_load16(addr + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[c + e] = fmaf(__uint_as_float(v[e]) * f.x, f.y, acc[c + e]);
  }
}

// The largest of four numbers of [0, 255], one of each thread of a row.  (`top` may be written
// again when all have passed another meeting.)
DCT_DEV int meet(uint32_t mine, uint8_t (&top)[kTile][4], int row, int quarter, int warp) {
  top[row][quarter] = (uint8_t)mine;
  rows_sync(warp);
  const uint32_t x = *reinterpret_cast<const uint32_t*>(top[row]);
  return (int)max(max(x & 255, x >> 8 & 255), max(x >> 16 & 255, x >> 24));
}
// dS = P (dP - delta) can be anything up to the sizes of dout and the largest v of the whole
// row, and is small where P is or where another row of the tile has the large dout.  So it is
// scaled by what it is: for each row of the product that takes it (a query in dq, a key in dk)
// the largest |dS| of the half tile comes to [2^14, 2^15), and the row's accumulator is drained
// with the reverse of that after every half tile.  (Bounds from the tiles' norms instead lost
// the accuracy of rows far below the bound, and passed float16 where delta came from
// other tiles' v.)  Returns the exponent.
template <int N>
DCT_DEV int scale_of_ds(const float (&ds)[N], uint8_t (&top)[kTile][4], int row, int quarter, int warp) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) m = fmaxf(m, fabsf(ds[e]));
  return min(14 + 127 - meet(__float_as_uint(m) >> 23, top, row, quarter, warp), 120);
}
// P = 2^y of a key's rows likewise: a key that no row gives much weight has a dv as small, with
// as many bits.  (Down to weights of 2^-36; smaller ones keep steps of 2^-75.)
template <int N>
DCT_DEV int scale_of_p(const float (&y)[N], uint8_t (&top)[kTile][4], int row, int quarter, int warp) {
  float m = y[0];
#pragma unroll
  for (int e = 1; e < N; ++e) m = fmaxf(m, y[e]);
  return 14 + 50 - meet(__float2int_rd(fminf(fmaxf(m, -36.f), 100.f)) + 50, top, row, quarter, warp);
}
// f 2^e as two factors, neither of which leaves float32 where their product with an
// accumulator does not
DCT_DEV float2 factors(float f, int e) { return make_float2(pow2(e >> 1), f * pow2(e - (e >> 1))); }

template <int BLOCKS>
struct Dq : Sizes<BLOCKS> {
  static constexpr int kKeys = BLOCKS == 1 ? 5 : 3, kValues = BLOCKS == 1 ? 4 : 2;   // halves of K, of V
  struct Control {
    Ring<kKeys> k;
    Ring<kValues> v;
    uint64_t q_full, go_full, s_full[2], ds_full[2], acc_full, acc_empty;
    uint32_t tmem;
    __align__(4) uint8_t top[2][kTile][4];
  };
  static constexpr uint32_t kK = Sizes<BLOCKS>::kTileBytes, kV = kK + kKeys * Sizes<BLOCKS>::kSlotBytes;
  static constexpr uint32_t kEnd = kV + kValues * Sizes<BLOCKS>::kSlotBytes;
  static constexpr size_t kSmem = kEnd + sizeof(Control);
  static_assert(kSmem <= 227 * 1024);
};

// dq of a tile of 128 rows: dS = P (dP - delta), dq = scale dS K.  Q rests in shared memory,
// dout in tensor memory; V and K come in half tiles of 64 keys.
template <int BLOCKS, bool FULL>
DCT_DEV void attn_dq(const AttnArgs& a, const Tiles& w, int block, int row_tiles, bool vec_out, uint32_t* err) {
  using S = Dq<BLOCKS>;
  extern __shared__ __align__(1024) uint8_t sm[];
  auto& ctl = *reinterpret_cast<typename S::Control*>(sm + S::kEnd);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (misaligned(sm, err)) return;
  if (threadIdx.x == 0) {
    mbar_init(&ctl.q_full, 1);
    mbar_init(&ctl.go_full, kSoft);
    ctl.k.init();
    ctl.v.init();
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctl.s_full[s], 1);
      mbar_init(&ctl.ds_full[s], kSoft);
    }
    mbar_init(&ctl.acc_full, 1);
    mbar_init(&ctl.acc_empty, kSoft);
    mbar_fence_init();
  }
  if (warp == kSoft + 1) tmem_alloc(&ctl.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // S and dP twice, the operand dout, the accumulator
  const uint32_t tm_s = ctl.tmem, tm_dp = tm_s + 128, tm_go = tm_s + 256, tm_acc = tm_s + 384;
  const int heads = a.batch * a.kv_heads, bh = block % heads, tile = row_tiles - 1 - block / heads;
  const int b = bh / a.kv_heads, hk = bh % a.kv_heads;
  const int rows = a.q_len * a.group, r0 = tile * kTile;
  const int i0 = r0 / a.group, i_end = (min(r0 + kTile, rows) - 1) / a.group;
  touch(a);
  touch(w);
  pdl_entry();
  const AttnStats stats = w.stats[bh];
  const AttnSpan span(a, b);
  const bool splits_head = head_splits(stats, a.scale, a.dim);
  if (!splits_head && threadIdx.x == 0) *w.any = 1;          // work for the float32 kernels
  const int i1 = min(i_end, span.m - 1);
  int t0 = 0, n = 0;
  if (splits_head && i0 < span.m) {
    const int k0 = span.lo(a, i0), k1 = span.hi(a, i1);
    t0 = k0 / kHalf;
    n = k1 > k0 ? (k1 + kHalf - 1) / kHalf - t0 : 0;
  }
  Waits wait{err};
  const int steps = FULL ? 4 * BLOCKS : (a.dim + 15) / 16;

  if (warp >= kSoft) {
    registers_down();
    if (warp == kSoft) {
      if (n && elect_one()) {
        mbar_arrive_expect_tx(&ctl.q_full, S::kTileBytes);
        load_tile<BLOCKS>(w, bh, 0, tile, sm, &ctl.q_full);
        ctl.k.fill(n, S::kSlotBytes, wait, [&](int it, int s, uint64_t* bar) {
          load_half<BLOCKS>(w, bh, 1, t0 + it, sm + S::kK + s * S::kSlotBytes, bar);
        });
        mbar_wait(&ctl.q_full, 0, err);
      }
    } else if (warp == kSoft + 2) {
      if (elect_one())
        ctl.v.fill(n, S::kSlotBytes, wait, [&](int it, int s, uint64_t* bar) {
          load_half<BLOCKS>(w, bh, 2, t0 + it, sm + S::kV + s * S::kSlotBytes, bar);
        });
    } else if (warp == kSoft + 1) {
      if (n && elect_one()) {
        wait(&ctl.q_full, 0);
        wait(&ctl.go_full, 0);
        const uint64_t q = umma_desc(smem_addr(sm), kChunkBytes, 1024);
        auto key = [&](int j) { return smem_addr(sm + S::kK + j % S::kKeys * S::kSlotBytes); };
        auto value = [&](int j) { return smem_addr(sm + S::kV + j % S::kValues * S::kSlotBytes); };
        auto scores = [&](int j) {                   // S(j) = Q K^T, dP(j) = dout V^T
          if (!ctl.k.ready(j, wait)) return;
          mma_features_ss<BLOCKS>(tm_s + (j & 1) * kHalf, q, umma_desc(key(j), kChunkBytes, 1024), steps);
          if (!ctl.v.ready(j, wait)) return;
          mma_features_ts<BLOCKS, kHalf>(tm_dp + (j & 1) * kHalf, tm_go, umma_desc(value(j), kChunkBytes, 1024), steps);
          ctl.v.release(j);
          umma_commit(&ctl.s_full[j & 1]);
        };
        scores(0);
        for (int j = 0; j < n && wait.ok; ++j) {
          if (j + 1 < n) scores(j + 1);
          wait(&ctl.ds_full[j & 1], j >> 1);
          wait(&ctl.acc_empty, j ^ 1);
          if (!wait.ok) break;
          mma_rows<BLOCKS, 16>(tm_acc, tm_s + (j & 1) * kHalf, umma_desc(key(j), 2 * kChunkBytes, 1024), false, steps);
          ctl.k.release(j);
          umma_commit(&ctl.acc_full);
        }
      }
    }
  } else if (splits_head) {
    registers_up();
    const int quarter = warp >> 2, row = (warp & 3) * 32 + lane, r = r0 + row;
    const RowAt at_row(a, hk, min(r, rows - 1));
    const bool in = r < rows && at_row.i < span.m;
    const int lo = in ? span.lo(a, at_row.i) : 0, hi = in ? span.hi(a, at_row.i) : 0;
    const AttnTile *ki = w.info[1] + bh * w.tiles[1], *vi = w.info[2] + bh * w.tiles[2];
    const int eq = w.info[0][bh * w.tiles[0] + tile].e;
    const int eg = w.info[3][bh * w.tiles[3] + tile].e;
    float acc[S::kF];
#pragma unroll
    for (int e = 0; e < S::kF; ++e) acc[e] = 0.f;
    if (n) {
      const int64_t at_stat = (int64_t)bh * row_tiles * kTile + r;
      const float lse2 = w.lse2[at_stat], delta = w.delta[at_stat];
      tile_to_tmem<BLOCKS>(w.p[3] + (bh * w.tiles[3] + tile) * (int64_t)S::kTileBytes, tm_go, warp, row);
      tmem_wait_st();
      arrive_warp(&ctl.go_full);
      float f = 0.f, fd = 0.f;
      float2 back = {};
      auto take = [&](int j) {
        wait(&ctl.acc_full, j);
        drain(tm_acc + lane_bits(warp) + quarter * S::kF, back, acc);
        arrive_warp(&ctl.acc_empty);
      };
      AttnTile kt = ki[t0 >> 1], vt = vi[t0 >> 1];
      int ek = 0;
      for (int j = 0; j < n; ++j) {
        const int key = (t0 + j) * kHalf + quarter * 16;
        if (j == 0 || !((t0 + j) & 1)) {           // another tile of K and V
          ek = kt.e;
          f = a.scale * kLog2e * pow2(-eq - ek);
          fd = pow2(-vt.e);
          const int next = ((t0 + j) >> 1) + 1;
          if (next <= (t0 + n - 1) >> 1) {
            kt = ki[next];
            vt = vi[next];
          }
        }
        wait(&ctl.s_full[j & 1], j >> 1);
        const uint32_t off = lane_bits(warp) + (j & 1) * kHalf + quarter * 16;
        uint32_t x[16], y[16];
        tmem_load16(tm_s + off, x);
        tmem_load16(tm_dp + off, y);
        tmem_wait_ld();
        float ds[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          ds[e] = ex2(fmaf(__uint_as_float(x[e]), f, -lse2)) * fmaf(__uint_as_float(y[e]), fd, -delta);
        if (__any_sync(0xffffffffu, key < lo || key + 16 > hi)) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (key + e < lo || key + e >= hi) ds[e] = 0.f;
        }
        const int eds = scale_of_ds(ds, ctl.top[j & 1], row, quarter, warp);
        const float up = pow2(eds);
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] *= up;
        store_operand<16>(tm_s + off, ds);
        tmem_wait_st();
        arrive_warp(&ctl.ds_full[j & 1]);
        if (j) take(j - 1);
        back = factors(a.scale, -eds - eg - ek);
      }
      take(n - 1);
    }
    if (r < rows) {
      store_features<S::kF>(a.dq + at(a.dqs, b, at_row.i, at_row.h), quarter * S::kF, a.dim, vec_out, acc);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kSoft + 1) tmem_free(tm_s, 512);
}

template <int BLOCKS>
struct Dkv : Sizes<BLOCKS> {
  static constexpr int kRowsQ = BLOCKS == 1 ? 5 : 3, kRowsGo = BLOCKS == 1 ? 4 : 2;  // halves of Q, of dout
  struct Control {
    float lse[kRowsQ][kHalf], delta[kRowsQ][kHalf];  // with Q; 16-byte aligned: the bulk copies' targets
    __align__(4) uint8_t top[2][kTile][4];
    Ring<kRowsQ> q;
    Ring<kRowsGo> go;
    uint64_t k_full, v_full, s_full, dp_full, p_full, ds_full, dv_full, dv_empty, dk_full, dk_empty;
    uint32_t tmem;
  };
  static constexpr uint32_t kQ = Sizes<BLOCKS>::kTileBytes, kGo = kQ + kRowsQ * Sizes<BLOCKS>::kSlotBytes;
  static constexpr uint32_t kEnd = kGo + kRowsGo * Sizes<BLOCKS>::kSlotBytes;
  static constexpr size_t kSmem = kEnd + sizeof(Control);
  static_assert(kSmem <= 227 * 1024);
};

// dk and dv of a tile of 128 keys: dv = P^T dout, dk = scale dS^T Q.  K rests in shared
// memory, V in tensor memory; Q and dout come in half tiles of 64 rows with their log-sums
// and deltas.  A thread holds (key, quarter): 16 rows of the scores and a quarter of the
// features of both gradients.
template <int BLOCKS, bool FULL>
DCT_DEV void attn_dkv(const AttnArgs& a, const Tiles& w, int block, int row_tiles, bool vec_out, uint32_t* err) {
  using S = Dkv<BLOCKS>;
  extern __shared__ __align__(1024) uint8_t sm[];
  auto& ctl = *reinterpret_cast<typename S::Control*>(sm + S::kEnd);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (misaligned(sm, err)) return;
  if (threadIdx.x == 0) {
    mbar_init(&ctl.k_full, 1);
    mbar_init(&ctl.v_full, kSoft);
    ctl.q.init();
    ctl.go.init();
    mbar_init(&ctl.s_full, 1);
    mbar_init(&ctl.dp_full, 1);
    mbar_init(&ctl.p_full, kSoft);
    mbar_init(&ctl.ds_full, kSoft);
    mbar_init(&ctl.dv_full, 1);
    mbar_init(&ctl.dv_empty, kSoft);
    mbar_init(&ctl.dk_full, 1);
    mbar_init(&ctl.dk_empty, kSoft);
    mbar_fence_init();
  }
  if (warp == kSoft + 1) tmem_alloc(&ctl.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // the accumulators, the operand V, S and dP (each also P's and dS's place)
  const uint32_t tm_dk = ctl.tmem, tm_dv = tm_dk + 128, tm_v = tm_dk + 256, tm_s = tm_dk + 384, tm_dp = tm_dk + 448;
  const int heads = a.batch * a.kv_heads, bh = block % heads, tile = block / heads;    // long ones first
  const int b = bh / a.kv_heads, hk = bh % a.kv_heads;
  touch(a);
  touch(w);
  pdl_entry();
  const AttnStats stats = w.stats[bh];
  const AttnSpan span(a, b);
  const bool splits_head = head_splits(stats, a.scale, a.dim);
  if (!splits_head && threadIdx.x == 0) *w.any = 1;          // work for the float32 kernels
  const int j0 = tile * kTile, j1 = min(j0 + kTile, span.n) - 1;
  int t0 = 0, n = 0;
  if (splits_head && j0 < span.n) {
    const int first = span.first(a, j0) * a.group, last = span.last(a, j1) * a.group;
    t0 = first / kHalf;
    n = last > first ? (last + kHalf - 1) / kHalf - t0 : 0;
  }
  Waits wait{err};
  const int steps = FULL ? 4 * BLOCKS : (a.dim + 15) / 16;

  if (warp >= kSoft) {
    registers_down();
    if (warp == kSoft) {
      if (n && elect_one()) {
        mbar_arrive_expect_tx(&ctl.k_full, S::kTileBytes);
        load_tile<BLOCKS>(w, bh, 1, tile, sm, &ctl.k_full);
        ctl.q.fill(n, S::kSlotBytes + 2 * kHalf * 4, wait, [&](int it, int s, uint64_t* bar) {
          const int64_t at_stat = (int64_t)bh * row_tiles * kTile + (int64_t)(t0 + it) * kHalf;
          load_half<BLOCKS>(w, bh, 0, t0 + it, sm + S::kQ + s * S::kSlotBytes, bar);
          bulk_load(ctl.lse[s], w.lse2 + at_stat, kHalf * 4, bar);
          bulk_load(ctl.delta[s], w.delta + at_stat, kHalf * 4, bar);
        });
        mbar_wait(&ctl.k_full, 0, err);
      }
    } else if (warp == kSoft + 2) {
      if (elect_one())
        ctl.go.fill(n, S::kSlotBytes, wait, [&](int it, int s, uint64_t* bar) {
          load_half<BLOCKS>(w, bh, 3, t0 + it, sm + S::kGo + s * S::kSlotBytes, bar);
        });
    } else if (warp == kSoft + 1) {
      if (n && elect_one()) {
        wait(&ctl.k_full, 0);
        wait(&ctl.v_full, 0);
        const uint64_t k = umma_desc(smem_addr(sm), kChunkBytes, 1024);
        auto query = [&](int j) { return smem_addr(sm + S::kQ + j % S::kRowsQ * S::kSlotBytes); };
        auto grad = [&](int j) { return smem_addr(sm + S::kGo + j % S::kRowsGo * S::kSlotBytes); };
        auto scores = [&](int j) {                   // S^T(j) = K Q^T
          if (!ctl.q.ready(j, wait)) return;
          mma_features_ss<BLOCKS>(tm_s, k, umma_desc(query(j), kChunkBytes, 1024), steps);
          umma_commit(&ctl.s_full);
        };
        auto dps = [&](int j) {                      // dP^T(j) = V dout^T
          if (!ctl.go.ready(j, wait)) return;
          mma_features_ts<BLOCKS, kHalf>(tm_dp, tm_v, umma_desc(grad(j), kChunkBytes, 1024), steps);
          umma_commit(&ctl.dp_full);
        };
        scores(0);
        dps(0);
        for (int j = 0; j < n && wait.ok; ++j) {
          wait(&ctl.p_full, j);
          wait(&ctl.dv_empty, j ^ 1);
          if (!wait.ok) break;
          mma_rows<BLOCKS, 16>(tm_dv, tm_s, umma_desc(grad(j), 2 * kChunkBytes, 1024), false, steps);
          ctl.go.release(j);
          umma_commit(&ctl.dv_full);
          if (j + 1 < n) scores(j + 1);
          wait(&ctl.ds_full, j);
          wait(&ctl.dk_empty, j ^ 1);
          if (!wait.ok) break;
          mma_rows<BLOCKS, 16>(tm_dk, tm_dp, umma_desc(query(j), 2 * kChunkBytes, 1024), false, steps);
          ctl.q.release(j);
          umma_commit(&ctl.dk_full);
          if (j + 1 < n) dps(j + 1);
        }
      }
    }
  } else if (splits_head) {
    registers_up();
    const int quarter = warp >> 2, row = (warp & 3) * 32 + lane, key = j0 + row;
    // rows that see the thread's key
    const int lo = key < span.n ? span.first(a, key) * a.group : 0, hi = key < span.n ? span.last(a, key) * a.group : 0;
    const AttnTile *qi = w.info[0] + bh * w.tiles[0], *gi = w.info[3] + bh * w.tiles[3];
    const int ek = w.info[1][bh * w.tiles[1] + tile].e;
    const int ev = w.info[2][bh * w.tiles[2] + tile].e;
    float dk[S::kF], dv[S::kF];
#pragma unroll
    for (int e = 0; e < S::kF; ++e) dk[e] = dv[e] = 0.f;
    if (n) {
      tile_to_tmem<BLOCKS>(w.p[2] + (bh * w.tiles[2] + tile) * (int64_t)S::kTileBytes, tm_v, warp, row);
      tmem_wait_st();
      arrive_warp(&ctl.v_full);
      // dv of a half tile is drained at the end of it, dk after the next one's P, when their
      // products are done and no matrix instruction yet waits for the accumulator.
      const float fd = pow2(-ev);
      float f = 0.f;
      float2 back_k = {};
      auto take_dk = [&](int j) {
        wait(&ctl.dk_full, j);
        drain(tm_dk + lane_bits(warp) + quarter * S::kF, back_k, dk);
        arrive_warp(&ctl.dk_empty);
      };
      AttnTile qt = qi[t0 >> 1], gt = gi[t0 >> 1];
      int eq = 0, eg = 0;
      const uint32_t off = lane_bits(warp) + quarter * 16;
      for (int j = 0; j < n; ++j) {
        const int r = (t0 + j) * kHalf + quarter * 16;
        if (j == 0 || !((t0 + j) & 1)) {                   // another tile of Q and dout
          eq = qt.e;
          f = a.scale * kLog2e * pow2(-eq - ek);
          eg = gt.e;
          const int next = ((t0 + j) >> 1) + 1;
          if (next <= (t0 + n - 1) >> 1) {
            qt = qi[next];
            gt = gi[next];
          }
        }
        ctl.q.ready(j, wait);                      // the log-sums and deltas
        wait(&ctl.s_full, j);
        const float4* lse = reinterpret_cast<const float4*>(ctl.lse[j % S::kRowsQ] + quarter * 16);
        const float4* del = reinterpret_cast<const float4*>(ctl.delta[j % S::kRowsQ] + quarter * 16);
        uint32_t x[16];
        float p[16];
        tmem_load16(tm_s + off, x);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 l = lse[e / 4];
          p[e] = fmaf(__uint_as_float(x[e]), f, -l.x);
          p[e + 1] = fmaf(__uint_as_float(x[e + 1]), f, -l.y);
          p[e + 2] = fmaf(__uint_as_float(x[e + 2]), f, -l.z);
          p[e + 3] = fmaf(__uint_as_float(x[e + 3]), f, -l.w);
        }
        if (__any_sync(0xffffffffu, r < lo || r + 16 > hi)) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (r + e < lo || r + e >= hi) p[e] = -INFINITY;
        }
        const int ep = scale_of_p(p, ctl.top[0], row, quarter, warp);
        const float up_p = pow2(ep);               // (not in the exponent, which would be rounded again)
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = ex2(p[e]) * up_p;
        store_operand<16>(tm_s + off, p);
        tmem_wait_st();
        arrive_warp(&ctl.p_full);
        if (j) take_dk(j - 1);
        wait(&ctl.dp_full, j);
        tmem_load16(tm_dp + off, x);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 d = del[e / 4];
          p[e] *= fmaf(__uint_as_float(x[e]), fd, -d.x);
          p[e + 1] *= fmaf(__uint_as_float(x[e + 1]), fd, -d.y);
          p[e + 2] *= fmaf(__uint_as_float(x[e + 2]), fd, -d.z);
          p[e + 3] *= fmaf(__uint_as_float(x[e + 3]), fd, -d.w);
        }
        const int eds = scale_of_ds(p, ctl.top[1], row, quarter, warp);
        const float up = pow2(eds);
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] *= up;
        back_k = factors(a.scale, -eds - ep - eg - eq);
        store_operand<16>(tm_dp + off, p);
        tmem_wait_st();
        arrive_warp(&ctl.ds_full);
        wait(&ctl.dv_full, j);
        drain(tm_dv + lane_bits(warp) + quarter * S::kF, pow2(-ep - eg), dv);
        arrive_warp(&ctl.dv_empty);
      }
      take_dk(n - 1);
    }
    if (key < a.kv_len) {
      store_features<S::kF>(a.dk + at(a.dks, b, key, hk), quarter * S::kF, a.dim, vec_out, dk);
      store_features<S::kF>(a.dv + at(a.dvs, b, key, hk), quarter * S::kF, a.dim, vec_out, dv);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kSoft + 1) tmem_free(tm_dk, 512);
}

// Both in one launch: the long tiles of keys first, then the tiles of rows, which fill the
// SMs that the last tiles of keys leave idle.
template <int BLOCKS, bool FULL>
__global__ void __launch_bounds__(kThreads, 1) k_attn_backward(const __grid_constant__ AttnArgs a,
                                                               const __grid_constant__ Tiles w, int row_tiles,
                                                               int key_blocks, bool vec_q, bool vec_kv, uint32_t* err) {
  if ((int)blockIdx.x < key_blocks) attn_dkv<BLOCKS, FULL>(a, w, blockIdx.x, row_tiles, vec_kv, err);
  else attn_dq<BLOCKS, FULL>(a, w, blockIdx.x - key_blocks, row_tiles, vec_q, err);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct Layout {
  int64_t heads, row_tiles, key_tiles, blocks;
  size_t stats, tile[4], info[4], lse2, delta, plain, part, total;
  int splits;
  Layout(const AttnArgs& a, bool backward) {
    heads = (int64_t)a.batch * a.kv_heads;
    row_tiles = padded_rows(a) / kTile;
    key_tiles = (a.kv_len + kTile - 1) / kTile;
    blocks = a.dim <= 64 ? 1 : 2;
    splits = 1;
    if (!backward && heads * row_tiles) {          // fill the SMs when there are few tiles of rows
      const int64_t want = dev_info().sm_count / (heads * row_tiles);
      splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, key_tiles / 2), 64));
    }
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += (n + 1023) & ~size_t(1023); return o; };
    stats = take(sizeof(AttnStats) * heads + sizeof(uint32_t));     // and the word `any`
    for (int t = 0; t < (backward ? 4 : 3); ++t) {
      const size_t tiles = (size_t)heads * (t == 1 || t == 2 ? key_tiles : row_tiles);
      tile[t] = take(tiles * blocks * kBlockBytes);
      info[t] = take(tiles * sizeof(AttnTile));
    }
    lse2 = delta = plain = part = 0;
    if (backward) {
      lse2 = take(sizeof(float) * heads * row_tiles * kTile);
      delta = take(sizeof(float) * heads * row_tiles * kTile);
      plain = take(sizeof(float) * heads * row_tiles * kTile);
    } else {
      part = take(std::max(attn_rows_ws_bytes(a),
                           splits > 1 ? sizeof(float) * heads * a.group * a.q_len * splits * (size_t)(a.dim + 2) : 0));
    }
    total = at;
  }
};

bool aligned(const float* p, const int64_t* s) {
  return aligned16_h(p) && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
}

cudaError_t prepare(const AttnArgs& a, const Layout& L, uint8_t* w, bool backward, Tiles& t, cudaStream_t st) {
  t = Tiles{};
  t.stats = reinterpret_cast<AttnStats*>(w + L.stats);
  t.any = reinterpret_cast<uint32_t*>(t.stats + L.heads);
  for (int i = 0; i < (backward ? 4 : 3); ++i) {
    t.p[i] = w + L.tile[i];
    t.info[i] = reinterpret_cast<AttnTile*>(w + L.info[i]);
    t.tiles[i] = i == 1 || i == 2 ? L.key_tiles : L.row_tiles;
  }
  t.lse2 = reinterpret_cast<float*>(w + L.lse2);
  t.delta = reinterpret_cast<float*>(w + L.delta);
  cudaError_t e = cudaMemsetAsync(t.stats, 0, sizeof(AttnStats) * L.heads + sizeof(uint32_t), st);
  if (e != cudaSuccess) return e;
  const int64_t split = L.heads * ((backward ? 2 : 1) * L.row_tiles + 2 * L.key_tiles);
  if (split > INT_MAX) return cudaErrorInvalidConfiguration;
  if (!split) return cudaSuccess;
  const bool vec = a.dim % 4 == 0 && aligned(a.q, a.qs) && aligned(a.k, a.ks) && aligned(a.v, a.vs) &&
                   (!backward || aligned(a.dout, a.os));
  const int tq = (int)L.row_tiles, tk = (int)L.key_tiles;
  return launch_pdl(L.blocks == 1 ? k_attn_split<1> : k_attn_split<2>, dim3((unsigned)split), dim3(512), 0, st, a, t,
                    tq, tk, vec);
}

template <typename K>
cudaError_t prepared(K kernel, size_t smem) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  return e == cudaSuccess ? launched_with(kernel, kThreads, kRegs) : e;
}

template <int BLOCKS, bool FULL>
cudaError_t forward(const AttnArgs& a, const Layout& L, const Tiles& t, float* part, cudaStream_t st) {
  using S = Forward<BLOCKS>;
  static const cudaError_t set = prepared(k_attn_forward<BLOCKS, FULL>, S::kSmem);
  if (set != cudaSuccess) return set;
  const int64_t blocks = L.heads * L.row_tiles * L.splits;
  if (blocks > INT_MAX) return cudaErrorInvalidConfiguration;
  return launch_pdl(k_attn_forward<BLOCKS, FULL>, dim3((unsigned)blocks), dim3(kThreads), S::kSmem, st, a, t,
                    (int)L.row_tiles, L.splits, part, a.dim % 4 == 0 && aligned(a.out, a.os), device_error_word());
}

template <int BLOCKS, bool FULL>
cudaError_t backward(const AttnArgs& a, const Layout& L, const Tiles& t, cudaStream_t st) {
  constexpr size_t kSmem = std::max(Dq<BLOCKS>::kSmem, Dkv<BLOCKS>::kSmem);
  static const cudaError_t set = prepared(k_attn_backward<BLOCKS, FULL>, kSmem);
  if (set != cudaSuccess) return set;
  const int64_t nq = L.heads * L.row_tiles, nk = L.heads * L.key_tiles;
  if (nq + nk > INT_MAX) return cudaErrorInvalidConfiguration;
  const bool vec = a.dim % 4 == 0;
  return launch_pdl(k_attn_backward<BLOCKS, FULL>, dim3((unsigned)(nq + nk)), dim3(kThreads), kSmem, st, a, t,
                    (int)L.row_tiles, (int)nk, vec && aligned(a.dq, a.dqs),
                    vec && aligned(a.dk, a.dks) && aligned(a.dv, a.dvs), device_error_word());
}

}  // namespace

// The tensor cores' way has more launches and a pass over the operands before it; the CUDA
// cores' time goes with the work (here all pairs times features), and for few rows with the
// bytes of the keys.  Microseconds, CUDA cores against tensor cores, forward: 8.4 million 20
// and 28, 50 million 40 and 29, 67 million 33 to 37 and 32 to 35, 262 million 116 and 66; 8
// rows a key head over 1000 keys 26 and 42, 16 rows over 2000 72 and 61.  Forward and
// backward: 11.5 million 42 and 50, 34 million 62 to 114 and 47 to 62, 67 million 96 and 52.
bool attn_tensor_fits(const AttnArgs& a, bool backward) {
  const double work = (double)a.batch * a.q_heads * a.q_len * a.kv_len * a.dim;
  return backward ? work >= 12e6 : work >= 30e6 && (int64_t)a.q_len * a.group >= 16;
}

size_t attn_tensor_ws_bytes(const AttnArgs& a, bool backward) { return Layout(a, backward).total; }

cudaError_t launch_attn_tensor_forward(const AttnArgs& args, void* ws, cudaStream_t st) {
  AttnArgs a = args;
  const Layout L(a, false);
  uint8_t* w = static_cast<uint8_t*>(ws);
  Tiles t;
  cudaError_t e = prepare(a, L, w, false, t, st);
  if (e != cudaSuccess) return e;
  a.stats = t.stats;
  a.any = t.any;
  float* part = reinterpret_cast<float*>(w + L.part);
  const auto run = L.blocks == 1 ? (a.dim == 64 ? forward<1, true> : forward<1, false>)
                                 : (a.dim == 128 ? forward<2, true> : forward<2, false>);
  e = run(a, L, t, part, st);
  if (e == cudaSuccess && L.splits > 1) e = launch_attn_join(a, L.splits, part, true, st);
  if (e == cudaSuccess) e = launch_attn_rows_forward(a, part, st);
  return e;
}

cudaError_t launch_attn_tensor_backward(const AttnArgs& args, void* ws, cudaStream_t st) {
  AttnArgs a = args;
  const Layout L(a, true);
  Tiles t;
  a.delta = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + L.plain);
  cudaError_t e = prepare(a, L, static_cast<uint8_t*>(ws), true, t, st);
  if (e != cudaSuccess) return e;
  a.stats = t.stats;
  a.any = t.any;
  const auto run = L.blocks == 1 ? (a.dim == 64 ? backward<1, true> : backward<1, false>)
                                 : (a.dim == 128 ? backward<2, true> : backward<2, false>);
  e = run(a, L, t, st);
  if (e == cudaSuccess) e = launch_attn_rows_backward(a, st);
  return e;
}

}  // namespace dct
