// Orthogonalisation by Newton-Schulz steps, and the optimizer update around it.
//
// X = u / (|u| + eps), then `steps` times A = X X^T, P = c A A + b A, X = P X + a X (for tall
// matrices A = X^T X, and P on the right).  The terms b A and a X are added in float32 after
// the products: inside them, as multiples of the identity, they would be rounded with every
// matrix instruction (see k_product), which measured 5 times the error.
//
// It is bound by the tensor cores: X, A and P live as split float16 chunks (dct_umma.cuh)
// from the first kernel to the last, and one persistent kernel forms each product at float32
// accuracy.  Of the symmetric A and P only the tiles up to the diagonal are formed and
// stored; a chunk above it is read as the transpose of its mirror image, which the matrix
// instructions do at no cost.  The powers of two are constants: no entry is larger than the
// matrix's norm, which the polynomial bounds from the start.
#include <algorithm>

#include "dct_common.cuh"
#include "dct_umma.cuh"
#include "kernels.h"

namespace dct {
namespace {

// ---------------------------------------------------------------------------
// C = sa A B + sd D over a batch, as chunks or as the final float32 result
// ---------------------------------------------------------------------------
struct Operand {
  const uint8_t* p;
  uint32_t cb;               // chunks per row of chunks
  uint64_t z;                // bytes between matrices
  bool mn;                   // its rows are the contraction
  bool half;                 // symmetric, the tiles above the diagonal are not stored
};
DCT_DEV const uint8_t* chunk_of(const Operand& o, uint32_t z, uint32_t rb, uint32_t cb) {
  return o.p + z * o.z + ((uint64_t)rb * o.cb + cb) * kPairBytes;
}
struct Product {
  Operand A, B, D;           // D.p null: no D; else stored where C is
  uint8_t* C;                // chunks, or null: final
  uint32_t c_cb;
  uint64_t c_z;
  float sa, sd;
  uint32_t M, N, kb;         // rows, columns, contraction in chunks of 64
  uint32_t mt, nt, tiles;    // rows and columns of tiles, tiles of a matrix
  bool half;                 // C is symmetric: only the tiles up to the diagonal
  // final result
  float* out;                // y, or w
  float keep, rate;
  bool update;               // out = keep out - rate C, else out = C
  float* parts;              // sums of cut tiles, two slots a worker and block
  uint32_t* arrived;         // segments of a worker's cut tile that are summed (zero between launches)
};

constexpr int kRows = 128, kEpi = 8;            // tile rows of a block, epilogue warps
constexpr int kThreads = 32 * (kEpi + 4);     // and warps that load, issue, and give up registers (two)
// 384 threads start with 168 registers, 64512 in all, and as many are taken
constexpr int kUpRegs = 232, kDownRegs = 40, kRegs = 32 * (kEpi * kUpRegs + 4 * kDownRegs);

constexpr uint32_t kStaging = 4096;              // of an epilogue warp: its 32 rows of a chunk

template <bool PAIR, int BN>
struct Shape {
  static constexpr uint32_t kTileRows = PAIR ? 2 * kRows : kRows;
  static constexpr uint32_t kBChunks = (PAIR ? BN / 2 : BN) / 64;    // chunks of B's columns in this block
  static constexpr uint32_t kA = 2 * kPairBytes, kB = kBChunks * kPairBytes, kStage = kA + kB;
  static constexpr int kStages = 196608 / kStage > 4 ? 4 : 196608 / kStage;
  static constexpr int kBufs = BN == 256 ? 2 : 4;                    // accumulators in tensor memory
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kEpi * kStaging;
};

// tile number -> batch entry, row and column of tiles
DCT_DEV void tile_at(const Product& g, uint32_t t, uint32_t& z, uint32_t& i, uint32_t& j) {
  z = t / g.tiles;
  uint32_t r = t - z * g.tiles;
  if (!g.half) {
    i = r % g.mt;            // neighbours share the B tile
    j = r / g.mt;
    return;
  }
  for (i = 0; r > i; ++i) r -= i + 1;      // row i holds the tiles 0 .. i
  j = r;
}

// A worker (a block, or a pair of blocks) takes every workers-th tile as far as they go
// around, so that the tiles at work at one time are neighbours and share their operands in
// L2.  The tiles that are left go whole to some workers, or their chunks are dealt to all in
// equal runs.  A worker's share of one tile is a segment.
struct Segment {
  uint32_t tile, k0, k1;     // chunks [k0, k1) of the tile
  uint32_t first, count;     // the worker with the tile's first segment, the tile's segments
};
struct Run {                 // fewer than `workers` tiles are left, of at most 2^17 chunks: 32 bits hold the products
  uint32_t at, end, units;   // of the tiles that are left
  uint32_t kb, unit, worker, workers, round, rounds, used;
  DCT_DEV Run(uint32_t tiles, uint32_t kb_, uint32_t unit_, uint32_t used_, uint32_t worker_, uint32_t workers_)
      : kb(kb_), unit(unit_), worker(worker_), workers(workers_), round(0), rounds(tiles / workers_), used(used_) {
    units = (tiles - rounds * workers) * (unit == 1 ? kb : 1);
    at = end = 0;
    if (worker < used) {
      at = worker * units / used * unit;
      end = (worker + 1) * units / used * unit;
    }
  }
  DCT_DEV uint32_t worker_of(uint32_t chunk) const {
    return (((unit == 1 ? chunk : chunk / unit) + 1) * used - 1) / units;
  }
  DCT_DEV bool next(Segment& s) {
    if (round < rounds) {
      s.tile = round++ * workers + worker;
      s.k0 = 0;
      s.k1 = kb;
      s.count = 1;
      return true;
    }
    if (at >= end) return false;
    const uint32_t t = at / kb, base = t * kb;
    s.tile = rounds * workers + t;
    s.k0 = at - base;
    s.k1 = min(kb, end - base);
    s.first = worker_of(base);
    s.count = worker_of(base + kb - 1) - s.first + 1;
    at = base + s.k1;
    return true;
  }
};

// acc[at .. at + 7] += f * the float16 numbers of v
template <int N>
DCT_DEV void add8(float (&acc)[N], int at, float f, uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
    acc[at + 2 * e] = fmaf(f, x.x, acc[at + 2 * e]);
    acc[at + 2 * e + 1] = fmaf(f, x.y, acc[at + 2 * e + 1]);
  }
}

DCT_DEV void prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
DCT_DEV void epilogue_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Warps 0..7 drain and store, warp 8 loads, warp 9 issues the matrix instructions.
//
// The tensor cores round every sum toward zero: a chain of n matrix instructions is off by
// about n/2 * 2^-24 of a sum that grows steadily (5e-5 after 8192 columns, measured), so the
// accumulator is drained to registers every kDrain chunks and added there with rounding to
// nearest, and within a chunk the small cross products come first.
//
// Tiles that several blocks share meet in memory: every block leaves its sum, and the last
// to arrive adds them in the order of the contraction, so the result does not depend on who
// that was.
// Draining costs about 230 cycles of the tensor cores: 5% of a large product every second
// chunk, 9% every chunk; the smaller tiles do it every chunk.
//
// PAIR: two blocks on one tile of twice the rows.  A chunk of the contraction then costs a
// block 64 KB of loads instead of 96 KB (tile 256 columns wide), and the loads are what
// bounds the large products: 6.4 TB/s out of L2 at 2048 x 8192 without pairs.
template <bool PAIR, int BN>
__global__ void __launch_bounds__(kThreads, 1) k_product(const __grid_constant__ Product g, uint32_t total,
                                                         uint32_t unit, uint32_t used, uint32_t* err) {
  using S = Shape<PAIR, BN>;
  constexpr uint32_t kDrain = PAIR ? 2 : 1;
  extern __shared__ uint8_t raw[];
  uint8_t* sm = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
  __shared__ uint64_t full[4], empty[4], there[4], done[4], freed[4];   // there: the other block's chunk is in
  __shared__ uint32_t tmem_base, order;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0, worker = PAIR ? blockIdx.x / 2 : blockIdx.x;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&there[s], 1);
    }
    for (int s = 0; s < S::kBufs; ++s) {
      mbar_init(&done[s], 1);
      mbar_init(&freed[s], PAIR ? 2 * kEpi : kEpi);
    }
    mbar_fence_init();
  }
  if (warp == kEpi + 1) {
    if constexpr (PAIR) tmem_alloc_pair(&tmem_base, S::kBufs * BN);
    else tmem_alloc(&tmem_base, S::kBufs * BN);
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  const uint32_t mchunks = (g.M + 63) / 64, nchunks = (g.N + 63) / 64;
  // the first segment before the wait for the kernel before: its divisions take 2 us
  Run run(total, g.kb, unit, used, worker, PAIR ? gridDim.x / 2 : gridDim.x);
  Segment sg;
  uint32_t z, ti, tj;
  auto next = [&]() {
    if (!run.next(sg)) return false;
    tile_at(g, sg.tile, z, ti, tj);
    return true;
  };
  bool more = next();
  pdl_entry();
  // whether chunk k of an operand's tile is read with its rows as the contraction: its own
  // layout, or the mirror image of a chunk above the diagonal
  auto transposed = [](const Operand& o, uint32_t tile, uint32_t k) {
    return o.half ? tile < k / (S::kTileRows / 64) : o.mn;
  };

  if (warp >= kEpi) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kDownRegs));
    if (warp == kEpi) {
      if (elect_one()) {
        uint32_t it = 0;
        bool ok = true;
          for (; ok && more; more = next()) {
          const uint32_t m0 = ti * (S::kTileRows / 64) + rank * 2, n0 = tj * (BN / 64) + rank * S::kBChunks;
          const uint32_t mc = m0 < mchunks ? min(2u, mchunks - m0) : 0;
          const uint32_t nc = n0 < nchunks ? min(S::kBChunks, nchunks - n0) : 0;
          for (uint32_t k = sg.k0; k < sg.k1; ++k, ++it) {
            const uint32_t s = it % S::kStages;
            ok = mbar_wait(&empty[s], ((it / S::kStages) & 1) ^ 1, err);
            if (!ok) break;
            mbar_arrive_expect_tx(&full[s], (mc + nc) * kPairBytes);
            const bool a_mn = transposed(g.A, ti, k), b_mn = transposed(g.B, tj, k);
            uint8_t* a = sm + s * S::kStage;
            for (uint32_t p = 0; p < mc; ++p) {
              const uint8_t* c = a_mn ? chunk_of(g.A, z, k, m0 + p) : chunk_of(g.A, z, m0 + p, k);
              bulk_load(a + p * kChunkBytes, c, kChunkBytes, &full[s]);
              bulk_load(a + (2 + p) * kChunkBytes, c + kChunkBytes, kChunkBytes, &full[s]);
            }
            uint8_t* b = a + S::kA;
            for (uint32_t p = 0; p < nc; ++p) {
              const uint8_t* c = b_mn ? chunk_of(g.B, z, k, n0 + p) : chunk_of(g.B, z, n0 + p, k);
              bulk_load(b + p * kChunkBytes, c, kChunkBytes, &full[s]);
              bulk_load(b + (S::kBChunks + p) * kChunkBytes, c + kChunkBytes, kChunkBytes, &full[s]);
            }
          }
        }
        // every copy has landed before the block may end
        for (uint32_t u = it > (uint32_t)S::kStages ? it - S::kStages : 0; u < it; ++u)
          mbar_wait(&full[u % S::kStages], (u / S::kStages) & 1, err);
      }
    } else if (warp == kEpi + 1 && rank != 0) {
      if (elect_one()) {                              // tells the even block of each chunk that has come in
        uint32_t it = 0;
        bool ok = true;
        for (; ok && more; more = next())
          for (uint32_t k = sg.k0; k < sg.k1 && ok; ++k, ++it) {
            const uint32_t s = it % S::kStages;
            ok = mbar_wait(&full[s], (it / S::kStages) & 1, err);
            if (ok) mbar_arrive_at(&there[s], 0);
          }
      }
    } else if (warp == kEpi + 1) {
      if (elect_one()) {
        auto mma = [](uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
          if constexpr (PAIR) umma_pair(d, a, b, idesc, add);
          else umma(d, a, b, idesc, add);
        };
        auto commit = [](uint64_t* bar) {
          if constexpr (PAIR) umma_commit_pair(bar);
          else umma_commit(bar);
        };
        uint32_t it = 0, part = 0;
        bool ok = true;
        for (; ok && more; more = next()) {
          for (uint32_t k0 = sg.k0; k0 < sg.k1 && ok; k0 += kDrain, ++part) {
            const uint32_t buf = part % S::kBufs, d = tmem + buf * BN, k1 = min(sg.k1, k0 + kDrain);
            ok = mbar_wait_cluster(&freed[buf], ((part / S::kBufs) & 1) ^ 1, err);
            tc_fence_after();
            for (uint32_t k = k0; k < k1 && ok; ++k, ++it) {
              const uint32_t s = it % S::kStages;
              ok = mbar_wait(&full[s], (it / S::kStages) & 1, err);
              if (PAIR && ok) ok = mbar_wait_cluster(&there[s], (it / S::kStages) & 1, err);
              if (!ok) break;
              tc_fence_after();
              const bool a_mn = transposed(g.A, ti, k), b_mn = transposed(g.B, tj, k);
              const uint32_t idesc = umma_idesc(S::kTileRows, BN, a_mn, b_mn);
              // 16 rows, or 16 columns
              const uint32_t step_a = (a_mn ? 2048 : 32) / 16, step_b = (b_mn ? 2048 : 32) / 16;
              const uint32_t a = smem_addr(sm + s * S::kStage), b = a + S::kA;
              const uint64_t ah = umma_desc(a, kChunkBytes, 1024), bh = umma_desc(b, kChunkBytes, 1024);
              const uint64_t al = ah + 2 * kChunkBytes / 16, bl = bh + S::kBChunks * kChunkBytes / 16;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                mma(d, al + q * step_a, bh + q * step_b, idesc, k != k0 || q != 0);
                mma(d, ah + q * step_a, bl + q * step_b, idesc, true);
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) mma(d, ah + q * step_a, bh + q * step_b, idesc, true);
              commit(&empty[s]);
            }
            commit(&done[buf]);
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kUpRegs));
    constexpr int W = BN / 2;                     // columns of a thread's row
    const uint32_t side = warp >> 2;
    uint8_t* stage = sm + S::kStages * S::kStage + warp * kStaging;
    uint32_t part = 0;
    // once a wait has run out the loop goes on without waiting: the other warps still count
    // on meeting this one
    bool ok = true;
    for (; more; more = next()) {
      // the warp's 32 rows from i0, the thread's columns from j0
      const uint32_t i0 = ti * S::kTileRows + rank * kRows + (warp & 3) * 32, j0 = tj * BN + side * W;
      // what the end of the tile reads, into L2 by then
      if (g.D.p && i0 < mchunks * 64)
        for (uint32_t c = 0; c < W && j0 + c < nchunks * 64; c += 64) {
          const uint8_t* d = chunk_of(g.D, z, i0 >> 6, (j0 + c) >> 6) + (i0 & 32) * 128 + lane * 128;
          prefetch(d);
          prefetch(d + kChunkBytes);
        }
      if (g.update && i0 + lane < g.M)
        for (uint32_t c = 0; c < W && j0 + c < g.N; c += 32)
          prefetch(g.out + ((uint64_t)z * g.M + i0 + lane) * g.N + j0 + c);
      float acc[W];
#pragma unroll
      for (int c = 0; c < W; ++c) acc[c] = 0.f;
      for (uint32_t k0 = sg.k0; k0 < sg.k1; k0 += kDrain, ++part) {
        const uint32_t buf = part % S::kBufs;
        ok = ok && mbar_wait(&done[buf], (part / S::kBufs) & 1, err);
        tc_fence_after();
        if (ok) {
#pragma unroll
          for (int c = 0; c < W; c += 32) {
            uint32_t v[32];
            tmem_load32(tmem + ((warp & 3) * 32u << 16) + buf * BN + side * W + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) acc[c + e] += __uint_as_float(v[e]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (rank == 0) mbar_arrive(&freed[buf]);
          else mbar_arrive_at(&freed[buf], 0);
        }
      }
      if (sg.count > 1) {                         // the tile is cut
        auto slot = [&](uint32_t w) {
          return reinterpret_cast<float4*>(
                     g.parts + (size_t)(2 * (PAIR ? 2 * w + rank : w) + (w == sg.first)) * (kRows * BN)) + threadIdx.x;
        };
        uint32_t* arrived = g.arrived + (PAIR ? 2 * sg.first + rank : sg.first);
        float4* mine = slot(worker);
#pragma unroll
        for (int c = 0; c < W / 4; ++c)
          __stcg(mine + c * 256, make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]));
        __threadfence();
        epilogue_sync();
        if (threadIdx.x == 0) order = atomicAdd(arrived, 1u);
        epilogue_sync();
        const bool last = order == sg.count - 1;
        if (!last) continue;
        __threadfence();
        if (threadIdx.x == 0) *arrived = 0;
        auto add = [&](uint32_t w) {
          const float4* p = slot(w);
#pragma unroll
          for (int c = 0; c < W / 4; ++c) {
            const float4 v = __ldcg(p + c * 256);
            acc[4 * c] += v.x;
            acc[4 * c + 1] += v.y;
            acc[4 * c + 2] += v.z;
            acc[4 * c + 3] += v.w;
          }
        };
        if (sg.count == 2) {                      // two sums: either order gives the same
          add(worker == sg.first ? sg.first + 1 : sg.first);
        } else {
#pragma unroll
          for (int c = 0; c < W; ++c) acc[c] = 0.f;
          for (uint32_t w = sg.first; w < sg.first + sg.count; ++w) add(w);
        }
      }
      const uint32_t i = i0 + lane;
#pragma unroll
      for (int c = 0; c < W; ++c) acc[c] *= g.sa;
      if (g.D.p && i0 < mchunks * 64) {
        if constexpr (W < 64) {
          const uint8_t* d = chunk_of(g.D, z, i >> 6, j0 >> 6);
#pragma unroll
          for (int e = 0; e < W; e += 8) {
            const uint8_t* p = d + chunk_at(i & 63, ((j0 & 63) + e) >> 3);
            add8(acc, e, g.sd, *reinterpret_cast<const uint4*>(p));
            add8(acc, e, g.sd, *reinterpret_cast<const uint4*>(p + kChunkBytes));
          }
        } else
#pragma unroll
        for (int c = 0; c < W; c += 64) {         // whole rows into the staging, then each thread its row
          if (j0 + c >= nchunks * 64) break;
          const uint8_t* d = chunk_of(g.D, z, i0 >> 6, (j0 + c) >> 6) + (i0 & 32) * 128;
#pragma unroll
          for (int low = 0; low < 2; ++low) {
            uint4 v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              v[e] = *reinterpret_cast<const uint4*>(d + low * kChunkBytes + (e * 32 + lane) * 16);
            if (lane == 0) bulk_store_read();     // an earlier tile's stores have left the staging
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) *reinterpret_cast<uint4*>(stage + (e * 32 + lane) * 16) = v[e];
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 64; e += 8)
              add8(acc, c + e, g.sd, *reinterpret_cast<const uint4*>(stage + chunk_at(lane, e >> 3)));
          }
        }
      }
      if (g.C) {
        // rows and columns behind M and N inside a chunk come out zero, as their operands are
        if (i0 >= mchunks * 64) continue;
        if constexpr (W < 64) {                   // half rows of a chunk do not lie together: no bulk copy
          uint8_t* o = g.C + z * g.c_z + ((uint64_t)(i0 >> 6) * g.c_cb + (j0 >> 6)) * kPairBytes;
#pragma unroll
          for (int e = 0; e < W; e += 8) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) split2(acc[e + 2 * q], acc[e + 2 * q + 1], h[q], l[q]);
            uint8_t* p = o + chunk_at(i & 63, ((j0 & 63) + e) >> 3);
            *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(p + kChunkBytes) = make_uint4(l[0], l[1], l[2], l[3]);
          }
        } else
#pragma unroll
        for (int c = 0; c < W; c += 64) {
          const uint32_t j = j0 + c;
          if (j >= nchunks * 64) break;
          uint8_t* o = g.C + z * g.c_z + ((uint64_t)(i0 >> 6) * g.c_cb + (j >> 6)) * kPairBytes + (i0 & 32) * 128;
#pragma unroll
          for (int low = 0; low < 2; ++low) {
            if (lane == 0) bulk_store_read();     // the staging is free again
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 64; e += 8) {
              uint32_t h[4], l[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) split2(acc[c + e + 2 * q], acc[c + e + 2 * q + 1], h[q], l[q]);
              *reinterpret_cast<uint4*>(stage + chunk_at(lane, e >> 3)) =
                  low ? make_uint4(l[0], l[1], l[2], l[3]) : make_uint4(h[0], h[1], h[2], h[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) bulk_store(o + low * kChunkBytes, stage, kStaging);
          }
        }
      } else {
        // through the staging, so that a warp reads and writes whole rows of 32 floats
#pragma unroll
        for (int c = 0; c < W; c += 32) {
          float* t = reinterpret_cast<float*>(stage);
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 32; ++e) t[lane * 32 + ((e + lane) & 31)] = acc[c + e];
          __syncwarp();
          const uint32_t j = j0 + c + lane;
          if (j < g.N) {
            float* o = g.out + ((uint64_t)z * g.M + i0) * g.N + j;
            const uint32_t rows = i0 < g.M ? min(32u, g.M - i0) : 0;
#pragma unroll
            for (uint32_t r = 0; r < 32; r += 16) {          // 16 rows of w in flight
              float old[16];
              if (g.update) {
#pragma unroll
                for (uint32_t e = 0; e < 16; ++e)
                  if (r + e < rows) old[e] = o[(uint64_t)(r + e) * g.N];
              }
#pragma unroll
              for (uint32_t e = 0; e < 16; ++e) {
                const float v = t[(r + e) * 32 + ((lane + r + e) & 31)];
                if (r + e < rows) o[(uint64_t)(r + e) * g.N] = g.update ? fmaf(-g.rate, v, g.keep * old[e]) : v;
              }
            }
          }
        }
      }
    }
    if (lane == 0) bulk_store_done();
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync();             // no arrival may reach a block that has ended
  else __syncthreads();
  tc_fence_after();
  if (warp == kEpi + 1) {
    if constexpr (PAIR) tmem_free_pair(tmem, S::kBufs * BN);
    else tmem_free(tmem, S::kBufs * BN);
  }
}

// ---------------------------------------------------------------------------
// momentum, norm, first split
// ---------------------------------------------------------------------------
constexpr int kMostParts = 1024;    // partial sums of squares per matrix

DCT_DEV float updated(const MuonArgs& a, float m, float g) { return fmaf(a.momentum, m, g); }
DCT_DEV float direction(const MuonArgs& a, float m, float g) {     // m after its update
  return !a.update ? g : a.nesterov ? fmaf(a.momentum, m, g) : m;
}

// m = momentum m + g, and the sums of squares of the direction, a part per block; 12 bytes
// an element (4 without the update), bound by memory
template <int V>
__global__ void __launch_bounds__(256) k_muon_momentum(const __grid_constant__ MuonArgs a, double* part,
                                                       uint32_t* arrived, uint32_t blocks) {
  __shared__ double sh[32];
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (uint32_t i = threadIdx.x; i < blocks; i += 256) arrived[i] = 0;
  const uint64_t n = (uint64_t)a.rows * a.cols / V, base = blockIdx.y * n;
  double s = 0.0;
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += 256ull * gridDim.x) {
    float g[V], m[V];
    if constexpr (V == 4) {
      *reinterpret_cast<float4*>(g) = reinterpret_cast<const float4*>(a.g)[base + i];
      if (a.update) *reinterpret_cast<float4*>(m) = reinterpret_cast<const float4*>(a.m)[base + i];
    } else {
      g[0] = a.g[base + i];
      if (a.update) m[0] = a.m[base + i];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      m[e] = a.update ? updated(a, m[e], g[e]) : 0.f;
      const float x = direction(a, m[e], g[e]);
      s += (double)x * x;
    }
    if (!a.update) continue;
    if constexpr (V == 4) reinterpret_cast<float4*>(a.m)[base + i] = *reinterpret_cast<const float4*>(m);
    else a.m[base + i] = m[0];
  }
  s = block_sum(s, sh);
  if (threadIdx.x == 0) part[blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// 1 / (norm + eps) of the block's matrix, in every thread
DCT_DEV double inverse_norm(const MuonArgs& a, const double* part, uint32_t parts) {
  __shared__ double sh[32], inv;
  const double s = block_sum(strided_sum(part + (uint64_t)blockIdx.y * parts, parts), sh);
  if (threadIdx.x == 0) inv = 1.0 / (sqrt(s) + a.eps);
  __syncthreads();
  return inv;
}

// the chunks of X = direction / (norm + eps), a thread per 8 columns of a row
template <int V>
__global__ void __launch_bounds__(256) k_muon_split(const __grid_constant__ MuonArgs a, const double* part,
                                                    uint32_t parts, uint8_t* x, uint32_t rb, uint32_t cb, float scale) {
  const uint32_t z = blockIdx.y;
  const double f = inverse_norm(a, part, parts) * scale;
  const uint64_t base = (uint64_t)z * a.rows * a.cols, groups = (uint64_t)rb * 64 * cb * 8;
  for (uint64_t t = blockIdx.x * 256ull + threadIdx.x; t < groups; t += 256ull * gridDim.x) {
    const uint32_t i = (uint32_t)(t / (cb * 8)), c = (uint32_t)(t % (cb * 8));
    const uint64_t at = base + (uint64_t)i * a.cols + c * 8;
    float g[8], m[8];
#pragma unroll
    for (int e = 0; e < 8; e += V) {
      const bool in = i < a.rows && c * 8 + e < a.cols;
      if constexpr (V == 4) {
        const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(g + e) = in ? *reinterpret_cast<const float4*>(a.g + at + e) : none;
        *reinterpret_cast<float4*>(m + e) = in && a.update ? *reinterpret_cast<const float4*>(a.m + at + e) : none;
      } else {
        g[e] = in ? a.g[at + e] : 0.f;
        m[e] = in && a.update ? a.m[at + e] : 0.f;
      }
    }
    uint32_t h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      split2((float)(direction(a, m[2 * e], g[2 * e]) * f), (float)(direction(a, m[2 * e + 1], g[2 * e + 1]) * f), h[e],
             l[e]);
    uint8_t* o = x + (((uint64_t)z * rb + (i >> 6)) * cb + (c >> 3)) * kPairBytes + chunk_at(i & 63, c & 7);
    *reinterpret_cast<uint4*>(o) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(o + kChunkBytes) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// no steps: the result is X itself
__global__ void __launch_bounds__(256) k_muon_apply(const __grid_constant__ MuonArgs a, const double* part,
                                                    uint32_t parts) {
  const uint64_t n = (uint64_t)a.rows * a.cols;
  const double inv = inverse_norm(a, part, parts);
  for (uint64_t t = blockIdx.x * 256ull + threadIdx.x; t < n; t += 256ull * gridDim.x) {
    const uint64_t i = blockIdx.y * n + t;
    const float x = (float)(direction(a, a.update ? a.m[i] : 0.f, a.g[i]) * inv);
    if (a.update) a.w[i] = fmaf(-a.rate, x, a.keep * a.w[i]);
    else a.y[i] = x;
  }
}

// ---------------------------------------------------------------------------
// short matrices: everything in one launch
// ---------------------------------------------------------------------------
// With a shorter side of 128 or less, what bounds the products above is not their work but
// their number: each is a launch of one or a few tiles, about 9 us from its first load to
// its last store.  Here a cluster holds a matrix: X^T or X as [shorter side][longer side],
// `chunks` columns of 64 a block in shared memory, from the first read of the gradient to
// the last step, and A and P in another 64 KB.  Only the blocks' sums of A meet, through L2
// (the cluster's shared memory measured slower: 81 us against 69 for 333 x 127).
constexpr int kMostChunks = 5;
struct Small {
  MuonArgs a;
  uint32_t side, length;         // the shorter and the longer side
  bool tall;                     // the matrix is [longer][shorter]
  int chunks;                    // of this cluster's blocks
  float *sums;                   // [matrix][block][128][128]
  float first;                   // scale of the first X
  float gram, poly_a, poly_b, next_p, next_x, last_p, last_x;    // powers of two and coefficients
};

DCT_DEV uint64_t at_small(const Small& g, uint32_t s, uint32_t t) {
  return g.tall ? (uint64_t)t * g.a.cols + s : (uint64_t)s * g.a.cols + t;
}

// a shared memory address in another block of the cluster
DCT_DEV uint32_t at_block(uint32_t addr, uint32_t block) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(block));
  return r;
}

// 16 warps: a thread holds a quarter (32 columns) of a row of A and P, and of every 64 columns
// of X.  The steps alternate between all threads and one that issues matrix instructions.
constexpr int kSmallThreads = 512;
__global__ void __launch_bounds__(kSmallThreads) k_muon_small(const __grid_constant__ Small g, uint32_t* err) {
  extern __shared__ __align__(1024) uint8_t sm[];
  __shared__ uint64_t bar, ready[kMostChunks];
  __shared__ uint32_t tmem_base;
  __shared__ double sh[32], square;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, C = g.chunks;
  uint8_t* ap = sm + C * 4 * kChunkBytes;         // A, then P: [64 columns][hi, lo][128 rows]
  const uint32_t rank = cluster_rank();
  uint32_t blocks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
  const uint32_t z = blockIdx.x / blocks, t0 = rank * C * 64;
  const uint64_t base = (uint64_t)z * g.a.rows * g.a.cols;
  if ((smem_addr(sm) & 1023) != 0) {              // uniform over the cluster
    if (err && threadIdx.x == 0) atomicOr(err, DCT_DEVERR_WAIT_TIMEOUT);
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    for (int k = 0; k < kMostChunks; ++k) mbar_init(&ready[k], 1);
    mbar_fence_init();
  }
  if (warp == 0) tmem_alloc(&tmem_base, 512);
  for (uint32_t i = threadIdx.x; i < C * 4 * kChunkBytes / 16; i += kSmallThreads)
    reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  // Momentum and norm.  The direction waits for its scale where the first X will lie, its
  // upper and lower 16 bits in the places of hi and lo.  A warp takes lines of memory.
  const uint32_t lines = g.tall ? min((uint32_t)C * 64, g.length > t0 ? g.length - t0 : 0) : g.side;
  const uint32_t across = g.tall ? g.side : min((uint32_t)C * 64, g.length > t0 ? g.length - t0 : 0);
  double part = 0.0;
  constexpr int kW = kSmallThreads / 32, kL = 4;  // lines in flight
  for (uint32_t l0 = warp; l0 < lines; l0 += kW * kL)
    for (uint32_t c0 = lane; c0 < across; c0 += 128) {
      float x[kL][4], m[kL][4];
#pragma unroll
      for (int j = 0; j < kL; ++j) {
        const uint32_t line = l0 + j * kW;
        const uint64_t from = base + (g.tall ? at_small(g, 0, t0 + line) : at_small(g, line, t0));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t c = c0 + e * 32;
          const bool in = line < lines && c < across;
          x[j][e] = in ? g.a.g[from + c] : 0.f;
          m[j][e] = g.a.update && in ? g.a.m[from + c] : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < kL; ++j) {
        const uint32_t line = l0 + j * kW;
        if (line >= lines) break;
        const uint64_t from = base + (g.tall ? at_small(g, 0, t0 + line) : at_small(g, line, t0));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t c = c0 + e * 32;
          if (c >= across) break;
          if (g.a.update) g.a.m[from + c] = m[j][e] = updated(g.a, m[j][e], x[j][e]);
          const float u = direction(g.a, m[j][e], x[j][e]);
          part += (double)u * u;
          const uint32_t s = g.tall ? c : line, k = g.tall ? line : c, bits = __float_as_uint(u);
          uint8_t* p = sm + (k >> 6) * 4 * kChunkBytes + chunk_at(s, (k & 63) >> 3) + 2 * (k & 7);
          *reinterpret_cast<uint16_t*>(p) = (uint16_t)(bits >> 16);
          *reinterpret_cast<uint16_t*>(p + 2 * kChunkBytes) = (uint16_t)bits;
        }
      }
    }
  part = block_sum(part, sh);
  if (threadIdx.x == 0) square = part;
  cluster_sync();
  double all = 0.0;
  for (uint32_t b = 0; b < blocks; ++b) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at_block(smem_addr(&square), b)) : "memory");
    all += v;
  }
  const double f = (double)g.first / (sqrt(all) + g.a.eps);
  for (uint32_t i = threadIdx.x; i < C * 2 * kChunkBytes / 16; i += kSmallThreads) {
    uint4* h = reinterpret_cast<uint4*>(sm + i / (2 * kChunkBytes / 16) * 4 * kChunkBytes) + i % (2 * kChunkBytes / 16);
    uint4* l = h + 2 * kChunkBytes / 16;
    const uint32_t hh[4] = {h->x, h->y, h->z, h->w}, ll[4] = {l->x, l->y, l->z, l->w};
    uint32_t u[4], v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      split2((float)(__uint_as_float(hh[e] << 16 | (ll[e] & 0xffff)) * f),
             (float)(__uint_as_float((hh[e] & 0xffff0000u) | ll[e] >> 16) * f), u[e], v[e]);
    *h = make_uint4(u[0], u[1], u[2], u[3]);
    *l = make_uint4(v[0], v[1], v[2], v[3]);
  }

  const uint32_t row = (warp & 3) * 32 + lane, quarter = warp >> 2, lanes = (uint32_t)(warp & 3) * 32u << 16;
  bool ok = true;
  uint32_t phase = 0;
  auto to_tensor = [&]() {
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };
  auto from_tensor = [&]() {
    ok = ok && mbar_wait(&bar, phase & 1, err);
    ++phase;
    tc_fence_after();
  };
  auto three = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t step_a, uint32_t step_b, uint64_t lo, uint32_t idesc,
                   bool add, int deep) {          // 16 `deep` of the contraction
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q >= deep) break;
      umma(d, a + lo + q * step_a, b + q * step_b, idesc, add || q != 0);
      umma(d, a + q * step_a, b + lo + q * step_b, idesc, true);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < deep) umma(d, a + q * step_a, b + q * step_b, idesc, true);
  };
  // rows of the shorter side in 16s: all the columns of A and P, and the contraction with them
  const int wide = (int)(g.side + 15) / 16, deep0 = min(wide, 4), deep1 = wide - deep0;
  const int cols = min(max(16 * wide - (int)quarter * 32, 0), 32);     // of the thread's columns (the rest stays 0)
  constexpr uint64_t kLow = 2 * kChunkBytes / 16;                 // from hi to lo of 128 rows
  constexpr uint32_t kBlock = 4 * kChunkBytes / 16;               // from 64 columns to the next
  const uint64_t x = umma_desc(smem_addr(sm), kChunkBytes, 1024), p = umma_desc(smem_addr(ap), kChunkBytes, 1024);
  for (uint32_t it = 0; it < g.a.steps; ++it) {
    const bool last = it + 1 == g.a.steps;
    // A = X X^T: every 64 columns an accumulator of their own (the fifth joins the first)
    to_tensor();
    if (warp == 0 && elect_one()) {
      const uint32_t id = umma_idesc(128, 16 * wide, false, false);
      for (int k = 0; k < C; ++k) three(tmem + (k & 3) * 128, x + k * kBlock, x + k * kBlock, 2, 2, kLow, id, k > 3, 4);
      umma_commit(&bar);
    }
    from_tensor();
    float acc[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) acc[e] = 0.f;
    for (int k = 0; k < min(C, 4) && cols > 0; ++k) {
      uint32_t v[32];
      tmem_load32(tmem + lanes + k * 128 + quarter * 32, v);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (e < cols) acc[e] += __uint_as_float(v[e]);
    }
    if (blocks > 1) {                             // the blocks' sums meet, added in the blocks' order
      float* mine = g.sums + ((uint64_t)z * blocks + rank) * 16384 + quarter * 32 * 128 + row;
      if (cols > 0) {
#pragma unroll
        for (int e = 0; e < 32; ++e) __stcg(mine + e * 128, acc[e]);
      }
      __threadfence();
      cluster_sync();
      if (cols > 0) {
        const float* from = g.sums + (uint64_t)z * blocks * 16384 + quarter * 32 * 128 + row;
#pragma unroll
        for (int e = 0; e < 32; ++e) acc[e] = 0.f;
        for (uint32_t b = 0; b < blocks; ++b) {
#pragma unroll
          for (int e = 0; e < 32; ++e) acc[e] += __ldcg(from + b * 16384 + e * 128);
        }
      }
      cluster_sync();                             // before the next step's sums
    }
    auto store = [&](const float (&v)[32]) {      // the thread's columns of A or P
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) split2(v[e + 2 * q], v[e + 2 * q + 1], h[q], l[q]);
        uint8_t* o = ap + (quarter >> 1) * 4 * kChunkBytes + chunk_at(row, (quarter & 1) * 4 + (e >> 3));
        *reinterpret_cast<uint4*>(o) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(o + 2 * kChunkBytes) = make_uint4(l[0], l[1], l[2], l[3]);
      }
    };
#pragma unroll
    for (int e = 0; e < 32; ++e) acc[e] *= g.gram;
    store(acc);
    // P = c A A + b A
    to_tensor();
    if (warp == 0 && elect_one()) {
      const uint32_t id = umma_idesc(128, 16 * wide, false, false);
      three(tmem, p, p, 2, 2, kLow, id, false, deep0);
      if (deep1) three(tmem + 128, p + kBlock, p + kBlock, 2, 2, kLow, id, false, deep1);
      umma_commit(&bar);
    }
    from_tensor();
    if (cols > 0) {
      uint32_t v[32], w[32];
      tmem_load32(tmem + lanes + quarter * 32, v);
      if (deep1) tmem_load32(tmem + lanes + 128 + quarter * 32, w);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        if (e >= cols) continue;
        const float s = deep1 ? __uint_as_float(v[e]) + __uint_as_float(w[e]) : __uint_as_float(v[e]);
        acc[e] = fmaf(g.poly_b, acc[e], g.poly_a * s);
      }
    }
    store(acc);
    // X = P X + a X, the two halves of the contraction apart where tensor memory has room
    to_tensor();
    const bool apart = C <= 4 && deep1;
    if (warp == 0 && elect_one()) {
      constexpr uint32_t id = umma_idesc(128, 64, false, true);
      for (int k = 0; k < C; ++k) {
        for (int h = 0; h < (deep1 ? 2 : 1); ++h)
          three(tmem + (apart ? 2 * k + h : k) * 64, p + h * kBlock, x + k * kBlock + h * (kChunkBytes / 16), 2, 128,
                kLow, id, !apart && h, h ? deep1 : deep0);
        umma_commit(&ready[k]);
      }
    }
    const float sp = last ? g.last_p : g.next_p, sx = last ? g.last_x : g.next_x;
    for (int k = 0; k < C; ++k) {
      ok = ok && mbar_wait(&ready[k], it & 1, err);
      tc_fence_after();
      uint32_t v[16];
      float y[16];
      tmem_load16(tmem + lanes + (apart ? 2 * k : k) * 64 + quarter * 16, v);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = __uint_as_float(v[e]);
      if (apart) {
        tmem_load16(tmem + lanes + (2 * k + 1) * 64 + quarter * 16, v);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] += __uint_as_float(v[e]);
      }
#pragma unroll
      for (int e = 0; e < 16; e += 8) {
        uint8_t* o = sm + k * 4 * kChunkBytes + chunk_at(row, quarter * 2 + (e >> 3));
        const uint4 h = *reinterpret_cast<const uint4*>(o), l = *reinterpret_cast<const uint4*>(o + 2 * kChunkBytes);
#pragma unroll
        for (int q = 0; q < 8; ++q) y[e + q] *= sp;
        add8(y, e, sx, h);
        add8(y, e, sx, l);
        if (!last) {
          uint32_t hh[4], ll[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) split2(y[e + 2 * q], y[e + 2 * q + 1], hh[q], ll[q]);
          *reinterpret_cast<uint4*>(o) = make_uint4(hh[0], hh[1], hh[2], hh[3]);
          *reinterpret_cast<uint4*>(o + 2 * kChunkBytes) = make_uint4(ll[0], ll[1], ll[2], ll[3]);
        }
      }
      if (last && row < g.side) {
        const uint32_t t = t0 + k * 64 + quarter * 16;
        const uint64_t first = base + at_small(g, row, t), step = g.tall ? g.a.cols : 1;
        float old[16];
        if (g.a.update) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (t + e < g.length) old[e] = g.a.w[first + e * step];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (t + e >= g.length) break;
          if (g.a.update) g.a.w[first + e * step] = fmaf(-g.a.rate, y[e], g.a.keep * old[e]);
          else g.a.y[first + e * step] = y[e];
        }
      }
    }
  }
  tc_fence_before();
  cluster_sync();                                 // the others have read this block's square
  tc_fence_after();
  if (warp == 0) tmem_free(tmem, 512);
}

// One block an SM, whatever it needs: each takes all 512 columns of tensor memory, and two
// clusters that share SMs could each hold the columns that the other waits for.
constexpr size_t kSmShared = 228 * 1024;          // of an SM
constexpr size_t small_smem(int chunks) {
  const size_t need = (size_t)(chunks + 2) * 4 * kChunkBytes, alone = kSmShared / 2 + 1024;
  return need > alone ? need : alone;
}
static_assert(2 * small_smem(1) > kSmShared && small_smem(kMostChunks) <= 227 * 1024);

// Blocks of a matrix's cluster, or 0 where the general way takes it.  A chunk costs a block
// about 2300 cycles a step, the meeting of several blocks' sums 6800.
int small_blocks(const MuonArgs& a) {
  const uint32_t s = std::min(a.rows, a.cols), chunks = (std::max(a.rows, a.cols) + 63) / 64;
  if (s > 128 || !a.steps || chunks > 8 * kMostChunks) return 0;
  int best = 0;
  uint32_t cost = ~0u;
  for (uint32_t n = 1; n <= 8; ++n) {
    const uint32_t c = (chunks + n - 1) / n, want = c * 2300 + (n > 1 ? 6800 : 0);
    if (c > kMostChunks || (n - 1) * c >= chunks || want >= cost) continue;
    cost = want;
    best = (int)n;
  }
  return best;
}

// Scratch of one launch's matrices.  A thin matrix is padded to 64 on its short side, up to 128
// times its data with both copies of X, so a batch goes in groups that stay below this.
constexpr uint64_t kMostScratch = 2ull << 30;

struct Layout {
  uint32_t rb, cb, sb;              // chunks of rows, columns, the shorter side
  uint64_t x, s;                    // bytes of X's and of a Gram matrix's chunks
  size_t x0 = 0, x1 = 0, gram = 0, poly = 0, part, cut = 0, arrived, total;
  explicit Layout(const MuonArgs& a) {
    rb = (a.rows + 63) / 64;
    cb = (a.cols + 63) / 64;
    sb = rb < cb ? rb : cb;
    x = (uint64_t)rb * cb * kPairBytes;
    s = (uint64_t)sb * sb * kPairBytes;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += (bytes + 1023) & ~size_t(1023); return o; };
    part = take(8 * kMostParts * (size_t)a.batch);
    arrived = take(sizeof(uint32_t) * dev_info().sm_count);
    if (a.steps) {                  // without, the direction is only scaled
      x0 = take(x * a.batch);
      x1 = take(x * a.batch);
      gram = take(s * a.batch);
      poly = take(s * a.batch);
      cut = take(2ull * dev_info().sm_count * kRows * 256 * sizeof(float));
    }
    total = at;
  }
  static uint64_t a_matrix(const MuonArgs& a) {
    MuonArgs one = a;
    one.batch = 1;
    const Layout l(one);
    return 8 * kMostParts + (a.steps ? 2 * (l.x + l.s) : 0);
  }
};

// Workers that run at once: every SM, or the pairs that the device can place.
template <typename K>
cudaError_t workers_of(K kernel, bool pair, size_t smem, int* workers) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) e = launched_with(kernel, kThreads, kRegs);
  *workers = dev_info().sm_count;
  if (e != cudaSuccess || !pair) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(2 * (dev_info().sm_count / 2));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(workers, kernel, &cfg);
}

template <bool PAIR, int BN>
cudaError_t product_as(Product g, uint32_t batch, cudaStream_t st) {
  using S = Shape<PAIR, BN>;
  const auto kernel = k_product<PAIR, BN>;
  static int most = 0;
  static const cudaError_t set = workers_of(kernel, PAIR, S::kSmem, &most);
  if (set != cudaSuccess) return set;
  if (most < 1 || (PAIR ? 2 : 1) * most > dev_info().sm_count) return cudaErrorInvalidConfiguration;
  g.mt = (g.M + S::kTileRows - 1) / S::kTileRows;
  g.nt = (g.N + BN - 1) / BN;
  g.tiles = g.mt * g.nt;
  if (g.half) g.tiles = g.mt * (g.mt + 1) / 2;
  const uint64_t total = (uint64_t)g.tiles * batch, work = total * g.kb;
  if (total >= (1ull << 31) || g.kb > (1u << 17)) return cudaErrorInvalidConfiguration;
  // The tiles that do not go around: whole, or cut in runs of 4 chunks or more (2 of the
  // smallest tiles), whichever ends first.  A cut tile's meeting in memory costs about as
  // much as 6 chunks (when this rule was chosen, one matrix of 1024 x 8192: 700 us cut,
  // 1079 us whole; twelve of 768 x 768: 552 and 550 us).
  constexpr uint64_t kShortest = BN == 64 ? 2 : 4, kMeeting = 6;
  const uint64_t workers = std::min<uint64_t>(work / kShortest + 1, most), left = total % workers;
  const uint64_t cut = std::max<uint64_t>(kShortest, (left * g.kb + workers - 1) / workers) + kMeeting;
  const uint32_t unit = g.kb <= cut ? g.kb : 1;
  const uint64_t used = std::min<uint64_t>(unit == 1 ? (left * g.kb + kShortest - 1) / kShortest : left, workers);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = PAIR ? 2 : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)workers * (PAIR ? 2 : 1));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, g, (uint32_t)total, unit, (uint32_t)used, device_error_word());
}

// The tile of a call's products: its rows and columns, of which symmetric results store
// the lower half (64: one tile of a result no larger than that).
cudaError_t product(int tile, const Product& g, uint32_t batch, cudaStream_t st) {
  if (tile == 64) return product_as<false, 64>(g, batch, st);
  if (tile == 128) return product_as<false, 128>(g, batch, st);
  return product_as<true, 256>(g, batch, st);
}

// Pairs with tiles of 256 where these fill a fifth of the SMs or more with one symmetric
// product (twelve of 768 x 768: 479 us, 509 with tiles of 128; 4096 x 4096: 3.3 ms, 4.9);
// below, smaller tiles divide better (1500 x 1500: 519 us, 419 with 128; 256 x 1000: 259, 173
// and 159 with 64; 512 x 2048: 327, 222 and 214).
int tile_of(const MuonArgs& a) {
  const uint64_t s = std::min(a.rows, a.cols), n = (s + 255) / 256;
  return n * (n + 1) / 2 * a.batch * 5 >= (uint64_t)dev_info().sm_count ? 256 : s <= 512 ? 64 : 128;
}

// the power of two that brings `most` to at most 2^15
int room(double most) {
  int e;
  frexp(most, &e);           // most <= 2^e
  return 15 - e;
}
float pow2(int e) { return (float)ldexp(1.0, e); }
// exponents at which X, A and P are held: no entry of X exceeds its largest singular value,
// none of A that squared, none of P b t + c t^2 on those
struct Powers {
  int x, g, p;
  explicit Powers(const MuonArgs& a) {
    const double top = a.bound * a.bound, most = std::max(1e-30, fabs(a.b) * top + fabs(a.c) * top * top);
    x = room(a.bound);
    g = room(top);
    p = room(most);
  }
};

// The matrices of a launch: all, or as many as the scratch allows, in groups of (almost) one size.
uint32_t group_of(const MuonArgs& a) {
  const int n = small_blocks(a);
  const uint64_t one = n ? (n > 1 ? n * 16384 * sizeof(float) : 0) : Layout::a_matrix(a);
  const uint64_t most = one ? std::max<uint64_t>(1, kMostScratch / one) : a.batch;
  if (a.batch <= most) return a.batch;
  const uint32_t groups = (uint32_t)((a.batch + most - 1) / most);
  return (a.batch + groups - 1) / groups;
}

cudaError_t launch_small(const MuonArgs& a, int blocks, void* ws, cudaStream_t st) {
  Small g{};
  g.a = a;
  g.tall = a.rows > a.cols;
  g.side = std::min(a.rows, a.cols);
  g.length = std::max(a.rows, a.cols);
  g.chunks = (int)(((g.length + 63) / 64 + blocks - 1) / blocks);
  g.sums = static_cast<float*>(ws);
  const Powers w(a);
  g.first = pow2(w.x);
  g.gram = pow2(w.g - 2 * w.x);
  g.poly_a = (float)(a.c * pow2(w.p - 2 * w.g));
  g.poly_b = (float)(a.b * pow2(w.p - w.g));
  g.next_p = pow2(-w.p);
  g.next_x = (float)a.a;
  g.last_p = pow2(-w.x - w.p);
  g.last_x = (float)(a.a * pow2(-w.x));
  const size_t smem = small_smem(g.chunks);
  static const cudaError_t set = cudaFuncSetAttribute(k_muon_small, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                      (int)small_smem(kMostChunks));
  if (set != cudaSuccess) return set;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(a.batch * blocks);
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_muon_small, g, device_error_word());
}

cudaError_t launch_group(const MuonArgs& a, void* ws, cudaStream_t st) {
  if (const int n = small_blocks(a)) return launch_small(a, n, ws, st);
  const Layout L(a);
  uint8_t* w = static_cast<uint8_t*>(ws);
  uint8_t *x = w + L.x0, *y = w + L.x1;
  double* part = reinterpret_cast<double*>(w + L.part);
  uint32_t* arrived = reinterpret_cast<uint32_t*>(w + L.arrived);
  const uint64_t n = (uint64_t)a.rows * a.cols;
  const bool vec = a.cols % 4 == 0 && aligned16_h(a.g) && (!a.update || aligned16_h(a.m));
  // blocks a matrix: a thread takes 16 elements or more, the batch eight blocks an SM
  const uint32_t across = (uint32_t)std::max<uint64_t>(
      1, std::min<uint64_t>(std::min<uint64_t>((n + 4095) / 4096, kMostParts), 8ull * dev_info().sm_count / a.batch));
  const dim3 grid(across, a.batch);
  if (vec) k_muon_momentum<4><<<grid, 256, 0, st>>>(a, part, arrived, dev_info().sm_count);
  else k_muon_momentum<1><<<grid, 256, 0, st>>>(a, part, arrived, dev_info().sm_count);
  if (!a.steps) {
    k_muon_apply<<<grid, 256, 0, st>>>(a, part, across);
    return cudaGetLastError();
  }
  const Powers powers(a);
  const int ex = powers.x, eg = powers.g, ep = powers.p;
  if (vec) k_muon_split<4><<<grid, 256, 0, st>>>(a, part, across, x, L.rb, L.cb, pow2(ex));
  else k_muon_split<1><<<grid, 256, 0, st>>>(a, part, across, x, L.rb, L.cb, pow2(ex));
  cudaError_t e = cudaGetLastError();
  const bool wide = a.rows <= a.cols;
  const uint32_t S = wide ? a.rows : a.cols;
  const int tile = tile_of(a);
  Product base{};
  base.parts = reinterpret_cast<float*>(w + L.cut);
  base.arrived = arrived;
  for (uint32_t i = 0; i < a.steps && e == cudaSuccess; ++i) {
    const Operand X{x, L.cb, L.x, false, false}, XT{x, L.cb, L.x, true, false};
    const Operand A{w + L.gram, L.sb, L.s, false, tile > 64}, P{w + L.poly, L.sb, L.s, false, tile > 64};
    Product g = base;
    g.A = g.B = wide ? X : XT;
    g.C = w + L.gram; g.c_cb = L.sb; g.c_z = L.s;
    g.sa = pow2(eg - 2 * ex);
    g.M = g.N = S; g.kb = wide ? L.cb : L.rb;
    g.half = tile > 64;
    e = product(tile, g, a.batch, st);
    if (e != cudaSuccess) break;
    Product p = base;
    p.A = p.B = p.D = A;
    p.C = w + L.poly; p.c_cb = L.sb; p.c_z = L.s;
    p.sa = (float)(a.c * pow2(ep - 2 * eg));
    p.sd = (float)(a.b * pow2(ep - eg));
    p.M = p.N = S; p.kb = L.sb;
    p.half = tile > 64;
    e = product(tile, p, a.batch, st);
    if (e != cudaSuccess) break;
    const bool last = i + 1 == a.steps;
    Product q = base;
    q.D = X;
    q.A = wide ? P : X;
    q.B = wide ? XT : P;
    q.M = a.rows; q.N = a.cols; q.kb = L.sb;
    q.sa = pow2((last ? 0 : ex) - ex - ep);
    q.sd = (float)(a.a * pow2((last ? 0 : ex) - ex));
    if (last) {
      q.out = a.update ? a.w : a.y;
      q.update = a.update; q.keep = a.keep; q.rate = a.rate;
    } else {
      q.C = y; q.c_cb = L.cb; q.c_z = L.x;
    }
    e = product(tile, q, a.batch, st);
    std::swap(x, y);
  }
  return e;
}

}  // namespace

size_t muon_ws_bytes(const MuonArgs& a) {
  if (!a.rows || !a.cols || !a.batch) return 0;
  MuonArgs g = a;
  g.batch = group_of(a);
  if (const int n = small_blocks(g)) return n > 1 ? (size_t)g.batch * n * 16384 * sizeof(float) : 0;
  return Layout(g).total;
}

cudaError_t launch_muon(const MuonArgs& a, void* ws, cudaStream_t st) {
  if (!a.rows || !a.cols || !a.batch) return cudaSuccess;
  const uint32_t most = group_of(a);
  cudaError_t e = cudaSuccess;
  for (uint32_t z = 0; z < a.batch && e == cudaSuccess; z += most) {
    MuonArgs g = a;
    const uint64_t at = (uint64_t)z * a.rows * a.cols;
    g.batch = std::min(most, a.batch - z);
    g.g += at;
    if (a.update) { g.w += at; g.m += at; }
    else g.y += at;
    e = launch_group(g, ws, st);
  }
  return e;
}

}  // namespace dct
