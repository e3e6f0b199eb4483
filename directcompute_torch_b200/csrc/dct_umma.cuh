// Fifth-generation tensor core helpers for sm_100a (tcgen05, tensor memory), as inline PTX,
// and float32 operands for them.
//
// A float32 operand is held as two float16 numbers, 2^e x = hi + lo with hi the nearest
// float16 and lo the nearest to the rest: |2^e x - hi - lo| <= max(2^-23 |hi|, 2^-25) (half
// a step of lo, whose own size is at most half a step of hi; 2^-25 is half float16's
// smallest step).  A product of two such operands is hi hi + hi lo + lo hi, three matrix
// instructions into one float32 accumulator; the lo lo that is left out is at most 2^-22 of
// the product.  The power of two e puts the largest magnitude near 2^15.
//
// Operands lie in memory as they will lie in shared memory: chunks of 64 rows x 64 columns
// of float16 (8 KB), row r at 128 r, its 16-byte column group c at 16 (c ^ (r & 7)), the
// 128-byte swizzle that the matrix instructions read without bank conflicts.  So a plain
// bulk copy brings a chunk in.  The same chunk serves with its columns as the contraction
// (K-major: 8-row groups 1024 bytes apart) and with its rows as the contraction (MN-major:
// 64 columns wide panels one chunk apart, 8-row groups 1024 bytes apart).
#pragma once
#include <cuda_fp16.h>

#include "dct_tma.cuh"

namespace dct {

constexpr uint32_t kChunkBytes = 8192;       // 64 x 64 float16
constexpr uint32_t kPairBytes = 2 * kChunkBytes;   // hi and lo

// byte offset of (row, 8-column group) inside a chunk
DCT_DEV uint32_t chunk_at(uint32_t row, uint32_t group) { return row * 128 + ((group ^ (row & 7)) << 4); }

// two scaled floats as packed hi and lo
DCT_DEV void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
// the sum of packed hi and lo
DCT_DEV float2 join2(uint32_t hi, uint32_t lo) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  return make_float2(h.x + l.x, h.y + l.y);
}

// bulk copy of shared memory to global memory (addresses and size multiples of 16), and the
// wait until the copies of this thread have been read out of shared memory / have landed
DCT_DEV void bulk_store(void* gmem_dst, const void* smem_src, uint32_t bytes) {
  asm volatile(
      "cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\t"
      "cp.async.bulk.commit_group;" ::"l"(gmem_dst),
      "r"(smem_addr(smem_src)), "r"(bytes)
      : "memory");
}
DCT_DEV void bulk_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
DCT_DEV void bulk_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ---- tensor memory ------------------------------------------------------------
// one warp allocates `cols` columns (a power of two >= 32) and later frees them
DCT_DEV void tmem_alloc(uint32_t* smem_out, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(smem_out)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
DCT_DEV void tmem_free(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
DCT_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
DCT_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
DCT_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
DCT_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: thread l gets columns addr .. addr + 31 of lane l
DCT_DEV void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
DCT_DEV void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

DCT_DEV void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
DCT_DEV void tmem_store8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
DCT_DEV void tmem_load(uint32_t addr, uint32_t (&r)[32]) { tmem_load32(addr, r); }
DCT_DEV void tmem_load(uint32_t addr, uint32_t (&r)[16]) { tmem_load16(addr, r); }
DCT_DEV void tmem_store(uint32_t addr, const uint32_t (&r)[16]) { tmem_store16(addr, r); }
DCT_DEV void tmem_store(uint32_t addr, const uint32_t (&r)[8]) { tmem_store8(addr, r); }

// Reads a kernel's parameters, a word of every 64 bytes, so that they are in the constant cache
// before the wait for the kernel before is over (attention of 4096 tokens: 1 to 2%).
template <typename T>
DCT_DEV void touch(const T& p) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&p);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); i += 16) asm volatile("" ::"r"(w[i]));
}

// One thread of a converged warp.  The compiler knows that a branch on it has one thread, and
// forms the operands of the instructions inside in uniform registers; behind `lane == 0` it
// moves each there, and with busy warps beside it the issuing warp then took 550 cycles for
// a matrix instruction of 64 (72 with this).
DCT_DEV bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}

// Whether a block of `kernel` is launched with at least `need` registers in all: what its
// warps take (setmaxnreg) from what they give up must be there, or they would wait for ever.
template <typename K>
inline cudaError_t launched_with(K kernel, int threads, int need) {
  cudaFuncAttributes a{};
  const cudaError_t e = cudaFuncGetAttributes(&a, kernel);
  if (e != cudaSuccess) return e;
  return (a.numRegs + 7) / 8 * 8 * threads >= need ? cudaSuccess : cudaErrorInvalidConfiguration;
}

// ---- matrix instructions ---------------------------------------------------------
// Shared memory descriptor of a 128-byte swizzled operand (start address, leading and
// stride byte offsets in units of 16; version 1; swizzle mode 2).
DCT_DEV uint64_t umma_desc(uint32_t addr, uint32_t leading, uint32_t stride) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((leading >> 4) & 0x3fff) << 16 |
         (uint64_t)((stride >> 4) & 0x3fff) << 32 | 1ull << 46 | 2ull << 61;
}
// Instruction descriptor: float32 accumulator, float16 operands, M x N tile; `mn` says that
// an operand's rows are the contraction
constexpr uint32_t umma_idesc(uint32_t M, uint32_t N, bool a_mn, bool b_mn) {
  return 1u << 4 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (N >> 3) << 17 | (M >> 4) << 24;
}
// D (tensor memory) = A B, or D += A B; 16 deep; one thread issues it
DCT_DEV void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
      "r"((uint32_t)add)
      : "memory");
}
// the same with A in tensor memory: lane = row, column c = elements 2c, 2c + 1
DCT_DEV void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
      "r"((uint32_t)add)
      : "memory");
}
// arrives on `bar` when the matrix instructions that this thread issued are done
DCT_DEV void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}

DCT_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// ---- pairs: two blocks of a cluster on one tile -----------------------------------
// The even block issues for both: the tile's rows are split over the blocks (each holds
// its accumulator rows), and so are the columns of B in shared memory, which both read.
DCT_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
DCT_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
DCT_DEV void tmem_alloc_pair(uint32_t* smem_out, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(smem_out)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
DCT_DEV void tmem_free_pair(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
DCT_DEV void umma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
      "r"((uint32_t)add)
      : "memory");
}
// arrives on `bar` of both blocks when this thread's matrix instructions are done
DCT_DEV void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// arrive on the same barrier of block `rank` of the cluster
DCT_DEV void mbar_arrive_at(uint64_t* bar, uint32_t rank) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\t"
      "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_addr(bar)),
      "r"(rank)
      : "memory");
}
// mbar_wait for arrivals from the other block too
DCT_DEV bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t limit = 1u << 22) {
  for (uint32_t spins = 0; spins < limit; ++spins) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  if (err) atomicOr(err, DCT_DEVERR_WAIT_TIMEOUT);
  return false;
}

}  // namespace dct
