// Orthogonalisation by Newton-Schulz steps, and the optimizer update around it.
#include "dct_common.cuh"
#include "kernels.h"

namespace dct {
namespace {

constexpr int kTile = 64, kDepth = 16;

// C = alpha op(A) op(B) + beta D over a batch of matrices; element (i, k) of A lies at
// i * ai + k * ak, likewise B (k, j).  64 x 64 tiles, 4 x 4 outputs a thread.
struct Gemm {
  const float *A, *B, *D;
  float* C;
  int64_t ai, ak, bk, bj, cs;       // C and D row stride
  int64_t az, bz, cz;               // between matrices
  int M, N, K;
  float alpha, beta;
};
__global__ void __launch_bounds__(256) k_gemm(const __grid_constant__ Gemm g) {
  __shared__ float as[kDepth][kTile + 1], bs[kDepth][kTile + 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int i0 = blockIdx.y * kTile, j0 = blockIdx.x * kTile;
  const float* A = g.A + blockIdx.z * g.az;
  const float* B = g.B + blockIdx.z * g.bz;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < g.K; k0 += kDepth) {
    for (int t = threadIdx.x; t < kTile * kDepth; t += 256) {
      const int i = t / kDepth, k = t % kDepth;
      as[k][i] = i0 + i < g.M && k0 + k < g.K ? A[(i0 + i) * g.ai + (k0 + k) * g.ak] : 0.f;
      bs[k][i] = j0 + i < g.N && k0 + k < g.K ? B[(k0 + k) * g.bk + (j0 + i) * g.bj] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(as[k][ty + 16 * u], bs[k][tx + 16 * v], acc[u][v]);
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int i = i0 + ty + 16 * u, j = j0 + tx + 16 * v;
      if (i < g.M && j < g.N) {
        const int64_t at = blockIdx.z * g.cz + i * g.cs + j;
        g.C[at] = g.D ? fmaf(g.alpha, acc[u][v], g.beta * g.D[at]) : g.alpha * acc[u][v];
      }
    }
}

constexpr int kChunks = 64;         // partial sums of squares per matrix

// u = the matrix to orthogonalise (with the momentum update), and its sums of squares
__global__ void __launch_bounds__(256) k_muon_momentum(const __grid_constant__ MuonArgs a, float* u, double* part) {
  __shared__ double sh[32];
  const uint64_t n = (uint64_t)a.rows * a.cols, per = (n + kChunks - 1) / kChunks;
  const uint64_t base = blockIdx.y * n, end = min(n, (blockIdx.x + 1) * per);
  double s = 0.0;
  for (uint64_t i = blockIdx.x * per + threadIdx.x; i < end; i += 256) {
    float x = a.g[base + i];
    if (a.update) {
      const float m = fmaf(a.momentum, a.m[base + i], x);
      a.m[base + i] = m;
      x = a.nesterov ? fmaf(a.momentum, m, x) : m;
    }
    u[base + i] = x;
    s += (double)x * x;
  }
  s = block_sum(s, sh);
  if (threadIdx.x == 0) part[blockIdx.y * kChunks + blockIdx.x] = s;
}

__global__ void __launch_bounds__(256) k_muon_scale(const __grid_constant__ MuonArgs a, float* x, const double* part) {
  const uint64_t n = (uint64_t)a.rows * a.cols;
  double s = 0.0;
  for (int i = 0; i < kChunks; ++i) s += part[blockIdx.y * kChunks + i];
  const double inv = 1.0 / (sqrt(s) + a.eps);
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += 256ull * gridDim.x)
    x[blockIdx.y * n + i] = (float)(x[blockIdx.y * n + i] * inv);
}

__global__ void __launch_bounds__(256) k_muon_apply(const __grid_constant__ MuonArgs a, const float* x) {
  const uint64_t n = (uint64_t)a.batch * a.rows * a.cols;
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += 256ull * gridDim.x) {
    if (a.update) a.w[i] = fmaf(-a.rate, x[i], a.keep * a.w[i]);
    else a.y[i] = x[i];
  }
}

struct Layout {
  uint64_t n, r;                    // elements of a matrix, and of its Gram matrix
  size_t x0, x1, gram, poly, part, total;
  explicit Layout(const MuonArgs& a) {
    n = (uint64_t)a.rows * a.cols;
    const uint64_t s = a.rows < a.cols ? a.rows : a.cols;
    r = s * s;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += (bytes + 255) & ~size_t(255); return o; };
    x0 = take(4 * n * a.batch);
    x1 = take(4 * n * a.batch);
    gram = take(4 * r * a.batch);
    poly = take(4 * r * a.batch);
    part = take(8 * kChunks * (size_t)a.batch);
    total = at;
  }
};

cudaError_t gemm(const Gemm& g, uint32_t batch, cudaStream_t st) {
  k_gemm<<<dim3((g.N + kTile - 1) / kTile, (g.M + kTile - 1) / kTile, batch), 256, 0, st>>>(g);
  return cudaGetLastError();
}

}  // namespace

size_t muon_ws_bytes(const MuonArgs& a) { return Layout(a).total; }

cudaError_t launch_muon(const MuonArgs& a, void* ws, cudaStream_t st) {
  const Layout L(a);
  if (!L.n || !a.batch) return cudaSuccess;
  char* w = static_cast<char*>(ws);
  float *x = reinterpret_cast<float*>(w + L.x0), *y = reinterpret_cast<float*>(w + L.x1);
  float *gram = reinterpret_cast<float*>(w + L.gram), *poly = reinterpret_cast<float*>(w + L.poly);
  double* part = reinterpret_cast<double*>(w + L.part);
  k_muon_momentum<<<dim3(kChunks, a.batch), 256, 0, st>>>(a, x, part);
  k_muon_scale<<<dim3(kChunks, a.batch), 256, 0, st>>>(a, x, part);
  cudaError_t e = cudaGetLastError();
  const int R = a.rows, C = a.cols;
  const bool wide = R <= C;
  const int S = wide ? R : C, T = wide ? C : R;
  for (uint32_t i = 0; i < a.steps && e == cudaSuccess; ++i) {
    const int64_t n = L.n, r = L.r;
    e = gemm(wide ? Gemm{x, x, nullptr, gram, C, 1, 1, C, S, n, n, r, S, S, T, 1.f, 0.f}
                  : Gemm{x, x, nullptr, gram, 1, C, C, 1, S, n, n, r, S, S, T, 1.f, 0.f}, a.batch, st);
    if (e == cudaSuccess)
      e = gemm(Gemm{gram, gram, gram, poly, S, 1, S, 1, S, r, r, r, S, S, S, (float)a.c, (float)a.b}, a.batch, st);
    if (e == cudaSuccess)
      e = gemm(wide ? Gemm{poly, x, x, y, S, 1, C, 1, C, r, n, n, R, C, S, 1.f, (float)a.a}
                    : Gemm{x, poly, x, y, C, 1, S, 1, C, n, r, n, R, C, S, 1.f, (float)a.a}, a.batch, st);
    float* t = x; x = y; y = t;
  }
  if (e != cudaSuccess) return e;
  k_muon_apply<<<grid_for((uint64_t)a.batch * L.n, 256), 256, 0, st>>>(a, x);
  return cudaGetLastError();
}

}  // namespace dct
