// Entry points of the transformer operators (dct_rotary, dct_attention_*, dct_orthogonalize,
// dct_muon): argument checks, scratch and launches.  The kernels are in k_rotary.cu,
// k_attention.cu and k_muon.cu.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>

#include "dct_common.cuh"
#include "kernels.h"
#include "runtime_internal.h"
#include "../../include/dct_cuda.h"

namespace dct {
namespace {

int refuse(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  note_error(code, buf);
  return code;
}

// The engine's device is current while this lives (a caller's thread may have another).
class OnDevice {
 public:
  OnDevice() {
    if (cudaGetDevice(&old_) != cudaSuccess) old_ = -1;
    if (old_ != dev_info().device) cudaSetDevice(dev_info().device);
    else old_ = -1;
  }
  ~OnDevice() {
    if (old_ >= 0) cudaSetDevice(old_);
  }

 private:
  int old_ = -1;
};

// engine up, and no capture of its stream under way
int ready(const char* what) {
  if (!rt_init()) return DCT_ERR_NO_DEVICE;
  cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(rt_stream(), &s) != cudaSuccess || s != cudaStreamCaptureStatusNone) {
    cudaGetLastError();
    return refuse(DCT_ERR_UNSUPPORTED, "%s: the library's stream is being captured into a graph", what);
  }
  return DCT_OK;
}

// A strided tensor argument [batch, position, head, feature].
struct Arg {
  const char* name;
  void* handle;
  uint64_t size[3], dim;
  const int64_t* stride;
  bool output;
  Buffer* buf = nullptr;
  uint64_t extent = 0;         // elements from the first to behind the last
  const char* lo() const { return reinterpret_cast<const char*>(buf->d); }
  const char* hi() const { return lo() + 4 * extent; }
};

int check(const char* what, Arg& a) {
  a.buf = rt_buf(a.handle);
  if (!a.buf) return refuse(DCT_ERR_HANDLE, "%s: %s is not a live buffer", what, a.name);
  a.extent = 0;
  if (!a.size[0] || !a.size[1] || !a.size[2] || !a.dim) return DCT_OK;
  unsigned __int128 last = a.dim;
  int order[3], n = 0;
  for (int i = 0; i < 3; ++i) {
    if (a.stride[i] < 0) return refuse(DCT_ERR_ARG, "%s: a stride of %s is negative", what, a.name);
    last += (unsigned __int128)(a.size[i] - 1) * (uint64_t)a.stride[i];
    if (a.size[i] > 1) order[n++] = i;
  }
  if (last > a.buf->count)
    return refuse(DCT_ERR_SIZE, "%s: %s holds %llu floats, its shape and strides reach further", what, a.name,
                  (unsigned long long)a.buf->count);
  a.extent = (uint64_t)last;
  if (a.output) {              // each dim steps over all that the smaller ones span
    std::sort(order, order + n, [&](int i, int j) { return a.stride[i] < a.stride[j]; });
    uint64_t span = a.dim;
    for (int i = 0; i < n; ++i) {
      const int d = order[i];
      if ((uint64_t)a.stride[d] < span)
        return refuse(DCT_ERR_ARG, "%s: elements of the output %s overlap", what, a.name);
      span += (a.size[d] - 1) * (uint64_t)a.stride[d];
    }
  }
  return DCT_OK;
}

bool overlap(const Arg& a, const Arg& b) { return a.extent && b.extent && a.lo() < b.hi() && b.lo() < a.hi(); }

// Whether no element of one output is one of the other.  Ranges that meet are told apart
// where the two lie side by side in every step of a common buffer, as the parts of a packed
// projection do: equal strides of batch and position, the heads of one behind the other's.
bool apart(const Arg& a, const Arg& b) {
  if (!overlap(a, b)) return true;
  const Arg &first = a.lo() <= b.lo() ? a : b, &second = a.lo() <= b.lo() ? b : a;
  auto width = [](const Arg& x) { return x.dim + (x.size[2] - 1) * (uint64_t)x.stride[2]; };
  const uint64_t ahead = (uint64_t)(second.lo() - first.lo()) / 4;
  if (ahead < width(first)) return false;
  uint64_t stride[2], size[2], span = ahead + width(second);
  for (int i = 0; i < 2; ++i) {
    if (a.size[i] > 1 && b.size[i] > 1 && a.stride[i] != b.stride[i]) return false;
    stride[i] = (uint64_t)(a.size[i] > 1 ? a : b).stride[i];
    size[i] = std::max(a.size[i], b.size[i]);
  }
  const int inner = size[0] > 1 && (size[1] <= 1 || stride[0] < stride[1]) ? 0 : 1;
  for (const int i : {inner, 1 - inner}) {
    if (size[i] <= 1) continue;
    if (stride[i] < span) return false;
    span += (size[i] - 1) * stride[i];
  }
  return true;
}

// an int32 tensor of n words, or null
int words(const char* what, const char* name, void* handle, uint64_t n, const int32_t** out) {
  *out = nullptr;
  if (!handle) return DCT_OK;
  Buffer* b = rt_buf(handle);
  if (!b) return refuse(DCT_ERR_HANDLE, "%s: %s is not a live buffer", what, name);
  if (b->count < n)
    return refuse(DCT_ERR_SIZE, "%s: %s holds %llu words, %llu are read", what, name, (unsigned long long)b->count,
                  (unsigned long long)n);
  *out = reinterpret_cast<const int32_t*>(b->d);
  return DCT_OK;
}

void copy3(int64_t* to, const int64_t* from) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

constexpr uint64_t kMost = 1ull << 30;       // tokens or features of one call
constexpr uint64_t kMostRows = 1ull << 28;   // positions times heads: sums of a few of them are 32-bit

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
int attention(const char* what, const DctAttention* p, void* q, void* k, void* v, void* q_lens, void* kv_lens,
              void* out, void* lse, bool backward, void* dout, void* dq, void* dk, void* dv) {
  if (const int rc = ready(what)) return rc;
  if (!p) return refuse(DCT_ERR_ARG, "%s: no parameters", what);
  if (p->head_dim < 1 || p->head_dim > 128)
    return refuse(DCT_ERR_ARG, "%s: head_dim is %u (1 to 128)", what, p->head_dim);
  if (!p->q_heads || !p->kv_heads || p->q_heads % p->kv_heads)
    return refuse(DCT_ERR_ARG, "%s: %u query heads over %u key heads", what, p->q_heads, p->kv_heads);
  // heads and batch entries count where there are no positions too: the kernels' are 32-bit
  if ((unsigned __int128)std::max(1u, p->q_len) * p->q_heads * std::max(1u, p->batch) >= kMostRows ||
      (unsigned __int128)std::max(1u, p->kv_len) * p->kv_heads * std::max(1u, p->batch) >= kMostRows)
    return refuse(DCT_ERR_ARG, "%s: too many rows in one call", what);
  if (!isfinite(p->scale)) return refuse(DCT_ERR_ARG, "%s: scale is not finite", what);
  const uint64_t B = p->batch, D = p->head_dim;
  Arg args[] = {{"q", q, {B, p->q_len, p->q_heads}, D, p->q_stride, false},
                {"k", k, {B, p->kv_len, p->kv_heads}, D, p->k_stride, false},
                {"v", v, {B, p->kv_len, p->kv_heads}, D, p->v_stride, false},
                {"out", out, {B, p->q_len, p->q_heads}, D, p->o_stride, !backward},
                {"dout", dout, {B, p->q_len, p->q_heads}, D, p->o_stride, false},
                {"dq", dq, {B, p->q_len, p->q_heads}, D, p->dq_stride, true},
                {"dk", dk, {B, p->kv_len, p->kv_heads}, D, p->dk_stride, true},
                {"dv", dv, {B, p->kv_len, p->kv_heads}, D, p->dv_stride, true}};
  const int n = backward ? 8 : 4;
  for (int i = 0; i < n; ++i)
    if (const int rc = check(what, args[i])) return rc;
  const int64_t lse_stride[3] = {(int64_t)p->q_heads * p->q_len, (int64_t)p->q_len, 1};
  Arg l{"lse", lse, {B, p->q_heads, p->q_len}, 1, lse_stride, !backward};
  if (lse || backward)
    if (const int rc = check(what, l)) return rc;
  for (int i = 0; i < n; ++i) {
    for (int j = 0; j < n; ++j)
      if (args[i].output && !args[j].output && overlap(args[i], args[j]))
        return refuse(DCT_ERR_ARG, "%s: %s overlaps %s", what, args[i].name, args[j].name);
    for (int j = i + 1; j < n; ++j)
      if (args[i].output && args[j].output && !apart(args[i], args[j]))
        return refuse(DCT_ERR_ARG, "%s: %s and %s share elements", what, args[i].name, args[j].name);
    if ((args[i].output || l.output) && overlap(args[i], l))
      return refuse(DCT_ERR_ARG, "%s: %s overlaps lse", what, args[i].name);
  }
  AttnArgs a{};
  if (const int rc = words(what, "q_lens", q_lens, B, &a.q_lens)) return rc;
  if (const int rc = words(what, "kv_lens", kv_lens, B, &a.kv_lens)) return rc;
  for (const int32_t* w : {a.q_lens, a.kv_lens}) {
    auto meets = [&](const Arg& x) {
      return w && x.output && x.extent && reinterpret_cast<const char*>(w) < x.hi() &&
             x.lo() < reinterpret_cast<const char*>(w + B);
    };
    for (int i = 0; i < n; ++i)
      if (meets(args[i])) return refuse(DCT_ERR_ARG, "%s: %s overlaps the lengths", what, args[i].name);
    if (meets(l)) return refuse(DCT_ERR_ARG, "%s: lse overlaps the lengths", what);
  }
  a.q = args[0].buf->d; a.k = args[1].buf->d; a.v = args[2].buf->d;
  a.out = args[3].buf->d;
  a.lse = l.buf ? l.buf->d : nullptr;
  copy3(a.qs, p->q_stride); copy3(a.ks, p->k_stride); copy3(a.vs, p->v_stride); copy3(a.os, p->o_stride);
  a.batch = p->batch; a.q_heads = p->q_heads; a.kv_heads = p->kv_heads; a.group = p->q_heads / p->kv_heads;
  a.q_len = p->q_len; a.kv_len = p->kv_len; a.dim = p->head_dim;
  a.causal = p->causal != 0;
  a.window = p->window >= p->q_len + p->kv_len ? 0 : (int)p->window;      // as wide as that hides nothing
  a.scale = p->scale != 0.f ? p->scale : (float)(1.0 / sqrt((double)p->head_dim));
  OnDevice guard;
  cudaStream_t st = rt_stream();
  if (backward) {
    a.dout = args[4].buf->d; a.dq = args[5].buf->d; a.dk = args[6].buf->d; a.dv = args[7].buf->d;
    copy3(a.dqs, p->dq_stride); copy3(a.dks, p->dk_stride); copy3(a.dvs, p->dv_stride);
  }
  cudaError_t e;
  if (attn_tensor_fits(a, backward)) {
    if (!rt_ensure_ws(attn_tensor_ws_bytes(a, backward))) return DCT_ERR_CUDA;
    e = backward ? launch_attn_tensor_backward(a, rt_ws(), st) : launch_attn_tensor_forward(a, rt_ws(), st);
  } else if (!backward) {
    if (!rt_ensure_ws(attn_rows_ws_bytes(a))) return DCT_ERR_CUDA;
    e = launch_attn_rows_forward(a, rt_ws(), st);
  } else {
    if (!rt_ensure_ws(sizeof(float) * B * p->kv_heads * padded_rows(a))) return DCT_ERR_CUDA;
    a.delta = static_cast<float*>(rt_ws());
    e = launch_attn_delta(a, st);
    if (e == cudaSuccess) e = launch_attn_rows_backward(a, st);
  }
  return rt_cuda_ok(e, what) ? DCT_OK : DCT_ERR_CUDA;
}

// ---------------------------------------------------------------------------
// orthogonalisation
// ---------------------------------------------------------------------------
// Fills the shape, the polynomial and the largest singular value that its steps can give.
int muon_args(const char* what, const DctMuon* p, MuonArgs& a) {
  if (!p) return refuse(DCT_ERR_ARG, "%s: no parameters", what);
  if (p->batch > 65535 || (uint64_t)p->rows * p->cols >= kMost || p->rows > (1u << 23) || p->cols > (1u << 23))
    return refuse(DCT_ERR_ARG, "%s: %u matrices of %u x %u are too many or too large", what, p->batch, p->rows,
                  p->cols);
  if (p->steps > 16) return refuse(DCT_ERR_ARG, "%s: %u steps (0 to 16)", what, p->steps);
  if (!(p->eps >= 0.f) || !isfinite(p->eps)) return refuse(DCT_ERR_ARG, "%s: eps is negative or not finite", what);
  a.a = p->a; a.b = p->b; a.c = p->c;
  if (a.a == 0 && a.b == 0 && a.c == 0) { a.a = 3.4445; a.b = -4.7750; a.c = 2.0315; }
  if (!isfinite(a.a) || !isfinite(a.b) || !isfinite(a.c))
    return refuse(DCT_ERR_ARG, "%s: a coefficient is not finite", what);
  // singular values start in [0, 1]; follow the largest that a step can give, on a grid
  // (and the slack that the grid's spacing and the arithmetic leave)
  double top = 1.0;
  a.bound = 1.0;
  for (uint32_t i = 0; i < p->steps; ++i) {
    double next = 0.0;
    for (int j = 0; j <= 256; ++j) {
      const double s = top * j / 256.0, t = s * s;
      next = std::max(next, fabs(s * (a.a + t * (a.b + t * a.c))));
    }
    top = 1.01 * next;
    a.bound = std::max(a.bound, top);
    if (!(a.bound < 64.0))
      return refuse(DCT_ERR_ARG, "%s: the steps' polynomial grows past 64", what);
  }
  a.batch = p->batch; a.rows = p->rows; a.cols = p->cols; a.steps = p->steps;
  a.eps = p->eps;
  return DCT_OK;
}

int muon_run(const char* what, const MuonArgs& a) {
  OnDevice guard;
  if (!rt_ensure_ws(muon_ws_bytes(a))) return DCT_ERR_CUDA;
  return rt_cuda_ok(launch_muon(a, rt_ws(), rt_stream()), what) ? DCT_OK : DCT_ERR_CUDA;
}

}  // namespace
}  // namespace dct

using namespace dct;
#define LOCK std::lock_guard<std::recursive_mutex> _lk(rt_mutex())

extern "C" {

DCT_API int dct_rotary(const DctRotary* p, void* x, void* positions, void* y) {
  LOCK;
  const char* what = "dct_rotary";
  if (const int rc = ready(what)) return rc;
  if (!p) return refuse(DCT_ERR_ARG, "%s: no parameters", what);
  if (p->rotated % 2 || p->rotated > p->head_dim || p->rotated > 256)
    return refuse(DCT_ERR_ARG, "%s: %u rotated features of %u (even, at most 256)", what, p->rotated, p->head_dim);
  if ((unsigned __int128)p->batch * p->length >= kMost || (unsigned __int128)p->heads * p->head_dim >= kMost)
    return refuse(DCT_ERR_ARG, "%s: too many tokens or features in one call", what);
  if (!(p->base > 0) || !(p->factor > 0) || !isfinite(p->base) || !isfinite(p->factor) || !isfinite(p->magnitude) ||
      !(p->original >= 0) || !isfinite(p->original))
    return refuse(DCT_ERR_ARG, "%s: base and factor are positive, original is not negative, all are finite", what);
  if (p->factor != 1.0 && p->original > 0 && !(p->high > p->low && isfinite(p->high) && isfinite(p->low)))
    return refuse(DCT_ERR_ARG, "%s: low must be below high", what);
  Arg ax{"x", x, {p->batch, p->length, p->heads}, p->head_dim, p->x_stride, false};
  Arg ay{"y", y, {p->batch, p->length, p->heads}, p->head_dim, p->y_stride, true};
  if (const int rc = check(what, ax)) return rc;
  if (const int rc = check(what, ay)) return rc;
  bool same = ax.buf->d == ay.buf->d;
  for (int i = 0; i < 3; ++i) same = same && (ax.size[i] <= 1 || p->x_stride[i] == p->y_stride[i]);
  if (!same && overlap(ax, ay)) return refuse(DCT_ERR_ARG, "%s: y overlaps x", what);
  RotaryArgs a{};
  const uint64_t tokens = (uint64_t)p->batch * p->length;
  if (const int rc = words(what, "positions", positions, tokens, &a.positions)) return rc;
  if (a.positions && ay.extent && reinterpret_cast<const char*>(a.positions) < ay.hi() &&
      ay.lo() < reinterpret_cast<const char*>(a.positions + tokens))
    return refuse(DCT_ERR_ARG, "%s: y overlaps the positions", what);
  if (!ax.extent) return DCT_OK;
  a.x = ax.buf->d; a.y = ay.buf->d;
  a.batch = p->batch; a.length = p->length; a.heads = p->heads; a.head_dim = p->head_dim; a.rotated = p->rotated;
  copy3(a.xs, p->x_stride); copy3(a.ys, p->y_stride);
  a.start = p->start; a.magnitude = (float)p->magnitude;
  a.interleaved = p->interleaved != 0; a.inverse = p->inverse != 0; a.in_place = same;
  RotaryTurns f;
  // powers by products in long double: 2^-64 a factor, at most 128 factors
  const double two_pi = 6.283185307179586476925286766559;
  const long double ratio = p->rotated ? powl((long double)p->base, -2.0L / p->rotated) : 1.0L;
  long double w = 1.0L;
  for (uint32_t j = 0; j < p->rotated / 2; ++j, w *= ratio) {
    double t = (double)(w / two_pi);             // turns a position
    if (p->factor != 1.0) {
      double keep = 0.0;
      if (p->original > 0) keep = std::min(1.0, std::max(0.0, (p->original * t - p->low) / (p->high - p->low)));
      t *= keep + (1.0 - keep) / p->factor;
    }
    f.turns[j] = t;
  }
  OnDevice guard;
  return rt_cuda_ok(launch_rotary(a, f, rt_stream()), what) ? DCT_OK : DCT_ERR_CUDA;
}

DCT_API int dct_attention_forward(const DctAttention* p, void* q, void* k, void* v, void* q_lens, void* kv_lens,
                                  void* out, void* lse) {
  LOCK;
  return attention("dct_attention_forward", p, q, k, v, q_lens, kv_lens, out, lse, false, nullptr, nullptr, nullptr,
                   nullptr);
}

DCT_API int dct_attention_backward(const DctAttention* p, void* q, void* k, void* v, void* q_lens, void* kv_lens,
                                   void* out, void* lse, void* dout, void* dq, void* dk, void* dv) {
  LOCK;
  return attention("dct_attention_backward", p, q, k, v, q_lens, kv_lens, out, lse, true, dout, dq, dk, dv);
}

DCT_API int dct_orthogonalize(const DctMuon* p, void* x, void* y) {
  LOCK;
  const char* what = "dct_orthogonalize";
  if (const int rc = ready(what)) return rc;
  MuonArgs a{};
  if (const int rc = muon_args(what, p, a)) return rc;
  const int64_t none[3] = {(int64_t)p->rows * p->cols, (int64_t)p->cols, (int64_t)p->cols};
  Arg ax{"x", x, {p->batch, p->rows, 1}, p->cols, none, false};
  Arg ay{"y", y, {p->batch, p->rows, 1}, p->cols, none, true};
  if (const int rc = check(what, ax)) return rc;
  if (const int rc = check(what, ay)) return rc;
  if (!ax.extent) return DCT_OK;
  if (ax.buf->d != ay.buf->d && overlap(ax, ay)) return refuse(DCT_ERR_ARG, "%s: y overlaps x", what);
  a.g = ax.buf->d;
  a.y = ay.buf->d;
  return muon_run(what, a);
}

DCT_API int dct_muon(const DctMuon* p, void* w, void* m, void* g) {
  LOCK;
  const char* what = "dct_muon";
  if (const int rc = ready(what)) return rc;
  MuonArgs a{};
  if (const int rc = muon_args(what, p, a)) return rc;
  const int64_t none[3] = {(int64_t)p->rows * p->cols, (int64_t)p->cols, (int64_t)p->cols};
  Arg aw{"w", w, {p->batch, p->rows, 1}, p->cols, none, true};
  Arg am{"m", m, {p->batch, p->rows, 1}, p->cols, none, true};
  Arg ag{"g", g, {p->batch, p->rows, 1}, p->cols, none, false};
  if (const int rc = check(what, aw)) return rc;
  if (const int rc = check(what, am)) return rc;
  if (const int rc = check(what, ag)) return rc;
  if (!aw.extent) return DCT_OK;
  if (overlap(aw, am) || overlap(aw, ag) || overlap(am, ag))
    return refuse(DCT_ERR_ARG, "%s: w, m and g overlap", what);
  a.w = aw.buf->d; a.m = am.buf->d; a.g = ag.buf->d;
  a.momentum = p->momentum;
  a.keep = (float)(1.0 - (double)p->lr * p->weight_decay);
  a.rate = (float)(p->lr * (p->scale != 0.f ? (double)p->scale : sqrt(std::max(1.0, (double)p->rows / p->cols))));
  a.nesterov = p->nesterov != 0;
  a.update = true;
  return muon_run(what, a);
}

}  // extern "C"
