// The norm over many gradient tensors together, and their scaling by it:
//   norm = (sum |g|^p)^(1/p) for p = 1, 2, or max |g|;   coef = min(1, max_norm / (norm + 1e-6));   g = g coef
//
// Bound by HBM: all gradients are read for the norm and, where coef < 1, read again and written.  The list of tensors travels in the kernel's arguments (up to
// GROUP tensors a launch: no table to upload, so a captured launch holds its own), a workgroup takes one piece of one tensor.
// Sums run in 64 bits (squares of fp32 and bf16 values leave the range of fp32, and a billion of them its precision), in a fixed order: the
// pieces' sums go to the workspace, one workgroup adds them.
#include "rows.h"
#include <stdlib.h>

namespace cagc {
namespace {

constexpr int GROUP = 120;
struct Group {
  void* p[GROUP];
  int64_t n[GROUP];
  uint32_t first[GROUP + 1];      // tensor i has the launch's workgroups first[i] .. first[i + 1] - 1
  uint8_t dtype[GROUP];
  int count;
  int piece;                      // elements of a workgroup
  double* part;                   // of the launch's first workgroup
  const float* coef;
};
static_assert(sizeof(Group) <= 4000, "kernel arguments");

// magnitudes as bit patterns: a NaN is above infinity and so is kept
__device__ __forceinline__ double larger(double a, double b) {
  const uint64_t x = __builtin_bit_cast(uint64_t, a), y = __builtin_bit_cast(uint64_t, b);
  return x > y ? a : b;
}
template <int P> __device__ __forceinline__ double take(double s, float g) {
  const double d = (double)fabsf(g);
  if (P == 2) return s + d * d;
  if (P == 1) return s + d;
  return larger(s, d);
}
template <int P> __device__ __forceinline__ double both(double a, double b) { return P == 0 ? larger(a, b) : a + b; }
template <int P> __device__ __forceinline__ double wave_all(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = both<P>(v, __shfl_xor(v, off, 64));
  return v;
}

__device__ __forceinline__ int tensor_of(const Group& a, uint32_t b) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.first[mid] <= b) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <class T, int P> __device__ __forceinline__ double piece_norm(const T* g, int64_t n) {
  constexpr int V = 16 / (int)sizeof(T);
  double s = 0., s2 = 0.;
  const int64_t whole = n / V;
  int64_t i = threadIdx.x;
  for (; i + 768 < whole; i += 1024) {       // four loads in flight
    T e[4][V];
#pragma unroll
    for (int k = 0; k < 4; ++k) { const Any16 a = reinterpret_cast<const Any16*>(g)[i + 256 * k]; __builtin_memcpy(e[k], &a, 16); }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) { if (k & 1) s2 = take<P>(s2, (float)e[k][j]); else s = take<P>(s, (float)e[k][j]); }
  }
  for (; i < whole; i += 256) {
    T e[V];
    const Any16 a = reinterpret_cast<const Any16*>(g)[i];
    __builtin_memcpy(e, &a, 16);
#pragma unroll
    for (int j = 0; j < V; ++j) s = take<P>(s, (float)e[j]);
  }
  if (whole * V + threadIdx.x < n) s = take<P>(s, (float)g[whole * V + threadIdx.x]);
  return both<P>(s, s2);
}

template <int P> __global__ __launch_bounds__(256) void k_grad_norm(Group a) {
  __shared__ double sh[4];
  const int i = tensor_of(a, blockIdx.x);
  const int64_t at = (int64_t)(blockIdx.x - a.first[i]) * a.piece, n = min((int64_t)a.piece, a.n[i] - at);
  double s;
  if (a.dtype[i] == CAGC_F32) s = piece_norm<float, P>(static_cast<const float*>(a.p[i]) + at, n);
  else if (a.dtype[i] == CAGC_F16) s = piece_norm<_Float16, P>(static_cast<const _Float16*>(a.p[i]) + at, n);
  else s = piece_norm<__bf16, P>(static_cast<const __bf16*>(a.p[i]) + at, n);
  s = wave_all<P>(s);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.part[blockIdx.x] = both<P>(both<P>(sh[0], sh[1]), both<P>(sh[2], sh[3]));
}

template <int P> __global__ __launch_bounds__(1024) void k_grad_norm_join(float* __restrict__ norm, float* __restrict__ coef, const double* __restrict__ part, int64_t parts, double max_norm) {
  __shared__ double sh[16];
  double s = 0.;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < parts; i += 1024) s = both<P>(s, part[i]);
  s = wave_all<P>(s);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 16; ++i) s = both<P>(s, sh[i]);
  if (P == 2) s = sqrt(s);
  *norm = (float)s;
  const double c = max_norm / (s + 1e-6);
  if (coef) *coef = c > 1. ? 1.f : (float)c;          // a NaN stays one
}

template <class T> __device__ __forceinline__ void piece_scale(T* g, int64_t n, float c) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t whole = n / V;
  auto one = [&](Any16 a) {
    T e[V];
    __builtin_memcpy(e, &a, 16);
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = (T)((float)e[j] * c);
    __builtin_memcpy(&a, e, 16);
    return a;
  };
  int64_t i = threadIdx.x;
  Any16* q = reinterpret_cast<Any16*>(g);
  for (; i + 768 < whole; i += 1024) {
    Any16 a[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = q[i + 256 * k];
#pragma unroll
    for (int k = 0; k < 4; ++k) q[i + 256 * k] = one(a[k]);
  }
  for (; i < whole; i += 256) q[i] = one(q[i]);
  if (whole * V + threadIdx.x < n) g[whole * V + threadIdx.x] = (T)((float)g[whole * V + threadIdx.x] * c);
}
__global__ __launch_bounds__(256) void k_grad_scale(Group a) {
  const float c = *a.coef;
  if (c == 1.f) return;                        // nothing to clip: every value times 1
  const int i = tensor_of(a, blockIdx.x);
  const int64_t at = (int64_t)(blockIdx.x - a.first[i]) * a.piece, n = min((int64_t)a.piece, a.n[i] - at);
  if (a.dtype[i] == CAGC_F32) piece_scale(static_cast<float*>(a.p[i]) + at, n, c);
  else if (a.dtype[i] == CAGC_F16) piece_scale(static_cast<_Float16*>(a.p[i]) + at, n, c);
  else piece_scale(static_cast<__bf16*>(a.p[i]) + at, n, c);
}

// elements of a workgroup: 16 KB of fp32 while that makes at most 8192 workgroups, then as many as keep it at that
int piece_of(const int64_t* n, int count) {
  int64_t total = 0;
  for (int i = 0; i < count; ++i) total += n[i];
  int64_t piece = 4096;
  while (total / piece > 8192 && piece < (1 << 30)) piece *= 2;
  return (int)piece;
}
int64_t pieces(const int64_t* n, int count, int piece) {
  int64_t b = 0;
  for (int i = 0; i < count; ++i) b += (n[i] + piece - 1) / piece;
  return b;
}

// calls `launch` for each group of tensors with its workgroups
template <class F> int for_groups(void* const* p, const int64_t* n, const int* dtype, int count, int piece, double* part, const float* coef, F launch, const char* what) {
  Group a;
  a.piece = piece; a.coef = coef; a.part = part;
  int i = 0;
  while (i < count) {
    a.count = 0;
    uint32_t b = 0;
    for (; i < count && a.count < GROUP; ++i) {
      if (n[i] == 0) continue;
      a.p[a.count] = p[i]; a.n[a.count] = n[i]; a.dtype[a.count] = (uint8_t)dtype[i]; a.first[a.count] = b;
      b += (uint32_t)((n[i] + piece - 1) / piece);
      ++a.count;
    }
    if (a.count == 0) break;
    a.first[a.count] = b;
    launch(a, b);
    const int rc = check_launch(what);
    if (rc != CAGC_OK) return rc;
    if (a.part) a.part += b;
  }
  return CAGC_OK;
}

int esize(int dtype) { return dtype == CAGC_F32 ? 4 : 2; }
struct Span { uintptr_t from, to; };
int by_start(const void* x, const void* y) {
  const uintptr_t a = static_cast<const Span*>(x)->from, b = static_cast<const Span*>(y)->from;
  return a < b ? -1 : a > b;
}
// two tensors of the list that share memory would be counted twice and scaled by two workgroups at once
bool apart(void* const* p, const int64_t* n, const int* dtype, int count) {
  if (count < 2) return true;
  Span few[256];
  Span* s = count <= 256 ? few : static_cast<Span*>(malloc(sizeof(Span) * (size_t)count));
  if (!s) return false;
  for (int i = 0; i < count; ++i) s[i] = Span{(uintptr_t)p[i], (uintptr_t)p[i] + (uintptr_t)(n[i] * esize(dtype[i]))};
  qsort(s, (size_t)count, sizeof(Span), by_start);
  bool ok = true;
  uintptr_t end = 0;
  for (int i = 0; i < count; ++i) {
    if (s[i].from == s[i].to) continue;
    if (s[i].from < end) ok = false;
    end = s[i].to;
  }
  if (s != few) free(s);
  return ok;
}

}  // namespace
}  // namespace cagc

using namespace cagc;

extern "C" int64_t cagc_grad_norm_workspace(const int64_t* n, int count) {
  if (!n || count <= 0) return 64;
  const int64_t b = pieces(n, count, piece_of(n, count));
  return 64 + 8 * b;
}

extern "C" int cagc_clip_grad_norm(float* norm, void* ws, void* const* p, const int64_t* n, const int* dtype, int count, int norm_type, double max_norm, int scale,
                                   cagc_stream_t stream) {
  const char* what = "cagc_clip_grad_norm";
  CAGC_REQUIRE(norm && ws && count >= 0 && (count == 0 || (p && n && dtype)), "%s: null pointer", what);
  CAGC_REQUIRE(norm_type == 0 || norm_type == 1 || norm_type == 2, "%s: norm type %d", what, norm_type);
  for (int i = 0; i < count; ++i) {
    CAGC_REQUIRE(dtype[i] == CAGC_F32 || dtype[i] == CAGC_F16 || dtype[i] == CAGC_BF16, "%s: element type %d of tensor %d", what, dtype[i], i);
    CAGC_REQUIRE(n[i] >= 0 && n[i] < (1ll << 40) && (n[i] == 0 || p[i]), "%s: tensor %d", what, i);
    CAGC_REQUIRE((uintptr_t)p[i] % esize(dtype[i]) == 0, "%s: address of tensor %d", what, i);
  }
  CAGC_REQUIRE(apart(p, n, dtype, count), "%s: two tensors of the list share memory", what);
  hipStream_t st = as_stream(stream);
  float* coef = static_cast<float*>(ws);
  double* part = reinterpret_cast<double*>(static_cast<char*>(ws) + 64);
  const int piece = count ? piece_of(n, count) : 1;
  const int64_t parts = count ? pieces(n, count, piece) : 0;
  int rc = for_groups(p, n, dtype, count, piece, part, nullptr, [&](const Group& a, uint32_t b) {
    if (norm_type == 2) hipLaunchKernelGGL((k_grad_norm<2>), dim3(b), dim3(256), 0, st, a);
    else if (norm_type == 1) hipLaunchKernelGGL((k_grad_norm<1>), dim3(b), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_grad_norm<0>), dim3(b), dim3(256), 0, st, a);
  }, what);
  if (rc != CAGC_OK) return rc;
  if (norm_type == 2) hipLaunchKernelGGL((k_grad_norm_join<2>), dim3(1), dim3(1024), 0, st, norm, scale ? coef : nullptr, part, parts, max_norm);
  else if (norm_type == 1) hipLaunchKernelGGL((k_grad_norm_join<1>), dim3(1), dim3(1024), 0, st, norm, scale ? coef : nullptr, part, parts, max_norm);
  else hipLaunchKernelGGL((k_grad_norm_join<0>), dim3(1), dim3(1024), 0, st, norm, scale ? coef : nullptr, part, parts, max_norm);
  if ((rc = check_launch(what)) != CAGC_OK || !scale) return rc;
  return for_groups(p, n, dtype, count, piece, nullptr, coef, [&](const Group& a, uint32_t b) {
    hipLaunchKernelGGL(k_grad_scale, dim3(b), dim3(256), 0, st, a);
  }, what);
}
