// Root-mean-square norm of rows, with the residual's addition before it and, for 8-bit products, e4m3 output with a scale per row.
//   h = x + residual (rounded to the type: it is an output),  rstd = (mean(h^2) + eps)^-1/2,  y = h rstd w
//   e4m3: scale = max |y| / 448, q = y / scale
//   backward, with t = dy w and n = h rstd:  dx = dresidual = rstd (t - n mean(t n)) + dh,   dw = sum over rows of dy n
//
// Bound by HBM: a row is read once and kept in registers between its sums and its output (TPR threads a row, NV chunks of 16 bytes each),
// so a forward moves x, residual, h and y once.  Sums are fp32.  Rows may start at any address.
#include "rows.h"

namespace cagc {
namespace {

template <class T> struct Row { static constexpr int V = 16 / (int)sizeof(T); };

// V e4m3 bytes of f / scale, `inv` = 1 / scale.  The quotient is the correctly rounded one: times the rounded reciprocal alone, values beside a tie of e4m3 would go to the other side.  Two residuals
// make it so (Markstein 1990: the first leaves it within a step, the second rounds it as the division does); a scale below 2^-90, whose residuals underflow, an infinite one and a NaN are divided by.
// 8191 x 5120 bf16: 57.8 us times the reciprocal, 62.1 divided, 58.8 this way.
template <int V> __device__ __forceinline__ void store_q(uint8_t* p, const float (&f)[V], float scale, float inv, int n) {
  float q[V];
  if (scale > 0x1p-90f && scale < __builtin_inff()) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float a = f[i] * inv, b = fmaf(fmaf(-a, scale, f[i]), inv, a);
      q[i] = fmaf(fmaf(-b, scale, f[i]), inv, b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = f[i] / scale;
  }
  uint32_t d[V / 4];
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
    d[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], v, true);
  }
  struct __attribute__((packed, aligned(1))) Any { uint32_t v[V / 4]; };
  if (n >= V) {
    Any a;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) a.v[i] = d[i];
    *reinterpret_cast<Any*>(p) = a;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) if (i < n) p[i] = (uint8_t)(d[i / 4] >> (8 * (i & 3)));
  }
}

// A thread's chunk of V elements.  The last chunk of a row whose length is no multiple of V begins V before the row's end: its first `skip` elements are the chunk before's too, which counts them;
// both store the same values there.  A thread behind the row's end stands at the last chunk and counts nothing (skip = V).  `n`: elements there (V, but in a row shorter than that).
template <int V> struct Chunk {
  int at, skip, n;
  __device__ __forceinline__ Chunk(int chunk, int dim) {
    const int start = chunk * V;
    at = max(0, min(start, dim - V));
    skip = min(V, start - at);
    n = min(V, dim);
  }
  __device__ __forceinline__ bool used() const { return skip < V; }
};

// sum / largest over the TPR threads of a row; every thread gets it.  `sh`: TPR / 64 words of this row's own, one use a call.
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* sh) {
  v = wave_sum(v);
  if (TPR == 64) return v;
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < TPR / 64; ++i) s += sh[i];
  return s;
}
// magnitudes compared as bit patterns: a NaN is above infinity and so is kept
template <int TPR> __device__ __forceinline__ float row_top(uint32_t v, uint32_t* sh) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, 64));
  if (TPR > 64) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v = max(v, sh[i]);
  }
  return __builtin_bit_cast(float, v);
}

struct Norm {
  void* y;               // [rows, dim]: the element type, or e4m3
  float* scale;          // [rows] (e4m3)
  void* h;               // [rows, dim] [nullable]
  float* rstd;           // [rows] [nullable]
  const void* x;
  const void* res;       // [nullable]
  const void* w;         // [dim] [nullable]
  int64_t rows, xs, rs;  // rows of x and residual are xs, rs elements apart
  int dim;
  float eps;
};

// threads of a workgroup: several rows of a wave each, or one row
constexpr int threads_of(int tpr) { return tpr == 64 ? 256 : tpr; }

// OUT: 0 = the element type, 1 = e4m3, 2 = e4m3 of the rows themselves, without the norm
template <class T, class W, int TPR, int NV, int OUT>
__global__ __launch_bounds__(threads_of(TPR)) void k_rms_norm(Norm a) {
  constexpr int V = Row<T>::V, RPB = threads_of(TPR) / TPR;
  __shared__ float sh[2][TPR / 64];
  const int t = threadIdx.x % TPR;
  const int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (r >= a.rows) return;                     // (a whole wave, and with more than 64 threads a row the whole workgroup)
  const T* x = static_cast<const T*>(a.x) + r * a.xs;
  const T* res = a.res ? static_cast<const T*>(a.res) + r * a.rs : nullptr;
  T* h = a.h ? static_cast<T*>(a.h) + r * a.dim : nullptr;
  float v[NV][V], ss = 0.f;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const Chunk<V> k(t + c * TPR, a.dim);
    load_v<V>(v[c], x + k.at, k.n);
  }
  if (res) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const Chunk<V> k(t + c * TPR, a.dim);
      float f[V];
      load_v<V>(f, res + k.at, k.n);
#pragma unroll
      for (int i = 0; i < V; ++i) v[c][i] = (float)(T)(v[c][i] + f[i]);
    }
  }
  if (h) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const Chunk<V> k(t + c * TPR, a.dim);
      if (k.used()) store_v<V>(h + k.at, v[c], k.n);
    }
  }
  if (OUT != 2) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const Chunk<V> k(t + c * TPR, a.dim);
#pragma unroll
      for (int i = 0; i < V; ++i) ss += i >= k.skip ? v[c][i] * v[c][i] : 0.f;
    }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(ss, sh[0]) / (float)a.dim + a.eps);
    if (a.rstd && t == 0) a.rstd[r] = rstd;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      if (a.w) {
        const Chunk<V> k(t + c * TPR, a.dim);
        float f[V];
        load_v<V>(f, static_cast<const W*>(a.w) + k.at, k.n);
#pragma unroll
        for (int i = 0; i < V; ++i) v[c][i] = v[c][i] * rstd * f[i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[c][i] *= rstd;
      }
    }
  }
  if (OUT == 0) {
    T* y = static_cast<T*>(a.y) + r * a.dim;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const Chunk<V> k(t + c * TPR, a.dim);
      if (k.used()) store_v<V>(y + k.at, v[c], k.n);
    }
    return;
  }
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[c][i]) & 0x7fffffffu);
  const float most = row_top<TPR>(top, reinterpret_cast<uint32_t*>(sh[1]));
  // a row of zeros (or of less than the smallest normal scale holds) has something to be divided by; a NaN stays one (the comparison is false)
  float scale = most / 448.f;
  if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;
  if (t == 0) a.scale[r] = scale;
  const float inv = 1.f / scale;
  uint8_t* q = static_cast<uint8_t*>(a.y) + r * a.dim;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const Chunk<V> k(t + c * TPR, a.dim);
    if (k.used()) store_q<V>(q + k.at, v[c], scale, inv, k.n);
  }
}

struct NormBwd {
  void* dx;              // [rows, dim]
  float* part;           // [gridDim.x][dim]: each workgroup's share of dw [nullable]
  void* dw;              // [dim], of a workgroup that is the only one [nullable]
  const void* dy;
  const void* dh;        // [nullable]
  const void* h;
  const void* w;         // [nullable]
  const float* rstd;
  int64_t rows, dys, dhs, hs;
  int dim;
};

// A workgroup takes rows blockIdx.x * RPB, + gridDim.x * RPB, ...: a thread keeps its columns of w and of dw in registers throughout.  16-bit rows of more than 16384 elements, four chunks of 1024 threads,
// want more than the 128 registers of a lane there: some 95 of them spill.  Reading w anew for each row (it stays in L2) still spills 75 and is slower: 2048 x 32768 bf16 467 us, so 423.
template <class T, class W, int TPR, int NV>
__global__ __launch_bounds__(threads_of(TPR)) void k_rms_norm_bwd(NormBwd a) {
  constexpr int V = Row<T>::V, RPB = threads_of(TPR) / TPR;
  __shared__ float sh[2][TPR / 64];
  __shared__ float join[RPB > 1 ? NV * V * TPR : 1];
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  float w[NV][V], dw[NV][V];
  auto weight = [&](int c, float (&f)[V]) {
    const Chunk<V> k(t + c * TPR, a.dim);
    if (a.w) { load_v<V>(f, static_cast<const W*>(a.w) + k.at, k.n); return; }
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = 1.f;
  };
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    weight(c, w[c]);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[c][i] = 0.f;
  }
  int turn = 0;
  for (int64_t r = (int64_t)blockIdx.x * RPB + slot; r < a.rows; r += (int64_t)gridDim.x * RPB, turn ^= 1) {
    const T* dy = static_cast<const T*>(a.dy) + r * a.dys;
    const T* h = static_cast<const T*>(a.h) + r * a.hs;
    const float rstd = a.rstd[r];
    float d[NV][V], n[NV][V], s = 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const Chunk<V> k(t + c * TPR, a.dim);
      load_v<V>(d[c], dy + k.at, k.n);
      load_v<V>(n[c], h + k.at, k.n);
    }
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const Chunk<V> k(t + c * TPR, a.dim);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        n[c][i] *= rstd;
        dw[c][i] += d[c][i] * n[c][i];
        d[c][i] *= w[c][i];
        s += i >= k.skip ? d[c][i] * n[c][i] : 0.f;
      }
    }
    s = row_sum<TPR>(s, sh[turn]) / (float)a.dim;      // two places in turn: one barrier a row
    if (!a.dx) continue;
    T* dx = static_cast<T*>(a.dx) + r * a.dim;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const Chunk<V> k(t + c * TPR, a.dim);
#pragma unroll
      for (int i = 0; i < V; ++i) d[c][i] = rstd * (d[c][i] - n[c][i] * s);
      if (a.dh) {
        float f[V];
        load_v<V>(f, static_cast<const T*>(a.dh) + r * a.dhs + k.at, k.n);
#pragma unroll
        for (int i = 0; i < V; ++i) d[c][i] += f[i];
      }
      if (k.used()) store_v<V>(dx + k.at, d[c], k.n);
    }
  }
  if (!a.part && !a.dw) return;
  if (RPB > 1) {                               // the workgroup's rows at once, joined in order
    for (int k = RPB - 1; k > 0; --k) {
      if (slot == k) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) join[(c * V + i) * TPR + t] = dw[c][i];
      }
      __syncthreads();
      if (slot == k - 1) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) dw[c][i] += join[(c * V + i) * TPR + t];
      }
      __syncthreads();
    }
    if (slot > 0) return;
  }
  float* part = a.part ? a.part + (int64_t)blockIdx.x * a.dim : nullptr;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const Chunk<V> k(t + c * TPR, a.dim);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i < k.skip || i >= k.n) continue;
      if (part) part[k.at + i] = dw[c][i];
      else static_cast<W*>(a.dw)[k.at + i] = (W)dw[c][i];
    }
  }
}

// Threads a row and chunks a thread: a wave for up to 128 chunks of 16 bytes (no barrier), then mostly two chunks a thread.  Four hold so many registers that few rows are on the way (backward of
// 4096 x 8192 bf16: 256 threads of four 86 us, 512 of two 66), workgroups of an odd number of waves do not fill the four SIMDs (8191 x 5120: 320 threads of two 115 us, 256 of three 91).
#define CAGC_ROW_SHAPES(chunks, CALL)       \
  if (chunks <= 64) { CALL(64, 1); }        \
  else if (chunks <= 128) { CALL(64, 2); }  \
  else if (chunks <= 256) { CALL(128, 2); } \
  else if (chunks <= 512) { CALL(256, 2); } \
  else if (chunks <= 768) { CALL(256, 3); } \
  else if (chunks <= 1024) { CALL(512, 2); } \
  else if (chunks <= 1536) { CALL(768, 2); } \
  else if (chunks <= 2048) { CALL(1024, 2); } \
  else { CALL(1024, 4); }

constexpr int MOST_CHUNKS = 4096;
int esize(int dtype) { return dtype == CAGC_F32 ? 4 : 2; }
bool row_type(int dtype) { return dtype == CAGC_F32 || dtype == CAGC_F16 || dtype == CAGC_BF16; }
int chunks_of(int64_t dim, int dtype) { return (int)((dim * esize(dtype) + 15) / 16); }
bool dim_ok(int64_t dim, int dtype) { return dim > 0 && dim * esize(dtype) <= (int64_t)MOST_CHUNKS * 16; }

template <class T, class W, int OUT> int launch_some(const Norm& a, hipStream_t st, const char* what) {
  const int chunks = (a.dim + Row<T>::V - 1) / Row<T>::V;
#define CAGC_CALL(TPR, NV) hipLaunchKernelGGL((k_rms_norm<T, W, TPR, NV, OUT>), dim3((unsigned)((a.rows + threads_of(TPR) / TPR - 1) / (threads_of(TPR) / TPR))), dim3(threads_of(TPR)), 0, st, a)
  CAGC_ROW_SHAPES(chunks, CAGC_CALL)
#undef CAGC_CALL
  return check_launch(what);
}
// a launch holds fewer than 2^32 threads: at most 2^21 rows at a time
template <class T, class W, int OUT> int launch_norm(Norm a, hipStream_t st, const char* what) {
  const int64_t rows = a.rows, most = 1 << 21, out = OUT == 0 ? (int64_t)sizeof(T) : 1;
  for (int64_t done = 0; done < rows; done += most) {
    a.rows = rows - done < most ? rows - done : most;
    const int rc = launch_some<T, W, OUT>(a, st, what);
    if (rc != CAGC_OK) return rc;
    a.y = static_cast<char*>(a.y) + most * a.dim * out;
    a.x = static_cast<const T*>(a.x) + most * a.xs;
    if (a.res) a.res = static_cast<const T*>(a.res) + most * a.rs;
    if (a.h) a.h = static_cast<T*>(a.h) + most * a.dim;
    if (a.rstd) a.rstd += most;
    if (a.scale) a.scale += most;
  }
  return CAGC_OK;
}
template <int OUT> int launch_norm_as(const Norm& a, int dtype, int wdtype, hipStream_t st, const char* what) {
  if (dtype == CAGC_F32) return launch_norm<float, float, OUT>(a, st, what);
  if (dtype == CAGC_F16) return wdtype == CAGC_F32 ? launch_norm<_Float16, float, OUT>(a, st, what) : launch_norm<_Float16, _Float16, OUT>(a, st, what);
  return wdtype == CAGC_F32 ? launch_norm<__bf16, float, OUT>(a, st, what) : launch_norm<__bf16, __bf16, OUT>(a, st, what);
}

// Workgroups of a backward: at most as many as 256 CUs hold at once (at these registers 16 waves each, in fp32, whose chunks have half the elements, 24), each taking rows in turn: with a quarter
// more, the rest runs by itself at the end (16384 x 4096 bf16: 1024 workgroups 110 us, 1280 145).  At least four turns each if that still makes 256: each writes a row of shares of dw (2048 x 2048
// fp32: 512 workgroups 19.5 us, 1536 22.4).  Up to four turns of rows are left to one workgroup, which then writes dw itself (16 rows of 512: one launch instead of two, and no workspace).
int bwd_wgs(int64_t rows, int chunks, int dtype) {
  const int rpb = chunks <= 128 ? 4 : 1;
  const int waves = chunks <= 256 && chunks > 128 ? 2 : chunks <= 768 ? 4 : chunks <= 1024 ? 8 : chunks <= 1536 ? 12 : 16;      // of a workgroup
  const int64_t most = 256 * (chunks > 512 && chunks <= 768 ? (dtype == CAGC_F32 ? 4 : 3) : (dtype == CAGC_F32 ? 24 : 16) / waves);
  const int64_t turns = (rows + rpb - 1) / rpb, want = turns / 4 > 256 ? turns / 4 : 256;
  if (turns <= 4) return 1;
  const int64_t wgs = want < most ? want : most;
  return (int)(turns < wgs ? turns : wgs);
}

template <class T, class W> int launch_bwd(const NormBwd& a, void* dw, hipStream_t st, const char* what) {
  const int chunks = (a.dim + Row<T>::V - 1) / Row<T>::V, wgs = bwd_wgs(a.rows, chunks, sizeof(T) == 4 ? CAGC_F32 : CAGC_BF16);
#define CAGC_CALL(TPR, NV) hipLaunchKernelGGL((k_rms_norm_bwd<T, W, TPR, NV>), dim3(wgs), dim3(threads_of(TPR)), 0, st, a)
  CAGC_ROW_SHAPES(chunks, CAGC_CALL)
#undef CAGC_CALL
  int rc = check_launch(what);
  if (rc != CAGC_OK || !a.part) return rc;
  hipLaunchKernelGGL((k_column_sums<W>), dim3((a.dim + 15) / 16), dim3(1024), 0, st, static_cast<W*>(dw), a.part, wgs, a.dim);
  return check_launch(what);
}

}  // namespace
}  // namespace cagc

using namespace cagc;

#define CAGC_NORM_CHECKS(what)                                                                                                          \
  CAGC_REQUIRE(row_type(dtype), "%s: element type %d", what, dtype);                                                                    \
  CAGC_REQUIRE(wdtype == dtype || wdtype == CAGC_F32, "%s: weight type %d for element type %d", what, wdtype, dtype);                   \
  CAGC_REQUIRE(rows >= 0 && rows < (1ll << 31) && dim_ok(dim, dtype), "%s: %lld rows of %lld (at most %d bytes a row)", what, (long long)rows, (long long)dim, MOST_CHUNKS * 16)

extern "C" int cagc_rms_norm_fwd(void* y, void* h, float* rstd, const void* x, const void* residual, const void* w, int64_t rows, int64_t dim, int64_t x_stride,
                                 int64_t res_stride, int dtype, int wdtype, float eps, cagc_stream_t stream) {
  const char* what = "cagc_rms_norm_fwd";
  CAGC_NORM_CHECKS(what);
  if (rows == 0) return CAGC_OK;
  CAGC_REQUIRE(y && x && (!residual || h), "%s: null pointer", what);
  const Norm a = {y, nullptr, h, rstd, x, residual, w, rows, x_stride, res_stride, (int)dim, eps};
  return launch_norm_as<0>(a, dtype, wdtype, as_stream(stream), what);
}
extern "C" int cagc_rms_norm_e4m3(void* q, float* scale, void* h, const void* x, const void* residual, const void* w, int64_t rows, int64_t dim, int64_t x_stride,
                                  int64_t res_stride, int dtype, int wdtype, float eps, cagc_stream_t stream) {
  const char* what = "cagc_rms_norm_e4m3";
  CAGC_NORM_CHECKS(what);
  if (rows == 0) return CAGC_OK;
  CAGC_REQUIRE(q && scale && x && (!residual || h), "%s: null pointer", what);
  const Norm a = {q, scale, h, nullptr, x, residual, w, rows, x_stride, res_stride, (int)dim, eps};
  return launch_norm_as<1>(a, dtype, wdtype, as_stream(stream), what);
}
extern "C" int cagc_quantize_rows_e4m3(void* q, float* scale, const void* x, int64_t rows, int64_t dim, int64_t x_stride, int dtype, cagc_stream_t stream) {
  const char* what = "cagc_quantize_rows_e4m3";
  const int wdtype = dtype;
  CAGC_NORM_CHECKS(what);
  if (rows == 0) return CAGC_OK;
  CAGC_REQUIRE(q && scale && x, "%s: null pointer", what);
  const Norm a = {q, scale, nullptr, nullptr, x, nullptr, nullptr, rows, x_stride, 0, (int)dim, 0.f};
  return launch_norm_as<2>(a, dtype, dtype, as_stream(stream), what);
}
extern "C" int64_t cagc_rms_norm_bwd_workspace(int64_t rows, int64_t dim, int dtype) {
  if (rows <= 0 || !row_type(dtype) || !dim_ok(dim, dtype)) return 0;
  const int wgs = bwd_wgs(rows, chunks_of(dim, dtype), dtype);
  return wgs > 1 ? 4 * dim * wgs : 0;
}
extern "C" int cagc_rms_norm_bwd(void* dx, void* dw, void* ws, const void* dy, const void* dh, const void* h, const void* w, const float* rstd, int64_t rows,
                                 int64_t dim, int64_t dy_stride, int64_t dh_stride, int64_t h_stride, int dtype, int wdtype, cagc_stream_t stream) {
  const char* what = "cagc_rms_norm_bwd";
  CAGC_NORM_CHECKS(what);
  CAGC_REQUIRE(rows > 0, "%s: no rows (the weight's gradient is zero)", what);
  if (!dx && !dw) return CAGC_OK;
  const bool alone = bwd_wgs(rows, chunks_of(dim, dtype), dtype) == 1;
  CAGC_REQUIRE(dy && h && rstd && (!dw || alone || ws), "%s: null pointer", what);
  const NormBwd a = {dx, dw && !alone ? static_cast<float*>(ws) : nullptr, alone ? dw : nullptr, dy, dh, h, w, rstd, rows, dy_stride, dh_stride, h_stride, (int)dim};
  hipStream_t st = as_stream(stream);
  if (dtype == CAGC_F32) return launch_bwd<float, float>(a, dw, st, what);
  if (dtype == CAGC_F16) return wdtype == CAGC_F32 ? launch_bwd<_Float16, float>(a, dw, st, what) : launch_bwd<_Float16, _Float16>(a, dw, st, what);
  return wdtype == CAGC_F32 ? launch_bwd<__bf16, float>(a, dw, st, what) : launch_bwd<__bf16, __bf16>(a, dw, st, what);
}
