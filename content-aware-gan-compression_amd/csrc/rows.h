// Loads and stores of rows of any alignment, 16 bytes at a time: gfx950's global accesses need none, only the piece that crosses a row's end goes
// element by element.
#pragma once
#include "common.h"

namespace cagc {

struct __attribute__((packed, aligned(1))) Any16 { uint32_t v[4]; };
struct __attribute__((packed, aligned(1))) Any8 { uint32_t v[2]; };

// V elements from p as floats; those from `left` on are zero and not read
template <int V, class T> __device__ __forceinline__ void load_v(float (&f)[V], const T* p, int64_t left) {
  T e[V];
  if (left >= V) {
    constexpr int N = V * (int)sizeof(T) / 16;
    static_assert(N >= 1, "whole 16-byte pieces");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Any16 a = reinterpret_cast<const Any16*>(p)[i];
      __builtin_memcpy(reinterpret_cast<char*>(e) + 16 * i, &a, 16);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (float)e[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i < left ? (float)p[i] : 0.f;
  }
}
template <int V, class T> __device__ __forceinline__ void store_v(T* p, const float (&f)[V], int64_t left) {
  if (left >= V) {
    T e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = (T)f[i];
    Any16 a;
    static_assert(V * sizeof(T) == 16, "one 16-byte piece");
    __builtin_memcpy(&a, e, 16);
    *reinterpret_cast<Any16*>(p) = a;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) if (i < left) p[i] = (T)f[i];
  }
}

// out[c] = sum over r of part[r][c], in a fixed order: a workgroup of 1024 makes 16 columns, 64 rows at a time
template <class T> __global__ __launch_bounds__(1024) void k_column_sums(T* __restrict__ out, const float* __restrict__ part, int rows, int cols) {
  __shared__ float sh[64][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
  float s = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int r = y; r < rows; r += 64) s += part[(int64_t)r * cols + c];
  sh[y][x] = s;
  __syncthreads();
  for (int half = 32; half > 0; half /= 2) {
    if (y < half) sh[y][x] += sh[y + half][x];
    __syncthreads();
  }
  if (y == 0 && c < cols) out[c] = (T)sh[0][x];
}

}  // namespace cagc
