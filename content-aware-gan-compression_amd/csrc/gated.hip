// Gated projection: out = act(s x Wg^T + bg) * (s x Wu^T + bu) with W = [Wg; Wu] of 2n rows, and its backward pass.
//
// Both projections are ONE product with the 2n weight rows; a workgroup's tile holds the gate rows and the up rows of the same
// columns, a wave both accumulators of an output, so the activation and the product are the epilogue of the matrix product and the
// pre-activations never travel (a training forward stores them once, for the backward).  Backward, with z = (g, u):
// dz = (dy u act'(g), dy act(g)) [rows, 2n], dx = s dz W, dW = s dz^T x, db = sum of dz's rows.
#include "gated.h"

namespace cagc {
namespace gated {
namespace {

enum { EPI_GATED = 0, EPI_PLAIN = 1 };

struct Product {
  const char* p;         // operand of the output's columns: [rows, K], rows ldp bytes apart (gated: gate rows, then up rows from p2)
  const char* p2;
  const char* q;         // operand of the output's rows
  int64_t ldp, ldq;
  int np, nq;            // columns and rows of the output
  int kbytes, ksteps;    // K in bytes and in steps of 128 bytes
  int splits;            // K is cut into this many pieces, each with a slab of its own
  int tiles_p, tiles_q;
  float* slab;           // [splits][nq][np or 2 np] fp32
  void* out;             // [nq, ldo]
  int64_t ldo;
  float alpha;
  const void* bias;      // [2 np] in the output's type [nullable]
  const float* sp;       // scales of p's rows [2 np] and of q's rows [nq] (e4m3) [nullable]
  const float* sq;
  void* saved;           // pre-activations [nullable]
  int act;
};

typedef __attribute__((address_space(3))) char lds_t;

template <class T> __device__ __forceinline__ void store4(T* p, f32x4 v, int n, bool vec) {
  typedef T tx4 __attribute__((ext_vector_type(4)));
  if (vec && n >= 4) { *reinterpret_cast<tx4*>(p) = tx4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]}; return; }
#pragma unroll
  for (int r = 0; r < 4; ++r) if (r < n) p[r] = (T)v[r];
}
// the gated epilogue for the (up to) four outputs [m][n .. n+3]
template <class O> __device__ __forceinline__ void gated_out(const Product& a, int m, int n, f32x4 g, f32x4 u) {
  const int left = a.np - n;
  const float sq = a.alpha * (a.sq ? a.sq[m] : 1.f);
  f32x4 o;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (r >= left) { g[r] = u[r] = o[r] = 0.f; continue; }
    g[r] *= a.sp ? sq * a.sp[n + r] : sq;
    u[r] *= a.sp ? sq * a.sp[a.np + n + r] : sq;
    if (a.bias) {
      g[r] += (float)static_cast<const O*>(a.bias)[n + r];
      u[r] += (float)static_cast<const O*>(a.bias)[a.np + n + r];
    }
    o[r] = act_of(a.act, g[r]) * u[r];
  }
  const bool vec = (a.np & 3) == 0;
  const int64_t at = (int64_t)m * a.ldo + n;
  store4(static_cast<O*>(a.out) + at, o, left, vec);
  if (!a.saved) return;
  const int64_t plane = (int64_t)a.nq * a.np, i = (int64_t)m * a.np + n;
  if (sizeof(O) == 4) {
    store4(static_cast<float*>(a.saved) + i, g, left, vec);
    store4(static_cast<float*>(a.saved) + plane + i, u, left, vec);
    return;
  }
  typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
  u16x4 hg, hu, lo;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint32_t tg = top24(g[r]), tu = top24(u[r]);
    hg[r] = (uint16_t)(tg >> 8); hu[r] = (uint16_t)(tu >> 8); lo[r] = (uint16_t)((tg & 0xffu) << 8 | (tu & 0xffu));
  }
  uint16_t* s = static_cast<uint16_t*>(a.saved) + i;
  if (vec && left >= 4) {
    *reinterpret_cast<u16x4*>(s) = hg; *reinterpret_cast<u16x4*>(s + plane) = hu; *reinterpret_cast<u16x4*>(s + 2 * plane) = lo;
    return;
  }
  for (int r = 0; r < 4; ++r) if (r < left) { s[r] = hg[r]; s[plane + r] = hu[r]; s[2 * plane + r] = lo[r]; }
}
template <class O> __device__ __forceinline__ void plain_out(const Product& a, int m, int n, f32x4 v) {
  store4(static_cast<O*>(a.out) + (int64_t)m * a.ldo + n, v * a.alpha, a.np - n, (a.ldo & 3) == 0);
}

// ---- tiled product --------------------------------------------------------------------------------------------------------------
// out[m][n] = sum_k q[m][k] p[n][k].  A workgroup of WP x WQ waves makes a tile of BQ rows (m) and BP rows of p (n; gated: BP/2 columns,
// gate and up); K goes by in stages of 128 bytes a row, two stages in LDS: while one is multiplied, the other is filled by loads that
// go straight to LDS.  A stage's row is 8 chunks of 16 bytes, chunk c kept at slot c ^ (row % 8): the 16 rows that a wave reads of one
// chunk then lie in different banks; the loads write LDS in lane order, so the lanes fetch their chunks in that order.
// Rows beyond the operand are read from its last row (their outputs are not stored), chunks beyond K come back as zero.
template <class T, class O, int BP, int BQ, int WP, int WQ, int EPI> struct Tile {      // (O: a class of its own for each kernel)
  static constexpr int NW = WP * WQ, TP = BP / WP, TQ = BQ / WQ, IP = TP / 16, IQ = TQ / 16;
  static constexpr int LOADS = (BP + BQ) / 8 / NW;                 // direct loads of a wave and stage, 8 rows each
  static constexpr int STAGE = (BP + BQ) * 128;
  static_assert((BP / 16) % NW == 0 && (BQ / 8) % NW == 0, "a load's 8 rows lie in one operand");
  f32x4 acc[IP][IQ];

  __device__ __forceinline__ void step(lds_t* __restrict__ cur, lds_t* __restrict__ nxt, const __amdgpu_buffer_rsrc_t (&rs)[3],
                                       const int (&off)[LOADS], int next, bool more, bool tail_ok, int w, int pa, int qa, int c0, int c1) {
    if (more) fill(nxt, rs, off, next, tail_ok, w);
    {
      i32x4 pf[IP][2], qf[IQ][2];
#pragma unroll
      for (int i = 0; i < IP; ++i) {
        const int row = EPI == EPI_GATED && i >= IP / 2 ? pa + BP / 2 * 128 + (i - IP / 2) * 2048 : pa + i * 2048;
        pf[i][0] = *reinterpret_cast<__attribute__((address_space(3))) i32x4*>(cur + row + c0);
        pf[i][1] = *reinterpret_cast<__attribute__((address_space(3))) i32x4*>(cur + row + c1);
      }
#pragma unroll
      for (int j = 0; j < IQ; ++j) {
        qf[j][0] = *reinterpret_cast<__attribute__((address_space(3))) i32x4*>(cur + qa + j * 2048 + c0);
        qf[j][1] = *reinterpret_cast<__attribute__((address_space(3))) i32x4*>(cur + qa + j * 2048 + c1);
      }
#pragma unroll
      for (int j = 0; j < IQ; ++j)
#pragma unroll
        for (int i = 0; i < IP; ++i) acc[i][j] = mma<T>(pf[i], qf[j], acc[i][j]);
    }
  }
  // the loads of a stage: number c of this wave fills the 8 rows from (c * NW + w) * 8
  static __device__ __forceinline__ void fill(lds_t* __restrict__ dst, const __amdgpu_buffer_rsrc_t (&rs)[3], const int (&off)[LOADS], int step,
                                              bool ok, int w) {
#pragma unroll
    for (int c = 0; c < LOADS; ++c) {
      const int first = c * NW * 8;
      const __amdgpu_buffer_rsrc_t r = first < BP / 2 ? rs[0] : (first < BP ? rs[1] : rs[2]);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(dst + (first + w * 8) * 128), 16,
                                               ok ? off[c] : (int)0x80000000, step * 128, 0, 0);
    }
  }
};

// The workgroup's tile: the hardware deals workgroups to the 8 dies in turn, so consecutive numbers of one die are made neighbours,
// and within a die tiles go by in bands of 8 tile rows, whose operands then stay in that die's L2.
__device__ __forceinline__ void tile_of(int b, int tiles_p, int tiles_q, int& tp, int& tq) {
  const int nb = tiles_p * tiles_q, per = nb / 8, rest = nb % 8;
  const int die = b % 8, k = b / 8;
  const int id = die * per + (die < rest ? die : rest) + k;
  const int band = 8 * tiles_p, g = id / band, first = g * 8, rows = min(8, tiles_q - first), in = id - g * band;
  tq = first + in % rows;
  tp = in / rows;
}

template <class T, class O, int BP, int BQ, int WP, int WQ, int EPI>
__global__ __launch_bounds__(WP* WQ * 64) void k_product(Product a) {
  typedef Tile<T, O, BP, BQ, WP, WQ, EPI> K;
  __shared__ __attribute__((aligned(1024))) char stage[2 * K::STAGE];
  lds_t* s0 = (lds_t*)stage;
  lds_t* s1 = s0 + K::STAGE;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wp = w % WP, wq = w / WP;
  int tp, tq;
  tile_of(blockIdx.x, a.tiles_p, a.tiles_q, tp, tq);
  constexpr int COLS = EPI == EPI_GATED ? BP / 2 : BP;
  const int n0 = tp * COLS, m0 = tq * BQ;
  // this split's K steps
  const int per = (a.ksteps + a.splits - 1) / a.splits, k0 = blockIdx.y * per, k1 = min(a.ksteps, k0 + per);

  __amdgpu_buffer_rsrc_t rs[3];
  const int lp0 = EPI == EPI_GATED ? n0 : n0 + BP / 2;
  const char* second = EPI == EPI_GATED ? a.p2 : a.p;
  rs[0] = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p + (int64_t)min(n0, a.np - 1) * a.ldp), 0, 0x7ffffff0, 0x00020000);
  rs[1] = __builtin_amdgcn_make_buffer_rsrc((void*)(second + (int64_t)min(lp0, a.np - 1) * a.ldp), 0, 0x7ffffff0, 0x00020000);
  rs[2] = __builtin_amdgcn_make_buffer_rsrc((void*)(a.q + (int64_t)m0 * a.ldq), 0, 0x7ffffff0, 0x00020000);
  const int chunk = (lane & 7) ^ (lane >> 3);
  int off[K::LOADS];
#pragma unroll
  for (int c = 0; c < K::LOADS; ++c) {
    const int row = (c * K::NW + w) * 8 + (lane >> 3);
    const int first = c * K::NW * 8;
    if (first < BP / 2) off[c] = min(row, max(0, a.np - 1 - n0)) * (int)a.ldp;
    else if (first < BP) off[c] = min(row - BP / 2, max(0, a.np - 1 - lp0)) * (int)a.ldp;
    else off[c] = min(row - BP, a.nq - 1 - m0) * (int)a.ldq;
    off[c] += chunk * 16;
  }
  const int pa = (wp * (EPI == EPI_GATED ? K::TP / 2 : K::TP) + (lane & 15)) * 128, qa = (BP + wq * K::TQ + (lane & 15)) * 128;
  const int c0 = ((lane >> 4) ^ (lane & 7)) * 16, c1 = ((4 + (lane >> 4)) ^ (lane & 7)) * 16;
  auto inside = [&](int step) { return step * 128 + chunk * 16 < a.kbytes; };

  K t;
#pragma unroll
  for (int i = 0; i < K::IP; ++i)
#pragma unroll
    for (int j = 0; j < K::IQ; ++j) t.acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (k0 < k1) K::fill(s0, rs, off, k0, inside(k0), w);
  for (int k = k0; k < k1; ++k) {
    __builtin_amdgcn_s_waitcnt(0x0f70);      // this wave's loads have reached LDS (issued a whole stage ago) ...
    __syncthreads();                         // ... and so have the others'; and everyone is done with the other stage
    t.step(s0, s1, rs, off, k + 1, k + 1 < k1, inside(k + 1), w, pa, qa, c0, c1);
    lds_t* x = s0; s0 = s1; s1 = x;
  }

  // a lane holds 4 consecutive columns of one output row: column 4 (lane / 16) + r, row lane % 16 of each 16 x 16 block
#pragma unroll
  for (int j = 0; j < K::IQ; ++j) {
    const int m = m0 + wq * K::TQ + j * 16 + (lane & 15);
    if (m >= a.nq) continue;
    constexpr int HALF = EPI == EPI_GATED ? K::IP / 2 : K::IP;
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
      const int n = n0 + wp * (EPI == EPI_GATED ? K::TP / 2 : K::TP) + i * 16 + (lane >> 4) * 4;
      if (n >= a.np) continue;
      if (a.splits > 1) {
        const int64_t width = EPI == EPI_GATED ? 2 * (int64_t)a.np : a.np;
        float* s = a.slab + ((int64_t)blockIdx.y * a.nq + m) * width + n;
        const bool vec = (a.np & 3) == 0;
        store4(s, t.acc[i][j], a.np - n, vec);
        if (EPI == EPI_GATED) store4(s + a.np, t.acc[EPI == EPI_GATED ? i + K::IP / 2 : i][j], a.np - n, vec);
      } else if (EPI == EPI_GATED) {
        gated_out<O>(a, m, n, t.acc[i][j], t.acc[EPI == EPI_GATED ? i + K::IP / 2 : i][j]);
      } else {
        plain_out<O>(a, m, n, t.acc[i][j]);
      }
    }
  }
}

// the pieces of a K split, added in order, and the epilogue: four outputs a thread
template <class O, int EPI> __global__ __launch_bounds__(256) void k_join(Product a) {
  const int quads = (a.np + 3) / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (int64_t)quads * a.nq) return;
  const int m = (int)(id / quads), n = (int)(id % quads) * 4, left = a.np - n;
  const int64_t width = EPI == EPI_GATED ? 2 * (int64_t)a.np : a.np;
  f32x4 v[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.slab + ((int64_t)s * a.nq + m) * width + n;
#pragma unroll
    for (int h = 0; h < (EPI == EPI_GATED ? 2 : 1); ++h) {
      if ((a.np & 3) == 0) v[h] += *reinterpret_cast<const f32x4*>(p + h * (int64_t)a.np);
      else
        for (int r = 0; r < 4; ++r) if (r < left) v[h][r] += p[h * (int64_t)a.np + r];
    }
  }
  if (EPI == EPI_GATED) gated_out<O>(a, m, n, v[0], v[1]);
  else plain_out<O>(a, m, n, v[0]);
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------------
// Up to 16 MQ rows of x: bound by the weights' bytes, each read once, straight into registers.  A workgroup makes 16 output columns (16 gate
// and 16 up rows); its waves share out K and are added through LDS.  Rows need no alignment: the loads are 16 bytes from any address.
struct __attribute__((packed, aligned(1))) Any16 { uint32_t v[4]; };
__device__ __forceinline__ i32x4 chunk_at(const char* row, int64_t at, int64_t kbytes) {
  if (at + 16 <= kbytes) return __builtin_bit_cast(i32x4, *reinterpret_cast<const Any16*>(row + at));
  union { uint8_t b[16]; i32x4 v; } u;
  u.v = i32x4{0, 0, 0, 0};
  for (int i = 0; i < 16; ++i) if (at + i < kbytes) u.b[i] = row[at + i];
  return u.v;
}
template <class T, class O, int MQ> __global__ __launch_bounds__(1024) void k_few_rows(Product a) {
  __shared__ f32x4 part[15 * 64 * 2 * MQ];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int n0 = blockIdx.x * 16, row = min(n0 + (lane & 15), a.np - 1);
  const char* pg = a.p + (int64_t)row * a.ldp;
  const char* pu = a.p2 + (int64_t)row * a.ldp;
  const char* q[MQ];
#pragma unroll
  for (int j = 0; j < MQ; ++j) q[j] = a.q + (int64_t)min(j * 16 + (lane & 15), a.nq - 1) * a.ldq;
  f32x4 g[MQ], u[MQ];
#pragma unroll
  for (int j = 0; j < MQ; ++j) g[j] = u[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int whole = a.kbytes / 128;
  const int64_t c0 = (lane >> 4) * 16, c1 = c0 + 64;
  for (int k = w; k < whole; k += nw) {
    const int64_t at = (int64_t)k * 128;
    i32x4 x[2] = {__builtin_bit_cast(i32x4, *reinterpret_cast<const Any16*>(pg + at + c0)), __builtin_bit_cast(i32x4, *reinterpret_cast<const Any16*>(pg + at + c1))};
    i32x4 y[2] = {__builtin_bit_cast(i32x4, *reinterpret_cast<const Any16*>(pu + at + c0)), __builtin_bit_cast(i32x4, *reinterpret_cast<const Any16*>(pu + at + c1))};
#pragma unroll
    for (int j = 0; j < MQ; ++j) {
      const i32x4 z[2] = {__builtin_bit_cast(i32x4, *reinterpret_cast<const Any16*>(q[j] + at + c0)), __builtin_bit_cast(i32x4, *reinterpret_cast<const Any16*>(q[j] + at + c1))};
      g[j] = mma<T>(x, z, g[j]);
      u[j] = mma<T>(y, z, u[j]);
    }
  }
  if (whole * 128 < a.kbytes && whole % nw == w) {
    const int64_t at = (int64_t)whole * 128;
    const i32x4 x[2] = {chunk_at(pg, at + c0, a.kbytes), chunk_at(pg, at + c1, a.kbytes)};
    const i32x4 y[2] = {chunk_at(pu, at + c0, a.kbytes), chunk_at(pu, at + c1, a.kbytes)};
#pragma unroll
    for (int j = 0; j < MQ; ++j) {
      const i32x4 z[2] = {chunk_at(q[j], at + c0, a.kbytes), chunk_at(q[j], at + c1, a.kbytes)};
      g[j] = mma<T>(x, z, g[j]);
      u[j] = mma<T>(y, z, u[j]);
    }
  }
  if (w > 0) {
#pragma unroll
    for (int j = 0; j < MQ; ++j) {
      part[((w - 1) * 2 * MQ + 2 * j) * 64 + lane] = g[j];
      part[((w - 1) * 2 * MQ + 2 * j + 1) * 64 + lane] = u[j];
    }
  }
  __syncthreads();
  if (w > 0) return;
  for (int s = 0; s + 1 < nw; ++s)
#pragma unroll
    for (int j = 0; j < MQ; ++j) {
      g[j] += part[(s * 2 * MQ + 2 * j) * 64 + lane];
      u[j] += part[(s * 2 * MQ + 2 * j + 1) * 64 + lane];
    }
  const int n = n0 + (lane >> 4) * 4;
#pragma unroll
  for (int j = 0; j < MQ; ++j) {
    const int m = j * 16 + (lane & 15);
    if (m < a.nq && n < a.np) gated_out<O>(a, m, n, g[j], u[j]);
  }
}

// ---- layout passes ----------------------------------------------------------------------------------------------------------------
// rows of any stride and alignment -> rows of `width16` chunks of 16 bytes, the rest of the last chunk zero
__global__ __launch_bounds__(256) void k_pad_rows(char* __restrict__ dst, const char* __restrict__ src, int64_t rows, int64_t kbytes, int64_t ld, int width16) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= rows * width16) return;
  const int64_t r = id / width16, c = (id % width16) * 16;
  *reinterpret_cast<i32x4*>(dst + (r * width16 * 16 + c)) = chunk_at(src + r * ld, c, kbytes);
}
// [rows, cols] -> [cols, ldd], zeros behind the last row's column up to ldd (elements; ldd >= rows)
template <class E> __global__ __launch_bounds__(256) void k_transpose(E* __restrict__ dst, const E* __restrict__ src, int rows, int cols, int64_t lds_, int64_t ldd) {
  __shared__ E t[64][65];
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  for (int i = y; i < 64; i += 4) t[i][x] = (r0 + i < rows && c0 + x < cols) ? src[(int64_t)(r0 + i) * lds_ + c0 + x] : E(0);
  __syncthreads();
  for (int i = y; i < 64; i += 4)
    if (c0 + i < cols && r0 + x < ldd) dst[(int64_t)(c0 + i) * ldd + r0 + x] = t[x][i];
}

// dz from the saved pre-activations and dy, in both layouts: z [rows, ldz] (zeros behind 2n) and zt [2n, ldzt] (zeros behind rows), and the
// column sums of each band of 64 rows for db.  A workgroup makes 64 rows x 64 columns, gate and up.
template <class T> __global__ __launch_bounds__(256) void k_dz(T* __restrict__ z, T* __restrict__ zt, float* __restrict__ dbpart, const T* __restrict__ dy, int64_t lddy,
                                                              const void* __restrict__ saved, int rows, int n, int64_t ldz, int64_t ldzt, int act) {
  __shared__ T t[2][64][65];
  __shared__ float col[4][2][64];
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const int64_t plane = (int64_t)rows * n;
  float sg = 0.f, su = 0.f;
  for (int i = y; i < 64; i += 4) {
    float dg = 0.f, du = 0.f;
    const int64_t at = (int64_t)(r0 + i) * n + c0 + x;
    if (r0 + i < rows && c0 + x < n) {
      float g, u, a, da;
      if (sizeof(T) == 4) {
        g = static_cast<const float*>(saved)[at];
        u = static_cast<const float*>(saved)[plane + at];
      } else {
        const uint16_t* s = static_cast<const uint16_t*>(saved) + at;
        const uint32_t lo = s[2 * plane];
        g = from24(s[0], lo >> 8);
        u = from24(s[plane], lo & 0xffu);
      }
      const float d = (float)dy[(int64_t)(r0 + i) * lddy + c0 + x];
      act_grad(act, g, a, da);
      dg = d * u * da;
      du = d * a;
    }
    sg += dg; su += du;
    t[0][i][x] = (T)dg; t[1][i][x] = (T)du;
    if (z && r0 + i < rows) {
      T* p = z + (int64_t)(r0 + i) * ldz;
      if (c0 + x < n) { p[c0 + x] = (T)dg; p[n + c0 + x] = (T)du; }
      if (c0 + x < ldz - 2 * n) p[2 * n + c0 + x] = (T)0.f;
    }
  }
  col[y][0][x] = sg; col[y][1][x] = su;
  __syncthreads();
  if (dbpart && threadIdx.x < 128) {
    const int h = threadIdx.x >> 6;
    if (c0 + x < n) dbpart[(int64_t)blockIdx.y * 2 * n + h * n + c0 + x] = (col[0][h][x] + col[1][h][x]) + (col[2][h][x] + col[3][h][x]);
  }
  if (!zt) return;
  for (int i = y; i < 64; i += 4)
    if (c0 + i < n && r0 + x < ldzt) {
      zt[(int64_t)(c0 + i) * ldzt + r0 + x] = t[0][x][i];
      zt[(int64_t)(n + c0 + i) * ldzt + r0 + x] = t[1][x][i];
    }
}
template <class T> __global__ __launch_bounds__(256) void k_db(T* __restrict__ db, const float* __restrict__ part, int bands, int cols) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int b = 0; b < bands; ++b) s += part[(int64_t)b * cols + c];
  db[c] = (T)s;
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
int esize(int dtype) { return dtype == CAGC_F32 ? 4 : dtype == CAGC_E4M3 ? 1 : 2; }
int64_t up16(int64_t b) { return (b + 15) / 16 * 16; }
int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

struct Plan { int bp, bq, splits; };      // bp = 0: the kernel for few rows (bq rows a workgroup)

// Tile and K split of a product with `cols` columns (of 2 `cols` rows of p when gated), `rows` rows and K of `ksteps` stages.
Plan plan_of(bool gated, int64_t rows, int64_t cols, int ksteps) {
  Plan p;
  const int64_t prows = gated ? 2 * cols : cols;
  auto wgs = [&](int bp, int bq) { return ((prows + bp - 1) / bp) * ((rows + bq - 1) / bq); };
  if (rows > 128 && wgs(256, 256) >= 192) { p = {256, 256, 1}; return p; }
  p = {128, rows <= 32 ? 32 : rows <= 64 ? 64 : 128, 1};
  const int64_t w = wgs(p.bp, p.bq);
  int64_t s = w >= 256 ? 1 : (512 + w - 1) / w;
  if (s > ksteps / 4) s = ksteps / 4;      // at least 4 stages a piece
  if (s > 16) s = 16;
  p.splits = s < 1 ? 1 : (int)s;
  return p;
}

template <class T, class O, int EPI> int launch_product(Product& a, const Plan& p, hipStream_t st, const char* what) {
  const int cols = EPI == EPI_GATED ? p.bp / 2 : p.bp;
  a.tiles_p = cdiv(a.np, cols);
  a.tiles_q = cdiv(a.nq, p.bq);
  const int per = cdiv(a.ksteps, p.splits);
  a.splits = cdiv(a.ksteps, per);          // no empty piece
  const dim3 grid((unsigned)(a.tiles_p * a.tiles_q), (unsigned)a.splits);
  if (p.bp == 256) hipLaunchKernelGGL((k_product<T, O, 256, 256, 4, 2, EPI>), grid, dim3(512), 0, st, a);
  else if (p.bq == 128) hipLaunchKernelGGL((k_product<T, O, 128, 128, 2, 2, EPI>), grid, dim3(256), 0, st, a);
  else if (p.bq == 64) hipLaunchKernelGGL((k_product<T, O, 128, 64, 4, 1, EPI>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_product<T, O, 128, 32, 4, 1, EPI>), grid, dim3(256), 0, st, a);
  int rc = check_launch(what);
  if (rc != CAGC_OK || a.splits == 1) return rc;
  const int64_t quads = (int64_t)((a.np + 3) / 4) * a.nq;
  hipLaunchKernelGGL((k_join<O, EPI>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, a);
  return check_launch(what);
}
// 16-byte alignment of a matrix's rows and row length: what the tiled product's loads want
bool aligned(const void* p, int64_t ld_bytes, int64_t kbytes) { return ((uintptr_t)p % 16) == 0 && ld_bytes % 16 == 0 && kbytes % 16 == 0; }

constexpr int64_t FEW = 32;               // rows up to which the weights are streamed through registers
constexpr int64_t MOST_LD = 7 << 20;      // 256 rows of a tile stay within 32-bit offsets

struct FwdLayout { bool few; Plan plan; int64_t xpad, wpad, slab, total; int64_t kpad; };
FwdLayout fwd_layout(int64_t rows, int64_t n, int64_t k, bool x_ok, bool w_ok, int dtype) {
  FwdLayout l = {};
  const int64_t kb = k * esize(dtype);
  l.kpad = up16(kb);
  l.few = rows <= FEW;
  if (l.few) return l;
  l.plan = plan_of(true, rows, n, (int)((l.kpad + 127) / 128));
  int64_t at = 0;
  if (!x_ok) { l.xpad = at; at += up256(rows * l.kpad); }
  if (!w_ok) { l.wpad = at; at += up256(2 * n * l.kpad); }
  l.slab = at;
  if (l.plan.splits > 1) at += up256(4 * (int64_t)l.plan.splits * rows * 2 * n);
  l.total = at;
  return l;
}

int pad_rows(void* dst, const void* src, int64_t rows, int64_t kbytes, int64_t ld, hipStream_t st, const char* what) {
  const int64_t w16 = up16(kbytes) / 16, total = rows * w16;
  hipLaunchKernelGGL(k_pad_rows, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st, (char*)dst, (const char*)src, rows, kbytes, ld, (int)w16);
  return check_launch(what);
}

template <class T, class O> int few_rows(Product& a, hipStream_t st, const char* what) {
  const int blocks = cdiv(a.np, 16);
  int nw = 4;                              // waves that share K: more where there are few workgroups, at least 2 stages each
  while (nw < 16 && blocks * nw < 4096 && a.ksteps >= 4 * nw) nw *= 2;
  if (a.nq <= 16) hipLaunchKernelGGL((k_few_rows<T, O, 1>), dim3(blocks), dim3(nw * 64), 0, st, a);
  else hipLaunchKernelGGL((k_few_rows<T, O, 2>), dim3(blocks), dim3(nw * 64), 0, st, a);
  return check_launch(what);
}

template <class T, class O> int forward(Product& a, const FwdLayout& l, hipStream_t st, const char* what) {
  return l.few ? few_rows<T, O>(a, st, what) : launch_product<T, O, EPI_GATED>(a, l.plan, st, what);
}

bool sizes_ok(int64_t rows, int64_t n, int64_t k, int dtype) {
  return rows >= 0 && n > 0 && k > 0 && rows < (1ll << 31) - 512 && n < (1 << 29) && k * esize(dtype) <= MOST_LD;
}

struct BwdLayout { int64_t z, zt, wt, xt, dbpart, slab, total; int64_t ldz, ldm; Plan dx, dw; };
BwdLayout bwd_layout(int64_t rows, int64_t n, int64_t k, int dtype, bool need_dx, bool need_dw, bool need_db) {
  BwdLayout l = {};
  const int e = esize(dtype), v = 16 / e;
  l.ldz = (2 * n + v - 1) / v * v;
  l.ldm = (rows + v - 1) / v * v;
  int64_t at = 0;
  if (need_dx) { l.z = at; at += up256(rows * l.ldz * e); l.wt = at; at += up256(k * l.ldz * e); l.dx = plan_of(false, rows, k, (int)((l.ldz * e + 127) / 128)); }
  if (need_dw) { l.zt = at; at += up256(2 * n * l.ldm * e); l.xt = at; at += up256(k * l.ldm * e); l.dw = plan_of(false, 2 * n, k, (int)((l.ldm * e + 127) / 128)); }
  if (need_db) { l.dbpart = at; at += up256(4 * ((rows + 63) / 64) * 2 * n); }
  l.slab = at;
  int64_t s = 0;
  if (need_dx && l.dx.splits > 1) s = 4 * (int64_t)l.dx.splits * rows * k;
  if (need_dw && l.dw.splits > 1) { const int64_t t = 4 * (int64_t)l.dw.splits * 2 * n * k; if (t > s) s = t; }
  l.total = at + up256(s);
  return l;
}

template <class E> int transpose(void* dst, const void* src, int64_t rows, int64_t cols, int64_t ld, int64_t ldd, hipStream_t st, const char* what) {
  const dim3 grid((unsigned)((cols + 63) / 64), (unsigned)((ldd + 63) / 64));
  hipLaunchKernelGGL((k_transpose<E>), grid, dim3(256), 0, st, (E*)dst, (const E*)src, (int)rows, (int)cols, ld, ldd);
  return check_launch(what);
}

template <class T> int backward(void* dx, void* dw, void* db, char* ws, const void* dy, const void* saved, const void* x, const void* w, int64_t rows, int64_t n,
                                int64_t k, int64_t ldx, int64_t ldw, int64_t lddy, int dtype, int act, float scale, hipStream_t st, const char* what) {
  typedef typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type E;
  const int e = sizeof(T);
  const BwdLayout l = bwd_layout(rows, n, k, dtype, dx != nullptr, dw != nullptr, db != nullptr);
  T* z = dx ? (T*)(ws + l.z) : nullptr;
  T* zt = dw ? (T*)(ws + l.zt) : nullptr;
  float* part = db ? (float*)(ws + l.dbpart) : nullptr;
  const int bands = cdiv(dw ? l.ldm : rows, 64);
  hipLaunchKernelGGL((k_dz<T>), dim3((unsigned)((n + 63) / 64), (unsigned)bands), dim3(256), 0, st, z, zt, part, (const T*)dy, lddy, saved, (int)rows, (int)n, l.ldz, l.ldm, act);
  int rc = check_launch(what);
  if (rc != CAGC_OK) return rc;
  if (db) {
    hipLaunchKernelGGL((k_db<T>), dim3((unsigned)((2 * n + 255) / 256)), dim3(256), 0, st, (T*)db, part, cdiv(rows, 64), (int)(2 * n));
    if ((rc = check_launch(what)) != CAGC_OK) return rc;
  }
  Product a = {};
  a.alpha = scale;
  a.slab = (float*)(ws + l.slab);
  a.ldo = k;
  a.np = (int)k;
  if (dx) {
    if ((rc = transpose<E>(ws + l.wt, w, 2 * n, k, ldw, l.ldz, st, what)) != CAGC_OK) return rc;
    a.p = ws + l.wt; a.p2 = a.p; a.ldp = l.ldz * e;
    a.q = (const char*)z; a.ldq = l.ldz * e;
    a.nq = (int)rows;
    a.kbytes = (int)(l.ldz * e); a.ksteps = cdiv(a.kbytes, 128);
    a.out = dx;
    if ((rc = launch_product<T, T, EPI_PLAIN>(a, l.dx, st, what)) != CAGC_OK) return rc;
  }
  if (dw) {
    if ((rc = transpose<E>(ws + l.xt, x, rows, k, ldx, l.ldm, st, what)) != CAGC_OK) return rc;
    a.p = ws + l.xt; a.p2 = a.p; a.ldp = l.ldm * e;
    a.q = (const char*)zt; a.ldq = l.ldm * e;
    a.nq = (int)(2 * n);
    a.kbytes = (int)(l.ldm * e); a.ksteps = cdiv(a.kbytes, 128);
    a.out = dw;
    if ((rc = launch_product<T, T, EPI_PLAIN>(a, l.dw, st, what)) != CAGC_OK) return rc;
  }
  return CAGC_OK;
}

}  // namespace
}  // namespace gated
}  // namespace cagc

using namespace cagc;
using namespace cagc::gated;

extern "C" int64_t cagc_gated_linear_workspace(const void* x, const void* w, int64_t rows, int64_t n, int64_t k, int64_t ldx, int64_t ldw, int dtype) {
  if (!sizes_ok(rows, n, k, dtype)) return 0;
  const int64_t e = esize(dtype);
  return fwd_layout(rows, n, k, aligned(x, ldx * e, k * e), aligned(w, ldw * e, k * e), dtype).total;
}

extern "C" int cagc_gated_linear_fwd(void* out, void* saved, void* ws, const void* x, const void* w, const void* bias, const float* x_scale, const float* w_scale,
                                     int64_t rows, int64_t n, int64_t k, int64_t ldx, int64_t ldw, int dtype, int out_dtype, int act, float scale, cagc_stream_t stream) {
  const char* what = "cagc_gated_linear_fwd";
  CAGC_REQUIRE(dtype == CAGC_F32 || dtype == CAGC_F16 || dtype == CAGC_BF16 || dtype == CAGC_E4M3, "%s: element type %d", what, dtype);
  CAGC_REQUIRE(sizes_ok(rows, n, k, dtype) && ldx >= k && ldw >= k, "%s: bad sizes (rows %lld, n %lld, k %lld)", what, (long long)rows, (long long)n, (long long)k);
  CAGC_REQUIRE(act == CAGC_ACT_SILU || act == CAGC_ACT_GELU, "%s: activation %d", what, act);
  CAGC_REQUIRE(dtype == CAGC_E4M3 ? (out_dtype == CAGC_F16 || out_dtype == CAGC_BF16 || out_dtype == CAGC_F32) && !saved : out_dtype == dtype && !x_scale && !w_scale,
               "%s: output type %d for element type %d", what, out_dtype, dtype);
  if (rows == 0) return CAGC_OK;
  CAGC_REQUIRE(out && x && w, "%s: null pointer", what);
  const int64_t e = esize(dtype), kb = k * e;
  CAGC_REQUIRE(ldx * e <= MOST_LD && ldw * e <= MOST_LD, "%s: rows more than %lld bytes apart", what, (long long)MOST_LD);
  const bool x_ok = aligned(x, ldx * e, kb), w_ok = aligned(w, ldw * e, kb);
  const FwdLayout l = fwd_layout(rows, n, k, x_ok, w_ok, dtype);
  CAGC_REQUIRE(l.total == 0 || ws, "%s: needs %lld bytes of workspace", what, (long long)l.total);
  hipStream_t st = as_stream(stream);
  Product a = {};
  a.p = (const char*)w; a.ldp = ldw * e;
  a.q = (const char*)x; a.ldq = ldx * e;
  a.np = (int)n; a.nq = (int)rows;
  a.kbytes = (int)kb; a.ksteps = cdiv(kb, 128);
  a.out = out; a.ldo = n;
  a.alpha = scale; a.bias = bias; a.sp = w_scale; a.sq = x_scale; a.saved = saved; a.act = act;
  a.splits = 1;
  char* base = (char*)ws;
  int rc;
  if (!l.few) {
    if (!x_ok) { if ((rc = pad_rows(base + l.xpad, x, rows, kb, a.ldq, st, what)) != CAGC_OK) return rc; a.q = base + l.xpad; a.ldq = l.kpad; }
    if (!w_ok) { if ((rc = pad_rows(base + l.wpad, w, 2 * n, kb, a.ldp, st, what)) != CAGC_OK) return rc; a.p = base + l.wpad; a.ldp = l.kpad; }
    a.kbytes = (int)l.kpad;
    a.slab = (float*)(base + l.slab);
  }
  a.p2 = a.p + n * a.ldp;
  if (dtype == CAGC_F32) return forward<float, float>(a, l, st, what);
  if (dtype == CAGC_F16) return forward<_Float16, _Float16>(a, l, st, what);
  if (dtype == CAGC_BF16) return forward<__bf16, __bf16>(a, l, st, what);
  if (out_dtype == CAGC_F32) return forward<e4m3, float>(a, l, st, what);
  if (out_dtype == CAGC_F16) return forward<e4m3, _Float16>(a, l, st, what);
  return forward<e4m3, __bf16>(a, l, st, what);
}

extern "C" int64_t cagc_gated_linear_bwd_workspace(int64_t rows, int64_t n, int64_t k, int dtype, int need_dx, int need_dw, int need_db) {
  if (!sizes_ok(rows, n, k, dtype)) return 0;
  return bwd_layout(rows, n, k, dtype, need_dx, need_dw, need_db).total;
}

extern "C" int cagc_gated_linear_bwd(void* dx, void* dw, void* db, void* ws, const void* dy, const void* saved, const void* x, const void* w, int64_t rows, int64_t n,
                                     int64_t k, int64_t ldx, int64_t ldw, int64_t lddy, int dtype, int act, float scale, cagc_stream_t stream) {
  const char* what = "cagc_gated_linear_bwd";
  CAGC_REQUIRE(dtype == CAGC_F32 || dtype == CAGC_F16 || dtype == CAGC_BF16, "%s: element type %d", what, dtype);
  CAGC_REQUIRE(sizes_ok(rows, n, k, dtype) && ldx >= k && ldw >= k && lddy >= n, "%s: bad sizes", what);
  CAGC_REQUIRE((2 * n + 16) * esize(dtype) <= MOST_LD && (rows + 16) * esize(dtype) <= MOST_LD, "%s: n or rows too large (reductions of at most %lld bytes a row)", what, (long long)MOST_LD);
  CAGC_REQUIRE(act == CAGC_ACT_SILU || act == CAGC_ACT_GELU, "%s: activation %d", what, act);
  CAGC_REQUIRE(rows > 0, "%s: no rows (the gradients of weight and bias are zero)", what);
  if (!dx && !dw && !db) return CAGC_OK;
  CAGC_REQUIRE(ws && dy && saved && (!dw || x) && (!dx || w), "%s: null pointer", what);
  hipStream_t st = as_stream(stream);
  if (dtype == CAGC_F32) return backward<float>(dx, dw, db, (char*)ws, dy, saved, x, w, rows, n, k, ldx, ldw, lddy, dtype, act, scale, st, what);
  if (dtype == CAGC_F16) return backward<_Float16>(dx, dw, db, (char*)ws, dy, saved, x, w, rows, n, k, ldx, ldw, lddy, dtype, act, scale, st, what);
  return backward<__bf16>(dx, dw, db, (char*)ws, dy, saved, x, w, rows, n, k, ldx, ldw, lddy, dtype, act, scale, st, what);
}
