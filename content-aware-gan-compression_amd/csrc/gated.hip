// Gated projection: out = act(s x Wg^T + bg) * (s x Wu^T + bu) with W = [Wg; Wu] of 2n rows, and its backward pass.
//
// Both projections are ONE product with the 2n weight rows; a workgroup's tile holds the gate rows and the up rows of the same
// columns, a wave both accumulators of an output, so the activation and the product are the epilogue of the matrix product and the
// pre-activations never travel (a training forward stores them once, for the backward).  Backward, with z = (g, u):
// dz = (dy u act'(g), dy act(g)) [rows, 2n], dx = s dz W, dW = s dz^T x, db = sum of dz's rows.
#include "gated.h"
#include <type_traits>

namespace cagc {
namespace gated {
namespace {

struct Product {
  const char* p;         // operand of the output's columns (gated: gate rows, then up rows from p2)
  const char* p2;
  const char* q;         // operand of the output's rows
  int64_t ldp, ldq;      // bytes from row to row
  int np, nq;            // columns and rows of the output
  int kbytes;            // K in bytes (a multiple of 16) where a row holds K ...
  int krows;             // ... and in rows where a column does
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
template <class V> __device__ __forceinline__ V lds_read(const lds_t* p) { return *reinterpret_cast<const __attribute__((address_space(3))) V*>(p); }

// ---- tiled product --------------------------------------------------------------------------------------------------------------
// out[m][n] = sum_k q[m][k] p[n][k].  A workgroup of WP x WQ waves makes a tile of BQ rows (m) and BP rows of p (n; gated: BP/2 columns,
// gate and up); K goes by in stages of SB bytes a row, NS stages in LDS: while one is multiplied, the next ones are filled by loads that
// go straight to LDS, in lane order, 16 bytes a lane.
//
// An operand lies in memory with K along its rows (x, W in the forward), or with K down its columns (W for dx; dz and x for dW).  In LDS a stage keeps that
// order: B rows of SB bytes, or SB / size rows of B elements.  Along rows, a wave reads 16 bytes of 16 rows at a time; down columns, the
// transposing read hands each lane 4 elements of a column (16-bit types), or it reads single elements (fp32).  Either way a lane ends up with the k that the other operand's lane
// has: chunk number lane / 16 (and 4 + lane / 16) of the stage's four (eight).  So that those reads fall into different banks, chunk c of LDS row r is kept at c ^ turn(r).
// Nothing outside the operands is read: rows beyond the last repeat it (their outputs are not stored), chunks beyond a row and rows beyond K come back as zero.
template <class T, int B, bool DOWN, int SB> struct Side {
  static constexpr int ES = Type<T>::size, RK = SB / ES;           // elements of K in a stage
  static constexpr int ROW = DOWN ? B * ES : SB, CH = ROW / 16;    // bytes and chunks of an LDS row
  static __device__ __forceinline__ int turn(int row) {
    if (!DOWN) return SB == 64 ? (row >> 2) & 3 : row & 7;
    if (ES == 2) return (((row & 3) | ((row >> 3) & 1) << 2) << 1) & (CH - 1);
    return (((row >> 2) & 3) << 2) & (CH - 1);
  }
  // where the 16 bytes at `at` of the stage come from, as an offset from the tile's first element of the stage.  Along rows: beyond the last row, that row.
  // Down columns: `columns` bytes are left of a row; a chunk beyond them is out of range for good.
  static __device__ __forceinline__ int source(int at, int64_t ld, int last, int columns) {
    const int row = at / ROW, chunk = ((at % ROW) / 16) ^ turn(row);
    if (!DOWN) return min(row, last) * (int)ld + chunk * 16;
    return chunk * 16 < columns ? row * (int)ld + chunk * 16 : (int)0x80000000;
  }
  // Load number c of a wave of NW begins c * NW KB behind load 0: the same chunk of later rows (along rows), a later row of K (down columns).  What decides whether a
  // load lies within K is `first` = its chunk's byte or its row of K for c = 0, and c times this:
  template <int NW> static constexpr int further() { return DOWN ? NW * 1024 / ROW : 0; }
  static __device__ __forceinline__ int first(int at) { return DOWN ? at / ROW : (((at % ROW) / 16) ^ turn(at / ROW)) * 16; }
  // LDS address of this lane's part of the 16 columns / rows `t` (in sixteens)
  static __device__ __forceinline__ int place(int t, int lane) {
    const int g = lane >> 4, l = lane & 15;
    if (!DOWN) return (t * 16 + l) * SB;
    if (ES == 2) { const int row = 8 * g + (l >> 2); return row * ROW + (((2 * t) ^ turn(row)) + ((l & 3) >> 1)) * 16 + (l & 1) * 8; }
    const int row = 4 * g;
    return row * ROW + (((4 * t) ^ turn(row)) + (l >> 2)) * 16 + (l & 3) * 4;
  }
  static __device__ __forceinline__ i32x4 read(const lds_t* stage, int at, int half, int c) {
    if (!DOWN) return lds_read<i32x4>(stage + at + c);
    if constexpr (ES == 2) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* tr_t;
      union { s16x4 h[2]; i32x4 v; } u;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_t)(stage + at + half * 32 * ROW));
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_t)(stage + at + half * 32 * ROW + 4 * ROW));
      return u.v;
    } else {
      i32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = lds_read<int>(stage + at + (half * 16 + j) * ROW);
      return v;
    }
  }
};

// Stages.  Two of 128 bytes a row; with K down the columns of 16-bit operands, where a row of LDS is 512 contiguous bytes of memory whatever SB is, the largest tile takes five of 64, so that a load has
// three stages' products to arrive in (dW of 8192 x 2048 -> 8192 bf16: 411 -> 396 us, with zeros for operands, which leave the clock alone, 376 -> 312).  Elsewhere five are slower: along rows a load
// would fetch half lines (the forward of that: 432 -> 457 us), two smaller workgroups on a CU cover each other's waits (1024 x 2048 ...: 26 -> 31 us), and fp32's products take 16 times as long.
template <class T, int BQ, bool DP> struct Stages {
  static constexpr bool FIVE = DP && BQ == 256 && Type<T>::size == 2;
  static constexpr int SB = FIVE ? 64 : 128, NS = FIVE ? 5 : 2;
};

template <class T, class O, int BP, int BQ, int WP, int WQ, bool DP, bool DQ> struct Tile {      // (O: a class of its own for each kernel)
  static constexpr int SB = Stages<T, BQ, DP>::SB, NS = Stages<T, BQ, DP>::NS;
  typedef Side<T, BP, DP, SB> P;
  typedef Side<T, BQ, DQ, SB> Q;
  static constexpr int NW = WP * WQ, TP = BP / WP, TQ = BQ / WQ, IP = TP / 16, IQ = TQ / 16;
  static constexpr int LP = BP * SB / 1024 / NW, LQ = BQ * SB / 1024 / NW;         // loads of 1 KB of a wave and stage
  static constexpr int STAGE = (BP + BQ) * SB, LDS = NS * STAGE;
  static_assert(BP / 2 * SB % (1024 * NW) == 0 && BQ * SB % (1024 * NW) == 0, "a wave's loads lie in one operand, and in one half of p");
  f32x4 acc[IP][IQ];
  int pa[IP], qa[IQ];              // LDS places of this lane's operands
  int po[LP], qo[LQ];              // sources of this lane's loads
  int pk, qk;                      // Side::first of them
  int ends_p, ends_q;              // where K ends, in rows of K (down columns) or bytes (along rows)

  // load number c of this wave and stage `step`: zeros where K (of this split) has ended
  __device__ __forceinline__ void load(lds_t* __restrict__ dst, int c, const char* p, const char* p2, const char* q, int step, int w) {
    const bool is_p = c < LP;
    const int at = is_p ? c * NW * 1024 : BP * SB + (c - LP) * NW * 1024;
    const char* from = is_p ? (!DP && at >= BP / 2 * SB ? p2 : p) : q;
    const bool ok = is_p ? pk + c * P::template further<NW>() < ends_p - step * (DP ? P::RK : SB) : qk + (c - LP) * Q::template further<NW>() < ends_q - step * (DQ ? Q::RK : SB);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, 0x7ffffff0, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(dst + at + w * 1024), 16, ok ? (is_p ? po[c < LP ? c : 0] : qo[c < LP ? 0 : c - LP]) : (int)0x80000000, 0, 0, 0);
  }
  // A stage goes by in H pieces of K; of a piece, p's IP parts are held in registers while q's IQ parts pass.
  typedef typename Piece<T>::type part;
  static constexpr int H = SB / 128 * (Piece<T>::count - 1) + 1, N = H * IQ, L = LP + LQ;
  static constexpr int LATE = IQ >= 4 ? (Type<T>::size > 1 ? 4 : 2) : IQ;      // parts of q read ahead, and multiplied behind the barrier
  template <class S> static __device__ __forceinline__ part read(const lds_t* side, int at, int h, int c0, int c1) {
    if constexpr (Piece<T>::count == 2) return S::read(side, at, h, h ? c1 : c0);
    else return join(S::read(side, at, 0, c0), S::read(side, at, 1, c1));
  }
  __device__ __forceinline__ part read_q(const lds_t* stage, int k, int c0, int c1) { return read<Q>(stage + BP * SB, qa[k % IQ], k / IQ, c0, c1); }
  // The first stages' loads, and the first reads (of stage 0, which `s0` is).
  __device__ __forceinline__ void begin(lds_t* __restrict__ s0, lds_t* __restrict__ s1, part (&first)[IP], part (&ahead)[LATE], const char* p, const char* p2, const char* q, int64_t dp, int64_t dq,
                                        int k0, int w, int c0, int c1) {
#pragma unroll
    for (int c = 0; c < L; ++c) load(s0, c, p, p2, q, k0, w);
#pragma unroll
    for (int n = 1; n < NS; ++n)
#pragma unroll
      for (int c = 0; c < L; ++c) load(s1 + (n - 1) * STAGE, c, p + n * dp, p2 + n * dp, q + n * dq, k0 + n, w);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 1) * L) : "memory");
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < IP; ++i) first[i] = read<P>(s0, pa[i], 0, c0, c1);
#pragma unroll
    for (int k = 0; k < LATE; ++k) ahead[k] = read_q(s0, k, c0, c1);
  }
  // One stage, in `cur`; the first piece of p is in `first`, the first parts of q in `ahead`.  q is read LATE parts ahead, each read and load between the products of one part and the next (the order is
  // pinned).  When the barrier comes, all of the stage has been read, and behind it the next one is in `nxt` for everyone and `cur` is free: the loads of the stage NS further on and the next stage's first
  // reads run under the last LATE parts' products.
  // (One function with both stages as restricted pointers: the compiler then knows that the loads do not touch what is read, and does not wait for them.)
  __device__ __forceinline__ void step(lds_t* __restrict__ cur, lds_t* __restrict__ nxt, part (&first)[IP], part (&then)[IP], part (&ahead)[LATE], const char* p, const char* p2, const char* q, int far,
                                       int w, int c0, int c1) {
    part last[IP], qf[N];
#pragma unroll
    for (int k = 0; k < LATE; ++k) qf[k] = ahead[k];
#pragma unroll
    for (int k = 0; k < N - LATE; ++k) {
      qf[k + LATE] = read_q(cur, k + LATE, c0, c1);
      if (H == 2 && k < IP) last[k] = read<P>(cur, pa[k < IP ? k : 0], 1, c0, c1);
      if (H == 2 && k == N - LATE - 1) {
#pragma unroll
        for (int i = k + 1; i < IP; ++i) last[i] = read<P>(cur, pa[i], 1, c0, c1);
      }
#pragma unroll
      for (int i = 0; i < IP; ++i) acc[i][k % IQ] = mma<T>(H == 2 && k >= IQ ? last[i] : first[i], qf[k], acc[i][k % IQ]);
      __builtin_amdgcn_sched_barrier(0);
    }
    // this wave's loads of the next stage have reached LDS (those of the NS - 2 behind it may be on their way), its reads are done; and so are the others'
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * L) : "memory");
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int l = 0; l < LATE; ++l) {
      ahead[l] = read_q(nxt, l, c0, c1);
#pragma unroll
      for (int i = 0; i < IP; ++i) if (i * LATE / IP == l) then[i] = read<P>(nxt, pa[i], 0, c0, c1);
#pragma unroll
      for (int c = 0; c < L; ++c) if (c * LATE / L == l) load(cur, c, p, p2, q, far, w);
#pragma unroll
      for (int i = 0; i < IP; ++i) acc[i][(N - LATE + l) % IQ] = mma<T>(H == 2 ? last[i] : first[i], qf[N - LATE + l], acc[i][(N - LATE + l) % IQ]);
      __builtin_amdgcn_sched_barrier(0);
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

// A tile's results leave through LDS, so that whole rows of the tile are written at once (a lane holds 4 columns of one row; stores of its 8 bytes, 32 contiguous
// bytes a row, took three times as long).  ROWS x COLS elements of type E at `lds`, chunk c of row r at c ^ (r % 16).
template <class E, int ROWS, int COLS, int NT> struct Out {
  static constexpr int ROW = COLS * (int)sizeof(E), CH = ROW / 16, BYTES = ROWS * ROW;
  typedef E e4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ void put(lds_t* lds, int row, int col, e4 v) {
    const int byte = col * (int)sizeof(E);
    *reinterpret_cast<__attribute__((address_space(3))) e4*>(lds + row * ROW + (((byte / 16) ^ (row & (CH < 16 ? CH - 1 : 15))) * 16) + byte % 16) = v;
  }
  static __device__ __forceinline__ void store(const lds_t* lds, E* base, int64_t ld, int rows, int cols) {
#pragma unroll
    for (int c = 0; c < (ROWS * CH + NT - 1) / NT; ++c) {
      const int id = c * NT + threadIdx.x, row = id / CH, chunk = id % CH, col = chunk * (16 / (int)sizeof(E));
      if (ROWS * CH % NT && id >= ROWS * CH) return;
      if (row >= rows || col >= cols) continue;
      const i32x4 v = lds_read<i32x4>(lds + row * ROW + ((chunk ^ (row & (CH < 16 ? CH - 1 : 15))) * 16));
      E* to = base + (int64_t)row * ld + col;
      if (col + 16 / (int)sizeof(E) <= cols) *reinterpret_cast<Any16*>(to) = __builtin_bit_cast(Any16, v);
      else {
        union { i32x4 v; E e[16 / sizeof(E)]; } u;
        u.v = v;
#pragma unroll
        for (int i = 0; i < 16 / (int)sizeof(E); ++i) if (i < cols - col) to[i] = u.e[i];
      }
    }
  }
};

// four values from s[n], those from s[last + 1] on repeating s[last]
template <class O> __device__ __forceinline__ f32x4 four_of(const O* s, int n, int last) {
  f32x4 b;
#pragma unroll
  for (int r = 0; r < 4; ++r) b[r] = (float)s[min(n + r, last)];
  return b;
}
template <int ACT> __device__ __forceinline__ f32x4 gate(f32x4 g, f32x4 u) {
  f32x4 o;
#pragma unroll
  for (int r = 0; r < 4; ++r) o[r] = act_of(ACT, g[r]) * u[r];
  return o;
}
template <class E> __device__ __forceinline__ void put4(E* p, f32x4 v, int left) {
#pragma unroll
  for (int r = 0; r < 4; ++r) if (r < left) p[r] = (E)v[r];
}

// The forward has K along the rows of both and the gated epilogue; the backward's products have it down p's columns (DP), and down q's for dW (DQ).
template <class T, class O, int BP, int BQ, int WP, int WQ, bool DP, bool DQ>
__global__ __launch_bounds__(WP* WQ * 64) void k_product(Product a) {
  typedef Tile<T, O, BP, BQ, WP, WQ, DP, DQ> K;
  constexpr bool GATED = !DP;
  constexpr int COLS = GATED ? BP / 2 : BP, NT = WP * WQ * 64;
  __shared__ __attribute__((aligned(1024))) char stage[K::LDS];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wp = w % WP, wq = w / WP;
  int tp, tq;
  tile_of(blockIdx.x, a.tiles_p, a.tiles_q, tp, tq);
  const int n0 = tp * COLS, m0 = tq * BQ;
  const int stages = DP ? (a.krows + K::P::RK - 1) / K::P::RK : (a.kbytes + K::SB - 1) / K::SB;
  const int per = (stages + a.splits - 1) / a.splits, k0 = blockIdx.y * per, k1 = min(stages, k0 + per);      // this split's stages

  K t;
  // first elements of the tile's operands at stage k0, and how far a stage moves them
  const int64_t dp = DP ? K::P::RK * a.ldp : K::SB, dq = DQ ? K::Q::RK * a.ldq : K::SB;
  const char* p = a.p + (DP ? (int64_t)n0 * K::P::ES : (int64_t)n0 * a.ldp) + k0 * dp;
  const char* p2 = GATED ? a.p2 + (int64_t)n0 * a.ldp + k0 * dp : nullptr;
  const char* q = a.q + (DQ ? (int64_t)m0 * K::Q::ES : (int64_t)m0 * a.ldq) + k0 * dq;
  const int mine = w * 1024 + lane * 16;
  t.pk = K::P::first(mine);
  t.qk = K::Q::first(mine);
#pragma unroll
  for (int c = 0; c < K::LP; ++c) {
    const int at = c * K::NW * 1024 + mine;
    const bool up = GATED && c * K::NW * 1024 >= BP / 2 * K::SB;
    t.po[c] = K::P::source(up ? at - BP / 2 * K::SB : at, a.ldp, a.np - 1 - n0, (a.np - n0) * K::P::ES);
  }
#pragma unroll
  for (int c = 0; c < K::LQ; ++c) t.qo[c] = K::Q::source(c * K::NW * 1024 + mine, a.ldq, a.nq - 1 - m0, (a.nq - m0) * K::Q::ES);
#pragma unroll
  for (int i = 0; i < K::IP; ++i)
    t.pa[i] = K::P::place(GATED ? (i < K::IP / 2 ? wp * (K::IP / 2) + i : BP / 32 + wp * (K::IP / 2) + i - K::IP / 2) : wp * K::IP + i, lane);
#pragma unroll
  for (int j = 0; j < K::IQ; ++j) t.qa[j] = K::Q::place(wq * K::IQ + j, lane);
  const int turn = K::SB == 64 ? (lane >> 2) & 3 : lane & 7, c0 = ((lane >> 4) ^ turn) * 16, c1 = ((4 + (lane >> 4)) ^ turn) * 16;
#pragma unroll
  for (int i = 0; i < K::IP; ++i)
#pragma unroll
    for (int j = 0; j < K::IQ; ++j) t.acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  t.ends_p = DP ? min(a.krows, k1 * K::P::RK) : min(a.kbytes, k1 * K::SB);
  t.ends_q = DQ ? min(a.krows, k1 * K::Q::RK) : min(a.kbytes, k1 * K::SB);
  typename K::part pf[2][K::IP], ahead[K::LATE];
  lds_t* cur = (lds_t*)stage;
  lds_t* const stop = cur + K::LDS;
  t.begin(cur, cur + K::STAGE, pf[0], ahead, p, p2, q, dp, dq, k0, w, c0, c1);
  p += K::NS * dp; p2 += K::NS * dp; q += K::NS * dq;
  for (int k = k0; k < k1; k += 2) {         // two stages a turn, each with registers of its own for p (an odd number of stages ends with one of zeros)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      lds_t* const nxt = cur + K::STAGE == stop ? (lds_t*)stage : cur + K::STAGE;
      t.step(cur, nxt, pf[h], pf[1 - h], ahead, p, p2, q, k + h + K::NS, w, c0, c1);
      p += dp; p2 += dp; q += dq;
      cur = nxt;
    }
  }
  // the last loads (zeros) and reads have ended: the stages are free for the results
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

  // a lane holds columns 4 (lane / 16) .. + 3 of row lane % 16 of each 16 x 16 block
  lds_t* const out = (lds_t*)stage;
  const int mw = wq * K::TQ + (lane & 15), nw = wp * (GATED ? K::TP / 2 : K::TP) + (lane >> 4) * 4;
  const int rows = a.nq - m0, cols = a.np - n0;
  constexpr int HI = GATED ? K::IP / 2 : 0, NI = GATED ? K::IP / 2 : K::IP;      // (accumulators of up: HI + i)
  if (BP < 256 && a.splits > 1) {            // (the largest tile is taken only where there are many)
    const int64_t width = GATED ? 2 * (int64_t)a.np : a.np;
    float* base = a.slab + ((int64_t)blockIdx.y * a.nq + m0) * width + n0;
#pragma unroll
    for (int j = 0; j < K::IQ; ++j) {
      const int m = mw + j * 16;
#pragma unroll
      for (int i = 0; i < K::IP; ++i) {
        const int h = GATED && i >= HI ? 1 : 0, n = nw + (i - h * HI) * 16;
        if (m < rows && n < cols) {
          float* to = base + m * width + h * (int64_t)a.np + n;
          if (n + 4 <= cols) *reinterpret_cast<Any16*>(to) = __builtin_bit_cast(Any16, t.acc[i][j]);
          else put4(to, t.acc[i][j], cols - n);
        }
      }
    }
    return;
  }
  typedef O o4 __attribute__((ext_vector_type(4)));
  if constexpr (!GATED) {
    // in as many turns over the tile's rows as its results are larger than the stages
    constexpr int TURNS = (BQ * COLS * (int)sizeof(O) + K::LDS - 1) / K::LDS, R = BQ / TURNS;
    typedef Out<O, R, COLS, NT> Z;
    static_assert(Z::BYTES <= K::LDS && (TURNS == 1 || TURNS == WQ), "a turn: the rows of one row of waves");
    O* base = static_cast<O*>(a.out) + (int64_t)m0 * a.ldo + n0;
#pragma unroll
    for (int turn = 0; turn < TURNS; ++turn) {
      if (TURNS == 1 || wq == turn) {
#pragma unroll
        for (int j = 0; j < K::IQ; ++j)
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const f32x4 v = t.acc[i][j] * a.alpha;
            Z::put(out, mw + j * 16 - turn * R, nw + i * 16, o4{(O)v[0], (O)v[1], (O)v[2], (O)v[3]});
          }
      }
      __syncthreads();
      Z::store(out, base + (int64_t)turn * R * a.ldo, a.ldo, rows - turn * R, cols);
      if (turn + 1 < TURNS) __syncthreads();
    }
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int n = n0 + nw + i * 16, last = a.np - 1;
      const O* bias = static_cast<const O*>(a.bias);
      f32x4 sg, su, bg, bu;
      sg = su = f32x4{a.alpha, a.alpha, a.alpha, a.alpha};
      bg = bu = f32x4{0.f, 0.f, 0.f, 0.f};
      if (a.sp) { sg *= four_of(a.sp, n, last); su *= four_of(a.sp + a.np, n, last); }
      if (bias) { bg = four_of(bias, n, last); bu = four_of(bias + a.np, n, last); }
#pragma unroll
      for (int j = 0; j < K::IQ; ++j) {
        if constexpr (Type<T>::size == 1) {      // one scale after the other: their product may leave fp32's range where the scaled sum does not
          const float q = a.sq ? a.sq[min(m0 + mw + j * 16, a.nq - 1)] : 1.f;
          t.acc[i][j] *= q;
          t.acc[HI + i][j] *= q;
        }
        t.acc[i][j] = t.acc[i][j] * sg + bg;
        t.acc[HI + i][j] = t.acc[HI + i][j] * su + bu;
      }
    }
    typedef Out<O, BQ, COLS, NT> Z;
    static_assert(Z::BYTES <= K::LDS, "the results fit the stages");
    auto put_out = [&](auto act) {
#pragma unroll
      for (int j = 0; j < K::IQ; ++j)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const f32x4 v = gate<decltype(act)::value>(t.acc[i][j], t.acc[HI + i][j]);
          Z::put(out, mw + j * 16, nw + i * 16, o4{(O)v[0], (O)v[1], (O)v[2], (O)v[3]});
        }
    };
    if (a.act == CAGC_ACT_SILU) put_out(std::integral_constant<int, CAGC_ACT_SILU>{});
    else put_out(std::integral_constant<int, CAGC_ACT_GELU>{});
    __syncthreads();
    Z::store(out, static_cast<O*>(a.out) + (int64_t)m0 * a.ldo + n0, a.ldo, rows, cols);
    if (!a.saved) return;
    const int64_t plane = (int64_t)a.nq * a.np, first = (int64_t)m0 * a.np + n0;
    if constexpr (sizeof(O) == 4) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < K::IQ; ++j)
#pragma unroll
          for (int i = 0; i < NI; ++i) Z::put(out, mw + j * 16, nw + i * 16, t.acc[h * HI + i][j]);
        __syncthreads();
        Z::store(out, static_cast<float*>(a.saved) + h * plane + first, a.np, rows, cols);
      }
    } else {
      typedef Out<uint16_t, BQ, COLS, NT> S;
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      uint16_t* saved = static_cast<uint16_t*>(a.saved) + first;
#pragma unroll
      for (int h = 0; h < 3; ++h) {            // two places in turn: one barrier a plane
        lds_t* const at = 2 * S::BYTES <= K::LDS ? out + (h & 1 ? 0 : S::BYTES) : out;
        if (2 * S::BYTES > K::LDS) __syncthreads();
#pragma unroll
        for (int j = 0; j < K::IQ; ++j)
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const f32x4 g = t.acc[i][j], u = t.acc[HI + i][j];
            const u32x2 v = h == 0 ? u32x2{upper2(g[0], g[1]), upper2(g[2], g[3])}
                                   : (h == 1 ? u32x2{upper2(u[0], u[1]), upper2(u[2], u[3])} : u32x2{third2(g[0], u[0], g[1], u[1]), third2(g[2], u[2], g[3], u[3])});
            S::put(at, mw + j * 16, nw + i * 16, __builtin_bit_cast(typename S::e4, v));
          }
        __syncthreads();
        S::store(at, saved + h * plane, a.np, rows, cols);
      }
    }
  }
}

// the gated epilogue for the (up to) four outputs [m][n .. n+3], straight to memory
template <class O> __device__ __forceinline__ void gated_out(const Product& a, int m, int n, f32x4 g, f32x4 u) {
  const int left = a.np - n, last = a.np - 1;
  const O* bias = static_cast<const O*>(a.bias);
  const float q = a.alpha * (a.sq ? a.sq[m] : 1.f);
  g *= q; u *= q;                                // (one scale after the other, as in the tiles' epilogue)
  if (a.sp) { g *= four_of(a.sp, n, last); u *= four_of(a.sp + a.np, n, last); }
  if (bias) { g += four_of(bias, n, last); u += four_of(bias + a.np, n, last); }
  put4(static_cast<O*>(a.out) + (int64_t)m * a.ldo + n, a.act == CAGC_ACT_SILU ? gate<CAGC_ACT_SILU>(g, u) : gate<CAGC_ACT_GELU>(g, u), left);
  if (!a.saved) return;
  const int64_t plane = (int64_t)a.nq * a.np, i = (int64_t)m * a.np + n;
  if (sizeof(O) == 4) {
    put4(static_cast<float*>(a.saved) + i, g, left);
    put4(static_cast<float*>(a.saved) + plane + i, u, left);
    return;
  }
  uint16_t* s = static_cast<uint16_t*>(a.saved) + i;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r < left) {
      s[r] = (uint16_t)(bits(g[r]) >> 16);
      s[plane + r] = (uint16_t)(bits(u[r]) >> 16);
      s[2 * plane + r] = (uint16_t)((bits(g[r]) & 0xff00u) | ((bits(u[r]) >> 8) & 0xffu));
    }
}

// the pieces of a K split, added in order, and the epilogue: four outputs a thread
template <class O, bool GATED> __global__ __launch_bounds__(256) void k_join(Product a) {
  const int quads = (a.np + 3) / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (int64_t)quads * a.nq) return;
  const int m = (int)(id / quads), n = (int)(id % quads) * 4, left = a.np - n;
  const int64_t width = GATED ? 2 * (int64_t)a.np : a.np;
  constexpr int HALVES = GATED ? 2 : 1, AHEAD = 8;
  const int64_t slab = a.nq * width;
  const float* p = a.slab + m * width + n;
  f32x4 v[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  int s = 0;
  if (left >= 4) {
    for (; s + AHEAD <= a.splits; s += AHEAD, p += AHEAD * slab) {      // (16 slabs of 256 x 128: one after the other 7.1 us, 4.7; 64: 19, 6.8)
      f32x4 e[AHEAD][HALVES];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
#pragma unroll
        for (int h = 0; h < HALVES; ++h) e[i][h] = __builtin_bit_cast(f32x4, *reinterpret_cast<const Any16*>(p + i * slab + h * (int64_t)a.np));
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
#pragma unroll
        for (int h = 0; h < HALVES; ++h) v[h] += e[i][h];
    }
  }
  for (; s < a.splits; ++s, p += slab)
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
      if (left >= 4) v[h] += __builtin_bit_cast(f32x4, *reinterpret_cast<const Any16*>(p + h * (int64_t)a.np));
      else
        for (int r = 0; r < 4; ++r) if (r < left) v[h][r] += p[h * (int64_t)a.np + r];
  if (GATED) gated_out<O>(a, m, n, v[0], v[1]);
  else put4(static_cast<O*>(a.out) + (int64_t)m * a.ldo + n, v[0] * a.alpha, left);
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------------
// Up to 16 MQ rows of x: bound by the weights' bytes, each read once, straight into registers.  A workgroup makes C output columns; its waves share out K, 128 bytes a turn, and are added
// through LDS.  C = 16: 16 gate rows and 16 up rows, a product for each; C = 8: 8 gate and 8 up rows in ONE product, twice the workgroups: a CU brings in about 40 GB/s whatever its
// waves have on the way (more turns' loads at once changed nothing), so where there are fewer workgroups than CUs their number decides.
// Rows need no alignment: the loads are 16 bytes from any address.
__device__ __forceinline__ i32x4 load16(const char* p) { return __builtin_bit_cast(i32x4, *reinterpret_cast<const Any16*>(p)); }
// chunk of 16 bytes at `at` of a row of kbytes: zero behind its end (the row's last 16 bytes, shifted down)
__device__ __forceinline__ i32x4 chunk_at(const char* row, int64_t at, int64_t kbytes) {
  if (at + 16 <= kbytes) return load16(row + at);
  union { uint8_t b[16]; uint64_t q[2]; i32x4 v; } u;
  u.v = i32x4{0, 0, 0, 0};
  if (at >= kbytes) return u.v;
  if (kbytes >= 16) {
    u.v = load16(row + kbytes - 16);
    const int s = (int)(at + 16 - kbytes) * 8;      // 8 .. 120 bits
    u.q[0] = s < 64 ? (u.q[0] >> s | u.q[1] << (64 - s)) : u.q[1] >> (s - 64);
    u.q[1] = s < 64 ? u.q[1] >> s : 0;
    return u.v;
  }
  for (int i = 0; i < 16; ++i) if (at + i < kbytes) u.b[i] = row[at + i];
  return u.v;
}
template <class T> __device__ __forceinline__ f32x4 mma128(const i32x4 (&a)[2], const i32x4 (&b)[2], f32x4 c) {
  if constexpr (Piece<T>::count == 2) return mma<T>(a[1], b[1], mma<T>(a[0], b[0], c));
  else return mma<T>(join(a[0], a[1]), join(b[0], b[1]), c);
}
template <class T, class O, int MQ, int C> __global__ __launch_bounds__(1024) void k_few_rows(Product a) {
  constexpr int P = C / 8;                 // products a turn
  extern __shared__ f32x4 part[];          // [nw / 2][MQ][P][64]
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6, r = lane & 15;
  const int n0 = blockIdx.x * C, c0 = (lane >> 4) * 16;
  // this lane's rows
  const char* row[P];
  const char* q[MQ];
#pragma unroll
  for (int i = 0; i < P; ++i) row[i] = ((P == 1 ? r >= 8 : i == 1) ? a.p2 : a.p) + (int64_t)min(n0 + r % C, a.np - 1) * a.ldp + c0;
#pragma unroll
  for (int j = 0; j < MQ; ++j) q[j] = a.q + (int64_t)min(j * 16 + r, a.nq - 1) * a.ldq + c0;
  f32x4 acc[MQ][P];
#pragma unroll
  for (int j = 0; j < MQ; ++j)
#pragma unroll
    for (int i = 0; i < P; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  i32x4 x[P][2], z[MQ][2];
  auto mul = [&]() {
#pragma unroll
    for (int j = 0; j < MQ; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) acc[j][i] = mma128<T>(x[i], z[j], acc[j][i]);
  };
  const int whole = a.kbytes / 128;
  // a piece of the rows each, in one stretch (every nw-th 128 bytes instead: 1 x 8192 -> 4096 bf16 33.6 instead of 29.0 us, 1 x 4096 -> 8192 fp32 56 instead of 48)
  const int q0 = (int)((int64_t)whole * w / nw), q1 = (int)((int64_t)whole * (w + 1) / nw);
  for (int k = q0; k < q1; ++k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < P; ++i) x[i][h] = load16(row[i] + k * 128ll + h * 64);
#pragma unroll
      for (int j = 0; j < MQ; ++j) z[j][h] = load16(q[j] + k * 128ll + h * 64);
    }
    mul();
  }
  if (whole * 128 < a.kbytes && w == nw - 1) {
    const int64_t o = whole * 128ll + c0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < P; ++i) x[i][h] = chunk_at(row[i] - c0, o + h * 64, a.kbytes);
#pragma unroll
      for (int j = 0; j < MQ; ++j) z[j][h] = chunk_at(q[j] - c0, o + h * 64, a.kbytes);
    }
    mul();
  }
  for (int half = nw / 2; half > 0; half /= 2) {      // the upper half of the waves hands its sums to the lower
    if (w >= half && w < 2 * half) {
#pragma unroll
      for (int j = 0; j < MQ; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) part[(((w - half) * MQ + j) * P + i) * 64 + lane] = acc[j][i];
    }
    __syncthreads();
    if (w < half) {
#pragma unroll
      for (int j = 0; j < MQ; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) acc[j][i] += part[((w * MQ + j) * P + i) * 64 + lane];
    }
    __syncthreads();
  }
  // the sums once more through LDS: every wave stores some rows, and gate and up meet (C = 8: up is in the upper 32 lanes)
  if (w == 0) {
#pragma unroll
    for (int j = 0; j < MQ; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) part[(j * P + i) * 64 + lane] = acc[j][i];
  }
  __syncthreads();
  const int n = n0 + (lane >> 4) * 4;
  if (P == 1 && lane >= 32) return;
  for (int j = w; j < MQ; j += nw) {
    const int m = j * 16 + r;
    if (m < a.nq && n < a.np) gated_out<O>(a, m, n, part[j * P * 64 + lane], P == 1 ? part[j * 64 + lane + 32] : part[(j * P + 1) * 64 + lane]);
  }
}

// ---- layout passes ----------------------------------------------------------------------------------------------------------------
// rows of any stride and alignment -> rows of whole 16-byte chunks, the rest of the last chunk zero; up to two operands in one launch
struct Pad { char* dst; const char* src; int64_t rows, kbytes, ld; };
__global__ __launch_bounds__(256) void k_pad_rows(Pad a, Pad b) {
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < a.rows + b.rows; i += (int64_t)gridDim.x * 4) {      // a row a wave
    const Pad p = i < a.rows ? a : b;
    const int64_t r = i < a.rows ? i : i - a.rows, width = (p.kbytes + 15) / 16 * 16;
    const char* src = p.src + r * p.ld;
    char* dst = p.dst + r * width;
    for (int64_t c = (threadIdx.x & 63) * 16; c < width; c += 1024) *reinterpret_cast<i32x4*>(dst + c) = chunk_at(src, c, p.kbytes);
  }
}

// dz [rows, ldz] from the saved pre-activations and dy (zeros behind 2n), 8 or 4 columns a thread (16 bytes of dz), and the column sums of a band of rows
// for db (in fp32, before dz is rounded).  dz is rounded to the type, because the matrix cores multiply 16-bit operands; with the 24 bits of the pre-activations the gradients' error in bf16 is 1.4 times that
// of one final rounding (dz as a sum of two values of the type would take twice the products).  In fp16 a |dz| above 65504 is infinite and one below 2^-14 loses bits, as the gradient of a
// pre-activation in fp16 does: loss scaling has to keep it in range.  Bound by its bytes: dy, 3 planes of 16 bits (2 of fp32) and dz's two halves.
template <class T> __global__ __launch_bounds__(256) void k_dz(T* __restrict__ z, float* __restrict__ dbpart, const T* __restrict__ dy, int64_t lddy, const void* __restrict__ saved,
                                                              int rows, int n, int64_t ldz, int act, int band) {
  constexpr int V = 16 / (int)sizeof(T), GROUPS = 32;      // 32 threads side by side, 8 rows at a time
  __shared__ float join[8][GROUPS][2 * V + 1];
  const int x = threadIdx.x % GROUPS, y = threadIdx.x / GROUPS;
  const int64_t c = ((int64_t)blockIdx.x * GROUPS + x) * V, plane = (int64_t)rows * n, left = n - c;
  const int r0 = blockIdx.y * band, r1 = r0 + min(band, rows - r0);
  float sg[V], su[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sg[i] = su[i] = 0.f;
  if (left > 0)
    for (int r = r0 + y; r < r1; r += 8) {
      const int64_t at = (int64_t)r * n + c;
      float d[V], g[V], u[V];
      load_v<V>(d, dy + r * lddy + c, left);
      if constexpr (sizeof(T) == 4) {
        load_v<V>(g, static_cast<const float*>(saved) + at, left);
        load_v<V>(u, static_cast<const float*>(saved) + plane + at, left);
      } else {
        const uint16_t* s = static_cast<const uint16_t*>(saved) + at;
        uint16_t hg[V], hu[V], lo[V];
        if (left >= V) {
          const Any16 a = *reinterpret_cast<const Any16*>(s), b = *reinterpret_cast<const Any16*>(s + plane), l = *reinterpret_cast<const Any16*>(s + 2 * plane);
          __builtin_memcpy(hg, &a, 16); __builtin_memcpy(hu, &b, 16); __builtin_memcpy(lo, &l, 16);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            hg[i] = i < left ? s[i] : 0; hu[i] = i < left ? s[plane + i] : 0; lo[i] = i < left ? s[2 * plane + i] : 0;
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) { g[i] = from24(hg[i], lo[i] >> 8); u[i] = from24(hu[i], lo[i] & 0xffu); }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float a, da;
        act_grad(act, g[i], a, da);
        const float dg = d[i] * u[i] * da, du = d[i] * a;
        sg[i] += i < left ? dg : 0.f; su[i] += i < left ? du : 0.f;
        g[i] = dg; u[i] = du;
      }
      if (z) {
        T* p = z + r * ldz;
        store_v<V>(p + c, g, left);
        store_v<V>(p + n + c, u, left);
        if (left <= V) for (int64_t i = 2 * (int64_t)n; i < ldz; ++i) p[i] = (T)0.f;
      }
    }
  if (!dbpart) return;
#pragma unroll
  for (int i = 0; i < V; ++i) { join[y][x][i] = sg[i]; join[y][x][V + i] = su[i]; }
  __syncthreads();
  for (int id = threadIdx.x; id < GROUPS * 2 * V; id += 256) {
    const int g = id / (2 * V), i = id % (2 * V);
    const int64_t col = ((int64_t)blockIdx.x * GROUPS + g) * V + i % V;
    if (col >= n) continue;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += join[k][g][i];
    dbpart[(int64_t)blockIdx.y * 2 * n + (i / V) * n + col] = s;
  }
}
// ---- host -------------------------------------------------------------------------------------------------------------------------
int esize(int dtype) { return dtype == CAGC_F32 ? 4 : dtype == CAGC_E4M3 ? 1 : 2; }
int64_t up16(int64_t b) { return (b + 15) / 16 * 16; }
int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

struct Plan { int bp, bq, splits; };

// Tile and K split of a product with `cols` columns (of 2 `cols` rows of p when gated), `rows` rows and K of `ksteps` times 128 bytes: the least of an estimate.  A workgroup's stage of 128 bytes takes
// its latency `least`, and n workgroups of a CU take n times `share`, whichever is longer (us, measured with 128 to 4500 rows of 256 to 4096: the estimates are within 15 % of most times); `turn` is what a
// round of workgroups spends outside its stages.  Small tiles share operands less, so they cost more a product, but come before a split of K, whose slabs want a launch of their own to be joined: 1024 x 1024 ->
// 1024 bf16 with tiles of 128 / 64 / 32 rows 12.0 / 9.4 / 8.8 us, of 128 in two pieces of K 19.9; 512 x 4096 -> 4096 43 / 40 / 58 us.
// Up to 64 pieces: with 16, dW of many rows and few columns leaves CUs idle (131072 x 64 -> 128 bf16 103 instead of 79 us with dz, 65536 x 128 -> 128 fp32 106 instead of 82); 128 help one and cost another (67; 65536 x
// 64 -> 64 41 instead of 37).
struct Cost { int bp, bq, slots; double least, share, turn; };
constexpr Cost COSTS_16[] = {{256, 256, 1, 1.05, 1.55, 8.}, {128, 128, 2, .65, .47, 3.}, {128, 64, 3, .45, .30, 2.5}, {128, 32, 4, .36, .23, 2.}};
// fp32: bound by the matrix cores at every tile
constexpr Cost COSTS_32[] = {{256, 256, 1, 8.2, 8.2, 8.}, {128, 128, 2, 2.1, 2.1, 3.}, {128, 64, 3, 1.1, 1.03, 2.5}, {128, 32, 4, .6, .52, 2.}};
Plan plan_of(bool gated, int64_t rows, int64_t cols, int ksteps, int dtype) {
  const int64_t prows = gated ? 2 * cols : cols;
  Plan best = {0, 0, 1};
  double least = 0.;
  for (const Cost& c : dtype == CAGC_F32 ? COSTS_32 : COSTS_16) {
    const int64_t tiles = ((prows + c.bp - 1) / c.bp) * ((rows + c.bq - 1) / c.bq);
    for (int s = 1; s <= (c.bq == 256 ? 1 : 64); ++s) {
      if (s > 1 && (s * 4 > ksteps || tiles * s > 1024)) break;      // at least 512 bytes of K a piece
      const int64_t wgs = tiles * s, n = (wgs + 255) / 256;
      // the largest tile's share falls towards its latency on a chip that is not full
      const double share = c.bq == 256 && n == 1 && dtype != CAGC_F32 ? c.least + (c.share - c.least) * wgs / 256. : n * c.share;
      double t = (double)((ksteps + s - 1) / s) * (share > c.least ? share : c.least) + c.turn * ((n + c.slots - 1) / c.slots);
      if (s > 1) t += 5. + 8e-6 / 5. * s * rows * prows;
      if (best.bp == 0 || t < least) { best = {c.bp, c.bq, s}; least = t; }
    }
  }
  return best;
}

template <class T, class O, bool DP, bool DQ> int launch_product(Product& a, const Plan& p, hipStream_t st, const char* what) {
  const int cols = DP ? p.bp : p.bp / 2;
  a.tiles_p = cdiv(a.np, cols);
  a.tiles_q = cdiv(a.nq, p.bq);
  a.splits = p.splits;
  const dim3 grid((unsigned)(a.tiles_p * a.tiles_q), (unsigned)a.splits);
  if (p.bp == 256) hipLaunchKernelGGL((k_product<T, O, 256, 256, 4, 2, DP, DQ>), grid, dim3(512), 0, st, a);
  else if (p.bq == 128) hipLaunchKernelGGL((k_product<T, O, 128, 128, 2, 2, DP, DQ>), grid, dim3(256), 0, st, a);
  else if (p.bq == 64) hipLaunchKernelGGL((k_product<T, O, 128, 64, 4, 1, DP, DQ>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_product<T, O, 128, 32, 4, 1, DP, DQ>), grid, dim3(256), 0, st, a);
  int rc = check_launch(what);
  if (rc != CAGC_OK || a.splits == 1) return rc;
  const int64_t quads = (int64_t)((a.np + 3) / 4) * a.nq;
  hipLaunchKernelGGL((k_join<O, !DP>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, a);
  return check_launch(what);
}
constexpr int64_t MOST_LD = 7 << 20;      // 256 rows of a tile stay within 32-bit offsets
// What the tiled product's loads want: 16-byte alignment of a matrix's rows and row length, and rows within the reach of a tile's offsets.  Other matrices are copied first (k_pad_rows);
// the kernel for few rows reads any.
bool aligned(const void* p, int64_t ld_bytes, int64_t kbytes) { return ((uintptr_t)p % 16) == 0 && ld_bytes % 16 == 0 && kbytes % 16 == 0 && ld_bytes <= MOST_LD; }

// Rows whose weights are streamed through registers: up to 32; up to 64 where the weights are small (one launch without padding or a join: 64 x 1001 -> 2731 fp16 18 instead of 24 us, 40 x 512 ->
// 512 6 instead of 8; with 134 MB of weights, 64 x 4096 -> 8192 bf16, 46 instead of 30) and K does not leave a few workgroups with long rows (61 x 3480 -> 78 fp32 59 instead of 31).
bool few_rows_do(int64_t rows, int64_t n, int64_t kbytes) { return rows <= 32 || (rows <= 64 && 2 * n * kbytes <= (16 << 20) && kbytes <= 8192); }

struct FwdLayout { bool few; Plan plan; int64_t xpad, wpad, slab, total; int64_t kpad; };
FwdLayout fwd_layout(int64_t rows, int64_t n, int64_t k, bool x_ok, bool w_ok, int dtype) {
  FwdLayout l = {};
  const int64_t kb = k * esize(dtype);
  l.kpad = up16(kb);
  l.few = few_rows_do(rows, n, kb);
  if (l.few) return l;
  l.plan = plan_of(true, rows, n, (int)((l.kpad + 127) / 128), dtype);
  int64_t at = 0;
  if (!x_ok) { l.xpad = at; at += up256(rows * l.kpad); }
  if (!w_ok) { l.wpad = at; at += up256(2 * n * l.kpad); }
  l.slab = at;
  if (l.plan.splits > 1) at += up256(4 * (int64_t)l.plan.splits * rows * 2 * n);
  l.total = at;
  return l;
}

int pad_rows(const Pad* jobs, int count, hipStream_t st, const char* what) {
  if (count == 0) return CAGC_OK;
  const Pad none = {};
  const Pad& second = count > 1 ? jobs[1] : none;
  const int64_t wgs = (jobs[0].rows + second.rows + 3) / 4, most = 1 << 20;
  hipLaunchKernelGGL(k_pad_rows, dim3((unsigned)(wgs < most ? wgs : most)), dim3(256), 0, st, jobs[0], second);
  return check_launch(what);
}

template <class T, class O, int MQ, int C> int launch_few(Product& a, hipStream_t st, const char* what) {
  const int blocks = cdiv(a.np, C);
  // Waves that share K, at least two turns each: mostly eight.  16 columns: four where a CU has more than one workgroup, rows are up to 8 KB and not both short and of a single product.  8 columns: sixteen
  // where rows are 8 KB and more and a CU has at most three workgroups, four where it has eight and rows are up to 8 KB.  With 4 / 8 / 16 waves, us (weights from HBM): 16 columns, 16 x 8192 -> 4096 bf16
  // 43.4 / 33.2 / 33.7, 16 x 1024 -> 8192 bf16 11.3 / 9.9 / 12.1, 32 x 4096 -> 5120 bf16 35.6 / 38.9 / 40.3, 16 x 8192 -> 8192 e4m3 26.5 / 28.6 / 30.9; 8 columns, 1 x 2048 -> 2048 bf16 7.5 / 5.9 / 6.1,
  // 1 x 4096 -> 4096 bf16 14.7 / 14.0 / 13.6, 1 x 4096 -> 8192 fp32 64.5 / 46.3 / 49.1, 1 x 4096 -> 16384 bf16 46.8 / 50.0 / 49.2.  Over 378 sizes (1 to 32 rows, n 512 to 24576, rows of 1 to 16 KB,
  // three types) the rule's choice takes 0.7 % (8 columns 1.5 %) longer than the best of the three in the mean, 7 (15) % at worst; eight everywhere would take 2.4 (2.2) % longer.
  int nw = 8;
  if (C == 16 && blocks > 256 && a.kbytes <= 8192 && (MQ > 1 || a.kbytes > 4096)) nw = 4;
  if (C == 8 && blocks <= 768 && a.kbytes >= 8192) nw = 16;
  if (C == 8 && blocks >= 2048 && a.kbytes <= 8192) nw = 4;
  if (a.kbytes < 256 * nw) nw = 4;
  hipLaunchKernelGGL((k_few_rows<T, O, MQ, C>), dim3(blocks), dim3(nw * 64), (size_t)nw / 2 * MQ * (C / 8) * 64 * sizeof(f32x4), st, a);      // (at most 32 KB)
  return check_launch(what);
}
template <class T, class O> int few_rows(Product& a, hipStream_t st, const char* what) {
  const bool narrow = a.np < 16 * 256 || a.nq <= 4;      // few rows of x: reading them in twice the workgroups costs little (1 x 4096 -> 8192 bf16 28.6 -> 25.3 us; with 16 rows 33.6 -> 35.4)
  if (a.nq <= 16) return narrow ? launch_few<T, O, 1, 8>(a, st, what) : launch_few<T, O, 1, 16>(a, st, what);
  if (a.nq <= 32) return narrow ? launch_few<T, O, 2, 8>(a, st, what) : launch_few<T, O, 2, 16>(a, st, what);
  return narrow ? launch_few<T, O, 4, 8>(a, st, what) : launch_few<T, O, 4, 16>(a, st, what);
}

template <class T, class O> int forward(Product& a, const FwdLayout& l, hipStream_t st, const char* what) {
  return l.few ? few_rows<T, O>(a, st, what) : launch_product<T, O, false, false>(a, l.plan, st, what);
}

bool sizes_ok(int64_t rows, int64_t n, int64_t k, int dtype) {
  return rows >= 0 && n > 0 && k > 0 && rows < (1ll << 31) - 512 && n <= (1 << 26) && k * esize(dtype) <= MOST_LD;
}

// dz's rows [2n] are read along K by the tiles, so they stay within a tile's offsets too; a forward pass that saves for a backward pass is held to it as well
bool dz_ok(int64_t n, int dtype) { return (2 * n + 16) * esize(dtype) <= MOST_LD; }

// rows of a workgroup of k_dz: 8, a row a thread, while that makes few workgroups; 16 (each band writes a row of shares of db); as many more as keep the grid to 65535 of them
int band_of(int64_t rows, int64_t n) {
  int64_t band = rows * n < (1 << 20) ? 8 : 16;
  while (rows > band * 65535) band *= 2;
  return (int)band;
}

struct BwdLayout { int64_t z, wpad, xpad, dbpart, slab, total; int64_t ldz, kpad; Plan dx, dw; };
BwdLayout bwd_layout(int64_t rows, int64_t n, int64_t k, bool x_ok, bool w_ok, int dtype, bool need_dx, bool need_dw, bool need_db) {
  BwdLayout l = {};
  const int e = esize(dtype), v = 16 / e, rk = 128 / e;
  l.ldz = (2 * n + v - 1) / v * v;
  l.kpad = up16(k * e);
  int64_t at = 0, s = 0;
  if (need_dx || need_dw) at += up256(rows * l.ldz * e);
  if (need_dx) {
    l.dx = plan_of(false, rows, k, (int)((2 * n + rk - 1) / rk), dtype);
    if (!w_ok) { l.wpad = at; at += up256(2 * n * l.kpad); }
    if (l.dx.splits > 1) s = 4 * (int64_t)l.dx.splits * rows * k;
  }
  if (need_dw) {
    l.dw = plan_of(false, 2 * n, k, (int)((rows + rk - 1) / rk), dtype);
    if (!x_ok) { l.xpad = at; at += up256(rows * l.kpad); }
    const int64_t t = l.dw.splits > 1 ? 4 * (int64_t)l.dw.splits * 2 * n * k : 0;
    if (t > s) s = t;
  }
  if (need_db) { l.dbpart = at; const int band = band_of(rows, n); at += up256(4 * ((rows + band - 1) / band) * 2 * n); }
  l.slab = at;
  l.total = at + up256(s);
  return l;
}

template <class T> int backward(void* dx, void* dw, void* db, char* ws, const void* dy, const void* saved, const void* x, const void* w, int64_t rows, int64_t n,
                                int64_t k, int64_t ldx, int64_t ldw, int64_t lddy, int dtype, int act, float scale, hipStream_t st, const char* what) {
  const int e = sizeof(T), v = 16 / e;
  const bool x_ok = !dw || aligned(x, ldx * e, k * e), w_ok = !dx || aligned(w, ldw * e, k * e);
  const BwdLayout l = bwd_layout(rows, n, k, x_ok, w_ok, dtype, dx != nullptr, dw != nullptr, db != nullptr);
  T* z = dx || dw ? (T*)(ws + l.z) : nullptr;
  float* part = db ? (float*)(ws + l.dbpart) : nullptr;
  const int band = band_of(rows, n), bands = cdiv(rows, band);
  hipLaunchKernelGGL((k_dz<T>), dim3((unsigned)((n + 32 * v - 1) / (32 * v)), (unsigned)bands), dim3(256), 0, st, z, part, (const T*)dy, lddy, saved, (int)rows, (int)n, l.ldz, act, band);
  int rc = check_launch(what);
  if (rc != CAGC_OK) return rc;
  if (db) {
    hipLaunchKernelGGL((k_column_sums<T>), dim3((unsigned)((2 * n + 15) / 16)), dim3(1024), 0, st, (T*)db, part, bands, (int)(2 * n));
    if ((rc = check_launch(what)) != CAGC_OK) return rc;
  }
  Product a = {};
  a.alpha = scale;
  a.slab = (float*)(ws + l.slab);
  a.ldo = k;
  a.np = (int)k;
  a.q = (const char*)z; a.ldq = l.ldz * e;
  Pad jobs[2];
  int count = 0;
  if (!w_ok) jobs[count++] = Pad{ws + l.wpad, (const char*)w, 2 * n, k * e, ldw * e};
  if (!x_ok) jobs[count++] = Pad{ws + l.xpad, (const char*)x, rows, k * e, ldx * e};
  if ((rc = pad_rows(jobs, count, st, what)) != CAGC_OK) return rc;
  if (dx) {                                  // dz [rows, 2n] along its rows, W [2n, k] down its columns
    a.p = w_ok ? (const char*)w : ws + l.wpad; a.ldp = w_ok ? ldw * e : l.kpad;
    a.nq = (int)rows;
    a.kbytes = (int)(l.ldz * e); a.krows = (int)(2 * n);
    a.out = dx;
    if ((rc = launch_product<T, T, true, false>(a, l.dx, st, what)) != CAGC_OK) return rc;
  }
  if (dw) {                                  // dz and x [rows, k] down their columns
    a.p = x_ok ? (const char*)x : ws + l.xpad; a.ldp = x_ok ? ldx * e : l.kpad;
    a.nq = (int)(2 * n);
    a.kbytes = 0; a.krows = (int)rows;
    a.out = dw;
    if ((rc = launch_product<T, T, true, true>(a, l.dw, st, what)) != CAGC_OK) return rc;
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
  CAGC_REQUIRE(!saved || dz_ok(n, dtype), "%s: n too large for a backward pass (2n values of at most %lld bytes)", what, (long long)MOST_LD);
  if (rows == 0) return CAGC_OK;
  CAGC_REQUIRE(out && x && w, "%s: null pointer", what);
  const int64_t e = esize(dtype), kb = k * e;
  const bool x_ok = aligned(x, ldx * e, kb), w_ok = aligned(w, ldw * e, kb);
  const FwdLayout l = fwd_layout(rows, n, k, x_ok, w_ok, dtype);
  CAGC_REQUIRE(l.total == 0 || ws, "%s: needs %lld bytes of workspace", what, (long long)l.total);
  hipStream_t st = as_stream(stream);
  Product a = {};
  a.p = (const char*)w; a.ldp = ldw * e;
  a.q = (const char*)x; a.ldq = ldx * e;
  a.np = (int)n; a.nq = (int)rows;
  a.kbytes = (int)kb;
  a.out = out; a.ldo = n;
  a.alpha = scale; a.bias = bias; a.sp = w_scale; a.sq = x_scale; a.saved = saved; a.act = act;
  a.splits = 1;
  char* base = (char*)ws;
  int rc;
  if (!l.few) {
    Pad jobs[2];
    int count = 0;
    if (!x_ok) { jobs[count++] = Pad{base + l.xpad, a.q, rows, kb, a.ldq}; a.q = base + l.xpad; a.ldq = l.kpad; }
    if (!w_ok) { jobs[count++] = Pad{base + l.wpad, a.p, 2 * n, kb, a.ldp}; a.p = base + l.wpad; a.ldp = l.kpad; }
    if ((rc = pad_rows(jobs, count, st, what)) != CAGC_OK) return rc;
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

extern "C" int cagc_gated_linear_plan(int* columns, int* tile_rows, int* pieces, int product, int64_t rows, int64_t n, int64_t k, int dtype) {
  const char* what = "cagc_gated_linear_plan";
  CAGC_REQUIRE(columns && tile_rows && pieces, "%s: null pointer", what);
  CAGC_REQUIRE(dtype == CAGC_F32 || dtype == CAGC_F16 || dtype == CAGC_BF16 || (dtype == CAGC_E4M3 && product == 0), "%s: element type %d", what, dtype);
  CAGC_REQUIRE(product >= 0 && product <= 2 && rows > 0 && sizes_ok(rows, n, k, dtype) && (product == 0 || dz_ok(n, dtype)), "%s: bad sizes or product", what);
  Plan p;
  if (product == 0) {
    const FwdLayout l = fwd_layout(rows, n, k, true, true, dtype);
    p = l.few ? Plan{0, 0, 1} : l.plan;
  } else {
    const BwdLayout l = bwd_layout(rows, n, k, true, true, dtype, product == 1, product == 2, false);
    p = product == 1 ? l.dx : l.dw;
  }
  *columns = p.bp; *tile_rows = p.bq; *pieces = p.splits;
  return CAGC_OK;
}

extern "C" int64_t cagc_gated_linear_bwd_workspace(const void* x, const void* w, int64_t rows, int64_t n, int64_t k, int64_t ldx, int64_t ldw, int dtype, int need_dx, int need_dw,
                                                   int need_db) {
  if (!sizes_ok(rows, n, k, dtype)) return 0;
  const int64_t e = esize(dtype);
  return bwd_layout(rows, n, k, aligned(x, ldx * e, k * e), aligned(w, ldw * e, k * e), dtype, need_dx, need_dw, need_db).total;
}

extern "C" int cagc_gated_linear_bwd(void* dx, void* dw, void* db, void* ws, const void* dy, const void* saved, const void* x, const void* w, int64_t rows, int64_t n,
                                     int64_t k, int64_t ldx, int64_t ldw, int64_t lddy, int dtype, int act, float scale, cagc_stream_t stream) {
  const char* what = "cagc_gated_linear_bwd";
  CAGC_REQUIRE(dtype == CAGC_F32 || dtype == CAGC_F16 || dtype == CAGC_BF16, "%s: element type %d", what, dtype);
  CAGC_REQUIRE(sizes_ok(rows, n, k, dtype) && ldx >= k && ldw >= k && lddy >= n, "%s: bad sizes", what);
  CAGC_REQUIRE(dz_ok(n, dtype), "%s: n too large (2n values of at most %lld bytes)", what, (long long)MOST_LD);
  CAGC_REQUIRE(act == CAGC_ACT_SILU || act == CAGC_ACT_GELU, "%s: activation %d", what, act);
  CAGC_REQUIRE(rows > 0, "%s: no rows (the gradients of weight and bias are zero)", what);
  if (!dx && !dw && !db) return CAGC_OK;
  CAGC_REQUIRE(ws && dy && saved && (!dw || x) && (!dx || w), "%s: null pointer", what);
  hipStream_t st = as_stream(stream);
  if (dtype == CAGC_F32) return backward<float>(dx, dw, db, (char*)ws, dy, saved, x, w, rows, n, k, ldx, ldw, lddy, dtype, act, scale, st, what);
  if (dtype == CAGC_F16) return backward<_Float16>(dx, dw, db, (char*)ws, dy, saved, x, w, rows, n, k, ldx, ldw, lddy, dtype, act, scale, st, what);
  return backward<__bf16>(dx, dw, db, (char*)ws, dy, saved, x, w, rows, n, k, ldx, ldw, lddy, dtype, act, scale, st, what);
}
