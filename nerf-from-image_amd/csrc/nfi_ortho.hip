// Orthogonalised updates (include/nfi_learn.h nfi_ortho): X0 = U / max(|U|_F, eps), taken with its smaller side as rows
// (m <= n), then `steps` times
//
//   A = X X^T        Q = a I + b A + c A A        X <- Q X
//
// which maps every singular value s to the odd polynomial a s + b s^3 + c s^5 and leaves the singular vectors; with
// U = G + beta M, M <- beta M + G (or U = M) before, and W <- (1 - decay) W - step X behind.  Per step m^2 n + m^3 + 2 m^2 n
// operations (A and A A are symmetric: half of each product is computed and mirrored).
//
// Small singular values grow by up to `a` each step, and rounding errors with them, so products are near 32-bit ones
// whatever the type of the weights: operands are pairs of halves hi = f16(v 2^s), lo = f16(v 2^s - hi), three
// products hi hi + hi lo + lo hi on the 16-bit matrix cores into 32-bit sums (lo lo is below 2^-22 of the product).  All
// operands are bounded (singular values start at <= 1 and the polynomial is known), so the scales are constants of the
// call; a value keeps 22 bits down to 2^-17 of its bound, and 2^-40 of the bound below (a lo half is subnormal there).  Two of
// 2048 x 2048: 2.4e-6 of the norm off after five steps, the formula in 32-bit products 3.8e-6.  Memory holds 32 hi and 32 lo halves of 32 neighbouring columns together: 128 bytes that are one step of a tile.
//
// Matrices of up to 64 rows that fit into LDS run whole in one workgroup each; the others run as tiles of 128 x 128, all
// matrices of the call in each launch: their grid holds one tile after the other.  Sides are padded to 128, and the padding is
// computed (64 x 576 takes what 128 x 1152 does, 180 us).
//
// Two of 2048 x 2048: A 76 us, Q 82, X' 96 a step (of 3 products: X' at 1080 TF, as fast as a large f16 product of a library;
// A and Q have 272 tiles for 256 compute units, one each, where two hide each other's waits).  A generator's 26 matrices up to
// 512 x 4608: 56 + 12 (A in pieces, joined), 25, 92 us a step, momentum and norm 61 (316 MB at 5.2 TB/s), the start 80.
#include <algorithm>
#include <cmath>

#include "nfi_mm.h"

namespace nfi {
namespace learn {

constexpr int ITEMS = 32;            // matrices (or runs of equal ones) of a launch
constexpr int NORM_CHUNK = 16384;    // elements of a partial sum of squares

struct Item {
  const void* g;
  float* mom;
  void* w;
  _Float16 *x, *y, *a, *q;    // workspace: X and the next X [mp][2 np], A and Q [mp][2 mp]
  double* sums;               // [count][chunks]
  float* part;                // partial tiles of A or Q where the contracted index is split
  float scale;                // the step's factor of this matrix
  int rows, cols, count, m, n, mp, np, chunks, split_a, split_q;
};

struct Args {
  int items, g_type, w_type, update, nesterov, last;
  float beta, keep, step, a, b, c, eps;   // keep = 1 - decay
  float up_x, up_a, up_q;                 // powers of two
};

// The launch's arguments: a kernel takes room for 1, 8 or 32 items (the 4 KB of 32 cost 10 us of a launch)
template <int N>
struct Table : Args {
  int first[N];   // the launch's first unit of each item (behind the last: beyond any)
  Item item[N];
};
static_assert(sizeof(Table<ITEMS>) <= 4096, "kernel arguments");

typedef _Float16 h4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float typed_at(const void* p, int type, int64_t i) {
  return type == NFI_F32 ? ((const float*)p)[i] : type == NFI_BF16 ? (float)((const bf16_t*)p)[i] : (float)((const f16_t*)p)[i];
}

// Work unit `id` of a launch: the item, the matrix of its run, and the unit within it (per(item) units each).  (The first units
// lie together and come with one or two loads; a walk over the items would wait for each.)
template <int N, class F>
__device__ __forceinline__ int locate(const Table<N>& p, int id, int& matrix, int& unit, F per) {
  int it = 0;
#pragma unroll
  for (int k = 1; k < N; ++k) it += id >= p.first[k];
  id -= p.first[it];
  const int u = per(p.item[it]);
  matrix = id / u;
  unit = id - matrix * u;
  return it;
}

// ---- momentum and norm -------------------------------------------------------------------------------------------

// M <- beta M + G, and the squares' sum of U over a chunk (64-bit: squares of bf16 values pass the 32-bit range)
template <int N>
__global__ void __launch_bounds__(256) ortho_norm(const Table<N> p) {
  __shared__ double red[256];
  int matrix, chunk;
  const int i = locate(p, blockIdx.x, matrix, chunk, [](const Item& t) { return t.chunks; });
  const Item& t = p.item[i];
  const int64_t size = (int64_t)t.rows * t.cols, base = matrix * size;
  const int64_t e0 = (int64_t)chunk * NORM_CHUNK, e1 = min(e0 + NORM_CHUNK, size);
  double s = 0.;
  for (int64_t e = e0 + threadIdx.x * 4; e < e1; e += 1024) {
    float g[4], m[4];
    if (e + 4 <= e1) {
      load_typed<4>(t.g, p.g_type, base + e, g);
      if (t.mom) load_piece<float, 4>(t.mom + base + e, m);
    } else {
      for (int j = 0; j < 4; ++j) {
        g[j] = e + j < e1 ? typed_at(t.g, p.g_type, base + e + j) : 0.f;
        m[j] = t.mom && e + j < e1 ? t.mom[base + e + j] : 0.f;
      }
    }
    if (t.mom) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] = fmaf(p.beta, m[j], g[j]);
        g[j] = p.nesterov ? fmaf(p.beta, m[j], g[j]) : m[j];
      }
      if (e + 4 <= e1) store_piece<float, 4>(t.mom + base + e, m);
      else
        for (int j = 0; e + j < e1; ++j) t.mom[base + e + j] = m[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fma((double)g[j], (double)g[j], s);
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int d = 128; d > 0; d >>= 1) {
    if (threadIdx.x < d) red[threadIdx.x] += red[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x == 0) t.sums[(int64_t)matrix * t.chunks + chunk] = red[0];
}

__device__ __forceinline__ float update_at(const Args& p, const Item& t, int64_t at) {
  const float g = typed_at(t.g, p.g_type, at);
  if (!t.mom) return g;
  const float m = t.mom[at];
  return p.nesterov ? fmaf(p.beta, m, g) : m;
}

// 1 / max(norm, eps) of the sums of a matrix, the same in every thread (64-bit: that of a large 32-bit norm is subnormal)
__device__ __forceinline__ double inverse_norm(const double* sums, int chunks, float eps, double* red) {
  double s = 0.;
  for (int k = threadIdx.x; k < chunks; k += blockDim.x) s += sums[k];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int d = blockDim.x / 2; d > 0; d >>= 1) {
    if ((int)threadIdx.x < d) red[threadIdx.x] += red[threadIdx.x + d];
    __syncthreads();
  }
  const double n = sqrt(red[0]);
  __syncthreads();
  return 1. / (n < (double)eps ? (double)eps : n);   // (a NaN stays one)
}

__device__ __forceinline__ void split4(const float (&v)[4], h4v& hi, h4v& lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    hi[j] = (_Float16)v[j];
    lo[j] = (_Float16)(v[j] - (float)hi[j]);
  }
}

// place of column c's hi half in a row; its lo half is 32 further
__device__ __forceinline__ int64_t half_at(int c) { return ((int64_t)(c >> 5) << 6) + (c & 31); }

// X0 in halves, 64 x 64 at a time, turned where the matrix is taller than wide; zeros in the padding
template <int N>
__global__ void __launch_bounds__(256) ortho_start(const Table<N> p) {
  __shared__ float tile[64][65];
  __shared__ double red[256];
  int matrix, unit;
  const int i = locate(p, blockIdx.x, matrix, unit, [](const Item& t) { return t.mp / 64 * (t.np / 64); });
  const Item& t = p.item[i];
  const double inv = inverse_norm(t.sums + (int64_t)matrix * t.chunks, t.chunks, p.eps, red) * p.up_x;
  const int r0 = unit / (t.np / 64) * 64, c0 = unit % (t.np / 64) * 64;
  const int64_t base = (int64_t)matrix * t.rows * t.cols;
  const bool turned = t.rows > t.cols;
  const int a = threadIdx.x & 63, b = threadIdx.x >> 6;
  for (int k = b; k < 64; k += 4) {
    // (a runs along memory)
    const int r = turned ? r0 + a : r0 + k, c = turned ? c0 + k : c0 + a;
    float v = 0.f;
    if (r < t.m && c < t.n) v = (float)(update_at(p, t, base + (turned ? (int64_t)c * t.cols + r : (int64_t)r * t.cols + c)) * inv);
    if (turned) tile[a][k] = v;
    else tile[k][a] = v;
  }
  __syncthreads();
  _Float16* x = t.x + (int64_t)matrix * t.mp * 2 * t.np;
  for (int k = threadIdx.x; k < 1024; k += 256) {
    const int r = k >> 4, c = (k & 15) * 4;
    const float v[4] = {tile[r][c], tile[r][c + 1], tile[r][c + 2], tile[r][c + 3]};
    h4v hi, lo;
    split4(v, hi, lo);
    _Float16* d = x + (int64_t)(r0 + r) * 2 * t.np + half_at(c0 + c);
    *reinterpret_cast<h4v*>(d) = hi;
    *reinterpret_cast<h4v*>(d + 32) = lo;
  }
}

// ---- products of pairs of halves -------------------------------------------------------------------------------------

// An operand whose contracted index runs over rows: LDS [32 rows][128 columns hi and lo: 512 bytes]
struct PairSlab {
  unsigned off[4];
  static __device__ __forceinline__ int lds_row(int j) { return ((threadIdx.x >> 6) * 4 + j) * 2 + (lane_id() >> 5); }
  __device__ __forceinline__ void init(unsigned ld) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = lds_row(j);
      off[j] = row * ld + (((lane_id() & 31) ^ (2 * (row & 7))) << 4);
    }
  }
  __device__ __forceinline__ void issue(const void* base, unsigned char* lds, bool in) const {
    const __amdgpu_buffer_rsrc_t r = descriptor(base);
    unsigned char* dst = lds + (threadIdx.x >> 6) * 4096;
#pragma unroll
    for (int j = 0; j < 4; ++j) load_to_lds(r, dst + j * 1024, in ? off[j] : NOWHERE);
  }
};

template <int N>
__device__ __forceinline__ void read_pair_slab(const unsigned char* lds, int line0, int plane, u4v (&f)[N]) {
  const int i = lane_id() & 15, g = lane_id() >> 4, r0 = 8 * g + (i >> 2), half = (i & 1) * 8;
#pragma unroll
  for (int x = 0; x < N; ++x) {
    const int c = line0 + 16 * x, piece = ((c >> 5) << 3) + ((c & 31) >> 3) + 4 * plane + ((i & 3) >> 1);
    u2v v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = r0 + 4 * h;
      const unsigned char* q = lds + row * 512 + ((piece ^ (2 * (row & 7))) << 4) + half;
      v[h] = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)q));
    }
    f[x] = u4v{v[0][0], v[0][1], v[1][0], v[1][1]};
  }
}

// acc (a's lines by lane, b's by register) of a 128 x 128 tile over `steps` steps of 32; everything inside the padding.
// a: lines; b: lines, or (SLAB) rows of the contracted index; SWAP: the roles of lane and register exchanged.  Two stages, loads
// two steps ahead (tile_product in nfi_mm.h).
template <bool SLAB, bool SWAP>
__device__ __forceinline__ void pair_product(const _Float16* a, unsigned lda, const _Float16* b, unsigned ldb, int steps, unsigned char* s0,
                                             unsigned char* s1, f4v (&acc)[4][4]) {
  TileLoad<_Float16, false, TILE> la, lb;
  PairSlab sb;
  la.init(TILE, lda);
  if (SLAB) sb.init(ldb);
  else lb.init(TILE, ldb);
  const int64_t step_b = SLAB ? (int64_t)32 * ldb : STEP_BYTES;
  const int wave = threadIdx.x >> 6, line_a = (wave & 1) * 64, line_b = (wave >> 1) * 64;
  const unsigned char *pa = (const unsigned char*)a, *pb = (const unsigned char*)b;
  auto issue = [&](int t, unsigned char* dst) {
    const bool in = t < steps;   // (a step behind the last reads nothing: every step waits for the same number of loads)
    la.issue(pa + (int64_t)t * STEP_BYTES, dst, in ? STEP_BYTES : 0);
    if (SLAB) sb.issue(pb + t * step_b, dst + TILE_BYTES, in);
    else lb.issue(pb + t * step_b, dst + TILE_BYTES, in ? STEP_BYTES : 0);
    __builtin_amdgcn_sched_barrier(0);   // the waits count on this order of the steps' loads
  };
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) acc[x][y] = f4v{0.f, 0.f, 0.f, 0.f};
  auto step = [&](int t, unsigned char* cur) {
    wait_loads<8>();
    bare_barrier();
    u4v fa[2][4], fb[2][4];
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      read_fragments<_Float16, false, TILE, 4>(cur, line_a, plane, fa[plane]);
      if (SLAB) read_pair_slab<4>(cur + TILE_BYTES, line_b, plane, fb[plane]);
      else read_fragments<_Float16, false, TILE, 4>(cur + TILE_BYTES, line_b, plane, fb[plane]);
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): this wave has read the step
    bare_barrier();
    issue(t + 2, cur);
#pragma unroll
    for (int pair = 0; pair < 3; ++pair)   // lo hi, hi lo, hi hi: the small ones first
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const u4v va = fa[pair == 0][x], vb = fb[pair == 1][y];
          acc[x][y] = SWAP ? product<_Float16>(va, vb, acc[x][y]) : product<_Float16>(vb, va, acc[x][y]);
        }
  };
  issue(0, s0);
  issue(1, s1);
  int t = 0;
  for (; t + 2 <= steps; t += 2) {
    step(t, s0);
    step(t + 1, s1);
  }
  if (t < steps) step(t, s0);
  wait_loads<0>();
  bare_barrier();   // the stages are free: no wave reads, and no load is on its way
}

// a wave's 64 x 64 part of a tile in halves to rows of `ld` halves from d, turned in LDS on the way (store_part in nfi_mm.h): 256
// bytes of a row at a time in place of 32 (X' of a generator's 26 matrices up to 512 x 4608: 108 -> 92 us)
__device__ __forceinline__ void store_pairs(const f4v (&acc)[4][4], float scale, unsigned char* lds, _Float16* d, int64_t ld) {
  const int l = lane_id(), i = l & 15, g = l >> 4;
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float v[4] = {acc[x][y][0] * scale, acc[x][y][1] * scale, acc[x][y][2] * scale, acc[x][y][3] * scale};
      h4v hi, lo;
      split4(v, hi, lo);
      const int row = 16 * x + i, col = 16 * y + 4 * g, piece = half_at(col) >> 3;   // of 8 halves; lo: 4 pieces on
      unsigned char* q = lds + row * 256 + (col & 4) * 2;
      lds_st_fenced((h4v*)(q + ((piece ^ i) << 4)), hi);
      lds_st_fenced((h4v*)(q + (((piece + 4) ^ i) << 4)), lo);
    }
  asm volatile("" ::: "memory");
#pragma unroll
  for (int j0 = 0; j0 < 16; j0 += 8) {
    u4v v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int row = 4 * (j0 + j) + g;
      v[j] = *reinterpret_cast<const u4v*>(lds + row * 256 + ((i ^ (row & 15)) << 4));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) *reinterpret_cast<u4v*>(d + (4 * (j0 + j) + g) * ld + 8 * i) = v[j];
  }
}

// a wave's 64 x 64 part, turned
__device__ __forceinline__ void turn_part(f4v (&v)[4][4], unsigned char* lds) {
  const int i = lane_id() & 15, g = lane_id() >> 4;
  float* f = (float*)lds;
  auto at = [](int row, int col) { return row * 64 + (col ^ (((row >> 2) & 3) << 4) ^ ((row & 3) << 2)); };
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) lds_st_fenced(reinterpret_cast<f4v*>(f + at(16 * x + i, 16 * y + 4 * g)), v[x][y]);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[x][y][r] = f[at(16 * y + 4 * g + r, 16 * x + i)];
  asm volatile("" ::: "memory");
}

// a 128 x 128 tile of a symmetric matrix in halves to (r0, c0), and mirrored to (c0, r0) off the diagonal
__device__ __forceinline__ void store_symmetric(_Float16* d, int ld, int r0, int c0, f4v (&v)[4][4], unsigned char* s0, unsigned char* s1) {
  typedef Share<TILE, TILE> S;
  unsigned char* room = S::room(s0, s1);
  r0 += S::line_a();
  c0 += S::line_b();
  store_pairs(v, 1.f, room, d + (int64_t)r0 * ld + half_at(c0), ld);
  if (r0 / TILE == c0 / TILE) return;
  turn_part(v, room);
  store_pairs(v, 1.f, room, d + (int64_t)c0 * ld + half_at(r0), ld);
}

__device__ __forceinline__ void triangle(int unit, int& ti, int& tj) {
  ti = 0;
  while (unit >= ti + 1) {
    unit -= ti + 1;
    ++ti;
  }
  tj = unit;
}

__device__ __forceinline__ int lower_tiles(const Item& t) { const int k = t.mp / TILE; return k * (k + 1) / 2; }

// The tile's sum scaled, or Q's other terms added, and stored
template <bool SQUARE>
__device__ __forceinline__ void finish_tile(const Args& p, const Item& t, int matrix, int ti, int tj, f4v (&acc)[4][4], unsigned char* s0,
                                            unsigned char* s1) {
  const int wave = threadIdx.x >> 6, i = lane_id() & 15, g = lane_id() >> 4;
  const int r0 = ti * TILE, c0 = tj * TILE;
  if constexpr (!SQUARE) {
    const float s = p.up_a / (p.up_x * p.up_x);
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) acc[x][y] *= s;
  } else {
    const float s = p.c * p.up_q / (p.up_a * p.up_a), sb = p.b * p.up_q / p.up_a, sa = p.a * p.up_q;
    const _Float16* src = t.a + (int64_t)matrix * t.mp * 2 * t.mp;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int row = r0 + (wave & 1) * 64 + 16 * x + i;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int col = c0 + (wave >> 1) * 64 + 16 * y + 4 * g;
        const _Float16* q = src + (int64_t)row * 2 * t.mp + half_at(col);
        const h4v hi = *reinterpret_cast<const h4v*>(q), lo = *reinterpret_cast<const h4v*>(q + 32);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float a = (float)hi[r] + (float)lo[r];
          acc[x][y][r] = fmaf(s, acc[x][y][r], fmaf(sb, a, row == col + r ? sa : 0.f));
        }
      }
    }
  }
  store_symmetric((SQUARE ? t.q : t.a) + (int64_t)matrix * t.mp * 2 * t.mp, 2 * t.mp, r0, c0, acc, s0, s1);
}

// A = X X^T (SQUARE false) or Q = a I + b A + c A A (SQUARE true), the tiles on and below the diagonal, in `split` pieces of the
// contracted index each
template <bool SQUARE, int N>
__global__ void __launch_bounds__(256, 2) ortho_gram(const Table<N> p) {
  __shared__ __attribute__((aligned(16))) unsigned char s0[2 * TILE_BYTES], s1[2 * TILE_BYTES];
  int matrix, unit, ti, tj;
  const int it = locate(p, xcd_order(blockIdx.x, gridDim.x), matrix, unit, [](const Item& t) { return lower_tiles(t) * (SQUARE ? t.split_q : t.split_a); });
  const Item& t = p.item[it];
  const int split = SQUARE ? t.split_q : t.split_a, tile = unit / split, piece = unit - tile * split;
  triangle(tile, ti, tj);
  const int k = SQUARE ? t.mp : t.np, steps = k / 32, k0 = steps * piece / split, k1 = steps * (piece + 1) / split;
  const _Float16* src = (SQUARE ? t.a : t.x) + (int64_t)matrix * t.mp * 2 * k + (int64_t)k0 * 64;
  const unsigned ld = 4u * k;
  f4v acc[4][4];
  pair_product<false, false>(src + (int64_t)ti * TILE * 2 * k, ld, src + (int64_t)tj * TILE * 2 * k, ld, k1 - k0, s0, s1, acc);
  if (split == 1) {
    finish_tile<SQUARE>(p, t, matrix, ti, tj, acc, s0, s1);
    return;
  }
  f4v* part = (f4v*)(t.part + (((int64_t)matrix * lower_tiles(t) + tile) * split + piece) * (TILE * TILE)) + threadIdx.x;
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) part[(4 * x + y) * 256] = acc[x][y];
}

// the pieces of a tile summed in their order
template <bool SQUARE, int N>
__global__ void __launch_bounds__(256, 2) ortho_join(const Table<N> p) {
  __shared__ __attribute__((aligned(16))) unsigned char s0[2 * TILE_BYTES], s1[2 * TILE_BYTES];
  int matrix, tile, ti, tj;
  const int it = locate(p, blockIdx.x, matrix, tile, [](const Item& t) { return (SQUARE ? t.split_q : t.split_a) > 1 ? lower_tiles(t) : 0; });
  const Item& t = p.item[it];
  const int split = SQUARE ? t.split_q : t.split_a;
  triangle(tile, ti, tj);
  const f4v* part = (const f4v*)(t.part + ((int64_t)matrix * lower_tiles(t) + tile) * split * (TILE * TILE)) + threadIdx.x;
  f4v acc[4][4];
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) acc[x][y] = part[(4 * x + y) * 256];
  for (int q = 1; q < split; ++q) {
    part += TILE * TILE / 4;
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) acc[x][y] += part[(4 * x + y) * 256];
  }
  finish_tile<SQUARE>(p, t, matrix, ti, tj, acc, s0, s1);
}

// X' = Q X, or with `last` the weights' step (or the result)
__device__ __forceinline__ void put_update(const Args& p, const Item& t, int64_t at, const f4v& acc, float s, int count) {
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = acc[r] * s;
  if (p.update) {
    const float step = p.step * t.scale;
    if (p.w_type == NFI_F32 && count == 4) {
      float w[4];
      load_piece<float, 4>((const float*)t.w + at, w);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = fmaf(p.keep, w[r], -step * v[r]);
    } else
      for (int r = 0; r < count; ++r) v[r] = fmaf(p.keep, typed_at(t.w, p.w_type, at + r), -step * v[r]);
  }
  if (p.w_type == NFI_F32) {
    if (count == 4) store_piece<float, 4>((float*)t.w + at, v);
    else
      for (int r = 0; r < count; ++r) ((float*)t.w)[at + r] = v[r];
  } else {
    for (int r = 0; r < count; ++r) store_typed(t.w, p.w_type, at + r, v[r]);
  }
}

template <int N>
__global__ void __launch_bounds__(256, 2) ortho_apply(const Table<N> p) {
  __shared__ __attribute__((aligned(16))) unsigned char s0[2 * TILE_BYTES], s1[2 * TILE_BYTES];
  int matrix, unit;
  const int it = locate(p, xcd_order(blockIdx.x, gridDim.x), matrix, unit, [](const Item& t) { return t.mp / TILE * (t.np / TILE); });
  const Item& t = p.item[it];
  const int tr = unit % (t.mp / TILE), tc = unit / (t.mp / TILE);   // the tiles of a block of X's columns follow each other
  const int r0 = tr * TILE, c0 = tc * TILE;
  const _Float16* q = t.q + (int64_t)matrix * t.mp * 2 * t.mp + (int64_t)r0 * 2 * t.mp;
  const _Float16* x = t.x + (int64_t)matrix * t.mp * 2 * t.np + half_at(c0);
  const int wave = threadIdx.x >> 6, i = lane_id() & 15, g = lane_id() >> 4;
  const int la = (wave & 1) * 64, lb = (wave >> 1) * 64;
  const float s = 1.f / (p.up_q * p.up_x), down = 1.f / p.up_q;
  const int64_t base = (int64_t)matrix * t.rows * t.cols;
  f4v acc[4][4];
  if (p.last && t.rows > t.cols) {   // (uniform) the turned matrix: a lane holds neighbours along X's rows
    pair_product<true, true>(q, 4u * t.mp, x, 4u * t.np, t.mp / 32, s0, s1, acc);
#pragma unroll
    for (int xx = 0; xx < 4; ++xx)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int row = r0 + la + 16 * xx + 4 * g, col = c0 + lb + 16 * y + i;
        if (row < t.m && col < t.n) put_update(p, t, base + (int64_t)col * t.cols + row, acc[xx][y], s, min(4, t.m - row));
      }
    return;
  }
  pair_product<true, false>(q, 4u * t.mp, x, 4u * t.np, t.mp / 32, s0, s1, acc);
  if (p.last) {
#pragma unroll
    for (int xx = 0; xx < 4; ++xx)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int row = r0 + la + 16 * xx + i, col = c0 + lb + 16 * y + 4 * g;
        if (row < t.m && col < t.n) put_update(p, t, base + (int64_t)row * t.cols + col, acc[xx][y], s, min(4, t.n - col));
      }
    return;
  }
  store_pairs(acc, down, Share<TILE, TILE>::room(s0, s1), t.y + ((int64_t)matrix * t.mp + r0 + la) * 2 * t.np + half_at(c0 + lb), 2 * t.np);
}

// ---- small matrices ----------------------------------------------------------------------------------------------------

constexpr int SMALL_WAVES = 16;
constexpr int SMALL_THREADS = 64 * SMALL_WAVES;

// g's value at `at` through `type`, 0 where at < 0 (the load is made all the same: loads in a row wait for each other's branches)
template <class T>
__device__ __forceinline__ float value_or_zero(const void* p, int64_t base, int at) {
  const float v = (float)((const T*)p)[base + (at < 0 ? 0 : at)];
  return at < 0 ? 0.f : v;
}

// Up to 16 rows: the waves hold X in registers, in 32 bits, as v_mfma_f32_16x16x4_f32 takes it for Q X: block b of wave w is the
// 16 columns from 16 (w + 16 b), lane (i, g) = (l & 15, l >> 4) holding rows 4 g .. + 3 of column i, which is also how the product
// leaves them.  For A the blocks are turned through LDS of the wave's own; its part of A is the only thing that the waves
// exchange (one barrier a step): each sums all parts in their order and has A, and by symmetry A A and Q, as an operand.
// (32-bit products, not pairs of halves: with few rows the pairs' errors, 2^-23 of A and Q each step, do not average out.)
constexpr int TURN = 16 * 20;   // floats of a turned block (rows of 20: those of one access lie in different banks)
constexpr int ROWS16_BYTES = 2 * SMALL_WAVES * 1024 + SMALL_WAVES * 2 * TURN * 4;

template <int B>
__device__ __forceinline__ void run_rows16(const Args& p, const Item& t, int matrix, int steps, unsigned char* lds, double* red) {
  constexpr int TURNS = B < 2 ? B : 2;
  float* parts = (float*)lds;                              // [2][waves][256]
  const int64_t base = (int64_t)matrix * t.rows * t.cols;
  const bool turned = t.rows > t.cols;
  const int wave = threadIdx.x >> 6, i = lane_id() & 15, g = lane_id() >> 4;
  float* turn = parts + 2 * SMALL_WAVES * 256 + wave * 2 * TURN;   // [TURNS][16][20], this wave's own
  auto place = [&](int b, int r) {   // of X's row 4 g + r, column i of block b; -1 outside
    const int row = 4 * g + r, col = 16 * (wave + SMALL_WAVES * b) + i;
    return row < t.m && col < t.n ? (turned ? col * t.cols + row : row * t.cols + col) : -1;
  };
  f4v x[B];
  auto fetch = [&](auto type, const void* from, f4v (&to)[B]) {
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) to[b][r] = value_or_zero<decltype(type)>(from, base, place(b, r));
  };
  auto fetch_typed = [&](int type, const void* from, f4v (&to)[B]) {
    if (type == NFI_F32) fetch(float(), from, to);
    else if (type == NFI_BF16) fetch(bf16_t(), from, to);
    else fetch(f16_t(), from, to);
  };
  fetch_typed(p.g_type, t.g, x);
  if (t.mom) {
    f4v m[B];
    fetch(float(), t.mom, m);
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = fmaf(p.beta, m[b][r], x[b][r]);
        x[b][r] = p.nesterov ? fmaf(p.beta, v, x[b][r]) : v;
        const int at = place(b, r);
        if (at >= 0) t.mom[base + at] = v;
      }
  }
  double s = 0.;
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) s = fma((double)x[b][r], (double)x[b][r], s);
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane_id() == 0) lds_st_fenced(red + wave, s);
  __syncthreads();
  s = 0.;
#pragma unroll
  for (int w = 0; w < SMALL_WAVES; ++w) s += red[w];
  const double norm = sqrt(s), inv = 1. / (norm < (double)p.eps ? (double)p.eps : norm);   // (a NaN stays one)
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) x[b][r] = (float)(x[b][r] * inv);
  const int used = min(SMALL_WAVES, (t.n + 15) / 16);   // waves that hold a column
  for (int step = 0; step < steps; ++step) {
    float* part = parts + (step & 1) * SMALL_WAVES * 256;
    if (wave < used) {
      f4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b0 = 0; b0 < B; b0 += TURNS) {
#pragma unroll
        for (int b = 0; b < TURNS; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) lds_st_fenced(turn + b * TURN + (4 * g + r) * 20 + i, x[b0 + b][r]);
#pragma unroll
        for (int b = 0; b < TURNS; ++b) {
          const u4v f = *reinterpret_cast<const u4v*>(turn + b * TURN + i * 20 + 4 * g);
          acc = product<float>(f, f, acc);
        }
      }
      // lane (i, g): rows 4 g + r, column i, and as well row i, columns 4 g + r
      lds_st_fenced(reinterpret_cast<f4v*>(part + wave * 256 + 16 * i + 4 * g), acc);
    }
    __syncthreads();
    if (wave < used) {
      f4v a = {0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < used; ++w) a += *reinterpret_cast<const f4v*>(part + w * 256 + 16 * i + 4 * g);
      const u4v af = __builtin_bit_cast(u4v, a);
      const f4v aa = product<float>(af, af, f4v{0.f, 0.f, 0.f, 0.f});
      f4v q;
#pragma unroll
      for (int r = 0; r < 4; ++r) q[r] = fmaf(p.c, aa[r], fmaf(p.b, a[r], i == 4 * g + r ? p.a : 0.f));
#pragma unroll
      for (int b = 0; b < B; ++b) x[b] = product<float>(__builtin_bit_cast(u4v, q), __builtin_bit_cast(u4v, x[b]), f4v{0.f, 0.f, 0.f, 0.f});
    }
  }
  const float step = p.step * t.scale;
  if (p.update) {
    f4v w[B];
    fetch_typed(p.w_type, t.w, w);
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[b][r] = fmaf(p.keep, w[b][r], -step * x[b][r]);
  }
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = place(b, r);
      if (at >= 0) store_typed(t.w, p.w_type, base + at, x[b][r]);
    }
}

// More rows: a workgroup of 16 waves holds X [16 nb][n], A and Q [m][m] in LDS, each as a plane of hi and one of lo halves, and runs
// every step there.  m16 = 16 nb rows are held; A and Q have rows and columns up to the next multiple of 32 (the contracted
// length of a product), zeros behind.  Rows are padded by 8 halves, so that those of one read lie in different banks.  Bound
// by the latency of a step's phases (A's pieces, A, Q, X), not by the products: 64 x 64 takes 18 products of 16 x 16 x 32 on
// the longest path.

struct SmallShape {
  int nb, m16, m32, n32, ldx, lda;   // leading dimensions in halves
  __host__ __device__ SmallShape(int m, int n) {
    nb = (m + 15) / 16;
    m16 = 16 * nb;
    m32 = (m + 31) / 32 * 32;
    n32 = (n + 31) / 32 * 32;
    ldx = n32 + 8;
    lda = m32 + 8;
  }
  // pieces of A (32 bits), X, A, Q in two planes each, 16 zeros
  __host__ __device__ int bytes() const { return SMALL_WAVES * 1024 + 4 * m16 * ldx + 2 * 4 * m32 * lda + 32; }
};

// acc += first second^T over 32 contracted values of pairs: registers hold first's lines 4 g + r, lanes second's line i
__device__ __forceinline__ f4v pair_products(const u4v (&first)[2], const u4v (&second)[2], f4v acc) {
  acc = product<_Float16>(first[1], second[0], acc);
  acc = product<_Float16>(first[0], second[1], acc);
  return product<_Float16>(first[0], second[0], acc);
}
__device__ __forceinline__ void store_pair4(_Float16* hi, _Float16* lo, int at, const float (&v)[4]) {
  h4v h, l;
  split4(v, h, l);
  lds_st_fenced(reinterpret_cast<h4v*>(hi + at), h);
  lds_st_fenced(reinterpret_cast<h4v*>(lo + at), l);
}

template <int NB>
__device__ __forceinline__ void run_lds(const Args& p, const Item& t, int matrix, int steps, unsigned char* lds, double* red) {
  const SmallShape d(t.m, t.n);
  float* P = (float*)lds;
  _Float16 *Xh = (_Float16*)(lds + SMALL_WAVES * 1024), *Xl = Xh + d.m16 * d.ldx;
  _Float16 *Ah = Xl + d.m16 * d.ldx, *Al = Ah + d.m32 * d.lda, *Qh = Al + d.m32 * d.lda, *Ql = Qh + d.m32 * d.lda;
  _Float16* zeros = Ql + d.m32 * d.lda;
  const int size = t.rows * t.cols;
  const int64_t base = (int64_t)matrix * size;
  const bool turned = t.rows > t.cols;
  const int tid = threadIdx.x, wave = tid >> 6, l = lane_id(), i = l & 15, g = l >> 4;
  const int words = (d.bytes() - SMALL_WAVES * 1024) / 16;
  for (int k = tid; k < words; k += SMALL_THREADS) lds_st_fenced((u4v*)Xh + k, u4v{0, 0, 0, 0});
  // the update's square sum (the momentum is updated by the way) ...
  double s = 0.;
  for (int e = tid * 4; e < size; e += SMALL_THREADS * 4) {
    float v[4], m[4];
    const int have = min(4, size - e);
    if (have == 4) {
      load_typed<4>(t.g, p.g_type, base + e, v);
      if (t.mom) load_piece<float, 4>(t.mom + base + e, m);
    } else {
      for (int j = 0; j < 4; ++j) {
        v[j] = j < have ? typed_at(t.g, p.g_type, base + e + j) : 0.f;
        m[j] = t.mom && j < have ? t.mom[base + e + j] : 0.f;
      }
    }
    if (t.mom) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] = fmaf(p.beta, m[j], v[j]);
        v[j] = p.nesterov ? fmaf(p.beta, m[j], v[j]) : m[j];
      }
      if (have == 4) store_piece<float, 4>(t.mom + base + e, m);
      else
        for (int j = 0; j < have; ++j) t.mom[base + e + j] = m[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fma((double)v[j], (double)v[j], s);
  }
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (l == 0) lds_st_fenced(red + wave, s);
  __syncthreads();
  s = 0.;
#pragma unroll
  for (int w = 0; w < SMALL_WAVES; ++w) s += red[w];
  const double norm = sqrt(s);
  const double inv = (double)p.up_x / (norm < (double)p.eps ? (double)p.eps : norm);   // (a NaN stays one)
  // ... and X0 (its own loads again, from the cache: each thread reads what it read and wrote)
  for (int e = tid * 4; e < size; e += SMALL_THREADS * 4) {
    const int have = min(4, size - e);
    int r = e / t.cols, c = e - r * t.cols;
    for (int j = 0; j < have; ++j) {
      const float v = (float)(update_at(p, t, base + e + j) * inv);
      const _Float16 h = (_Float16)v;
      const int at = turned ? c * d.ldx + r : r * d.ldx + c;
      Xh[at] = h;
      Xl[at] = (_Float16)(v - (float)h);
      if (++c == t.cols) c = 0, ++r;
    }
  }
  const float to_a = p.up_a / (p.up_x * p.up_x), to_x = 1.f / p.up_q;
  const float qs = p.c * p.up_q / (p.up_a * p.up_a), qb = p.b * p.up_q / p.up_a, qa = p.a * p.up_q;
  // each wave's place in a step's phases: a block of A on or below the diagonal (in ks pieces of X's columns where the blocks
  // are few), a block of Q, and blocks of X
  constexpr int LOWER = NB * (NB + 1) / 2, KS = SMALL_WAVES / LOWER, DEEP_M = (NB + 1) / 2;
  const int deep = d.n32 / 32, cbs = d.n32 / 16, plane_x = d.m16 * d.ldx, plane_a = d.m32 * d.lda;
  int bi, bj;
  triangle(wave / KS, bi, bj);
  const bool has_a = wave < LOWER * KS, has_q = wave < NB * NB;
  const int k0 = deep * (wave % KS) / KS, k1 = deep * (wave % KS + 1) / KS;
  const _Float16 *xa = Xh + (bi * 16 + i) * d.ldx + 8 * g, *xb = Xh + (bj * 16 + i) * d.ldx + 8 * g;
  _Float16 *a_to = Ah + (bi * 16 + i) * d.lda + bj * 16 + 4 * g, *a_mirror = Ah + (bj * 16 + 4 * g) * d.lda + bi * 16 + i;
  const int qi = wave / NB, qj = wave % NB;
  const _Float16 *qa_from = Ah + (qi * 16 + i) * d.lda + 8 * g, *qb_from = Ah + (qj * 16 + i) * d.lda + 8 * g;
  const int q_at = (qi * 16 + i) * d.lda + qj * 16 + 4 * g;
  const bool split = NB * cbs <= 2 * SMALL_WAVES;
  auto pair_at = [](const _Float16* q, int plane, u4v (&v)[2]) {
    v[0] = *reinterpret_cast<const u4v*>(q);
    v[1] = *reinterpret_cast<const u4v*>(q + plane);
  };
  // rows of X that a lane reads for Q X (16 lanes read 4 rows of 16 columns, and each gets a column's 4 rows)
  int x_row[DEEP_M][2];
  bool x_in[DEEP_M][2];
#pragma unroll
  for (int k = 0; k < DEEP_M; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 32 * k + 8 * g + 4 * h + (i >> 2);
      x_in[k][h] = row < d.m16;
      x_row[k][h] = row * d.ldx + 4 * (i & 3);
    }
  auto read_x = [&](int cb, int k, u4v (&x)[2]) {
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      u2v v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const _Float16* q = x_in[k][h] ? Xh + plane * plane_x + x_row[k][h] + cb * 16 : zeros;
        v[h] = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)q));
      }
      x[plane] = u4v{v[0][0], v[0][1], v[1][0], v[1][1]};
    }
  };
  auto put_x = [&](int b, int cb, const f4v& acc) {
    const float v[4] = {acc[0] * to_x, acc[1] * to_x, acc[2] * to_x, acc[3] * to_x};
    store_pair4(Xh, Xl, (b * 16 + i) * d.ldx + cb * 16 + 4 * g, v);
  };
  for (int step = 0; step < steps; ++step) {
    __syncthreads();
    if (has_a) {
      f4v acc = {0.f, 0.f, 0.f, 0.f};
      u4v a[2], b[2];
      if (k0 < k1) {
        pair_at(xa + 32 * k0, plane_x, a);
        pair_at(xb + 32 * k0, plane_x, b);
      }
      for (int k = k0; k < k1; ++k) {
        u4v na[2], nb[2];
        const int next = k + 1 < k1 ? k + 1 : k;
        pair_at(xa + 32 * next, plane_x, na);
        pair_at(xb + 32 * next, plane_x, nb);
        acc = pair_products(b, a, acc);
        a[0] = na[0], a[1] = na[1], b[0] = nb[0], b[1] = nb[1];
      }
      if constexpr (KS > 1) {
        lds_st_fenced(reinterpret_cast<f4v*>(P + wave * 256 + i * 16 + 4 * g), acc);
      } else {
        const float v[4] = {acc[0] * to_a, acc[1] * to_a, acc[2] * to_a, acc[3] * to_a};
        store_pair4(a_to, a_to + plane_a, 0, v);
        if (bi != bj) {
          h4v h, lo;
          split4(v, h, lo);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            a_mirror[r * d.lda] = h[r];
            a_mirror[r * d.lda + plane_a] = lo[r];
          }
        }
      }
    }
    __syncthreads();
    if constexpr (KS > 1) {
      for (int e = tid; e < LOWER * 256; e += SMALL_THREADS) {
        int ei, ej;
        triangle(e >> 8, ei, ej);
        const int r = (e >> 4) & 15, c = e & 15;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < KS; ++q) v += P[((e >> 8) * KS + q) * 256 + (e & 255)];
        v *= to_a;
        const _Float16 h = (_Float16)v, lo = (_Float16)(v - (float)h);
        Ah[(ei * 16 + r) * d.lda + ej * 16 + c] = h;
        Al[(ei * 16 + r) * d.lda + ej * 16 + c] = lo;
        if (ei != ej) {
          Ah[(ej * 16 + c) * d.lda + ei * 16 + r] = h;
          Al[(ej * 16 + c) * d.lda + ei * 16 + r] = lo;
        }
      }
      __syncthreads();
    }
    if (has_q) {
      f4v acc = {0.f, 0.f, 0.f, 0.f};
      u4v a[DEEP_M][2], b[DEEP_M][2];
#pragma unroll
      for (int k = 0; k < DEEP_M; ++k) {
        pair_at(qa_from + 32 * k, plane_a, a[k]);
        pair_at(qb_from + 32 * k, plane_a, b[k]);
      }
      const h4v h = *reinterpret_cast<const h4v*>(Ah + q_at), lo = *reinterpret_cast<const h4v*>(Al + q_at);
#pragma unroll
      for (int k = 0; k < DEEP_M; ++k) acc = pair_products(b[k], a[k], acc);
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        v[r] = fmaf(qs, acc[r], fmaf(qb, (float)h[r] + (float)lo[r], qi == qj && i == 4 * g + r ? qa : 0.f));
      store_pair4(Qh, Ql, q_at, v);
    }
    __syncthreads();
    // X, in place.  With few blocks each wave takes one or two of 16 x 16, and everything is read before anything is written;
    // with many it takes whole blocks of columns, which no other wave reads
    if (split) {
      f4v acc[2];
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        acc[k2] = f4v{0.f, 0.f, 0.f, 0.f};
        const int task = wave + SMALL_WAVES * k2, b = task % NB, cb = task / NB;
        if (cb >= cbs) continue;
        u4v x[DEEP_M][2], q[DEEP_M][2];
#pragma unroll
        for (int k = 0; k < DEEP_M; ++k) {
          read_x(cb, k, x[k]);
          pair_at(Qh + (b * 16 + i) * d.lda + 8 * g + 32 * k, plane_a, q[k]);
        }
#pragma unroll
        for (int k = 0; k < DEEP_M; ++k) acc[k2] = pair_products(x[k], q[k], acc[k2]);
      }
      __syncthreads();
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        const int task = wave + SMALL_WAVES * k2, b = task % NB, cb = task / NB;
        if (cb < cbs) put_x(b, cb, acc[k2]);
      }
    } else {
      for (int cb = wave; cb < cbs; cb += SMALL_WAVES) {
        f4v acc[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < DEEP_M; ++k) {
          u4v x[2];
          read_x(cb, k, x);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            u4v q[2];
            pair_at(Qh + (b * 16 + i) * d.lda + 8 * g + 32 * k, plane_a, q);
            acc[b] = pair_products(x, q, acc[b]);
          }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) put_x(b, cb, acc[b]);
      }
    }
  }
  __syncthreads();
  const float step = p.step * t.scale, down = 1.f / p.up_x;
  for (int e = tid * 4; e < size; e += SMALL_THREADS * 4) {
    const int have = min(4, size - e);
    int r = e / t.cols, c = e - r * t.cols;
    float v[4];
    for (int j = 0; j < have; ++j) {
      const int at = turned ? c * d.ldx + r : r * d.ldx + c;
      v[j] = ((float)Xh[at] + (float)Xl[at]) * down;
      if (p.update) v[j] = fmaf(p.keep, typed_at(t.w, p.w_type, base + e + j), -step * v[j]);
      if (++c == t.cols) c = 0, ++r;
    }
    if (have == 4 && p.w_type == NFI_F32) store_piece<float, 4>((float*)t.w + base + e, v);
    else
      for (int j = 0; j < have; ++j) store_typed(t.w, p.w_type, base + e + j, v[j]);
  }
}

// Both: one workgroup for each matrix.  Its 16 waves of 128 registers fill a compute unit, whatever LDS it takes
constexpr int SMALL_BYTES = 155648;
static_assert(ROWS16_BYTES <= SMALL_BYTES, "rows16 fits");
template <int N>
__global__ void __launch_bounds__(SMALL_THREADS) ortho_small(const Table<N> p, int steps) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[SMALL_BYTES];
  __shared__ double red[SMALL_WAVES];
  int matrix, unit;
  const int it = locate(p, blockIdx.x, matrix, unit, [](const Item&) { return 1; });
  const Item& t = p.item[it];
  if (t.m > 48) run_lds<4>(p, t, matrix, steps, lds, red);
  else if (t.m > 32) run_lds<3>(p, t, matrix, steps, lds, red);
  else if (t.m > 16) run_lds<2>(p, t, matrix, steps, lds, red);
  else if (t.n <= 256) run_rows16<1>(p, t, matrix, steps, lds, red);
  else if (t.n <= 512) run_rows16<2>(p, t, matrix, steps, lds, red);
  else run_rows16<8>(p, t, matrix, steps, lds, red);
}

// ---- host --------------------------------------------------------------------------------------------------------------

static inline int ceil_to(int v, int k) { return (v + k - 1) / k * k; }
static inline int64_t up(int64_t v) { return (v + 255) / 256 * 256; }

// Does a matrix run in one workgroup (else as tiles)?
static bool is_small(const nfi_ortho_item& q) {
  const int m = std::min(q.rows, q.cols), n = std::max(q.rows, q.cols);
  if (m <= 16) return n <= 2048;
  return m <= 64 && n <= 65536 && SmallShape(m, n).bytes() <= SMALL_BYTES;
}

constexpr int MOST_SMALL = 1 << 21;   // workgroups of a launch (a launch has fewer than 2^32 threads)

// a table in the smallest size that holds its items
template <int N>
static Table<N> smaller(const Table<ITEMS>& t) {
  Table<N> r;
  (Args&)r = t;
  std::copy(t.item, t.item + std::min(t.items, N), r.item);
  return r;
}
// the items' first units, per(item) for each matrix; returns all
template <int N, class F>
static unsigned number_units(Table<N>& t, F per) {
  int64_t all = 0;
  for (int i = 0; i < N; ++i) {
    t.first[i] = i < t.items ? (int)all : 0x7fffffff;
    if (i < t.items) all += (int64_t)per(t.item[i]) * t.item[i].count;
  }
  return (unsigned)all;
}
template <int N>
static void launch_small(const Table<ITEMS>& a, int steps, hipStream_t s) {
  Table<N> t = smaller<N>(a);
  const unsigned blocks = number_units(t, [](const Item&) { return 1; });
  ortho_small<N><<<blocks, SMALL_THREADS, 0, s>>>(t, steps);
}
template <int N>
static void launch_tiles(const Table<ITEMS>& a, int steps, hipStream_t s) {
  Table<N> t = smaller<N>(a);
  auto lower = [](const Item& q) { return (q.mp / TILE) * (q.mp / TILE + 1) / 2; };
  auto launch = [&](auto kernel, auto per) {
    const unsigned blocks = number_units(t, per);
    if (blocks) kernel<<<blocks, 256, 0, s>>>(t);
  };
  launch(ortho_norm<N>, [](const Item& q) { return q.chunks; });
  launch(ortho_start<N>, [](const Item& q) { return q.mp / 64 * (q.np / 64); });
  for (int k = 0; k < steps; ++k) {
    t.last = k == steps - 1;
    launch(ortho_gram<false, N>, [&](const Item& q) { return lower(q) * q.split_a; });
    launch(ortho_join<false, N>, [&](const Item& q) { return q.split_a > 1 ? lower(q) : 0; });
    launch(ortho_gram<true, N>, [&](const Item& q) { return lower(q) * q.split_q; });
    launch(ortho_join<true, N>, [&](const Item& q) { return q.split_q > 1 ? lower(q) : 0; });
    launch(ortho_apply<N>, [](const Item& q) { return q.mp / TILE * (q.np / TILE); });
    for (int i = 0; i < t.items; ++i) std::swap(t.item[i].x, t.item[i].y);
  }
}

static int64_t padded_side(int v) { return ceil_to(v, TILE); }
static int64_t lower_of(int64_t mp) { return (mp / TILE) * (mp / TILE + 1) / 2; }
constexpr int MOST_SPLIT = 8;

static int64_t item_bytes(const nfi_ortho_item& s) {
  const int m = std::min(s.rows, s.cols), n = std::max(s.rows, s.cols);
  if (is_small(s)) return 0;
  const int64_t mp = padded_side(m), np = padded_side(n), size = (int64_t)s.rows * s.cols;
  return s.count * (2 * up(mp * np * 4) + 2 * up(mp * mp * 4)) + up(s.count * ((size + NORM_CHUNK - 1) / NORM_CHUNK) * 8);
}

// Tiles of A are few and long where matrices are wide: with fewer than the 256 compute units' one each, the contracted index is
// divided so that two fit on every unit, in pieces of 12 steps at least (a shorter one costs more in the join).  The partial tiles
// of A, and after them those of Q, lie from `part` on; returns their bytes.
static int64_t choose_splits(Item* items, int count, unsigned char* part) {
  int64_t tiles = 0, steps_a = 0, steps_q = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t t = lower_of(items[i].mp) * items[i].count;
    tiles += t;
    steps_a += t * (items[i].np / 32);
    steps_q += t * (items[i].mp / 32);
  }
  auto split = [&](int64_t all, int64_t own) {
    if (tiles >= 256) return 1;
    const int64_t piece = std::max<int64_t>(12, (all + 511) / 512);
    return (int)std::min<int64_t>(MOST_SPLIT, std::max<int64_t>(1, own / piece));
  };
  int64_t used = 0;
  for (int i = 0; i < count; ++i) {
    Item& t = items[i];
    t.split_a = split(steps_a, t.np / 32);
    t.split_q = split(steps_q, t.mp / 32);
    t.part = (float*)(part + used);
    const int most = std::max(t.split_a, t.split_q);
    if (most > 1) used += lower_of(t.mp) * t.count * TILE * TILE * 4 * most;
  }
  return used;
}

// largest |s q(s^2)| and |q| over s in [0, top], q(t) = a + b t + c t^2: at the ends or where a derivative is 0
static void bounds(double a, double b, double c, double top, double& x, double& q) {
  x = q = 0.;
  auto at = [&](double t) {
    if (!(t >= 0. && t <= top * top)) return;
    const double v = std::fabs(a + t * (b + t * c));
    x = std::max(x, std::sqrt(t) * v);
    q = std::max(q, v);
  };
  at(0.);
  at(top * top);
  at(-b / (2. * c));
  const double root = std::sqrt(9. * b * b - 20. * a * c);   // a + 3 b t + 5 c t^2 = 0
  at((-3. * b + root) / (10. * c));
  at((-3. * b - root) / (10. * c));
  at(-a / (3. * b));
}

static int check_items(const nfi_ortho_item* items, int n_items) {
  for (int i = 0; i < n_items; ++i) {
    const nfi_ortho_item& s = items[i];
    NFI_REQUIRE(s.rows > 0 && s.cols > 0 && s.count > 0 && s.rows <= NFI_ORTHO_MAX_SIDE && s.cols <= NFI_ORTHO_MAX_SIDE,
                "ortho: matrix %d is %d x %d x %d (sides 1 .. %d)", i, s.count, s.rows, s.cols, NFI_ORTHO_MAX_SIDE);
    const int64_t tr = (s.rows + TILE - 1) / TILE, tc = (s.cols + TILE - 1) / TILE;
    NFI_REQUIRE(4 * tr * tc * s.count < (1ll << 26), "ortho: matrix %d is too large", i);
  }
  return NFI_OK;
}

static int check(const nfi_ortho_args* p, double& most_x, double& most_q) {
  NFI_REQUIRE(p && p->items && p->n_items > 0, "ortho: no matrices");
  NFI_REQUIRE(type_ok(p->g_type) && type_ok(p->w_type), "ortho: bad type");
  NFI_REQUIRE(p->steps >= 1 && p->steps <= 64, "ortho: %d steps (1 .. 64)", p->steps);
  NFI_REQUIRE(p->eps > 0.f && std::isfinite(p->eps), "ortho: eps %g", (double)p->eps);
  const int e = check_items(p->items, p->n_items);
  if (e) return e;
  for (int i = 0; i < p->n_items; ++i) NFI_REQUIRE(p->items[i].g && p->items[i].w, "ortho: null tensor");
  // the iterates stay bounded under this polynomial
  double top = 1., x, q;
  most_x = 1.;
  most_q = 0.;
  for (int k = 0; k < p->steps; ++k) {
    bounds(p->a, p->b, p->c, top * 1.0001, x, q);   // (a division by 0 gives a point outside)
    most_x = std::max(most_x, x);
    most_q = std::max(most_q, q);
    top = x;
    NFI_REQUIRE(std::isfinite(x) && x < 64. && q > 0. && q < 4096., "ortho: the polynomial %g, %g, %g leaves its range", (double)p->a, (double)p->b,
                (double)p->c);
  }
  return NFI_OK;
}

static float power_below(double limit) { return (float)std::ldexp(1., (int)std::floor(std::log2(limit))); }

}  // namespace learn
}  // namespace nfi

using namespace nfi::learn;

extern "C" {

int64_t nfi_ortho_work_bytes(const nfi_ortho_item* items, int32_t n_items) {
  if (check_items(items, n_items) != NFI_OK) return -1;
  int64_t most = 0, sum = 0;
  int held = 0;
  Item table[ITEMS];
  for (int i = 0; i <= n_items; ++i) {
    const int64_t b = i < n_items ? item_bytes(items[i]) : 0;
    if (b > 0) {
      Item& t = table[held++];
      t = {};
      t.count = items[i].count;
      t.mp = (int)padded_side(std::min(items[i].rows, items[i].cols));
      t.np = (int)padded_side(std::max(items[i].rows, items[i].cols));
      sum += b;
    }
    if (held == ITEMS || (i == n_items && held > 0)) {
      most = std::max(most, sum + choose_splits(table, held, nullptr));
      held = 0;
      sum = 0;
    }
  }
  return most;
}

int32_t nfi_ortho(const nfi_ortho_args* p, void* stream) {
  double most_x, most_q;
  const int e = check(p, most_x, most_q);
  if (e) return e;
  const int64_t need = nfi_ortho_work_bytes(p->items, p->n_items);
  NFI_REQUIRE(p->work_bytes >= need && (need == 0 || p->work), "ortho: %lld bytes of work, %lld wanted", (long long)p->work_bytes, (long long)need);
  hipStream_t s = (hipStream_t)stream;
  Args base = {};
  base.g_type = p->g_type;
  base.w_type = p->w_type;
  base.update = p->update;
  base.nesterov = p->nesterov;
  base.beta = p->momentum;
  base.keep = 1.f - p->decay;
  base.step = p->step;
  base.a = p->a;
  base.b = p->b;
  base.c = p->c;
  base.eps = p->eps;
  // largest halves: entries of a matrix are at most its largest singular value (with room for rounding)
  base.up_x = power_below(60000. / (1.001 * most_x));
  base.up_a = power_below(60000. / (1.002 * most_x * most_x));
  base.up_q = power_below(60000. / (1.002 * most_q));
  auto item = [&](const nfi_ortho_item& q, int unit) {
    Item t = {};
    t.g = q.g;
    t.mom = (float*)q.momentum;
    t.w = q.w;
    t.scale = q.scale;
    t.rows = q.rows;
    t.cols = q.cols;
    t.count = q.count;
    t.m = std::min(q.rows, q.cols);
    t.n = std::max(q.rows, q.cols);
    t.mp = ceil_to(t.m, unit);
    t.np = ceil_to(t.n, unit);
    return t;
  };
  Table<ITEMS> a;
  (Args&)a = base;
  auto flush_small = [&]() {
    if (a.items == 1) launch_small<1>(a, p->steps, s);
    else if (a.items > 0 && a.items <= 8) launch_small<8>(a, p->steps, s);
    else if (a.items > 8) launch_small<ITEMS>(a, p->steps, s);
    a.items = 0;
  };
  int64_t held = 0;   // workgroups of the launch
  for (int i = 0; i < p->n_items; ++i) {
    const nfi_ortho_item& q = p->items[i];
    if (!is_small(q)) continue;
    const int64_t size = (int64_t)q.rows * q.cols;
    for (int done = 0; done < q.count;) {   // (a run of more matrices than a launch takes leaves in pieces)
      Item t = item(q, 16);
      t.g = (const unsigned char*)q.g + done * size * type_bytes(p->g_type);
      if (t.mom) t.mom += done * size;
      t.w = (unsigned char*)q.w + done * size * type_bytes(p->w_type);
      t.count = (int)std::min<int64_t>(q.count - done, MOST_SMALL - held);
      done += t.count;
      held += t.count;
      a.item[a.items++] = t;
      if (a.items == ITEMS || held == MOST_SMALL) {
        flush_small();
        held = 0;
      }
    }
  }
  flush_small();
  unsigned char* work = (unsigned char*)p->work;
  auto flush = [&]() {
    choose_splits(a.item, a.items, work);   // (behind the last item)
    if (a.items == 1) launch_tiles<1>(a, p->steps, s);
    else if (a.items > 0 && a.items <= 8) launch_tiles<8>(a, p->steps, s);
    else if (a.items > 8) launch_tiles<ITEMS>(a, p->steps, s);
    a.items = 0;
    work = (unsigned char*)p->work;
  };
  for (int i = 0; i < p->n_items; ++i) {
    const nfi_ortho_item& q = p->items[i];
    if (is_small(q)) continue;
    Item t = item(q, TILE);
    const int64_t sx = up((int64_t)t.mp * t.np * 4) * t.count, sa = up((int64_t)t.mp * t.mp * 4) * t.count;
    t.x = (_Float16*)work;
    t.y = (_Float16*)(work + sx);
    t.a = (_Float16*)(work + 2 * sx);
    t.q = (_Float16*)(work + 2 * sx + sa);
    t.sums = (double*)(work + 2 * sx + 2 * sa);
    t.chunks = (int)(((int64_t)q.rows * q.cols + NORM_CHUNK - 1) / NORM_CHUNK);
    work += item_bytes(q);
    a.item[a.items++] = t;
    if (a.items == ITEMS) flush();
  }
  flush();
  NFI_CHECK_LAUNCH("ortho");
  return NFI_OK;
}

}  // extern "C"
