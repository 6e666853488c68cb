// Products grouped by ragged runs of rows (include/nfi_learn.h nfi_grouped_*): rows off[e] .. off[e+1] of x
// [T][K] meet w[e] [N][K]
//
//   y[r] = w[e] x[r] + b[e]      d x[r] = w[e]^T dy[r]      d w[e] = sum_r dy[r] x[r]^T      d b[e] = sum_r dy[r]
//
// 2 T K N operations each way and product; the offsets stay on the device: a launch covers every tile that
// any division into groups could need, and a workgroup finds its group by a scan of the tile counts.
//
// 16 experts, 32,749 rows of 1024 -> 4096 in bf16: forward 358 us, dx 347, dw 355 (275 GF each: 770 .. 790 TF).  Per step
// a compute unit's LDS takes 32 KB of loads and gives 64 KB of fragments, 768 clocks against 512 of its matrix cores, which
// bounds these tiles: the matrix cores are busy 0.39 .. 0.42 of the cycles (at 1.9 GHz), the waves ready but not issued half of
// theirs.  Tiles of 256 x 256 on eight waves read less but spill, and hide neither their first loads nor their last stores: not
// taken.  16,411 rows of 512 -> 512, 32-bit as three bf16 parts: 73, 74 and 64 .. 76 us (116 TF of 192 that six products
// leave), bound by cutting the parts, 5 operations for each value and part.  Few rows are bound by reading the weights (48
// rows, 67 MB: 14 us).
#include <algorithm>

#include "nfi_mm.h"

namespace nfi {
namespace learn {

struct GroupedArgs {
  const unsigned char *a, *b;      // operands of the product (see the kernels)
  const void *offsets, *bias;
  void* out;
  float* part;                     // partial results where the rows of a group are split
  int64_t rows;
  int groups, n, k;                // the product's columns (of out) and contracted length
  unsigned lda, ldb;               // bytes between rows
  int64_t sb;                      // bytes between w's matrices
  int offsets64, splits, col_tiles, row_tiles, by_xcd;
};
constexpr int BAND = 8;

__device__ __forceinline__ int64_t offset_at(const void* p, int is64, int e, int64_t rows) {
  const int64_t v = is64 ? ((const int64_t*)p)[e] : (int64_t)((const int32_t*)p)[e];
  return v < 0 ? 0 : (v > rows ? rows : v);
}

// Row tile `tile` over the groups' tiles one after the other, then those of the rows that no group holds.
// Returns the group (groups: rows of none; -1: past the end) and its rows [r0, r1).
__device__ __forceinline__ int find_tile(const GroupedArgs& p, int64_t tile, int64_t& r0, int64_t& r1) {
  const int l = lane_id();
  int64_t before = 0;
  for (int e0 = 0; e0 < p.groups + 2; e0 += 64) {
    // two runs of no group follow the last: the rows before the first group and behind the last
    const int e = e0 + l;
    int64_t s = e == p.groups ? 0 : offset_at(p.offsets, p.offsets64, min(e, p.groups), p.rows);
    int64_t t = offset_at(p.offsets, p.offsets64, e < p.groups ? e + 1 : 0, p.rows);
    if (e > p.groups) t = e == p.groups + 1 ? p.rows : 0;
    const int mine = t > s ? (int)((t - s + TILE - 1) / TILE) : 0;
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(incl, d);
      if (l >= d) incl += v;
    }
    const int64_t at = tile - before - (incl - mine);   // this lane's tile, if it is one of its own
    const unsigned long long hit = __ballot(at >= 0 && at < mine);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      const int64_t first = s + at * TILE, last = min(first + TILE, t);
      r0 = __shfl((int)(first & 0xffffffff), src) & 0xffffffffll;
      r0 |= (int64_t)__shfl((int)(first >> 32), src) << 32;
      r1 = r0 + __shfl((int)(last - first), src);
      return min(e0 + src, p.groups);
    }
    before += __shfl(incl, 63);
  }
  return -1;
}

// y (SLAB_B false: b = w[e], rows of K) and d x (SLAB_B true: a = dy, b = w[e] as slabs): rows of `a` by tiles of 128 x LB
template <class T, bool SLAB_B, int LB>
__global__ void __launch_bounds__(256, 2) grouped_rows(const GroupedArgs p) {
  typedef Share<TILE, LB> S;
  __shared__ __attribute__((aligned(16))) unsigned char s0[(TILE + LB) * STEP_BYTES], s1[(TILE + LB) * STEP_BYTES];
  // bands of BAND row tiles, a band's rows first, so that what an XCD's compute units read at a time is a square of tiles
  const unsigned unit = p.by_xcd ? xcd_order(blockIdx.x, gridDim.x) : blockIdx.x, band = unit / (BAND * p.col_tiles), in_band = unit - band * BAND * p.col_tiles;
  const unsigned rows_of_band = min((unsigned)BAND, (unsigned)p.row_tiles - band * BAND);
  const int64_t tile = band * BAND + in_band % rows_of_band;
  const int c0 = (int)(in_band / rows_of_band) * LB;
  int64_t r0, r1;
  const int e = find_tile(p, tile, r0, r1);
  if (e < 0) return;
  const int rows = (int)(r1 - r0), cols = min(LB, p.n - c0);
  const unsigned char* b = p.b + min(e, p.groups - 1) * p.sb + (SLAB_B ? (int64_t)c0 * (int)sizeof(T) : (int64_t)c0 * p.ldb);
  const int line_a = S::line_a(), line_b = S::line_b();
  T* corner = (T*)p.out + (r0 + line_a) * p.n + c0 + line_b;
  Accumulate<T, S::NA, S::NB, false> out;
  auto add_bias = [&]() {
    if constexpr (!SLAB_B) {
      if (p.bias && e < p.groups) {
        const int g = lane_id() >> 4;
#pragma unroll
        for (int y = 0; y < S::NB; ++y) {
          f4v bias;   // (all in flight: clamped, not skipped)
#pragma unroll
          for (int r = 0; r < 4; ++r) bias[r] = (float)((const T*)p.bias)[(int64_t)e * p.n + c0 + min(line_b + y * 16 + 4 * g + r, cols - 1)];
#pragma unroll
          for (int x = 0; x < S::NA; ++x) out.acc[x][y] += bias;
        }
      }
    }
  };
  out.clear();
  const bool live = e < p.groups;
  if (live) tile_product<T, false, SLAB_B, TILE, LB, sizeof(T) == 4>(p.a + r0 * p.lda, p.lda, rows, b, p.ldb, cols, p.k, s0, s1, out, false);
  bool again = false;
  unsigned long long which = 0;
  unsigned lines;
  if constexpr (sizeof(T) == 4) {
    again = live && any_wave(out.overflowed(), s0);
    if (again) out.broken(which, lines);
  }
  add_bias();
  store_part<T, S::NA, S::NB>(out.acc, S::room(s0, s1), corner, p.n, rows - line_a, cols - line_b);
  if constexpr (sizeof(T) == 4) {
    if (!again) return;
    __syncthreads();   // (the stages are free of what was stored)
    out.clear();
    tile_product<T, false, SLAB_B, TILE, LB, false>(p.a + r0 * p.lda, p.lda, rows, b, p.ldb, cols, p.k, s0, s1, out, false);
    add_bias();
    store_broken(out.acc, which, corner, p.n, rows - line_a, cols - line_b);
  }
}

// d w[e] [N][K] and d b[e]: a = dy as slabs (its columns are the lines), b = x as slabs, tiles of L x L.  Partial results: part [split][group][N][K], then part_b [split][group][N].
template <class T, int L>
__global__ void __launch_bounds__(256, 2) grouped_weights(const GroupedArgs p, int n_rows, void* gb, float* part_b) {
  typedef Share<L, L> S;
  __shared__ __attribute__((aligned(16))) unsigned char s0[2 * L * STEP_BYTES], s1[2 * L * STEP_BYTES];
  const unsigned tile = blockIdx.x % p.row_tiles, place = blockIdx.x / p.row_tiles;   // place: split, group
  const int e = (int)(place % p.groups), z = (int)(place / p.groups);
  const int m0 = (int)(tile / p.col_tiles) * L, c0 = (int)(tile % p.col_tiles) * L;
  const int64_t s = offset_at(p.offsets, p.offsets64, e, p.rows), t = max(s, offset_at(p.offsets, p.offsets64, e + 1, p.rows));
  // pieces of whole steps
  constexpr int KSTEP = STEP_BYTES / sizeof(T);
  const int64_t piece = ((t - s + p.splits - 1) / p.splits + KSTEP - 1) / KSTEP * KSTEP;
  const int64_t r0 = min(t, s + z * piece), r1 = min(t, r0 + piece);
  const int lines = min(L, n_rows - m0), cols = min(L, p.n - c0);
  Accumulate<T, S::NA, S::NB, true> acc;
  acc.clear();
  const bool sums = gb != nullptr && c0 == 0;
  const unsigned char *pa = p.a + r0 * p.lda + m0 * (int64_t)sizeof(T), *pb = p.b + r0 * p.ldb + c0 * (int64_t)sizeof(T);
  tile_product<T, true, true, L, L, sizeof(T) == 4>(pa, p.lda, lines, pb, p.ldb, cols, r1 - r0, s0, s1, acc, sums);
  const int i = lane_id() & 15, g = lane_id() >> 4, line_a = S::line_a(), line_b = S::line_b();
  bool again = false;
  unsigned long long which = 0;
  unsigned which_lines = 0;
  if constexpr (sizeof(T) == 4) {
    again = any_wave(acc.overflowed(), s0);
    if (again) acc.broken(which, which_lines);
  }
  auto put_sums = [&](unsigned of) {
    if (sums && line_b == 0 && g == 0) {
#pragma unroll
      for (int x = 0; x < S::NA; ++x) {
        const int row = line_a + x * 16 + i;
        if (row >= lines || !(of >> x & 1)) continue;
        if (p.splits == 1) ((T*)gb)[(int64_t)e * n_rows + m0 + row] = (T)acc.sum[x][0];
        else part_b[(int64_t)place * n_rows + m0 + row] = acc.sum[x][0];
      }
    }
  };
  put_sums(~0u);
  const int64_t matrix = (int64_t)n_rows * p.n, at = (int64_t)(m0 + line_a) * p.n + c0 + line_b;
  if (p.splits == 1) store_part<T, S::NA, S::NB>(acc.acc, S::room(s0, s1), (T*)p.out + e * matrix + at, p.n, lines - line_a, cols - line_b);
  else store_part<float, S::NA, S::NB>(acc.acc, S::room(s0, s1), p.part + place * matrix + at, p.n, lines - line_a, cols - line_b);
  if constexpr (sizeof(T) == 4) {
    if (!again) return;
    __syncthreads();   // (the stages are free of what was stored)
    acc.clear();
    tile_product<T, true, true, L, L, false>(pa, p.lda, lines, pb, p.ldb, cols, r1 - r0, s0, s1, acc, sums);
    put_sums(which_lines);
    store_broken(acc.acc, which, p.splits == 1 ? (float*)p.out + e * matrix + at : p.part + place * matrix + at, p.n, lines - line_a, cols - line_b);
  }
}

// d b[e] alone: 64 columns x 4 rows at a time; blockIdx.y the group, .z the split
template <class T>
__global__ void __launch_bounds__(256) grouped_bias(const GroupedArgs p) {
  __shared__ float lds[4][64];
  const int e = blockIdx.y, col = blockIdx.x * 64 + (threadIdx.x & 63), slot = threadIdx.x >> 6;
  const int64_t s = offset_at(p.offsets, p.offsets64, e, p.rows), t = max(s, offset_at(p.offsets, p.offsets64, e + 1, p.rows));
  const int64_t piece = (t - s + p.splits - 1) / p.splits;
  const int64_t r0 = min(t, s + blockIdx.z * piece), r1 = min(t, r0 + piece);
  float v = 0.f;
  if (col < p.n) {
#pragma unroll 4
    for (int64_t r = r0 + slot; r < r1; r += 4) v += (float)((const T*)p.a)[r * p.n + col];
  }
  lds[slot][threadIdx.x & 63] = v;
  __syncthreads();
  if (slot == 0 && col < p.n) {
    v = (lds[0][threadIdx.x] + lds[1][threadIdx.x]) + (lds[2][threadIdx.x] + lds[3][threadIdx.x]);
    if (p.splits == 1) ((T*)p.out)[(int64_t)e * p.n + col] = (T)v;
    else p.part[((int64_t)blockIdx.z * p.groups + e) * p.n + col] = v;
  }
}

// Partial results [splits][count] (and of a second array behind) summed in a fixed order and rounded once: 16 neighbours x 16
// slices of the splits at a time
template <class T>
__global__ void __launch_bounds__(256) join_parts(const float* __restrict__ part, T* __restrict__ out, int64_t count,
                                                  const float* __restrict__ part_b, T* __restrict__ out_b, int64_t count_b, int splits) {
  __shared__ float lds[16][68];
  int64_t at = (int64_t)blockIdx.x * 64 + (threadIdx.x & 15) * 4;
  const int64_t first = (count + 63) / 64;   // (uniform) blocks of the first array
  if (blockIdx.x >= first) {
    at -= first * 64;
    part = part_b;
    out = out_b;
    count = count_b;
  }
  const int slice = threadIdx.x >> 4, have = (int)min((int64_t)4, count - at);
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (have == 4) {
#pragma unroll 4
    for (int s = slice; s < splits; s += 16) {
      float u[4];
      load_piece<float, 4>(part + s * count + at, u);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += u[r];
    }
  } else {
    for (int s = slice; s < splits; s += 16)
      for (int r = 0; r < have; ++r) v[r] += part[s * count + at + r];
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) lds_st_fenced(&lds[slice][(threadIdx.x & 15) * 4 + r], v[r]);
  __syncthreads();
  if (threadIdx.x >= 64) return;
  at += threadIdx.x - (int64_t)(threadIdx.x & 15) * 4;
  if (at >= count) return;
  float sum = 0.f;
  const int used = splits < 16 ? splits : 16;
  for (int k = 0; k < used; ++k) sum += lds[k][threadIdx.x];
  out[at] = (T)sum;
}

// The same for few splits, where 16 slices would be mostly empty: a thread takes 4 neighbours of every split
template <class T>
__global__ void __launch_bounds__(256) join_few(const float* __restrict__ part, T* __restrict__ out, int64_t count,
                                                const float* __restrict__ part_b, T* __restrict__ out_b, int64_t count_b, int splits) {
  int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const int64_t first = (count + 1023) / 1024;   // (uniform) blocks of the first array
  if (blockIdx.x >= first) {
    at -= first * 1024;
    part = part_b;
    out = out_b;
    count = count_b;
  }
  const int have = (int)min((int64_t)4, count - at);
  if (have == 4) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      float u[4];
      load_piece<float, 4>(part + s * count + at, u);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += u[r];
    }
    store_piece<T, 4>(out + at, v);
  } else {
    for (int r = 0; r < have; ++r) {
      float v = 0.f;
      for (int s = 0; s < splits; ++s) v += part[s * count + at + r];
      out[at + r] = (T)v;
    }
  }
}

// by slices where there are many splits of few sums (256 of 4 x 64 x 64: 4 us), a thread each where there are few (4 of 8 x 512 x
// 512: 16 -> 8 us)
template <class T>
static void join(const float* part, void* out, int64_t count, const float* part_b, void* out_b, int64_t count_b, int splits, hipStream_t s) {
  if (splits <= 8) join_few<T><<<(unsigned)((count + 1023) / 1024 + (count_b + 1023) / 1024), 256, 0, s>>>(part, (T*)out, count, part_b, (T*)out_b, count_b, splits);
  else join_parts<T><<<(unsigned)((count + 63) / 64 + (count_b + 63) / 64), 256, 0, s>>>(part, (T*)out, count, part_b, (T*)out_b, count_b, splits);
}

// rows of `width` elements to rows of `padded`, zeros behind: a matrix whose rows are not aligned to 16 bytes
template <class T>
__global__ void __launch_bounds__(256) pad_rows(const T* __restrict__ src, T* __restrict__ dst, int64_t rows, int width, int padded) {
  constexpr int V = 16 / sizeof(T);
  const int per = padded / V;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= rows * per) return;
  const int64_t row = id / per;
  const int col = (int)(id - row * per) * V;
  T v[V];
  if (col + V <= width) {
    __builtin_memcpy(v, src + row * width + col, 16);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = col + j < width ? src[row * width + col + j] : (T)0.f;
  }
  __builtin_memcpy(dst + row * padded + col, v, 16);
}

static inline int padded_width(int width, int es) { return (width * es + 15) / 16 * 16 / es; }
static inline bool rows_aligned(const void* p, int width, int es) { return ((uintptr_t)p & 15) == 0 && width * es % 16 == 0; }
static inline int64_t up(int64_t v) { return (v + 255) / 256 * 256; }

// Tiles of the weights' gradients: 64 where a side is no larger (a 128 tile would be half empty)
static int weight_tile(int n, int k) { return std::min(n, k) <= 64 ? 64 : TILE; }
static int64_t tiles_of(int n, int k, int tile) { return (int64_t)((n + tile - 1) / tile) * ((k + tile - 1) / tile); }

// The rows of a group are divided where the tiles alone are too few for 256 compute units with two workgroups (of 128 tiles) or
// three (of 64) each; a piece keeps at least 128 rows of an average group
static int weight_splits(int64_t rows, int groups, int n, int k) {
  const int tile = weight_tile(n, k);
  const int64_t tiles = groups * tiles_of(n, k, tile);
  const int64_t want = (tile == 64 ? 768 : 512) / tiles, most = rows / groups / 128;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 256));
}
static int bias_splits(int64_t rows, int groups, int n) {
  const int64_t tiles = (int64_t)groups * ((n + 63) / 64);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(1024 / tiles, rows / groups / 32), 64));
}

template <class T, bool SLAB>
static void launch_rows(GroupedArgs& p, hipStream_t s) {
  const int lb = p.n <= 64 ? 64 : TILE;   // (64: half of a 128 tile would be empty)
  p.col_tiles = (p.n + lb - 1) / lb;
  p.row_tiles = (int)((p.rows + TILE - 1) / TILE + std::min<int64_t>(p.groups + 2, p.rows));
  // neighbouring tiles to an XCD where they share both operands (16 experts' 32,749 rows of 1024 -> 4096: 388 -> 374 us, back
  // 364 -> 320); weights that a few rows read once, and single columns of tiles, go to all of them in turn (48 rows of 512 ->
  // 2048: 19 -> 15 us)
  p.by_xcd = p.col_tiles > 1 && p.rows / p.groups >= 2 * TILE;
  const unsigned tiles = (unsigned)((int64_t)p.row_tiles * p.col_tiles);
  if (lb == 64) grouped_rows<T, SLAB, 64><<<tiles, 256, 0, s>>>(p);
  else grouped_rows<T, SLAB, TILE><<<tiles, 256, 0, s>>>(p);
}

template <class T>
static const unsigned char* padded(const void* src, int64_t rows, int width, unsigned char*& work, unsigned& ld, hipStream_t s) {
  const int es = sizeof(T), pw = padded_width(width, es);
  ld = (unsigned)pw * es;
  if (rows_aligned(src, width, es)) return (const unsigned char*)src;
  T* dst = (T*)work;
  work += up(rows * (int64_t)ld);
  const int64_t pieces = rows * (pw / (16 / es));
  pad_rows<T><<<(unsigned)((pieces + 255) / 256), 256, 0, s>>>((const T*)src, dst, rows, width, pw);
  return (const unsigned char*)dst;
}

template <class T>
static void forward(const nfi_grouped_args& a, hipStream_t s) {
  unsigned char* work = (unsigned char*)a.work;
  GroupedArgs p = {};
  p.a = padded<T>(a.x, a.rows, a.in_width, work, p.lda, s);
  p.b = padded<T>(a.w, (int64_t)a.groups * a.out_width, a.in_width, work, p.ldb, s);
  p.sb = (int64_t)p.ldb * a.out_width;
  p.offsets = a.offsets;
  p.offsets64 = a.offsets64;
  p.bias = a.bias;
  p.out = a.y;
  p.rows = a.rows;
  p.groups = a.groups;
  p.n = a.out_width;
  p.k = a.in_width;
  launch_rows<T, false>(p, s);
}

template <class T>
static void backward(const nfi_grouped_args& a, hipStream_t s) {
  unsigned char* work = (unsigned char*)a.work;
  GroupedArgs p = {};
  p.offsets = a.offsets;
  p.offsets64 = a.offsets64;
  p.rows = a.rows;
  p.groups = a.groups;
  unsigned ldg = 0;
  const unsigned char* g = a.gx || a.gw ? padded<T>(a.gy, a.rows, a.out_width, work, ldg, s) : nullptr;
  if (a.gx) {
    p.a = g;
    p.lda = ldg;
    p.b = padded<T>(a.w, (int64_t)a.groups * a.out_width, a.in_width, work, p.ldb, s);
    p.sb = (int64_t)p.ldb * a.out_width;
    p.out = a.gx;
    p.n = a.in_width;
    p.k = a.out_width;
    launch_rows<T, true>(p, s);
  }
  if (a.gw) {
    p.a = g;
    p.lda = ldg;
    p.b = padded<T>(a.x, a.rows, a.in_width, work, p.ldb, s);
    p.out = a.gw;
    p.n = a.in_width;
    const int tile = weight_tile(a.out_width, a.in_width);
    p.col_tiles = (a.in_width + tile - 1) / tile;
    p.splits = weight_splits(a.rows, a.groups, a.out_width, a.in_width);
    p.part = (float*)work;
    const int64_t count = (int64_t)a.groups * a.out_width * a.in_width, count_b = a.gb ? (int64_t)a.groups * a.out_width : 0;
    float* part_b = p.part + count * p.splits;
    p.row_tiles = (int)tiles_of(a.out_width, a.in_width, tile);   // (of one matrix)
    const unsigned grid = (unsigned)((int64_t)p.row_tiles * a.groups * p.splits);
    if (tile == 64) grouped_weights<T, 64><<<grid, 256, 0, s>>>(p, a.out_width, a.gb, part_b);
    else grouped_weights<T, TILE><<<grid, 256, 0, s>>>(p, a.out_width, a.gb, part_b);
    if (p.splits > 1)
      join<T>(p.part, a.gw, count, part_b, a.gb, count_b, p.splits, s);
  } else if (a.gb) {
    p.a = (const unsigned char*)a.gy;
    p.out = a.gb;
    p.n = a.out_width;
    p.splits = bias_splits(a.rows, a.groups, a.out_width);
    p.part = (float*)work;
    const int64_t count = (int64_t)a.groups * a.out_width;
    grouped_bias<T><<<dim3((unsigned)((a.out_width + 63) / 64), (unsigned)a.groups, (unsigned)p.splits), 256, 0, s>>>(p);
    if (p.splits > 1) join<T>(p.part, a.gb, count, p.part, a.gb, 0, p.splits, s);
  }
}

static int check(const nfi_grouped_args* a, const char* what) {
  NFI_REQUIRE(a && a->offsets, "%s: null input", what);
  NFI_REQUIRE(type_ok(a->dtype), "%s: bad type", what);
  NFI_REQUIRE(a->rows > 0 && a->rows < (1ll << 31), "%s: %lld rows", what, (long long)a->rows);
  NFI_REQUIRE(a->groups > 0 && a->groups <= NFI_GROUPED_MAX_GROUPS, "%s: %d groups (1 .. %d)", what, a->groups, NFI_GROUPED_MAX_GROUPS);
  // (a tile's offsets are 32-bit: 128 rows of at most 8 MB)
  NFI_REQUIRE(a->in_width > 0 && a->in_width <= NFI_GROUPED_MAX_WIDTH && a->out_width > 0 && a->out_width <= NFI_GROUPED_MAX_WIDTH,
              "%s: widths %d -> %d (1 .. %d)", what, a->in_width, a->out_width, NFI_GROUPED_MAX_WIDTH);
  const int64_t widest = std::max(a->in_width, a->out_width);
  NFI_REQUIRE(((a->rows + TILE - 1) / TILE + a->groups + 2) * ((widest + 63) / 64) < (1ll << 31), "%s: too many tiles", what);
  NFI_REQUIRE(a->groups * tiles_of(a->out_width, a->in_width, 64) < (1ll << 31), "%s: too many tiles", what);
  return NFI_OK;
}

// (a matrix of whatever alignment may be padded: room is kept where its rows are not of whole pieces, or its address
// may not be)
static int64_t pad_bytes(const void* p, int64_t rows, int width, int es) {
  return rows_aligned(p, width, es) ? 0 : up(rows * (int64_t)padded_width(width, es) * es);
}

}  // namespace learn
}  // namespace nfi

using namespace nfi::learn;

extern "C" {

int64_t nfi_grouped_forward_work_bytes(const nfi_grouped_args* a) {
  if (check(a, "grouped_forward") != NFI_OK) return -1;
  const int es = type_bytes(a->dtype);
  return pad_bytes(a->x, a->rows, a->in_width, es) + pad_bytes(a->w, (int64_t)a->groups * a->out_width, a->in_width, es);
}

int64_t nfi_grouped_backward_work_bytes(const nfi_grouped_args* a) {
  if (check(a, "grouped_backward") != NFI_OK) return -1;
  const int es = type_bytes(a->dtype);
  int64_t n = 0;
  if (a->gx || a->gw) n += pad_bytes(a->gy, a->rows, a->out_width, es);
  if (a->gx) n += pad_bytes(a->w, (int64_t)a->groups * a->out_width, a->in_width, es);
  if (a->gw) {
    n += pad_bytes(a->x, a->rows, a->in_width, es);
    const int s = weight_splits(a->rows, a->groups, a->out_width, a->in_width);
    if (s > 1) n += up((int64_t)a->groups * a->out_width * (a->in_width + (a->gb ? 1 : 0)) * 4 * s);
  } else if (a->gb) n += up((int64_t)a->groups * a->out_width * 4 * bias_splits(a->rows, a->groups, a->out_width));
  return n;
}

int32_t nfi_grouped_forward(const nfi_grouped_args* a, void* stream) {
  const int e = check(a, "grouped_forward");
  if (e) return e;
  NFI_REQUIRE(a->x && a->w && a->y, "grouped_forward: null tensor");
  const int64_t need = nfi_grouped_forward_work_bytes(a);
  NFI_REQUIRE(a->work_bytes >= need && (need == 0 || a->work), "grouped_forward: %lld bytes of work, %lld wanted", (long long)a->work_bytes,
              (long long)need);
  hipStream_t s = (hipStream_t)stream;
  if (a->dtype == NFI_F32) forward<float>(*a, s);
  else if (a->dtype == NFI_BF16) forward<bf16_t>(*a, s);
  else forward<f16_t>(*a, s);
  NFI_CHECK_LAUNCH("grouped_forward");
  return NFI_OK;
}

int32_t nfi_grouped_backward(const nfi_grouped_args* a, void* stream) {
  const int e = check(a, "grouped_backward");
  if (e) return e;
  NFI_REQUIRE(a->gy && (!a->gx || a->w) && (!a->gw || a->x), "grouped_backward: null tensor");
  const int64_t need = nfi_grouped_backward_work_bytes(a);
  NFI_REQUIRE(a->work_bytes >= need && (need == 0 || a->work), "grouped_backward: %lld bytes of work, %lld wanted", (long long)a->work_bytes,
              (long long)need);
  hipStream_t s = (hipStream_t)stream;
  if (a->dtype == NFI_F32) backward<float>(*a, s);
  else if (a->dtype == NFI_BF16) backward<bf16_t>(*a, s);
  else backward<f16_t>(*a, s);
  NFI_CHECK_LAUNCH("grouped_backward");
  return NFI_OK;
}

}  // extern "C"
