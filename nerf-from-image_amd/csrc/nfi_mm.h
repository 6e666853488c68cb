// Tiles of a matrix product on the matrix cores, fed by loads that go straight to LDS (gfx950).
//
// An operand tile is 64 or 128 "lines" of 128 bytes of the contracted index (64 16-bit or 32 32-bit values), in one of
// two layouts:
//   lines   the operand's rows hold the contracted index contiguously: LDS [lines][8 pieces of 16 B], piece p of line
//           r stored at p ^ (r & 7), so that the 16-byte reads of 8 lines use all banks
//   slabs   the contracted index runs over rows and the lines are columns (a transposed operand): LDS
//           [64 or 32 rows][columns]; 16-bit fragments are read with the transposing LDS load, 32-bit ones word by
//           word.  Pieces are exchanged by the row so that the rows of one read lie in different banks.
// Both give a lane the same contracted indices in the same order, so any two layouts meet in one product:
// 16-bit: lane (i, g) = (l & 15, l >> 4) holds k = 32 sub + 8 g .. + 7;  32-bit: k = 16 sub + 4 g .. + 3.
// Loads go through a buffer descriptor whose range no lane out of the matrix falls into: such a lane's
// offset is 2^31, and the hardware writes zeros.
//
// 32-bit values meet as three bf16 ones each, v = h + m + l (24 bits in 8 + 8 + 8, exactly), in six products l h + h l + m m +
// m h + h m + h h on the bf16 matrix cores: 96 clocks of them for 32 contracted values against 256 of
// v_mfma_f32_16x16x4_f32, and what is left out is at most 2^-24 of a product (a value below
// 2^-110 keeps fewer bits: its parts' last step is 2^-133, bf16's smallest).  An infinity, or a value that bf16 rounds to
// one, has parts that are no numbers: sums that do not come out finite are taken again in 32-bit products (any_wave).
#pragma once
#include "nfi_learn.h"

namespace nfi {
namespace learn {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef unsigned u4v __attribute__((ext_vector_type(4)));
typedef unsigned u2v __attribute__((ext_vector_type(2)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) unsigned char* lds_bytes;

constexpr int TILE = 128;              // lines of an operand tile
constexpr int STEP_BYTES = 128;        // contracted bytes of a step
constexpr int TILE_BYTES = TILE * STEP_BYTES;
constexpr unsigned NOWHERE = 0x80000000u;

// (uniform by construction, and told so: descriptors live in scalar registers)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(const void* p) {
  const unsigned long long a = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((unsigned long long)hi << 32) | lo), 0, 0x7fffffff, 0x00020000);
}

__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, unsigned char* lds, unsigned offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, (int)offset, 0, 0, 0);
}

// The loads of one operand tile of LINES lines by a workgroup: LINES / 32 a wave, of 1 KB each, at fixed offsets
// from an address that moves by a step (lines: 128 bytes, slabs: a step's rows)
template <class T, bool SLAB, int LINES>
struct TileLoad {
  static constexpr int KSTEP = STEP_BYTES / sizeof(T);
  static constexpr int LOADS = LINES / 32;
  static constexpr int PIECES = SLAB ? LINES * (int)sizeof(T) / 16 : 8;   // 16-byte pieces of an LDS row
  unsigned off[LOADS];    // byte offset of each of this lane's pieces, NOWHERE out of the lines
  int k[LOADS];           // contracted byte (lines) or row (slabs) of the piece within the step

  static __device__ __forceinline__ int lds_row(int j) { return ((threadIdx.x >> 6) * LOADS + j) * (64 / PIECES) + (lane_id() / PIECES); }
  static __device__ __forceinline__ int swizzle(int row) {
    if (!SLAB) return row & 7;
    return sizeof(T) == 2 ? (2 * row) & (PIECES - 1) & 15 : 4 * ((row >> 2) & 3);
  }
  // `lines` valid lines (rows of the operand, or columns of a slab); ld: bytes between the operand's rows
  __device__ __forceinline__ void init(int lines, unsigned ld) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int row = lds_row(j), piece = (lane_id() & (PIECES - 1)) ^ swizzle(row);
      if (SLAB) {
        k[j] = row;
        off[j] = piece * (16 / (int)sizeof(T)) < lines ? row * ld + piece * 16 : NOWHERE;
      } else {
        k[j] = piece * 16;
        off[j] = row < lines ? row * ld + piece * 16 : NOWHERE;
      }
    }
  }
  // left: contracted bytes (lines) or rows (slabs) that remain at this step
  __device__ __forceinline__ void issue(const void* base, unsigned char* lds, int left) const {
    const __amdgpu_buffer_rsrc_t r = descriptor(base);
    unsigned char* dst = lds + (threadIdx.x >> 6) * (LOADS * 1024);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load_to_lds(r, dst + j * 1024, k[j] < left ? off[j] : NOWHERE);
  }
};

// Fragments of N 16-line blocks from line `line0`, for one sub-step, of a tile of LINES lines
template <class T, bool SLAB, int LINES, int N>
__device__ __forceinline__ void read_fragments(const unsigned char* lds, int line0, int sub, u4v (&f)[N]) {
  typedef TileLoad<T, SLAB, LINES> L;
  const int i = lane_id() & 15, g = lane_id() >> 4;
  if constexpr (!SLAB) {
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int row = line0 + 16 * x + i;
      f[x] = *reinterpret_cast<const u4v*>(lds + row * STEP_BYTES + (((4 * sub + g) ^ (row & 7)) << 4));
    }
  } else if constexpr (sizeof(T) == 2) {
    // 16 lanes read 4 rows of 16 columns and each gets a column's 4 rows; twice for 8 rows
    const int r0 = 32 * sub + 8 * g + (i >> 2);
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int piece = (line0 >> 3) + 2 * x + ((i & 3) >> 1), half = (i & 1) * 8;
      u2v v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = r0 + 4 * h;
        const unsigned char* p = lds + row * (L::PIECES * 16) + ((piece ^ L::swizzle(row)) << 4) + half;
        v[h] = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)p));
      }
      f[x] = u4v{v[0][0], v[0][1], v[1][0], v[1][1]};
    }
  } else {
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int col = line0 + 16 * x + i;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int row = 16 * sub + 4 * g + s;   // (row >> 2) & 3 == g
        f[x][s] = *reinterpret_cast<const unsigned*>(lds + row * (L::PIECES * 16) + (((col >> 2) ^ (4 * g)) << 4) + (col & 3) * 4);
      }
    }
  }
}

// acc += b a^T for one sub-step: the accumulator's lane (i, g) register r is a's line i, b's line 4 g + r
template <class T>
__device__ __forceinline__ f4v product(u4v b, u4v a, f4v acc) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b[s]), __uint_as_float(a[s]), acc, 0, 0, 0);
    return acc;
  } else if constexpr (TypeCode<T>::V == NFI_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, b), __builtin_bit_cast(b8v, a), acc, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, b), __builtin_bit_cast(h8v, a), acc, 0, 0, 0);
  }
}

// 8 32-bit values as three bf16 each (to nearest: each part's remainder is half a step of it, so that the products left out,
// m l and l m, are 2^-25 of the whole)
typedef float f2v __attribute__((ext_vector_type(2)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
struct Thirds {
  u4v h, m, l;
  static __device__ __forceinline__ unsigned part(f2v& v) {
    const unsigned p = __builtin_bit_cast(unsigned, __builtin_convertvector(v, b2v));
    v[0] -= __uint_as_float(p << 16);
    v[1] -= __uint_as_float(p & 0xffff0000u);
    return p;
  }
  __device__ __forceinline__ void set(const u4v& v0, const u4v& v1) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f2v v = k < 2 ? f2v{__uint_as_float(v0[2 * k]), __uint_as_float(v0[2 * k + 1])}
                    : f2v{__uint_as_float(v1[2 * k - 4]), __uint_as_float(v1[2 * k - 3])};
      h[k] = part(v);
      m[k] = part(v);
      l[k] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, b2v));
    }
  }
};
__device__ __forceinline__ f4v product(const Thirds& b, const Thirds& a, f4v acc) {
  acc = product<bf16_t>(b.l, a.h, acc);
  acc = product<bf16_t>(b.h, a.l, acc);
  acc = product<bf16_t>(b.m, a.m, acc);
  acc = product<bf16_t>(b.m, a.h, acc);
  acc = product<bf16_t>(b.h, a.m, acc);
  return product<bf16_t>(b.h, a.h, acc);
}

// Workgroups go to the 8 XCDs (each with an L2 of its own) in turn: the unit of work of workgroup b of n, such that
// each XCD gets neighbouring units, which share operands
__device__ __forceinline__ unsigned xcd_order(unsigned b, unsigned n) {
  const unsigned x = b & 7, q = n >> 3, r = n & 7;
  return x * q + min(x, r) + (b >> 3);
}

// vmcnt(n), nothing else (n < 64)
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}

// A barrier alone: __syncthreads() also waits for every load on its way to LDS, those of the next step too
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// How four waves share an LA x LB product tile: two along a's lines, two along b's
template <int LA, int LB>
struct Share {
  static constexpr int NA = LA / 32, NB = LB / 32;   // blocks of 16 lines of a wave
  static __device__ __forceinline__ int line_a() { return ((threadIdx.x >> 6) & 1) * (LA / 2); }
  static __device__ __forceinline__ int line_b() { return (threadIdx.x >> 7) * (LB / 2); }
  // a wave's room for its part, of at most 4 bytes an element, in the stages of a product that has ended
  static __device__ __forceinline__ unsigned char* room(unsigned char* s0, unsigned char* s1) {
    return (threadIdx.x >> 7 ? s1 : s0) + ((threadIdx.x >> 6) & 1) * (LA / 2 * LB / 2 * 4);
  }
};

// What is done with fragments: acc[x][y] += a's block x, b's block y; with SUM also sum[x] += a's lines
template <class T, int NA, int NB, bool SUM>
struct Accumulate {
  f4v acc[NA][NB], sum[NA];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int x = 0; x < NA; ++x) {
      sum[x] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int y = 0; y < NB; ++y) acc[x][y] = f4v{0.f, 0.f, 0.f, 0.f};
    }
  }
  // one sub-step, of 16-bit values or in 32-bit products
  __device__ __forceinline__ void add(const u4v (&fa)[NA], const u4v (&fb)[NB], bool sums) {
#pragma unroll
    for (int x = 0; x < NA; ++x)
#pragma unroll
      for (int y = 0; y < NB; ++y) acc[x][y] = product<T>(fb[y], fa[x], acc[x][y]);
    if (SUM && sums) {
      const unsigned one = TypeCode<T>::V == NFI_F32 ? 0x3f800000u : TypeCode<T>::V == NFI_BF16 ? 0x3f803f80u : 0x3c003c00u;
      const u4v ones = {one, one, one, one};
#pragma unroll
      for (int x = 0; x < NA; ++x) sum[x] = product<T>(ones, fa[x], sum[x]);
    }
  }
  // a step of 32-bit values; the next block of a is cut into its parts while a block's products run
  __device__ __forceinline__ void add32(const u4v (&fa)[2][NA], const u4v (&fb)[2][NB], bool sums) {
    Thirds a[NA], b[NB];
#pragma unroll
    for (int y = 0; y < NB; ++y) b[y].set(fb[0][y], fb[1][y]);
    a[0].set(fa[0][0], fa[1][0]);
#pragma unroll
    for (int x = 0; x < NA; ++x) {
      __builtin_amdgcn_sched_barrier(0);
      if (x + 1 < NA) a[x + 1].set(fa[0][x + 1], fa[1][x + 1]);
#pragma unroll
      for (int y = 0; y < NB; ++y) acc[x][y] = product(b[y], a[x], acc[x][y]);
#pragma unroll
      for (int k = 0; k < 6 * NB; ++k) {   // a product, two other instructions, and so on
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      }
    }
    if (SUM && sums) {
      const unsigned one = 0x3f803f80u;
      const u4v ones = {one, one, one, one};
#pragma unroll
      for (int x = 0; x < NA; ++x) {
        sum[x] = product<bf16_t>(ones, a[x].l, sum[x]);
        sum[x] = product<bf16_t>(ones, a[x].m, sum[x]);
        sum[x] = product<bf16_t>(ones, a[x].h, sum[x]);
      }
    }
  }
  // is a sum of this lane not finite?
  __device__ __forceinline__ bool overflowed() const {
    float z = 0.f;   // (a number times 0, added: 0, or no number)
#pragma unroll
    for (int x = 0; x < NA; ++x) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (SUM) z = fmaf(sum[x][r], 0.f, z);
#pragma unroll
        for (int y = 0; y < NB; ++y) z = fmaf(acc[x][y][r], 0.f, z);
      }
    }
    return z != 0.f;
  }
  // which of them (bit 4 (NB x + y) + r), and which of its lines' sums (bit x)
  __device__ __forceinline__ void broken(unsigned long long& which, unsigned& lines) const {
    static_assert(NA * NB * 4 <= 64, "a bit for each sum");
    which = 0;
    lines = 0;
#pragma unroll
    for (int x = 0; x < NA; ++x) {
      if (SUM) lines |= (unsigned)!(fabsf(sum[x][0]) < INFINITY) << x;
#pragma unroll
      for (int y = 0; y < NB; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) which |= (unsigned long long)!(fabsf(acc[x][y][r]) < INFINITY) << (4 * (NB * x + y) + r);
    }
  }
};

// An LA x LB product tile: steps over the contracted index through two stages of LDS, each of (LA + LB) x 128 bytes.  A step's
// fragments go to registers, its stage is free after a barrier, and the loads of the step after next are made into it while the
// step's (last) products run: loads have a whole step to arrive.  (The stages are two variables of their own: the compiler waits
// for all loads into the one that is read, and for no others.)
template <class T, bool SLAB_A, bool SLAB_B, int LA, int LB, bool PARTS, bool SUM>
__device__ __forceinline__ void tile_product(const unsigned char* a, unsigned lda, int lines_a, const unsigned char* b, unsigned ldb,
                                             int lines_b, int64_t contracted, unsigned char* s0, unsigned char* s1,
                                             Accumulate<T, Share<LA, LB>::NA, Share<LA, LB>::NB, SUM>& out, bool sums) {
  typedef Share<LA, LB> S;
  typedef TileLoad<T, SLAB_A, LA> LoadA;
  typedef TileLoad<T, SLAB_B, LB> LoadB;
  constexpr int KSTEP = STEP_BYTES / sizeof(T), NA = S::NA, NB = S::NB, LOADS = LoadA::LOADS + LoadB::LOADS;
  LoadA la;
  LoadB lb;
  la.init(lines_a, lda);
  lb.init(lines_b, ldb);
  const int64_t step_a = SLAB_A ? (int64_t)KSTEP * lda : STEP_BYTES, step_b = SLAB_B ? (int64_t)KSTEP * ldb : STEP_BYTES;
  const int steps = (int)((contracted + KSTEP - 1) / KSTEP), line_a = S::line_a(), line_b = S::line_b();
  // (a step behind the last reads nothing and clears its stage: every step waits for the same number of loads)
  auto issue = [&](int t, unsigned char* dst) {
    const int64_t k = contracted - (int64_t)t * KSTEP;
    const int left = (int)(k < KSTEP ? k : KSTEP);
    la.issue(a + t * step_a, dst, SLAB_A ? left : left * (int)sizeof(T));
    lb.issue(b + t * step_b, dst + LA * STEP_BYTES, SLAB_B ? left : left * (int)sizeof(T));
    __builtin_amdgcn_sched_barrier(0);   // the waits count on this order of the steps' loads
  };
  auto read = [&](const unsigned char* cur, int sub, u4v (&fa)[NA], u4v (&fb)[NB]) {
    read_fragments<T, SLAB_A, LA, NA>(cur, line_a, sub, fa);
    read_fragments<T, SLAB_B, LB, NB>(cur + LA * STEP_BYTES, line_b, sub, fb);
  };
  auto step = [&](int t, unsigned char* cur) {
    wait_loads<LOADS>();   // step t's loads are in LDS, those of step t + 1 may be on their way
    bare_barrier();
    u4v fa[2][NA], fb[2][NB];
    read(cur, 0, fa[0], fb[0]);
    read(cur, 1, fa[1], fb[1]);
    __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): this wave has read the step
    bare_barrier();
    issue(t + 2, cur);
    if constexpr (PARTS) {   // (of 32-bit values)
      out.add32(fa, fb, sums);
    } else {
      out.add(fa[0], fb[0], sums);
      out.add(fa[1], fb[1], sums);
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

// Has any wave of the workgroup, behind its product, a sum that is not finite?  (32-bit values in parts: an infinity's are no
// numbers.  The sums that are finite stay, and keep their bits whatever another row holds; the others are taken again in 32-bit
// products and stored over them.  The test costs less than 1 % of a tile of 512 contracted values.)
__device__ __forceinline__ bool any_wave(bool mine, unsigned char* free_stage) {
  int* votes = (int*)free_stage;
  const bool wave = __ballot(mine) != 0;
  if (lane_id() == 0) votes[threadIdx.x >> 6] = wave;
  __syncthreads();
  const bool any = (votes[0] | votes[1] | votes[2] | votes[3]) != 0;
  __syncthreads();
  return any;
}

// A wave's part of a product tile to rows of `out` (ld elements apart; `rows` x `cols` of them from this wave's
// corner are the matrix's).  A lane holds 4 columns of a row, 32 bytes of a row's line in a 16-bit store: the part is turned in
// LDS first, where the wave has room for it, and leaves in pieces of 16 bytes, a row's one after the other (32,749 rows of
// 1024 -> 4096 in bf16: 410 -> 365 us).
template <class O, int NA, int NB>
__device__ __forceinline__ void store_part(const f4v (&acc)[NA][NB], unsigned char* lds, O* out, int64_t ld, int rows, int cols) {
  constexpr int V = 16 / (int)sizeof(O), PIECES = NB * (int)sizeof(O), AT_ONCE = 64 / PIECES;   // pieces of a row; rows of a store
  const int l = lane_id(), i = l & 15, g = l >> 4;
#pragma unroll
  for (int x = 0; x < NA; ++x)
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      const int row = 16 * x + i, byte = (16 * y + 4 * g) * (int)sizeof(O);
      unsigned char* p = lds + row * (PIECES * 16) + (((byte >> 4) ^ (row & (PIECES - 1))) << 4) + (byte & 15);
      const f4v v = acc[x][y];
      if constexpr (sizeof(O) == 4) {
        lds_st_fenced((f4v*)p, v);
      } else {
        O t[4] = {(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
        u2v u;
        __builtin_memcpy(&u, t, 8);
        lds_st_fenced((u2v*)p, u);
      }
    }
  asm volatile("" ::: "memory");
  const int piece = l & (PIECES - 1), row0 = l / PIECES, have = cols - piece * V;
  constexpr int STORES = 16 * NA / AT_ONCE, GROUP = STORES < 8 ? STORES : 8;
#pragma unroll
  for (int j0 = 0; j0 < STORES; j0 += GROUP) {
    u4v v[GROUP];
#pragma unroll
    for (int j = 0; j < GROUP; ++j) {
      const int row = row0 + (j0 + j) * AT_ONCE;
      v[j] = *reinterpret_cast<const u4v*>(lds + row * (PIECES * 16) + ((piece ^ (row & (PIECES - 1))) << 4));
    }
#pragma unroll
    for (int j = 0; j < GROUP; ++j) {
      const int row = row0 + (j0 + j) * AT_ONCE;
      O* d = out + row * ld + piece * V;
      if (row < rows && have >= V) {
        __builtin_memcpy(d, &v[j], 16);
      } else if (row < rows) {
        O t[V];
        __builtin_memcpy(t, &v[j], 16);
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (k < have) d[k] = t[k];
      }
    }
  }
}

// The sums of `which` (Accumulate::broken) alone, to the same places
template <int NA, int NB>
__device__ __forceinline__ void store_broken(const f4v (&acc)[NA][NB], unsigned long long which, float* out, int64_t ld, int rows, int cols) {
  const int i = lane_id() & 15, g = lane_id() >> 4;
#pragma unroll
  for (int x = 0; x < NA; ++x)
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * x + i, col = 16 * y + 4 * g + r;
        if ((which >> (4 * (NB * x + y) + r) & 1) && row < rows && col < cols) out[row * ld + col] = acc[x][y][r];
      }
}

}  // namespace learn
}  // namespace nfi
