// Tiles of a matrix product on the matrix cores, fed by loads that go straight to LDS (gfx950).
//
// An operand tile is 128 "lines" of 128 bytes of the contracted index (64 16-bit or 32 32-bit values),
// 16 KB, in one of two layouts:
//   lines   the operand's rows hold the contracted index contiguously: LDS [128 lines][8 pieces of 16 B],
//           piece p of line r stored at p ^ (r & 7), so that the 16-byte reads of 8 lines use all banks
//   slabs   the contracted index runs over rows and the lines are columns (a transposed operand): LDS
//           [64 or 32 rows][128 columns]; 16-bit fragments are read with the transposing LDS load, 32-bit
//           ones word by word.  Pieces are exchanged by the row so that the rows of one read lie in
//           different banks.
// Both give a lane the same contracted indices in the same order, so any two layouts meet in one product:
// 16-bit: lane (i, g) = (l & 15, l >> 4) holds k = 32 sub + 8 g .. + 7;  32-bit: k = 16 sub + 4 g + s for
// the s-th product of a sub-step.
// Loads go through a buffer descriptor whose range no lane out of the matrix falls into: such a lane's
// offset is 2^31, and the hardware writes zeros.
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

// The loads of one operand tile by a workgroup of 4 waves: 4 of 1 KB for each wave, at fixed offsets from
// an address that moves by a step (lines: 128 bytes, slabs: a step's rows)
template <class T, bool SLAB>
struct TileLoad {
  static constexpr int KSTEP = STEP_BYTES / sizeof(T);
  static constexpr int PIECES = SLAB ? TILE * (int)sizeof(T) / 16 : 8;   // 16-byte pieces of an LDS row
  unsigned off[4];    // byte offset of each of this lane's pieces, NOWHERE out of the lines
  int k[4];           // contracted byte (lines) or row (slabs) of the piece within the step

  static __device__ __forceinline__ int lds_row(int j) { return ((threadIdx.x >> 6) * 4 + j) * (64 / PIECES) + (lane_id() / PIECES); }
  static __device__ __forceinline__ int swizzle(int row) {
    if (!SLAB) return row & 7;
    return sizeof(T) == 2 ? 2 * (row & 7) : 4 * ((row >> 2) & 3);
  }
  // `lines` valid lines (rows of the operand, or columns of a slab); ld: bytes between the operand's rows
  __device__ __forceinline__ void init(int lines, unsigned ld) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
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
    unsigned char* dst = lds + (threadIdx.x >> 6) * 4096;
    if (left >= (SLAB ? KSTEP : STEP_BYTES)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) load_to_lds(r, dst + j * 1024, off[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) load_to_lds(r, dst + j * 1024, k[j] < left ? off[j] : NOWHERE);
    }
  }
};

// Fragments of N 16-line blocks from line `line0`, for one sub-step
template <class T, bool SLAB, int N>
__device__ __forceinline__ void read_fragments(const unsigned char* lds, int line0, int sub, u4v (&f)[N]) {
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
        const unsigned char* p = lds + row * 256 + ((piece ^ (2 * (row & 7))) << 4) + half;
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
        f[x][s] = *reinterpret_cast<const unsigned*>(lds + row * 512 + (((col >> 2) ^ (4 * g)) << 4) + (col & 3) * 4);
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

// A 128 x 128 product tile by 4 waves of 64 x 64: steps over the contracted index, two stages of LDS (2 x 32
// KB), the next step's loads in flight during a step's products.  `left` and the strides: TileLoad::issue.
template <class T, bool SLAB_A, bool SLAB_B>
__device__ __forceinline__ void tile_product(const unsigned char* a, unsigned lda, int lines_a, const unsigned char* b, unsigned ldb,
                                             int lines_b, int64_t contracted, unsigned char* lds, f4v (&acc)[4][4]) {
  constexpr int KSTEP = STEP_BYTES / sizeof(T);
  TileLoad<T, SLAB_A> la;
  TileLoad<T, SLAB_B> lb;
  la.init(lines_a, lda);
  lb.init(lines_b, ldb);
  const int64_t step_a = SLAB_A ? (int64_t)KSTEP * lda : STEP_BYTES, step_b = SLAB_B ? (int64_t)KSTEP * ldb : STEP_BYTES;
  const int steps = (int)((contracted + KSTEP - 1) / KSTEP);
  const int wave = threadIdx.x >> 6, line_a = (wave & 1) * 64, line_b = (wave >> 1) * 64;
  auto issue = [&](int t, unsigned char* dst) {
    const int64_t k = contracted - (int64_t)t * KSTEP;
    const int left = (int)(k < KSTEP ? k : KSTEP);
    la.issue(a + t * step_a, dst, SLAB_A ? left : left * (int)sizeof(T));
    lb.issue(b + t * step_b, dst + TILE_BYTES, SLAB_B ? left : left * (int)sizeof(T));
  };
  if (steps > 0) issue(0, lds);
  for (int t = 0; t < steps; ++t) {
    const unsigned char* cur = lds + (t & 1) * 2 * TILE_BYTES;
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's loads of step t are in LDS
    __syncthreads();
    u4v fa[2][4], fb[2][4];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      read_fragments<T, SLAB_A, 4>(cur, line_a, sub, fa[sub]);
      read_fragments<T, SLAB_B, 4>(cur + TILE_BYTES, line_b, sub, fb[sub]);
    }
    if (t + 1 < steps) issue(t + 1, lds + ((t + 1) & 1) * 2 * TILE_BYTES);   // (last read before the barrier above)
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = product<T>(fb[sub][y], fa[sub][x], acc[x][y]);
  }
}

}  // namespace learn
}  // namespace nfi
