// The residual norm (include/nfi_learn.h nfi_resnorm_*): per row r of width D
//
//   n = (h - mean) rstd      u = n w + b      v = max(u, slope u)      x = scale (res + gate v)
//   m = (x - mean2) rstd2    y = m w2 + b2
//
// and, with g = gx + rstd2 (gy w2 - mean(gy w2) - m mean(gy w2 m)) (the middle mean only for LayerNorm),
//
//   d res = scale g     d gate = sum scale g v     gu = scale g gate (u > 0 ? 1 : slope)
//   d w = sum gu n      d b = sum gu               d h = rstd (gu w - mean(gu w) - n mean(gu w n))
//   d w2 = sum gy m     d b2 = sum gy
//
// Bound by memory: forward reads h and res and writes x and y once, backward reads h, res, gx, gy and
// writes d h and d res once (x is recomputed from h and res: reading it back would cost as much).  A
// row is held in registers by TPR lanes, NC pieces of 16 bytes each, so that every statistic is one
// pass of lane moves: variances are sums of squared differences from the mean, not differences of
// squares.  TPR is the smallest power of two that holds a row (8 rows of 64 bf16 share a wave); wide rows
// take a workgroup, in the backward of twice or four times as many lanes as in the forward (dispatch).  The parameter
// gradients stay in registers over a workgroup's rows and leave as one partial per workgroup, summed by a second launch in a
// fixed order.  16,384 rows of 1024 bf16, both norms, eight gates: forward 31 us (134 MB, 4.3 TB/s), backward 57 + 5 us
// (201 MB, 3.5 TB/s: vector instructions issue in 0.55 of the cycles, with 2 x 2 sums over four waves and 50 operations an
// element, and its two waves a SIMD wait in 0.59 of theirs).  131,072 rows of 64 32-bit values: 17 us (101 MB), and with their
// gradients 50 (269 MB), or 52 where each of 8 groups has parameters of its own.
#include <algorithm>

#include "nfi_learn.h"

namespace nfi {
namespace learn {

constexpr int PARAMS = 5;       // d weight, d bias, d next_weight, d next_bias, d gate

// Workgroups of the backward, as many as 256 compute units hold at a time: two each; three where a row's four waves meet twice a
// row and wait (16,384 rows of 1024 bf16: 66 -> 58 us; 131,072 rows of 64, a wave each, lose by it, 31 -> 35); one of eight
// waves where a row is wider, whose partial results cost most (2048 rows of 8192 bf16: 117 us in place of 143)
__host__ inline int blocks_of(int width) { return width <= 512 ? 512 : width <= 1024 ? 768 : width <= 2048 ? 512 : 256; }

// sum over TPR lanes (a power of two up to 64), in every one of them
template <int TPR>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (TPR >= 2) v += dpp_mov<0xB1>(v);
  if constexpr (TPR >= 4) v += dpp_mov<0x4E>(v);
  if constexpr (TPR >= 8) v += dpp_mov<0x141>(v);
  if constexpr (TPR >= 16) v += dpp_mov<0x140>(v);
  if constexpr (TPR >= 32) v += __shfl_xor(v, 16);
  if constexpr (TPR >= 64) {
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(s[0]) + __int_as_float(s[1]);
  }
  return v;
}

// N sums over a row's lanes; `turn` alternates the exchange buffer, so one barrier is enough
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*buf)[2][16], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<(TPR < 64 ? TPR : 64)>(v[i]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    if (lane_id() == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds_st_fenced(&buf[turn][i][threadIdx.x >> 6], v[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += buf[turn][i][w];
      v[i] = s;
    }
    turn ^= 1;
  }
}

// A row over TPR lanes: piece c of lane t is V elements from column (c TPR + t) V.  Where the width is no
// multiple, the piece that would pass its end ends with the row instead and repeats elements of its
// neighbour: loaded and stored twice with the same values, counted once (mine).
template <class T, int V_, int TPR, int NC, bool EXACT>
struct Row {
  static constexpr int V = V_;
  static constexpr int BLK = TPR > 256 ? TPR : 256;
  static constexpr int SLOTS = BLK / TPR;   // rows that a workgroup holds at a time
  float v[NC][V];

  static __device__ __forceinline__ int first(int c) { return (c * TPR + (int)(threadIdx.x & (TPR - 1))) * V; }
  static __device__ __forceinline__ int col(int c, int width) { return EXACT ? first(c) : min(first(c), width - V); }
  static __device__ __forceinline__ bool mine(int c, int j, int width) { return EXACT || first(c) <= col(c, width) + j; }
  __device__ __forceinline__ void load(const void* p, int64_t at, int width) {
#pragma unroll
    for (int c = 0; c < NC; ++c) load_piece<T, V>((const T*)p + at + col(c, width), v[c]);
  }
  // the same in two steps: the bits, and later their values
  struct Bits { T t[NC][V]; };
  static __device__ __forceinline__ void load_bits(Bits& b, const void* p, int64_t at, int width) {
#pragma unroll
    for (int c = 0; c < NC; ++c) __builtin_memcpy(b.t[c], (const T*)p + at + col(c, width), sizeof(T) * V);
  }
  __device__ __forceinline__ void set(const Bits& b) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) v[c][j] = (float)b.t[c][j];
  }
  __device__ __forceinline__ void load_param(const void* p, int type, int64_t at, int width, float fill) {
    if (p == nullptr) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) v[c][j] = fill;
      return;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) load_typed<V>(p, type, at + col(c, width), v[c]);
  }
  __device__ __forceinline__ void store(void* p, int64_t at, int width) const {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (EXACT || first(c) < width) store_piece<T, V>((T*)p + at + col(c, width), v[c]);
  }
};

__device__ __forceinline__ int64_t gate_of(int64_t row, int64_t per_gate) {
  if (per_gate == 1) return row;
  if (((row | per_gate) >> 32) == 0) return (uint32_t)row / (uint32_t)per_gate;
  return row / per_gate;
}

// mean and 1 / sqrt(var + eps) of a row in registers
template <class R, int TPR, int NC>
__device__ __forceinline__ void statistics(const R& r, int kind, int width, float inv_d, float eps, float& mean, float& rstd,
                                           float (*buf)[2][16], int& turn) {
  mean = 0.f;
  rstd = 1.f;
  if (kind == NFI_NORM_NONE) return;
  if (kind == NFI_NORM_LAYER) {
    float s[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < R::V; ++j) s[0] += r.mine(c, j, width) ? r.v[c][j] : 0.f;
    row_sums<TPR, 1>(s, buf, turn);
    mean = s[0] * inv_d;
  }
  float s[1] = {0.f};
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int j = 0; j < R::V; ++j) {
      const float d = r.mine(c, j, width) ? r.v[c][j] - mean : 0.f;
      s[0] = fmaf(d, d, s[0]);
    }
  row_sums<TPR, 1>(s, buf, turn);
  rstd = 1.f / sqrtf(fmaf(s[0], inv_d, eps));
}

template <class T, int V, int TPR, int NC, bool EXACT>
__global__ void __launch_bounds__((TPR > 256 ? TPR : 256)) resnorm_fwd(const nfi_resnorm_args a) {
  typedef Row<T, V, TPR, NC, EXACT> R;
  __shared__ float buf[2][2][16];
  int turn = 0;
  const int width = a.width;
  const float inv_d = 1.f / (float)width;
  const int64_t per_gate = a.groups ? a.rows / a.groups : 1;
  // the parameters are held in registers over the rows where that is cheap
  const bool keep = NC * R::V <= 8 && !a.affine_groups;
  R w, b, w2, b2;
  if (keep) {
    w.load_param(a.weight, a.param_dtype, 0, width, 1.f);
    b.load_param(a.bias, a.param_dtype, 0, width, 0.f);
    if (a.next_norm) {
      w2.load_param(a.next_weight, a.param_dtype, 0, width, 1.f);
      b2.load_param(a.next_bias, a.param_dtype, 0, width, 0.f);
    }
  }
  for (int64_t row = (int64_t)blockIdx.x * R::SLOTS + threadIdx.x / TPR; row < a.rows; row += (int64_t)gridDim.x * R::SLOTS) {
    const int64_t at = row * width;
    R x, res, gate;
    x.load(a.h, at, width);
    if (a.residual) res.load(a.residual, at, width);
    const int64_t group = a.groups > 1 ? gate_of(row, per_gate) : 0, param_at = a.affine_groups ? group * width : 0;
    if (a.gate) gate.load_param(a.gate, a.gate_dtype, group * width, width, 1.f);
    if (!keep) {
      w.load_param(a.weight, a.param_dtype, param_at, width, 1.f);
      b.load_param(a.bias, a.param_dtype, param_at, width, 0.f);
    }
    float mean, rstd, mean2 = 0.f, rstd2 = 1.f;
    statistics<R, TPR, NC>(x, a.norm, width, inv_d, a.eps, mean, rstd, buf, turn);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < R::V; ++j) {
        const float u = fmaf((x.v[c][j] - mean) * rstd, w.v[c][j], b.v[c][j]);
        float s = u > 0.f ? u : u * a.slope;
        if (a.gate) s *= gate.v[c][j];
        if (a.residual) s += res.v[c][j];
        x.v[c][j] = s * a.scale;
      }
    x.store(a.x, at, width);
    if (a.next_norm) {
      statistics<R, TPR, NC>(x, a.next_norm, width, inv_d, a.eps, mean2, rstd2, buf, turn);
      if (!keep) {
        w2.load_param(a.next_weight, a.param_dtype, param_at, width, 1.f);
        b2.load_param(a.next_bias, a.param_dtype, param_at, width, 0.f);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < R::V; ++j) x.v[c][j] = fmaf((x.v[c][j] - mean2) * rstd2, w2.v[c][j], b2.v[c][j]);
      x.store(a.y, at, width);
    }
    if (a.stats && (threadIdx.x & (TPR - 1)) == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(mean, rstd, mean2, rstd2);
  }
}

// Rows in segments: a segment is a piece of one group's rows (`splits` pieces each), or all rows in `splits` pieces
// without groups.  A workgroup takes `per` consecutive segments; with several pieces for each group per is 1 and the
// group's sums leave as partials, otherwise the workgroup holds whole groups.
struct Plan {
  int64_t segments, per, rows_per_gate, rows_per_split;
  int splits, blocks;
};

// (a gate for each row alone needs no sum)
__host__ inline int64_t summed_groups(int64_t rows, int64_t groups, bool affine) { return groups > 0 && (groups < rows || affine) ? groups : 1; }

__host__ inline Plan make_plan(int64_t rows, int64_t groups, bool affine, int width, int slots) {
  Plan p;
  const int64_t blocks = blocks_of(width);
  const int64_t g = summed_groups(rows, groups, affine);
  p.rows_per_gate = rows / g;
  const int64_t want = std::max<int64_t>(1, blocks / g);
  const int64_t most = (p.rows_per_gate + slots - 1) / slots;
  p.splits = (int)std::min(want, most);
  p.rows_per_split = (p.rows_per_gate + p.splits - 1) / p.splits;
  p.segments = g * p.splits;
  p.per = p.splits > 1 ? 1 : (p.segments + blocks - 1) / blocks;
  p.blocks = (int)((p.segments + p.per - 1) / p.per);
  return p;
}

// sums acc over the workgroup's SLOTS rows and hands column sums to put(col, value)
template <class R, int TPR, int NC, class F>
__device__ __forceinline__ void slots_sum(const float (&acc)[NC][R::V], float* lds, int width, F put) {
  if constexpr (R::SLOTS == 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < R::V; ++j)
        if (R::mine(c, j, width)) put(R::col(c, width) + j, acc[c][j]);
  } else {
    constexpr int W = TPR * NC * R::V;   // columns that the lanes of a row hold
    __syncthreads();
    const int slot = threadIdx.x / TPR;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < R::V; ++j)
        if (R::mine(c, j, width)) lds[slot * W + R::col(c, width) + j] = acc[c][j];
    __syncthreads();
    for (int col = threadIdx.x; col < width; col += R::BLK) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < R::SLOTS; ++k) s += lds[k * W + col];
      put(col, s);
    }
  }
}

template <class T, int V, int TPR, int NC, bool EXACT>
__global__ void __launch_bounds__((TPR > 256 ? TPR : 256)) resnorm_bwd(const nfi_resnorm_args a, const Plan p) {
  typedef Row<T, V, TPR, NC, EXACT> R;
  __shared__ float buf[2][2][16];
  __shared__ float lds[R::SLOTS == 1 ? 1 : R::BLK * NC * R::V];
  int turn = 0;
  const int width = a.width;
  const float inv_d = 1.f / (float)width;
  const bool layer = a.norm == NFI_NORM_LAYER, layer2 = a.next_norm == NFI_NORM_LAYER;
  const bool row_gate = a.groups == a.rows && a.groups > 0 && !a.affine_groups;
  const bool gate_sum = a.gate && a.dgate && !row_gate;
  float acc[4][NC][R::V], accg[NC][R::V];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int j = 0; j < R::V; ++j) {
      acc[0][c][j] = acc[1][c][j] = acc[2][c][j] = acc[3][c][j] = 0.f;
      accg[c][j] = 0.f;
    }
  // up to one piece of 16 bytes a lane there are registers for the next row's bits, which arrive while a row is worked on, and for the
  // parameters that the rows share (16,384 rows of 1024 bf16, together: 88 -> 58 us)
  constexpr bool AHEAD = NC * R::V * (int)sizeof(T) <= 16 && TPR < 1024;
  const bool keep = AHEAD && !a.affine_groups;
  R gate, w, b, w2;
  auto load_params = [&](int64_t at) {
    w.load_param(a.weight, a.param_dtype, at, width, 1.f);
    b.load_param(a.bias, a.param_dtype, at, width, 0.f);
    if (a.gy) w2.load_param(a.next_weight, a.param_dtype, at, width, 1.f);
  };
  if (keep) load_params(0);
  const int64_t last = min((int64_t)(blockIdx.x + 1) * p.per, p.segments);
  for (int64_t seg = (int64_t)blockIdx.x * p.per; seg < last; ++seg) {
    const int64_t gi = seg / p.splits, piece = seg - gi * p.splits;
    const int64_t r0 = gi * p.rows_per_gate + piece * p.rows_per_split;
    const int64_t r1 = min(r0 + p.rows_per_split, (gi + 1) * p.rows_per_gate);
    const bool keep_gate = AHEAD && a.gate && !row_gate;
    if (keep_gate) gate.load_param(a.gate, a.gate_dtype, gi * width, width, 1.f);
    typename R::Bits bh, bres, bg, bgy;
    float4 next_st;
    auto ahead = [&](int64_t row) {
      const int64_t at = row * width;
      R::load_bits(bh, a.h, at, width);
      if (a.residual) R::load_bits(bres, a.residual, at, width);
      if (a.gx) R::load_bits(bg, a.gx, at, width);
      if (a.gy) R::load_bits(bgy, a.gy, at, width);
      next_st = *reinterpret_cast<const float4*>(a.stats + 4 * row);
    };
    const int64_t mine = r0 + threadIdx.x / TPR;
    if (AHEAD && mine < r1) ahead(mine);
    for (int64_t row = mine; row < r1; row += R::SLOTS) {
      const int64_t at = row * width;
      R h, res, g, gy;
      if constexpr (!AHEAD) {
        R none;   // (nothing is carried from row to row)
        gate = w = b = w2 = none;
        h.load(a.h, at, width);
        if (a.residual) res.load(a.residual, at, width);
        if (a.gx) g.load(a.gx, at, width);
        if (a.gy) gy.load(a.gy, at, width);
        next_st = *reinterpret_cast<const float4*>(a.stats + 4 * row);
      } else {
        h.set(bh);
        if (a.residual) res.set(bres);
        if (a.gx) g.set(bg);
        if (a.gy) gy.set(bgy);
      }
      const float4 st = next_st;
      if (AHEAD && row + R::SLOTS < r1) ahead(row + R::SLOTS);
      if (a.gate && !keep_gate) gate.load_param(a.gate, a.gate_dtype, (row_gate ? row : gi) * width, width, 1.f);
      if (!keep) load_params(a.affine_groups ? gi * width : 0);
      // h becomes n, res becomes v (the gated value is scale (res + gate v))
      float s[2] = {0.f, 0.f};
      R m2, &m_of = AHEAD ? m2 : w2;   // (w2 is not needed again, but for the next row)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < R::V; ++j) {
          const bool ok = R::mine(c, j, width);
          const float n = (h.v[c][j] - st.x) * st.y;
          const float u = fmaf(n, w.v[c][j], b.v[c][j]);
          const float v = u > 0.f ? u : u * a.slope;
          float x = a.gate ? v * gate.v[c][j] : v;
          if (a.residual) x += res.v[c][j];
          x *= a.scale;
          h.v[c][j] = n;
          res.v[c][j] = v;
          if (a.gy) {
            const float m = (x - st.z) * st.w;
            const float q = gy.v[c][j];
            acc[2][c][j] = fmaf(q, m, acc[2][c][j]);
            acc[3][c][j] += q;
            const float qw = q * w2.v[c][j];
            gy.v[c][j] = qw;
            m_of.v[c][j] = m;
            s[0] += ok ? qw : 0.f;
            s[1] += ok ? qw * m : 0.f;
          }
        }
      if (a.gy) {
        row_sums<TPR, 2>(s, buf, turn);
        s[0] = layer2 ? s[0] * inv_d : 0.f;
        s[1] *= inv_d;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < R::V; ++j) {
            const float q = st.w * (gy.v[c][j] - s[0] - m_of.v[c][j] * s[1]);
            g.v[c][j] = a.gx ? g.v[c][j] + q : q;
          }
      }
      s[0] = s[1] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < R::V; ++j) {
          const bool ok = R::mine(c, j, width);
          const float gs = g.v[c][j] * a.scale;
          g.v[c][j] = gs;   // d residual
          const float dg = gs * res.v[c][j];
          if (row_gate) gy.v[c][j] = dg;
          else accg[c][j] += dg;
          const float n = h.v[c][j];
          const float u = fmaf(n, w.v[c][j], b.v[c][j]);
          float gu = a.gate ? gs * gate.v[c][j] : gs;
          gu = u > 0.f ? gu : gu * a.slope;
          acc[0][c][j] = fmaf(gu, n, acc[0][c][j]);
          acc[1][c][j] += gu;
          const float q = gu * w.v[c][j];
          res.v[c][j] = q;
          s[0] += ok ? q : 0.f;   // (repeated elements are computed like their twins, and counted once)
          s[1] += ok ? q * n : 0.f;
        }
      if (a.dresidual) g.store(a.dresidual, at, width);
      if (row_gate && a.dgate) {
        if (a.gate_dtype == TypeCode<T>::V) gy.store(a.dgate, at, width);
        else
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < R::V; ++j)
              if (R::mine(c, j, width)) store_typed(a.dgate, a.gate_dtype, at + R::col(c, width) + j, gy.v[c][j]);
      }
      if (a.dh) {
        if (a.norm != NFI_NORM_NONE) {
          row_sums<TPR, 2>(s, buf, turn);
          s[0] = layer ? s[0] * inv_d : 0.f;
          s[1] *= inv_d;
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < R::V; ++j) res.v[c][j] = st.y * (res.v[c][j] - s[0] - h.v[c][j] * s[1]);
        }
        res.store(a.dh, at, width);
      }
    }
    // a whole group: its sums are final
    if (p.splits == 1 && gate_sum) {
      slots_sum<R, TPR, NC>(accg, lds, width, [&](int col, float v) { store_typed(a.dgate, a.gate_dtype, gi * width + col, v); });
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < R::V; ++j) accg[c][j] = 0.f;
    }
    if (p.splits == 1 && a.affine_groups) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        void* out = k == 0 ? a.dweight : k == 1 ? a.dbias : k == 2 ? a.dnext_weight : a.dnext_bias;
        if (out) slots_sum<R, TPR, NC>(acc[k], lds, width, [&](int col, float v) { store_typed(out, a.param_dtype, gi * width + col, v); });
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < R::V; ++j) acc[k][c][j] = 0.f;
      }
    }
  }
  float* part = a.work + (int64_t)blockIdx.x * PARAMS * width;
  if (p.splits > 1 || !a.affine_groups) {
    if (a.dweight) slots_sum<R, TPR, NC>(acc[0], lds, width, [&](int col, float v) { part[col] = v; });
    if (a.dbias) slots_sum<R, TPR, NC>(acc[1], lds, width, [&](int col, float v) { part[width + col] = v; });
    if (a.dnext_weight) slots_sum<R, TPR, NC>(acc[2], lds, width, [&](int col, float v) { part[2 * width + col] = v; });
    if (a.dnext_bias) slots_sum<R, TPR, NC>(acc[3], lds, width, [&](int col, float v) { part[3 * width + col] = v; });
  }
  if (gate_sum && p.splits > 1) slots_sum<R, TPR, NC>(accg, lds, width, [&](int col, float v) { part[4 * width + col] = v; });
}

// The workgroups' partials summed in their order, COLS columns x 1024 / COLS slices of workgroups at a time: blockIdx.y the
// parameter (4: the gate), blockIdx.z the group (its own workgroups), or 0 for parameters of all rows
template <int COLS>
__global__ void __launch_bounds__(1024) resnorm_join(const nfi_resnorm_args a, const Plan p) {
  constexpr int SLICES = 1024 / COLS;
  __shared__ float lds[SLICES][COLS + 1];
  const int which = blockIdx.y;
  void* out = which == 0 ? a.dweight : which == 1 ? a.dbias : which == 2 ? a.dnext_weight : which == 3 ? a.dnext_bias : a.dgate;
  const bool grouped = which == 4 || a.affine_groups;
  const int64_t gi = blockIdx.z;
  if (out == nullptr || (!grouped && gi > 0) || (grouped && p.splits == 1)) return;
  const int first = grouped ? (int)(gi * p.splits) : 0, count = grouped ? p.splits : p.blocks;
  const int col = blockIdx.x * COLS + (threadIdx.x & (COLS - 1)), slice = threadIdx.x / COLS;
  float s = 0.f;
  if (col < a.width) {
    const float* q = a.work + ((int64_t)first * PARAMS + which) * a.width + col;
#pragma unroll 8
    for (int k = slice; k < count; k += SLICES) s += q[(int64_t)k * PARAMS * a.width];
  }
  lds[slice][threadIdx.x & (COLS - 1)] = s;
  __syncthreads();
  if (slice == 0 && col < a.width) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < SLICES; ++k) t += lds[k][threadIdx.x & (COLS - 1)];
    store_typed(out, which < 4 ? a.param_dtype : a.gate_dtype, gi * a.width + col, t);
  }
}

enum Way { BOTH, FORWARD, BACKWARD };

template <class T, int V, int TPR, int NC, bool EXACT, Way WAY>
static void launch(const nfi_resnorm_args& a, bool backward, hipStream_t s) {
  typedef Row<T, V, TPR, NC, EXACT> R;
  if constexpr (WAY != BACKWARD) {
    if (!backward) {
      const int64_t need = (a.rows + R::SLOTS - 1) / R::SLOTS;
      resnorm_fwd<T, V, TPR, NC, EXACT><<<(unsigned)std::min<int64_t>(need, 8192), R::BLK, 0, s>>>(a);
      return;
    }
  }
  if constexpr (WAY == FORWARD) return;
  else {
  const Plan p = make_plan(a.rows, a.groups, a.affine_groups, a.width, R::SLOTS);
  resnorm_bwd<T, V, TPR, NC, EXACT><<<(unsigned)p.blocks, R::BLK, 0, s>>>(a, p);
  const bool params = (a.dweight || a.dbias || a.dnext_weight || a.dnext_bias) && (p.splits > 1 || !a.affine_groups);
  const bool gate = a.dgate && (a.groups < a.rows || a.affine_groups) && p.splits > 1;
  const bool each = gate || (params && a.affine_groups);   // (a group's own sums: fewer groups than workgroups)
  if (params || gate) {
    // (few columns need every slice, many want whole lines: 256 partial results of 8192 columns, 37 -> 13 us)
    const int cols = a.width >= 512 ? 64 : 16;
    const dim3 grid((unsigned)((a.width + cols - 1) / cols), gate ? 5 : 4, (unsigned)(each ? a.groups : 1));
    if (cols == 64) resnorm_join<64><<<grid, 1024, 0, s>>>(a, p);
    else resnorm_join<16><<<grid, 1024, 0, s>>>(a, p);
  }
  }
}

template <class T, int V, int TPR, int NC, Way WAY = BOTH>
static void pick_exact(const nfi_resnorm_args& a, bool backward, hipStream_t s) {
  if (a.width == TPR * NC * V) launch<T, V, TPR, NC, true, WAY>(a, backward, s);
  else launch<T, V, TPR, NC, false, WAY>(a, backward, s);
}

template <class T>
static void dispatch(const nfi_resnorm_args& a, bool backward, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int n = (a.width + V - 1) / V;
  if (a.width < V) launch<T, 1, 8, 1, false, BOTH>(a, backward, s);   // (a piece does not fit into the row)
  else if (n <= 8) pick_exact<T, V, 8, 1>(a, backward, s);
  else if (n <= 16) pick_exact<T, V, 16, 1>(a, backward, s);
  else if (n <= 32) pick_exact<T, V, 32, 1>(a, backward, s);
  else if (n <= 64) pick_exact<T, V, 64, 1>(a, backward, s);
  else if constexpr (sizeof(T) == 2) {
    // the backward of wide 16-bit rows: a lane's registers hold a row's four tensors, so few elements to a lane, in more waves
    // (16,384 rows of 1024: two pieces of 8 in one wave 83 us, one of 4 in four waves 57; 4096 rows of 4096: two of 8 in four
    // waves 101 us, one in eight 49; 2048 rows of 8192: two in eight 117, one in sixteen 79); the forward holds less, and wants the wider loads (30 us, and 37)
    if (n <= 128) {
      if (backward) pick_exact<T, 4, 256, 1, BACKWARD>(a, backward, s);
      else pick_exact<T, V, 64, 2, FORWARD>(a, backward, s);
    } else if (n <= 256) {
      pick_exact<T, V, 256, 1>(a, backward, s);
    } else if (n <= 512) {
      if (backward) pick_exact<T, V, 512, 1, BACKWARD>(a, backward, s);
      else pick_exact<T, V, 256, 2, FORWARD>(a, backward, s);
    } else {
      if (backward) pick_exact<T, V, 1024, 1, BACKWARD>(a, backward, s);
      else pick_exact<T, V, 512, 2, FORWARD>(a, backward, s);
    }
  } else {
    if (n <= 128) pick_exact<T, V, 64, 2>(a, backward, s);
    else if (n <= 256) pick_exact<T, V, 256, 1>(a, backward, s);
    else if (n <= 512) pick_exact<T, V, 256, 2>(a, backward, s);
    else if (n <= 1024) pick_exact<T, V, 512, 2>(a, backward, s);
    else if (backward) pick_exact<T, V, 1024, 2, BACKWARD>(a, backward, s);   // (2048 rows of 8192: four pieces in eight waves 179 us, two in sixteen 127)
    else pick_exact<T, V, 512, 4, FORWARD>(a, backward, s);
  }
}

static int check(const nfi_resnorm_args* a, const char* what) {
  NFI_REQUIRE(a && a->h, "%s: null input", what);
  NFI_REQUIRE(a->rows > 0 && a->width > 0 && a->width <= NFI_RESNORM_MAX_WIDTH, "%s: rows %lld, width %d (1 .. %d)", what,
              (long long)a->rows, a->width, NFI_RESNORM_MAX_WIDTH);
  NFI_REQUIRE(type_ok(a->dtype) && type_ok(a->param_dtype) && type_ok(a->gate_dtype), "%s: bad type", what);
  NFI_REQUIRE(a->norm >= 0 && a->norm <= 2 && a->next_norm >= 0 && a->next_norm <= 2, "%s: bad norm kind", what);
  NFI_REQUIRE(a->groups >= 0 && ((a->gate == nullptr && !a->affine_groups) || a->groups > 0) && (a->groups == 0 || a->rows % a->groups == 0),
              "%s: %lld groups of %lld rows", what, (long long)a->groups, (long long)a->rows);
  NFI_REQUIRE(a->eps >= 0.f, "%s: eps %g", what, (double)a->eps);
  return NFI_OK;
}

static void run(const nfi_resnorm_args& a, bool backward, hipStream_t s) {
  if (a.dtype == NFI_F32) dispatch<float>(a, backward, s);
  else if (a.dtype == NFI_BF16) dispatch<bf16_t>(a, backward, s);
  else dispatch<f16_t>(a, backward, s);
}

}  // namespace learn
}  // namespace nfi

using namespace nfi::learn;

extern "C" {

int64_t nfi_resnorm_work_bytes(int64_t rows, int64_t groups, int32_t affine_groups, int32_t width) {
  if (rows <= 0 || groups < 0 || width <= 0) return 0;
  // (the plan's workgroups, whatever number of rows one holds)
  const int64_t g = summed_groups(rows, groups, affine_groups != 0);
  const int64_t most = blocks_of(width), blocks = g >= most ? most : g * std::max<int64_t>(1, most / g);
  return blocks * PARAMS * (int64_t)width * 4;
}

int32_t nfi_resnorm_forward(const nfi_resnorm_args* a, void* stream) {
  const int e = check(a, "resnorm_forward");
  if (e) return e;
  NFI_REQUIRE(a->x && (a->y != nullptr || a->next_norm == NFI_NORM_NONE), "resnorm_forward: null output");
  run(*a, false, (hipStream_t)stream);
  NFI_CHECK_LAUNCH("resnorm_forward");
  return NFI_OK;
}

int32_t nfi_resnorm_backward(const nfi_resnorm_args* a, void* stream) {
  const int e = check(a, "resnorm_backward");
  if (e) return e;
  NFI_REQUIRE(a->stats && a->work, "resnorm_backward: null statistics or work buffer");
  NFI_REQUIRE(a->gx || a->gy, "resnorm_backward: no gradient");
  NFI_REQUIRE(!a->gy || a->next_norm != NFI_NORM_NONE, "resnorm_backward: gy without a next norm");
  NFI_REQUIRE(!a->dgate || a->gate, "resnorm_backward: dgate without a gate");
  run(*a, true, (hipStream_t)stream);
  NFI_CHECK_LAUNCH("resnorm_backward");
  return NFI_OK;
}

}  // extern "C"
