// Shared by the operators of include/nfi_learn.h: element types and 16-byte pieces of rows.
#pragma once
#include "nfi_common.h"
#include "nfi_host.h"
#include "../../include/nfi_learn.h"

namespace nfi {
namespace learn {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

template <class T> struct TypeCode;
template <> struct TypeCode<float> { static constexpr int V = NFI_F32; };
template <> struct TypeCode<bf16_t> { static constexpr int V = NFI_BF16; };
template <> struct TypeCode<f16_t> { static constexpr int V = NFI_F16; };

__host__ __device__ __forceinline__ int type_bytes(int t) { return t == NFI_F32 ? 4 : 2; }
inline bool type_ok(int t) { return t == NFI_F32 || t == NFI_BF16 || t == NFI_F16; }

// V elements at p; rows need no alignment beyond their element's (global loads and stores of 16 bytes take any
// address on this target)
template <class T, int V>
__device__ __forceinline__ void load_piece(const T* __restrict__ p, float (&v)[V]) {
  T t[V];
  __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = (float)t[j];
}

template <class T, int V>
__device__ __forceinline__ void store_piece(T* __restrict__ p, const float (&v)[V]) {
  T t[V];
#pragma unroll
  for (int j = 0; j < V; ++j) t[j] = (T)v[j];
  __builtin_memcpy(p, t, sizeof(t));
}

// the same from a buffer whose type is known at run time (parameters; the branch is uniform)
template <int V>
__device__ __forceinline__ void load_typed(const void* p, int type, int64_t at, float (&v)[V]) {
  if (type == NFI_F32) load_piece<float, V>((const float*)p + at, v);
  else if (type == NFI_BF16) load_piece<bf16_t, V>((const bf16_t*)p + at, v);
  else load_piece<f16_t, V>((const f16_t*)p + at, v);
}

__device__ __forceinline__ void store_typed(void* p, int type, int64_t at, float v) {
  if (type == NFI_F32) ((float*)p)[at] = v;
  else if (type == NFI_BF16) ((bf16_t*)p)[at] = (bf16_t)v;
  else ((f16_t*)p)[at] = (f16_t)v;
}

}  // namespace learn
}  // namespace nfi
