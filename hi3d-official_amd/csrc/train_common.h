// What the training kernels share: element types, vector loads of any element alignment, sums over a group of lanes.
#pragma once
#include "common.h"

namespace {

typedef _Float16 half_t;
struct bf16_t { unsigned short u; };

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int VEC = 4, CODE = HI3D_F32;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<half_t> {
  static constexpr int VEC = 8, CODE = HI3D_F16;
  static __device__ __forceinline__ float get(half_t v) { return (float)v; }
  static __device__ __forceinline__ half_t put(float v) { return (half_t)v; }      // round to nearest even, overflow to infinity
};
template <> struct Elem<bf16_t> {
  static constexpr int VEC = 8, CODE = HI3D_BF16;
  static __device__ __forceinline__ float get(bf16_t v) { return bf16_to_f32(v.u); }
  static __device__ __forceinline__ bf16_t put(float v) { return bf16_t{f32_to_bf16(v)}; }
};

// N elements in one access.  The alignment asked for is the element's own: gfx950 takes global vector accesses at any byte
// address (unaligned access mode), so views at odd offsets and rows of odd length use the same 16-byte loads.
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[N]; };

// The first n of N elements of a row's vector (n <= 0: none), the others zero, as raw bits: a full vector is one masked load whose
// result nothing waits for until it is unpacked, so that a row's loads are all in flight together.
template <typename T, int N>
__device__ __forceinline__ void fetch(const T* p, int n, Pack<T, N>& k) {
  k = Pack<T, N>{};
  if (n >= N) k = *(const Pack<T, N>*)p;
  else if (n > 0) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) k.v[j] = p[j];
  }
}
template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& k, float (&f)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = Elem<T>::get(k.v[j]);
}
template <typename T, int N>
__device__ __forceinline__ void store_some(T* p, int n, const float (&f)[N]) {
  if (n >= N) {
    Pack<T, N> k;
#pragma unroll
    for (int j = 0; j < N; ++j) k.v[j] = Elem<T>::put(f[j]);
    *(Pack<T, N>*)p = k;
  } else if (n > 0) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) p[j] = Elem<T>::put(f[j]);
  }
}
// elements [e, e + n) of a tensor whose type is known at run time only (weights: read once per block)
template <int N>
__device__ __forceinline__ void load_vec_as(const void* p, int code, int e, int n, float (&f)[N]) {
  if (code == HI3D_F32) { Pack<float, N> k; fetch((const float*)p + e, n, k); unpack(k, f); }
  else if (code == HI3D_BF16) { Pack<bf16_t, N> k; fetch((const bf16_t*)p + e, n, k); unpack(k, f); }
  else { Pack<half_t, N> k; fetch((const half_t*)p + e, n, k); unpack(k, f); }
}

// one element of a tensor whose type is known at run time only (weights, biases: read or written once per block)
__device__ __forceinline__ float load_as(const void* p, int code, long i) {
  if (code == HI3D_F32) return ((const float*)p)[i];
  if (code == HI3D_BF16) return bf16_to_f32(((const unsigned short*)p)[i]);
  return (float)((const half_t*)p)[i];
}
__device__ __forceinline__ void store_as(void* p, int code, long i, float v) {
  if (code == HI3D_F32) ((float*)p)[i] = v;
  else if (code == HI3D_BF16) ((unsigned short*)p)[i] = f32_to_bf16(v);
  else ((half_t*)p)[i] = (half_t)v;
}

// the sum of v over the aligned group of L lanes that this lane is in, in every one of them
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

}  // namespace

// o0[0, C) and o1[0, width - C) = the column sums of part[nblk][width], in a fixed order (norm_train.hip)
int hi3d_column_reduce(const float* part, void* o0, void* o1, int code0, int code1, int nblk, int C, int width, hipStream_t st);

namespace {

inline bool hi3d_known_dtype(int c) { return c == HI3D_F32 || c == HI3D_BF16 || c == HI3D_F16; }
inline int hi3d_dtype_size(int c) { return c == HI3D_F32 ? 4 : 2; }

}  // namespace
