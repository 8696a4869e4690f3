// What the training kernels share: element types, vector loads of any element alignment, sums over a group of lanes.
#pragma once
#include "common.h"
#include <type_traits>

namespace {

typedef _Float16 half_t;
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
struct bf16_t { unsigned short u; };

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<half_t> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(half_t v) { return (float)v; }
  static __device__ __forceinline__ half_t put(float v) { return (half_t)v; }      // round to nearest even, overflow to infinity
};
template <> struct Elem<bf16_t> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(bf16_t v) { return bf16_to_f32(v.u); }
  static __device__ __forceinline__ bf16_t put(float v) { return bf16_t{f32_to_bf16(v)}; }
};

// N elements in one access, as raw 32-bit words.  The alignment asked for is the element's own: gfx950 takes global vector accesses at any
// byte address (unaligned access mode), so views at odd offsets and rows of odd length use the same 16-byte loads.
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  static constexpr int W = N * (int)sizeof(T) / 4;
  static_assert(W * 4 == N * (int)sizeof(T), "whole words");
  unsigned w[W];
};

template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& k, float (&f)[N]) {
#pragma unroll
  for (int j = 0; j < Pack<T, N>::W; ++j) {
    if constexpr (sizeof(T) == 4) f[j] = __uint_as_float(k.w[j]);
    else if constexpr (std::is_same<T, bf16_t>::value) { f[2 * j] = __uint_as_float(k.w[j] << 16); f[2 * j + 1] = __uint_as_float(k.w[j] & 0xffff0000u); }
    else {
      const half2_t h = __builtin_bit_cast(half2_t, k.w[j]);
      f[2 * j] = (float)h[0]; f[2 * j + 1] = (float)h[1];
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack(const float (&f)[N]) {
  Pack<T, N> k;
#pragma unroll
  for (int j = 0; j < Pack<T, N>::W; ++j) {
    if constexpr (sizeof(T) == 4) k.w[j] = __float_as_uint(f[j]);
    else if constexpr (std::is_same<T, bf16_t>::value) k.w[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
    else k.w[j] = __builtin_bit_cast(unsigned, half2_t{(half_t)f[2 * j], (half_t)f[2 * j + 1]});
  }
  return k;
}
// k moved down by s of its N elements (0 <= s < N), zeros behind
template <typename T, int N>
__device__ __forceinline__ void shift_down(Pack<T, N>& k, int s) {
  constexpr int W = Pack<T, N>::W, PER = 4 / (int)sizeof(T);
#pragma unroll
  for (int step = W / 2; step > 0; step >>= 1) {
    const bool on = s & (step * PER);
#pragma unroll
    for (int j = 0; j < W; ++j) k.w[j] = on ? (j + step < W ? k.w[j + step] : 0u) : k.w[j];
  }
  if constexpr (PER == 2) {
    const bool on = s & 1;
#pragma unroll
    for (int j = 0; j < W; ++j) k.w[j] = on ? (k.w[j] >> 16) | (j + 1 < W ? k.w[j + 1] << 16 : 0u) : k.w[j];
  }
}
// The first n of N elements at p (n <= 0: none), the others zero.  A vector that the row's end cuts is loaded so that it ends there, and moved down
// afterwards: one access, nothing is read outside the row; `before` elements precede p in its row, and where those are too few the elements come one by one.
template <typename T, int N>
__device__ __forceinline__ void fetch(const T* p, int n, long before, Pack<T, N>& k) {
#pragma unroll
  for (int j = 0; j < Pack<T, N>::W; ++j) k.w[j] = 0;
  if (n >= N) k = *(const Pack<T, N>*)p;
  else if (n > 0) {
    Pack<T, N> t = {};
    if (before >= N - n) {
      t = *(const Pack<T, N>*)(p - (N - n));
      shift_down(t, N - n);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) {
          if constexpr (sizeof(T) == 4) t.w[j] = *(const unsigned*)(p + j);
          else t.w[j / 2] |= (unsigned)*(const unsigned short*)(p + j) << (16 * (j & 1));
        }
    }
#pragma unroll
    for (int j = 0; j < Pack<T, N>::W; ++j) k.w[j] = t.w[j];
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_some(T* p, int n, const float (&f)[N]) {
  if (n >= N) *(Pack<T, N>*)p = pack<T, N>(f);
  else if (n > 0) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) p[j] = Elem<T>::put(f[j]);
  }
}
// elements [e, e + n) of a tensor whose type is known at run time only (weights: read once per block)
template <int N>
__device__ __forceinline__ void load_vec_as(const void* p, int code, int e, int n, float (&f)[N]) {
  if (code == HI3D_F32) { Pack<float, N> k; fetch((const float*)p + e, n, e, k); unpack(k, f); }
  else if (code == HI3D_BF16) { Pack<bf16_t, N> k; fetch((const bf16_t*)p + e, n, e, k); unpack(k, f); }
  else { Pack<half_t, N> k; fetch((const half_t*)p + e, n, e, k); unpack(k, f); }
}

// one element of a tensor whose type is known at run time only (gradients of weights: written once)
__device__ __forceinline__ void store_as(void* p, int code, long i, float v) {
  if (code == HI3D_F32) ((float*)p)[i] = v;
  else if (code == HI3D_BF16) ((unsigned short*)p)[i] = f32_to_bf16(v);
  else ((half_t*)p)[i] = (half_t)v;
}

// The sum of v over the aligned group of L lanes that this lane is in, in every one of them: lane exchanges inside the vector unit (quad
// permutations, mirrors of 8 and 16 lanes, swaps of rows and of halves), no LDS round trip.
template <int CTRL>
__device__ __forceinline__ float plus_dpp(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  static_assert(L == 8 || L == 16 || L == 32 || L == 64, "lanes of a row");
  v = plus_dpp<0xB1>(v);                       // lane ^ 1
  v = plus_dpp<0x4E>(v);                       // lane ^ 2
  v = plus_dpp<0x141>(v);                      // the other four of 8
  if constexpr (L >= 16) v = plus_dpp<0x140>(v);
  if constexpr (L >= 32) {
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (L >= 64) {
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

}  // namespace

// o0[0, C) and o1[0, width - C) = the column sums of part[nblk][width], in a fixed order (norm_train.hip)
int hi3d_column_reduce(const float* part, void* o0, void* o1, int code0, int code1, int nblk, int C, int width, hipStream_t st);

namespace {

inline bool hi3d_known_dtype(int c) { return c == HI3D_F32 || c == HI3D_BF16 || c == HI3D_F16; }

}  // namespace
