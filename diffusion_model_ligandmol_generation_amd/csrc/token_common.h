// Element types, 16-byte packs and block reductions shared by the token kernels (embed.hip, tokens.hip).
#pragma once
#include <type_traits>
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// A pack is the 16 bytes one lane moves per memory instruction: 4 fp32 or 8 half-precision elements.  Rows of an odd
// number of elements start anywhere, so a pack is only as aligned as its element: global_load / store_dwordx4 take any
// address on this chip, and one that straddles a cache line costs one more line.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct Pack {
  enum { N = 16 / sizeof(T), PER = 4 / sizeof(T) };   // elements of a pack, of one 32-bit register
  typedef typename std::conditional<sizeof(T) == 2, u32x4_a2, u32x4_a4>::type Mem;
};
template <typename T> __device__ __forceinline__ u32x4 load_raw(const T* p) { return *reinterpret_cast<const typename Pack<T>::Mem*>(p); }
__device__ __forceinline__ float raw_at(const u32x4& r, int j, float) { return __uint_as_float(r[j]); }
__device__ __forceinline__ float raw_at(const u32x4& r, int j, bf16_t) {
  return __uint_as_float(j & 1 ? r[j >> 1] & 0xffff0000u : r[j >> 1] << 16);
}
typedef f16_t f16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float raw_at(const u32x4& r, int j, f16_t) {
  return (float)__builtin_bit_cast(f16x2, (uint32_t)r[j >> 1])[j & 1];
}
template <typename T> __device__ __forceinline__ float raw_get(const u32x4& r, int j) { return raw_at(r, j, T()); }
template <typename T> __device__ __forceinline__ u32x4 raw_minus_inf() {
  const uint32_t v = sizeof(T) == 4 ? 0xff800000u : __builtin_bit_cast(uint16_t, (typename std::conditional<sizeof(T) == 4, bf16_t, T>::type)-__builtin_inff()) * 0x10001u;
  return u32x4{v, v, v, v};
}
// The first `live` elements of a pack, zeros behind them.
template <typename T> __device__ __forceinline__ u32x4 load_raw_part(const T* p, int live) {
  typedef typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type Bits;
  u32x4 r = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < Pack<T>::N; ++j)
    if (j < live) r[j / Pack<T>::PER] |= (uint32_t)reinterpret_cast<const Bits*>(p)[j] << (j % Pack<T>::PER * 16);
  return r;
}
template <typename T> __device__ __forceinline__ void load_pack(const T* p, float (&v)[Pack<T>::N]) {
  const u32x4 r = load_raw(p);
#pragma unroll
  for (int j = 0; j < Pack<T>::N; ++j) v[j] = raw_get<T>(r, j);
}
// (a conversion to half precision rounds to nearest even: the one rounding of a result that was computed in 32 bits)
__device__ __forceinline__ uint32_t pack_word(const float* v, float) { return __float_as_uint(v[0]); }
__device__ __forceinline__ uint32_t pack_word(const float* v, bf16_t) { return __builtin_bit_cast(uint32_t, bf16x2{(bf16_t)v[0], (bf16_t)v[1]}); }
__device__ __forceinline__ uint32_t pack_word(const float* v, f16_t) { return __builtin_bit_cast(uint32_t, f16x2{(f16_t)v[0], (f16_t)v[1]}); }
template <typename T> __device__ __forceinline__ void store_pack(T* p, const float (&v)[Pack<T>::N]) {
  u32x4 r;
#pragma unroll
  for (int w = 0; w < 4; ++w) r[w] = pack_word(v + w * Pack<T>::PER, T());
  *reinterpret_cast<typename Pack<T>::Mem*>(p) = r;
}

// Token i of an int32 or int64 array; -1 when it lies outside [0, n_rows).
struct TokenView {
  const void* p;
  int32_t bytes;     // 4 or 8
  int32_t n_rows;
  __device__ __forceinline__ int at(int64_t i) const {
    const int64_t v = bytes == 8 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
    return v >= 0 && v < n_rows ? (int)v : -1;
  }
};

// Sum / maximum over the TPR consecutive lanes of a row group (8, 16 or 64), every lane receives it.
template <int TPR> __device__ __forceinline__ float group_sum(float v) {
  v += dpp_move<0xB1>(v);
  v += dpp_move<0x4E>(v);
  v += dpp_move<0x141>(v);
  if (TPR >= 16) v += dpp_move<0x140>(v);
  if (TPR >= 64) { v = add_xor16(v); v += __shfl_xor(v, 32); }
  return v;
}
template <int TPR> __device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  if (TPR >= 16) v = fmaxf(v, dpp_move<0x140>(v));
  if (TPR >= 64) { v = fmaxf(v, __shfl_xor(v, 16)); v = fmaxf(v, __shfl_xor(v, 32)); }
  return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ int wave_sum_i32(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// Sum over a block of NT threads, in the fixed order of its waves; every thread receives it.  `red` holds NT / 64 values
// and is free again when the call returns.
template <int NT, typename S> __device__ __forceinline__ S block_sum(S v, S* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  S s = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) s += red[w];
  __syncthreads();
  return s;
}
