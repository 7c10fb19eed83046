// Element types, 16-byte packs and block reductions shared by the token kernels (embed.hip, tokens.hip).
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// A pack is the 16 bytes one lane moves per memory instruction: 4 fp32 or 8 half-precision elements.  Rows of an odd
// number of elements start anywhere, so a pack is only as aligned as its element: global_load / store_dwordx4 take any
// address on this chip, and one that straddles a cache line costs one more line.
template <typename T> struct Pack {
  enum { N = 16 / sizeof(T) };
  typedef T Raw __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};
template <typename T> __device__ __forceinline__ void load_pack(const T* p, float (&v)[Pack<T>::N]) {
  const typename Pack<T>::Raw r = *reinterpret_cast<const typename Pack<T>::Raw*>(p);
#pragma unroll
  for (int j = 0; j < Pack<T>::N; ++j) v[j] = (float)r[j];
}
// (a conversion to half precision rounds to nearest even: the one rounding of a result that was computed in 32 bits)
template <typename T> __device__ __forceinline__ void store_pack(T* p, const float (&v)[Pack<T>::N]) {
  typename Pack<T>::Raw r;
#pragma unroll
  for (int j = 0; j < Pack<T>::N; ++j) r[j] = (T)v[j];
  *reinterpret_cast<typename Pack<T>::Raw*>(p) = r;
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

// Sum / maximum over the TPR consecutive lanes of a row group (16 or 64), every lane receives it.
template <int TPR> __device__ __forceinline__ float group_sum(float v) {
  v += dpp_move<0xB1>(v);
  v += dpp_move<0x4E>(v);
  v += dpp_move<0x141>(v);
  v += dpp_move<0x140>(v);
  if (TPR >= 64) { v = add_xor16(v); v += __shfl_xor(v, 32); }
  return v;
}
template <int TPR> __device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  v = fmaxf(v, dpp_move<0x140>(v));
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

// True in every thread of the block that arrives last; what the other blocks wrote before their call is then visible to
// it.  `counter` is zero before the launch.
__device__ __forceinline__ bool last_block(uint32_t* counter) {
  __shared__ int is_last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    is_last = atomicAdd(counter, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  const bool last = is_last != 0;
  if (last) __threadfence();
  return last;
}
