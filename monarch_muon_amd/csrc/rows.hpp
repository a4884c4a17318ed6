// Rows of a bf16 or fp32 matrix in 16-B chunks of consecutive elements, at any element's
// address: gfx950 loads and stores 16 B that start at any byte, so rows of odd widths and
// strides go by the same chunks as aligned ones, and only a row's last, shorter chunk an
// element at a time.
#pragma once

#include "common.hpp"

namespace mmuon {
namespace {

typedef uint32_t u32x4_v __attribute__((ext_vector_type(4)));
typedef u32x4_v u32x4_any __attribute__((aligned(2)));
typedef float f32x4_v __attribute__((ext_vector_type(4)));
typedef f32x4_v f32x4_any __attribute__((aligned(4)));
typedef float f32x2_v __attribute__((ext_vector_type(2)));
typedef f32x2_v f32x2_any __attribute__((aligned(4)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// Elements of a chunk
template <class T>
constexpr int ROW_CHUNK = 16 / int(sizeof(typename T::storage));

__device__ __forceinline__ void unpack_chunk(const u32x4_v& u, float (&v)[8]) {
  Vec8<BF16T>::unpack(make_uint4(u.x, u.y, u.z, u.w), v);
}
__device__ __forceinline__ void unpack_chunk(const u32x4_v& u, float (&v)[4]) {
  v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ u32x4_v pack_chunk(const float (&v)[8]) {
  return u32x4_v{f2bf2(v[0], v[1]), f2bf2(v[2], v[3]), f2bf2(v[4], v[5]), f2bf2(v[6], v[7])};
}
__device__ __forceinline__ u32x4_v pack_chunk(const float (&v)[4]) {
  return u32x4_v{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}

// A chunk's bits: `left` elements of the row from p on are there (left >= N: the whole chunk; the
// others are 0).
template <class T>
__device__ __forceinline__ u32x4_v load_bits(const typename T::storage* p, int left) {
  constexpr int N = ROW_CHUNK<T>;
  if (left >= N) return *reinterpret_cast<const u32x4_any*>(p);
  float v[N];
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = k < left ? T::load(p, k) : 0.f;
  return pack_chunk(v);
}
template <class T>
__device__ __forceinline__ void store_bits(typename T::storage* p, const u32x4_v& u, int left) {
  constexpr int N = ROW_CHUNK<T>;
  if (left >= N) {
    *reinterpret_cast<u32x4_any*>(p) = u;
    return;
  }
  float v[N];
  unpack_chunk(u, v);
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (k < left) T::store(p, k, v[k]);
}
template <class T>
__device__ __forceinline__ void load_chunk(const typename T::storage* p, int left, float (&v)[ROW_CHUNK<T>]) {
  unpack_chunk(load_bits<T>(p, left), v);
}
template <class T>
__device__ __forceinline__ void store_chunk(typename T::storage* p, const float (&v)[ROW_CHUNK<T>], int left) {
  store_bits<T>(p, pack_chunk(v), left);
}
// N floats (2, or a multiple of 4), `left` of them there
template <int N>
__device__ __forceinline__ void load_floats(const float* p, int left, float (&v)[N]) {
  if (left >= N) {
    if constexpr (N == 2) {
      const f32x2_v f = *reinterpret_cast<const f32x2_any*>(p);
      v[0] = f.x, v[1] = f.y;
      return;
    }
#pragma unroll
    for (int k = 0; k + 3 < N; k += 4) {
      const f32x4_v f = *reinterpret_cast<const f32x4_any*>(p + k);
      v[k] = f.x, v[k + 1] = f.y, v[k + 2] = f.z, v[k + 3] = f.w;
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = k < left ? p[k] : 0.f;
}

// Sum over the `lanes` (a power of two) lanes of a row, the same in each; rows of over 64 lanes
// join their waves through scratch[waves], in order.
__device__ __forceinline__ float row_sum(float v, int lanes, float* scratch) {
  for (int o = min(lanes, 64) >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if (lanes <= 64) return v;
  const int wave = threadIdx.x >> 6, first = wave & ~((lanes >> 6) - 1);
  __syncthreads();  // what the scratch held before has been read
  if ((threadIdx.x & 63) == 0) scratch[wave] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < lanes >> 6; ++w) v += scratch[first + w];
  return v;
}
__device__ __forceinline__ float row_max(float v, int lanes, float* scratch) {
  for (int o = min(lanes, 64) >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  if (lanes <= 64) return v;
  const int wave = threadIdx.x >> 6, first = wave & ~((lanes >> 6) - 1);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[wave] = v;
  __syncthreads();
  for (int w = 0; w < lanes >> 6; ++w) v = fmaxf(v, scratch[first + w]);
  return v;
}

}  // namespace
}  // namespace mmuon
