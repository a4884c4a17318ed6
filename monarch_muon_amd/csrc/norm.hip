// Root-mean-square norm with the residual's addition, and its gradients.
//
//   h = round(x + r)      s = (mean of h^2 + eps)^-1/2      y = h s w
//   dx = dr = dh + s w dy - h s^3 mean(w dy h)              dw = sum over rows of dy h s
//
// h is what the residual stream keeps, so the norm is of its rounded values, and the backward
// has what the forward had.  A row is held in registers by a power of two of lanes, up to eight
// 16-B chunks each, so each input is read once and each output written once: bound by HBM.
//
// Output in 8 bits: a scale for each `group` columns (or the row), scale = max |y| / MAX (1 where
// that is no normal number), code = y / scale to the nearest even; y goes from fp32 to its code in one rounding.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "fp8codec.hpp"
#include "kernels.hpp"
#include "rows.hpp"

namespace mmuon {
namespace {

// w's values of a chunk; bits of another type than the row's only where w is fp32 and the row bf16
template <class T>
__device__ __forceinline__ void load_weight(const mmuon_norm_args& a, int col, int left, float (&v)[ROW_CHUNK<T>]) {
  if (a.w_dtype == MMUON_F32) load_floats(static_cast<const float*>(a.w) + col, left, v);
  else load_chunk<BF16T>(static_cast<const uint16_t*>(a.w) + col, left, v);
}
template <>
__device__ __forceinline__ void load_weight<F32T>(const mmuon_norm_args& a, int col, int left, float (&v)[4]) {
  load_chunk<F32T>(static_cast<const float*>(a.w) + col, left, v);
}

// A scale that is no normal number, of values that are 0 or next to it, has no reciprocal.
template <class F>
__device__ __forceinline__ float code_scale(float most) {
  const float scale = most / F::MAX;
  return scale < 0x1p-126f ? 1.f : scale;
}

// y / scale as y (1 / scale): two roundings of 2^-24, where the code's own is 2^-4 or 2^-3
template <class F, int N>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&y)[N], float scale, int left) {
  uint32_t code[N / 4];
  const float by = 1.f / scale;
#pragma unroll
  for (int k = 0; k < N; k += 4) {
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      z[e] = y[k + e] * by;
      if (fabsf(z[e]) > F::MAX) z[e] = copysignf(F::MAX, z[e]);  // (a NaN stays one)
    }
    code[k / 4] = encode4<F>(z);
  }
#pragma unroll
  for (int k = 0; k < N / 4; ++k) {
    if (left >= 4 * k + 4) {
      *reinterpret_cast<u32_any*>(p + 4 * k) = code[k];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * k + e < left) p[4 * k + e] = uint8_t(code[k] >> (8 * e));
    }
  }
}

// OUT: MMUON_F8E4M3 or MMUON_F8E5M2, or anything else for y in T.  BLOCK: threads at most.
template <class T, int CPT, int BLOCK, int OUT>
__global__ __launch_bounds__(BLOCK) void norm_rows(mmuon_norm_args a, int lanes) {
  using S = typename T::storage;
  constexpr int N = ROW_CHUNK<T>;
  __shared__ float scratch[BLOCK / 64];
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t row = int64_t(blockIdx.x) * (blockDim.x / lanes) + threadIdx.x / lanes;
  const bool in = row < a.rows;  // (rows of over 64 lanes meet at barriers)
  const S* x = static_cast<const S*>(a.x) + (in ? row : 0) * a.x_stride;
  const S* r = a.residual ? static_cast<const S*>(a.residual) + (in ? row : 0) * a.residual_stride : nullptr;
  float h[CPT][N];
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    const int col = (i * lanes + lane) * N, left = in ? a.width - col : 0;
    load_chunk<T>(x + col, left, h[i]);
  }
  if (r != nullptr) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int col = (i * lanes + lane) * N, left = in ? a.width - col : 0;
      float v[N];
      load_chunk<T>(r + col, left, v);
#pragma unroll
      for (int k = 0; k < N; ++k) h[i][k] = T::round(h[i][k] + v[k]);
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    if (a.h != nullptr) {
      const int col = (i * lanes + lane) * N, left = in ? a.width - col : 0;
      store_chunk<T>(static_cast<S*>(a.h) + row * a.width + col, h[i], left);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) sum = fmaf(h[i][k], h[i][k], sum);
  }
  sum = row_sum(sum, lanes, scratch);
  const float inv = 1.f / sqrtf(sum / float(a.width) + a.eps);
  if (in && lane == 0 && a.inv != nullptr) a.inv[row] = inv;
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    const int col = (i * lanes + lane) * N, left = in ? a.width - col : 0;
    float w[N];
    load_weight<T>(a, col, left, w);
#pragma unroll
    for (int k = 0; k < N; ++k) h[i][k] = h[i][k] * inv * w[k];
    if constexpr (OUT == MMUON_F8E4M3 || OUT == MMUON_F8E5M2) {
#pragma unroll
      for (int k = 0; k < N; ++k) most = fmaxf(most, fabsf(h[i][k]));
      if (a.group > 0) {  // a group lies in 128 / N lanes that follow one another
        using F = std::conditional_t<OUT == MMUON_F8E4M3, E4M3, E5M2>;
        for (int o = min(lanes, 128 / N) >> 1; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
        const float scale = code_scale<F>(most);
        if (left > 0) {
          store_codes<F>(static_cast<uint8_t*>(a.y) + row * a.width + col, h[i], scale, left);
          if (col % 128 == 0) a.scale[row * ((a.width + 127) / 128) + col / 128] = scale;
        }
        most = 0.f;
      }
    } else {
      store_chunk<T>(static_cast<S*>(a.y) + row * a.width + col, h[i], left);
    }
  }
  if constexpr (OUT == MMUON_F8E4M3 || OUT == MMUON_F8E5M2) {
    if (a.group > 0) return;
    using F = std::conditional_t<OUT == MMUON_F8E4M3, E4M3, E5M2>;
    most = row_max(most, lanes, scratch);
    const float scale = code_scale<F>(most);
    if (in && lane == 0) a.scale[row] = scale;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int col = (i * lanes + lane) * N, left = in ? a.width - col : 0;
      if (left > 0) store_codes<F>(static_cast<uint8_t*>(a.y) + row * a.width + col, h[i], scale, left);
    }
  }
}

// dx, and this workgroup's part of dw: its rows' sums in fp32 in registers, joined row after row.
template <class T, int CPT, int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_grad(mmuon_norm_args a, int lanes) {
  using S = typename T::storage;
  constexpr int N = ROW_CHUNK<T>;
  __shared__ float scratch[BLOCK / 64];
  extern __shared__ float joined[];
  const int lane = threadIdx.x & (lanes - 1), mine = threadIdx.x / lanes, each = blockDim.x / lanes;
  float dw[CPT][N] = {};
  for (int64_t r0 = int64_t(blockIdx.x) * each; r0 < a.rows; r0 += int64_t(gridDim.x) * each) {
    const int64_t row = r0 + mine;
    const bool in = row < a.rows;
    const S* hp = static_cast<const S*>(a.x) + (in ? row : 0) * a.x_stride;
    const S* gp = static_cast<const S*>(a.dy) + (in ? row : 0) * a.dy_stride;
    const S* dhp = a.dh ? static_cast<const S*>(a.dh) + (in ? row : 0) * a.dh_stride : nullptr;
    const float inv = in ? a.inv[row] : 0.f;
    u32x4_v h[CPT], g[CPT], dh[CPT];
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int col = (i * lanes + lane) * N, left = in ? a.width - col : 0;
      h[i] = load_bits<T>(hp + col, left);
      g[i] = load_bits<T>(gp + col, left);
      if (dhp != nullptr) dh[i] = load_bits<T>(dhp + col, left);
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int col = (i * lanes + lane) * N, left = in ? a.width - col : 0;
      float hv[N], gv[N], w[N];
      unpack_chunk(h[i], hv);
      unpack_chunk(g[i], gv);
      load_weight<T>(a, col, left, w);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        dw[i][k] = fmaf(gv[k], hv[k] * inv, dw[i][k]);
        dot = fmaf(gv[k] * w[k], hv[k], dot);
      }
    }
    dot = row_sum(dot, lanes, scratch);
    const float c = dot / float(a.width) * inv * inv * inv;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int col = (i * lanes + lane) * N, left = in ? a.width - col : 0;
      float hv[N], gv[N], w[N], d[N];
      unpack_chunk(h[i], hv);
      unpack_chunk(g[i], gv);
      load_weight<T>(a, col, left, w);
      if (dhp != nullptr) unpack_chunk(dh[i], d);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float v = fmaf(gv[k] * w[k], inv, -(hv[k] * c));
        d[k] = dhp != nullptr ? d[k] + v : v;
      }
      store_chunk<T>(static_cast<S*>(a.dx) + row * a.width + col, d, left);
    }
  }
  if (a.dw == nullptr) return;
  float* part = static_cast<float*>(a.workspace) + int64_t(blockIdx.x) * a.width;
  for (int j = 0; j < each; ++j) {
    if (mine == j) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int col = (i * lanes + lane) * N + k;
          if (col >= a.width) continue;
          if (each == 1) part[col] = dw[i][k];
          else joined[col] = j == 0 ? dw[i][k] : joined[col] + dw[i][k];
        }
      }
    }
    __syncthreads();
  }
  if (each == 1) return;
  for (int col = threadIdx.x; col < a.width; col += blockDim.x) part[col] = joined[col];
}

// dw of `parts` sums for each column: 64 columns to a workgroup, 16 runs of the parts side by side
__global__ __launch_bounds__(1024) void norm_join(mmuon_norm_args a, int parts) {
  __shared__ float sums[16][64];
  const int c = threadIdx.x & 63, run = threadIdx.x >> 6, col = blockIdx.x * 64 + c;
  const int each = (parts + 15) / 16, p1 = min((run + 1) * each, parts);
  const float* part = static_cast<const float*>(a.workspace);
  float s = 0.f;
  if (col < a.width) {
#pragma unroll 8
    for (int p = run * each; p < p1; ++p) s += part[int64_t(p) * a.width + col];
  }
  sums[run][c] = s;
  __syncthreads();
  if (run != 0 || col >= a.width) return;
  s = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) s += sums[k][c];
  if (a.w_dtype == MMUON_F32) static_cast<float*>(a.dw)[col] = s;
  else static_cast<uint16_t*>(a.dw)[col] = f2bf(s);
}

// Lanes of a row and chunks of a lane.  Two chunks to a lane, or one where the rows are too few to fill
// the chip's threads (2048 to a CU): many waves with little in flight each hide one another's latency
// better than few with much.  16384 x 4096 in bf16 with a residual, 1, 2, 4 and 8 chunks: gradient 120,
// 117, 147 and 221 us (512 MiB: 4.6 TB/s at best); forward, 2, 4 and 8: 85, 86 and 97 us (6.3 TB/s); 8-bit
// output of 4096 x 4096: 23.3, 24.1 and 30 us (5.1 TB/s).  Rows of over 8192 bf16 columns take 4 and 8.
constexpr int64_t FILL = 524288;
constexpr int GRAD_BLOCK = 512;
struct RowPlan {
  int lanes, chunks;
};
RowPlan row_plan(int64_t rows, int width, int columns) {
  const int all = (width + columns - 1) / columns;
  int most = 1;
  while (most < all && most < 512) most *= 2;
  int lanes = std::min(most, 64);
  while (lanes < 512 && lanes * 2 < all) lanes *= 2;
  while (lanes < most && rows * lanes < FILL) lanes *= 2;
  RowPlan p{lanes, 1};
  while (p.chunks * lanes < all) p.chunks *= 2;
  return p;
}

template <class T, int CPT, int OUT>
void norm_launch(const mmuon_norm_args& all, int lanes, hipStream_t s) {
  using S = typename T::storage;
  const int block = std::max(lanes, 256), each = block / lanes;
  // a launch holds fewer than 2^32 threads: more rows take several
  const int64_t most = (int64_t(1) << 31) / lanes;
  for (int64_t r = 0; r < all.rows; r += most) {
    mmuon_norm_args a = all;
    a.rows = std::min(all.rows - r, most);
    a.x = static_cast<const S*>(all.x) + r * all.x_stride;
    if (all.residual != nullptr) a.residual = static_cast<const S*>(all.residual) + r * all.residual_stride;
    if (all.h != nullptr) a.h = static_cast<S*>(all.h) + r * all.width;
    if (all.inv != nullptr) a.inv = all.inv + r;
    constexpr bool codes = OUT == MMUON_F8E4M3 || OUT == MMUON_F8E5M2;
    a.y = static_cast<char*>(all.y) + r * all.width * int64_t(codes ? 1 : sizeof(S));
    if (codes) a.scale = all.scale + r * (all.group > 0 ? (all.width + 127) / 128 : 1);
    const dim3 grid(unsigned((a.rows + each - 1) / each));
    if (block == 256) hipLaunchKernelGGL((norm_rows<T, CPT, 256, OUT>), grid, dim3(256), 0, s, a, lanes);
    else hipLaunchKernelGGL((norm_rows<T, CPT, 512, OUT>), grid, dim3(block), 0, s, a, lanes);
  }
}
template <class T, int OUT>
void norm_forward(const mmuon_norm_args& a, hipStream_t s) {
  const RowPlan p = row_plan(a.rows, a.width, ROW_CHUNK<T>);
  switch (p.chunks) {
    case 1: return norm_launch<T, 1, OUT>(a, p.lanes, s);
    case 2: return norm_launch<T, 2, OUT>(a, p.lanes, s);
    case 4: return norm_launch<T, 4, OUT>(a, p.lanes, s);
    default: return norm_launch<T, 8, OUT>(a, p.lanes, s);
  }
}
template <class T>
void norm_forward(const mmuon_norm_args& a, hipStream_t s) {
  if (a.out_dtype == MMUON_F8E4M3) norm_forward<T, MMUON_F8E4M3>(a, s);
  else if (a.out_dtype == MMUON_F8E5M2) norm_forward<T, MMUON_F8E5M2>(a, s);
  else norm_forward<T, MMUON_BF16>(a, s);
}

// Workgroups of the gradient: each leaves a row of sums.  Two to a CU, which their registers allow; a third
// would wait for one of them (768: 132 us in place of 117), and 1024 leave twice the sums.
int grad_parts(const mmuon_norm_args& a, int lanes) {
  const int each = GRAD_BLOCK / lanes;
  return int(std::min<int64_t>((a.rows + each - 1) / each, 512));
}
template <class T, int CPT>
void grad_launch(const mmuon_norm_args& a, int lanes, hipStream_t s) {
  const size_t shared = lanes < GRAD_BLOCK ? size_t(a.width) * 4 : 0;
  hipLaunchKernelGGL((norm_grad<T, CPT, GRAD_BLOCK>), dim3(unsigned(grad_parts(a, lanes))), dim3(GRAD_BLOCK), shared, s, a, lanes);
}
template <class T>
void norm_backward(const mmuon_norm_args& a, hipStream_t s) {
  const RowPlan p = row_plan(a.rows, a.width, ROW_CHUNK<T>);
  switch (p.chunks) {
    case 1: grad_launch<T, 1>(a, p.lanes, s); break;
    case 2: grad_launch<T, 2>(a, p.lanes, s); break;
    case 4: grad_launch<T, 4>(a, p.lanes, s); break;
    default: grad_launch<T, 8>(a, p.lanes, s); break;
  }
  if (a.dw == nullptr) return;
  hipLaunchKernelGGL(norm_join, dim3(unsigned((a.width + 63) / 64)), dim3(1024), 0, s, a, grad_parts(a, p.lanes));
}

}  // namespace

size_t norm_workspace(const mmuon_norm_args& a) {
  if (a.rows == 0) return 0;
  const RowPlan p = row_plan(a.rows, a.width, a.dtype == MMUON_BF16 ? ROW_CHUNK<BF16T> : ROW_CHUNK<F32T>);
  return size_t(grad_parts(a, p.lanes)) * size_t(a.width) * 4;
}

int launch_norm_fwd(const mmuon_norm_args& a, hipStream_t s) {
  if (a.rows == 0) return 0;
  if (a.dtype == MMUON_BF16) norm_forward<BF16T>(a, s);
  else norm_forward<F32T>(a, s);
  return 0;
}

int launch_norm_bwd(const mmuon_norm_args& a, hipStream_t s) {
  if (a.rows == 0) {
    if (a.dw != nullptr) hipLaunchKernelGGL(norm_join, dim3(unsigned((a.width + 63) / 64)), dim3(1024), 0, s, a, 0);
    return 0;
  }
  if (a.dtype == MMUON_BF16) norm_backward<BF16T>(a, s);
  else norm_backward<F32T>(a, s);
  return 0;
}

}  // namespace mmuon
