// Token embedding and the gradient of its table.
//
//   out[t] = scale w[i_t]            dw[v] = scale sum over t with i_t = v of dout[t]
//
// The gradient is dense, one launch, and does not depend on timing: rows are dealt to
// classes (row v to class v % C), one workgroup each.  A workgroup reads all ids, places
// the positions of its rows in token order (counts per row and wave, then a stable rank),
// and writes its rows: zeros, or the fp32 sum of the row's gradients in token order,
// rounded once.  Common words have neighbouring ids, so the rows of a class are far apart.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace mmuon {
namespace {

// N consecutive elements; N == 1 for rows that are not whole aligned 16-B chunks
template <class T, int N>
__device__ __forceinline__ void load_n(const typename T::storage* p, float (&v)[N]) {
  if constexpr (N == 8) Vec8<T>::load(p, v);
  else v[0] = T::load(p, 0);
}
template <class T, int N>
__device__ __forceinline__ void store_n(typename T::storage* p, const float (&v)[N]) {
  if constexpr (N == 8) Vec8<T>::store(p, v);
  else T::store(p, 0, v[0]);
}

// `lanes` (a power of two) threads per row
template <class T, int N>
__global__ __launch_bounds__(256) void embed_lookup(mmuon_embedding_args a, int lanes) {
  const int64_t t = int64_t(blockIdx.x) * (256 / lanes) + threadIdx.x / lanes;
  if (t >= a.tokens) return;
  const int64_t v = a.index[t];
  const bool in = v >= 0 && v < a.vocab;
  const auto* src = static_cast<const typename T::storage*>(a.w) + (in ? v : 0) * a.w_stride;
  auto* dst = static_cast<typename T::storage*>(a.out) + t * a.width;
#pragma unroll 4
  for (int c = (threadIdx.x & (lanes - 1)) * N; c < a.width; c += lanes * N) {
    float x[N];
    load_n<T, N>(src + c, x);
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = in ? x[k] * a.scale : NAN;  // no such row: the output shows it
    store_n<T, N>(dst + c, x);
  }
}

constexpr int GT = 1024, GW = GT / 64;  // threads and waves of a gradient workgroup
constexpr int MAX_ROWS = 1024;          // rows of a class

template <class T, int N>
__global__ __launch_bounds__(GT) void embed_grad(mmuon_embedding_args a, int log2c, int* order) {
  __shared__ int at[GW][MAX_ROWS];     // counts, then the next place, of a row's positions in a wave's tokens
  __shared__ int first[MAX_ROWS + 1];  // the row's first place
  __shared__ int below[GW], wsum[GW];
  const int c = blockIdx.x, C = 1 << log2c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rows = int((a.vocab - c + C - 1) >> log2c);
  for (int i = threadIdx.x; i < GW * MAX_ROWS; i += GT) (&at[0][0])[i] = 0;
  __syncthreads();
  // a wave's tokens: a run of whole 64s
  const int64_t run = (a.tokens + 64 * GW - 1) / (64 * GW) * 64, t0 = wave * run, t1 = min(a.tokens, t0 + run);
  const auto row_of = [&](int64_t t, int& less) {  // the token's row of this class, or -1
    const int64_t v = t < t1 ? a.index[t] : -1;
    if (v < 0 || v >= a.vocab || v == a.padding_idx) return -1;
    less += int(v & (C - 1)) < c;
    return int(v & (C - 1)) == c ? int(v >> log2c) : -1;
  };
  int less = 0;
#pragma unroll 4
  for (int64_t t = t0 + lane; t < t1; t += 64) {
    const int r = row_of(t, less);
    if (r >= 0) atomicAdd(&at[wave][r], 1);
  }
  less = wave_isum(less);
  if (lane == 0) below[wave] = less;
  __syncthreads();
  // places: class after class, row after row, wave after wave
  int n = 0;
  if (threadIdx.x < rows)
    for (int w = 0; w < GW; ++w) n += at[w][threadIdx.x];
  int incl = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(incl, o, 64);
    if (lane >= o) incl += u;
  }
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < GW; ++w) base += below[w] + (w < wave ? wsum[w] : 0);
  first[threadIdx.x] = base + incl - n;
  if (threadIdx.x == GT - 1) first[GT] = base + incl;
  int place = base + incl - n;
  for (int w = 0; w < GW; ++w) {
    const int k = at[w][threadIdx.x];
    at[w][threadIdx.x] = place;
    place += k;
  }
  __syncthreads();
  volatile int* next = at[wave];  // one lane's store is another's next load
  for (int64_t t = t0; t < t1; t += 64) {
    const int r = row_of(t + lane, less);
    uint64_t left = __ballot(r >= 0);
    while (left != 0) {  // row by row of these 64 tokens, in lane order
      const int lead = __ffsll(static_cast<unsigned long long>(left)) - 1;
      const uint64_t same = __ballot(r >= 0 && r == __shfl(r, lead, 64));
      const int p = next[__shfl(r, lead, 64)];
      if (same >> lane & 1) order[p + __popcll(same & ((uint64_t(1) << lane) - 1))] = int(t + lane);
      if (lane == lead) next[r] = p + __popcll(same);
      left &= ~same;
    }
  }
  __syncthreads();
  const auto* dout = static_cast<const typename T::storage*>(a.dout);
  for (int r = wave; r < rows; r += GW) {
    const int p0 = first[r], p1 = first[r + 1];
    auto* dst = static_cast<typename T::storage*>(a.dw) + (int64_t(r) * C + c) * a.width;
    for (int col = lane * N; col < a.width; col += 64 * N) {
      float s[N];
#pragma unroll
      for (int k = 0; k < N; ++k) s[k] = 0.f;
#pragma unroll 4
      for (int p = p0; p < p1; ++p) {
        float x[N];
        load_n<T, N>(dout + order[p] * a.dout_stride + col, x);
#pragma unroll
        for (int k = 0; k < N; ++k) s[k] += x[k];
      }
#pragma unroll
      for (int k = 0; k < N; ++k) s[k] *= a.scale;
      store_n<T, N>(dst + col, s);
    }
  }
}

// Whether rows are whole 16-B chunks (8 elements in bf16, and two chunks of fp32)
bool whole_chunks(const void* base, int64_t stride, int64_t width) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && stride % 8 == 0 && width % 8 == 0;
}

template <class T>
void lookup(const mmuon_embedding_args& a, hipStream_t s) {
  const bool vec = whole_chunks(a.w, a.w_stride, a.width) && whole_chunks(a.out, a.width, a.width);
  const int chunks = vec ? a.width / 8 : a.width;
  int lanes = 16;  // about four chunks per thread
  while (lanes < 256 && lanes * 4 < chunks) lanes *= 2;
  const dim3 grid(unsigned((a.tokens + 256 / lanes - 1) / (256 / lanes))), block(256);
  if (vec) hipLaunchKernelGGL((embed_lookup<T, 8>), grid, block, 0, s, a, lanes);
  else hipLaunchKernelGGL((embed_lookup<T, 1>), grid, block, 0, s, a, lanes);
}

// Classes: a power of two, at most MAX_ROWS rows each; 256, one workgroup per CU, where
// that suffices
int log2_classes(int64_t vocab) {
  int l = 8;
  while ((vocab + (int64_t(1) << l) - 1) >> l > MAX_ROWS) ++l;
  return l;
}

template <class T>
void gradient(const mmuon_embedding_args& a, hipStream_t s) {
  const bool vec = whole_chunks(a.dout, a.dout_stride, a.width) && whole_chunks(a.dw, a.width, a.width);
  const int l = log2_classes(a.vocab);
  const dim3 grid(unsigned(std::min<int64_t>(int64_t(1) << l, a.vocab))), block(GT);
  int* order = static_cast<int*>(a.workspace);
  if (vec) hipLaunchKernelGGL((embed_grad<T, 8>), grid, block, 0, s, a, l, order);
  else hipLaunchKernelGGL((embed_grad<T, 1>), grid, block, 0, s, a, l, order);
}

}  // namespace

size_t embedding_workspace(const mmuon_embedding_args& a) { return size_t(std::max<int64_t>(a.tokens, 1)) * 4; }

int launch_embedding_fwd(const mmuon_embedding_args& a, hipStream_t s) {
  if (a.tokens == 0) return 0;
  if (a.dtype == MMUON_BF16) lookup<BF16T>(a, s);
  else lookup<F32T>(a, s);
  return 0;
}

int launch_embedding_bwd(const mmuon_embedding_args& a, hipStream_t s) {
  if (a.dtype == MMUON_BF16) gradient<BF16T>(a, s);
  else gradient<F32T>(a, s);
  return 0;
}

}  // namespace mmuon
