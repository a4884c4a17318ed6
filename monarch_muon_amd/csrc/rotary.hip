// Rotary positions of queries and keys, and of their gradients.
//
//   (a, b) -> (a c - b s, a s + b c),   c, s = table[position][pair]
//
// for the pairs (i, i + part / 2) or, interleaved, (2 i, 2 i + 1) of a head's first `part` columns;
// the others are copied.  The gradient's rotation is by -s.  The table holds cosines and sines (times
// the scaling's factor) in fp32, made once in 64 bits, where the angles of far positions need them.
//
// A lane takes one chunk of 16 B (or two that are pairs) of a head.  Bound by HBM: queries and keys are
// read and written once, both in one launch (16384 tokens x 64 heads of 128, bf16: 92 us, 5.8 TB/s); the
// table comes from the caches, so that four heads to a lane, which read it once, are no faster (in graphs of ten
// calls 107 us, one head 98; 2048 tokens 13.1 one head, 12.6 four; 1024 7.5, 8.1; 256 5.0, 5.6).
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"
#include "rows.hpp"

namespace mmuon {
namespace {

template <class T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_rows(mmuon_rotary_args a, int64_t first, int64_t tokens, int turned, int items, float sign) {
  using S = typename T::storage;
  constexpr int N = ROW_CHUNK<T>, M = INTERLEAVED ? N / 2 : N;
  const int heads = a.q_heads + a.k_heads;
  const int64_t id = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (id >= tokens * (heads * items)) return;
  const int64_t of = id / (heads * items), token = first + of;
  const int rest = int(id - of * (heads * items)), h = rest / items, item = rest - h * items;
  const int64_t b = token / a.tokens, t = token - b * a.tokens;
  const int half = a.part / 2;
  const bool turn = item < turned;
  const int col = turn ? item * N : a.part + (item - turned) * N;
  const int left = turn ? (INTERLEAVED ? a.part : half) - col : a.dim - col;
  float c[M], s[M];
  if (turn) {
    const int64_t p = a.positions != nullptr ? a.positions[token] : t;
    const bool in = p >= 0 && p < a.table_rows;
    const float* row = a.table + (in ? p : 0) * int64_t(a.part) + (INTERLEAVED ? col / 2 : col);
    load_floats(row, INTERLEAVED ? (left + 1) / 2 : left, c);
    load_floats(row + half, INTERLEAVED ? (left + 1) / 2 : left, s);
#pragma unroll
    for (int k = 0; k < M; ++k) {
      c[k] = in ? c[k] : NAN;  // no such position: the output shows it
      s[k] *= sign;
    }
  }
  const S* from = h < a.q_heads ? static_cast<const S*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + h * a.q_stride[2]
                                : static_cast<const S*>(a.k) + b * a.k_stride[0] + t * a.k_stride[1] + (h - a.q_heads) * a.k_stride[2];
  S* to = h < a.q_heads ? static_cast<S*>(a.q_out) + (token * a.q_heads + h) * a.dim
                        : static_cast<S*>(a.k_out) + (token * a.k_heads + h - a.q_heads) * a.dim;
  u32x4_v u = load_bits<T>(from + col, left);
  if (turn) {
    float x[N], y[N];
    unpack_chunk(u, x);
    if constexpr (INTERLEAVED) {
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        y[k] = fmaf(x[k], c[k / 2], -(x[k + 1] * s[k / 2]));
        y[k + 1] = fmaf(x[k], s[k / 2], x[k + 1] * c[k / 2]);
      }
      u = pack_chunk(y);
    } else {
      float z[N];
      load_chunk<T>(from + col + half, left, z);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        y[k] = fmaf(x[k], s[k], z[k] * c[k]);
        x[k] = fmaf(x[k], c[k], -(z[k] * s[k]));
      }
      u = pack_chunk(x);
      store_chunk<T>(to + col + half, y, left);
    }
  }
  store_bits<T>(to + col, u, left);
}

template <class T, bool INTERLEAVED>
void rotary_launch(const mmuon_rotary_args& a, bool back, hipStream_t s) {
  constexpr int N = ROW_CHUNK<T>;
  const int rotated = INTERLEAVED ? a.part : a.part / 2;
  const int turned = (rotated + N - 1) / N, items = turned + (a.dim - a.part + N - 1) / N;
  const int64_t each = int64_t(a.q_heads + a.k_heads) * items;
  // a launch holds fewer than 2^32 threads: more tokens, of one sequence or several, take several
  const int64_t all = a.batch * a.tokens, most = std::max<int64_t>(1, (int64_t(1) << 31) / each);
  for (int64_t first = 0; first < all; first += most) {
    const int64_t tokens = std::min(all - first, most);
    hipLaunchKernelGGL((rotary_rows<T, INTERLEAVED>), dim3(unsigned((tokens * each + 255) / 256)), dim3(256), 0, s, a, first, tokens,
                       turned, items, back ? -1.f : 1.f);
  }
}
template <class T>
void rotary(const mmuon_rotary_args& a, bool back, hipStream_t s) {
  if (a.interleaved) rotary_launch<T, true>(a, back, s);
  else rotary_launch<T, false>(a, back, s);
}

}  // namespace

int launch_rotary(const mmuon_rotary_args& a, bool back, hipStream_t s) {
  if (a.batch == 0 || a.tokens == 0 || a.q_heads + a.k_heads == 0) return 0;
  if (a.dtype == MMUON_BF16) rotary<BF16T>(a, back, s);
  else rotary<F32T>(a, back, s);
  return 0;
}

}  // namespace mmuon
