// What the kernels of differential attention share: tiles of rows in LDS, loaded past the
// registers, and the two ways in which they are read as MFMA operands.
//
// A tile has ROWS rows of three matrices: two of D columns (the two maps' queries or keys) and one
// of 2 D (the values, or the output's gradient).  A row of CH 16-B chunks keeps chunk c at c ^ g(row):
//   CH >= 16: g = 4 (r & 3) + (r >> 2 & 3);  CH = 8: 4 (r >> 1 & 1) + (r >> 2 & 3);  CH = 4: r >> 2 & 3.
// So the 16 rows that a quarter-wave's ds_read_b128 takes of one chunk column, and the 4 rows of 64 B
// that a half-wave's ds_read_b64_tr_b16 takes, each cover all 64 banks once.
//
// 32x32x16 products: a lane's accumulator i belongs to row 8 (i / 4) + 4 (lane / 32) + i % 4 and column
// lane % 32.  A product's 16 consecutive values of a lane, rounded to bf16, are two operands of the
// next one as they stand, if its other operand is read with the rows in that order: half h of a
// 16-row step holds rows 4 h .. 4 h + 3 and 8 + 4 h .. 8 + 4 h + 3 (read_turned).
#pragma once

#include <algorithm>

#include "mfma_tile.hpp"

namespace mmuon {
namespace {

// The scores' factor, for powers of 2: rounded once, since what it is off by is the same for all scores and
// shows in dlam, a sum that cancels
__device__ __forceinline__ float scale_of(const mmuon_attention_args& a) { return float(double(a.scale) * 1.4426950408889634); }

template <int CH>
__device__ __forceinline__ int chunk_mask(int r) {
  static_assert(CH >= 4 && (CH & (CH - 1)) == 0, "rows of whole 64-B lines");
  if constexpr (CH >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (CH == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  else return (r >> 2) & 3;
}

// A per-lane address of each reading; what depends on compile-time indexes is XORed or added.
template <int CH>
__device__ __forceinline__ uint32_t row_base(int lane) {
  const int r = lane & 31;
  return uint32_t((r * CH + ((lane >> 5) ^ chunk_mask<CH>(r))) * 16);
}
template <int CH>
__device__ __forceinline__ uint32_t turned_base(int lane) {
  const int l = lane & 15, r = 4 * (lane >> 5) + (l >> 2);
  const int c = 2 * ((lane >> 4) & 1) + ((l & 3) >> 1);
  return uint32_t((r * CH + (c ^ chunk_mask<CH>(r))) * 16 + (l & 1) * 8);
}
// Rows r0 + lane % 32 (r0 a multiple of 32), columns 16 kk + 8 (lane / 32) + [0, 8)
template <int CH>
__device__ __forceinline__ bf16x8 read_rows(const char* m, uint32_t base, int r0, int kk) {
  return *reinterpret_cast<const bf16x8*>(m + r0 * CH * 16 + (base ^ uint32_t(kk * 32)));
}
// Column 32 jb + lane % 32, rows r0 + 4 (lane / 32) + [0, 4) and 8 more on (r0 a multiple of 16)
template <int CH>
__device__ __forceinline__ bf16x8 read_turned(const char* m, uint32_t base, int r0, int jb) {
  const char* p = m + r0 * CH * 16;
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + (base ^ uint32_t(jb * 64))));
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 8 * CH * 16 + (base ^ uint32_t(jb * 64 + 32))));
  typedef short i16x8 __attribute__((ext_vector_type(8)));
  const i16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf16x8, v);
}

// Values 8 s .. 8 s + 7 of a lane as an operand
__device__ __forceinline__ bf16x8 operand(const float* v) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 u = {f2bf2(v[0], v[1]), f2bf2(v[2], v[3]), f2bf2(v[4], v[5]), f2bf2(v[6], v[7])};
  return __builtin_bit_cast(bf16x8, u);
}

// What the rounding of those values to the operand left
__device__ __forceinline__ bf16x8 operand_rest(const float* v, const bf16x8& rounded) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 u = __builtin_bit_cast(u32x4, rounded);
  float r[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    r[2 * k] = v[2 * k] - __uint_as_float(u[k] << 16);
    r[2 * k + 1] = v[2 * k + 1] - __uint_as_float(u[k] & 0xffff0000u);
  }
  return operand(r);
}

// c + the sum of an operand's eight values
__device__ __forceinline__ float operand_sum(const bf16x8& v, float c) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 one = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
#pragma unroll
  for (int k = 0; k < 8; k += 2) c = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[k], v[k + 1]}, one, c, false);
  return c;
}

// Sum and maximum of a lane's and the other half-wave's value for the same column
__device__ __forceinline__ float half_sum(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
__device__ __forceinline__ float half_max(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}

// Wait for every load in flight, in a form that the compiler counts: registers that were loaded
// before a loop would else be waited for inside it, and with them, in issue order, the tiles that
// are on their way past the registers.
__device__ __forceinline__ void wait_loaded() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0) alone

// A uniform value by the scalar unit, whose loads do not queue behind the tiles'
__device__ __forceinline__ float load_uniform(const float* p) {
  return *(const __attribute__((address_space(4))) float*)(uintptr_t)p;
}

// A value that the compiler takes for new: what is formed from it is formed here, not before the loop,
// where it would hold registers.
__device__ __forceinline__ uint32_t fresh(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// A tile's rows: of both kinds of matrix
struct TileRows {
  uint32_t a_stride, b_stride;  // bytes from one row to the next
  int a_last, b_last;           // the last chunk of a row that is there
};

template <int D, int ROWS, int WAVES>
struct Tile {
  static constexpr int CA = D / 8, CB = D / 4;        // chunks of a row
  static constexpr int NA = ROWS * CA / 64, NB = 2 * NA;  // loads of a wave that fill a matrix
  static constexpr int LOADS = (2 * NA + NB) / WAVES;     // of each wave
  static constexpr int A2 = ROWS * CA * 16, B = 2 * A2, BYTES = 4 * A2;
  static_assert((2 * NA + NB) % WAVES == 0, "each wave has as many loads");

  // A wave's k-th load fills 1 KiB: its matrix, where in the tile, and each lane's offset in the
  // matrix's rows.  Rows from `left` on repeat the last one there, rows before `skip` that one, and chunks a
  // row does not have its last: what is read is always there, and what comes of it is masked, multiplied by
  // zeros or not stored.
  static __device__ __forceinline__ uint32_t offset(const TileRows& s, int n, int lane, int left, int skip = 0) {
    if (n < 2 * NA) {
      const int at = (n >= NA ? n - NA : n) * 64 + lane, r = at / CA, c = min((at % CA) ^ chunk_mask<CA>(r), s.a_last);
      return uint32_t(min(max(r, skip), left - 1)) * s.a_stride + uint32_t(c) * 16;
    }
    const int at = (n - 2 * NA) * 64 + lane, r = at / CB, c = min((at % CB) ^ chunk_mask<CB>(r), s.b_last);
    return uint32_t(min(max(r, skip), left - 1)) * s.b_stride + uint32_t(c) * 16;
  }
  // (of whole tiles: made once, so that a load in the loop is a load and little else)
  static __device__ __forceinline__ void offsets(const TileRows& s, int wave, int lane, uint32_t (&off)[LOADS]) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) off[k] = offset(s, wave + WAVES * k, lane, ROWS);
  }
  // a1, a2, b: the tile's first row in each matrix (values: a select between members of a struct goes through memory)
  static __device__ __forceinline__ void load(uint32_t lds, const char* a1, const char* a2, const char* b, const TileRows& s,
                                              const uint32_t (&off)[LOADS], int left, int wave, int lane, int skip = 0) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int n = wave + WAVES * k;
      const char* from = uniform_ptr(n < NA ? a1 : n < 2 * NA ? a2 : b);
      dma16(from, left >= ROWS && skip <= 0 ? off[k] : offset(s, n, lane, left, skip), lds + n * 1024);
    }
  }
};

// A row of `dim` columns (a multiple of 8) as operands: columns first + 16 kk + 8 (lane / 32) + [0, 8), zeros
// behind the last
template <int N>
__device__ __forceinline__ void load_operands(const uint16_t* row, int dim, int half, bf16x8 (&v)[N], int first = 0) {
#pragma unroll
  for (int kk = 0; kk < N; ++kk) {
    const int col = first + 16 * kk + 8 * half;
    v[kk] = bf16x8{};
    if (col < dim) v[kk] = *reinterpret_cast<const bf16x8*>(row + col);
  }
}

// Accumulators of 32 rows (columns of the output) and 32 columns (its rows) to bf16, a lane's row `out`
// (null: none) from column 32 jb on: the half-waves exchange 4 values, so that each stores 16 B.
__device__ __forceinline__ void store_turned(uint16_t* out, const f32x16& acc, int jb, int dim, int half) {
#pragma unroll
  for (int g = 0; g < 4; g += 2) {
    uint32_t a0 = f2bf2(acc[4 * g], acc[4 * g + 1]), a1 = f2bf2(acc[4 * g + 2], acc[4 * g + 3]);
    uint32_t b0 = f2bf2(acc[4 * g + 4], acc[4 * g + 5]), b1 = f2bf2(acc[4 * g + 6], acc[4 * g + 7]);
    const auto x = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
    const int col = 32 * jb + 8 * (g + half);
    if (out != nullptr && col < dim) *reinterpret_cast<uint4*>(out + col) = make_uint4(x[0], y[0], x[1], y[1]);
  }
}

// Which group (sequence and key head) and which of its items a workgroup takes.  `across` 8: a group's
// workgroups are on one XCD, whose L2 holds its keys and values; 1: groups are spread over all of them.
// Items are in falling order of their work, and a block of groups is dealt item by item: the largest
// first, so that the smallest fill the end, but no more groups at a time than that takes.
struct Dealing {
  int across;
  int groups;  // of one XCD
  int block;
  int each;    // items of a group
};
__device__ __forceinline__ bool deal(const Dealing& d, int all, int& group, int& item) {
  const int local = d.across == 8 ? blockIdx.x >> 3 : blockIdx.x;
  const int full = d.block * d.each, at = local / full, rest = local - at * full;
  const int n = min(d.block, d.groups - at * d.block);
  item = rest / n;
  const int of = at * d.block + rest - item * n;
  group = d.across == 8 ? (blockIdx.x & 7) + 8 * of : of;
  return group < all;
}
inline Dealing dealing(int64_t groups, int64_t each) {
  Dealing d;
  d.across = groups % 8 == 0 || groups >= 64 ? 8 : 1;
  d.groups = int((groups + d.across - 1) / d.across);
  d.each = int(each);
  d.block = int(std::max<int64_t>(1, std::min<int64_t>(d.groups, 128 * (8 / d.across) / std::max<int64_t>(each, 1))));
  return d;
}
inline unsigned blocks_of(const Dealing& d) { return unsigned(int64_t(d.across) * d.groups * d.each); }

// Workgroups of a launch, and the length of the longest, the mean and the shortest one's loop
struct Items {
  int64_t count;
  double most, mean, fewest;
};
// us of a unit of that length: with as many workgroups resident as there is room for, and by itself where
// others are through; of a workgroup beside its loop; bytes a us at which parts are written and joined
struct Pace {
  int64_t resident;
  double full, alone, beside, parts;
};
// us of a launch with its loops in `splits` parts, and of joining them: the longest workgroup, all of them over
// those that are resident, or rounds of the shortest
inline double estimate(const Items& n, const Pace& p, int64_t splits, double part_bytes) {
  const double rounds = double((n.count * splits + p.resident - 1) / p.resident);
  const double t = std::max({n.most * p.alone / splits + p.beside, double(n.count) * splits * (n.mean * p.full / splits + p.beside) / p.resident,
                             rounds * (n.fewest * p.full / splits + p.beside)});
  return splits == 1 ? t : t + 5 + 2 * splits * part_bytes / p.parts;
}

// The sequence's keys and the place of its first query among them
struct Span {
  int keys;       // visible ones, of those there is room for
  int64_t first;  // query t sees keys up to first + t, where the mask is causal
};
__device__ __forceinline__ Span span_of(const mmuon_attention_args& a, int b) {
  constexpr int64_t FAR = int64_t(1) << 32;  // as good as any place farther off
  const int64_t n = a.lengths != nullptr ? a.lengths[b] : a.keys;
  Span s;
  s.keys = int(n < 0 ? 0 : n > a.keys ? a.keys : n);
  s.first = a.starts != nullptr ? a.starts[b] : s.keys - a.queries;
  s.first = s.first < -FAR ? -FAR : s.first > FAR ? FAR : s.first;
  return s;
}
// Keys that query t sees
__device__ __forceinline__ int seen(const mmuon_attention_args& a, const Span& s, int t) {
  if (!a.causal) return s.keys;
  const int64_t n = s.first + t + 1;
  return n <= 0 ? 0 : n < s.keys ? int(n) : s.keys;
}

}  // namespace
}  // namespace mmuon
