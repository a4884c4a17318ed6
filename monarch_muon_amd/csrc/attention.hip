// Differential attention, forward: for each head the difference of two softmax maps over shared values.
//
//   s_m = scale q_m . k_m    P_m = exp(s_m - max) / sum    o = sum_j P_1 v - lam sum_j P_2 v
//
// One pass over the keys with a running reference and sum for each map.  A wave has 32 queries and
// both maps, so that a value read from LDS serves two products; with heads of over 64 columns, whose
// sums for both maps would be all of a SIMD's registers, and where there are few rows, two waves have a
// map each and join them at the end (two waves to a SIMD, one's exponentials beside the other's products;
// 3 x 1001 tokens, 6 heads of 2 x 64: one wave for both maps 63 us, a pair 40).  Scores are made transposed
// (keys x queries): a lane's values all belong to one query, the row's statistics are the lane's own
// but for one exchange between the half-waves, and the probabilities are the next product's operand as
// they stand.  The reference moves only where a score exceeds it by 2^8: what is exact needs no
// maximum, and the accumulators are left alone but for a few tiles at a row's begin.
//
// Probabilities are rounded to bf16 for their product, and the output is divided by the sum of the
// rounded ones: its weights add up to one.  The gradient needs that: D_m = dO . o_m is subtracted from
// dO . v, and where one key has most of the weight little is left, of which the weights' error must be
// a small part.  (Divided by the exact sum, the gradients of two queries were 0.65% off.)  o_m goes to the
// backward in fp32 for the same reason; the backward's own probabilities are made with the exact sum.
//
// Rows are the query heads that share a key head, token after token, so that single tokens of several
// heads are one tile of rows and a cache is read once.  Where there are few rows the
// keys are split over workgroups, and a second launch joins the parts in order.
#include <algorithm>

#include "attention_tile.hpp"
#include "kernels.hpp"

namespace mmuon {
namespace {

// A part's place in the workspace: for each row the sums of both maps (2 x 2 D floats, the reference's
// scale still on them) and (reference, sum, weight) of each map
struct Parts {
  float* sums;
  float4* stats;  // [row][map]
};

// log2 of the sum of a row's 2^(s - shift), shift still on it, and what 2^(s - that) is to be multiplied by
// for what the logarithm's rounding took: half of its last place, 2^(e - 24) ln 2 of each probability of the row for one
// of 2^e and more (1.3e-6 from 32 on, 4e-5 from 1024 on; the scores' own fp32 sums are off by as much).  dq and dlam, where
// rows cancel, take that factor; dk and dv, whose P and dS are rounded to bf16 (2^-9), do not.  Of a row that sees
// nothing +inf, so that its probabilities are 0.
__device__ __forceinline__ void store_lse(float* to, float shift, float sum) {
  const float lse = sum == 0.f ? INFINITY : shift + __builtin_amdgcn_logf(sum);
  *reinterpret_cast<float2*>(to) = make_float2(lse, sum == 0.f ? 1.f : __builtin_amdgcn_exp2f(lse - shift) / sum);
}

// MAPS: maps of a wave.  (Heads of over 64 columns, eight waves, keys in parts: 2 registers go to scratch.)
template <int D, int TK, int WAVES, int MAPS, int SLOTS, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 ? 2 : 1) void attend(mmuon_attention_args a, int tiles, int splits, Dealing dealt, Parts parts) {
  constexpr int CA = D / 8, CB = D / 4, PANELS = D / 16;  // of the values: 2 D / 32
  using T = Tile<D, TK, WAVES>;
  __shared__ __attribute__((aligned(1024))) char ring[SLOTS * T::BYTES];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int PAIRS = WAVES * MAPS / 2;  // waves of 32 rows: one, or two that are a pair
  const int m0 = MAPS == 2 ? 0 : wave & 1;
  int group, item;
  if (!deal(dealt, a.batch * a.kv_heads, group, item)) return;
  // the last queries see the most keys: first
  const int tile = tiles - 1 - item / splits, split = item % splits;
  const int b = group / a.kv_heads, g = group % a.kv_heads, share = a.heads / a.kv_heads;
  const int rows = share * a.queries, r0 = tile * 32 * PAIRS;
  const Span span = span_of(a, b);
  // keys that any row of the workgroup sees, and the wave's: most and fewest
  const auto most_of = [&](int first, int n) {  // rows first .. first + n - 1
    if (first >= rows) return 0;
    return seen(a, span, (min(first + n, rows) - 1) / share);
  };
  const int w0 = r0 + 32 * (MAPS == 2 ? wave : wave >> 1);
  const int keys = most_of(r0, 32 * PAIRS), mine = most_of(w0, 32);
  const int row = w0 + (lane & 31);
  const bool in = row < rows;
  const int t = (in ? row : rows - 1) / share, h = g * share + (in ? row : rows - 1) - t * share;
  const int limit = in ? seen(a, span, t) : keys;
  int fewest = limit;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) fewest = min(fewest, __shfl_xor(fewest, o, 64));
  fewest = __builtin_amdgcn_readfirstlane(fewest);
  const int all = (keys + TK - 1) / TK;
  int t0 = 0, t1 = all;
  if constexpr (SPLIT) {
    const int part = (all + splits - 1) / splits;
    t0 = min(split * part, all);
    t1 = min(t0 + part, all);
  }

  const char* k1 = static_cast<const char*>(a.k) + 2 * (b * a.k_stride[0] + 2 * g * a.k_stride[2]);
  TileRows src;
  src.a_stride = uint32_t(2 * a.k_stride[1]);
  src.b_stride = uint32_t(2 * a.v_stride[1]);
  src.a_last = a.dim / 8 - 1;
  src.b_last = a.dim / 4 - 1;
  const char* v0 = static_cast<const char*>(a.v) + 2 * (b * a.v_stride[0] + g * a.v_stride[2]);
  const uint32_t lds = lds_addr(ring);
  uint32_t off[T::LOADS];
  T::offsets(src, wave, lane, off);
  const auto load = [&](int i) {  // the i-th of this workgroup's tiles
    const int64_t first = int64_t(t0 + i) * TK;
    const char* k = k1 + 2 * first * a.k_stride[1];
    T::load(lds + (i % SLOTS) * T::BYTES, k, k + 2 * a.k_stride[2], v0 + 2 * first * a.v_stride[1], src, off, span.keys - int(first), wave, lane);
  };

  bf16x8 q[MAPS][D / 16];
  {
    const uint16_t* p = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + 2 * h * a.q_stride[2];
#pragma unroll
    for (int m = 0; m < MAPS; ++m) load_operands(p + (m0 + m) * a.q_stride[2], a.dim, half, q[m]);
  }
  f32x16 acc[MAPS][PANELS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int j = 0; j < PANELS; ++j) acc[m][j] = f32x16{};
  float ref[MAPS], shift[MAPS], sum[MAPS], weight[MAPS];  // sum: of exact probabilities; weight: of the rounded ones
#pragma unroll
  for (int m = 0; m < MAPS; ++m) ref[m] = -INFINITY, shift[m] = sum[m] = weight[m] = 0.f;
  const float scale = scale_of(a);

  const int n = t1 - t0;
#pragma unroll
  for (int i = 0; i < SLOTS - 1; ++i)
    if (i < n) load(i);
  wait_loaded();
  const uint32_t kbase = row_base<CA>(lane), vbase = turned_base<CB>(lane);
  for (int i = 0; i < n; ++i) {
    // this wave's part of tile i is there; behind the barrier all of it, and tile i - 1 has been read
    if (i + SLOTS - 2 < n) wait_vm<(SLOTS - 2) * T::LOADS>();
    else wait_vm<0>();
    barrier_after_lds_writes();
    if (i + SLOTS - 1 < n) load(i + SLOTS - 1);
    const char* tile_at = ring + (i % SLOTS) * T::BYTES;
    const int key0 = (t0 + i) * TK;
#pragma unroll
    for (int u = 0; u < TK; u += 32) {
      if (key0 + u >= mine) break;  // no row of this wave sees these
      f32x16 s[MAPS] = {};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
          s[m] = mfma(read_rows<CA>(tile_at + (m0 + m) * T::A2, kbase, u, kk), q[m][kk], s[m]);
      if (key0 + u + 32 > fewest) {
        const int left = limit - (key0 + u) - 4 * half;
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
          for (int m = 0; m < MAPS; ++m)
            if (8 * (e / 4) + e % 4 >= left) s[m][e] = -INFINITY;
      }
      bf16x8 p[MAPS][2];
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        float top = s[m][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[m][e]);
        top = half_max(top);
        if (__any(top * scale > shift[m] + 8.f || (ref[m] == -INFINITY && top > -INFINITY))) {
          const float next = fmaxf(ref[m], top);
          const float by = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((ref[m] - next) * scale);
          ref[m] = next;
          shift[m] = next == -INFINITY ? 0.f : next * scale;
          sum[m] *= by;
          weight[m] *= by;
#pragma unroll
          for (int j = 0; j < PANELS; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][j][e] *= by;
        }
        float w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          w[e] = __builtin_amdgcn_exp2f(fmaf(s[m][e], scale, -shift[m]));
          sum[m] += w[e];
        }
        p[m][0] = operand(w);
        p[m][1] = operand(w + 8);
        weight[m] = operand_sum(p[m][1], operand_sum(p[m][0], weight[m]));
      }
#pragma unroll
      for (int j = 0; j < PANELS; ++j)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const bf16x8 v = read_turned<CB>(tile_at + T::B, vbase, u + 16 * x, j);
#pragma unroll
          for (int m = 0; m < MAPS; ++m) acc[m][j] = mfma(v, p[m][x], acc[m][j]);
        }
    }
  }
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    sum[m] = half_sum(sum[m]);
    weight[m] = half_sum(weight[m]);
  }

  if constexpr (SPLIT) {
    if (!in) return;
    const int64_t at = (int64_t(group) * splits + split) * rows + row;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      if (half == 0) parts.stats[2 * at + m0 + m] = make_float4(shift[m], sum[m], weight[m], 0.f);
      if (sum[m] == 0.f) continue;  // nothing seen: not read
      float* to = parts.sums + (2 * at + m0 + m) * (2 * D);
#pragma unroll
      for (int j = 0; j < PANELS; ++j)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<float4*>(to + 32 * j + 2 * e + 4 * half) =
              make_float4(acc[m][j][e], acc[m][j][e + 1], acc[m][j][e + 2], acc[m][j][e + 3]);
    }
    return;
  }
  const int64_t at = (int64_t(b) * a.queries + t) * a.heads + h;
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    const float inv = 1.f / weight[m];
    float* own = in && a.o1 != nullptr ? (m0 + m ? a.o2 : a.o1) + at * 2 * a.dim : nullptr;
#pragma unroll
    for (int j = 0; j < PANELS; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[m][j][e] = weight[m] == 0.f ? 0.f : acc[m][j][e] * inv;  // (0 * NaN of a hidden key is NaN)
      if (own != nullptr) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int col = 32 * j + 2 * e + 4 * half;
          if (col < 2 * a.dim)
            *reinterpret_cast<float4*>(own + col) = make_float4(acc[m][j][e], acc[m][j][e + 1], acc[m][j][e + 2], acc[m][j][e + 3]);
        }
      }
    }
    if (a.lse != nullptr && in && half == 0)
      store_lse(a.lse + ((int64_t(b) * a.heads + h) * a.queries + t) * 4 + 2 * (m0 + m), shift[m], sum[m]);
  }
  const float lam = a.lam[int64_t(h) * a.lam_stride];
  uint16_t* o = in ? static_cast<uint16_t*>(a.o) + at * 2 * a.dim : nullptr;
  if constexpr (MAPS == 2) {
#pragma unroll
    for (int j = 0; j < PANELS; ++j) {
      f32x16 d;
#pragma unroll
      for (int e = 0; e < 16; ++e) d[e] = fmaf(-lam, acc[1][j][e], acc[0][j][e]);
      store_turned(o, d, j, 2 * a.dim, half);
    }
  } else {  // the second map's sums go through the ring, half of the columns at a time
    static_assert(PAIRS * (PANELS / 2) * 4096 <= SLOTS * T::BYTES, "half of the columns fit");
    float* pass = reinterpret_cast<float*>(ring) + (wave >> 1) * (PANELS / 2) * 1024 + lane;
#pragma unroll
    for (int j0 = 0; j0 < PANELS; j0 += PANELS / 2) {
      __syncthreads();
      if (m0 == 1) {
#pragma unroll
        for (int j = 0; j < PANELS / 2; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) pass[j * 1024 + e * 64] = acc[0][j0 + j][e];
      }
      __syncthreads();
      if (m0 == 1) continue;
#pragma unroll
      for (int j = 0; j < PANELS / 2; ++j) {
        f32x16 d;
#pragma unroll
        for (int e = 0; e < 16; ++e) d[e] = fmaf(-lam, pass[j * 1024 + e * 64], acc[0][j0 + j][e]);
        store_turned(o, d, j0 + j, 2 * a.dim, half);
      }
    }
  }
}

// The parts of a row's keys, joined by WAVES waves: each part's factor first, then the sums of every
// WAVES-th part to a wave, which are added in order.
constexpr int JOIN = 8;            // waves of a workgroup
constexpr int ALONE_PARTS = 32;  // parts that a wave can join alone
constexpr int MOST_PARTS = 1024;
template <int D, int WAVES>
__global__ __launch_bounds__(64 * JOIN) void attend_join(mmuon_attention_args a, int splits, Parts parts) {
  constexpr int N = D / 32, ROWS = JOIN / WAVES;  // columns of a lane, of each map; rows of a workgroup
  __shared__ float2 by[ROWS][WAVES == 1 ? ALONE_PARTS : MOST_PARTS];
  __shared__ float found[2][JOIN];
  __shared__ float4 total[JOIN];
  __shared__ float sums[JOIN][2][2 * D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part0 = wave % WAVES, mine = wave / WAVES;
  const int share = a.heads / a.kv_heads, rows = share * a.queries;
  const int64_t all = int64_t(a.batch) * a.kv_heads * rows, id = int64_t(blockIdx.x) * ROWS + mine;
  const bool in = id < all;  // (a workgroup's waves meet at barriers)
  const int group = int((in ? id : 0) / rows), row = int((in ? id : 0) - int64_t(group) * rows);
  const int64_t at = int64_t(group) * splits * rows + row;
  const float4* stats = parts.stats + 2 * at;
  const int step = 64 * WAVES, first = part0 * 64 + lane;
  float top1 = -INFINITY, top2 = -INFINITY;
  for (int p = first; p < splits; p += step) {
    const float4 s1 = stats[int64_t(p) * 2 * rows], s2 = stats[int64_t(p) * 2 * rows + 1];
    if (s1.y != 0.f) top1 = fmaxf(top1, s1.x);
    if (s2.y != 0.f) top2 = fmaxf(top2, s2.x);
  }
  top1 = wave_max(top1);
  top2 = wave_max(top2);
  if constexpr (WAVES > 1) {
    if (lane == 0) found[0][wave] = top1, found[1][wave] = top2;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JOIN; ++w) top1 = fmaxf(top1, found[0][w]), top2 = fmaxf(top2, found[1][w]);
  }
  float l1 = 0.f, l2 = 0.f, n1 = 0.f, n2 = 0.f;
  for (int p = first; p < splits; p += step) {
    const float4 s1 = stats[int64_t(p) * 2 * rows], s2 = stats[int64_t(p) * 2 * rows + 1];
    const float2 w = make_float2(s1.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(s1.x - top1),
                                 s2.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(s2.x - top2));
    by[mine][p] = w;
    if (s1.y != 0.f) l1 = fmaf(s1.y, w.x, l1), n1 = fmaf(s1.z, w.x, n1);
    if (s2.y != 0.f) l2 = fmaf(s2.y, w.y, l2), n2 = fmaf(s2.z, w.y, n2);
  }
  l1 = wave_sum(l1), l2 = wave_sum(l2), n1 = wave_sum(n1), n2 = wave_sum(n2);
  if (lane == 0) total[wave] = make_float4(l1, l2, n1, n2);
  __syncthreads();
  float x1[N] = {}, x2[N] = {};
  const float* from = parts.sums + at * (4 * D) + lane * N;
#pragma unroll 8
  for (int p = part0; p < splits; p += WAVES) {
    const float2 w = by[mine][p];
    const float* y = from + int64_t(p) * rows * (4 * D);
#pragma unroll
    for (int k = 0; k < N; ++k) {  // (what a part did not write counts for nothing, whatever it holds)
      const float y1 = y[k], y2 = y[2 * D + k];
      x1[k] = fmaf(w.x == 0.f ? 0.f : y1, w.x, x1[k]);
      x2[k] = fmaf(w.y == 0.f ? 0.f : y2, w.y, x2[k]);
    }
  }
  if constexpr (WAVES > 1) {
    l1 = l2 = n1 = n2 = 0.f;
#pragma unroll
    for (int w = 0; w < JOIN; ++w) l1 += total[w].x, l2 += total[w].y, n1 += total[w].z, n2 += total[w].w;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    sums[wave][0][lane * N + k] = x1[k];
    sums[wave][1][lane * N + k] = x2[k];
  }
  __syncthreads();
  const int b = group / a.kv_heads, g = group % a.kv_heads;
  const int t = row / share, h = g * share + row - t * share;
  const float lam = a.lam[int64_t(h) * a.lam_stride];
  const float i1 = n1 == 0.f ? 0.f : 1.f / n1, i2 = n2 == 0.f ? 0.f : 1.f / n2;
  const int64_t to = ((int64_t(b) * a.queries + t) * a.heads + h) * 2 * a.dim;
  if (!in) return;
  for (int c = part0 * 64 + lane; c < 2 * a.dim; c += 64 * WAVES) {
    float y1 = 0.f, y2 = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) y1 += sums[mine * WAVES + w][0][c], y2 += sums[mine * WAVES + w][1][c];
    y1 *= i1;
    y2 *= i2;
    static_cast<uint16_t*>(a.o)[to + c] = f2bf(fmaf(-lam, y2, y1));
    if (a.o1 != nullptr) {
      a.o1[to + c] = y1;
      a.o2[to + c] = y2;
    }
  }
  if (a.lse != nullptr && part0 == 0 && lane == 0) {
    float* lse = a.lse + ((int64_t(b) * a.heads + h) * a.queries + t) * 4;
    store_lse(lse, top1, l1);
    store_lse(lse + 2, top2, l2);
  }
}

struct ForwardPlan {
  bool wide;   // workgroups of eight waves, else of two that are a pair
  int tiles;   // of rows
  int splits;  // of the keys
};
// Rows of a workgroup of eight waves
constexpr int wide_rows(int dim) { return dim > 64 ? 128 : 256; }

ForwardPlan forward_plan(const mmuon_attention_args& a) {
  const int64_t rows = int64_t(a.heads / a.kv_heads) * a.queries, groups = int64_t(a.batch) * a.kv_heads;
  const int wide = wide_rows(a.dim);
  ForwardPlan p{false, 0, 1};
  if (rows == 0 || groups == 0) return p;
  // Pairs: as many workgroups as are resident, each of four tiles of keys at least
  p.tiles = int((rows + 31) / 32);
  const Pace pair = a.dim > 64 ? Pace{512, 0.049, 0.049, 5, 4e6} : Pace{1024, 0.050, 0.030, 5, 4e6};
  const int64_t most = std::min<int64_t>(MOST_PARTS, std::max(1, (a.keys + 127) / 128));
  p.splits = int(std::max<int64_t>(1, std::min(most, pair.resident / (groups * p.tiles))));
  const int64_t wide_tiles = (rows + wide - 1) / wide, wides = groups * wide_tiles;
  if (rows * 4 <= wide) {
    // Few rows of a group, over which eight waves would not be spread, are bound by the loads.  512 groups over
    // 4096 keys, heads of 2 x 64, eight waves / pairs: 1 row 296 / 193 us, 64 rows 305 / 220; of 2 x 128: 1 row 361 / 351;
    // 16384 groups of 16 rows and keys 341 / 105 and 502 / 279.  One row of 2 x 128: 128 groups 136 / 112, 192 140 / 159,
    // 256 183 / 196 (eight waves to a CU have as many loads on their way as two pairs, and need no join), 320 310 / 251.
    p.wide = a.dim > 64 && groups > 160 && groups <= 256;
    if (p.wide) p.tiles = int(wide_tiles), p.splits = 1;
    return p;
  }
  // More are bound by products and exponentials: what the estimate finds shortest.  us measured, pairs / eight waves in
  // one part / in the parts that it takes: heads of 2 x 128, 1 x 8192 tokens, 1 head 212 / 334 / 104 (6), 4 heads 402 /
  // 342 / 272 (2); 4096, 4 heads 197 / 174 / 106 (3); 1024, 4 heads 34 / 50 / -; of 2 x 64, 8192, 4 heads 243 / 354 / 173 (4);
  // 2048, 8 heads 61 / 94 / -; 3 x 1001, 6 heads on 2 36 / 51 / -; 2 x 128, 3 x 208 over 5102, 12 heads on 6 143 / 211 / 111 (3).
  const double fewest = a.causal ? std::max(0, a.keys - a.queries) : a.keys, mean = 0.5 * (a.keys + fewest);
  const double part = double(groups) * rows * (4 * (a.dim > 64 ? 128 : a.dim > 32 ? 64 : 32) + 8) * 4;
  double best = 0.95 * estimate({groups * p.tiles, double(a.keys), mean, fewest}, pair, p.splits, part);  // pairs where the two are near
  const Pace eight = a.dim > 64 ? Pace{256, 0.042, 0.042, 5, 4e6} : Pace{256, 0.0435, 0.0435, 5, 4e6};
  for (int splits = 1; splits <= ALONE_PARTS && (splits == 1 || (wides * splits <= 512 && splits * 64 <= a.keys)); ++splits) {
    const double t = estimate({wides, double(a.keys), mean, fewest}, eight, splits, part);
    if (t >= best) continue;
    best = t;
    p = {true, int(wide_tiles), splits};
  }
  return p;
}

template <int D, int TK, int WAVES, int MAPS, int SLOTS, bool SPLIT>
void attend_launch(const mmuon_attention_args& a, const ForwardPlan& p, const Parts& parts, hipStream_t s) {
  const Dealing d = dealing(int64_t(a.batch) * a.kv_heads, int64_t(p.tiles) * p.splits);
  hipLaunchKernelGGL((attend<D, TK, WAVES, MAPS, SLOTS, SPLIT>), dim3(blocks_of(d)), dim3(64 * WAVES), 0, s, a, p.tiles, p.splits, d,
                     parts);
}
template <int D>
void attend_dim(const mmuon_attention_args& a, hipStream_t s) {
  const ForwardPlan p = forward_plan(a);
  Parts parts{};
  constexpr int MAPS = D == 128 ? 1 : 2;
  constexpr int TK = D == 128 ? 32 : 64;
  if (p.wide && p.splits == 1) return attend_launch<D, TK, 8, MAPS, 3, false>(a, p, parts, s);
  if (p.splits == 1) return attend_launch<D, 32, 2, 1, 2, false>(a, p, parts, s);
  const int64_t rows = int64_t(a.heads / a.kv_heads) * a.queries * a.batch * a.kv_heads;
  parts.stats = static_cast<float4*>(a.workspace);
  parts.sums = static_cast<float*>(a.workspace) + rows * p.splits * 8;
  if (p.wide) attend_launch<D, TK, 8, MAPS, 3, true>(a, p, parts, s);
  else attend_launch<D, 32, 2, 1, 2, true>(a, p, parts, s);
  // A wave to a row where the parts are few or the rows alone fill the chip (8192 rows of 2 x 64, 9 parts: forward 120
  // us with eight waves to a row, 82 with one)
  if (p.splits <= 8 || (p.splits <= ALONE_PARTS && rows >= 2048))
    hipLaunchKernelGGL((attend_join<D, 1>), dim3(unsigned((rows + JOIN - 1) / JOIN)), dim3(64 * JOIN), 0, s, a, p.splits, parts);
  else hipLaunchKernelGGL((attend_join<D, JOIN>), dim3(unsigned(rows)), dim3(64 * JOIN), 0, s, a, p.splits, parts);
}

}  // namespace

size_t attention_forward_workspace(const mmuon_attention_args& a) {
  const ForwardPlan p = forward_plan(a);
  if (p.splits == 1) return 0;
  const int d = a.dim > 64 ? 128 : a.dim > 32 ? 64 : 32;
  return size_t(a.batch) * a.heads * a.queries * p.splits * (4 * size_t(d) + 8) * 4;
}

int launch_attention_fwd(const mmuon_attention_args& a, hipStream_t s) {
  if (a.batch == 0 || a.queries == 0 || a.heads == 0) return 0;
  if (a.dim > 64) attend_dim<128>(a, s);
  else if (a.dim > 32) attend_dim<64>(a, s);
  else attend_dim<32>(a, s);
  return 0;
}

}  // namespace mmuon
