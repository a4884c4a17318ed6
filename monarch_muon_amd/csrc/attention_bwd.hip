// Differential attention, backward.
//
//   dP = dO v^T (both maps')   D_m = dO . o_m      dS_1 = P_1 (dP - D_1)   dS_2 = -lam P_2 (dP - D_2)
//   dq_m = scale dS_m k_m      dk_m = scale dS_m^T q_m      dv = (P_1 - lam P_2)^T dO      dlam = -sum P_2 dP
//
// The maps share dP and one product for dv.  Two kernels make the scores again, one for a block of
// queries (dq) and one for a block of keys (dk, dv), so that every sum stays in one wave's registers in
// a fixed order: nothing is added by atomics.  Scores are made so that the index which is summed over
// next is that of a lane's registers (keys x queries for dq, queries x keys for dk and dv), and P and dS,
// rounded to bf16, are the next products' operands as they stand.  dlam takes P_2 dP in fp32 as dq's
// kernel has them: o_2, from rounded probabilities, would give it their error.
//
// dq's dS goes in as two bf16 terms (dS and what its rounding left): D's error, from rounded weights, and dS's
// rounding together would make it 2.4e-3 to 2.6e-3 off, where rounding the result alone makes 1.7e-3; so it is 1.7e-3 to
// 1.8e-3, for 10 us of 85 to 95 (16 x 1024 tokens, 8 heads of 2 x 64: 88 -> 99; 4 x 1024, 16 of 2 x 128: 94 -> 105).
// dk and dv, 2.4e-3 off, have one.
//
// Both kernels have both maps in a wave, which makes no product twice.  With heads of up to 64 columns
// two waves fit a SIMD, whose products and exponentials run side by side; with more a wave's sums for dk
// and dv alone are half of its registers.  (A map to each of two waves that pass dP and P through LDS:
// 16 x 1024 tokens, 8 heads of 2 x 64, dq 123 us, dk and dv 186; 4 x 1024, 16 of 2 x 128, 92 and 210.)
#include <algorithm>

#include "attention_tile.hpp"
#include "kernels.hpp"

namespace mmuon {
namespace {

// For each query row (b, h, t): (lse_1, D_1, lse_2, D_2); and its part of dlam
struct RowSpace {
  float4* stats;
  float* dlam;  // [part]
  float* dq;    // parts: (part, row, dq_1 dq_2)
  float* dkv;   // (group, part, key, dv dk_1 dk_2)
};

// A wave to four rows' D: 16 lanes each
__global__ __launch_bounds__(256) void attention_rows(mmuon_attention_args a, RowSpace space) {
  const int64_t rows = int64_t(a.batch) * a.heads * a.queries;
  const int64_t row = int64_t(blockIdx.x) * 16 + threadIdx.x / 16;
  if (row >= rows) return;
  const int lane = threadIdx.x & 15, t = int(row % a.queries);
  const int64_t bh = row / a.queries, b = bh / a.heads, h = bh - b * a.heads;
  const int64_t at = ((b * a.queries + t) * a.heads + h) * 2 * a.dim;
  float d1 = 0.f, d2 = 0.f;
  for (int c = lane * 8; c < 2 * a.dim; c += 128) {
    float g[8], x[8], y[8];
    Vec8<BF16T>::load(static_cast<const uint16_t*>(a.dout) + at + c, g);
    Vec8<F32T>::load(a.o1 + at + c, x);
    Vec8<F32T>::load(a.o2 + at + c, y);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      d1 = fmaf(g[k], x[k], d1);
      d2 = fmaf(g[k], y[k], d2);
    }
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    d1 += __shfl_xor(d1, o, 64);
    d2 += __shfl_xor(d2, o, 64);
  }
  if (lane == 0) space.stats[row] = make_float4(a.lse[4 * row], d1, a.lse[4 * row + 2], d2);
}

// dq and each row's part of dlam: 32 queries to a wave, over tiles of 32 keys
template <int D, int WAVES, int SLOTS, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES, D == 128 ? 1 : 2) void attention_dq(mmuon_attention_args a, Dealing dealt, int parts,
                                                                             RowSpace space) {
  constexpr int CA = D / 8, CB = D / 4, TK = 32;
  using T = Tile<D, TK, WAVES>;
  __shared__ __attribute__((aligned(1024))) char ring[SLOTS * T::BYTES];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int group, item;
  if (!deal(dealt, a.batch * a.kv_heads, group, item)) return;
  const int tile = SPLIT ? dealt.each / parts - 1 - item / parts : dealt.each - 1 - item, part = SPLIT ? item % parts : 0;
  const int b = group / a.kv_heads, g = group % a.kv_heads, share = a.heads / a.kv_heads;
  const int rows = share * a.queries, r0 = tile * 32 * WAVES;
  const Span span = span_of(a, b);
  const auto most_of = [&](int first, int n) {
    if (first >= rows) return 0;
    return seen(a, span, (min(first + n, rows) - 1) / share);
  };
  const int w0 = r0 + 32 * wave;
  const int keys = most_of(r0, 32 * WAVES), mine = most_of(w0, 32);
  const int row = w0 + (lane & 31);
  const bool in = row < rows;
  const int t = (in ? row : rows - 1) / share, h = g * share + (in ? row : rows - 1) - t * share;
  const int limit = in ? seen(a, span, t) : keys;
  int fewest = limit;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) fewest = min(fewest, __shfl_xor(fewest, o, 64));
  fewest = __builtin_amdgcn_readfirstlane(fewest);

  const char* k1 = static_cast<const char*>(a.k) + 2 * (b * a.k_stride[0] + 2 * g * a.k_stride[2]);
  const char* v0 = static_cast<const char*>(a.v) + 2 * (b * a.v_stride[0] + g * a.v_stride[2]);
  TileRows src;
  src.a_stride = uint32_t(2 * a.k_stride[1]);
  src.b_stride = uint32_t(2 * a.v_stride[1]);
  src.a_last = a.dim / 8 - 1;
  src.b_last = a.dim / 4 - 1;
  const uint32_t lds = lds_addr(ring);
  uint32_t off[T::LOADS];
  T::offsets(src, wave, lane, off);
  const int all = (keys + TK - 1) / TK, i0 = SPLIT ? int(int64_t(all) * part / parts) : 0;
  const auto load = [&](int i) {
    const int64_t first = int64_t(i0 + i) * TK;
    const char* k = k1 + 2 * first * a.k_stride[1];
    T::load(lds + (i % SLOTS) * T::BYTES, k, k + 2 * a.k_stride[2], v0 + 2 * first * a.v_stride[1], src, off, span.keys - int(first), wave, lane);
  };

  bf16x8 q[2][D / 16], dout[D / 8];
  {
    const uint16_t* p = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + 2 * h * a.q_stride[2];
    load_operands(p, a.dim, half, q[0]);
    load_operands(p + a.q_stride[2], a.dim, half, q[1]);
    load_operands(static_cast<const uint16_t*>(a.dout) + ((int64_t(b) * a.queries + t) * a.heads + h) * 2 * a.dim, 2 * a.dim, half, dout);
  }
  const int64_t at = (int64_t(b) * a.heads + h) * a.queries + t;
  const float4 st = space.stats[at];
  const float by1 = a.lse[4 * at + 1], by2 = a.lse[4 * at + 3];
  const float scale = scale_of(a);
  f32x16 acc[2][D / 32];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) acc[m][j] = f32x16{};
  float along = 0.f;

  const int n = (SPLIT ? int(int64_t(all) * (part + 1) / parts) : all) - i0;
#pragma unroll
  for (int i = 0; i < SLOTS - 1; ++i)
    if (i < n) load(i);
  wait_loaded();
  const uint32_t kbase0 = row_base<CA>(lane), vbase0 = row_base<CB>(lane), tbase0 = turned_base<CA>(lane);
  for (int i = 0; i < n; ++i) {
    if (i + SLOTS - 2 < n) wait_vm<(SLOTS - 2) * T::LOADS>();
    else wait_vm<0>();
    barrier_after_lds_writes();
    if (i + SLOTS - 1 < n) load(i + SLOTS - 1);
    const char* tile_at = ring + (i % SLOTS) * T::BYTES;
    const int key0 = (i0 + i) * TK;
    if (key0 >= mine) continue;
    const uint32_t kbase = fresh(kbase0), vbase = fresh(vbase0), tbase = fresh(tbase0);
    f32x16 s[2] = {f32x16{}, f32x16{}}, dp = f32x16{};
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      s[0] = mfma(read_rows<CA>(tile_at, kbase, 0, kk), q[0][kk], s[0]);
      s[1] = mfma(read_rows<CA>(tile_at + T::A2, kbase, 0, kk), q[1][kk], s[1]);
    }
    if (key0 + TK > fewest) {
      const int left = limit - key0 - 4 * half;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (8 * (e / 4) + e % 4 >= left) s[0][e] = s[1][e] = -INFINITY;
    }
#pragma unroll
    for (int kk = 0; kk < D / 8; ++kk) dp = mfma(read_rows<CB>(tile_at + T::B, vbase, 0, kk), dout[kk], dp);
    float d1[16], d2[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      d1[e] = __builtin_amdgcn_exp2f(fmaf(s[0][e], scale, -st.x));
      d2[e] = __builtin_amdgcn_exp2f(fmaf(s[1][e], scale, -st.z));
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) d1[e] *= dp[e] - st.y;
    const bf16x8 x1[2] = {operand(d1), operand(d1 + 8)}, y1[2] = {operand_rest(d1, x1[0]), operand_rest(d1 + 8, x1[1])};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const bf16x8 k = read_turned<CA>(tile_at, tbase, 16 * y, j);
        acc[0][j] = mfma(k, x1[y], acc[0][j]);
        acc[0][j] = mfma(k, y1[y], acc[0][j]);
      }
    float tile_along = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      tile_along = fmaf(d2[e], dp[e], tile_along);
      d2[e] *= dp[e] - st.w;
    }
    along += tile_along;
    const bf16x8 x2[2] = {operand(d2), operand(d2 + 8)}, y2[2] = {operand_rest(d2, x2[0]), operand_rest(d2 + 8, x2[1])};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const bf16x8 k = read_turned<CA>(tile_at + T::A2, tbase, 16 * y, j);
        acc[1][j] = mfma(k, x2[y], acc[1][j]);
        acc[1][j] = mfma(k, y2[y], acc[1][j]);
      }
  }
  along = half_sum(along) * by2;
  if (limit == 0) {  // nothing is seen: 0, where the products have 0 * NaN if a hidden key, q or dO holds one
    along = 0.f;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < D / 32; ++j) acc[m][j] = f32x16{};
  }
  const int64_t total = int64_t(a.batch) * a.heads * a.queries;
  if (in && half == 0) space.dlam[part * total + at] = -along;
  if constexpr (SPLIT) {
    if (!in) return;
    float* to = space.dq + (part * total + at) * (2 * D) + 4 * half;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float by = m ? by2 : by1;
          *reinterpret_cast<float4*>(to + m * D + 32 * j + 2 * e) =
              make_float4(acc[m][j][e] * by, acc[m][j][e + 1] * by, acc[m][j][e + 2] * by, acc[m][j][e + 3] * by);
        }
    return;
  }
  const float lam = a.lam[int64_t(h) * a.lam_stride];
  uint16_t* dq = in ? static_cast<uint16_t*>(a.dq) + ((int64_t(b) * a.queries + t) * 2 * a.heads + 2 * h) * a.dim : nullptr;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      acc[0][j][e] *= a.scale * by1;
      acc[1][j][e] *= -(lam * a.scale) * by2;
    }
    store_turned(dq, acc[0][j], j, a.dim, half);
    store_turned(dq != nullptr ? dq + a.dim : nullptr, acc[1][j], j, a.dim, half);
  }
}

// dq of the parts of the keys, in order: 4 columns of a row
template <int D>
__device__ __forceinline__ void join_dq(const mmuon_attention_args& a, int parts, const RowSpace& space, int64_t id) {
  const int64_t row = id / (D / 2), all = int64_t(a.batch) * a.heads * a.queries;
  if (row >= all) return;
  const int c = int(id - row * (D / 2)) * 4, m = c >= D, col = c - m * D, t = int(row % a.queries);
  const int64_t bh = row / a.queries, b = bh / a.heads, h = bh - b * a.heads;
  const float* from = space.dq + row * (2 * D) + c;
  float s[4] = {};
#pragma unroll 8
  for (int p = 0; p < parts; ++p) {
    const float4 x = *reinterpret_cast<const float4*>(from + p * all * (2 * D));
    s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w;
  }
  if (col >= a.dim) return;
  const float by = m ? -(a.lam[h * a.lam_stride] * a.scale) : a.scale;
  uint16_t* to = static_cast<uint16_t*>(a.dq) + ((b * a.queries + t) * 2 * a.heads + 2 * h + m) * a.dim + col;
  *reinterpret_cast<uint2*>(to) = make_uint2(f2bf2(s[0] * by, s[1] * by), f2bf2(s[2] * by, s[3] * by));
}

// dlam[h]: its rows of all sequences and parts, which may cancel, in 64 bits, in order by thread and then in a
// tree; 256 threads, each with loads in flight also where sequences are short (4096 x 4 tokens, 8 heads: a pass
// 2800 us with a sequence after the other, 1610 so)
__device__ __forceinline__ void sum_dlam(const mmuon_attention_args& a, int parts, const RowSpace& space, int h, double* scratch) {
  double s = 0.0;
  const int64_t all = int64_t(parts) * a.batch * a.queries;
  const int over = 256 / max(a.queries, 1), rest = 256 - over * a.queries;
  int i = int(threadIdx.x) / max(a.queries, 1), t = int(threadIdx.x) - i * a.queries;
#pragma unroll 8
  for (int64_t n = threadIdx.x; n < all; n += 256) {
    s += space.dlam[(int64_t(i) * a.heads + h) * a.queries + t];
    i += over;
    t += rest;
    if (t >= a.queries) t -= a.queries, ++i;
  }
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.dlam[h] = float(scratch[0] + scratch[1] + scratch[2] + scratch[3]);
}
__global__ __launch_bounds__(256) void attention_dlam(mmuon_attention_args a, int parts, RowSpace space) {
  __shared__ double scratch[4];
  sum_dlam(a, parts, space, blockIdx.x, scratch);
}

// dk and dv: 32 keys to a wave, over the query rows of the heads that share them, 32 at a time.  The
// keys are operands in registers, the values, whose product comes once for both maps, in LDS.  With heads of
// 2 x 64 a lane has 14 registers too few for two waves to a SIMD, 60 B of scratch (16 x 1024 tokens, 8 heads: 20
// of the 88 MB that are written); two waves are worth it (188 -> 128 us).  The
// workgroups from `dlam_at` on sum dlam, a head each, which would take a launch of its own (5 to 8 us).
template <int D, int WAVES, int SLOTS, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES, D == 128 ? 1 : 2) void attention_dkv(mmuon_attention_args a, Dealing dealt, int parts,
                                                                              int dlam_at, int of_keys, RowSpace space) {
  constexpr int CA = D / 8, CB = D / 4, TQ = 32;
  using T = Tile<D, TQ, WAVES>;
  constexpr int BYTES = T::BYTES + 1024;  // and the rows' statistics
  constexpr int LOADS = T::LOADS + 1;
  __shared__ __attribute__((aligned(1024))) char ring[SLOTS * BYTES];
  __shared__ __attribute__((aligned(1024))) char values[WAVES * 32 * CB * 16];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (int(blockIdx.x) >= dlam_at) {
    static_assert(WAVES == 4, "256 threads");
    return sum_dlam(a, of_keys, space, blockIdx.x - dlam_at, reinterpret_cast<double*>(ring));
  }
  int group, item;
  if (!deal(dealt, a.batch * a.kv_heads, group, item)) return;
  // the first keys are seen by the most queries: first
  const int tile = SPLIT ? item / parts : item, part = SPLIT ? item % parts : 0;
  const int b = group / a.kv_heads, g = group % a.kv_heads, share = a.heads / a.kv_heads;
  const Span span = span_of(a, b);
  const int c0 = tile * 32 * WAVES, w0 = c0 + 32 * wave;  // first key of the workgroup, the wave
  const int key = w0 + (lane & 31);
  // the first query that sees a key
  const auto first_of = [&](int k) -> int {
    if (k >= span.keys) return a.queries;
    if (!a.causal) return 0;
    const int64_t t = k - span.first;
    return t <= 0 ? 0 : t < a.queries ? int(t) : a.queries;
  };
  const int from = first_of(c0) / TQ * TQ, mine = first_of(w0), own = first_of(key);
  const int full = first_of(w0 + 31);  // from here on every key of the wave is seen
  const int none = first_of(0);        // the queries before see nothing, and their rows may hold anything
  const int steps = (a.queries - from + TQ - 1) / TQ, all = steps * share;
  const int i0 = SPLIT ? int(int64_t(all) * part / parts) : 0, n = (SPLIT ? int(int64_t(all) * (part + 1) / parts) : all) - i0;
  const int head0 = SPLIT && n > 0 ? i0 / steps : 0, first0 = from + (i0 - head0 * steps) * TQ;

  const char* q1 = static_cast<const char*>(a.q) + 2 * (b * a.q_stride[0] + 2 * g * share * a.q_stride[2]);
  const char* g0 = static_cast<const char*>(a.dout) + 2 * (int64_t(b) * a.queries * a.heads + g * share) * 2 * a.dim;
  TileRows src;
  src.a_stride = uint32_t(2 * a.q_stride[1]);
  src.b_stride = uint32_t(2) * a.heads * 2 * a.dim;
  src.a_last = a.dim / 8 - 1;
  src.b_last = a.dim / 4 - 1;
  const uint32_t lds = lds_addr(ring);
  uint32_t off[T::LOADS];
  T::offsets(src, wave, lane, off);
  int next_head = head0, next_first = first0;  // of the tile that is loaded next
  const auto load = [&](int i) {
    const int head = next_head, first = next_first;
    next_first += TQ;
    if (next_first >= a.queries) next_first = from, ++next_head;
    const char* q = q1 + 2 * (2 * head * a.q_stride[2] + first * a.q_stride[1]);
    const uint32_t to = lds + (i % SLOTS) * BYTES;
    T::load(to, q, q + 2 * a.q_stride[2], g0 + 2 * (int64_t(first) * a.heads + head) * 2 * a.dim, src, off, a.queries - first, wave, lane, none - first);
    // (every wave loads them, so that each has as many loads)
    const float4* stats = space.stats + (int64_t(b) * a.heads + g * share + head) * a.queries + first;
    dma16(uniform_ptr(stats), uint32_t(min(lane, a.queries - first - 1)) * 16, to + T::BYTES);
  };

  // a sequence without keys reads its first row; nothing of it is stored
  const int last = max(span.keys, 1) - 1;
  bf16x8 k[2][D / 16];
  {
    const uint16_t* p = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + min(key, last) * a.k_stride[1] + 2 * g * a.k_stride[2];
    load_operands(p, a.dim, half, k[0]);
    load_operands(p + a.k_stride[2], a.dim, half, k[1]);
    const uint16_t* v = static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + g * a.v_stride[2];
#pragma unroll
    for (int i = 0; i < CB / 2; ++i) {  // the wave's own rows
      const int r = (i * 64 + lane) / CB, c = min(((i * 64 + lane) % CB) ^ chunk_mask<CB>(r), src.b_last);
      const int row = min(w0 + r, last) - min(w0, last);
      dma16(uniform_ptr(v + min(w0, last) * a.v_stride[1]), uint32_t(row) * uint32_t(2 * a.v_stride[1]) + uint32_t(c) * 16,
            lds_addr(values) + (wave * (CB / 2) + i) * 1024);
    }
  }
  const float scale = scale_of(a);
  f32x16 dv[D / 16], dk[2][D / 32];
#pragma unroll
  for (int j = 0; j < D / 16; ++j) dv[j] = f32x16{};
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) dk[m][j] = f32x16{};

#pragma unroll
  for (int i = 0; i < SLOTS - 1; ++i)
    if (i < n) load(i);
  wait_loaded();
  const uint32_t abase0 = row_base<CA>(lane), bbase0 = row_base<CB>(lane), ta0 = turned_base<CA>(lane), tb0 = turned_base<CB>(lane);
  char* mine_v = values + wave * (CB / 2) * 1024;
  if (a.dim < D) {  // columns that are not there: the other operand's repeat its last ones
#pragma unroll
    for (int i = 0; i < CB / 2; ++i) {
      const int r = (i * 64 + lane) / CB, c = ((i * 64 + lane) % CB) ^ chunk_mask<CB>(r);
      if (c > src.b_last) *reinterpret_cast<uint4*>(mine_v + (i * 64 + lane) * 16) = make_uint4(0, 0, 0, 0);
    }
  }
  int head = head0, first = first0 - TQ;
  for (int i = 0; i < n; ++i) {
    first += TQ;
    if (first >= a.queries) first = from, ++head;
    if (i + SLOTS - 2 < n) wait_vm<(SLOTS - 2) * LOADS>();
    else wait_vm<0>();
    barrier_after_lds_writes();
    if (i + SLOTS - 1 < n) load(i + SLOTS - 1);
    const char* tile_at = ring + (i % SLOTS) * BYTES;
    if (first + TQ <= mine) continue;  // no key of this wave is seen
    const float4* stats = reinterpret_cast<const float4*>(tile_at + T::BYTES) + 4 * half;
    const float lam = load_uniform(a.lam + int64_t(g * share + head) * a.lam_stride);
    f32x16 s[2] = {f32x16{}, f32x16{}}, dp = f32x16{};
    const uint32_t abase = fresh(abase0), bbase = fresh(bbase0);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      s[0] = mfma(read_rows<CA>(tile_at, abase, 0, kk), k[0][kk], s[0]);
      s[1] = mfma(read_rows<CA>(tile_at + T::A2, abase, 0, kk), k[1][kk], s[1]);
    }
#pragma unroll
    for (int kk = 0; kk < D / 8; ++kk) dp = mfma(read_rows<CB>(tile_at + T::B, bbase, 0, kk), read_rows<CB>(mine_v, bbase, 0, kk), dp);
    float p[16], d1[16], d2[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float4 st = stats[8 * (e / 4) + e % 4];
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][e], scale, -st.x));
      const float p2 = __builtin_amdgcn_exp2f(fmaf(s[1][e], scale, -st.z)) * lam;
      p[e] = p1 - p2;
      d1[e] = p1 * (dp[e] - st.y);
      d2[e] = p2 * (st.w - dp[e]);
    }
    if (first < full || first + TQ > a.queries) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int t = first + 8 * (e / 4) + 4 * half + e % 4;
        if (t < own || t >= a.queries) p[e] = d1[e] = d2[e] = 0.f;
      }
    }
    const bf16x8 x[2] = {operand(p), operand(p + 8)}, x1[2] = {operand(d1), operand(d1 + 8)}, x2[2] = {operand(d2), operand(d2 + 8)};
    const uint32_t ta = fresh(ta0), tb = fresh(tb0);
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int y = 0; y < 2; ++y) dv[j] = mfma(read_turned<CB>(tile_at + T::B, tb, 16 * y, j), x[y], dv[j]);
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        dk[0][j] = mfma(read_turned<CA>(tile_at, ta, 16 * y, j), x1[y], dk[0][j]);
        dk[1][j] = mfma(read_turned<CA>(tile_at + T::A2, ta, 16 * y, j), x2[y], dk[1][j]);
      }
  }
  if (own >= a.queries) {  // nobody sees the key: 0, where the products have 0 * NaN if a query or its dO holds one
#pragma unroll
    for (int j = 0; j < D / 16; ++j) dv[j] = f32x16{};
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < D / 32; ++j) dk[m][j] = f32x16{};
  }
  const bool in = key < a.keys;
  if constexpr (SPLIT) {
    if (!in) return;
    float* to = space.dkv + ((int64_t(group) * parts + part) * a.keys + key) * (4 * D) + 4 * half;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {  // dv, dk of both maps
      const f32x16& acc = j < D / 16 ? dv[j] : j < 3 * D / 32 ? dk[0][j - D / 16] : dk[1][j - 3 * D / 32];
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<float4*>(to + 32 * j + 2 * e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
    }
    return;
  }
  uint16_t* to_k = in ? static_cast<uint16_t*>(a.dk) + ((int64_t(b) * a.keys + key) * 2 * a.kv_heads + 2 * g) * a.dim : nullptr;
  uint16_t* to_v = in ? static_cast<uint16_t*>(a.dv) + ((int64_t(b) * a.keys + key) * a.kv_heads + g) * 2 * a.dim : nullptr;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) store_turned(to_v, dv[j], j, 2 * a.dim, half);
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int e = 0; e < 16; ++e) dk[m][j][e] *= a.scale;
      store_turned(in ? to_k + m * a.dim : nullptr, dk[m][j], j, a.dim, half);
    }
  }
}

// dk and dv of the parts of the queries, in order: 4 columns of a key
template <int D>
__device__ __forceinline__ void join_dkv(const mmuon_attention_args& a, int parts, const RowSpace& space, int64_t id) {
  const int64_t row = id / D, all = int64_t(a.batch) * a.kv_heads * a.keys;
  if (row >= all) return;
  const int c = int(id - row * D) * 4, key = int(row % a.keys);
  const int64_t group = row / a.keys, b = group / a.kv_heads, g = group - b * a.kv_heads;
  const float* from = space.dkv + (group * parts * a.keys + key) * (4 * D) + c;
  float s[4] = {};
#pragma unroll 8
  for (int p = 0; p < parts; ++p) {
    const float4 x = *reinterpret_cast<const float4*>(from + int64_t(p) * a.keys * (4 * D));
    s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w;
  }
  const bool is_v = c < 2 * D;
  const int m = c >= 3 * D, col = is_v ? c : c - (2 + m) * D;
  if (col >= (is_v ? 2 * a.dim : a.dim)) return;
  const float by = is_v ? 1.f : a.scale;
  const int64_t at = b * a.keys + key;
  uint16_t* to = is_v ? static_cast<uint16_t*>(a.dv) + (at * a.kv_heads + g) * 2 * a.dim + col
                      : static_cast<uint16_t*>(a.dk) + (at * 2 * a.kv_heads + 2 * g + m) * a.dim + col;
  *reinterpret_cast<uint2*>(to) = make_uint2(f2bf2(s[0] * by, s[1] * by), f2bf2(s[2] * by, s[3] * by));
}
// Both: the first `of_dq` workgroups dq's
template <int D>
__global__ __launch_bounds__(256) void attention_join(mmuon_attention_args a, int of_dq, int of_keys, int of_rows, RowSpace space) {
  if (int(blockIdx.x) < of_dq) join_dq<D>(a, of_keys, space, int64_t(blockIdx.x) * 256 + threadIdx.x);
  else join_dkv<D>(a, of_rows, space, int64_t(blockIdx.x - of_dq) * 256 + threadIdx.x);
}

int template_dim(const mmuon_attention_args& a) { return a.dim > 64 ? 128 : a.dim > 32 ? 64 : 32; }
// Parts of a loop of `most` steps that the estimate finds shortest, each of eight steps at least.  Parts whose sums take
// over 4 GiB have to make it 5% shorter: rounds of hundreds of workgroups that end a little earlier do not (no mask, 1 x 52858
// tokens, 22 heads of 2 x 112: two parts 292 ms and 15.6 GB held in a pass, one 290 and 10.8; 35 x 10013, 16 of 2 x 96 on 2: three
// 279 and 31.5, one 282 and 27.2; 4 x 222563, 96 of 2 x 72 on 24 would have taken 89 GB for them).
int fewest_us(const Items& n, const Pace& p, double part_bytes) {
  int best = 1;
  double least = estimate(n, p, 1, part_bytes);
  for (int splits = 2; splits <= 16 && splits * 8 <= n.most; ++splits) {
    const double t = estimate(n, p, splits, part_bytes);
    if (t < (splits * part_bytes > 4294967296.0 ? 0.95 : 1.0) * least) least = t, best = splits;
  }
  return best;
}
// Pairs of a query and a key that it sees, of one head
double seen_pairs(const mmuon_attention_args& a) {
  const double q = a.queries, k = a.keys;
  return !a.causal ? q * k : k >= q ? q * k - q * q / 2 : k * k / 2;
}
constexpr int KEY_WAVES = 4, ROW_WAVES = 4;
// Parts of the queries (of all heads that share the keys).  Units of the estimate are steps of 32 queries.  us
// of all launches of a pass, dk and dv in one part / in as many as fill the chip / in those that the estimate takes:
// heads of 2 x 64, 3 x 1001 tokens, 6 heads on 2 231 / 86 / 86 (10); 1 x 8192, 4 heads 670 / 433 / 385 (3), 1 head 534 / 149 /
// 149; of 2 x 128, 8192, 4 heads 1192 / 1192 / 910 (2), 4096, 16 heads on 4 1772 / 1071 / 751 (4): under a causal mask
// the first keys' workgroups are much longer than the mean.
int key_parts(const mmuon_attention_args& a) {
  const int64_t tiles = int64_t(a.batch) * a.kv_heads * ((a.keys + 32 * KEY_WAVES - 1) / (32 * KEY_WAVES));
  if (tiles == 0 || a.queries == 0 || a.heads == 0) return 1;
  const double share = a.heads / a.kv_heads / 32.0;
  const Items n{tiles, share * (a.causal ? std::min(a.queries, a.keys) : a.queries), share * seen_pairs(a) / a.keys,
                share * (!a.causal || a.keys / 2 >= a.queries ? a.queries : 0)};
  const Pace p = a.dim > 64 ? Pace{256, 2.7, 2.7, 22, 8e6} : Pace{512, 2.3, 1.7, 20, 8e6};
  return fewest_us(n, p, double(a.batch) * a.kv_heads * a.keys * 4 * template_dim(a) * 4);
}
// Parts of the keys, likewise.  8192 tokens, 4 heads of 2 x 128: dq in one part 1192 us, in two 1036; 4096 tokens,
// 4 heads of 2 x 64: one 233, four 148.
int64_t row_tiles(const mmuon_attention_args& a) {
  return (int64_t(a.heads / a.kv_heads) * a.queries + 32 * ROW_WAVES - 1) / (32 * ROW_WAVES);
}
int row_parts(const mmuon_attention_args& a) {
  const int64_t tiles = int64_t(a.batch) * a.kv_heads * row_tiles(a);
  if (tiles == 0 || a.keys == 0) return 1;
  const Items n{tiles, a.keys / 32.0, seen_pairs(a) / a.queries / 32, (a.causal ? std::max(0, a.keys - a.queries) : a.keys) / 32.0};
  const Pace p = a.dim > 64 ? Pace{256, 1.6, 1.6, 20, 8e6} : Pace{512, 1.45, 0.95, 18, 8e6};
  return fewest_us(n, p, double(a.batch) * a.heads * a.queries * 2 * template_dim(a) * 4);
}

struct BackwardLayout {
  size_t dlam, dq, dkv, total;  // floats; the rows' statistics come first
};
BackwardLayout backward_layout(const mmuon_attention_args& a) {
  const size_t rows = size_t(a.batch) * a.heads * a.queries, keys = size_t(a.batch) * a.kv_heads * a.keys;
  const size_t d = template_dim(a), of_keys = row_parts(a), of_rows = key_parts(a);
  const auto up = [](size_t n) { return (n + 63) / 64 * 64; };
  BackwardLayout l;
  l.dlam = up(rows * 4);
  l.dq = l.dlam + up(rows * of_keys);
  l.dkv = l.dq + (of_keys > 1 ? up(rows * of_keys * 2 * d) : 0);
  l.total = l.dkv + (of_rows > 1 ? up(keys * of_rows * 4 * d) : 0);
  return l;
}

template <int D>
void backward_dim(const mmuon_attention_args& a, hipStream_t s) {
  const int64_t rows = int64_t(a.batch) * a.heads * a.queries, keys = int64_t(a.batch) * a.kv_heads * a.keys;
  const int64_t groups = int64_t(a.batch) * a.kv_heads;
  const BackwardLayout l = backward_layout(a);
  float* ws = static_cast<float*>(a.workspace);
  const RowSpace space{reinterpret_cast<float4*>(ws), ws + l.dlam, ws + l.dq, ws + l.dkv};
  const int of_keys = row_parts(a), of_rows = key_parts(a);
  const bool dq = a.dq != nullptr && rows > 0, dkv = a.dk != nullptr && keys > 0;
  if (rows > 0) hipLaunchKernelGGL(attention_rows, dim3(unsigned((rows + 15) / 16)), dim3(256), 0, s, a, space);
  if (dq) {
    const Dealing d = dealing(groups, row_tiles(a) * of_keys);
    const dim3 grid(blocks_of(d)), block(64 * ROW_WAVES);
    if (of_keys == 1) hipLaunchKernelGGL((attention_dq<D, ROW_WAVES, 3, false>), grid, block, 0, s, a, d, of_keys, space);
    else hipLaunchKernelGGL((attention_dq<D, ROW_WAVES, 3, true>), grid, block, 0, s, a, d, of_keys, space);
  }
  const int heads = a.dlam != nullptr ? a.heads : 0, summed = rows > 0 ? of_keys : 0;
  if (dkv) {
    const Dealing d = dealing(groups, (a.keys + 32 * KEY_WAVES - 1) / (32 * KEY_WAVES) * int64_t(of_rows));
    const unsigned blocks = blocks_of(d);
    const dim3 grid(blocks + heads), block(64 * KEY_WAVES);
    if (of_rows == 1) hipLaunchKernelGGL((attention_dkv<D, KEY_WAVES, 2, false>), grid, block, 0, s, a, d, of_rows, int(blocks), summed, space);
    else hipLaunchKernelGGL((attention_dkv<D, KEY_WAVES, 2, true>), grid, block, 0, s, a, d, of_rows, int(blocks), summed, space);
  } else if (heads > 0) {
    hipLaunchKernelGGL(attention_dlam, dim3(unsigned(heads)), dim3(256), 0, s, a, summed, space);
  }
  const int64_t q = dq && of_keys > 1 ? (rows * (D / 2) + 255) / 256 : 0, k = dkv && of_rows > 1 ? (keys * D + 255) / 256 : 0;
  if (q + k > 0) hipLaunchKernelGGL(attention_join<D>, dim3(unsigned(q + k)), dim3(256), 0, s, a, int(q), of_keys, of_rows, space);
}

}  // namespace

size_t attention_backward_workspace(const mmuon_attention_args& a) { return backward_layout(a).total * 4; }

int launch_attention_bwd(const mmuon_attention_args& a, hipStream_t s) {
  if (a.dim > 64) backward_dim<128>(a, s);
  else if (a.dim > 32) backward_dim<64>(a, s);
  else backward_dim<32>(a, s);
  return 0;
}

}  // namespace mmuon
