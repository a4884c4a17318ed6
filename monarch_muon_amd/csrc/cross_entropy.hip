// Softmax cross entropy of a linear head, loss and gradients, without keeping the logits.
//
// x (T, D), w (V, D) bf16, target y (T):
//   l_tv = x_t . w_v      lse_t = log sum_v exp l_tv      nll_t = lse_t - l_{t, y_t}
//   dl_tv = g_t (exp(l_tv - lse_t) - [v == y_t])          dx = dl w      dw = dl^T x
// g_t: the gradient of the loss by nll_t (1 / valid tokens, 1, or given), 0 for ignored ones.
//
// Tokens whose target is ignored take no part: head_compact lists the others, every
// product runs over that list (its length stays on the device), and x is gathered first where
// the list is not all tokens, so what such a row of x holds reaches nothing.
//
// The logits are made once, 6 T V D operations in all.  A piece of tokens at a time: the
// first product's epilogue (logits as vocabulary x tokens, so that a lane holds 64 or so
// logits of one token) takes the maximum and the sum of exponentials of each part of the
// vocabulary that a wave holds, and stores every logit as a 16-bit code: its distance below
// the part's maximum in base-2 fixed point, step 64 / 65535.  head_rows joins the parts'
// statistics into lse and turns the codes of a row into bf16 dl where they stand.  A code
// gives p with a relative error of 3.4e-4 at most, however small p is, a tenth of bf16's own
// rounding of dl (exponentials kept in bf16 would be rounded twice); what lies 64 binades
// below its part's maximum (p < 6e-20) counts as zero.  The target's logit is kept in fp32: the loss
// and p_y - 1 do not go through a code.  One factor 1 / valid tokens is applied to the
// fp32 sums of dx and dw and not to dl, and dx adds what bf16 took from its largest term,
// p_y - 1: with them in dl, its rounding was one for all tokens, up to 2^-8.
//
// What bounds it, at 4096 tokens of 50304 x 4096: three products of 1.69 TFLOP, 1.42 ms with
// statistics and codes, 1.23 (dx) and 1.21 (dw), 1.19 to 1.40 PFLOP/s; the matrix cores are 63,
// 76 and 79% busy at 1.7 to 1.8 GHz, and the package-power limit holds the clock 80% of the
// time.  One token: the read of the head, 412 MB in 89 us.  Narrow models (16384 tokens x 1024):
// 10 B of memory traffic per logit (code out, in, dl out, in twice) beside 6144 operations.
#include <float.h>

#include <algorithm>

#include "common.hpp"
#include "gemm_pipe.hpp"
#include "head_plan.hpp"
#include "kernels.hpp"

namespace mmuon {
namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.693147180559945309417f;
constexpr float CODE_RANGE = 64.f;               // binades below the part's maximum
constexpr float CODE_STEP = CODE_RANGE / 65535.f;
constexpr int CODE_ZERO = 65535;                 // p = 0

// What a product's epilogue does
enum {
  EP_STATS = 0,  // logits: statistics of each part, the targets' logits
  EP_CODES = 1,  // the same, and the codes
  EP_CODES_PAST = 2,  // the same, stored past the caches
  EP_ROWS = 3,   // bf16 result, rows = columns of the tile; or fp32 accumulators of a part of K
  EP_PAST = 4    // the same, rows stored past the caches
};

// D (M x N) = A (M x K) B^T (N x K), where N (logits, dx) or K (dw) are the piece's tokens:
// compact tokens t0 .. of *count, at most `piece`.
struct HeadGemm {
  GOp a, b;
  int M, N, K;
  int tiles_m, tiles_n;
  int full, S;                   // tiles from `full` on are split over K in S
  const int* count;
  int t0, piece, tokens;
  const char* x;                 // x itself, read instead of the gathered rows where no token is ignored
  int64_t xstride;
  char* out;                     // EP_ROWS: column n at out + n ostride
  int64_t ostride;
  const int* rows;               // dx: the output row of a compact token
  const float* factor;           // the result's factor (device), or null
  const float* resid;            // dx: what rounding took from dl at the target, per compact token
  const uint16_t* w;
  int64_t wstride;
  int64_t vocab;
  float* frag;                   // accumulators in fragment order: BM x BN floats per virtual tile,
  int frag_first;                //   from this one on
  bool start;                    // they are what the sums begin with (a later piece of the tokens)
  bool keep;                     // they are kept for the next piece, of every tile
  uint16_t* codes;               // EP_CODES: [token][ldc]
  int64_t ldc;
  float2* parts;                 // [token][nparts]: maximum (base 2), sum of 2^(l - maximum)
  int nparts;
  const int64_t* target;         // of the compact tokens of the piece
  const float* nll;              // dw: sums the loss too, or null
  float* loss;
  int mean;
  float* tlogit;                 // [token]
};

// The sizes that the number of compact tokens decides
struct HeadSize {
  int N, K, tiles_m, tiles_n, full, splits;  // unsplit tiles, and parts of the others
  int S, kchunk;                             // K of a part
  bool all;                                  // no token is ignored
  // virtual tiles: both dealt to the XCDs by themselves
  __device__ __forceinline__ int vfull() const { return (full + 7) / 8 * 8; }
  __device__ __forceinline__ int vtiles() const { return vfull() + (splits + 7) / 8 * 8; }
};
enum { X_IS_A = 0, X_IS_B = 1, X_IS_NONE = 2 };  // which operand x is: of dw, of the logits, of dx
template <class GE, int X>
__device__ __forceinline__ HeadSize head_size(const HeadGemm& a) {
  // (no list: every token of the piece)
  const int count = a.count != nullptr ? *a.count : a.tokens, n = min(max(count - a.t0, 0), a.piece);
  HeadSize z;
  z.N = X == X_IS_A ? a.N : n;
  z.K = X == X_IS_A ? n : a.K;
  z.tiles_m = a.tiles_m;
  z.tiles_n = X == X_IS_A ? a.tiles_n : (n + GE::BN - 1) / GE::BN;
  z.full = min(a.full, z.tiles_m * z.tiles_n);
  z.splits = (z.tiles_m * z.tiles_n - z.full) * a.S;
  z.S = a.S;
  z.kchunk = ((z.K + a.S - 1) / a.S + BK - 1) / BK * BK;
  z.all = count == a.tokens;
  return z;
}

// The kernel's arguments, read again where they are used: held in scalar registers from the
// start, they would be spilled around the main loop.
__device__ __forceinline__ const HeadGemm& late_args() {
  auto p = (const __attribute__((address_space(4))) void*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const HeadGemm*)p;
}

// Virtual tile -> tile row and column, part of K.  Each XCD (v % 8) takes a contiguous run of
// tiles; the tiles of a run are numbered in patches PATCH tile columns wide, so the 32 tiles
// that an XCD's CUs hold at a time share 4 column and 8 row operand bands.
constexpr int PATCH = 4;
struct HeadTile {
  int idx;                       // < 0: none
  int m0, n0, kbeg, kend;
  bool split;
  __device__ __forceinline__ int slices() const { return max(kend - kbeg + BK - 1, 0) / BK; }
};
__device__ __forceinline__ int2 tile_place(int t, int tiles_m, int tiles_n) {  // (row, column) of tile t
  const int g = t / (tiles_m * PATCH), r = t - g * tiles_m * PATCH, width = min(PATCH, tiles_n - g * PATCH);
  const int tm = r / width;
  return make_int2(tm, g * PATCH + r - tm * width);
}
template <class GE>
__device__ __forceinline__ HeadTile head_tile(const HeadSize& z, int v) {
  const bool split = v >= z.vfull();
  const int w = split ? v - z.vfull() : v, n = split ? z.splits : z.full;
  const int per = (n + 7) >> 3, local = w >> 3, i = (w & 7) * per + local;
  if (local >= per || i >= n) return HeadTile{-1, 0, 0, 0, 0, split};
  // part by part: neighbours read the same slices of K
  const int tail = z.tiles_m * z.tiles_n - z.full, part = split ? i / tail : 0, t = split ? z.full + i - part * tail : i;
  const int2 at = tile_place(t, z.tiles_m, z.tiles_n);
  return HeadTile{split ? z.full + (t - z.full) * z.S + part : i, at.x * GE::BM, at.y * GE::BN,
                  split ? part * z.kchunk : 0, split ? min(z.K, (part + 1) * z.kchunk) : z.K, split};
}

// The K slices of a workgroup's tiles as one stream through the LDS ring: behind the last
// slice of a tile come the first of the next, so its operands are on their way while the
// tile before is finished and stored, and the ring is filled once per launch.  (Filled anew
// for every tile, with the result staged in it, a tile of 1024 of K took 4 us more of 40.)
template <class GE, bool AT, bool BT, int X>
struct Stream {
  static constexpr int RING = GE::RING, WI = GE::WI, WJ = GE::WJ, NM = WI * WJ, NR = WI + WJ;
  struct Fr {
    bf16x8 r[WI];
    bf16x8 c[WJ];
  };
  typedef f32x16 Acc[WI][WJ];
  // what is loaded next
  const char *pa, *pb;     // the operands' slices
  int64_t sa, sb;          // bytes to the next ones
  int left;                // slices of its tile from it on
  int v;                   // its virtual tile
  uint32_t loff[GE::DMA];  // per-lane byte offsets of the loads (OOB: beyond the extent, or no tile left)
  uint32_t tail[GE::DMA];  // OOB where the load's element lies beyond the last slice's K
  int wave, lane, wm, wn;
  char* lds;
  uint32_t lds0;
  uint32_t kfrag[BK / 16];
  uint32_t tfrag_r, tfrag_c;

  __device__ __forceinline__ const uint16_t* slot(uint32_t pos) const {
    return reinterpret_cast<const uint16_t*>(lds + (pos % RING) * GE::SLOTB);
  }
  __device__ __forceinline__ void open(const HeadSize& z) {  // the first tile from v on
    const int vtiles = z.vtiles();
    HeadTile t{-1, 0, 0, 0, 0, false};
    for (; v < vtiles; v += gridDim.x) {
      t = head_tile<GE>(z, v);
      if (t.idx >= 0 && t.slices() > 0) break;
      t.idx = -1;
    }
    left = 1;
    if (t.idx < 0) {  // nothing left: loads that read zeros
#pragma unroll
      for (int q = 0; q < GE::DMA; ++q) loff[q] = OOB;
      v = vtiles - int(gridDim.x);
      return;
    }
    const HeadGemm& a = late_args();
    GOp oa = a.a, ob = a.b;
    if (X != X_IS_A) ob.extent = z.N;
    if (X == X_IS_A && z.all) oa.base = a.x, oa.kstride = a.xstride;
    if (X == X_IS_B && z.all) ob.base = a.x, ob.mstride = a.xstride;
    pa = oa.base + mn_off(oa, t.m0) + t.kbeg * oa.kstride;
    pb = ob.base + mn_off(ob, t.n0) + t.kbeg * ob.kstride;
    sa = BK * oa.kstride;
    sb = BK * ob.kstride;
    left = t.slices();
    const int rem = t.kend - t.kbeg - (left - 1) * BK;  // K of the last slice
#pragma unroll
    for (int q = 0; q < GE::DMA; ++q) {
      const bool row = q < GE::RL;
      const int u = row ? GE::RL * wave + q : GE::CL * wave + q - GE::RL;
      loff[q] = row ? lane_offset<AT>(oa, t.m0, u, lane) : lane_offset<BT>(ob, t.n0, u, lane);
      const int kd = (row ? AT : BT) ? 16 * (u & 1) + (lane >> 2) : 8 * ((lane & 3) ^ ((lane >> 4) & 3));
      tail[q] = kd >= rem ? OOB : 0;
    }
  }
  // behind a load: the next slice, of the same tile (!SWITCH: known to be one) or the next
  template <bool SWITCH>
  __device__ __forceinline__ void advance(const HeadSize& z) {
    --left;
    if (!SWITCH || left > 0) {
      pa += sa;
      pb += sb;
    } else {
      v += gridDim.x;
      open(z);
    }
  }

  // Load Q (row operand first) of the next slice into the slot of stream position pos.  Load
  // u of an operand, K form: rows 16 u + lane/4, chunk (lane%4) ^ ((lane>>4)&3); T form: k rows
  // 16 (u%2) + lane/4, MN 32 (u/2) + 8 (lane%4).  Either lands at byte 1024 u of its slice.
  template <bool LAST, int Q>
  __device__ __forceinline__ void issue_one(uint32_t pos) const {
    constexpr bool ROW = Q < GE::RL;
    const int u = ROW ? GE::RL * wave + Q : GE::CL * wave + Q - GE::RL;
    const uint32_t dst = lds0 + (pos % RING) * GE::SLOTB + (ROW ? 0 : GE::RSLB) + u * 1024;
    bdma16(buffer_rsrc(ROW ? pa : pb), LAST && left == 1 ? loff[Q] | tail[Q] : loff[Q], dst);
  }
  template <bool LAST, int Q0, int Q1>
  __device__ __forceinline__ void issue(uint32_t pos) const {
    if constexpr (Q0 < Q1) {
      issue_one<LAST, Q0>(pos);
      issue<LAST, Q0 + 1, Q1>(pos);
    }
  }

  template <int KK, int G>
  __device__ __forceinline__ void load_one(uint32_t pos, Fr& f) const {
    const uint16_t* sr = slot(pos);
    const uint16_t* sc = sr + GE::RSLB / 2;
    if constexpr (G < WJ)
      f.c[G] = BT ? frag_rowmajor_tr(sc, tfrag_c + G * 2048, KK) : frag_kmajor(sc, kfrag[KK], (wn * WJ + G) * 32);
    else
      f.r[G - WJ] = AT ? frag_rowmajor_tr(sr, tfrag_r + (G - WJ) * 2048, KK)
                       : frag_kmajor(sr, kfrag[KK], (wm * WI + G - WJ) * 32);
  }
  template <int KK, int G0, int G1>
  __device__ __forceinline__ void load(uint32_t pos, Fr& f) const {
    if constexpr (G0 < G1) {
      load_one<KK, G0>(pos, f);
      load<KK, G0 + 1, G1>(pos, f);
    }
  }

  // MFMA g of a k step, with its share of the fragment reads of the next step and, in the
  // second k step, of the direct loads
  template <bool LAST, int KK, int g>
  __device__ __forceinline__ void half(uint32_t pos, const Fr& f, Fr& n, Acc& acc) const {
    if constexpr (g < NM) {
      acc[g / WJ][g % WJ] = mfma(f.r[g / WJ], f.c[g % WJ], acc[g / WJ][g % WJ]);
      if constexpr (KK == 0) {
        load<1, g * NR / NM, (g + 1) * NR / NM>(pos, n);
      } else {
        load<0, g * NR / NM, (g + 1) * NR / NM>(pos + 1, n);
        issue<LAST, g * GE::DMA / NM, (g + 1) * GE::DMA / NM>(pos + RING - 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      half<LAST, KK, g + 1>(pos, f, n, acc);
    }
  }
  // The slice at stream position pos (fa: its first k step's fragments, then the next slice's).
  // !LAST: the slice to load is not the last of its tile
  template <bool LAST>
  __device__ __forceinline__ void body(const HeadSize& z, uint32_t pos, Fr& fa, Fr& fb, Acc& acc) {
    half<LAST, 0, 0>(pos, fa, fb, acc);
    wait_vm<(RING - 3) * GE::DMA>();  // slice pos + 1 landed
    barrier();
    // raised wave priority from the barrier to the end of k step 1, so the SIMD's wave still in
    // this phase wins issue over one already in the next step
    __builtin_amdgcn_s_setprio(1);
    half<LAST, 1, 0>(pos, fb, fa, acc);
    __builtin_amdgcn_s_setprio(0);
    advance<LAST>(z);
  }
  // n slices from stream position pos on
  __device__ __forceinline__ void run(const HeadSize& z, int n, uint32_t& pos, Fr& fa, Fr& fb, Acc& acc) {
    while (n > 0) {
      for (int m = min(n, left - 1); m > 0; --m, --n) body<false>(z, pos++, fa, fb, acc);
      if (n > 0) {
        body<true>(z, pos++, fa, fb, acc);
        --n;
      }
    }
  }
  __device__ __forceinline__ void fill(const HeadSize& z, Fr& fa) {
    open(z);
    for (uint32_t q = 0; q < RING - 1; ++q) {
      issue<true, 0, GE::DMA>(q);
      advance<true>(z);
    }
    wait_vm<(RING - 2) * GE::DMA>();  // slice 0 landed
    barrier();
    load<0, 0, NR>(0, fa);
  }
};

// A 32 x 32 MFMA tile as 16-bit values, D[row][column] with a lane = one column, to memory in
// rows of its columns: w[q] holds rows 8 q + 4 (lane/32) .. + 3 of column lane%32.  Exchanged
// between halves and between rows of 16 lanes, a lane ends up with eight rows (16 B) of one
// column and a store of a wave writes 64 B of 16 columns.  fn(column, first row, 16 B)
template <class Fn>
__device__ __forceinline__ void store_block(uint2 (&w)[4], int lane, Fn&& fn) {
  uint32_t x[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const auto lo = __builtin_amdgcn_permlane32_swap(w[2 * h].x, w[2 * h + 1].x, false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap(w[2 * h].y, w[2 * h + 1].y, false, false);
    x[h][0] = lo[0];
    x[h][1] = hi[0];
    x[h][2] = lo[1];
    x[h][3] = hi[1];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const auto t = __builtin_amdgcn_permlane16_swap(x[0][k], x[1][k], false, false);
    x[0][k] = t[0];
    x[1][k] = t[1];
  }
  const int r = lane >> 4, row = ((r & 1) << 1 | r >> 1) * 8;
#pragma unroll
  for (int h = 0; h < 2; ++h) fn(h * 16 + (lane & 15), row, make_uint4(x[h][0], x[h][1], x[h][2], x[h][3]));
}

// Statistics and codes of a tile of logits: rows m0.. are vocabulary, columns n0.. tokens.
template <class GE, int EP>
__device__ __forceinline__ void loss_epilogue(const HeadGemm& a, int N, int m0, int n0, int wave, int lane,
                                              f32x16 (&acc)[GE::WI][GE::WJ]) {
  const int wm = wave / GE::GN, wn = wave % GE::GN;
  constexpr int PW = 32 * GE::WI;               // vocabulary of a part
  const int v0 = m0 + wm * PW, left = a.M - v0;  // rows from `left` on do not exist
  const int half = lane >> 5;
#pragma unroll
  for (int j = 0; j < GE::WJ; ++j) {
    const int row = (wn * GE::WJ + j) * 32 + (lane & 31), tok = n0 + row;
    const bool live = tok < N;
    const int64_t y = live ? a.target[tok] : -1;
    const int64_t rel = y - v0;
    const bool hit = rel >= 0 && rel < PW && rel < left && ((int(rel) >> 2) & 1) == half;
    if (__any(hit)) {
      // element (rel % 4) + 4 (rel / 8 % 4) + 16 (rel / 32) of the lane's, bit by bit, by masks
      // (a choice between elements becomes an index, and an index 2048 comparisons)
      const int at = (int(rel) >> 5) * 16 + ((int(rel) >> 3) & 3) * 4 + (int(rel) & 3);
      uint32_t l[GE::WI * 16];
#pragma unroll
      for (int i = 0; i < GE::WI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) l[i * 16 + r] = __float_as_uint(acc[i][j][r]);
#pragma unroll
      for (int n = GE::WI * 8; n > 0; n /= 2) {
        const uint32_t upper = at & n ? ~0u : 0u;
#pragma unroll
        for (int k = 0; k < n; ++k) l[k] = (l[k + n] & upper) | (l[k] & ~upper);
      }
      if (hit) a.tlogit[tok] = __uint_as_float(l[0]);
    }
    if (left < PW) {
      int limit = left - half * 4;
      asm volatile("" : "+v"(limit));  // (the comparisons of every j at once would take 128 registers)
#pragma unroll
      for (int i = 0; i < GE::WI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (i * 32 + (r >> 2) * 8 + (r & 3) >= limit) acc[i][j][r] = -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < GE::WI; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[i][j][r]);
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    // (bounded below: a part that is all -inf, or nearly, has sum 0)
    const float m2 = fmaxf(m * LOG2E, -FLT_MAX);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < GE::WI; ++i) {
      uint2 codes[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[e] = __builtin_fmaf(acc[i][j][4 * q + e], LOG2E, -m2);
          s += __builtin_amdgcn_exp2f(d[e]);
        }
        if constexpr (EP != EP_STATS) {
          constexpr float K = -1.f / CODE_RANGE;
          const uint32_t lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(d[0] * K, d[1] * K));
          const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(d[2] * K, d[3] * K));
          codes[q] = make_uint2(lo, hi);
        }
      }
      if constexpr (EP != EP_STATS) {
        store_block(codes, lane, [&](int c, int r, const uint4& u) {
          const int t = n0 + (wn * GE::WJ + j) * 32 + c;
          if (t >= N) return;
          uint16_t* to = a.codes + int64_t(t) * a.ldc + v0 + i * 32 + r;
          if constexpr (EP == EP_CODES_PAST) store16_nt(to, u);
          else *reinterpret_cast<uint4*>(to) = u;
        });
      }
    }
    s += __shfl_xor(s, 32, 64);
    if (m2 == INFINITY) s = NAN;  // beyond what 32 bits hold in base 2 (every distance would be infinite, the sum 0)
    if (live && half == 0 && left > 0) a.parts[int64_t(tok) * a.nparts + v0 / PW] = make_float2(m2, s);
  }
}

// The compact token's term that bf16 took from dl: v[0..3] (columns m .. m + 3 of dx) += resid w[y]
__device__ __forceinline__ void add_resid(const HeadGemm& a, int n, int m, float (&v)[4]) {
  const int64_t y = a.target[n];
  if (y < 0 || y >= a.vocab) return;
  const uint2 u = *reinterpret_cast<const uint2*>(a.w + y * a.wstride + m);
  const float r = a.resid[n];
  v[0] += r * __uint_as_float(u.x << 16);
  v[1] += r * __uint_as_float(u.x & 0xffff0000u);
  v[2] += r * __uint_as_float(u.y << 16);
  v[3] += r * __uint_as_float(u.y & 0xffff0000u);
}

// Accumulators in fragment order: float4 q of MFMA tile (i, j) of a wave at 64 lanes x 16 B.
// Where a lane's begin:
template <class GE>
__device__ __forceinline__ int64_t fragment(int64_t idx, int wave, int lane) {
  return (idx * GE::NW + wave) * (GE::WI * GE::WJ * 16 * 64) + lane * 4;
}
template <class GE>
__device__ __forceinline__ void add_fragments(const float* frag, f32x16 (&acc)[GE::WI][GE::WJ]) {
#pragma unroll
  for (int i = 0; i < GE::WI; ++i)
#pragma unroll
    for (int j = 0; j < GE::WJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 f = *reinterpret_cast<const float4*>(frag + ((i * GE::WJ + j) * 4 + q) * 256);
        acc[i][j][4 * q] += f.x;
        acc[i][j][4 * q + 1] += f.y;
        acc[i][j][4 * q + 2] += f.z;
        acc[i][j][4 * q + 3] += f.w;
      }
}

// What becomes of a tile's accumulators
template <class GE, int EP, int X>
__device__ __forceinline__ void finish(int N, const HeadTile& t, f32x16 (&acc)[GE::WI][GE::WJ]) {
  const HeadGemm& a = late_args();
  const int tid = fresh_tid();
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / GE::GN, wn = wave % GE::GN;
  float* frag = a.frag + fragment<GE>(t.idx - a.frag_first, wave, lane);
  if (EP >= EP_ROWS && a.start) add_fragments<GE>(frag, acc);
  if ((EP >= EP_ROWS && a.keep) || t.split) {
#pragma unroll
    for (int i = 0; i < GE::WI; ++i)
#pragma unroll
      for (int j = 0; j < GE::WJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(frag + ((i * GE::WJ + j) * 4 + q) * 256) =
              make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
    return;
  }
  if constexpr (EP >= EP_ROWS) {
    const float factor = a.factor != nullptr ? *a.factor : 1.f;
#pragma unroll
    for (int j = 0; j < GE::WJ; ++j) {
      const int n1 = t.n0 + (wn * GE::WJ + j) * 32, n = n1 + (lane & 31);
#pragma unroll
      for (int i = 0; i < GE::WI; ++i) {
        const int m1 = t.m0 + (wm * GE::WI + i) * 32;
        uint2 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          const int m = m1 + q * 8 + (lane >> 5) * 4;
          if (X == X_IS_NONE && n < N && m < a.M) add_resid(a, n, m, v);
          w[q] = make_uint2(f2bf2(v[0] * factor, v[1] * factor), f2bf2(v[2] * factor, v[3] * factor));
        }
        store_block(w, lane, [&](int c, int r, const uint4& u) {
          if (n1 + c >= N || m1 + r >= a.M) return;
          const int row = X == X_IS_NONE ? a.rows[n1 + c] : n1 + c;
          char* to = a.out + int64_t(row) * a.ostride + int64_t(m1 + r) * 2;
          if constexpr (EP == EP_PAST) store16_nt(to, u);
          else *reinterpret_cast<uint4*>(to) = u;
        });
      }
    }
  } else {
    loss_epilogue<GE, EP>(a, N, t.m0, t.n0, wave, lane, acc);
  }
}

// Sum of nll, divided by the number of targets that are not ignored where mean (NaN if there
// is none): each thread's share in order, then a tree (the same order every time for NTH threads)
template <int NTH>
__device__ __forceinline__ void sum_loss(const float* nll, int tokens, int count, int mean, float* loss,
                                         float* scratch) {
  float s = 0.f;
#pragma unroll 8
  for (int i = threadIdx.x; i < tokens; i += NTH) s += nll[i];
  s = block_sum<NTH>(s, scratch);
  if (threadIdx.x == 0) *loss = mean ? s / float(count) : s;
}

template <class GE, bool AT, bool BT, int EP, int X>
__global__ __launch_bounds__(GE::NTH, GE::PER_CU * GE::NW / 4) void head_gemm(HeadGemm a) {
  __shared__ __attribute__((aligned(1024))) char lds[GE::LDS];
  const HeadSize z = head_size<GE, X>(a);
  const int vtiles = z.vtiles();
  typedef Stream<GE, AT, BT, X> Pipe;
  Pipe p;
  p.lane = threadIdx.x & 63;
  p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  p.wm = p.wave / GE::GN;
  p.wn = p.wave % GE::GN;
  p.lds = lds;
  p.lds0 = lds_addr(lds);
#pragma unroll
  for (int kk = 0; kk < BK / 16; ++kk) p.kfrag[kk] = kmajor_frag_base(kk, p.lane);
  p.tfrag_r = rowmajor_frag_base(p.wm * GE::WI, p.lane);
  p.tfrag_c = rowmajor_frag_base(p.wn * GE::WJ, p.lane);
  p.v = blockIdx.x;
  typename Pipe::Fr fa, fb;
  p.fill(z, fa);
  uint32_t pos = 0;
  for (int v = blockIdx.x; v < vtiles; v += gridDim.x) {
    const HeadTile t = head_tile<GE>(z, v);
    if (t.idx < 0) continue;
    f32x16 acc[GE::WI][GE::WJ];
#pragma unroll
    for (int i = 0; i < GE::WI; ++i)
#pragma unroll
      for (int j = 0; j < GE::WJ; ++j) acc[i][j] = f32x16{};
    p.run(z, t.slices(), pos, fa, fb, acc);
    finish<GE, EP, X>(z.N, t, acc);
  }
  wait_vm<0>();  // no load is left in flight to LDS that another workgroup may own next
  // dw sums the loss: the last workgroup has no more tiles than any other
  if (X == X_IS_A && a.nll != nullptr && blockIdx.x == gridDim.x - 1) {
    barrier();  // every wave is done with the ring
    sum_loss<GE::NTH>(a.nll, a.tokens, *a.count, a.mean, a.loss, reinterpret_cast<float*>(lds));
  }
}

// The split tiles of the logits: a workgroup of one wave sums the parts of what one wave of the
// product held, in order, and goes on as if it had multiplied.
template <class GE, int EP>
__global__ __launch_bounds__(64) void head_logits_join(HeadGemm a) {
  const HeadSize z = head_size<GE, X_IS_B>(a);
  const int nth = blockIdx.x / GE::NW, wave = blockIdx.x % GE::NW, lane = threadIdx.x, t = z.full + nth;
  if (t >= z.tiles_m * z.tiles_n) return;
  const int2 at = tile_place(t, z.tiles_m, z.tiles_n);
  f32x16 acc[GE::WI][GE::WJ];
#pragma unroll
  for (int i = 0; i < GE::WI; ++i)
#pragma unroll
    for (int j = 0; j < GE::WJ; ++j) acc[i][j] = f32x16{};
  const float* f = a.frag + fragment<GE>(z.full + int64_t(nth) * z.S - a.frag_first, wave, lane);
  for (int k = 0; k < z.S; ++k) add_fragments<GE>(f + int64_t(k) * GE::BM * GE::BN, acc);
  loss_epilogue<GE, EP>(a, z.N, at.x * GE::BM, at.y * GE::BN, wave, lane, acc);
}

// Sum over the parts of K, in order, of one 32 x 32 MFMA tile of a split tile per workgroup:
// the fp32 partials in fragment order -> bf16 rows.
template <class GE, int X>
__global__ __launch_bounds__(256) void head_join(HeadGemm a) {
  constexpr int PER = GE::NW * GE::WI * GE::WJ;  // MFMA tiles of a tile
  const HeadSize z = head_size<GE, X>(a);
  const int nth = blockIdx.x / PER, in = blockIdx.x % PER, t = z.full + nth;
  if (t >= z.tiles_m * z.tiles_n) return;
  const int2 at = tile_place(t, z.tiles_m, z.tiles_n);
  const int wave = in / (GE::WI * GE::WJ), ij = in % (GE::WI * GE::WJ);
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int m = at.x * GE::BM + (wave / GE::GN * GE::WI + ij / GE::WJ) * 32 + q * 8 + (lane >> 5) * 4;
  const int n = at.y * GE::BN + (wave % GE::GN * GE::WJ + ij % GE::WJ) * 32 + (lane & 31);
  if (m >= a.M || n >= z.N) return;
  const float* f = a.frag + (int64_t(z.full + nth * z.S - a.frag_first) * PER + in) * 1024 + threadIdx.x * 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = 0; k < z.S; ++k) {
    const float4 u = *reinterpret_cast<const float4*>(f + int64_t(k) * PER * 1024);
    v[0] += u.x;
    v[1] += u.y;
    v[2] += u.z;
    v[3] += u.w;
  }
  if (X == X_IS_NONE) add_resid(a, n, m, v);
  const float c = a.factor != nullptr ? *a.factor : 1.f;
  *reinterpret_cast<uint2*>(a.out + int64_t(X == X_IS_NONE ? a.rows[n] : n) * a.ostride + int64_t(m) * 2) =
      make_uint2(f2bf2(v[0] * c, v[1] * c), f2bf2(v[2] * c, v[3] * c));
}

// ---------------------------------------------------------------------------
// Rows
// ---------------------------------------------------------------------------
struct RowArgs {
  uint16_t* codes;  // in: codes; out: dl (bf16)
  int64_t ldc;
  const float2* parts;
  int nparts, part_shift;  // parts of 2^part_shift
  const float* tlogit;
  const int64_t* target;   // compact
  const int* rows;         // the token of a compact token
  const int* count;
  int t0, piece;
  int64_t vocab, ignore;
  const float* grad;       // per token, or null: 1
  float* nll;              // per token
  float* resid;            // per compact token
  __device__ __forceinline__ int live() const { return min(max(*count - t0, 0), piece); }
};

// log2 of a token's sum of exponentials, joined from its parts by NTHR threads
// (one wave where NTHR == 64); valid in every thread.
template <int NTHR>
__device__ __forceinline__ float join_parts(const float2* p, int n, float* scratch) {
  constexpr int U = 4;
  float m = -INFINITY, s = 0.f;
  for (int i = threadIdx.x % NTHR; i < n; i += NTHR * U) {
    float2 t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) t[u] = i + u * NTHR < n ? p[i + u * NTHR] : make_float2(0.f, 0.f);
    float top = m;  // a part that is empty or all -inf has sum 0 and no maximum
#pragma unroll
    for (int u = 0; u < U; ++u) top = t[u].y == 0.f ? top : fmaxf(top, t[u].x);
    const bool any = top != -INFINITY;
    s = any ? s * __builtin_amdgcn_exp2f(m - top) : s;
#pragma unroll
    for (int u = 0; u < U; ++u) s += any && t[u].y != 0.f ? t[u].y * __builtin_amdgcn_exp2f(t[u].x - top) : t[u].y;
    m = top;
  }
  float top = wave_max(m);
  const int wave = threadIdx.x / 64 % (NTHR / 64);
  if constexpr (NTHR > 64) {
    if ((threadIdx.x & 63) == 0) scratch[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NTHR / 64; ++w) top = fmaxf(top, scratch[w]);
  }
  s = wave_sum(m == -INFINITY ? s : s * __builtin_amdgcn_exp2f(m - top));
  if constexpr (NTHR > 64) {
    if ((threadIdx.x & 63) == 0) scratch[NTHR / 64 + wave] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int w = 0; w < NTHR / 64; ++w) s += scratch[NTHR / 64 + w];
  }
  return top + __builtin_log2f(s);
}

__device__ __forceinline__ float token_nll(float lse2, float tlogit, int64_t y, int64_t vocab) {
  if (y < 0 || y >= vocab) return NAN;  // no such token: the loss shows it
  return (lse2 - tlogit * LOG2E) * LN2;
}

// The loss alone: NTHR threads per token.  Without a list of compact tokens (rows null) every
// token is one, ignored or not.
template <int NTHR>
__global__ __launch_bounds__(256) void head_nll(RowArgs a) {
  __shared__ float scratch[8];
  const int tok = blockIdx.x * (256 / NTHR) + threadIdx.x / NTHR;
  if (tok >= (a.rows != nullptr ? a.live() : a.piece)) return;
  const float lse2 = join_parts<NTHR>(a.parts + int64_t(tok) * a.nparts, a.nparts, scratch);
  if (threadIdx.x % NTHR != 0) return;
  const int64_t y = a.target[tok];
  const float nll = y == a.ignore ? 0.f : token_nll(lse2, a.tlogit[tok], y, a.vocab);
  a.nll[a.rows != nullptr ? a.rows[tok] : tok] = nll;
}

// One workgroup per token: lse, nll, and the row's codes -> dl.  Bound by its traffic, 4 B per
// logit: 4096 x 50304 in 149 us, 5.5 TB/s, where a large copy reaches 5.1.
template <bool PAST>
__global__ __launch_bounds__(256) void head_rows(RowArgs a) {
  __shared__ float scratch[8];
  const int tok = blockIdx.x;
  if (tok >= a.live()) return;
  const float2* parts = a.parts + int64_t(tok) * a.nparts;
  const float lse2 = join_parts<256>(parts, a.nparts, scratch);
  const int64_t y = a.target[tok];
  const int at = a.rows[tok];
  const float nll = token_nll(lse2, a.tlogit[tok], y, a.vocab);
  float g = a.grad != nullptr ? a.grad[at] : 1.f;
  if (y < 0 || y >= a.vocab) g = NAN;
  const float term = g * expm1f(-nll);  // g (p_y - 1), p_y near 1 included
  const uint16_t at_target = f2bf(term);
  if (threadIdx.x == 0) {
    a.nll[at] = nll;
    a.resid[tok] = term - bf2f(at_target);
  }
  uint16_t* row = a.codes + int64_t(tok) * a.ldc;
  const float none = lse2 * 0.f;  // a code of zero: p = 0, and no number where the token has no softmax
  for (int64_t c = threadIdx.x * 8; c < a.ldc; c += 256 * 8) {
    const uint4 in = PAST ? load16_nt(row + c) : *reinterpret_cast<const uint4*>(row + c);
    const uint32_t w[4] = {in.x, in.y, in.z, in.w};
    const int part = int(c >> a.part_shift);
    const float top = part < a.nparts ? parts[part].x - lse2 : 0.f;  // beyond: codes of zero
    uint32_t r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = w[k] & 0xffff, hi = w[k] >> 16;
      const float p0 = lo == CODE_ZERO ? none : __builtin_amdgcn_exp2f(__builtin_fmaf(float(lo), -CODE_STEP, top));
      const float p1 = hi == CODE_ZERO ? none : __builtin_amdgcn_exp2f(__builtin_fmaf(float(hi), -CODE_STEP, top));
      r[k] = f2bf2(g * p0, g * p1);
    }
    if (y >= c && y < c + 8) {
      const int e = int(y - c);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e >> 1 == k) r[k] = e & 1 ? (r[k] & 0xffff) | (uint32_t(at_target) << 16) : (r[k] & 0xffff0000u) | at_target;
    }
    *reinterpret_cast<uint4*>(row + c) = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

// The tokens that are not ignored, in order: rows[j], their targets, their number, and its
// inverse (0 where there is none).  A wave takes a run of the tokens.
__global__ __launch_bounds__(1024) void head_compact(const int64_t* target, int tokens, int64_t ignore, int* rows,
                                                     int64_t* compact, int* count, float* inverse) {
  __shared__ int found[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int run = (tokens + 1023) / 1024 * 64, t0 = wave * run, t1 = min(tokens, t0 + run);
  int c = 0;
#pragma unroll 4
  for (int t = t0 + lane; t < t1; t += 64) c += target[t] != ignore;
  c = wave_isum(c);
  if (lane == 0) found[wave] = c;
  __syncthreads();
  int at = 0, all = 0;
  for (int w = 0; w < 16; ++w) {
    at += w < wave ? found[w] : 0;
    all += found[w];
  }
#pragma unroll 4
  for (int t = t0; t < t1; t += 64) {
    const int64_t y = t + lane < t1 ? target[t + lane] : ignore;
    const uint64_t kept = __ballot(y != ignore);
    if (y != ignore) {
      const int j = at + __popcll(kept & ((uint64_t(1) << lane) - 1));
      rows[j] = t + lane;
      compact[j] = y;
    }
    at += __popcll(kept);
  }
  if (threadIdx.x == 0) {
    *count = all;
    *inverse = all > 0 ? 1.f / float(all) : 0.f;
  }
}

// One workgroup per row: the piece's rows of x gathered (nothing where no token is ignored),
// and, with the first piece, the zeros of ignored tokens in dx and nll.  head_list: both for
// one piece of few tokens, each workgroup counting the tokens before its own.
struct GatherArgs {
  const uint16_t* x;
  int64_t xstride;
  uint16_t* xc;
  int width, tokens, t0, piece;
  const int* rows;
  const int* count;
  const int64_t* target;
  int64_t ignore;
  uint16_t* dx;  // or null
  float* nll;
  int* list_rows;  // head_list: what head_compact writes
  int64_t* list_target;
  int* list_count;
  float* list_inverse;
};
__device__ __forceinline__ void copy_row(const GatherArgs& a, int to, int token) {
  const uint16_t* src = a.x + int64_t(token) * a.xstride;
  for (int c = threadIdx.x * 8; c < a.width; c += 128 * 8)
    *reinterpret_cast<uint4*>(a.xc + int64_t(to) * a.width + c) = *reinterpret_cast<const uint4*>(src + c);
}
__device__ __forceinline__ void ignored_row(const GatherArgs& a, int token) {
  if (threadIdx.x == 0) a.nll[token] = 0.f;
  if (a.dx != nullptr)
    for (int c = threadIdx.x * 8; c < a.width; c += 128 * 8)
      *reinterpret_cast<uint4*>(a.dx + int64_t(token) * a.width + c) = make_uint4(0, 0, 0, 0);
}
__global__ __launch_bounds__(128) void head_gather(GatherArgs a) {
  const int n = *a.count, j = blockIdx.x;
  if (n == a.tokens) return;
  if (j < a.piece && a.t0 + j < n) copy_row(a, j, a.rows[a.t0 + j]);
  if (a.t0 == 0 && j < a.tokens && a.target[j] == a.ignore) ignored_row(a, j);
}
constexpr int LIST_TOKENS = 1024;
__global__ __launch_bounds__(128) void head_list(GatherArgs a) {
  __shared__ int part[4];
  const int token = blockIdx.x;
  int before = 0, all = 0;
#pragma unroll
  for (int u = 0; u < LIST_TOKENS / 128; ++u) {
    const int t = u * 128 + threadIdx.x;
    const bool is = t < a.tokens && a.target[t] != a.ignore;
    before += is && t < token;
    all += is;
  }
  before = wave_isum(before);
  all = wave_isum(all);
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x >> 6] = before;
    part[2 + (threadIdx.x >> 6)] = all;
  }
  __syncthreads();
  before = part[0] + part[1];
  all = part[2] + part[3];
  const int64_t y = a.target[token];
  if (threadIdx.x == 0 && token == 0) {
    *a.list_count = all;
    *a.list_inverse = all > 0 ? 1.f / float(all) : 0.f;
  }
  if (y == a.ignore) {
    ignored_row(a, token);
    return;
  }
  if (threadIdx.x == 0) {
    a.list_rows[before] = token;
    a.list_target[before] = y;
  }
  if (all != a.tokens) copy_row(a, before, token);
}

// The loss without a list: the targets are counted here
__global__ __launch_bounds__(1024) void head_loss(const float* nll, int tokens, const int* count,
                                                  const int64_t* target, int64_t ignore, int mean, float* loss) {
  __shared__ float scratch[16];
  __shared__ int found[16];
  int c = 0;
  if (count == nullptr) {
    for (int i = threadIdx.x; i < tokens; i += 1024) c += target[i] != ignore;
    c = wave_isum(c);
    if ((threadIdx.x & 63) == 0) found[threadIdx.x >> 6] = c;
    c = 0;
    __syncthreads();
    for (int w = 0; w < 16; ++w) c += found[w];
  } else {
    c = *count;
  }
  sum_loss<1024>(nll, tokens, c, mean, loss, scratch);
}

__global__ __launch_bounds__(256) void head_zero(uint4* x, int64_t chunks) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < chunks; i += int64_t(gridDim.x) * 256)
    x[i] = make_uint4(0, 0, 0, 0);
}

// x and y *= *c, in 16-B chunks; nothing is touched where *c == 1.  Rounds once more, to bf16,
// where *c is no power of two.  4 B of traffic per element.
__global__ __launch_bounds__(256) void head_scale(uint16_t* x, int64_t nx, uint16_t* y, int64_t ny, const float* c) {
  const float f = *c;
  if (f == 1.f) return;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < nx + ny; i += int64_t(gridDim.x) * 256) {
    uint16_t* p = i < nx ? x + i * 8 : y + (i - nx) * 8;
    float v[8];
    Vec8<BF16T>::load(p, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= f;
    Vec8<BF16T>::store(p, v);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Tiles: 256 of the first operand (vocabulary, or width) x 256 or 128 of the second, eight
// waves, one workgroup per CU; 128 x 64, four waves, three workgroups per CU
typedef Geo<2, 4, 4, 2, 4> H256;
typedef Geo<4, 2, 2, 2, 4> H128;
typedef Geo<4, 1, 1, 2, 4> H64;

// M, N, K with all of the piece's tokens valid (head_size: the real ones)
void set_tiles(HeadGemm& a, int M, int N, int K, HeadPlan p) {
  a.M = M;
  a.N = N;
  a.K = K;
  a.tiles_m = cdiv(M, p.rows());
  a.tiles_n = cdiv(N, p.cols());
  a.full = p.full;
  a.S = p.S;
}

template <class GE, bool AT, bool BT, int EP, int X>
void launch_tile(const HeadGemm& a, int tiles, hipStream_t s) {
  const int grid = std::min((tiles + 7) / 8 * 8, resident_grid(1 << 30) * GE::PER_CU);
  hipLaunchKernelGGL((head_gemm<GE, AT, BT, EP, X>), dim3(grid), dim3(GE::NTH), 0, s, a);
}
template <bool AT, bool BT, int EP, int X>
void launch_head(const HeadGemm& a, HeadPlan p, hipStream_t s) {
  const int tiles = p.virtual_tiles(a.M, a.N);
  if (p.tile == T128) launch_tile<H128, AT, BT, EP, X>(a, tiles, s);
  else launch_tile<H256, AT, BT, EP, X>(a, tiles, s);
}
template <class GE, int X>
void launch_join_tile(const HeadGemm& a, hipStream_t s) {
  const int split = a.tiles_m * a.tiles_n - a.full;
  if (split > 0)
    hipLaunchKernelGGL((head_join<GE, X>), dim3(split * GE::NW * GE::WI * GE::WJ), dim3(256), 0, s, a);
}
template <int X>
void launch_join(const HeadGemm& a, HeadPlan p, hipStream_t s) {
  if (p.tile == T128) launch_join_tile<H128, X>(a, s);
  else launch_join_tile<H256, X>(a, s);
}

template <int EP>
void launch_logits(const HeadGemm& a, HeadPlan p, hipStream_t s) {
  if constexpr (EP == EP_STATS)
    if (p.tile == T64) return launch_tile<H64, false, false, EP, X_IS_B>(a, p.virtual_tiles(a.M, a.N), s);
  launch_head<false, false, EP, X_IS_B>(a, p, s);
  const int split = a.tiles_m * a.tiles_n - a.full;
  if (split > 0 && p.tile == T128) hipLaunchKernelGGL((head_logits_join<H128, EP>), dim3(split * H128::NW), dim3(64), 0, s, a);
  else if (split > 0) hipLaunchKernelGGL((head_logits_join<H256, EP>), dim3(split * H256::NW), dim3(64), 0, s, a);
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct Layout : HeadPlans {
  int64_t piece, ldc;
  int nparts;
  size_t codes, xc, parts, tlogit, resid, frag, dwfrag, nll, rows, compact, count, inverse, total;
};

Layout head_layout(const mmuon_ce_args& x, bool train) {
  Layout l{};
  const int64_t T = std::max<int64_t>(x.tokens, 1);
  l.piece = std::min(T, std::max<int64_t>(1, x.piece_tokens));
  l.ldc = int64_t(cdiv(x.vocab, 256)) * 256;
  static_cast<HeadPlans&>(l) = head_plans(l.piece, x.width, x.vocab, train);
  l.nparts = cdiv(x.vocab, 1 << l.logits.part_shift());
  size_t at = 0;
  const auto take = [&at](size_t n) {
    const size_t here = at;
    at += up256(n);
    return here;
  };
  const size_t P = size_t(l.piece);
  l.codes = take(train ? P * l.ldc * 2 : 0);
  l.xc = take(P * x.width * 2);
  l.parts = take(P * l.nparts * 8);
  l.tlogit = take(P * 4);
  l.resid = take(train ? P * 4 : 0);
  l.frag = take(std::max(l.logits.frag(x.vocab, l.piece, false),
                         train && x.dx != nullptr ? l.dx.frag(x.width, l.piece, false) : 0));
  l.dwfrag = take(train && x.dw != nullptr ? l.dw.frag(x.width, x.vocab, T > l.piece) : 0);
  l.nll = take(x.nll == nullptr ? size_t(T) * 4 : 0);
  l.rows = take(size_t(T) * 4);
  l.compact = take(size_t(T) * 8);
  l.count = take(4);
  l.inverse = take(4);
  l.total = at;
  return l;
}

}  // namespace

size_t ce_workspace(const mmuon_ce_args& x, bool train) { return head_layout(x, train).total; }

int launch_ce(const mmuon_ce_args& x, bool train, hipStream_t st) {
  const Layout l = head_layout(x, train);
  char* ws = static_cast<char*>(x.workspace);
  float* nll = x.nll != nullptr ? x.nll : reinterpret_cast<float*>(ws + l.nll);
  int* rows = reinterpret_cast<int*>(ws + l.rows);
  int64_t* target = reinterpret_cast<int64_t*>(ws + l.compact);
  int* count = reinterpret_cast<int*>(ws + l.count);
  float* inverse = reinterpret_cast<float*>(ws + l.inverse);
  const bool mean = x.reduction == MMUON_CE_MEAN, reduced = x.reduction != MMUON_CE_NONE;
  const int T = int(x.tokens), V = int(x.vocab), P = int(l.piece);
  if (train && x.dw != nullptr && T == 0)
    hipLaunchKernelGGL(head_zero, dim3(1024), dim3(256), 0, st, static_cast<uint4*>(x.dw), x.vocab * x.width / 8);
  // the loss of one column of tiles: leaving tokens out would not make it less
  const bool list = train || T > 256 || T > P;
  const bool one = T <= LIST_TOKENS && T <= P;  // head_list
  if (list && !one)
    hipLaunchKernelGGL(head_compact, dim3(1), dim3(1024), 0, st, x.target, T, x.ignore_index, rows, target, count,
                       inverse);
  for (int t0 = 0; t0 < T; t0 += P) {
    const int n = std::min(P, T - t0);
    GatherArgs ga{};
    ga.x = static_cast<const uint16_t*>(x.x);
    ga.xstride = x.x_stride;
    ga.xc = reinterpret_cast<uint16_t*>(ws + l.xc);
    ga.width = x.width;
    ga.tokens = T;
    ga.t0 = t0;
    ga.piece = n;
    ga.rows = rows;
    ga.count = count;
    ga.target = x.target;
    ga.ignore = x.ignore_index;
    ga.dx = train ? static_cast<uint16_t*>(x.dx) : nullptr;
    ga.nll = nll;
    ga.list_rows = rows;
    ga.list_target = target;
    ga.list_count = count;
    ga.list_inverse = inverse;
    if (list && one) hipLaunchKernelGGL(head_list, dim3(T), dim3(128), 0, st, ga);
    else if (list) hipLaunchKernelGGL(head_gather, dim3(t0 == 0 ? T : n), dim3(128), 0, st, ga);

    HeadGemm f{};  // logits (vocabulary x tokens) = w . x^T
    f.a = make_op(x.w, 0, x.w_stride * 2, 2, V);
    f.b = make_op(ga.xc, 0, int64_t(x.width) * 2, 2, n);
    f.count = list ? count : nullptr;
    f.t0 = t0;
    f.piece = n;
    f.tokens = T;
    f.x = static_cast<const char*>(x.x) + int64_t(t0) * x.x_stride * 2;
    f.xstride = x.x_stride * 2;
    f.vocab = V;
    f.codes = reinterpret_cast<uint16_t*>(ws + l.codes);
    f.ldc = l.ldc;
    f.parts = reinterpret_cast<float2*>(ws + l.parts);
    f.nparts = l.nparts;
    f.target = list ? target + t0 : x.target;
    f.tlogit = reinterpret_cast<float*>(ws + l.tlogit);
    set_tiles(f, V, n, x.width, l.logits);
    f.frag = reinterpret_cast<float*>(ws + l.frag);
    f.frag_first = std::min(f.full, f.tiles_m * f.tiles_n);
    // Codes of twice the Infinity Cache go past it, out and back (6000 tokens of 50304 x 1024 with
    // gradients 2012 -> 1943 us, 8192 2606 -> 2572; 2000, a cache of them, 698 -> 711)
    const bool past = int64_t(n) * l.ldc * 2 > (int64_t(512) << 20);
    if (train && past) launch_logits<EP_CODES_PAST>(f, l.logits, st);
    else if (train) launch_logits<EP_CODES>(f, l.logits, st);
    else launch_logits<EP_STATS>(f, l.logits, st);

    RowArgs r{};
    r.codes = f.codes;
    r.ldc = l.ldc;
    r.parts = f.parts;
    r.nparts = l.nparts;
    r.part_shift = l.logits.part_shift();
    r.tlogit = f.tlogit;
    r.target = f.target;
    r.rows = list ? rows + t0 : nullptr;
    r.count = count;
    r.t0 = t0;
    r.piece = n;
    r.vocab = V;
    r.ignore = x.ignore_index;
    r.grad = x.grad;
    r.nll = nll;
    r.resid = reinterpret_cast<float*>(ws + l.resid);
    if (!train) {
      if (n <= 2048) hipLaunchKernelGGL(head_nll<256>, dim3(n), dim3(256), 0, st, r);
      else hipLaunchKernelGGL(head_nll<64>, dim3(cdiv(n, 4)), dim3(256), 0, st, r);
      continue;
    }
    if (past) hipLaunchKernelGGL(head_rows<true>, dim3(n), dim3(256), 0, st, r);
    else hipLaunchKernelGGL(head_rows<false>, dim3(n), dim3(256), 0, st, r);
    const float* factor = mean && x.grad == nullptr ? inverse : nullptr;
    if (x.dx != nullptr) {
      HeadGemm d = f;  // dx^T (width x tokens) = w^T dl^T
      d.a = make_op(x.w, 0, 2, x.w_stride * 2, x.width);
      d.b = make_op(f.codes, 0, l.ldc * 2, 2, n);
      d.out = static_cast<char*>(x.dx);
      d.ostride = int64_t(x.width) * 2;
      d.rows = r.rows;
      d.factor = factor;
      d.resid = r.resid;
      d.w = static_cast<const uint16_t*>(x.w);
      d.wstride = x.w_stride;
      d.frag = reinterpret_cast<float*>(ws + l.frag);
      set_tiles(d, x.width, n, V, l.dx);
      d.frag_first = std::min(d.full, d.tiles_m * d.tiles_n);
      launch_head<true, false, EP_ROWS, X_IS_NONE>(d, l.dx, st);
      launch_join<X_IS_NONE>(d, l.dx, st);
    }
    if (x.dw != nullptr) {
      HeadGemm d = f;  // dw^T (width x vocabulary) = x^T dl
      d.a = make_op(ga.xc, 0, 2, int64_t(x.width) * 2, x.width);
      d.b = make_op(f.codes, 0, 2, l.ldc * 2, V);
      d.out = static_cast<char*>(x.dw);
      d.ostride = int64_t(x.width) * 2;
      d.factor = factor;
      d.frag = reinterpret_cast<float*>(ws + l.dwfrag);
      // Few tokens: dw is bound by its writes, and one that fills the Infinity Cache leaves past it
      // (128 tokens of 50304 x 4096 155 -> 115 us, x 2048 87 -> 55, x 1024 35 -> 38; 800 of x 4096
      // with the other products 1035 -> 1044).
      const bool dwpast = n <= 512 && x.vocab * x.width * 2 > (int64_t(160) << 20);
      d.start = t0 > 0;
      d.keep = t0 + n < T;
      set_tiles(d, x.width, V, n, l.dw);
      d.frag_first = T > P ? 0 : std::min(d.full, d.tiles_m * d.tiles_n);
      if (!d.keep) {
        d.nll = reduced ? nll : nullptr;
        d.loss = x.loss;
        d.mean = mean ? 1 : 0;
      }
      if (dwpast) launch_head<true, true, EP_PAST, X_IS_A>(d, l.dw, st);
      else launch_head<true, true, EP_ROWS, X_IS_A>(d, l.dw, st);
      if (!d.keep) launch_join<X_IS_A>(d, l.dw, st);
    }
  }
  if (reduced && !(train && x.dw != nullptr && T > 0))
    hipLaunchKernelGGL(head_loss, dim3(1), dim3(1024), 0, st, nll, T, list && T > 0 ? count : nullptr, x.target,
                       x.ignore_index, mean ? 1 : 0, x.loss);
  return 0;
}

int launch_ce_scale(void* x, int64_t nx, void* y, int64_t ny, const float* c, hipStream_t st) {
  const int64_t chunks = (nx + ny) / 8;
  if (chunks > 0)
    hipLaunchKernelGGL(head_scale, dim3(unsigned(std::min<int64_t>((chunks + 255) / 256, 2048))), dim3(256), 0, st,
                       static_cast<uint16_t*>(x), nx / 8, static_cast<uint16_t*>(y), ny / 8, c);
  return 0;
}

}  // namespace mmuon
