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
// gives p with a relative error of 3.4e-4 at most, however small p is (2e-3 is bf16's own
// rounding of dl; bf16 exponentials would round twice); what lies 64 binades below its
// part's maximum (p < 6e-20) counts as zero.  The target's logit is kept in fp32: the loss
// and p_y - 1 do not go through a code.  One factor 1 / valid tokens is applied to the
// fp32 sums of dx and dw and not to dl, and dx adds what bf16 took from its largest term,
// p_y - 1: with them in dl, its rounding was one for all tokens, up to 2^-8.
#include <algorithm>

#include "common.hpp"
#include "gemm_pipe.hpp"
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
  EP_ROWS = 2,   // bf16 result, rows = columns of the tile
  EP_FRAG = 3    // fp32 accumulators in fragment order (a split of K, or a piece of the tokens)
};

// D (M x N) = A (M x K) B^T (N x K), where N (logits, dx) or K (dw) are the piece's tokens:
// compact tokens t0 .. of *count, at most `piece`.
struct HeadGemm {
  GOp a, b;
  int M, N, K, S, kchunk;
  int tiles_m, tiles_n;
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
  float* frag;                   // EP_FRAG: BM x BN floats per virtual tile
  const float* start;            // accumulators to start from, same order; or null
  uint16_t* codes;               // EP_CODES: [token][ldc]
  int64_t ldc;
  float2* parts;                 // [token][nparts]: maximum (base 2), sum of 2^(l - maximum)
  int nparts;
  const int64_t* target;         // of the compact tokens of the piece
  float* tlogit;                 // [token]
  __device__ __forceinline__ int live() const { return min(max(*count - t0, 0), piece); }
  __device__ __forceinline__ int total() const { return tiles_m * tiles_n * S; }
};

// Virtual tile -> (split, tile row, tile column).  Each XCD (v % 8) takes a contiguous run
// of tiles; the tiles of a run are numbered in patches PATCH tile columns wide, so the 32
// tiles that an XCD's CUs hold at a time share 4 column and 8 row operand bands.
constexpr int PATCH = 4;
__device__ __forceinline__ bool head_tile(const HeadGemm& a, int v, int& sp, int& tm, int& tn, int& idx) {
  const int total = a.total(), per = (total + 7) >> 3, local = v >> 3;
  idx = (v & 7) * per + local;
  if (local >= per || idx >= total) return false;
  const int plane = a.tiles_m * a.tiles_n;
  sp = idx / plane;
  const int t = idx - sp * plane, g = t / (a.tiles_m * PATCH), r = t - g * a.tiles_m * PATCH;
  const int width = min(PATCH, a.tiles_n - g * PATCH);
  tm = r / width;
  tn = g * PATCH + r - tm * width;
  return true;
}

// Statistics and codes of a tile of logits: rows m0.. are vocabulary, columns n0.. tokens.
template <class GE, bool CODES>
__device__ __forceinline__ void loss_epilogue(const HeadGemm& a, char* lds, int m0, int n0,
                                              f32x16 (&acc)[GE::WI][GE::WJ]) {
  const int tid = fresh_tid();
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / GE::GN, wn = wave % GE::GN;
  constexpr int PW = 32 * GE::WI;               // vocabulary of a part
  const int v0 = m0 + wm * PW, left = a.M - v0;  // rows from `left` on do not exist
  const int half = lane >> 5;
  if constexpr (CODES) barrier();  // every wave is done with the ring
#pragma unroll
  for (int j = 0; j < GE::WJ; ++j) {
    const int row = (wn * GE::WJ + j) * 32 + (lane & 31), tok = n0 + row;
    const bool live = tok < a.N;
    const int64_t y = live ? a.target[tok] : -1;
    const int64_t rel = y - v0;
    const bool hit = rel >= 0 && rel < PW && rel < left && ((int(rel) >> 2) & 1) == half;
    if (__any(hit)) {
      const int at = (int(rel) >> 5) * 16 + ((int(rel) >> 3) & 3) * 4 + (int(rel) & 3);
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < GE::WI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) l = at == i * 16 + r ? acc[i][j][r] : l;
      if (hit) a.tlogit[tok] = l;
    }
    if (left < PW) {
#pragma unroll
      for (int i = 0; i < GE::WI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (i * 32 + (r >> 2) * 8 + half * 4 + (r & 3) >= left) acc[i][j][r] = -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < GE::WI; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[i][j][r]);
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const float m2 = m == -INFINITY ? 0.f : m * LOG2E;  // a part that is all -inf: sum 0
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < GE::WI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[e] = __builtin_fmaf(acc[i][j][4 * q + e], LOG2E, -m2);
          s += __builtin_amdgcn_exp2f(d[e]);
        }
        if constexpr (CODES) {
          constexpr float K = -1.f / CODE_RANGE;
          const uint32_t lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(d[0] * K, d[1] * K));
          const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(d[2] * K, d[3] * K));
          const int col = (wm * GE::WI + i) * 32 + q * 8 + half * 4;
          *reinterpret_cast<uint2*>(lds + GE::tile_at(row, col)) = make_uint2(lo, hi);
        }
      }
    s += __shfl_xor(s, 32, 64);
    if (live && half == 0 && left > 0) a.parts[int64_t(tok) * a.nparts + v0 / PW] = make_float2(m2, s);
  }
}

// Staged tile -> rows of 16-B chunks: fn(row, first column, chunk)
template <class GE, class Fn>
__device__ __forceinline__ void staged_rows(const char* stage, Fn&& fn) {
  constexpr int CPR = GE::BM / 8;
  const int tid = fresh_tid();
#pragma unroll 4
  for (int it = 0; it < GE::BN * CPR / GE::NTH; ++it) {
    const int idx = tid + it * GE::NTH, row = idx / CPR, col = idx % CPR * 8;
    fn(row, col, *reinterpret_cast<const uint4*>(stage + GE::tile_at(row, col)));
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

template <class GE, bool AT, bool BT, int EP>
__device__ __forceinline__ void head_work(const HeadGemm& a, char* lds, int v) {
  int sp, tm, tn, idx;
  if (!head_tile(a, v, sp, tm, tn, idx)) return;
  const int m0 = tm * GE::BM, n0 = tn * GE::BN;
  GPipe<GE, AT, BT> p;
  p.lane = threadIdx.x & 63;
  p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  p.wm = p.wave / GE::GN;
  p.wn = p.wave % GE::GN;
  const int kbeg = sp * a.kchunk, kend = min(a.K, kbeg + a.kchunk);
  p.ak.start(a.a, a.a.base + mn_off(a.a, m0), kbeg);
  p.bk.start(a.b, a.b.base + mn_off(a.b, n0), kbeg);
  p.nxt = 0;
  p.KT = (kend - kbeg + BK - 1) / BK;
  const int rem = kend - kbeg - (p.KT - 1) * BK;  // K of the last slice
#pragma unroll
  for (int q = 0; q < GE::DMA; ++q) {
    const bool row = q < GE::RL;
    const int u = row ? GE::RL * p.wave + q : GE::CL * p.wave + q - GE::RL;
    p.loff[q] = row ? lane_offset<AT>(a.a, m0, u, p.lane) : lane_offset<BT>(a.b, n0, u, p.lane);
    const int kd = (row ? AT : BT) ? 16 * (u & 1) + (p.lane >> 2) : 8 * ((p.lane & 3) ^ ((p.lane >> 4) & 3));
    p.tail[q] = kd >= rem ? OOB : 0;
  }
  p.lds = lds;
  p.lds0 = lds_addr(lds);
#pragma unroll
  for (int kk = 0; kk < BK / 16; ++kk) p.kfrag[kk] = kmajor_frag_base(kk, p.lane);
  p.tfrag_r = rowmajor_frag_base(p.wm * GE::WI, p.lane);
  p.tfrag_c = rowmajor_frag_base(p.wn * GE::WJ, p.lane);
  f32x16 acc[GE::WI][GE::WJ];
  if (p.KT > 0) {
    p.run(acc);
  } else {  // an empty piece
#pragma unroll
    for (int i = 0; i < GE::WI; ++i)
#pragma unroll
      for (int j = 0; j < GE::WJ; ++j) acc[i][j] = f32x16{};
  }

  // fragment order: float4 q of MFMA tile (i, j) of a wave at 64 lanes x 16 B
  const int64_t f0 = ((int64_t(idx) * GE::NW + p.wave) * (GE::WI * GE::WJ * 16) * 64 + p.lane * 4);
  if (a.start != nullptr) {
#pragma unroll
    for (int i = 0; i < GE::WI; ++i)
#pragma unroll
      for (int j = 0; j < GE::WJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 t = *reinterpret_cast<const float4*>(a.start + f0 + ((i * GE::WJ + j) * 4 + q) * 256);
          acc[i][j][4 * q] += t.x;
          acc[i][j][4 * q + 1] += t.y;
          acc[i][j][4 * q + 2] += t.z;
          acc[i][j][4 * q + 3] += t.w;
        }
  }
  if constexpr (EP == EP_FRAG) {
#pragma unroll
    for (int i = 0; i < GE::WI; ++i)
#pragma unroll
      for (int j = 0; j < GE::WJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(a.frag + f0 + ((i * GE::WJ + j) * 4 + q) * 256) =
              make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
  } else if constexpr (EP == EP_ROWS) {
    const float factor = a.factor != nullptr ? *a.factor : 1.f;
#pragma unroll
    for (int i = 0; i < GE::WI; ++i)
#pragma unroll
      for (int j = 0; j < GE::WJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          if (a.resid != nullptr) {
            const int n = n0 + (p.wn * GE::WJ + j) * 32 + (p.lane & 31);
            const int m = m0 + (p.wm * GE::WI + i) * 32 + q * 8 + (p.lane >> 5) * 4;
            if (n < a.N && m < a.M) add_resid(a, n, m, v);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = v[e] * factor;
        }
    barrier();  // every wave is done with the ring
    stage_acc<GE>(lds, acc);
    barrier_after_lds_writes();
    staged_rows<GE>(lds, [&](int r, int c, const uint4& u) {
      if (n0 + r >= a.N || m0 + c >= a.M) return;
      const int row = a.rows != nullptr ? a.rows[n0 + r] : n0 + r;
      *reinterpret_cast<uint4*>(a.out + int64_t(row) * a.ostride + int64_t(m0 + c) * 2) = u;
    });
  } else {
    loss_epilogue<GE, EP == EP_CODES>(a, lds, m0, n0, acc);
    if constexpr (EP == EP_CODES) {
      barrier_after_lds_writes();
      staged_rows<GE>(lds, [&](int r, int c, const uint4& u) {
        if (n0 + r < a.N) *reinterpret_cast<uint4*>(a.codes + int64_t(n0 + r) * a.ldc + m0 + c) = u;
      });
    }
  }
}

// The sizes that the number of compact tokens decides
enum { X_IS_A = 0, X_IS_B = 1, X_IS_NONE = 2 };  // which operand x is: of dw, of the logits, of dx
template <class GE, int X>
__device__ __forceinline__ void settle(HeadGemm& a) {
  const int n = a.live();
  if constexpr (X == X_IS_A) {
    a.K = n;
    a.kchunk = max(n, 1);
  } else {
    a.N = n;
    a.b.extent = n;
    a.tiles_n = (n + GE::BN - 1) / GE::BN;
  }
  if (X == X_IS_A && *a.count == a.tokens) {
    a.a.base = a.x;
    a.a.kstride = a.xstride;
  }
  if (X == X_IS_B && *a.count == a.tokens) {
    a.b.base = a.x;
    a.b.mstride = a.xstride;
  }
}

template <class GE, bool AT, bool BT, int EP, int X>
__global__ __launch_bounds__(GE::NTH, GE::PER_CU * GE::NW / 4) void head_gemm(HeadGemm a) {
  __shared__ __attribute__((aligned(1024))) char lds[GE::LDS];
  settle<GE, X>(a);
  const int vtiles = (a.total() + 7) / 8 * 8;
  for (int v = blockIdx.x; v < vtiles; v += gridDim.x) {
    head_work<GE, AT, BT, EP>(a, lds, v);
    barrier();  // the staging area is read before the next tile's loads refill the ring
  }
}

// Sum over the splits of K, in split order, of one 32 x 32 MFMA tile per workgroup: the
// fp32 partials in fragment order -> bf16 rows of dx.
template <class GE>
__global__ __launch_bounds__(256) void head_join(HeadGemm a) {
  constexpr int PER = GE::NW * GE::WI * GE::WJ;  // MFMA tiles of a tile
  settle<GE, X_IS_NONE>(a);
  const int plane = a.tiles_m * a.tiles_n, t = blockIdx.x / PER, in = blockIdx.x % PER;
  if (t >= plane) return;
  const int g = t / (a.tiles_m * PATCH), r = t - g * a.tiles_m * PATCH, width = min(PATCH, a.tiles_n - g * PATCH);
  const int tm = r / width, tn = g * PATCH + r - tm * width;
  const int wave = in / (GE::WI * GE::WJ), ij = in % (GE::WI * GE::WJ);
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int m = tm * GE::BM + (wave / GE::GN * GE::WI + ij / GE::WJ) * 32 + q * 8 + (lane >> 5) * 4;
  const int n = tn * GE::BN + (wave % GE::GN * GE::WJ + ij % GE::WJ) * 32 + (lane & 31);
  if (m >= a.M || n >= a.N) return;
  const float* f = a.frag + (int64_t(t) * PER + in) * 1024 + threadIdx.x * 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < a.S; ++k) {
    const float4 u = *reinterpret_cast<const float4*>(f + int64_t(k) * plane * PER * 1024);
    v[0] += u.x;
    v[1] += u.y;
    v[2] += u.z;
    v[3] += u.w;
  }
  add_resid(a, n, m, v);
  const float c = a.factor != nullptr ? *a.factor : 1.f;
  *reinterpret_cast<uint2*>(a.out + int64_t(a.rows[n]) * a.ostride + int64_t(m) * 2) =
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
  int64_t vocab;
  const float* grad;       // per token, or null: 1
  float* nll;              // per token
  float* resid;            // per compact token
  __device__ __forceinline__ int live() const { return min(max(*count - t0, 0), piece); }
};

// log2 of a token's sum of exponentials, joined from its parts by NTHR threads
// (one wave where NTHR == 64); valid in every thread.
template <int NTHR>
__device__ __forceinline__ float join_parts(const float2* p, int n, float* scratch) {
  float m = -INFINITY, s = 0.f;
  for (int i = threadIdx.x % NTHR; i < n; i += NTHR) {
    const float2 t = p[i];
    // a part that is empty or all -inf has sum 0 and no maximum
    const float top = t.y == 0.f ? m : fmaxf(m, t.x);
    if (top != -INFINITY) s = s * __builtin_amdgcn_exp2f(m - top) + t.y * __builtin_amdgcn_exp2f(t.x - top);
    else s += t.y;
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

// The loss alone: one wave per token.
__global__ __launch_bounds__(256) void head_nll(RowArgs a) {
  const int tok = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tok >= a.live()) return;
  const float lse2 = join_parts<64>(a.parts + int64_t(tok) * a.nparts, a.nparts, nullptr);
  if ((threadIdx.x & 63) == 0) a.nll[a.rows[tok]] = token_nll(lse2, a.tlogit[tok], a.target[tok], a.vocab);
}

// One workgroup per token: lse, nll, and the row's codes -> dl.
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
  for (int64_t c = threadIdx.x * 8; c < a.ldc; c += 256 * 8) {
    const uint4 in = *reinterpret_cast<const uint4*>(row + c);
    const uint32_t w[4] = {in.x, in.y, in.z, in.w};
    const int part = int(c >> a.part_shift);
    const float top = part < a.nparts ? parts[part].x - lse2 : 0.f;  // beyond: codes of zero
    uint32_t r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = w[k] & 0xffff, hi = w[k] >> 16;
      const float p0 = lo == CODE_ZERO ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(float(lo), -CODE_STEP, top));
      const float p1 = hi == CODE_ZERO ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(float(hi), -CODE_STEP, top));
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
// and, with the first piece, the zeros of ignored tokens in dx and nll.
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
};
__global__ __launch_bounds__(128) void head_gather(GatherArgs a) {
  const int n = *a.count, j = blockIdx.x;
  if (n == a.tokens) return;
  if (j < a.piece && a.t0 + j < n) {
    const uint16_t* src = a.x + int64_t(a.rows[a.t0 + j]) * a.xstride;
    for (int c = threadIdx.x * 8; c < a.width; c += 128 * 8)
      *reinterpret_cast<uint4*>(a.xc + int64_t(j) * a.width + c) = *reinterpret_cast<const uint4*>(src + c);
  }
  if (a.t0 == 0 && j < a.tokens && a.target[j] == a.ignore) {
    if (threadIdx.x == 0) a.nll[j] = 0.f;
    if (a.dx != nullptr)
      for (int c = threadIdx.x * 8; c < a.width; c += 128 * 8)
        *reinterpret_cast<uint4*>(a.dx + int64_t(j) * a.width + c) = make_uint4(0, 0, 0, 0);
  }
}

// sum of nll, divided by the number of targets that are not ignored where mean (NaN if there
// is none): each thread's share in order, then a tree (the same order every time)
__global__ __launch_bounds__(1024) void head_loss(const float* nll, int tokens, const int* count, int mean,
                                                  float* loss) {
  __shared__ float scratch[16];
  float s = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < tokens; i += 1024) s += nll[i];
  s = block_sum<1024>(s, scratch);
  if (threadIdx.x == 0) *loss = mean ? s / float(*count) : s;
}

__global__ __launch_bounds__(256) void head_zero(uint4* x, int64_t chunks) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < chunks; i += int64_t(gridDim.x) * 256)
    x[i] = make_uint4(0, 0, 0, 0);
}

// x *= *c, in 16-B chunks; nothing is touched where *c == 1
__global__ __launch_bounds__(256) void head_scale(uint16_t* x, int64_t chunks, const float* c) {
  const float f = *c;
  if (f == 1.f) return;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < chunks; i += int64_t(gridDim.x) * 256) {
    float v[8];
    Vec8<BF16T>::load(x + i * 8, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= f;
    Vec8<BF16T>::store(x + i * 8, v);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
typedef Geo<2, 4, 4, 2, 4> H256;  // 256 x 256 tiles, one workgroup per CU

// M, N, K with all of the piece's tokens valid (settle: the real ones)
template <class GE>
void set_tiles(HeadGemm& a, int M, int N, int K, int S) {
  a.M = M;
  a.N = N;
  a.K = K;
  a.kchunk = cdiv(cdiv(K, S), BK) * BK;
  a.S = cdiv(K, a.kchunk);
  a.tiles_m = cdiv(M, GE::BM);
  a.tiles_n = cdiv(N, GE::BN);
}

template <class GE, bool AT, bool BT, int EP, int X>
void launch_head(const HeadGemm& a, hipStream_t s) {
  const int grid = std::min(cdiv(int64_t(a.tiles_m) * a.tiles_n * a.S, 8) * 8, resident_grid(1 << 30) * GE::PER_CU);
  hipLaunchKernelGGL((head_gemm<GE, AT, BT, EP, X>), dim3(grid), dim3(GE::NTH), 0, s, a);
}

// Splits of K = V of the dx product: its tiles (tokens x width) may not fill the chip.
// At least 2048 of K per split.
int dx_splits(int64_t tokens, int64_t width, int64_t vocab) {
  const int64_t tiles = cdiv(tokens, 256) * int64_t(cdiv(width, 256));
  return int(std::max<int64_t>(1, std::min<int64_t>(256 / tiles, vocab / 2048)));
}

constexpr int PART_SHIFT = 7;  // a wave of the 256-wide tile holds 128 of the vocabulary

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct Layout {
  int64_t piece, ldc;
  int nparts, splits;
  size_t codes, xc, parts, tlogit, resid, dxfrag, dwfrag, nll, rows, compact, count, inverse, total;
};

Layout head_layout(const mmuon_ce_args& x, bool train) {
  Layout l{};
  const int64_t T = std::max<int64_t>(x.tokens, 1);
  l.piece = std::min(T, std::max<int64_t>(1, x.piece_tokens));
  l.ldc = int64_t(cdiv(x.vocab, 256)) * 256;
  l.nparts = cdiv(x.vocab, 1 << PART_SHIFT);
  l.splits = dx_splits(l.piece, x.width, x.vocab);
  size_t at = 0;
  const auto take = [&at](size_t n) {
    const size_t here = at;
    at += up256(n);
    return here;
  };
  const size_t P = size_t(l.piece), tile = 256 * 256 * 4;
  l.codes = take(train ? P * l.ldc * 2 : 0);
  l.xc = take(P * x.width * 2);
  l.parts = take(P * l.nparts * 8);
  l.tlogit = take(P * 4);
  l.resid = take(train ? P * 4 : 0);
  l.dxfrag = take(train && l.splits > 1 ? tile * l.splits * cdiv(l.piece, 256) * cdiv(x.width, 256) : 0);
  l.dwfrag = take(train && T > l.piece ? tile * cdiv(x.width, 256) * cdiv(x.vocab, 256) : 0);
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
  const bool mean = x.reduction == MMUON_CE_MEAN;
  const int T = int(x.tokens), V = int(x.vocab), P = int(l.piece);
  if (train && x.dw != nullptr && T == 0)
    hipLaunchKernelGGL(head_zero, dim3(1024), dim3(256), 0, st, static_cast<uint4*>(x.dw), x.vocab * x.width / 8);
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
    hipLaunchKernelGGL(head_gather, dim3(t0 == 0 ? T : n), dim3(128), 0, st, ga);

    HeadGemm f{};  // logits (vocabulary x tokens) = w . x^T
    f.a = make_op(x.w, 0, x.w_stride * 2, 2, V);
    f.b = make_op(ga.xc, 0, int64_t(x.width) * 2, 2, n);
    f.count = count;
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
    f.target = target + t0;
    f.tlogit = reinterpret_cast<float*>(ws + l.tlogit);
    set_tiles<H256>(f, V, n, x.width, 1);
    if (train) launch_head<H256, false, false, EP_CODES, X_IS_B>(f, st);
    else launch_head<H256, false, false, EP_STATS, X_IS_B>(f, st);

    RowArgs r{};
    r.codes = f.codes;
    r.ldc = l.ldc;
    r.parts = f.parts;
    r.nparts = l.nparts;
    r.part_shift = PART_SHIFT;
    r.tlogit = f.tlogit;
    r.target = f.target;
    r.rows = rows + t0;
    r.count = count;
    r.t0 = t0;
    r.piece = n;
    r.vocab = V;
    r.grad = x.grad;
    r.nll = nll;
    r.resid = reinterpret_cast<float*>(ws + l.resid);
    if (!train) {
      hipLaunchKernelGGL(head_nll, dim3(cdiv(n, 4)), dim3(256), 0, st, r);
      continue;
    }
    hipLaunchKernelGGL(head_rows, dim3(n), dim3(256), 0, st, r);
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
      d.frag = reinterpret_cast<float*>(ws + l.dxfrag);
      set_tiles<H256>(d, x.width, n, V, l.splits);
      if (d.S > 1) {
        launch_head<H256, true, false, EP_FRAG, X_IS_NONE>(d, st);
        hipLaunchKernelGGL(head_join<H256>, dim3(d.tiles_m * d.tiles_n * H256::NW * H256::WI * H256::WJ), dim3(256), 0,
                           st, d);
      } else {
        launch_head<H256, true, false, EP_ROWS, X_IS_NONE>(d, st);
      }
    }
    if (x.dw != nullptr) {
      HeadGemm d = f;  // dw^T (width x vocabulary) = x^T dl
      d.a = make_op(ga.xc, 0, 2, int64_t(x.width) * 2, x.width);
      d.b = make_op(f.codes, 0, 2, l.ldc * 2, V);
      d.out = static_cast<char*>(x.dw);
      d.ostride = int64_t(x.width) * 2;
      d.factor = factor;
      d.frag = reinterpret_cast<float*>(ws + l.dwfrag);
      d.start = t0 > 0 ? d.frag : nullptr;
      set_tiles<H256>(d, x.width, V, n, 1);
      if (t0 + n < T) launch_head<H256, true, true, EP_FRAG, X_IS_A>(d, st);
      else launch_head<H256, true, true, EP_ROWS, X_IS_A>(d, st);
    }
  }
  if (x.loss != nullptr && x.reduction != MMUON_CE_NONE)
    hipLaunchKernelGGL(head_loss, dim3(1), dim3(1024), 0, st, nll, T, count, mean ? 1 : 0, x.loss);
  return 0;
}

int launch_ce_scale(void* x, int64_t numel, const float* c, hipStream_t st) {
  const int64_t chunks = numel / 8;
  if (chunks > 0)
    hipLaunchKernelGGL(head_scale, dim3(unsigned(std::min<int64_t>((chunks + 255) / 256, 4096))), dim3(256), 0, st,
                       static_cast<uint16_t*>(x), chunks, c);
  return 0;
}

}  // namespace mmuon
