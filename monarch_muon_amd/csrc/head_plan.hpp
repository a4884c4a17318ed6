// Which tiles the products of the head's loss take, and which of them are split over K (host
// code only; a function of the sizes alone).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace mmuon {
namespace {

enum { T256 = 0, T128 = 1, T64 = 2 };  // 256 x 256, 256 x 128, 128 x 64

inline int parts_of(int64_t n, int64_t each) { return int((n + each - 1) / each); }

// A product's tile, and the parts of K (S) of the tiles from `full` on.
struct HeadPlan {
  int tile;
  int full, S;
  int rows() const { return tile == T64 ? 128 : 256; }
  int cols() const { return 256 >> tile; }
  int part_shift() const { return 7 - tile; }  // vocabulary of a wave of the logits
  int tiles(int64_t m, int64_t n) const { return parts_of(m, rows()) * parts_of(n, cols()); }
  int virtual_tiles(int64_t m, int64_t n) const {
    const int t = tiles(m, n), f = std::min(full, t);
    return f + (t - f) * S;
  }
  // fp32 accumulators: of the split tiles, or of all
  size_t frag(int64_t m, int64_t n, bool all) const {
    return size_t(virtual_tiles(m, n) - (all ? 0 : std::min(full, tiles(m, n)))) * rows() * cols() * 4;
  }
};

// Time in ns of a product M x N x K on a 256-CU part (a function of the sizes only, so the order
// of the sums does not depend on the device): rounds of 256 tiles, each its slices of K at the
// rate of full rounds and what its start and end cost.  Logits with codes for the gradients end
// later than that (1000 x 512 90 us, 61 by this): what that costs is not in here.  Measured
// at V = 50304, the loss alone: 4096 x 4096 1.40 ms in 256-wide tiles, 1.83 in 128-wide; 1000 x
// 1024 123 / 145 us, 300 x 4096 196 / 213, 600 x 512 59.5 / 60.6, 128 x 2048 50 / 49, 33 x 2048
// 47 / 41.
inline int64_t round_time(bool narrow, int64_t K) { return narrow ? 1500 + 18 * K : 2500 + 25 * K; }
inline int64_t plan_time(const HeadPlan& p, int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = p.tiles(M, N), full = std::min<int64_t>(p.full, tiles), parts = (tiles - full) * p.S;
  const bool narrow = p.tile == T128;
  int64_t t = parts_of(full, 256) * round_time(narrow, K) + parts_of(parts, 256) * round_time(narrow, parts_of(K, p.S));
  // the partials' write and read, the join's launch
  if (parts > 0) t += 5000 + parts * 256 * p.cols() * 8 / 4500;
  return t;
}
constexpr int WHOLE = 1 << 30;  // no tile is split

// All tiles split (few tokens or a narrow model: dx has few tiles), or those of the last round,
// that would leave most CUs idle.  At least 256 of K in a part; partials of at most 256 MiB.
// The logits split where that should take 8% off at least (600 tokens of 50304 x 4096 312 ->
// 273 us, 1000 430 -> 392, x 1024 121 -> 124).
inline HeadPlan head_plan(int64_t M, int64_t N, int64_t K, bool narrow_too, bool logits) {
  HeadPlan best{T256, WHOLE, 1};
  int64_t best_time = plan_time(best, M, N, K);
  for (int tile = T256; tile <= (narrow_too ? T128 : T256); ++tile) {
    const int tiles = HeadPlan{tile, WHOLE, 1}.tiles(M, N);
    for (const int full : {WHOLE, 0, tiles / 256 * 256})
      for (int S = full == WHOLE ? 1 : 2; S <= (full == WHOLE ? 1 : 256) && (S == 1 || K / S >= 256); ++S) {
        const HeadPlan p{tile, full, S};
        if (p.frag(M, N, false) > (size_t(1) << 28)) break;
        const int64_t t = plan_time(p, M, N, K) * (logits && full != WHOLE ? 109 : 100) / 100;
        if (t < best_time) best = p, best_time = t;
      }
  }
  return best;
}

// The three products of a piece of the tokens
struct HeadPlans {
  HeadPlan logits, dx, dw;
};
inline HeadPlans head_plans(int64_t tokens, int64_t width, int64_t vocab, bool train) {
  HeadPlans p;
  // The loss alone of up to 64 tokens reads the head and little else: small tiles keep every CU
  // at it (256 x 128: 197 tiles of 50304).  1 token x 4096 103.5 -> 96.8 us, x 1024 27.5 -> 25.6,
  // 33 x 2048 41.6 -> 40.8, 64 x 512 21.6 -> 20.5, x 4096 106.5 -> 107.5; with gradients no gain.
  p.logits = !train && tokens <= 64 ? HeadPlan{T64, WHOLE, 1} : head_plan(vocab, tokens, width, true, true);
  p.dx = head_plan(width, tokens, vocab, true, false);
  // (128-wide tiles gained nothing there: 1000 x 512 54 us in 256-wide, 68 in 128-wide)
  p.dw = head_plan(width, vocab, tokens, false, false);
  return p;
}

}  // namespace
}  // namespace mmuon
