// Token embedding and the gradient of its table.
//
//   out[t] = scale w[i_t]            dw[v] = scale sum over t with i_t = v of dout[t]
//
// The gradient is dense and does not depend on timing: rows are dealt to classes (row v to
// class v % C), one workgroup each.  A workgroup reads all ids, places the positions of its
// rows in token order (counts per row and wave, then a stable rank), and writes zeros to the
// rows that no token has.  Common words have neighbouring ids, so the rows of a class are far
// apart.  A second launch sums the positions in fp32, a segment of them to a wave whatever
// rows they are of; a third joins the pieces of rows that lie in several segments, in order.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace mmuon {
namespace {

// N consecutive elements: 16 B, or one where rows are not whole aligned 16-B chunks.  (Two
// 16-B accesses to a lane, 8 floats, leave half of each line to the second: zeros to 50304 x 512
// floats 23 us, 16 B at a time 18.)
template <class T>
constexpr int CHUNK = 16 / int(sizeof(typename T::storage));
template <class T, int N>
__device__ __forceinline__ void load_n(const typename T::storage* p, float (&v)[N]) {
  if constexpr (N == 8) {
    Vec8<T>::load(p, v);
  } else if constexpr (N == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  } else {
    v[0] = T::load(p, 0);
  }
}
template <class T, int N, bool NT = false>
__device__ __forceinline__ void store_n(typename T::storage* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    T::store(p, 0, v[0]);
    return;
  } else {
    uint4 u;
    if constexpr (sizeof(typename T::storage) == 2) u = Vec8<T>::pack(v);
    else u = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    if constexpr (NT) store16_nt(p, u);
    else *reinterpret_cast<uint4*>(p) = u;
  }
}
// fp32 sums of N columns
template <int N>
__device__ __forceinline__ void load_sums(const float* p, float (&v)[N]) {
  if constexpr (N == 8) Vec8<F32T>::load(p, v);
  else load_n<F32T, N>(p, v);
}
template <int N>
__device__ __forceinline__ void store_sums(float* p, const float (&v)[N]) {
  if constexpr (N == 8) Vec8<F32T>::store(p, v);
  else store_n<F32T, N>(p, v);
}

// `lanes` (a power of two) threads per row; NT: past the L2s
template <class T, int N, bool NT>
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
    store_n<T, N, NT>(dst + c, x);
  }
}

constexpr int MAX_SEG = 32;  // positions that one wave sums, at most; 8, 16 or 32 (segment)

// The positions that have a gradient, class after class, row after row, in token order: the
// token and the row of each, at a row's first one how many it has, and how many there are.
struct GradSpace {
  int* token;
  int* row;
  int* count;
  int* all;
  float* sums;  // of the pieces of rows that lie in several segments: two for each segment
};

// WAVES waves, ROWS rows of a class at most, LIST ids of a class that a wave keeps from its scan;
// FIRST: zeros to all rows before, not to the empty ones behind.  Bound by the zeros (16384 bf16
// tokens of 50304 x 4096: 80 us for most of 412 MB), then by reading all ids in each of 256
// workgroups (65536 tokens of 50304 x 1024: 33 us); 1000 tokens of 50304 x 512 floats 19 us.
template <class T, int N, int WAVES, int ROWS, int LIST, bool FIRST>
__global__ __launch_bounds__(64 * WAVES) void embed_rows(mmuon_embedding_args a, int log2c, bool past, GradSpace space) {
  constexpr int NTH = 64 * WAVES;
  static_assert(ROWS % NTH == 0 || NTH % ROWS == 0, "rows are scanned by whole workgroups");
  __shared__ int at[WAVES][ROWS];     // counts, then the next place, of a row's positions in a wave's tokens
  __shared__ int first[ROWS + 1];     // the row's first place
  __shared__ uint32_t kept[WAVES][LIST];  // ids of the class: row << 22 | token of the run
  __shared__ int below[WAVES], wsum[WAVES];
  const int c = blockIdx.x, C = 1 << log2c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = int((a.vocab - c + C - 1) >> log2c);
  const uint64_t before = (uint64_t(1) << lane) - 1;
  const auto zero_rows = [&](auto which) {
    const float zero[N] = {};
    const int chunks = (a.width + 64 * N - 1) / (64 * N);
    for (int task = wave; task < rows * chunks; task += WAVES) {
      const int r = task / chunks, col = (task - r * chunks) * 64 * N + lane * N;
      if (!which(r) || col >= a.width) continue;
      auto* dst = static_cast<typename T::storage*>(a.dw) + (int64_t(r) * C + c) * a.width + col;
      if (past) store_n<T, N, true>(dst, zero);
      else store_n<T, N>(dst, zero);
    }
  };
  // few ids: most rows are empty, and all zeros are on their way while the ids are read
  if constexpr (FIRST) zero_rows([](int) { return true; });
  for (int i = threadIdx.x; i < WAVES * rows; i += NTH) at[i / rows][i % rows] = 0;
  __syncthreads();
  // a wave's tokens: a run of whole 64s
  const int64_t run = (a.tokens + NTH - 1) / NTH * 64, t0 = wave * run, t1 = min(a.tokens, t0 + run);
  int less = 0, found = 0;
  const auto row_of = [&](int64_t v) {  // the id's row of this class, or -1
    if (v < 0 || v >= a.vocab || v == a.padding_idx) return -1;
    less += int(v & (C - 1)) < c;
    return int(v & (C - 1)) == c ? int(v >> log2c) : -1;
  };
  constexpr int U = 8;
  for (int64_t t = t0; t < t1; t += 64 * U) {
    int64_t v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = t + u * 64 + lane < t1 ? a.index[t + u * 64 + lane] : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = row_of(v[u]);
      const uint64_t hit = __ballot(r >= 0);
      if (r >= 0) {
        atomicAdd(&at[wave][r], 1);
        const int j = found + __popcll(hit & before);
        if (j < LIST) kept[wave][j] = uint32_t(r) << 22 | uint32_t(t - t0 + u * 64 + lane);
      }
      found += __popcll(hit);
    }
  }
  less = wave_isum(less);
  if (lane == 0) below[wave] = less;
  __syncthreads();
  // places: class after class, row after row, wave after wave
  int base = 0;
  for (int w = 0; w < WAVES; ++w) base += below[w];
  for (int r0 = 0; r0 < rows; r0 += NTH) {
    const int r = r0 + threadIdx.x;
    int n = 0;
    if (r < rows)
      for (int w = 0; w < WAVES; ++w) n += at[w][r];
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(incl, o, 64);
      if (lane >= o) incl += u;
    }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int place = base + incl - n;
    for (int w = 0; w < WAVES; ++w) {
      place += w < wave ? wsum[w] : 0;
      base += wsum[w];
    }
    if (r < rows) {
      first[r] = place;
      if (n > 0) space.count[place] = n;
      for (int w = 0; w < WAVES; ++w) {
        const int k = at[w][r];
        at[w][r] = place;
        place += k;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    first[rows] = base;
    if (c == int(gridDim.x) - 1) *space.all = base;
  }
  // positions, row by row of 64 tokens, in lane order
  volatile int* next = at[wave];  // one lane's store is another's next load
  const auto put = [&](int r, int64_t t) {
    uint64_t left = __ballot(r >= 0);
    while (left != 0) {
      const int lead = __ffsll(static_cast<unsigned long long>(left)) - 1, row = __shfl(r, lead, 64);
      const uint64_t same = __ballot(r == row);
      const int p = next[row];
      if (r == row) {
        space.token[p + __popcll(same & before)] = int(t);
        space.row[p + __popcll(same & before)] = row * C + c;
      }
      if (lane == lead) next[row] = p + __popcll(same);
      left &= ~same;
    }
  };
  if (found <= LIST) {
    for (int j = 0; j < found; j += 64) {
      const uint32_t k = j + lane < found ? kept[wave][j + lane] : 0;
      put(j + lane < found ? int(k >> 22) : -1, t0 + (k & ((1u << 22) - 1)));
    }
  } else {
    for (int64_t t = t0; t < t1; t += 64) put(row_of(t + lane < t1 ? a.index[t + lane] : -1), t + lane);
  }
  __syncthreads();
  if constexpr (!FIRST) zero_rows([&](int r) { return first[r + 1] == first[r]; });
}

// Sums in fp32: a wave takes 64 N columns of a segment, eight loads in flight, and writes
// the rows that end in it; a row's piece that goes on, or began before, is left in sums (the
// first piece of segment i in 2 i, the last in 2 i + 1).  Segments seg0 .. seg1 - 1.  Bound by its
// reads at random rows: 16384 x 4096 in bf16 33 us (5.6 TB/s with the rows it writes), 57344 x 1024
// 28 us (4.2 of reads alone).
template <class T, int N>
__global__ __launch_bounds__(256) void embed_sum(mmuon_embedding_args a, int each, int seg0, int seg1, GradSpace space) {
  const int all = *space.all;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunks = (a.width + 64 * N - 1) / (64 * N);
  const int64_t item = int64_t(blockIdx.x) * 4 + wave;
  const int s0 = int(item / chunks), seg = seg0 + s0, col = int(item - int64_t(s0) * chunks) * 64 * N + lane * N;
  const int p0 = seg * each, n = min(each, all - p0);
  if (seg >= seg1 || n <= 0) return;
  // lanes 0 .. n - 1: the positions; lane n: the one after, lane 63: the one before (rows only)
  const int at = lane <= n ? p0 + lane : p0 - 1;
  const bool is = (lane <= n || lane == 63) && at >= 0 && at < all;
  const int token = is && lane < n ? space.token[at] : 0, row = is ? space.row[at] : -1;
  const int after = __shfl_down(row, 1, 64);  // (all lanes take part)
  const uint64_t ends = __ballot(lane < n && row != after);
  const bool began = __builtin_amdgcn_readlane(row, 63) == __builtin_amdgcn_readlane(row, 0);  // before this SEG
  if (col >= a.width) return;
  const auto* dout = static_cast<const typename T::storage*>(a.dout) + col;
  float s[N];
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = 0.f;
  bool first = true;
  const auto piece = [&](int slot) { store_sums<N>(space.sums + (int64_t(seg) * 2 + slot) * a.width + col, s); };
  constexpr int U = 8;
  for (int p = 0; p < n; p += U) {
    float x[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
      load_n<T, N>(dout + __builtin_amdgcn_readlane(token, min(p + u, n - 1)) * a.dout_stride, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p + u >= n) break;
#pragma unroll
      for (int k = 0; k < N; ++k) s[k] += x[u][k];
      if (!(ends >> (p + u) & 1)) continue;
      if (first && began) {
        piece(0);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) s[k] *= a.scale;
        store_n<T, N>(static_cast<typename T::storage*>(a.dw) + int64_t(__builtin_amdgcn_readlane(row, p + u)) * a.width + col, s);
      }
      first = false;
#pragma unroll
      for (int k = 0; k < N; ++k) s[k] = 0.f;
    }
  }
  if (!(ends >> (n - 1) & 1)) piece(first ? 0 : 1);  // goes on in the next segment
}

// The rows that lie in several segments: a workgroup sums 32 N columns of the row that goes on
// from its segment (seg0 on), if it begins there; 8 runs of the row's pieces side by side, joined
// in order.  Bound by its latency: 3 to 8 us, where one word is not most of the tokens.
template <class T, int N>
__global__ __launch_bounds__(256) void embed_join(mmuon_embedding_args a, int size, int seg0, GradSpace space) {
  constexpr int LANES = 32, RUNS = 256 / LANES, SLICE = LANES * N;
  __shared__ float sums[RUNS][SLICE];
  const int all = *space.all, slices = (a.width + SLICE - 1) / SLICE;
  const int seg = seg0 + blockIdx.x / slices, slice = blockIdx.x % slices, p0 = seg * size;
  if (p0 + size >= all) return;
  const int r = space.row[p0 + size];
  if (space.row[p0 + size - 1] != r) return;
  const int lead = threadIdx.x & (size - 1);  // the row's first position, among this segment's
  const uint64_t mine = __ballot(space.row[p0 + lead] == r);
  const int f = p0 + __ffsll(static_cast<unsigned long long>(mine)) - 1;
  if (f == p0 && p0 > 0 && space.row[p0 - 1] == r) return;  // began before
  const int pieces = (f + space.count[f] - 1) / size - seg + 1;
  const int run = threadIdx.x / LANES, lane = threadIdx.x % LANES, col = slice * SLICE + lane * N;
  const int each = (pieces + RUNS - 1) / RUNS, k1 = min((run + 1) * each, pieces);
  float s[N];
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = 0.f;
  if (col < a.width) {
#pragma unroll 8
    for (int i = run * each; i < k1; ++i) {
      // the row is the last of its first segment and the first of the others
      const int slot = 2 * (seg + i) + (i == 0 && f > p0 ? 1 : 0);
      float x[N];
      load_sums<N>(space.sums + int64_t(slot) * a.width + col, x);
#pragma unroll
      for (int k = 0; k < N; ++k) s[k] += x[k];
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) sums[run][lane * N + k] = s[k];
  __syncthreads();
  auto* dst = static_cast<typename T::storage*>(a.dw) + int64_t(r) * a.width + slice * SLICE;
  for (int e = threadIdx.x; e < min(SLICE, a.width - slice * SLICE); e += 256) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < RUNS; ++k) v += sums[k][e];
    T::store(dst, e, v * a.scale);
  }
}

// Whether rows are whole 16-B chunks (8 elements of bf16, 4 of fp32).  Others go an element to a
// lane (16384 tokens of 50304 rows, Zipf's ids: 1024 columns of bf16 lookup 9.2 us, gradient 39, 1028
// of them 20 and 93; 1028 of fp32, which are whole chunks, 17 and 64).
template <class T>
bool whole_chunks(const void* base, int64_t stride, int64_t width) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && stride % CHUNK<T> == 0 && width % CHUNK<T> == 0;
}

// Workgroups of 256 threads in a launch, which holds fewer than 2^32 threads: more tokens or
// segments take several
constexpr int64_t MOST_BLOCKS = int64_t(1) << 23;

template <class T, int N>
void lookup_n(const mmuon_embedding_args& a, hipStream_t s) {
  const int chunks = a.width / N;
  int lanes = 16;  // about four chunks per thread
  while (lanes < 256 && lanes * 4 < chunks) lanes *= 2;
  const int each = 256 / lanes;
  // An output that the L2s (32 MiB) cannot hold is stored past them: 16384 x 4096 in bf16 40.0 ->
  // 34.0 us, 8192 x 4096 18.7 -> 17.6; a smaller one is read from there by what comes next.
  const bool past = a.tokens * a.width * int64_t(sizeof(typename T::storage)) > (int64_t(32) << 20);
  for (int64_t t = 0; t < a.tokens; t += MOST_BLOCKS * each) {
    mmuon_embedding_args p = a;
    p.tokens = std::min(a.tokens - t, MOST_BLOCKS * each);
    p.index = a.index + t;
    p.out = static_cast<typename T::storage*>(a.out) + t * a.width;
    const dim3 grid(unsigned((p.tokens + each - 1) / each)), block(256);
    if (past) hipLaunchKernelGGL((embed_lookup<T, N, true>), grid, block, 0, s, p, lanes);
    else hipLaunchKernelGGL((embed_lookup<T, N, false>), grid, block, 0, s, p, lanes);
  }
}
template <class T>
void lookup(const mmuon_embedding_args& a, hipStream_t s) {
  if (whole_chunks<T>(a.w, a.w_stride, a.width) && whole_chunks<T>(a.out, a.width, a.width)) lookup_n<T, CHUNK<T>>(a, s);
  else lookup_n<T, 1>(a, s);
}

// Classes: a power of two.  Many small workgroups (2048, eight per CU) where the ids are few
// enough for each to read them all; else 256, or what 1024 rows of a class need.
constexpr int64_t FEW_IDS = 4096;
int log2_classes(int64_t tokens, int64_t vocab) {
  int l = tokens <= FEW_IDS ? 11 : 8;
  const int most = tokens <= FEW_IDS ? 256 : 1024;
  while ((vocab + (int64_t(1) << l) - 1) >> l > most) ++l;
  while (l > 0 && int64_t(1) << (l - 1) >= vocab) --l;
  return l;
}

// Positions of a segment: the most that leave eight waves per CU something to sum (1000 tokens
// of 512 columns: 32 at a time 10.5 us, 8 at a time 5).
int segment(int64_t tokens, int64_t width, int columns) {
  int n = MAX_SEG;
  while (n > 8 && (tokens + n - 1) / n * ((width + columns - 1) / columns) < 2048) n /= 2;
  return n;
}

struct GradLayout {
  size_t token, row, count, all, total;  // the sums come first
};
GradLayout grad_layout(int64_t tokens, int64_t width) {
  GradLayout l;
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const int seg = segment(tokens, width, 512);  // (of fewer columns at a time it is no shorter)
  l.token = up(size_t(tokens > seg ? (tokens + seg - 1) / seg : 0) * 2 * width * 4);
  l.row = l.token + up(size_t(tokens) * 4);
  l.count = l.row + up(size_t(tokens) * 4);
  l.all = l.count + up(size_t(tokens) * 4);
  l.total = l.all + 256;
  return l;
}

template <class T, int N>
void gradient_n(const mmuon_embedding_args& a, hipStream_t s) {
  const int l = log2_classes(a.tokens, a.vocab);
  const int classes = int(std::min<int64_t>(int64_t(1) << l, a.vocab));
  const GradLayout at = grad_layout(a.tokens, a.width);
  char* ws = static_cast<char*>(a.workspace);
  const GradSpace space{reinterpret_cast<int*>(ws + at.token), reinterpret_cast<int*>(ws + at.row),
                        reinterpret_cast<int*>(ws + at.count), reinterpret_cast<int*>(ws + at.all),
                        reinterpret_cast<float*>(ws)};
  // A table that the Infinity Cache (256 MiB) cannot hold gets its zeros past the caches: 16384
  // tokens of 50304 x 4096 in bf16 135 -> 125 us; 50304 x 512 floats 27 -> 30.
  const bool past = a.vocab * a.width * int64_t(sizeof(typename T::storage)) > (int64_t(256) << 20);
  if (a.tokens <= FEW_IDS)
    hipLaunchKernelGGL((embed_rows<T, N, 4, 256, 64, true>), dim3(classes), dim3(256), 0, s, a, l, past, space);
  else hipLaunchKernelGGL((embed_rows<T, N, 16, 1024, 512, false>), dim3(classes), dim3(1024), 0, s, a, l, past, space);
  if (a.tokens == 0) return;
  const int seg = segment(a.tokens, a.width, 64 * N);
  const int segs = int((a.tokens + seg - 1) / seg);
  const int64_t chunks = (a.width + 64 * N - 1) / (64 * N), slices = (a.width + 32 * N - 1) / (32 * N);
  const auto launches = [](int n, int64_t each, const auto& fn) {  // n segments of `each` workgroups
    const int most = int(std::max<int64_t>(1, std::min<int64_t>(n, MOST_BLOCKS / each)));
    for (int i = 0; i < n; i += most) fn(i, std::min(n, i + most));
  };
  launches(segs, (chunks + 3) / 4, [&](int s0, int s1) {
    hipLaunchKernelGGL((embed_sum<T, N>), dim3(unsigned(((s1 - s0) * chunks + 3) / 4)), dim3(256), 0, s, a, seg, s0, s1,
                       space);
  });
  launches(segs - 1, slices, [&](int s0, int s1) {
    hipLaunchKernelGGL((embed_join<T, N>), dim3(unsigned((s1 - s0) * slices)), dim3(256), 0, s, a, seg, s0, space);
  });
}

template <class T>
void gradient(const mmuon_embedding_args& a, hipStream_t s) {
  if (whole_chunks<T>(a.dout, a.dout_stride, a.width) && whole_chunks<T>(a.dw, a.width, a.width)) gradient_n<T, CHUNK<T>>(a, s);
  else gradient_n<T, 1>(a, s);
}

}  // namespace

size_t embedding_workspace(const mmuon_embedding_args& a) {
  return grad_layout(a.tokens, a.width).total;
}

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
