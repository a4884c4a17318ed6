// The pipelined bf16 MFMA main loop of the batched products (butterfly.hip) and of the
// language-model head (cross_entropy.hip): operands described by strides and segments,
// staged by buffer loads straight into an LDS ring, in the slice forms of mfma_tile.hpp.
#pragma once

#include "common.hpp"
#include "mfma_tile.hpp"

namespace mmuon {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Lane offset that reads zeros: the resource covers [0, OOB) bytes.
constexpr uint32_t OOB = 0x80000000u;

// Raw buffer resource over [base, base + OOB): base address, stride 0,
// num_records OOB, the gfx9 data-format word.
__device__ __forceinline__ i32x4 buffer_rsrc(const char* base) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane(int(low_word(a)));
  r[1] = __builtin_amdgcn_readfirstlane(int(high_word(a) & 0xffffu));
  r[2] = int(OOB);
  r[3] = 0x00020000;
  return r;
}

// 16-B buffer load straight into LDS: lane l lands at lds + 16 l (M0 holds the
// wave-uniform LDS address).  Inline assembly for the same reason as dma16: the
// pipeline waits for exactly the slice it reads.
// m0 is listed as clobbered (the asm writes it); clang warns that m0 is a
// register it reserves for its own uses, which it sets right before each.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void bdma16(i32x4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(voff), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory", "m0");
}
#pragma clang diagnostic pop

// floor(n / d) for 0 <= n < 2^24, 1 <= d < 2^16, with magic = ceil(2^40 / d)
// (exact because n d < 2^40).
__host__ __device__ __forceinline__ int64_t seg_div(int64_t n, uint64_t magic) {
  return int64_t((uint64_t(n) * magic) >> 40);
}
uint64_t seg_magic(int64_t d) { return ((uint64_t(1) << 40) + uint64_t(d) - 1) / uint64_t(d); }

// GEMM operand: element (mn, k) of batch g sits at
//   base + g bstride + seg(mn) + seg(k),
//   seg(x) = (x / xseg) xseg_stride + (x % xseg) xstride.
// Segments express the riffle permutations; an unsegmented index has
// xseg > its extent.  K form: kstride == 2 (rows of K contiguous); T form:
// mstride == 2 (MN contiguous).  Indices mn >= extent read as zeros.
struct GOp {
  const char* base;
  int64_t bstride;
  int64_t mstride, mseg_stride;
  int64_t kstride, kseg_stride;
  uint64_t mmagic, kmagic;
  int32_t mseg, kseg;
  int32_t extent;
  int32_t pad;
};

__device__ __forceinline__ int64_t mn_off(const GOp& o, int64_t m) {
  const int64_t s = seg_div(m, o.mmagic);
  return s * o.mseg_stride + (m - s * o.mseg) * o.mstride;
}
// An operand's walk over K, one slice of BK at a time.  Segments are whole slices
// (multiples of 32), so a slice lies in one.  (Forming each slice's address from its
// index, a 64-bit division and three products, and testing every load for the end of K
// paced the small tiles: 8 tokens of 4 x 1024 x 1024 11.5 -> 10.4 us, 500 tokens of 4 x
// 512 x 1376 12.7 -> 11.4.  Rings of 8 or 16 slots, and reading a whole slice's fragments
// behind the barrier, did not help them.)
struct KWalk {
  const char* p;       // the slice's first element (tile row 0)
  int64_t step, wrap;  // bytes to the next slice, and beyond that into the next segment
  int pos, seg;        // the slice's place in its segment, the segment's length
  __device__ __forceinline__ void start(const GOp& o, const char* base, int k) {
    const int64_t s = seg_div(k, o.kmagic);
    pos = k - int(s) * o.kseg;
    seg = o.kseg;
    p = base + s * o.kseg_stride + int64_t(pos) * o.kstride;
    step = int64_t(BK) * o.kstride;
    wrap = o.kseg_stride - int64_t(o.kseg) * o.kstride;
  }
  __device__ __forceinline__ void next() {
    p += step;
    pos += BK;
    if (pos == seg) {
      p += wrap;
      pos = 0;
    }
  }
};

// ---------------------------------------------------------------------------
// Tile geometries: GM x GN waves, each WI x WJ MFMA tiles of 32 x 32; RING slices
// of 32 k in LDS.
// ---------------------------------------------------------------------------
template <int GM_, int GN_, int WI_, int WJ_, int RING_>
struct Geo {
  static constexpr int GM = GM_, GN = GN_, WI = WI_, WJ = WJ_, RING = RING_;
  static constexpr int NW = GM * GN, NTH = 64 * NW;
  static constexpr int BM = 32 * WI * GM, BN = 32 * WJ * GN;
  static constexpr int RSLB = BM * BK * 2, SLOTB = (BM + BN) * BK * 2;  // bytes of a row slice, of a slot
  static constexpr int RL = BM / 16 / NW, CL = BN / 16 / NW;            // 1 KiB loads per wave and operand slice
  static constexpr int DMA = RL + CL;
  static constexpr int LDS = RING * SLOTB;
  static constexpr int PER_CU = 160 * 1024 / LDS < 4 ? 160 * 1024 / LDS : 4;  // workgroups resident per CU
  static_assert(RL * NW * 16 == BM && CL * NW * 16 == BN, "whole loads per wave");
  static_assert(BM * BN * 2 <= LDS && LDS <= 160 * 1024, "the staged tile fits in the ring");
  // Staged tile T[j][i] = D[i][j]: rows of BM bf16, 16-B chunk c of row r at c ^ g(r),
  // g distinct over the rows that one access touches (mfma_tile.hpp, tile_off; rows of
  // 128 B take two per pass over the banks)
  static __device__ __forceinline__ uint32_t tile_at(int r, int c) {
    const int g = BM >= 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (r >> 1) & 7;
    return uint32_t(r * BM * 2 + (((c >> 3) ^ g) << 4) + ((c & 7) << 1));
  }
};

// ---------------------------------------------------------------------------
// The pipelined main loop (the NS kernels' schedule with both operand forms
// fixed per launch): slice kt in ring slot kt % RING, RING - 2 slices in flight
// behind the one being read, fragment reads and buffer loads interleaved with the
// MFMAs.  (256 x 256 tiles: a fifth slot, the whole LDS, measured slightly slower.)
// ---------------------------------------------------------------------------
template <class GE, bool AT, bool BT>
struct GPipe {
  static constexpr int RING = GE::RING, WI = GE::WI, WJ = GE::WJ, NM = WI * WJ, NR = WI + WJ;
  struct Fr {
    bf16x8 r[WI];
    bf16x8 c[WJ];
  };
  typedef f32x16 Acc[WI][WJ];
  KWalk ak, bk;            // the slice to load next, of the two operands
  int nxt;                 // its index (the last slice stays: it refills consumed slots)
  uint32_t loff[GE::DMA];  // per-lane byte offsets of the loads (OOB: beyond the extent)
  uint32_t tail[GE::DMA];  // OOB where the load's element lies beyond the last slice's K
  int KT;
  int wave, lane, wm, wn;
  char* lds;
  uint32_t lds0;
  uint32_t kfrag[BK / 16];
  uint32_t tfrag_r, tfrag_c;

  __device__ __forceinline__ const uint16_t* slot(int kt) const {
    return reinterpret_cast<const uint16_t*>(lds + (uint32_t(kt) % RING) * GE::SLOTB);
  }

  // Load Q (row operand first) of the next slice into the slot of slice slot_kt.
  // Load u = RL wave + Q (CL wave + Q - RL) of the operand's BM / 16 (BN / 16).
  // K form: operand rows 16 u + lane/4, chunk (lane%4) ^ ((lane>>4)&3); T form: k rows
  // 16 (u%2) + lane/4 of the slice, MN 32 (u/2) + 8 (lane%4).  Either way the load
  // lands at byte 1024 u of the operand's slice.
  template <int Q>
  __device__ __forceinline__ void issue_one(int slot_kt) const {
    constexpr bool ROW = Q < GE::RL;
    const int u = ROW ? GE::RL * wave + Q : GE::CL * wave + Q - GE::RL;
    const uint32_t dst = lds0 + (uint32_t(slot_kt) % RING) * GE::SLOTB + (ROW ? 0 : GE::RSLB) + u * 1024;
    const uint32_t last = nxt == KT - 1 ? OOB : 0;
    bdma16(buffer_rsrc(ROW ? ak.p : bk.p), loff[Q] | (tail[Q] & last), dst);
  }
  template <int Q0, int Q1>
  __device__ __forceinline__ void issue(int slot_kt) const {
    if constexpr (Q0 < Q1) {
      issue_one<Q0>(slot_kt);
      issue<Q0 + 1, Q1>(slot_kt);
    }
  }
  __device__ __forceinline__ void advance() {
    if (nxt + 1 < KT) {
      ak.next();
      bk.next();
      ++nxt;
    }
  }

  template <int KK, int G>
  __device__ __forceinline__ void load_one(int kt, Fr& f) const {
    const uint16_t* sr = slot(kt);
    const uint16_t* sc = sr + GE::RSLB / 2;
    if constexpr (G < WJ)
      f.c[G] = BT ? frag_rowmajor_tr(sc, tfrag_c + G * 2048, KK) : frag_kmajor(sc, kfrag[KK], (wn * WJ + G) * 32);
    else
      f.r[G - WJ] = AT ? frag_rowmajor_tr(sr, tfrag_r + (G - WJ) * 2048, KK)
                       : frag_kmajor(sr, kfrag[KK], (wm * WI + G - WJ) * 32);
  }
  template <int KK, int G0, int G1>
  __device__ __forceinline__ void load(int kt, Fr& f) const {
    if constexpr (G0 < G1) {
      load_one<KK, G0>(kt, f);
      load<KK, G0 + 1, G1>(kt, f);
    }
  }

  // MFMA g of a k step, with its share of the fragment reads of the next step and,
  // in the second k step, of the direct loads
  template <int KK, int g>
  __device__ __forceinline__ void half(int kt, const Fr& f, Fr& n, Acc& acc) const {
    if constexpr (g < NM) {
      acc[g / WJ][g % WJ] = mfma(f.r[g / WJ], f.c[g % WJ], acc[g / WJ][g % WJ]);
      if constexpr (KK == 0) {
        load<1, g * NR / NM, (g + 1) * NR / NM>(kt, n);
      } else {
        load<0, g * NR / NM, (g + 1) * NR / NM>(kt + 1, n);
        issue<g * GE::DMA / NM, (g + 1) * GE::DMA / NM>(kt + RING - 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      half<KK, g + 1>(kt, f, n, acc);
    }
  }

  __device__ __forceinline__ void body(int kt, Fr& fa, Fr& fb, Acc& acc) {
    half<0, 0>(kt, fa, fb, acc);
    wait_vm<(RING - 3) * GE::DMA>();  // slice kt+1 landed
    barrier();
    // raised wave priority from the barrier to the end of k step 1, so the
    // SIMD's wave still in this phase wins issue over one already in the next
    // step and catches up before the next barrier
    __builtin_amdgcn_s_setprio(1);
    half<1, 0>(kt, fb, fa, acc);
    __builtin_amdgcn_s_setprio(0);
    advance();
  }

  __device__ __forceinline__ void run(Acc& acc) {
#pragma unroll
    for (int i = 0; i < WI; ++i)
#pragma unroll
      for (int j = 0; j < WJ; ++j) acc[i][j] = f32x16{};
#pragma unroll
    for (int q = 0; q < RING - 1; ++q) {
      issue<0, GE::DMA>(q);
      advance();
    }
    wait_vm<(RING - 2) * GE::DMA>();  // slice 0 landed
    barrier();
    Fr fa, fb;
    load<0, 0, NR>(0, fa);
    for (int kt = 0; kt < KT; ++kt) body(kt, fa, fb, acc);
    wait_vm<0>();  // the refills of the last steps land before the ring is reused
  }
};

// Per-lane byte offset of load u of an operand (tile origin mn0), OOB beyond
// its extent.
template <bool T>
__device__ __forceinline__ uint32_t lane_offset(const GOp& o, int mn0, int u, int lane) {
  int mn;
  int64_t off;
  if (T) {
    mn = mn0 + 32 * (u >> 1) + 8 * (lane & 3);
    off = int64_t(16 * (u & 1) + (lane >> 2)) * o.kstride;
  } else {
    mn = mn0 + 16 * u + (lane >> 2);
    off = int64_t((lane & 3) ^ ((lane >> 4) & 3)) * 16;
  }
  if (mn >= o.extent) return OOB;
  return uint32_t(off + mn_off(o, mn) - mn_off(o, mn0));
}

// Accumulators -> the staging area as T[j][i] = D[i][j], bf16.
template <class GE>
__device__ __forceinline__ void stage_acc(char* stage, const f32x16 (&acc)[GE::WI][GE::WJ]) {
  const int tid = fresh_tid();
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / GE::GN, wn = wave % GE::GN;
#pragma unroll
  for (int i = 0; i < GE::WI; ++i)
#pragma unroll
    for (int j = 0; j < GE::WJ; ++j)
#pragma unroll
      for (int qg = 0; qg < 4; ++qg) {
        const f32x16& v = acc[i][j];
        const int row = (wn * GE::WJ + j) * 32 + (lane & 31);
        const int col = (wm * GE::WI + i) * 32 + qg * 8 + (lane >> 5) * 4;
        *reinterpret_cast<uint2*>(stage + GE::tile_at(row, col)) =
            make_uint2(f2bf2(v[qg * 4], v[qg * 4 + 1]), f2bf2(v[qg * 4 + 2], v[qg * 4 + 3]));
      }
}

constexpr int64_t UNSEG = int64_t(1) << 24;  // segment length of an unsegmented index

GOp make_op(const void* base, int64_t bstride, int64_t mstride, int64_t kstride, int extent,
            int64_t mseg = UNSEG, int64_t mseg_stride = 0, int64_t kseg = UNSEG, int64_t kseg_stride = 0) {
  GOp o{};
  o.base = static_cast<const char*>(base);
  o.bstride = bstride;
  o.mstride = mstride;
  o.kstride = kstride;
  o.mseg = int32_t(mseg);
  o.mseg_stride = mseg_stride;
  o.kseg = int32_t(kseg);
  o.kseg_stride = kseg_stride;
  o.mmagic = seg_magic(mseg);
  o.kmagic = seg_magic(kseg);
  o.extent = extent;
  return o;
}

int cdiv(int64_t a, int64_t b) { return int((a + b - 1) / b); }

}  // namespace
}  // namespace mmuon
