// Product of two matrices held in 8-bit blocks: C[M,N] = A . B^T, A [M,K] and B [N,K] e4m3, contiguous along the contraction,
// one power-of-two scale per row and block of 128 contraction elements, fp32 accumulation, bf16 store.
//
//   C[m, n] (+)= sum_kb 2^(sa[kb, m] - 127 + sb[kb, n] - 127) sum_{k in block kb} a[m, k] b[n, k]
//
// The matrix instruction (v_mfma_scale_f32_32x32x64_f8f6f4, 131072 FLOP in 64 cycles, twice the rate of the unscaled 8-bit ones)
// multiplies by 2^(scale - 127) of both operands' rows on its way into the sum, so the scales cost nothing but their loads.
//
// Precision: a product of two e4m3 values has 8 bits and is exact in the unit.  The instruction adds fewer than 32 bits of it: of each
// eight consecutive contraction elements it takes E, the largest sum of two exponents, and cuts all eight products, towards zero, to
// multiples of 2^(E - 13); 64 elements' groups and the accumulator are then added exactly and rounded once to fp32 (reproduced bit for
// bit on random operands).  That is the format's full rate and cannot be asked for otherwise; it leaves sums 1.5e-5 off (256 x 512 x
// 30000, relative to 64 bits, in the norm), where a bf16 store leaves 1.7e-3, and turns one store's rounding in a hundred to the other
// neighbour.  Sums over the cuts of a contraction, over waves and with C are fp32; the one rounding to bf16 is the store's.
//
// What bounds it: large products the card's power.  16384 x 28672 x 4096 takes 1403 us (2.74 PFLOP/s) on normally distributed values
// and 1033 (3.73) on operands of one value, with the same instructions; 16384 x 7168 x 4096 353 and 262 us, 16384 x 4096 x 7168 337
// and 254.  Products of few rows are bound by B's bytes (1 x 28672 x 4096 18.4 us: 6.4 TB/s, from the 256 MiB cache), those of one
// tile per unit by their loads' latency and the launch.  The tiles below 192 x 256 need LDS for longer than the matrix pipe: a K-step of
// 128 x 256 writes 48 KB and reads 96, 0.5 us at 128 bytes a cycle where its MFMAs are 0.43; it takes 0.73, and what the rest is has not
// been shown (three K-steps under way instead of two: no faster).
#include "kr_common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

namespace {

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8;
typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;

constexpr int BK = 128;        // contraction elements (and bytes) of a K-step: one scale block
constexpr int NTHREADS = 256;
constexpr int kXcds = 8;
constexpr int kGroupM = 4;
enum Out { kStore, kAccumulate, kPartial };

struct Args {
  const uint8_t* a;
  const uint8_t* sa;
  const uint8_t* b;
  const uint8_t* sb;
  bf16* c;
  float* partial;
  int64_t lda, ldb, ldc;
  int lsa, lsb;            // bytes from one scale block's row to the next (multiples of 4)
  int m, n, ksteps, steps_per, splits;
};
// The pieces that a contraction lies in, one behind the other, each of whole blocks (Args: m, n, ksteps of all of them, the output)
constexpr int kMostSegments = KR_BLOCK_GEMM_MAX_SEGMENTS;
struct Segments {
  const uint8_t *a[kMostSegments], *sa[kMostSegments], *b[kMostSegments], *sb[kMostSegments];
  int lda[kMostSegments], ldb[kMostSegments], lsa[kMostSegments], lsb[kMostSegments], ksteps[kMostSegments];
};
struct OnePiece {};

__device__ __forceinline__ uint32_t lds_addr(const uint8_t* p) { return (uint32_t)(uintptr_t)(KR_LDS const uint8_t*)p; }

// One direct global -> LDS load: lane p's 16 bytes land at lds + 16 p (lds wave-uniform).  Inline assembly, so that the compiler does
// not drain it in front of every barrier; the K loop waits for all of them by hand.
template <int IMM>
__device__ __forceinline__ void dma_b128(const void* base, uint32_t byte_off, uint32_t lds_base) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds_base), "v"(byte_off), "s"(base), "n"(IMM)
               : "memory", "m0", "scc");
}

__device__ __forceinline__ void dma_b32(const void* base, uint32_t byte_off, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(lds_base), "v"(byte_off), "s"(base)
               : "memory", "m0");
}
// s_waitcnt immediate for vmcnt(n); lgkmcnt and expcnt untouched
constexpr int vm_wait(int n) { return 0x0f70 | (n & 15) | ((n >> 4) << 14); }

// ids congruent mod 8 run on one XCD: each XCD takes a compact band of C
__device__ __forceinline__ void tile_of(int pid, int nblocks, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int q = nblocks / kXcds, r = nblocks % kXcds;
  const int xcd = pid % kXcds, local = pid / kXcds;
  const int lid = xcd * q + (xcd < r ? xcd : r) + local;
  const int per_band = kGroupM * tiles_n;
  const int band = lid / per_band;
  const int first_m = band * kGroupM;
  const int band_rows = (tiles_m - first_m) < kGroupM ? (tiles_m - first_m) : kGroupM;
  const int in_band = lid - band * per_band;
  tn = in_band / band_rows;
  tm = first_m + in_band - tn * band_rows;
}

template <int W>
__device__ __forceinline__ int lds_scales(uint32_t a) {
  if constexpr (W == 4) return *(KR_LDS const int*)a;
  if constexpr (W == 3) return *(KR_LDS const uint8_t*)a | *(KR_LDS const uint8_t*)(a + 1) << 8 | *(KR_LDS const uint8_t*)(a + 2) << 16;
  if constexpr (W == 2) return *(KR_LDS const uint16_t*)a;
  return *(KR_LDS const uint8_t*)a;
}
template <int N>
using Int = std::integral_constant<int, N>;
template <class F, int... I>
__device__ __forceinline__ void each(F&& f, std::integer_sequence<int, I...>) {
  (f(Int<I>{}), ...);
}

// LDS of one instance: eight blocks of 64 contraction bytes (both operands' halves of two K-steps), two K-steps' scales, staging
constexpr int stage_row(int wn) { return wn == 4 ? 128 : 64; }
constexpr uint32_t block_bytes(int w) { return 64 * w * 64; }
constexpr size_t lds_bytes(int wt, int wn) {
  return 4 * (size_t)(block_bytes(wt > wn ? wt : wn) * 2) + 2 * 512 + 4 * 32 * stage_row(wn);
}

// WT x WN tiles of 32 x 32 per wave, four waves as 2 x 2: 64 WT x 64 WN of C per workgroup.
//   * Row j of a wave's MFMA tile g is row W j + g of its 32 W rows (W = WT for A, WN for B), so that the scales of all its tiles for a
//     K-step are W consecutive bytes, as the instruction's byte selector takes them, and a lane ends up with 4 WN consecutive columns
//     of C.  Rows lie in LDS in tile order: the load of a tile places them.
//   * A K-step is two phases, one per half of 64 contraction elements: a phase is the MFMAs on the fragments in registers, and between
//     them the fragment reads of the next phase and the loads of one operand two K-steps ahead.  In LDS the halves are blocks of
//     their own: the block that a phase has read is free behind the barrier at its end, so eight blocks hold the two K-steps that the
//     loads run ahead, every phase loads as much as the others, and every load has one phase to land at least.
//   * The barrier stands in front of a phase's last MFMAs, which run while the waves meet.
//   * A block's row is 64 bytes, its 16-byte chunks XORed with (row >> 2) & 3: the 16 rows that a fragment read takes at a time cover
//     all banks once.  Both halves of a row's 128 bytes are requested one behind the other: one line fetched from the L2.
//   * A contraction in pieces (Segments) moves the requests from one piece's operands to the next's between two K-steps; the computation
//     does not know of it.  (us, one operand, two and four pieces: 7168 x 4096 x 16384 339, 346, 343; 4096 x 3584 x 16384 170, 171, 171;
//     1536 x 4096 x 6144 39, 41, 42.)
template <int WT, int WN, int OUT, class Contraction>
__global__ __launch_bounds__(NTHREADS, WT * WN == 1 ? 3 : WT * WN == 4 ? 2 : 1) void block_gemm_kernel(Args g, Contraction pieces) {
#ifdef __HIP_DEVICE_COMPILE__   // (the host's pass over this file cannot place the registers that the assembly names)
  constexpr int BM = 64 * WT, BN = 64 * WN;
  constexpr int NA = 2 * WT, NB = 2 * WN;                       // loads per wave of an operand's K-step, both halves
  constexpr uint32_t BLK = block_bytes(WT > WN ? WT : WN);
  constexpr int SLOTS = WT * WN;                                // MFMAs of a phase
  constexpr bool SEGMENTS = std::is_same_v<Contraction, Segments>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const uint32_t smem_b = lds_addr(smem);
  const uint32_t scales_b = smem_b + 8 * BLK;
  const uint32_t stage = scales_b + 1024 + (uint32_t)wave * (32 * stage_row(WN));
  const int tiles_m = (g.m + BM - 1) / BM, tiles_n = (g.n + BN - 1) / BN;
  const int ntiles = tiles_m * tiles_n;
  const int total = ntiles * (OUT == kPartial ? g.splits : 1);

  struct Item {
    int m0, n0, k0, nk, split;
  };
  auto select = [&](int v) {
    Item it;
    it.split = v / ntiles;
    int tm, tn;
    tile_of(v - it.split * ntiles, ntiles, tiles_m, tiles_n, tm, tn);
    it.m0 = tm * BM;
    it.n0 = tn * BN;
    it.k0 = OUT == kPartial ? it.split * g.steps_per : 0;
    it.nk = OUT == kPartial ? (g.ksteps - it.k0 < g.steps_per ? g.ksteps - it.k0 : g.steps_per) : g.ksteps;
    return it;
  };

  // ---- requests: a cursor over the K-steps of all items of this workgroup, two steps ahead of the computation ----
  int r_item = blockIdx.x;
  int r_left;
  const uint8_t *ra, *rb, *rs;          // of the K-step to request next (wave-uniform); rs: the scales this wave loads
  uint32_t la[WT], lb[WN], ls;
  int64_t rs_step = wn ? g.lsb : g.lsa;
  int r_m0, r_n0, r_piece, r_left_piece;   // SEGMENTS
  // rows of the tile at (m0, n0), `lda` and `ldb` bytes apart
  auto address = [&](int m0, int n0, uint32_t lda, uint32_t ldb) {
    int l2 = lane;
    asm volatile("" : "+v"(l2));
    // load i of a wave fills block rows 16 (wave + 4 i) .. + 15; beyond the matrix: its last row (never stored)
    const int sub = l2 >> 2;
    const int chunk = ((l2 & 3) ^ ((sub >> 2) & 3)) << 4;
#pragma unroll
    for (int i = 0; i < WT; ++i) {
      const int row = 16 * (wave + 4 * i) + sub;
      const int w = row / (32 * WT), t = row % (32 * WT) / 32, j = row % 32;
      int r = 32 * WT * w + WT * j + t;
      r = m0 + r < g.m ? r : g.m - 1 - m0;
      la[i] = (uint32_t)r * lda + (uint32_t)chunk;
    }
#pragma unroll
    for (int i = 0; i < WN; ++i) {
      const int row = 16 * (wave + 4 * i) + sub;
      const int w = row / (32 * WN), t = row % (32 * WN) / 32, j = row % 32;
      int r = 32 * WN * w + WN * j + t;
      r = n0 + r < g.n ? r : g.n - 1 - n0;
      lb[i] = (uint32_t)r * ldb + (uint32_t)chunk;
    }
    // four rows' scales a lane; beyond the matrix: those of its last row
    const int sr = (wn ? n0 : m0) + 4 * l2, most = ((wn ? g.n : g.m) - 1) & ~3;
    ls = (uint32_t)(sr < most ? sr : most);
  };
  auto enter = [&](int piece, int step) {   // (SEGMENTS: K-step `step` of a piece, for the tile at r_m0, r_n0)
    if constexpr (SEGMENTS) {
      r_piece = piece;
      r_left_piece = pieces.ksteps[piece] - step;
      const int lda = pieces.lda[piece], ldb = pieces.ldb[piece];
      ra = pieces.a[piece] + (int64_t)r_m0 * lda + (int64_t)step * BK;
      rb = pieces.b[piece] + (int64_t)r_n0 * ldb + (int64_t)step * BK;
      rs_step = wn ? pieces.lsb[piece] : pieces.lsa[piece];
      rs = (wn ? pieces.sb[piece] : pieces.sa[piece]) + (int64_t)step * rs_step;
      address(r_m0, r_n0, (uint32_t)lda, (uint32_t)ldb);
    }
  };
  auto aim = [&](int v) {
    const Item it = select(v);
    r_left = it.nk;
    if constexpr (SEGMENTS) {
      r_m0 = it.m0;
      r_n0 = it.n0;
      int piece = 0, step = it.k0;
      while (step >= pieces.ksteps[piece]) step -= pieces.ksteps[piece++];
      enter(piece, step);
    } else {
      ra = g.a + (int64_t)it.m0 * g.lda + (int64_t)it.k0 * BK;
      rb = g.b + (int64_t)it.n0 * g.ldb + (int64_t)it.k0 * BK;
      rs = (wn ? g.sb : g.sa) + (int64_t)it.k0 * rs_step;
      address(it.m0, it.n0, (uint32_t)g.lda, (uint32_t)g.ldb);
    }
  };
  // (behind the last item's last K-step it stays there: the K loop requests that one again rather than branch, two steps in all)
  auto advance = [&]() {
    if (--r_left > 0) {
      if constexpr (SEGMENTS) {
        if (--r_left_piece == 0) {
          enter(r_piece + 1, 0);
          return;
        }
      }
      ra += BK;
      rb += BK;
      rs += rs_step;
    } else if (r_item + (int)gridDim.x < total) {
      r_item += gridDim.x;
      aim(r_item);
    } else {
      r_left = 1;
    }
  };
  // load d of an operand's K-step: half d & 1 of the rows of load d / 2; to block k0 (half 0) or k1
  auto request_a = [&](auto d, uint32_t k0, uint32_t k1) {
    constexpr int i = decltype(d)::value;
    dma_b128<(i >> 1) * 4096>(ra + 64 * (i & 1), la[i >> 1], (i & 1 ? k1 : k0) + (uint32_t)wave * 1024u);
  };
  auto request_b = [&](auto d, uint32_t k0, uint32_t k1) {
    constexpr int i = decltype(d)::value;
    dma_b128<(i >> 1) * 4096>(rb + 64 * (i & 1), lb[i >> 1], (i & 1 ? k1 : k0) + (uint32_t)wave * 1024u);
  };
  // a K-step's scales: waves 0 and 2 load A's 256 bytes, 1 and 3 B's (the same bytes to the same place)
  auto request_scales = [&](uint32_t slot) { dma_b32(rs, ls, slot + (uint32_t)wn * 256u); };

  // The accumulators of the large tile are the wave's 256 accumulation registers (its MFMAs are inline assembly, to pin them there:
  // with the builtin the compiler moves and spills them); smaller tiles leave them to the compiler.
  constexpr bool PINNED = WT * WN > 4;
  f32x16 acc[WT][WN];
  struct Frags {
    i32x8 a[WT], b[WN];
  } X, Y;
  auto clear = [&]() {
    if constexpr (!PINNED) {
#pragma unroll
      for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    }
  };

  // fragment addresses: lane l takes row l % 32 of a tile, chunks 2 (l / 32) and + 1 of a half
  const uint32_t frag0 = (uint32_t)((lane & 31) * 64 + (((2 * (lane >> 5)) ^ ((lane >> 2) & 3)) << 4));
  const uint32_t fa = (uint32_t)(wm * 32 * WT * 64) + frag0, fb = (uint32_t)(wn * 32 * WN * 64) + frag0;
  auto frag = [&](uint32_t a) {
    const i32x4 lo = *(KR_LDS const i32x4*)a, hi = *(KR_LDS const i32x4*)(a ^ 16u);
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  const uint32_t sca = (uint32_t)(32 * WT * wm + WT * (lane & 31)), scb = 256u + (uint32_t)(32 * WN * wn + WN * (lane & 31));

  // One phase: the MFMAs on `cur`, and between them the fragments of the next from blocks na / nb, `loads` (called with 0 ..
  // NLOADS - 1) and, in front of the last ones, `meet`.
  // FIRST: of an item; the pinned accumulators start from the instruction's constant 0 instead of being cleared.
  auto phase = [&](auto first_tag, Frags& cur, Frags& nxt, int sa, int sb, uint32_t na, uint32_t nb, auto nloads_tag, auto loads, auto meet) {
    constexpr bool FIRST = decltype(first_tag)::value;
    constexpr int NLOADS = decltype(nloads_tag)::value;
    const uint32_t a0 = fa + na, b0 = fb + nb;
    auto fetch = [&](auto f) {   // fragments in the order that the next phase takes them
      constexpr int i = decltype(f)::value;
      if constexpr (i == 0) nxt.a[0] = frag(a0);
      else if constexpr (i <= WN) nxt.b[i - 1] = frag(b0 + (i - 1) * 32 * 64);
      else nxt.a[i - WN] = frag(a0 + (i - WN) * 32 * 64);
    };
    constexpr int NF = WT + WN;
    // the MFMA that `meet` stands in front of.  (Large tile, behind all, in front of the last, the last two, the last three, us: 16384 x
    // 7168 x 4096 359, 359, 357, 359; 16384 x 28672 x 4096 1440, 1473, 1430, 1454; 16384 x 4096 x 7168 345, 344, 342, 344.)
    constexpr int LAST = SLOTS >= 12 ? SLOTS - 2 : SLOTS >= 4 ? SLOTS - 1 : SLOTS;
    // fragment f is read behind MFMA f * (LAST - 2) / NF, load d behind MFMA d * (LAST - 1) / NLOADS
    each([&](auto s) {
      constexpr int slot = decltype(s)::value, gi = slot / WN, ni = slot % WN;
      if constexpr (slot == LAST) meet();
      if constexpr (PINNED) {
        if constexpr (slot == 0) asm volatile("s_nop 3" ::: "memory");   // (the scales may just have been moved)
        if constexpr (FIRST)
          asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0]"
                       : "=a"(acc[gi][ni])
                       : "v"(cur.b[ni]), "v"(cur.a[gi]), "v"(sb), "v"(sa), "n"(ni & 1), "n"(gi & 1), "n"(ni >> 1), "n"(gi >> 1));
        else
          asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0]"
                       : "+a"(acc[gi][ni])
                       : "v"(cur.b[ni]), "v"(cur.a[gi]), "v"(sb), "v"(sa), "n"(ni & 1), "n"(gi & 1), "n"(ni >> 1), "n"(gi >> 1));
      } else {
        acc[gi][ni] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(cur.b[ni], cur.a[gi], acc[gi][ni], 0, 0, ni, sb, gi, sa);
      }
      each([&](auto f) {
        constexpr int span = LAST - 2 > 1 ? LAST - 2 : 1;
        if constexpr (decltype(f)::value * span / NF == slot) fetch(f);
      }, std::make_integer_sequence<int, NF>{});
      each([&](auto d) {
        constexpr int span = LAST - 1 > 1 ? LAST - 1 : 1;
        if constexpr (decltype(d)::value * span / NLOADS == slot) loads(d);
      }, std::make_integer_sequence<int, NLOADS>{});
      __builtin_amdgcn_sched_barrier(0);
    }, std::make_integer_sequence<int, SLOTS>{});
    if constexpr (LAST == SLOTS) meet();
  };

  // ---- start: K-steps 0 and 1 requested, half 0 of step 0 read ----
  struct Blocks {
    uint32_t a0, a1, b0, b1, sc;
  };
  Blocks now = {smem_b, smem_b + BLK, smem_b + 2 * BLK, smem_b + 3 * BLK, scales_b};
  Blocks next = {smem_b + 4 * BLK, smem_b + 5 * BLK, smem_b + 6 * BLK, smem_b + 7 * BLK, scales_b + 512};
  auto request_step = [&](const Blocks& to) {
    each([&](auto d) { request_a(d, to.a0, to.a1); }, std::make_integer_sequence<int, NA>{});
    request_scales(to.sc);
    each([&](auto d) { request_b(d, to.b0, to.b1); }, std::make_integer_sequence<int, NB>{});
    advance();
  };
  Item it = select(blockIdx.x);
  int item = blockIdx.x;
  aim(r_item);
  request_step(now);
  request_step(next);
  clear();
  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
  kr_barrier();
#pragma unroll
  for (int i = 0; i < WT; ++i) X.a[i] = frag(fa + now.a0 + i * 32 * 64);
#pragma unroll
  for (int i = 0; i < WN; ++i) X.b[i] = frag(fb + now.b0 + i * 32 * 64);
  int sa = lds_scales<WT>(now.sc + sca), sb = lds_scales<WN>(now.sc + scb);
  kr_barrier();                         // (every wave has read what the first phase's loads overwrite)
  auto k_step = [&](auto first) {
    // half 0: half 1 of this step is read; A two steps ahead goes where both operands' half 0 lay
    phase(first, X, Y, sa, sb, now.a1, now.b1, Int<NA + 1>{},
          [&](auto d) {
            if constexpr (decltype(d)::value < NA) request_a(d, now.a0, now.b0);
            else request_scales(now.sc);
          },
          [&]() {
            __builtin_amdgcn_s_waitcnt(vm_wait(NA + 1));   // the next step has landed
            kr_barrier();
          });
    // half 1: half 0 of the next step and its scales are read; B two steps ahead goes where this step's half 1 lay
    const int sa1 = lds_scales<WT>(next.sc + sca), sb1 = lds_scales<WN>(next.sc + scb);
    phase(std::false_type{}, Y, X, sa, sb, next.a0, next.b0, Int<NB>{}, [&](auto d) { request_b(d, now.a1, now.b1); }, [&]() { kr_barrier(); });
    advance();
    sa = sa1;
    sb = sb1;
    const Blocks ahead = {now.a0, now.b0, now.a1, now.b1, now.sc};
    now = next;
    next = ahead;
  };
  for (;;) {
    k_step(std::integral_constant<bool, PINNED>{});
    for (int t = 1; t < it.nk; ++t) k_step(std::false_type{});

    // the compiler does not know the latency of MFMAs in assembly: let the last ones finish before their results are read
    if constexpr (PINNED) asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");

    // ---- epilogue: lane l holds row WT (l % 32) + g of its wave, columns WN (8 q + 4 (l / 32)) .. + 4 WN - 1 for q = 0..3 ----
    {
      int le = lane;
      asm volatile("" : "+v"(le));
      const int j = le & 31, hi = le >> 5;
      const int m_wave = it.m0 + 32 * WT * wm, n_wave = it.n0 + 32 * WN * wn;
      constexpr int SW = stage_row(WN), PASSES = 64 * WN / SW, QP = 4 / PASSES, PIECES = SW / 16, RPP = 64 / PIECES, PER = 32 / RPP;
      const int piece = le % PIECES, r0 = le / PIECES;
      bf16x8 held[PER];   // the pass before
      auto store_pass = [&](int pass) {
        const int gi = pass / PASSES, col = n_wave + pass % PASSES * (SW / 2) + 8 * piece;
#pragma unroll
        for (int p = 0; p < PER; ++p) {
          const int rr = m_wave + WT * (p * RPP + r0) + gi;
          if (rr < g.m && col < g.n) stg8_stream(g.c + (int64_t)rr * g.ldc + col, held[p]);
        }
      };
#pragma unroll
      for (int gi = 0; gi < WT; ++gi) {
        const int row = m_wave + WT * j + gi;
        f32x16 val[WN];
#pragma unroll
        for (int ni = 0; ni < WN; ++ni) {
          if constexpr (PINNED) asm volatile("" : "+a"(acc[gi][ni]));
          val[ni] = acc[gi][ni];
          if constexpr (PINNED) asm volatile("" : "+v"(val[ni]));
        }
        if constexpr (OUT == kPartial) {
          float* const p = g.partial + ((int64_t)it.split * g.m + row) * g.n;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int col = n_wave + WN * (8 * q + 4 * hi);
#pragma unroll
            for (int v = 0; v < WN; ++v) {
              f32x4 o;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int c = 4 * v + e;
                o[e] = val[c % WN][4 * q + c / WN];
              }
              if (row < g.m && col + 4 * v < g.n) *reinterpret_cast<f32x4*>(p + col + 4 * v) = o;
            }
          }
        } else {
          // rows of the block through LDS (64 or 128 bytes of each at a time), then whole pieces of rows to memory.  A wave's LDS
          // instructions run in order, so nothing waits between a pass's writes and reads, nor before the next pass's writes; a
          // pass is stored when the next has been written and asked for.
#pragma unroll
          for (int h = 0; h < PASSES; ++h) {
#pragma unroll
            for (int ql = 0; ql < QP; ++ql) {
              const int q = h * QP + ql;
              const int col = n_wave + WN * (8 * q + 4 * hi);
              float v[4 * WN];
#pragma unroll
              for (int c = 0; c < 4 * WN; ++c) v[c] = val[c % WN][4 * q + c / WN];
              if constexpr (OUT == kAccumulate) {
#pragma unroll
                for (int c4 = 0; c4 < WN; ++c4) {
                  const bool in = row < g.m && col + 4 * c4 < g.n;
                  const bf16x4 old = in ? *reinterpret_cast<const bf16x4*>(g.c + (int64_t)row * g.ldc + col + 4 * c4) : bf16x4{};
#pragma unroll
                  for (int e = 0; e < 4; ++e) v[4 * c4 + e] += (float)old[e];
                }
              }
              if constexpr (WN == 1) {
                const bf16x4 o = {(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
                *(KR_LDS bf16x4*)(stage + j * SW + ((q ^ ((j >> 2) & 3)) << 4) + 8 * hi) = o;
              } else {
#pragma unroll
                for (int w = 0; w < WN / 2; ++w) {
                  bf16x8 o;
#pragma unroll
                  for (int e = 0; e < 8; ++e) o[e] = (bf16)v[8 * w + e];
                  const int piece = WN / 2 * (2 * ql + hi) + w;
                  *(KR_LDS bf16x8*)(stage + j * SW + ((piece ^ (SW == 128 ? (j >> 1) & 7 : (j >> 2) & 3)) << 4)) = o;
                }
              }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
            bf16x8 read[PER];
#pragma unroll
            for (int p = 0; p < PER; ++p) {
              const int jj = p * RPP + r0;
              read[p] = *(KR_LDS const bf16x8*)(stage + jj * SW + ((piece ^ (SW == 128 ? (jj >> 1) & 7 : (jj >> 2) & 3)) << 4));
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
            if (gi * PASSES + h > 0) store_pass(gi * PASSES + h - 1);
#pragma unroll
            for (int p = 0; p < PER; ++p) held[p] = read[p];
            __builtin_amdgcn_sched_barrier(0);
          }
          if (gi == WT - 1) store_pass(WT * PASSES - 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      clear();
    }
    item += gridDim.x;
    if (item >= total) break;
    it = select(item);
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);   // the loads requested again: LDS is given up only when they have landed
#endif
}

// Few rows (up to 16 MT of A): bound by the bytes of B, which stream from memory into registers.  A workgroup owns 16 rows of B; its
// eight waves take every eighth K-step each, FEW_AHEAD of them requested at a time, and their sums meet in LDS in wave order.
constexpr int FEW_WAVES = 8, FEW_AHEAD = 4;
template <int MT, bool ACCUMULATE>
__global__ __launch_bounds__(64 * FEW_WAVES) void block_gemm_few_rows_kernel(Args g) {
  __shared__ float sums[FEW_WAVES][MT * 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * 16, r16 = lane & 15, k32 = (lane >> 4) * 32;
  const int nrow = n0 + r16 < g.n ? n0 + r16 : g.n - 1;
  const uint8_t* const b = g.b + (int64_t)nrow * g.ldb + k32;
  const uint8_t* a[MT];
  int mrow[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    mrow[i] = 16 * i + r16 < g.m ? 16 * i + r16 : g.m - 1;
    a[i] = g.a + (int64_t)mrow[i] * g.lda + k32;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto load = [](const uint8_t* p) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(p), hi = *reinterpret_cast<const i32x4*>(p + 16);
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto steps = [&](int t0, auto count) {
    constexpr int U = decltype(count)::value;
    i32x8 fb[U], fa[U][MT];
    int sb[U], sa[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + u * FEW_WAVES;
      fb[u] = load(b + t * BK);
      sb[u] = g.sb[t * g.lsb + nrow];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        fa[u][i] = load(a[i] + t * BK);
        sa[u][i] = g.sa[t * g.lsa + mrow[i]];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[u], fa[u][i], acc[i], 0, 0, 0, sb[u], 0, sa[u][i]);
  };
  int t = wave;
  for (; t + (FEW_AHEAD - 1) * FEW_WAVES < g.ksteps; t += FEW_AHEAD * FEW_WAVES) steps(t, Int<FEW_AHEAD>{});
  for (; t < g.ksteps; t += FEW_WAVES) steps(t, Int<1>{});
  // lane l: row l % 16 of A's tile, columns 4 (l / 16) .. + 3
#pragma unroll
  for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4*>(&sums[wave][i * 256 + r16 * 16 + (lane >> 4) * 4]) = acc[i];
  kr_barrier();
  for (int i = threadIdx.x; i < MT * 64; i += 64 * FEW_WAVES) {   // four columns each
    const int row = i / 4, col = n0 + (i & 3) * 4;
    if (row >= g.m || col >= g.n) continue;
    f32x4 v = *reinterpret_cast<const f32x4*>(&sums[0][i * 4]);
#pragma unroll
    for (int w = 1; w < FEW_WAVES; ++w) {
      const f32x4 o = *reinterpret_cast<const f32x4*>(&sums[w][i * 4]);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += o[e];
    }
    bf16* const c = g.c + (int64_t)row * g.ldc + col;
    if constexpr (ACCUMULATE) {
      const bf16x4 old = *reinterpret_cast<const bf16x4*>(c);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += (float)old[e];
    }
    *reinterpret_cast<bf16x4*>(c) = bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
  }
}

// C = bf16(sum of the cuts' fp32 partial products, in order [+ C]).  (The whole product, us, a cut's loads at a time and four cuts':
// 75 x 608 x 17951 in twelve 13.2, 11.0; 91 x 272 x 3875 in sixteen 10.2, 7.0; 1536 x 2048 x 32768 in four 100, 100.)
// STRIDED: for a caller that has named the units, a workgroup each; otherwise one piece a thread (75 x 608 x 17951 11.4 us, 11.8 with
// the loop).
template <bool STRIDED>
__global__ __launch_bounds__(256) void block_gemm_reduce_kernel(const float* __restrict__ partial, bf16* __restrict__ C,
                                                                int64_t ldc, int M, int N, int splits, int accumulate) {
  const int nv = N / 8;
  for (int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; idx < (int64_t)M * nv; idx += (int64_t)gridDim.x * 256) {
    const int m = (int)(idx / nv), n = (int)(idx % nv) * 8;
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    const float* src = partial + (int64_t)m * N + n;
    const int64_t step = (int64_t)M * N;
    auto add = [&](auto count) {   // cuts whose loads are all asked for before the first is used
      constexpr int U = decltype(count)::value;
      f32x4 a[U], b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a[u] = *reinterpret_cast<const f32x4*>(src);
        b[u] = *reinterpret_cast<const f32x4*>(src + 4);
        src += step;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[e] += a[u][e];
          acc[4 + e] += b[u][e];
        }
    };
    int left = splits;
    for (; left >= 4; left -= 4) add(Int<4>{});
    for (; left > 0; --left) add(Int<1>{});
    bf16* dst = C + (int64_t)m * ldc + n;
    if (accumulate) {
      const bf16x8 old = ldg8(dst);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += (float)old[e];
    }
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (bf16)acc[e];
    stg8(dst, o);
    if constexpr (!STRIDED) return;
  }
}

// The tiles, and what a launch of them takes in us as measured (256 compute units): per round of workgroups, and per K-step, for each
// round and for each tile of a unit's share, but no less than `step_min` (a unit with one tile waits for its loads).
// us, model and measured: 16384 x 7168 x 4096, 256 x 256 346, 349; 192 x 256 409, 408; 256 x 128 409, 412; 128 x 128 499, 489; 64 x
// 64 824, 790.  6023 x 4096 x 3584: 90, 83; 74, 75; 81, 81; 97, 92; 167, 151.  1536 x 4096 x 6023: 74, 57; 60, 46; 43, 41; 57, 46; 55,
// 68.  512 x 4096 x 4096: 52, 40; 43, 32; 31, 25; 25, 24; 18, 18.  1024 x 1024 x 1024: 18, 15; 17, 13; 13, 10; 9, 8; 6, 5.
struct Tile {
  int wt, wn;       // MFMA tiles per wave: 64 wt x 64 wn of C per workgroup
  int per_cu;       // workgroups that a compute unit holds
  float round, step_round, step_tile, step_min;
};
constexpr Tile kTiles[] = {{4, 4, 1, 5.4f, 0.f, 1.38f, 1.38f}, {3, 4, 1, 5.3f, 0.f, 1.1f, 1.1f},   {4, 2, 1, 3.5f, 0.f, 0.8f, 0.8f},
                           {2, 4, 1, 3.5f, 0.f, 0.79f, 0.79f}, {2, 2, 2, 1.5f, 0.1f, 0.5f, 0.66f}, {1, 1, 3, 0.5f, 0.1f, 0.19f, 0.38f}};
constexpr int kNumTiles = 6, kFewRows = kNumTiles;   // behind the tiles: block_gemm_few_rows_kernel
constexpr int kFewRowsMost = 64, kMostSplits = 16;
constexpr float kLaunch = 2.f, kCutLaunch = 3.6f;

struct Plan {
  int tile, splits, steps_per;
};

size_t partial_bytes(int splits, int M, int N) { return splits > 1 ? (size_t)splits * M * N * sizeof(float) : 0; }

// The plan of the least time by the figures above, with at most `most_bytes` of workspace.
//   * A contraction is cut (partial tiles written and read again at 5 TB/s, and a second launch) only while all pieces fit into one
//     round: 1536 x 2048 x 32768 whole 159 us, in four pieces 100; 64 x 4096 x 4096 12 and 10; 1024 x 1024 x 1024 5 and 11.
//   * Few rows: a workgroup reads 16 rows of B and all of A, 33.6 GB/s per unit (us, 16 x 4096 x 4096 5.9 where tiles take 8.3, 64 x 4096
//     x 4096 11.8 and 10.0, 1 x 28672 x 4096 24.9 and 18.7).
// limited: the caller has named the units; a workgroup of each launch for each, and no kernel that takes more.
// segments: the contraction lies in pieces, which the kernel for few rows does not know.
Plan choose_plan(int M, int N, int K, int cus, bool limited, size_t most_bytes, bool segments = false) {
  const int ksteps = (K + BK - 1) / BK;
  Plan best{0, 1, ksteps};
  float least = INFINITY;
  if (M <= kFewRowsMost && !limited && !segments) {
    const float groups = std::max(1.f, (float)((N + 15) / 16) / cus), rows = 16.f + (M == 1 ? 1.f : 16.f * ((M + 15) / 16));
    least = 1.5f + std::max(groups * K * rows / 33.6e3f, (float)N * K / 5.5e6f);
    best.tile = kFewRows;
  }
  for (int t = 0; t < kNumTiles; ++t) {
    const Tile& tile = kTiles[t];
    const int per_cu = limited ? 1 : tile.per_cu;
    const int64_t tiles = (int64_t)((M + 64 * tile.wt - 1) / (64 * tile.wt)) * ((N + 64 * tile.wn - 1) / (64 * tile.wn));
    int last = 0;
    for (int want = 1; want <= kMostSplits && want <= ksteps; ++want) {
      const int per = (ksteps + want - 1) / want, splits = (ksteps + per - 1) / per;
      if (splits == last) continue;
      last = splits;
      if (splits > 1 && kLaunch + kCutLaunch + tile.round >= least) break;   // (whatever it is cut into)
      if (splits > 1 && (tiles * splits > (int64_t)cus * per_cu || partial_bytes(splits, M, N) > most_bytes)) break;
      const int64_t of_unit = splits > 1 ? ((int)tiles * splits + cus - 1) / cus : (tiles + cus - 1) / cus;
      const float share = (float)of_unit, rounds = (float)((of_unit + per_cu - 1) / per_cu);
      float us = kLaunch + rounds * tile.round + per * std::max(tile.step_min, rounds * tile.step_round + share * tile.step_tile);
      if (splits > 1) us += kCutLaunch + (2.f * splits + 0.5f) * M * N * 4.f / 5e6f;
      if (us < least) {
        least = us;
        best = Plan{t, splits, per};
      }
    }
  }
  return best;
}
constexpr size_t kMostWorkspace = (size_t)1 << 30;

int device_cus() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return 256;
  return n;
}

template <int T, int OUT, class Contraction>
int launch(const Args& g, const Contraction& pieces, int cus, bool limited, hipStream_t stream) {
  constexpr Tile t = kTiles[T];
  constexpr size_t lds = lds_bytes(t.wt, t.wn);
  static_assert(lds * t.per_cu <= 160 * 1024, "LDS of a compute unit");
  static const hipError_t raised = hipFuncSetAttribute((const void*)block_gemm_kernel<t.wt, t.wn, OUT, Contraction>,
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (raised != hipSuccess) return KR_ELAUNCH;
  const int64_t tiles = (int64_t)((g.m + 64 * t.wt - 1) / (64 * t.wt)) * ((g.n + 64 * t.wn - 1) / (64 * t.wn)) * g.splits;
  if (tiles > 0x3fffffff) return KR_EUNSUPPORTED;
  const int64_t grid = std::min<int64_t>(tiles, (int64_t)cus * (limited ? 1 : t.per_cu));
  hipLaunchKernelGGL((block_gemm_kernel<t.wt, t.wn, OUT, Contraction>), dim3((unsigned)grid), dim3(NTHREADS), lds, stream, g, pieces);
  return kr_launch_status();
}

template <int MT>
int launch_few(const Args& g, int accumulate, hipStream_t stream) {
  const dim3 grid((unsigned)((g.n + 15) / 16)), block(64 * FEW_WAVES);
  if (accumulate) hipLaunchKernelGGL((block_gemm_few_rows_kernel<MT, true>), grid, block, 0, stream, g);
  else hipLaunchKernelGGL((block_gemm_few_rows_kernel<MT, false>), grid, block, 0, stream, g);
  return kr_launch_status();
}
int launch_few_rows(const Args& g, int accumulate, hipStream_t stream) {
  if (g.m <= 16) return launch_few<1>(g, accumulate, stream);
  if (g.m <= 32) return launch_few<2>(g, accumulate, stream);
  return launch_few<4>(g, accumulate, stream);
}

template <int OUT, class Contraction>
int launch_tile(const Plan& p, const Args& g, const Contraction& pieces, int cus, bool limited, hipStream_t stream) {
  switch (p.tile) {
    case 0: return launch<0, OUT>(g, pieces, cus, limited, stream);
    case 1: return launch<1, OUT>(g, pieces, cus, limited, stream);
    case 2: return launch<2, OUT>(g, pieces, cus, limited, stream);
    case 3: return launch<3, OUT>(g, pieces, cus, limited, stream);
    case 4: return launch<4, OUT>(g, pieces, cus, limited, stream);
    case 5: return launch<5, OUT>(g, pieces, cus, limited, stream);
  }
  return KR_EUNSUPPORTED;
}

int launch_reduce(const Plan& p, const Args& g, int accumulate, int cus, bool limited, hipStream_t stream) {
  const int64_t groups = ((int64_t)g.m * (g.n / 8) + 255) / 256;
  const int64_t grid = std::min<int64_t>(groups, limited ? cus : 0x7fffffff);
  hipLaunchKernelGGL((grid < groups ? block_gemm_reduce_kernel<true> : block_gemm_reduce_kernel<false>), dim3((unsigned)grid), dim3(256), 0,
                     stream, g.partial, g.c, g.ldc, g.m, g.n, p.splits, accumulate);
  return kr_launch_status();
}

}  // namespace

extern "C" size_t kr_block_gemm_workspace_bytes(int M, int N, int K, int max_cus) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const int all = device_cus();
  const bool limited = max_cus > 0 && max_cus < all;
  return partial_bytes(choose_plan(M, N, K, limited ? max_cus : all, limited, kMostWorkspace).splits, M, N);
}

extern "C" int kr_block_gemm(int M, int N, int K, const void* A, int64_t lda, const void* sa, int64_t lsa, const void* B,
                             int64_t ldb, const void* sb, int64_t lsb, void* C, int64_t ldc, int accumulate, int max_cus,
                             void* workspace, size_t workspace_bytes, void* stream) {
  if (!A || !sa || !B || !sb || !C || M <= 0 || N <= 0 || K <= 0) return KR_EINVAL;
  if (N % 8 || ldc % 8 || lda % 16 || ldb % 16 || lsa % 4 || lsb % 4) return KR_EUNSUPPORTED;
  const int64_t kp = ((int64_t)K + BK - 1) / BK * BK;
  if (lda < kp || ldb < kp || lsa < M || lsb < N || ldc < N) return KR_EINVAL;
  if (!kr_aligned16(A) || !kr_aligned16(B) || !kr_aligned16(C) || !kr_aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(sa) & 3) || (reinterpret_cast<uintptr_t>(sb) & 3))
    return KR_EINVAL;
  // a tile's rows are addressed with 32-bit offsets from its first
  if (lda > (1 << 23) || ldb > (1 << 23) || lsa > 0x7fffffff || lsb > 0x7fffffff || M > 0x7fffff00 || N > 0x7fffff00)
    return KR_EUNSUPPORTED;
  const int all = device_cus();
  const bool limited = max_cus > 0 && max_cus < all;
  const int cus = limited ? max_cus : all;
  const Plan p = choose_plan(M, N, K, cus, limited, workspace ? std::min(workspace_bytes, kMostWorkspace) : 0);
  Args g{(const uint8_t*)A, (const uint8_t*)sa, (const uint8_t*)B, (const uint8_t*)sb, (bf16*)C, (float*)workspace,
         lda, ldb, ldc, (int)lsa, (int)lsb, M, N, (K + BK - 1) / BK, p.steps_per, p.splits};
  if (p.tile == kFewRows) return launch_few_rows(g, accumulate, (hipStream_t)stream);
  const hipStream_t st = (hipStream_t)stream;
  if (p.splits > 1) {
    const int rc = launch_tile<kPartial>(p, g, OnePiece{}, cus, limited, st);
    return rc != KR_OK ? rc : launch_reduce(p, g, accumulate, cus, limited, st);
  }
  return accumulate ? launch_tile<kAccumulate>(p, g, OnePiece{}, cus, limited, st) : launch_tile<kStore>(p, g, OnePiece{}, cus, limited, st);
}

extern "C" size_t kr_block_gemm_segments_workspace_bytes(int M, int N, int blocks, int max_cus) {
  if (M <= 0 || N <= 0 || blocks <= 0 || blocks > 0x7fffffff / BK) return 0;
  const int all = device_cus();
  const bool limited = max_cus > 0 && max_cus < all;
  return partial_bytes(choose_plan(M, N, blocks * BK, limited ? max_cus : all, limited, kMostWorkspace, true).splits, M, N);
}

extern "C" int kr_block_gemm_segments(int M, int N, int nseg, const int* K, const void* const* A, const int64_t* lda, const void* const* sa,
                                      const int64_t* lsa, const void* const* B, const int64_t* ldb, const void* const* sb,
                                      const int64_t* lsb, void* C, int64_t ldc, int max_cus, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  if (!K || !A || !lda || !sa || !lsa || !B || !ldb || !sb || !lsb || !C || M <= 0 || N <= 0 || nseg <= 0) return KR_EINVAL;
  if (nseg > kMostSegments || N % 8 || ldc % 8 || M > 0x7fffff00 || N > 0x7fffff00) return KR_EUNSUPPORTED;
  if (ldc < N || !kr_aligned16(C) || !kr_aligned16(workspace)) return KR_EINVAL;
  Segments pieces{};
  int64_t blocks = 0;
  for (int i = 0; i < nseg; ++i) {
    if (!A[i] || !sa[i] || !B[i] || !sb[i] || K[i] <= 0) return KR_EINVAL;
    if (lda[i] % 16 || ldb[i] % 16 || lsa[i] % 4 || lsb[i] % 4) return KR_EUNSUPPORTED;
    const int64_t steps = ((int64_t)K[i] + BK - 1) / BK;
    if (lda[i] < steps * BK || ldb[i] < steps * BK || lsa[i] < M || lsb[i] < N) return KR_EINVAL;
    if (!kr_aligned16(A[i]) || !kr_aligned16(B[i]) || (reinterpret_cast<uintptr_t>(sa[i]) & 3) || (reinterpret_cast<uintptr_t>(sb[i]) & 3))
      return KR_EINVAL;
    if (lda[i] > (1 << 23) || ldb[i] > (1 << 23) || lsa[i] > 0x7fffffff || lsb[i] > 0x7fffffff) return KR_EUNSUPPORTED;
    pieces.a[i] = (const uint8_t*)A[i];
    pieces.sa[i] = (const uint8_t*)sa[i];
    pieces.b[i] = (const uint8_t*)B[i];
    pieces.sb[i] = (const uint8_t*)sb[i];
    pieces.lda[i] = (int)lda[i];
    pieces.ldb[i] = (int)ldb[i];
    pieces.lsa[i] = (int)lsa[i];
    pieces.lsb[i] = (int)lsb[i];
    pieces.ksteps[i] = (int)steps;
    blocks += steps;
  }
  if (blocks > 0x7fffffff / BK) return KR_EUNSUPPORTED;
  const int all = device_cus();
  const bool limited = max_cus > 0 && max_cus < all;
  const int cus = limited ? max_cus : all;
  const Plan p = choose_plan(M, N, (int)blocks * BK, cus, limited, workspace ? std::min(workspace_bytes, kMostWorkspace) : 0, true);
  const Args g{nullptr, nullptr, nullptr, nullptr, (bf16*)C, (float*)workspace, 0, 0, ldc, 0, 0, M, N, (int)blocks, p.steps_per, p.splits};
  const hipStream_t st = (hipStream_t)stream;
  if (p.splits > 1) {
    const int rc = launch_tile<kPartial>(p, g, pieces, cus, limited, st);
    return rc != KR_OK ? rc : launch_reduce(p, g, 0, cus, limited, st);
  }
  return launch_tile<kStore>(p, g, pieces, cus, limited, st);
}
