// bf16 matrix -> 8-bit blocks (the operands of kr_block_gemm.hip): e4m3 values and one power-of-two scale per block of 128.
//
//   e = smallest whole number with amax 2^-e <= 448 (of the block's finite values; -127 for a block of zeros), -127 <= e <= 127
//   q = x 2^-e rounded to e4m3 (nearest even), scale byte = e + 127
//
// By row a block is 128 consecutive columns of a row; by column it is 128 consecutive rows of a column and the result is transposed,
// so that either way a row of the result is contiguous along the contraction it is made for.  With one scale per 128 x 128 tile
// (weights) both orientations hold the same values.
#include "kr_common.h"

namespace {

constexpr int kThreads = 256;

struct QArgs {
  const bf16* x;
  int64_t ld, run_ld;
  int run_sh;               // rows come in runs of 2^run_sh rows (stride ld) whose starts are run_ld apart; 0: one stride
  int rows, cols;
  uint8_t* q;               // [rows, ldq], by row (null: not wanted)
  uint8_t* s;               // [ceil(cols / 128), lds]
  uint8_t* qt;              // [cols, ldqt], by column
  uint8_t* st;              // [ceil(rows / 128), ldst]
  int64_t ldq, ldqt;
  int64_t lds, ldst;
};

// exponent of a block from the bf16 bits (without sign) of its largest finite magnitude
__device__ __forceinline__ int block_exponent(unsigned amax) {
  // amax = 1.m 2^p (or less, where subnormal: the bound holds all the same); 448 = 1.75 2^8
  const int p = (int)(amax >> 7) - 127;
  const int e = p - 8 + ((amax & 127u) > 0x60u ? 1 : 0);
  return amax == 0 || e < -127 ? -127 : e;   // (at most 127 - 7)
}
// 2^-e for -127 <= e <= 126
__device__ __forceinline__ float exp2_neg(int e) { return __uint_as_float((unsigned)(127 - e) << 23); }

__device__ __forceinline__ unsigned finite_bits(unsigned short b) {
  const unsigned a = b & 0x7fffu;
  return a < 0x7f80u ? a : 0u;
}
__device__ __forceinline__ float widen(unsigned short b) { return __uint_as_float((unsigned)b << 16); }
// two values as e4m3 in the low (HI: high) half of a word; what is not finite becomes NaN
template <bool HI>
__device__ __forceinline__ int pack2(float a, float b, int old) {
  a = __builtin_isfinite(a) ? a : __builtin_nanf("");
  b = __builtin_isfinite(b) ? b : __builtin_nanf("");
  return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, HI);
}

typedef __attribute__((__vector_size__(8 * sizeof(unsigned short)))) unsigned short u16x8;

// One workgroup per 128 x 128 tile.  Thread t holds rows 8 (t / 16) .. + 7, columns 8 (t % 16) .. + 7 of it.
template <bool ROWS, bool COLS, bool TILE>
__global__ __launch_bounds__(kThreads) void block_quantize_kernel(QArgs g) {
  __shared__ unsigned red[4][128];
  __shared__ __attribute__((aligned(16))) uint8_t turned[COLS ? 128 * 128 : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c8 = tid & 15, r8 = tid >> 4;
  const int cb = blockIdx.x, rb = blockIdx.y;
  const int col = cb * 128 + c8 * 8, row = rb * 128 + r8 * 8;
  u16x8 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = row + i;
    v[i] = u16x8{};
    if (r < g.rows && col < g.cols) {
      const int64_t off = (int64_t)(r >> g.run_sh) * g.run_ld + (int64_t)(r & ((1 << g.run_sh) - 1)) * g.ld;
      v[i] = *reinterpret_cast<const u16x8*>(g.x + off + col);
    }
  }
  unsigned ramax[8], camax[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) ramax[i] = camax[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned a = finite_bits(v[i][e]);
      ramax[i] = ramax[i] > a ? ramax[i] : a;
      camax[e] = camax[e] > a ? camax[e] : a;
    }
  if constexpr (TILE) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = m > ramax[i] ? m : ramax[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const unsigned other = __shfl_xor(m, o, 64);
      m = m > other ? m : other;
    }
    if (lane == 0) red[wave][0] = m;
    kr_barrier();
    m = red[0][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = m > red[w][0] ? m : red[w][0];
#pragma unroll
    for (int i = 0; i < 8; ++i) ramax[i] = camax[i] = m;
  } else {
    if constexpr (ROWS) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          const unsigned other = __shfl_xor(ramax[i], o, 64);
          ramax[i] = ramax[i] > other ? ramax[i] : other;
        }
    }
    if constexpr (COLS) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int o = 32; o > 8; o >>= 1) {
          const unsigned other = __shfl_xor(camax[e], o, 64);
          camax[e] = camax[e] > other ? camax[e] : other;
        }
      if (lane < 16)
#pragma unroll
        for (int e = 0; e < 8; ++e) red[wave][8 * c8 + e] = camax[e];
      kr_barrier();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        unsigned m = red[0][8 * c8 + e];
#pragma unroll
        for (int w = 1; w < 4; ++w) m = m > red[w][8 * c8 + e] ? m : red[w][8 * c8 + e];
        camax[e] = m;
      }
    }
  }
  if constexpr (ROWS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = block_exponent(ramax[i]);
      const float f = exp2_neg(e);
      int lo = 0, hi = 0;
      lo = pack2<false>(widen(v[i][0]) * f, widen(v[i][1]) * f, lo);
      lo = pack2<true>(widen(v[i][2]) * f, widen(v[i][3]) * f, lo);
      hi = pack2<false>(widen(v[i][4]) * f, widen(v[i][5]) * f, hi);
      hi = pack2<true>(widen(v[i][6]) * f, widen(v[i][7]) * f, hi);
      const int r = row + i;
      if (r < g.rows) {
        *reinterpret_cast<u32x2*>(g.q + (int64_t)r * g.ldq + col) = u32x2{(unsigned)lo, (unsigned)hi};
        if (c8 == 0) g.s[(int64_t)cb * g.lds + r] = (uint8_t)(e + 127);
      }
    }
  }
  if constexpr (COLS) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int ex = block_exponent(camax[e]);
      const float f = exp2_neg(ex);
      int lo = 0, hi = 0;
      lo = pack2<false>(widen(v[0][e]) * f, widen(v[1][e]) * f, lo);
      lo = pack2<true>(widen(v[2][e]) * f, widen(v[3][e]) * f, lo);
      hi = pack2<false>(widen(v[4][e]) * f, widen(v[5][e]) * f, hi);
      hi = pack2<true>(widen(v[6][e]) * f, widen(v[7][e]) * f, hi);
      const int c = 8 * c8 + e;
      *reinterpret_cast<u32x2*>(turned + c * 128 + (((r8 >> 1) ^ (c8 & 7)) << 4) + 8 * (r8 & 1)) = u32x2{(unsigned)lo, (unsigned)hi};
      if (r8 == 0 && cb * 128 + c < g.cols) g.st[(int64_t)rb * g.ldst + cb * 128 + c] = (uint8_t)(ex + 127);
    }
    kr_barrier();
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int c = 32 * p + (tid >> 3), chunk = tid & 7;
      if (cb * 128 + c < g.cols) {
        const u32x4 o = *reinterpret_cast<const u32x4*>(turned + c * 128 + ((chunk ^ ((c >> 3) & 7)) << 4));
        *reinterpret_cast<u32x4*>(g.qt + (int64_t)(cb * 128 + c) * g.ldqt + rb * 128 + chunk * 16) = o;
      }
    }
  }
}

}  // namespace

extern "C" int kr_block_quantize(const void* x, int rows, int cols, int64_t ld, int run_rows, int64_t run_ld, int tiles,
                                 void* q, int64_t ldq, void* s, int64_t lds, void* qt, int64_t ldqt, void* st, int64_t ldst,
                                 void* stream) {
  if (!x || rows <= 0 || cols <= 0 || (!q && !qt) || (q && !s) || (qt && !st)) return KR_EINVAL;
  if (run_rows <= 0 || (run_rows & (run_rows - 1))) return KR_EINVAL;
  if (cols % 8 || ld % 8 || (run_rows > 1 && run_ld % 8)) return KR_EUNSUPPORTED;
  if (ld < cols || (run_rows > 1 && (rows % run_rows || run_ld < run_rows * ld))) return KR_EINVAL;
  const int64_t cb = ((int64_t)cols + 127) / 128, rb = ((int64_t)rows + 127) / 128;
  if (q && (ldq % 16 || ldq < cb * 128 || lds < rows)) return KR_EINVAL;
  if (qt && (ldqt % 16 || ldqt < rb * 128 || ldst < cols)) return KR_EINVAL;
  if (!kr_aligned16(x) || !kr_aligned16(q) || !kr_aligned16(qt)) return KR_EINVAL;
  if (rb > 65535) return KR_EUNSUPPORTED;
  int sh = 0;
  while ((1 << sh) < run_rows) ++sh;
  const QArgs g{(const bf16*)x, ld, run_rows > 1 ? run_ld : ld, sh, rows, cols, (uint8_t*)q, (uint8_t*)s, (uint8_t*)qt,
                (uint8_t*)st, ldq, ldqt, lds, ldst};
  const dim3 grid((unsigned)cb, (unsigned)rb);
#define KR_Q(R, C, T) hipLaunchKernelGGL((block_quantize_kernel<R, C, T>), grid, dim3(kThreads), 0, (hipStream_t)stream, g)
  if (q && qt) { if (tiles) KR_Q(true, true, true); else KR_Q(true, true, false); }
  else if (q) { if (tiles) KR_Q(true, false, true); else KR_Q(true, false, false); }
  else { if (tiles) KR_Q(false, true, true); else KR_Q(false, true, false); }
#undef KR_Q
  return kr_launch_status();
}
