// bf16 matrix -> 8-bit blocks (the operands of kr_block_gemm.hip): e4m3 values and one power-of-two scale per block of 128.
//
//   e = smallest whole number with amax 2^-e <= 448 (of the block's finite values; -127 for a block of zeros), -127 <= e <= 127
//   q = x 2^-e rounded to e4m3 (nearest even), scale byte = e + 127
//
// Bound by the bytes: 2 read per value and 1 written per orientation.  16384 x 4096 by row 31 us (6.4 TB/s), both ways 46 us (5.8 TB/s, a
// large copy runs at 5.1-5.4); 6023 x 3584 both ways 18 us.  Small matrices take a kernel's latency, about 4 us.
//
// By row a block is 128 consecutive columns of a row; by column it is 128 consecutive rows of a column and the result is transposed,
// so that either way a row of the result is contiguous along the contraction it is made for.  With one scale per 128 x 128 tile
// (weights) both orientations hold the same values.
#include "kr_common.h"

#include <type_traits>

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
__device__ __forceinline__ float exp2_bits(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }   // 2^e, -126 <= e <= 127

typedef __attribute__((__vector_size__(2 * sizeof(unsigned short)))) unsigned short u16x2;
typedef __attribute__((__vector_size__(2 * sizeof(short)))) short s16x2;

// larger halves of two words
__device__ __forceinline__ unsigned max2(unsigned a, unsigned b) {
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// the largest of 16 neighbouring lanes, in each of them: lanes exchanged in pairs, quads, half rows and rows inside the vector unit
__device__ __forceinline__ unsigned max_of_16(unsigned m) {
  m = max2(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));    // quad_perm 1 0 3 2
  m = max2(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));    // quad_perm 2 3 0 1
  m = max2(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));   // row_half_mirror
  return max2(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xf, 0xf, true));   // row_mirror
}
// magnitudes of a word's two values; FINITE: 0 in the place of infinities and NaN
template <bool FINITE>
__device__ __forceinline__ unsigned mags(unsigned w) {
  const unsigned a = w & 0x7fff7fffu;
  if (!FINITE) return a;
  return ((a & 0xffffu) < 0x7f80u ? a & 0xffffu : 0u) | (a >> 16 < 0x7f80u ? a & 0xffff0000u : 0u);
}

// Four values (two words) times 2^-e as e4m3.  The instruction divides by its scale's power of two before it rounds (nearest, ties to
// even; what is not finite becomes NaN; tests check every bf16 value at every scale).  TINY: the
// block's scale may be 2^-127, which is no normal fp32 number: multiplied in two steps.
template <bool TINY>
__device__ __forceinline__ unsigned pack4(unsigned lo, unsigned hi, int e, float scale) {
  s16x2 r = {0, 0};
  if (!TINY) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, lo), scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, hi), scale, true);
    return __builtin_bit_cast(unsigned, r);
  }
  float v[4] = {__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u), __uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u)};
  const int first = -e < 120 ? -e : 120;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = v[i] * exp2_bits(first) * exp2_bits(-e - first);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __builtin_isfinite(v[i]) ? v[i] : __builtin_nanf("");
  int o = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], o, true);
}
__device__ __forceinline__ float scale_of(int e) { return exp2_bits(e > -127 ? e : 0); }   // (-127: a block of zeros, or TINY)

// One workgroup per 128 x 128 tile.  Thread t holds rows 8 (t / 16) .. + 7, columns 8 (t % 16) .. + 7 of it.
template <bool ROWS, bool COLS, bool TILE>
__device__ __forceinline__ void quantize_tile(const QArgs& g) {
  // largest magnitudes of each wave's part of the columns (two columns a word), or of the tile; behind them, whether a wave has seen
  // what is not finite
  __shared__ unsigned red[4][64];
  __shared__ unsigned odd[4];
  __shared__ __attribute__((aligned(16))) uint8_t turned[COLS ? 128 * 128 : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c8 = tid & 15, r8 = tid >> 4;
  const int cb = blockIdx.x, rb = blockIdx.y;
  const int col = cb * 128 + c8 * 8, row = rb * 128 + r8 * 8;
  u32x4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = row + i;
    v[i] = u32x4{0, 0, 0, 0};
    if (r < g.rows && col < g.cols) {
      const int64_t off = (int64_t)(r >> g.run_sh) * g.run_ld + (int64_t)(r & ((1 << g.run_sh) - 1)) * g.ld;
      v[i] = *reinterpret_cast<const u32x4*>(g.x + off + col);
    }
  }
  unsigned ramax[8], camax[4];   // of a row; of columns 2 d and 2 d + 1
  auto largest = [&](auto finite) {
    constexpr bool FINITE = decltype(finite)::value;
#pragma unroll
    for (int d = 0; d < 4; ++d) camax[d] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ramax[i] = 0;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const unsigned a = mags<FINITE>(v[i][d]);
        if (ROWS || TILE) ramax[i] = max2(ramax[i], a);
        if (COLS && !TILE) camax[d] = max2(camax[d], a);
      }
    }
    if constexpr (TILE) {
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max2(m, ramax[i]);
      m = max_of_16(m);
#pragma unroll
      for (int o = 32; o > 8; o >>= 1) m = max2(m, __shfl_xor(m, o, 64));
      ramax[0] = m;
    } else {
      if constexpr (ROWS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) ramax[i] = max_of_16(ramax[i]);
      }
      if constexpr (COLS) {
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int o = 32; o > 8; o >>= 1) camax[d] = max2(camax[d], __shfl_xor(camax[d], o, 64));
      }
    }
  };
  auto halves = [](unsigned m) { return (m & 0xffffu) > m >> 16 ? m & 0xffffu : m >> 16; };
  auto not_finite = [&]() {      // in this thread's magnitudes: a half of 0x7f80 or more
    unsigned m = 0;
    if constexpr (TILE) m = ramax[0];
    else {
      if constexpr (ROWS)
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max2(m, ramax[i]);
      if constexpr (COLS)
#pragma unroll
        for (int d = 0; d < 4; ++d) m = max2(m, camax[d]);
    }
    return halves(m) >= 0x7f80u;
  };
  auto publish = [&]() {
    if constexpr (TILE) {
      if (lane == 0) red[wave][0] = ramax[0];
    } else {
      if (lane < 16)
#pragma unroll
        for (int d = 0; d < 4; ++d) red[wave][4 * c8 + d] = camax[d];
    }
  };
  largest(std::false_type{});
  const bool seen = __ballot(not_finite()) != 0;
  if constexpr (TILE || COLS) {
    publish();
    if (lane == 0) odd[wave] = seen;
    kr_barrier();
    if (odd[0] | odd[1] | odd[2] | odd[3]) {   // (uniform: once more, without them)
      largest(std::true_type{});
      kr_barrier();
      publish();
      kr_barrier();
    }
    if constexpr (TILE) {
      ramax[0] = max2(max2(red[0][0], red[1][0]), max2(red[2][0], red[3][0]));
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d)
        camax[d] = max2(max2(red[0][4 * c8 + d], red[1][4 * c8 + d]), max2(red[2][4 * c8 + d], red[3][4 * c8 + d]));
    }
  } else {
    if (seen) largest(std::true_type{});
  }

  auto store = [&](auto tiny) {
    constexpr bool TINY = decltype(tiny)::value;
    const int et = TILE ? block_exponent(halves(ramax[0])) : 0;
    if constexpr (ROWS) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = TILE ? et : block_exponent(halves(ramax[i]));
        const float f = scale_of(e);
        const int r = row + i;
        const u32x2 o = {pack4<TINY>(v[i][0], v[i][1], e, f), pack4<TINY>(v[i][2], v[i][3], e, f)};
        if (r < g.rows) {
          *reinterpret_cast<u32x2*>(g.q + (int64_t)r * g.ldq + col) = o;
          if (c8 == 0) g.s[(int64_t)cb * g.lds + r] = (uint8_t)(e + 127);
        }
      }
    }
    if constexpr (COLS) {
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e = TILE ? et : block_exponent(h ? camax[d] >> 16 : camax[d] & 0xffffu);
          const float f = scale_of(e);
          unsigned p[4];                       // the column's values, two rows a word
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_perm(v[2 * i + 1][d], v[2 * i][d], h ? 0x07060302u : 0x05040100u);
          const int c = 8 * c8 + 2 * d + h;
          *reinterpret_cast<u32x2*>(turned + c * 128 + (((r8 >> 1) ^ (c8 & 7)) << 4) + 8 * (r8 & 1)) =
              u32x2{pack4<TINY>(p[0], p[1], e, f), pack4<TINY>(p[2], p[3], e, f)};
          if (r8 == 0 && cb * 128 + c < g.cols) g.st[(int64_t)rb * g.ldst + cb * 128 + c] = (uint8_t)(e + 127);
        }
    }
  };
  bool tiny = false;                           // a block that is not zero below 448 * 2^-127
  auto is_tiny = [&](unsigned m) { return m != 0 && block_exponent(m) == -127; };
  if constexpr (TILE) tiny = is_tiny(halves(ramax[0]));
  else {
    if constexpr (ROWS)
#pragma unroll
      for (int i = 0; i < 8; ++i) tiny |= is_tiny(halves(ramax[i]));
    if constexpr (COLS)
#pragma unroll
      for (int d = 0; d < 4; ++d) tiny |= is_tiny(camax[d] & 0xffffu) || is_tiny(camax[d] >> 16);
  }
  if (__ballot(tiny) == 0) store(std::false_type{});
  else store(std::true_type{});
  if constexpr (COLS) {
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

template <bool ROWS, bool COLS, bool TILE>
__global__ __launch_bounds__(kThreads) void block_quantize_kernel(QArgs g) {
  quantize_tile<ROWS, COLS, TILE>(g);
}
// Few tiles: a workgroup of its own for each orientation (x is read twice, the second time from a cache).  us, one workgroup for both
// and two: 257 x 512 5.9, 4.5; 2048 x 1024 (128 tiles) 6.5, 5.1; 2048 x 2048 (256) 7.2, 6.1; 4096 x 2048 (512) 9.3, 8.8, with one scale per
// tile 7.6, 7.9; 4096 x 4096 (1024) 15.3, 16.0.
constexpr int kApartTiles = 256;
template <bool TILE>
__global__ __launch_bounds__(kThreads) void block_quantize_apart_kernel(QArgs g) {
  if (blockIdx.z == 0) quantize_tile<true, false, TILE>(g);
  else quantize_tile<false, true, TILE>(g);
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
  if (q && qt && cb * rb <= kApartTiles) {
    const dim3 twice((unsigned)cb, (unsigned)rb, 2);
    if (tiles) hipLaunchKernelGGL(block_quantize_apart_kernel<true>, twice, dim3(kThreads), 0, (hipStream_t)stream, g);
    else hipLaunchKernelGGL(block_quantize_apart_kernel<false>, twice, dim3(kThreads), 0, (hipStream_t)stream, g);
    return kr_launch_status();
  }
#define KR_Q(R, C, T) hipLaunchKernelGGL((block_quantize_kernel<R, C, T>), grid, dim3(kThreads), 0, (hipStream_t)stream, g)
  if (q && qt) { if (tiles) KR_Q(true, true, true); else KR_Q(true, true, false); }
  else if (q) { if (tiles) KR_Q(true, false, true); else KR_Q(true, false, false); }
  else { if (tiles) KR_Q(false, true, true); else KR_Q(false, true, false); }
#undef KR_Q
  return kr_launch_status();
}
