// Layer norm forward and backward:
//   mean = sum x / n,  rstd = 1 / sqrt(sum (x - mean)^2 / n + eps),  xh = (x - mean) rstd,  y = xh gamma + beta
//   g = dy gamma,  dx = rstd (g - mean(g) - xh mean(g xh)) (+ the residual branch's gradient),  dgamma = sum dy xh,  dbeta = sum dy
// HBM-bound: the forward reads x and writes y (+ 8 bytes of statistics a row), the backward reads dy, x and the residual gradient and
// writes dx.  A group of LPR lanes owns a row and keeps it in registers, so that every element is read once and the variance is
// taken from the differences to the mean (of sum x^2 - n mean^2 nothing is left where the mean is large): 8 to 32 lanes, several rows
// to a wave, for rows of 64 to 256 elements, a wave, or two, four or eight waves where a lane would hold too much.
// The weight's and the bias' gradients are column sums over all rows: a lane has the same columns of every row it comes by and sums
// them in registers, a workgroup adds its rows' through LDS in a fixed order and leaves one fp32 row of both, [2][cols], and a
// second launch adds the workgroups' rows.
// 32768 x 4096: forward 95 us (5.6 TB/s), backward 137 (5.9), with a residual 180 (6.0); right behind the forward, of whose rows the caches
// still hold some, 154 with its sums' launch.  (The times below are of operands that come from memory.)
#include "kr_common.h"

namespace {

constexpr int kMaxCols = 16384;
// Up to this many rows one launch does both (two launches -> one, us from Python: 257 x 512 13.9 -> 8.8, 1024 x 512 11.1 -> 8.6, 512 x 8192
// 25.3 -> 12.1, 1024 x 4096 20.5 -> 14.9; 2048 x 4096 26.0 -> 26.8, 4096 x 512 11.1 -> 32.9).
constexpr int kFewRows = KR_LAYERNORM_FEW_ROWS;

template <int LPR>
constexpr int kBlock = LPR > 256 ? LPR : 256;

// Sum over the LPR lanes of a row; every lane gets it.  Of waves that share a row one lane each leaves its part in `slots`
// [row of the workgroup][wave of the row], and all add them in one order.  (Every wave of the workgroup has to come by.)
template <int LPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*slots)[kBlock<LPR> / 64], int wave, int lane) {
#pragma unroll
  for (int off = (LPR < 64 ? LPR : 64) / 2; off > 0; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off, KR_WAVE);
  if constexpr (LPR > 64) {
    constexpr int WPR = LPR / 64;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slots[i][wave] = v[i];
    }
    kr_barrier();
    const int first = wave / WPR * WPR;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) v[i] += slots[i][first + w];
    }
  }
}

// KEEP: plain stores for small results, which the next launch finds in the caches (as the RMS norm's).
template <int LPR, int NCH, bool KEEP>
__global__ __launch_bounds__(kBlock<LPR>) void layernorm_fwd_kernel(
    const bf16* __restrict__ x, const bf16* __restrict__ gamma, const bf16* __restrict__ beta, bf16* __restrict__ y,
    float* __restrict__ mean, float* __restrict__ rstd, int rows, int cols, int64_t x_ld, KrRuns x_runs, float eps) {
  constexpr int kRows = kBlock<LPR> / LPR;
  __shared__ float slots[4][1][kBlock<LPR> / 64];  // [use][sum][wave]: sums two barriers apart have slots of their own
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int at = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const int nvec = cols / 8;
  const float inv_cols = 1.0f / (float)cols;
  bf16x8 g[NCH], b[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int v = at + c * LPR;
    g[c] = v < nvec ? ldg8(gamma + v * 8) : zero8();
    b[c] = v < nvec ? ldg8(beta + v * 8) : zero8();
  }
  int use = 0;
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < rows; base += (int64_t)gridDim.x * kRows) {
    const int64_t row = base + slot;
    const bool active = row < rows;
    const bf16* xr = x + kr_row_at(active ? row : 0, x_ld, x_runs);
    bf16x8 xv[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int v = at + c * LPR;
      xv[c] = active && v < nvec ? ldg8(xr + v * 8) : zero8();
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[0] += (float)xv[c][e];
    row_sums<LPR>(sum, slots[use], wave, lane);
    const float mu = sum[0] * inv_cols;
    sum[0] = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (at + c * LPR < nvec) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float d = (float)xv[c][e] - mu;
          sum[0] = __builtin_fmaf(d, d, sum[0]);
        }
      }
    }
    row_sums<LPR>(sum, slots[use + 1], wave, lane);
    use ^= 2;
    const float rs = rsqrtf(sum[0] * inv_cols + eps);
    if (!active) continue;
    if (at == 0) {
      mean[row] = mu;
      rstd[row] = rs;
    }
    bf16* yr = y + row * cols;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int v = at + c * LPR;
      if (v < nvec) {
        bf16x8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          o[e] = (bf16)__builtin_fmaf(((float)xv[c][e] - mu) * rs, (float)g[c][e], (float)b[c][e]);
        if constexpr (KEEP)
          stg8(yr + v * 8, o);
        else
          stg8_stream(yr + v * 8, o);
      }
    }
  }
}

// The gradients of weight and bias in 32 columns, by one workgroup: 64 lanes along the rows with 8 columns each, their sums added in a
// fixed order.
constexpr int kFewCols = 32;
__device__ __forceinline__ void column_sums(const bf16* dy, const bf16* x, const float* mean, const float* rstd, bf16* dgamma,
                                            bf16* dbeta, int rows, int cols, int64_t dy_ld, int64_t x_ld, KrRuns x_runs, int block) {
  __shared__ float red[2][64][kFewCols + 1];
  const int vec = threadIdx.x & 3, rl = threadIdx.x >> 2, col = block * kFewCols + vec * 8;
  float dg[8], db[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dg[e] = db[e] = 0.f;
  if (col < cols) {
#pragma unroll 4
    for (int row = rl; row < rows; row += 64) {
      const bf16x8 xv = ldg8(x + kr_row_at(row, x_ld, x_runs) + col), dv = ldg8(dy + row * dy_ld + col);
      const float mu = mean[row], rs = rstd[row];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dg[e] = __builtin_fmaf((float)dv[e], ((float)xv[e] - mu) * rs, dg[e]);
        db[e] += (float)dv[e];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    red[0][rl][vec * 8 + e] = dg[e];
    red[1][rl][vec * 8 + e] = db[e];
  }
  kr_barrier();
  if (threadIdx.x < 2 * kFewCols) {
    const int which = threadIdx.x / kFewCols, c = threadIdx.x % kFewCols;
    if (block * kFewCols + c < cols) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 64; ++r) sum[r & 3] += red[which][r][c];
      (which ? dbeta : dgamma)[block * kFewCols + c] = (bf16)((sum[0] + sum[1]) + (sum[2] + sum[3]));
    }
  }
}

// Where a row's loads are asked for while the row before is worked on: eight waves to a row, which have no other workgroup beside them, and
// a wave to a row (without -> with a residual, us, at once -> ahead: 12000 x 8200 140 -> 111, 166 -> 146, 8192 x 12288 124 -> 108, 154 -> 141,
// 65536 x 512 49.5 -> 42, 55 -> 49, 50000 x 768 50 -> 44, 56 -> 58, 32768 x 1024 39.6 -> 39.8, 49.4 -> 48.7; two waves: 32768 x 4096 136 -> 142,
// 180 -> 175, 2560 89 -> 89, 115 -> 122, four: 11577 x 6552 97 -> 99, 117 -> 130; four vectors to a lane leave no registers, 7395 x 15696
// 145 -> 174, 182 -> 285).
template <int LPR, int NCH>
constexpr bool kAhead = (LPR == 64 && NCH <= 2) || (LPR == 512 && NCH <= 3);

// ADD: the gradient of the residual branch forked off in front of the norm is added before the one rounding.  dx may be dres (neither is
// __restrict__): a lane reads its piece before it writes there, and the row asked for ahead is another one.
// FEW: the workgroups from `row_blocks` on have the columns, and no partial rows are left.
template <int LPR, int NCH, bool ADD, bool FEW>
__global__ __launch_bounds__(kBlock<LPR>) void layernorm_bwd_kernel(
    const bf16* __restrict__ dy, const bf16* __restrict__ x, const float* __restrict__ mean, const float* __restrict__ rstd,
    const bf16* __restrict__ gamma, const bf16* dres, bf16* dx, float* __restrict__ partial, int rows,
    int cols, int64_t dy_ld, int64_t x_ld, int64_t dres_ld, int64_t dx_ld, KrRuns x_runs, KrRuns dres_runs, KrRuns dx_runs,
    int row_blocks, bf16* __restrict__ dgamma, bf16* __restrict__ dbeta) {
  if constexpr (FEW) {
    if ((int)blockIdx.x >= row_blocks) {
      column_sums(dy, x, mean, rstd, dgamma, dbeta, rows, cols, dy_ld, x_ld, x_runs, blockIdx.x - row_blocks);
      return;
    }
  }
  constexpr int kRows = kBlock<LPR> / LPR;
  __shared__ float slots[2][2][kBlock<LPR> / 64];
  __shared__ float red[kRows > 1 && !FEW ? kBlock<LPR> * 8 : 1];  // a chunk's column sums of every lane
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int at = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const int nvec = cols / 8;
  const float inv_cols = 1.0f / (float)cols;
  bf16x8 g[NCH];
  float dg[NCH][8], db[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int v = at + c * LPR;
    g[c] = v < nvec ? ldg8(gamma + v * 8) : zero8();
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[c][e] = db[c][e] = 0.f;
  }
  constexpr bool AHEAD = kAhead<LPR, NCH>;
  bf16x8 xn[NCH], dn[NCH], rn[ADD ? NCH : 1];
  float mu_n = 0.f, rs_n = 0.f;
  auto load = [&](int64_t row) {
    const bool active = row < rows;
    const int64_t r = active ? row : 0;
    const bf16* xr = x + kr_row_at(r, x_ld, x_runs);
    const bf16* dr = dy + r * dy_ld;
    const bf16* rr = ADD ? dres + kr_row_at(r, dres_ld, dres_runs) : nullptr;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int v = at + c * LPR;
      const bool in = active && v < nvec;
      xn[c] = in ? ldg8_stream(xr + v * 8) : zero8();
      dn[c] = in ? ldg8_stream(dr + v * 8) : zero8();
      if (ADD) rn[c] = in ? ldg8_stream(rr + v * 8) : zero8();
    }
    mu_n = active ? mean[r] : 0.f;
    rs_n = active ? rstd[r] : 0.f;
  };
  int use = 0;
  const int64_t step = (int64_t)(FEW ? row_blocks : gridDim.x) * kRows;
  if (AHEAD) load((int64_t)blockIdx.x * kRows + slot);
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < rows; base += step) {
    const int64_t row = base + slot;
    const bool active = row < rows;
    const int64_t r = active ? row : 0;
    if (!AHEAD) load(row);
    bf16x8 xv[NCH], dv[NCH], rv[ADD ? NCH : 1];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      xv[c] = xn[c];
      dv[c] = dn[c];
      if (ADD) rv[c] = rn[c];
    }
    const float mu = mu_n, rs = rs_n;
    if (AHEAD && base + step < rows) load(row + step);
    float sum[2] = {0.f, 0.f};  // of g and of g xh
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = ((float)xv[c][e] - mu) * rs, d = (float)dv[c][e], gv = d * (float)g[c][e];
        sum[0] += gv;
        sum[1] = __builtin_fmaf(gv, xh, sum[1]);
        if (!FEW) {
          dg[c][e] = __builtin_fmaf(d, xh, dg[c][e]);
          db[c][e] += d;
        }
      }
    row_sums<LPR>(sum, slots[use], wave, lane);
    use ^= 1;
    if (!active) continue;
    const float c1 = sum[0] * inv_cols, c2 = sum[1] * inv_cols;
    bf16* oxr = dx + kr_row_at(r, dx_ld, dx_runs);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int v = at + c * LPR;
      if (v < nvec) {
        bf16x8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float xh = ((float)xv[c][e] - mu) * rs;
          float d = rs * ((float)dv[c][e] * (float)g[c][e] - c1 - xh * c2);
          if (ADD) d += (float)rv[c][e];
          o[e] = (bf16)d;
        }
        stg8_stream(oxr + v * 8, o);
      }
    }
  }
  if constexpr (FEW) return;
  float* const mine = partial + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float total[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) total[e] = which ? db[c][e] : dg[c][e];
      if constexpr (kRows > 1) {
        kr_barrier();
#pragma unroll
        for (int e = 0; e < 8; ++e) red[e * kBlock<LPR> + threadIdx.x] = total[e];
        kr_barrier();
        if (slot == 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            total[e] = 0.f;
#pragma unroll
            for (int w = 0; w < kRows; ++w) total[e] += red[e * kBlock<LPR> + w * LPR + at];
          }
        }
      }
      const int v = at + c * LPR;
      if (slot == 0 && v < nvec) {
        f32x4* p = reinterpret_cast<f32x4*>(mine + which * cols + v * 8);
        p[0] = f32x4{total[0], total[1], total[2], total[3]};
        p[1] = f32x4{total[4], total[5], total[6], total[7]};
      }
    }
}

// dgamma[c], dbeta[c] = sums over the partial rows, [nparts][2 cols].  A workgroup has 32 columns and 32 lanes along the rows, each
// with four sums so that loads are in flight; the lanes' are added in a fixed order.
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void layernorm_dparams_kernel(const float* __restrict__ partial, bf16* __restrict__ dgamma,
                                                                        bf16* __restrict__ dbeta, int nparts, int cols) {
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c;
  const int64_t ld = 2 * (int64_t)cols;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (col < 2 * cols) {
    const float* src = partial + col;
    int p = rl;
    for (; p + 96 < nparts; p += 128) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] += src[(p + 32 * i) * ld];
    }
    for (; p < nparts; p += 32) a[0] += src[p * ld];
  }
  red[rl][c] = (a[0] + a[1]) + (a[2] + a[3]);
  kr_barrier();
  if (rl == 0 && col < 2 * cols) {
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) sum += red[r][c];
    if (col < cols)
      dgamma[col] = (bf16)sum;
    else
      dbeta[col - cols] = (bf16)sum;
  }
}

// Lanes that share a row: enough that a lane holds at most `most` vectors of 8.
int lanes_per_row(int cols, int most) {
  const int nvec = cols / 8;
  if (nvec <= 64) {
    int l = 8;
    while (l < nvec) l *= 2;
    return l;
  }
  int l = 64;
  while (l * most < nvec) l *= 2;
  return l;
}
// (8 -> 4 in the forward, us: 6023 x 3584 17.9 -> 15.3, 8192 x 8192 50.7 -> 48.4, 4096 x 16384 50.9 -> 49.5; 2: 16.8, 48.2, and 32768 x
// 4096, a wave a row or two, 95.5, 96.6, 108; backward 4 -> 2: 32768 x 4096 181 -> 183, without a residual 137 -> 144)
constexpr int kFwdVectors = 4, kBwdVectors = 4;
// In the backward rows of more than 5632 columns take eight waves, with loads ahead (four waves of 4 vectors -> those, without and with a
// residual, us: 11577 x 6552 94 -> 93, 117 -> 110, 12000 x 8192 109 -> 105, 140 -> 131, 16384 x 6144 109 -> 103, 144 -> 137, 5120 92 -> 92, 119
// -> 121), unless they are few and their columns are read in the same launch.
int bwd_lanes(int rows, int cols) { return cols > 5632 && rows > kFewRows ? 512 : lanes_per_row(cols, kBwdVectors); }

// Workgroups of the backward, each of which leaves 8 cols bytes that are read again: two a unit, what the registers of wide rows
// allow, one where it has eight waves (4096 x 16384 in 512 and 256, us: 121, 109; 32768 x 4096 181, 220), four where rows share a
// wave (100000 x 256 in 512 and 1024: 43.6, 40.4, without a residual 40.0, 32.6; 32768 x 1024 50.7, 53.5).
int bwd_blocks(int rows, int cols) {
  const int lpr = bwd_lanes(rows, cols), per = lpr > 256 ? 1 : 256 / lpr;
  const int most = lpr > 256 ? 256 : lpr < 64 ? 1024 : 512, blocks = (rows + per - 1) / per;
  return blocks < most ? blocks : most;
}

template <int LPR>
int launch_fwd(int nch, bool keep, int blocks, hipStream_t stream, const bf16* x, const bf16* gamma, const bf16* beta, bf16* y,
               float* mean, float* rstd, int rows, int cols, int64_t x_ld, KrRuns runs, float eps) {
#define KR_LN_FWD(NCH)                                                                                                            \
  hipLaunchKernelGGL((keep ? layernorm_fwd_kernel<LPR, NCH, true> : layernorm_fwd_kernel<LPR, NCH, false>), dim3(blocks),       \
                     dim3(kBlock<LPR>), 0, stream, x, gamma, beta, y, mean, rstd, rows, cols, x_ld, runs, eps)
  if constexpr (LPR < 64) {
    KR_LN_FWD(1);
  } else {
    switch (nch) {
      case 1: KR_LN_FWD(1); break;
      case 2: KR_LN_FWD(2); break;
      case 3: KR_LN_FWD(3); break;
      default: KR_LN_FWD(4);
    }
  }
#undef KR_LN_FWD
  return kr_launch_status();
}

struct BwdArgs {
  const bf16 *dy, *x;
  const float *mean, *rstd;
  const bf16 *gamma, *dres;
  bf16* dx;
  float* partial;
  int rows, cols;
  int64_t dy_ld, x_ld, dres_ld, dx_ld;
  KrRuns x_runs{0, 0}, dres_runs{0, 0}, dx_runs{0, 0};
  bf16 *dgamma = nullptr, *dbeta = nullptr;  // few rows: theirs in the same launch
};

template <int LPR>
int launch_bwd(int nch, int blocks, hipStream_t stream, const BwdArgs& a) {
#define KR_LN_BWD(NCH)                                                                                                            \
  hipLaunchKernelGGL((a.dgamma ? a.dres ? layernorm_bwd_kernel<LPR, NCH, true, kBlock<LPR> == 256>                               \
                                        : layernorm_bwd_kernel<LPR, NCH, false, kBlock<LPR> == 256>                              \
                      : a.dres ? layernorm_bwd_kernel<LPR, NCH, true, false>                                                     \
                               : layernorm_bwd_kernel<LPR, NCH, false, false>),                                                  \
                     dim3(blocks + (a.dgamma ? (a.cols + kFewCols - 1) / kFewCols : 0)), dim3(kBlock<LPR>), 0, stream, a.dy, a.x, \
                     a.mean, a.rstd, a.gamma, a.dres, a.dx, a.partial, a.rows, a.cols, a.dy_ld, a.x_ld, a.dres_ld, a.dx_ld,      \
                     a.x_runs, a.dres_runs, a.dx_runs, blocks, a.dgamma, a.dbeta)
  if constexpr (LPR < 64) {
    KR_LN_BWD(1);
  } else {
    switch (nch) {
      case 1: KR_LN_BWD(1); break;
      case 2: KR_LN_BWD(2); break;
      case 3: KR_LN_BWD(3); break;
      default: KR_LN_BWD(4);
    }
  }
#undef KR_LN_BWD
  return kr_launch_status();
}

}  // namespace

extern "C" int kr_layernorm_fwd(const void* x, const void* gamma, const void* beta, void* y, float* mean, float* rstd, int rows,
                                int cols, int64_t x_ld, int x_run_rows, int64_t x_run_ld, float eps, void* stream) {
  if (!x || !gamma || !beta || !y || !mean || !rstd || rows <= 0 || cols <= 0 || x_ld < cols) return KR_EINVAL;
  if (cols % 8 || x_ld % 8 || cols > kMaxCols) return KR_EUNSUPPORTED;
  if (!kr_aligned16(x) || !kr_aligned16(y) || !kr_aligned16(gamma) || !kr_aligned16(beta)) return KR_EINVAL;
  KrRuns runs;
  if (const int rc = kr_make_runs(x_run_rows, x_run_ld, rows, &runs)) return rc;
  const int lpr = lanes_per_row(cols, kFwdVectors), per = lpr > 256 ? 1 : 256 / lpr, nch = (cols / 8 + lpr - 1) / lpr;
  int blocks = (rows + per - 1) / per;
  if (blocks > 256 * 8) blocks = 256 * 8;
  const bool keep = (int64_t)rows * cols <= (int64_t)8 << 20;  // (as the RMS norm's results)
#define KR_LN_CALL(LPR)                                                                                                          \
  return launch_fwd<LPR>(nch, keep, blocks, (hipStream_t)stream, (const bf16*)x, (const bf16*)gamma, (const bf16*)beta, (bf16*)y, \
                         mean, rstd, rows, cols, x_ld, runs, eps)
  switch (lpr) {
    case 8: KR_LN_CALL(8);
    case 16: KR_LN_CALL(16);
    case 32: KR_LN_CALL(32);
    case 64: KR_LN_CALL(64);
    case 128: KR_LN_CALL(128);
    case 256: KR_LN_CALL(256);
    default: KR_LN_CALL(512);
  }
#undef KR_LN_CALL
}

extern "C" int kr_layernorm_bwd_partial_rows(int rows, int cols) {
  if (rows <= 0 || cols <= 0 || cols % 8 || cols > kMaxCols) return 0;
  return bwd_blocks(rows, cols);
}

extern "C" size_t kr_layernorm_bwd_workspace_bytes(int rows, int cols) {
  return (size_t)kr_layernorm_bwd_partial_rows(rows, cols) * 2 * (size_t)(cols > 0 ? cols : 0) * sizeof(float);
}

extern "C" int kr_layernorm_dparams(const float* partial, int nparts, int cols, void* dgamma, void* dbeta, void* stream) {
  if (!partial || !dgamma || !dbeta || nparts <= 0 || cols <= 0 || !kr_aligned16(partial)) return KR_EINVAL;
  if (cols > kMaxCols) return KR_EUNSUPPORTED;
  hipLaunchKernelGGL(layernorm_dparams_kernel, dim3((2 * cols + 31) / 32), dim3(kSumThreads), 0, (hipStream_t)stream, partial,
                     (bf16*)dgamma, (bf16*)dbeta, nparts, cols);
  return kr_launch_status();
}

extern "C" int kr_layernorm_bwd(const void* dy, const void* x, const float* mean, const float* rstd, const void* gamma,
                                const void* dres, void* dx, void* dgamma, void* dbeta, void* workspace, int rows, int cols,
                                int64_t dy_ld, int64_t x_ld, int x_run_rows, int64_t x_run_ld, int64_t dres_ld,
                                int dres_run_rows, int64_t dres_run_ld, int64_t dx_ld, int dx_run_rows, int64_t dx_run_ld,
                                void* stream) {
  const bool few = dgamma && rows <= kFewRows && cols <= KR_LAYERNORM_FEW_COLS;  // (workgroups of 256)
  if (!dy || !x || !mean || !rstd || !gamma || !dx || (!workspace && !few) || rows <= 0 || cols <= 0 || dy_ld < cols || x_ld < cols ||
      dx_ld < cols || (dres && dres_ld < cols) || !dgamma != !dbeta)
    return KR_EINVAL;
  if (cols % 8 || dy_ld % 8 || x_ld % 8 || dx_ld % 8 || (dres && dres_ld % 8) || cols > kMaxCols) return KR_EUNSUPPORTED;
  if (!kr_aligned16(x) || !kr_aligned16(dy) || !kr_aligned16(dx) || !kr_aligned16(gamma) || !kr_aligned16(workspace) ||
      (dres && !kr_aligned16(dres)))
    return KR_EINVAL;
  // (the gradients of the parameters are summed by other workgroups of the same launch, and a row's own may have left its place by then)
  if (dx == dy || dx == x) return KR_EINVAL;
  if (dx == dres && rows > 1 && (dx_ld != dres_ld || dx_run_rows != dres_run_rows || (dx_run_rows > 1 && dx_run_ld != dres_run_ld)))
    return KR_EINVAL;
  BwdArgs a{(const bf16*)dy, (const bf16*)x, mean, rstd, (const bf16*)gamma, (const bf16*)dres, (bf16*)dx, (float*)workspace,
            rows, cols, dy_ld, x_ld, dres ? dres_ld : 0, dx_ld};
  if (const int rc = kr_make_runs(x_run_rows, x_run_ld, rows, &a.x_runs)) return rc;
  if (dres)
    if (const int rc = kr_make_runs(dres_run_rows, dres_run_ld, rows, &a.dres_runs)) return rc;
  if (const int rc = kr_make_runs(dx_run_rows, dx_run_ld, rows, &a.dx_runs)) return rc;
  const int lpr = bwd_lanes(rows, cols), nch = (cols / 8 + lpr - 1) / lpr, blocks = bwd_blocks(rows, cols);
  const hipStream_t s = (hipStream_t)stream;
  if (few) a.dgamma = (bf16*)dgamma, a.dbeta = (bf16*)dbeta;
  int rc;
  switch (lpr) {
    case 8: rc = launch_bwd<8>(nch, blocks, s, a); break;
    case 16: rc = launch_bwd<16>(nch, blocks, s, a); break;
    case 32: rc = launch_bwd<32>(nch, blocks, s, a); break;
    case 64: rc = launch_bwd<64>(nch, blocks, s, a); break;
    case 128: rc = launch_bwd<128>(nch, blocks, s, a); break;
    case 256: rc = launch_bwd<256>(nch, blocks, s, a); break;
    default: rc = launch_bwd<512>(nch, blocks, s, a);
  }
  if (rc != KR_OK || !dgamma || few) return rc;  // without a destination the caller sums the partial rows later
  return kr_layernorm_dparams((const float*)workspace, blocks, cols, dgamma, dbeta, stream);
}
