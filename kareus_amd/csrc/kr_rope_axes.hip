// Rotary position embedding by positions on several axes (time, height and width of images and video):
//   angle(token, f) = position[axis(f)][token] * inv_freq[f],  (a, b) -> (a cos - b sin, b cos + a sin),
// a and b being channels f and f + hd / 2 of a head.  HBM-bound: every rotated head is read and written once, and a token brings 8
// bytes per axis of positions where a table of angles would be hd * 4 bytes for each.
// A wave takes a token.  A lane has 8 frequencies and every 64 / (hd / 16)-th head: the angles of a token are formed by each of
// those lanes anew, which costs some 400 instructions a token against the 2000 and more cycles that its heads take from memory.
// Angles are taken in 64 bits, as turns, and only what is left of the whole turns is rounded to 32: in 32 bits a position of a
// million at frequency 1 would be off by a sixteenth of a radian.
#include "kr_common.h"

namespace {

constexpr int kThreads = 256;
constexpr double kTurnsPerRadian = 0.15915494309189533577;

struct RopeAxes {
  int n, interleaved;
  int sections[KR_ROPE_MAX_AXES];
};

__device__ __forceinline__ int axis_of(const RopeAxes& a, int f) {
  if (a.interleaved) {
    const int axis = f % a.n, turn = f / a.n;
    int left = 0;
#pragma unroll
    for (int i = 0; i < KR_ROPE_MAX_AXES; ++i) left = i == axis ? a.sections[i] : left;
    return turn < left ? axis : 0;
  }
  int axis = 0, end = 0;
#pragma unroll
  for (int i = 0; i + 1 < KR_ROPE_MAX_AXES; ++i) {
    end += a.sections[i];
    axis += f >= end && i + 1 < a.n;
  }
  return axis;
}

__global__ __launch_bounds__(kThreads) void rope_axes_kernel(
    const bf16* t, bf16* out, const int64_t* __restrict__ positions, int64_t p_sa, int64_t p_sb, int64_t p_ss,
    const double* __restrict__ inv_freq, RopeAxes axes, int64_t tokens, int b, int heads, int hd, int64_t t_ss, int64_t t_sb,
    int64_t t_sh, int64_t o_ss, int64_t o_sb, int64_t o_sh, float sign, int group_size, int group_rotate) {
  const int lane = threadIdx.x & 63;
  const int nfg = hd / 16, at_once = 64 / nfg;  // lanes of a head; heads of a wave's step
  const int fg = lane % nfg, first = lane / nfg;
  const bool copies = out != t;                 // heads that are not rotated have to be carried over
  double per_turn[8];
  int axis[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    per_turn[e] = inv_freq[fg * 8 + e] * kTurnsPerRadian;
    axis[e] = axis_of(axes, fg * 8 + e);
  }
  const int64_t waves = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t token = (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); token < tokens;
       token += waves) {
    const int64_t si = token / b;
    const int64_t bi = token - si * b;
    double place[KR_ROPE_MAX_AXES];
#pragma unroll
    for (int a = 0; a < KR_ROPE_MAX_AXES; ++a)
      place[a] = a < axes.n ? (double)positions[a * p_sa + bi * p_sb + si * p_ss] : 0.0;
    float co[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      double p = place[0];
#pragma unroll
      for (int a = 1; a < KR_ROPE_MAX_AXES; ++a) p = axis[e] == a ? place[a] : p;
      const double turns = p * per_turn[e];
      sincospif((float)(2.0 * (turns - __builtin_rint(turns))), &sn[e], &co[e]);
      sn[e] *= sign;
    }
    if (first >= at_once) continue;
    const bf16* const tp = t + si * t_ss + bi * t_sb + fg * 8;
    bf16* const op = out + si * o_ss + bi * o_sb + fg * 8;
    for (int head = first; head < heads; head += at_once) {
      const bool turned = head % group_size < group_rotate;
      if (!turned && !copies) continue;
      bf16x8 x = ldg8(tp + head * t_sh), y = ldg8(tp + head * t_sh + hd / 2);
      if (turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = (float)x[e], c = (float)y[e];
          x[e] = (bf16)(a * co[e] - c * sn[e]);
          y[e] = (bf16)(c * co[e] + a * sn[e]);
        }
      }
      stg8(op + head * o_sh, x);
      stg8(op + head * o_sh + hd / 2, y);
    }
  }
}

}  // namespace

extern "C" int kr_rope_axes(const void* t, void* out, const int64_t* positions, int64_t p_stride_axis, int64_t p_stride_b,
                            int64_t p_stride_s, int axes, const double* inv_freq, const int* sections, int interleaved, int s,
                            int b, int heads, int hd, int64_t t_stride_s, int64_t t_stride_b, int64_t t_stride_h,
                            int64_t o_stride_s, int64_t o_stride_b, int64_t o_stride_h, int backward, int group_size,
                            int group_rotate, void* stream) {
  if (!t || !out || !positions || !inv_freq || !sections || s <= 0 || b <= 0 || heads <= 0 || hd <= 0 || axes <= 0)
    return KR_EINVAL;
  if (group_size <= 0 || group_rotate <= 0 || group_rotate > group_size || heads % group_size) return KR_EINVAL;
  if (hd % 16 || hd > 256 || axes > KR_ROPE_MAX_AXES) return KR_EUNSUPPORTED;
  RopeAxes a{axes, interleaved != 0, {0, 0, 0, 0}};
  int total = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0 || sections[i] > hd / 2) return KR_EINVAL;
    a.sections[i] = sections[i];
    total += sections[i];
  }
  if (total != hd / 2) return KR_EINVAL;
  if (!kr_aligned16(t) || !kr_aligned16(out) || (reinterpret_cast<uintptr_t>(positions) & 7u) ||
      (reinterpret_cast<uintptr_t>(inv_freq) & 7u))
    return KR_EINVAL;
  if ((t_stride_s | t_stride_b | t_stride_h | o_stride_s | o_stride_b | o_stride_h) % 8) return KR_EINVAL;
  if (t_stride_s <= 0 || t_stride_b <= 0 || t_stride_h <= 0 || o_stride_s <= 0 || o_stride_b <= 0 || o_stride_h <= 0)
    return KR_EUNSUPPORTED;
  const int64_t tokens = (int64_t)s * b, blocks = (tokens + 3) / 4;
  hipLaunchKernelGGL(rope_axes_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(kThreads), 0, (hipStream_t)stream,
                     (const bf16*)t, (bf16*)out, positions, p_stride_axis, p_stride_b, p_stride_s, inv_freq, a, tokens, b, heads,
                     hd, t_stride_s, t_stride_b, t_stride_h, o_stride_s, o_stride_b, o_stride_h, backward ? -1.0f : 1.0f,
                     group_size, group_rotate);
  return kr_launch_status();
}
