// Rotary position embedding by positions on several axes (time, height and width of images and video):
//   angle(token, f) = position[axis(f)][token] * inv_freq[f],  (a, b) -> (a cos - b sin, b cos + a sin),
// a and b being channels f and f + hd / 2 of a head.  HBM-bound: every rotated head is read and written once, and a token brings 8
// bytes per axis of positions where a table of angles would be hd * 4 bytes for each.
// A wave takes a token.  A lane has 8 frequencies and every 64 / (hd / 16)-th head, whose 16 bytes of either half it turns; the angles
// themselves, some hundred instructions each, are formed one to a lane and handed over through LDS.  (Formed by every lane that turns by
// them, 4 x 4096 tokens of 8/2 heads took 26.5 us for 18.5.  Vectors of whole rows to a wave, the halves exchanged between its lanes: 154.4
// at best for 154.4, and 19.7 for 18.5.)  In place, as a layer turns its fused buffer, value heads are left alone: 4 x 8191 tokens of 32/8
// heads of 128 take 121 us (5.5 TB/s), into a new buffer 154.
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

// Only lanes of one wave exchange data: the program order of its LDS instructions is all the ordering needed.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// Heads that a lane asks for at once, and workgroups of a launch (4 x 8191 tokens of 32/8 heads of 128, 1.6 GB read and written, and 4 x 4096
// of 8/2, us: 1 head 156.1, 18.5, 2 154.4, 18.5, 3 156.0, 19.0; 1024 workgroups of 2 heads as said, 2048 160.5, 18.9, a wave to a token
// 155.6, 19.9: 5.2 TB/s).
constexpr int kAhead = 2, kBlocks = 1024;
__global__ __launch_bounds__(kThreads) void rope_axes_kernel(
    const bf16* t, bf16* out, const int64_t* __restrict__ positions, int64_t p_sa, int64_t p_sb, int64_t p_ss,
    const double* __restrict__ inv_freq, RopeAxes axes, int64_t tokens, int b, int heads, int hd, int64_t t_ss, int64_t t_sb,
    int64_t t_sh, int64_t o_ss, int64_t o_sb, int64_t o_sh, float sign, int group_size, int group_rotate) {
  const int lane = threadIdx.x & 63;
  const int nfg = hd / 16, at_once = 64 / nfg;  // lanes of a head; heads of a wave's step
  const int fg = lane % nfg, first = lane / nfg;
  const bool copies = out != t;                 // heads that are not rotated have to be carried over
  const bool mine = first < at_once;            // (64 lanes are not whole heads of every size)
  // the angles of a token, one lane to a frequency (or to two, of 256 channels), come to the lanes that turn by them through LDS
  __shared__ __attribute__((aligned(16))) float turns[kThreads / 64][2][128];
  float* const cos_of = turns[threadIdx.x >> 6][0];
  float* const sin_of = turns[threadIdx.x >> 6][1];
  double per_turn[2];
  int axis[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int f = lane + 64 * i < hd / 2 ? lane + 64 * i : 0;
    per_turn[i] = inv_freq[f] * kTurnsPerRadian;
    axis[i] = axis_of(axes, f);
  }
  const int64_t waves = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t token = (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); token < tokens;
       token += waves) {
    const int64_t si = token / b;
    const int64_t bi = token - si * b;
    const bf16* const tp = t + si * t_ss + bi * t_sb + fg * 8;
    bf16* const op = out + si * o_ss + bi * o_sb + fg * 8;
    // the first heads are asked for in front of the angles
    bf16x8 x[kAhead], y[kAhead];
    auto load = [&](int base) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int head = base + i * at_once;
        if (mine && head < heads && (copies || head % group_size < group_rotate)) {
          x[i] = ldg8(tp + head * t_sh);
          y[i] = ldg8(tp + head * t_sh + hd / 2);
        }
      }
    };
    load(first);
    double place[KR_ROPE_MAX_AXES];
#pragma unroll
    for (int a = 0; a < KR_ROPE_MAX_AXES; ++a)
      place[a] = a < axes.n ? (double)positions[a * p_sa + bi * p_sb + si * p_ss] : 0.0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int f = lane + 64 * i;
      if (f >= hd / 2) break;
      double p = place[0];
#pragma unroll
      for (int a = 1; a < KR_ROPE_MAX_AXES; ++a) p = axis[i] == a ? place[a] : p;
      const double angle = p * per_turn[i];
      float sn, co;
      sincospif((float)(2.0 * (angle - __builtin_rint(angle))), &sn, &co);
      cos_of[f] = co;
      sin_of[f] = sn * sign;
    }
    wave_order();
    float co[8], sn[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 c4 = *reinterpret_cast<const f32x4*>(cos_of + fg * 8 + 4 * i);
      const f32x4 s4 = *reinterpret_cast<const f32x4*>(sin_of + fg * 8 + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) co[4 * i + e] = c4[e], sn[4 * i + e] = s4[e];
    }
    wave_order();  // (the next token's are written behind these reads)
    for (int base = first; base < heads; base += kAhead * at_once) {
      if (base > first) load(base);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int head = base + i * at_once;
        const bool turned = head % group_size < group_rotate;
        if (!mine || head >= heads || !(turned || copies)) continue;
        if (turned) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = (float)x[i][e], c = (float)y[i][e];
            x[i][e] = (bf16)(a * co[e] - c * sn[e]);
            y[i][e] = (bf16)(c * co[e] + a * sn[e]);
          }
        }
        if (copies) {
          stg8_stream(op + head * o_sh, x[i]);
          stg8_stream(op + head * o_sh + hd / 2, y[i]);
        } else {
          stg8(op + head * o_sh, x[i]);
          stg8(op + head * o_sh + hd / 2, y[i]);
        }
      }
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
  hipLaunchKernelGGL(rope_axes_kernel, dim3((unsigned)(blocks < kBlocks ? blocks : kBlocks)), dim3(kThreads), 0, (hipStream_t)stream,
                     (const bf16*)t, (bf16*)out, positions, p_stride_axis, p_stride_b, p_stride_s, inv_freq, a, tokens, b, heads,
                     hd, t_stride_s, t_stride_b, t_stride_h, o_stride_s, o_stride_b, o_stride_h, backward ? -1.0f : 1.0f,
                     group_size, group_rotate);
  return kr_launch_status();
}
