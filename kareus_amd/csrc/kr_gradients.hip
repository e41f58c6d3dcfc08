// The norm of all gradients that a process holds and clipping by it: norm = sqrt(sum g^2) over all tensors, factor = min(1, max_norm /
// (norm + eps)), g factor in place or in fp32 elsewhere.  HBM-bound: the norm reads every gradient once, clipping once more, and
// writes it.
// Tensors come as a table in the launch's own arguments, kTensors to a launch: nothing has to be copied to the device first, and a
// captured launch holds what it needs.  Each is cut in chunks of 4096 elements, and a workgroup takes a contiguous range of all
// chunks, so that it looks its first tensor up once and then only walks on.
// Sums are 64 bits from the first square on: the square of a bf16 or fp32 value is exact and never overflows or vanishes there,
// whatever the gradients' size, and the conversion and the multiply-add are a fraction of the time that the values take to arrive.
// Each workgroup leaves its sum in its own place and one more adds them in order: no atomics, the norm is reproducible.
// The pass that scales goes through the chunks from the last to the first, which are the ones the caches still hold; what it writes
// elsewhere goes past them, in whole 1 KB pieces to a wave.  Norm and scaled copy of 218 M bf16 and 131 M fp32 elements (0.96 GB read twice, 1.4
// GB written), us: 8 elements to a lane, 1024 workgroups of 8192 elements 237 + 479, 2048 209 + 482, from the last chunk on 209 + 472; 4
// elements to a lane 209 + 443; its stores past the caches, which leave the next step's first pass clean ones, 164 + 464; 4096 workgroups of
// 4096 elements 156 + 460: 5.4 TB/s.  In place, norm and scaling of 0.96 GB in bf16 and fp32 544 (5.3 TB/s of two reads and a write), of 0.35
// GB 209; with a factor of 1 170 and 87, the norm's own time.
#include "kr_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 128;
constexpr int kBlocks = 4096;                 // workgroups of a launch, and sums that it leaves
constexpr int kUnroll = 2;
constexpr int kChunk = kThreads * 8 * kUnroll;  // elements

// (tensors may begin at any element: the hardware takes such loads as they are)
typedef bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef bf16 bf16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct Table {
  const void* grad[kTensors];
  int64_t count[kTensors];        // elements; negative: fp32
  uint32_t first[kTensors];       // chunk
  int n;
  uint32_t chunks;
};
struct Outputs {
  float* to[kTensors];
};

// The chunks of this workgroup, REV: all from the last to the first: f(tensor, first element, its tensor's elements, fp32)
template <bool REV, typename F>
__device__ __forceinline__ void for_chunks(const Table& t, F&& f) {
  const uint32_t at = REV ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const uint32_t lo = (uint32_t)((uint64_t)t.chunks * at / gridDim.x);
  const uint32_t hi = (uint32_t)((uint64_t)t.chunks * (at + 1) / gridDim.x);
  if (lo >= hi) return;
  uint32_t c = REV ? hi - 1 : lo;
  int i = 0;
  for (int step = kTensors / 2; step > 0; step >>= 1)
    if (i + step < t.n && t.first[i + step] <= c) i += step;
  for (;;) {
    const int64_t n = t.count[i];
    f(i, (int64_t)(c - t.first[i]) * kChunk, n < 0 ? -n : n, n < 0);
    if (REV) {
      if (c == lo) return;
      --c;
      while (c < t.first[i]) --i;
    } else {
      if (++c == hi) return;
      while (i + 1 < t.n && c >= t.first[i + 1]) ++i;
    }
  }
}

__device__ __forceinline__ void load8(const void* g, int64_t at, bool fp32, float (&v)[8]) {
  if (fp32) {
    const f32x4u a = *reinterpret_cast<const f32x4u*>((const float*)g + at);
    const f32x4u b = *reinterpret_cast<const f32x4u*>((const float*)g + at + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  } else {
    const bf16x8u a = *reinterpret_cast<const bf16x8u*>((const bf16*)g + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
  }
}
__device__ __forceinline__ float load1(const void* g, int64_t at, bool fp32) {
  return fp32 ? ((const float*)g)[at] : (float)((const bf16*)g)[at];
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, KR_WAVE);
  return v;
}

__global__ __launch_bounds__(kThreads) void grad_square_kernel(Table t, double* __restrict__ sums) {
  __shared__ double parts[kThreads / 64];
  double acc[2] = {0.0, 0.0};
  for_chunks<false>(t, [&](int i, int64_t first, int64_t n, bool fp32) {
    const void* const g = t.grad[i];
    if (first + kChunk <= n) {
      float v[kUnroll][8];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) load8(g, first + ((int64_t)u * kThreads + threadIdx.x) * 8, fp32, v[u]);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e & 1] = __builtin_fma((double)v[u][e], (double)v[u][e], acc[e & 1]);
    } else {
      for (int64_t at = first + threadIdx.x; at < n; at += kThreads) {
        const double v = load1(g, at, fp32);
        acc[0] = __builtin_fma(v, v, acc[0]);
      }
    }
  });
  const double w = wave_sum64(acc[0] + acc[1]);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = w;
  kr_barrier();
  if (threadIdx.x == 0) sums[blockIdx.x] = (parts[0] + parts[1]) + (parts[2] + parts[3]);
}

// result: the norm in 64 bits, for the launches that clip; norm: in 32
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void grad_norm_kernel(const double* __restrict__ sums, int n, double* __restrict__ result,
                                                                float* __restrict__ norm) {
  __shared__ double parts[kSumThreads / 64];
  double acc = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += kSumThreads) acc += sums[i];
  acc = wave_sum64(acc);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = acc;
  kr_barrier();
  if (threadIdx.x == 0) {
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kSumThreads / 64; ++w) total += parts[w];
    const double r = sqrt(total);
    *result = r;
    *norm = (float)r;
  }
}

// IN_PLACE: bf16 stays bf16, rounded once; a factor of 1 leaves everything as it is
template <bool IN_PLACE>
__global__ __launch_bounds__(kThreads) void grad_scale_kernel(Table t, Outputs out, const double* __restrict__ norm, double max_norm,
                                                              double eps) {
  const double quotient = max_norm / (*norm + eps);
  const float factor = quotient >= 1.0 ? 1.0f : (float)quotient;  // (not a number: that)
  if (IN_PLACE && factor == 1.0f) return;
  for_chunks<true>(t, [&](int i, int64_t first, int64_t n, bool fp32) {
    const void* const g = t.grad[i];
    if (first + kChunk <= n) {
      if (IN_PLACE && !fp32) {
        bf16* const p = (bf16*)g + first + threadIdx.x * 8;
        bf16x8u v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u] = *reinterpret_cast<const bf16x8u*>(p + u * kThreads * 8);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[u][e] = (bf16)((float)v[u][e] * factor);
          *reinterpret_cast<bf16x8u*>(p + u * kThreads * 8) = v[u];
        }
        return;
      }
      // four elements to a lane, so that a wave's store is one piece of 1 KB
      f32x4u v[2 * kUnroll];
      const int64_t at = first + threadIdx.x * 4;
#pragma unroll
      for (int u = 0; u < 2 * kUnroll; ++u) {
        if (fp32) {
          v[u] = *reinterpret_cast<const f32x4u*>((const float*)g + at + u * kThreads * 4);
        } else {
          const bf16x4u h = *reinterpret_cast<const bf16x4u*>((const bf16*)g + at + u * kThreads * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = (float)h[e];
        }
      }
      float* const to = (IN_PLACE ? (float*)g : out.to[i]) + at;
#pragma unroll
      for (int u = 0; u < 2 * kUnroll; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[u][e] *= factor;
        if (!IN_PLACE)
          __builtin_nontemporal_store(v[u], reinterpret_cast<f32x4u*>(to + u * kThreads * 4));
        else
          *reinterpret_cast<f32x4u*>(to + u * kThreads * 4) = v[u];
      }
    } else {
      for (int64_t at = first + threadIdx.x; at < n; at += kThreads) {
        const float v = load1(g, at, fp32) * factor;
        if (IN_PLACE && !fp32)
          ((bf16*)g)[at] = (bf16)v;
        else
          (IN_PLACE ? (float*)g : out.to[i])[at] = v;
      }
    }
  });
}

int check(int n, const void* const* grads, const int64_t* counts, const int* fp32, void* const* out) {
  if (n <= 0 || !grads || !counts || !fp32) return KR_EINVAL;
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0) return KR_EINVAL;
    if (counts[i] == 0) continue;
    const uintptr_t at = reinterpret_cast<uintptr_t>(grads[i]);
    if (!at || at % (fp32[i] ? 4 : 2)) return KR_EINVAL;
    if (out && (!out[i] || reinterpret_cast<uintptr_t>(out[i]) % 4)) return KR_EINVAL;
    if (counts[i] > ((int64_t)1 << 37) - kChunk) return KR_EUNSUPPORTED;  // (kTensors of them: below 2^32 chunks)
  }
  return KR_OK;
}

// Tensors from `*at` on, as many as fit; false: none was left
bool next_table(int n, const void* const* grads, const int64_t* counts, const int* fp32, void* const* out, int* at, Table* t,
                Outputs* o) {
  t->n = 0;
  t->chunks = 0;
  for (; *at < n && t->n < kTensors; ++*at) {
    const int64_t count = counts[*at];
    if (!count) continue;
    t->grad[t->n] = grads[*at];
    t->count[t->n] = fp32[*at] ? -count : count;
    t->first[t->n] = t->chunks;
    if (o) o->to[t->n] = (float*)out[*at];
    t->chunks += (uint32_t)((count + kChunk - 1) / kChunk);
    ++t->n;
  }
  return t->n > 0;
}

unsigned blocks_of(const Table& t) { return t.chunks < (uint32_t)kBlocks ? t.chunks : (unsigned)kBlocks; }

}  // namespace

extern "C" size_t kr_grad_norm_workspace_bytes(int n) {
  return n <= 0 ? 0 : 16 + (size_t)((n + kTensors - 1) / kTensors) * kBlocks * sizeof(double);
}

extern "C" int kr_grad_norm(int n, const void* const* grads, const int64_t* counts, const int* fp32, float* norm, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (const int rc = check(n, grads, counts, fp32, nullptr)) return rc;
  if (!norm || !workspace || !kr_aligned16(workspace) || workspace_bytes < kr_grad_norm_workspace_bytes(n)) return KR_EINVAL;
  double* const sums = (double*)workspace + 2;
  Table t;
  int at = 0, left = 0;
  while (next_table(n, grads, counts, fp32, nullptr, &at, &t, nullptr)) {
    const unsigned blocks = blocks_of(t);
    hipLaunchKernelGGL(grad_square_kernel, dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, t, sums + left);
    left += (int)blocks;
    if (hipGetLastError() != hipSuccess) return KR_ELAUNCH;
  }
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kSumThreads), 0, (hipStream_t)stream, (const double*)sums, left,
                     (double*)workspace, norm);
  return kr_launch_status();
}

extern "C" int kr_grad_clip(int n, const void* const* grads, const int64_t* counts, const int* fp32, void* const* out,
                            double max_norm, double eps, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (!(max_norm >= 0.0) || !(eps >= 0.0)) return KR_EINVAL;
  if (const int rc = check(n, grads, counts, fp32, out)) return rc;
  if (const int rc = kr_grad_norm(n, grads, counts, fp32, norm, workspace, workspace_bytes, stream)) return rc;
  Table t;
  Outputs o{};
  int at = 0;
  while (next_table(n, grads, counts, fp32, out, &at, &t, out ? &o : nullptr)) {
    if (out)
      hipLaunchKernelGGL(grad_scale_kernel<false>, dim3(blocks_of(t)), dim3(kThreads), 0, (hipStream_t)stream, t, o,
                         (const double*)workspace, max_norm, eps);
    else
      hipLaunchKernelGGL(grad_scale_kernel<true>, dim3(blocks_of(t)), dim3(kThreads), 0, (hipStream_t)stream, t, o,
                         (const double*)workspace, max_norm, eps);
    if (hipGetLastError() != hipSuccess) return KR_ELAUNCH;
  }
  return KR_OK;
}
