// Token embedding with a factor, and its gradient by sorted tokens.
//
//   forward   out[si, bi, :] = bf16(scale * weight[ids[bi, si] - vocab_start, :]), zeros for ids of other shards
//   gradient  dweight[r, :] (+)= scale * sum over tokens t with id vocab_start + r of dout[t, :], fp32 sums, rounded once
//
// The gradient sorts the tokens by row (stable: equal rows stay in the order of dout), cuts the sorted tokens into chunks of equal
// length whatever the ids, sums each chunk's runs of equal rows, and joins the runs that chunks share in chunk order.  No sum
// depends on scheduling, and an id that fills the batch is spread over the device like any other.
#include "kr_common.h"

#include <algorithm>

namespace {

constexpr int kThreads = 256;

// ---- forward -----------------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void embedding_scaled_kernel(const int64_t* __restrict__ ids, const bf16* __restrict__ weight,
                                                                   bf16* __restrict__ out, int s, int b, int hidden,
                                                                   int64_t vocab_start, int64_t vocab_rows, float scale) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tokens = (int64_t)s * b;
  const int nvec = hidden / 8;
  for (int64_t t = (int64_t)blockIdx.x * 4 + wave; t < tokens; t += (int64_t)gridDim.x * 4) {
    const int si = (int)(t / b), bi = (int)(t % b);
    const int64_t row = ids[(int64_t)bi * s + si] - vocab_start;
    const bool mine = row >= 0 && row < vocab_rows;
    const bf16* src = weight + (mine ? row : 0) * hidden;
    bf16* dst = out + t * hidden;
    for (int v = lane; v < nvec; v += 64) {
      bf16x8 x = mine ? ldg8(src + v * 8) : zero8();
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (bf16)((float)x[e] * scale);
      stg8(dst + v * 8, mine ? x : zero8());
    }
  }
}

// ---- sort: least significant digit first, blocks of kBlock tokens --------------------------------
constexpr int kBlock = 2048, kPerWave = kBlock / 4;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;

// A token's row, or vocab_rows (behind all others) where its id belongs to another shard.
__device__ __forceinline__ unsigned row_of(const int64_t* ids, int64_t t, int s, int b, int64_t vocab_start, int64_t vocab_rows) {
  const int64_t si = t / b, bi = t - si * b;
  const int64_t row = ids[bi * s + si] - vocab_start;
  return (unsigned)(row >= 0 && row < vocab_rows ? row : vocab_rows);
}

struct SortArgs {
  const int64_t* ids;
  int s, b;
  int64_t vocab_start, vocab_rows;
  const unsigned *keys, *pos;     // input of a pass behind the first
  unsigned *keys_out, *pos_out;
  unsigned* counts;               // [bins][blocks]
  unsigned* totals;               // [bins]
  uint8_t* seen;                  // [vocab_rows]: cleared by the first pass's count
  int tokens, blocks, shift, bits;
};

template <bool FIRST>
__device__ __forceinline__ unsigned key_at(const SortArgs& g, int t) {
  return FIRST ? row_of(g.ids, t, g.s, g.b, g.vocab_start, g.vocab_rows) : g.keys[t];
}

template <bool FIRST>
__global__ __launch_bounds__(kThreads) void sort_count_kernel(SortArgs g) {
  __shared__ unsigned hist[kMaxBins];
  const int tid = threadIdx.x, bins = 1 << g.bits;
  if (FIRST)
    for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < g.vocab_rows; i += (int64_t)gridDim.x * kThreads) g.seen[i] = 0;
  for (int i = tid; i < bins; i += kThreads) hist[i] = 0;
  kr_barrier();
  for (int i = tid; i < kBlock; i += kThreads) {
    const int64_t t = (int64_t)blockIdx.x * kBlock + i;
    if (t < g.tokens) atomicAdd(&hist[(key_at<FIRST>(g, (int)t) >> g.shift) & (bins - 1)], 1u);
  }
  kr_barrier();
  for (int i = tid; i < bins; i += kThreads) g.counts[(int64_t)i * g.blocks + blockIdx.x] = hist[i];
}

// One workgroup per digit value: its counts over the blocks become running sums, its total goes to totals.
__global__ __launch_bounds__(kThreads) void sort_scan_kernel(unsigned* counts, unsigned* totals, int blocks) {
  __shared__ unsigned part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned* c = counts + (int64_t)blockIdx.x * blocks;
  unsigned before = 0;
  for (int i0 = 0; i0 < blocks; i0 += kThreads) {
    const int i = i0 + tid;
    const unsigned v = i < blocks ? c[i] : 0;
    unsigned inc = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned up = __shfl_up(inc, o, 64);
      if (lane >= o) inc += up;
    }
    if (lane == 63) part[wave] = inc;
    kr_barrier();
    unsigned base = before;
    for (int w = 0; w < wave; ++w) base += part[w];
    if (i < blocks) c[i] = base + inc - v;
    before += part[0] + part[1] + part[2] + part[3];
    kr_barrier();
  }
  if (tid == 0) totals[blockIdx.x] = before;
}

template <bool FIRST>
__global__ __launch_bounds__(kThreads) void sort_scatter_kernel(SortArgs g) {
  __shared__ unsigned start[4][kMaxBins];   // where the next token of a wave with this digit goes
  __shared__ unsigned part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = 1 << g.bits;
  for (int w = 0; w < 4; ++w)
    for (int i = tid; i < bins; i += kThreads) start[w][i] = 0;
  kr_barrier();
  const int64_t first = (int64_t)blockIdx.x * kBlock + wave * kPerWave;
  for (int i = lane; i < kPerWave; i += 64) {
    const int64_t t = first + i;
    if (t < g.tokens) atomicAdd(&start[wave][(key_at<FIRST>(g, (int)t) >> g.shift) & (bins - 1)], 1u);
  }
  kr_barrier();
  // running sums of the digits' totals: thread t takes the digits 2 t and 2 t + 1
  {
    const unsigned a = 2 * tid < bins ? g.totals[2 * tid] : 0, c = 2 * tid + 1 < bins ? g.totals[2 * tid + 1] : 0;
    unsigned inc = a + c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned up = __shfl_up(inc, o, 64);
      if (lane >= o) inc += up;
    }
    if (lane == 63) part[wave] = inc;
    kr_barrier();
    unsigned base = inc - a - c;
    for (int w = 0; w < wave; ++w) base += part[w];
    for (int d = 0; d < 2; ++d) {
      const int i = 2 * tid + d;
      if (i < bins) {
        unsigned at = base + (d ? a : 0) + g.counts[(int64_t)i * g.blocks + blockIdx.x];
        for (int w = 0; w < 4; ++w) {
          const unsigned n = start[w][i];
          start[w][i] = at;
          at += n;
        }
      }
    }
  }
  kr_barrier();
  for (int i0 = 0; i0 < kPerWave; i0 += 64) {   // (a wave's tokens in order, 64 at a time)
    const int64_t t = first + i0 + lane;
    const bool in = t < g.tokens;
    const unsigned key = in ? key_at<FIRST>(g, (int)t) : 0;
    const unsigned pos = in ? (FIRST ? (unsigned)t : g.pos[t]) : 0;
    const unsigned digit = (key >> g.shift) & (bins - 1);
    unsigned long long same = __ballot(in);
    for (int bit = 0; bit < g.bits; ++bit) {
      const unsigned long long set = __ballot(digit >> bit & 1);
      same &= digit >> bit & 1 ? set : ~set;
    }
    if (in) {
      const unsigned rank = __popcll(same & ((1ull << lane) - 1));
      const unsigned at = start[wave][digit] + rank;
      g.keys_out[at] = key;
      g.pos_out[at] = pos;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    if (in && (same >> lane) == 1) start[wave][digit] += __popcll(same);   // the last lane of each digit
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- sums --------------------------------------------------------------------------------------
struct SumArgs {
  const unsigned *keys, *pos;
  const bf16* dout;
  void* out;
  float* partial;     // [chunks][2][hidden]: the run a chunk shares with the chunks before it, and the one with those behind
  uint8_t* seen;
  int tokens, hidden, chunk, chunks;
  unsigned vocab_rows;
  float scale;
  int accumulate;
};

template <typename T>
__device__ __forceinline__ void put_row(const SumArgs& g, unsigned row, int col, float (&sum)[8]) {
  T* const p = reinterpret_cast<T*>(g.out) + (int64_t)row * g.hidden + col;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] *= g.scale;
  if (g.accumulate) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += (float)p[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) p[e] = (T)sum[e];
}

// One wave per chunk of sorted tokens and 512 columns.
template <typename T>
__global__ __launch_bounds__(64) void sorted_sum_kernel(SumArgs g) {
  const int lane = threadIdx.x, c = blockIdx.x;
  const int col = blockIdx.y * 512 + lane * 8;
  const bool live = col < g.hidden;
  const int lo = c * g.chunk, hi = lo + g.chunk < g.tokens ? lo + g.chunk : g.tokens;
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  unsigned row = g.keys[lo];
  bool shared = lo > 0 && g.keys[lo - 1] == row;   // the run has begun in an earlier chunk
  for (int i = lo; i < hi; ++i) {
    if (row >= g.vocab_rows) break;                // (tokens of other shards come last)
    if (live) {
      const bf16x8 v = ldg8(g.dout + (int64_t)g.pos[i] * g.hidden + col);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += (float)v[e];
    }
    const unsigned next = i + 1 < g.tokens ? g.keys[i + 1] : g.vocab_rows;
    const bool ends = i + 1 >= g.tokens || next != row;
    if (ends || i + 1 == hi) {
      if (blockIdx.y == 0 && lane == 0) g.seen[row] = 1;
      if (live) {
        if (shared || !ends) {
          float* const p = g.partial + ((int64_t)c * 2 + (shared ? 0 : 1)) * g.hidden + col;
#pragma unroll
          for (int e = 0; e < 8; ++e) p[e] = sum[e];
        } else {
          put_row<T>(g, row, col, sum);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = 0.f;
      shared = false;
      row = next;
    }
  }
}

// Joins the runs that go on behind the chunk they begin in (one wave per chunk and 512 columns).
template <typename T>
__global__ __launch_bounds__(64) void sorted_join_kernel(SumArgs g) {
  const int lane = threadIdx.x, c = blockIdx.x;
  const int col = blockIdx.y * 512 + lane * 8;
  const int last = c * g.chunk + g.chunk - 1;
  if (last + 1 >= g.tokens) return;
  const unsigned row = g.keys[last];
  if (row >= g.vocab_rows || g.keys[last + 1] != row) return;
  const int lo = c * g.chunk;
  if (lo > 0 && g.keys[lo - 1] == row) return;     // begun before this chunk (and all of it)
  if (col >= g.hidden) return;
  float sum[8];
  const float* p = g.partial + ((int64_t)c * 2 + 1) * g.hidden + col;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = p[e];
  for (int n = c + 1; n < g.chunks && g.keys[n * g.chunk] == row; ++n) {
    p = g.partial + (int64_t)n * 2 * g.hidden + col;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += p[e];
  }
  put_row<T>(g, row, col, sum);
}

// Zeros for the rows without a token.
template <typename T>
__global__ __launch_bounds__(kThreads) void unseen_rows_kernel(const uint8_t* seen, T* out, int64_t rows, int hidden) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
    if (seen[r]) continue;
    constexpr int V = 16 / sizeof(T);
    for (int v = lane; v < hidden / V; v += 64) *reinterpret_cast<u32x4*>(out + r * hidden + v * V) = u32x4{0, 0, 0, 0};
  }
}

struct Layout {
  int tokens, blocks, chunk, chunks, bits, passes;
  size_t counts, keys_a, pos_a, keys_b, pos_b, seen, partial, bytes;
};
Layout layout(int64_t tokens, int hidden, int64_t vocab_rows) {
  Layout l{};
  l.tokens = (int)tokens;
  l.blocks = (int)((tokens + kBlock - 1) / kBlock);
  int need = 1;
  while ((vocab_rows >> need) != 0) ++need;   // bits of vocab_rows itself: the mark of other shards' tokens
  l.passes = (need + kMaxBits - 1) / kMaxBits;
  l.bits = (need + l.passes - 1) / l.passes;
  l.chunk = 16;
  while ((tokens + l.chunk - 1) / l.chunk > 4096) l.chunk *= 2;
  l.chunks = (int)((tokens + l.chunk - 1) / l.chunk);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t here = at;
    at += (n + 255) / 256 * 256;
    return here;
  };
  l.counts = take(4 * ((size_t)kMaxBins * l.blocks + kMaxBins));
  l.keys_a = take(4 * tokens);
  l.pos_a = take(4 * tokens);
  l.keys_b = take(4 * tokens);
  l.pos_b = take(4 * tokens);
  l.seen = take(vocab_rows);
  l.partial = take((size_t)l.chunks * 2 * hidden * 4);
  l.bytes = at;
  return l;
}

}  // namespace

extern "C" int kr_embedding_fwd_scaled(const int64_t* ids, const void* weight, void* out, int s, int b, int hidden,
                                       int64_t vocab_start, int64_t vocab_rows, float scale, void* stream) {
  if (!ids || !weight || !out || s <= 0 || b <= 0 || hidden <= 0 || vocab_rows <= 0) return KR_EINVAL;
  if (hidden % 8) return KR_EUNSUPPORTED;
  if (!kr_aligned16(weight) || !kr_aligned16(out)) return KR_EINVAL;
  int64_t blocks = ((int64_t)s * b + 3) / 4;
  if (blocks > 256 * 16) blocks = 256 * 16;
  hipLaunchKernelGGL(embedding_scaled_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, ids,
                     (const bf16*)weight, (bf16*)out, s, b, hidden, vocab_start, vocab_rows, scale);
  return kr_launch_status();
}

extern "C" size_t kr_embedding_bwd_sorted_workspace_bytes(int s, int b, int hidden, int64_t vocab_rows) {
  if (s <= 0 || b <= 0 || hidden <= 0 || vocab_rows <= 0 || vocab_rows >= (1 << 27) || (int64_t)s * b >= (1 << 26)) return 0;
  return layout((int64_t)s * b, hidden, vocab_rows).bytes;
}

extern "C" int kr_embedding_bwd_sorted(const int64_t* ids, const void* dout, void* dweight, int out_fp32, int s, int b, int hidden,
                                       int64_t vocab_start, int64_t vocab_rows, float scale, int accumulate, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  if (!ids || !dout || !dweight || !workspace || s <= 0 || b <= 0 || hidden <= 0 || vocab_rows <= 0) return KR_EINVAL;
  if (hidden % 8 || vocab_rows >= (1 << 27) || (int64_t)s * b >= (1 << 26)) return KR_EUNSUPPORTED;
  if (!kr_aligned16(dout) || !kr_aligned16(dweight) || !kr_aligned16(workspace)) return KR_EINVAL;
  const Layout l = layout((int64_t)s * b, hidden, vocab_rows);
  if (workspace_bytes < l.bytes) return KR_EINVAL;
  char* const ws = (char*)workspace;
  const hipStream_t st = (hipStream_t)stream;
  SortArgs a{};
  a.ids = ids;
  a.s = s;
  a.b = b;
  a.vocab_start = vocab_start;
  a.vocab_rows = vocab_rows;
  a.counts = (unsigned*)(ws + l.counts);
  a.totals = a.counts + (size_t)kMaxBins * l.blocks;
  a.seen = (uint8_t*)(ws + l.seen);
  a.tokens = l.tokens;
  a.blocks = l.blocks;
  a.bits = l.bits;
  unsigned *ka = (unsigned*)(ws + l.keys_a), *pa = (unsigned*)(ws + l.pos_a);
  unsigned *kb = (unsigned*)(ws + l.keys_b), *pb = (unsigned*)(ws + l.pos_b);
  for (int p = 0; p < l.passes; ++p) {
    a.shift = p * l.bits;
    a.keys = kb;
    a.pos = pb;
    a.keys_out = ka;
    a.pos_out = pa;
    if (p == 0) hipLaunchKernelGGL(sort_count_kernel<true>, dim3(l.blocks), dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL(sort_count_kernel<false>, dim3(l.blocks), dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL(sort_scan_kernel, dim3(1 << l.bits), dim3(kThreads), 0, st, a.counts, a.totals, l.blocks);
    if (p == 0) hipLaunchKernelGGL(sort_scatter_kernel<true>, dim3(l.blocks), dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL(sort_scatter_kernel<false>, dim3(l.blocks), dim3(kThreads), 0, st, a);
    std::swap(ka, kb);
    std::swap(pa, pb);
  }
  const SumArgs g{kb, pb, (const bf16*)dout, dweight, (float*)(ws + l.partial), a.seen, l.tokens, hidden, l.chunk, l.chunks,
                  (unsigned)vocab_rows, scale, accumulate};
  const dim3 grid(l.chunks, (hidden + 511) / 512);
  const unsigned zero_blocks = (unsigned)std::min<int64_t>((vocab_rows + 3) / 4, 256 * 32);
  if (out_fp32) {
    hipLaunchKernelGGL(sorted_sum_kernel<float>, grid, dim3(64), 0, st, g);
    hipLaunchKernelGGL(sorted_join_kernel<float>, grid, dim3(64), 0, st, g);
    if (!accumulate) hipLaunchKernelGGL(unseen_rows_kernel<float>, dim3(zero_blocks), dim3(kThreads), 0, st, a.seen, (float*)dweight, vocab_rows, hidden);
  } else {
    hipLaunchKernelGGL(sorted_sum_kernel<bf16>, grid, dim3(64), 0, st, g);
    hipLaunchKernelGGL(sorted_join_kernel<bf16>, grid, dim3(64), 0, st, g);
    if (!accumulate) hipLaunchKernelGGL(unseen_rows_kernel<bf16>, dim3(zero_blocks), dim3(kThreads), 0, st, a.seen, (bf16*)dweight, vocab_rows, hidden);
  }
  return kr_launch_status();
}
