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
// A workgroup takes `TOKENS` tokens and a vector of eight columns per thread: all rows' pieces are asked for before the first is used.
// Bytes: 2 * T * hidden * 2 (+ ids).
template <int TOKENS>
__global__ __launch_bounds__(kThreads) void embedding_scaled_kernel(const int64_t* __restrict__ ids, const bf16* __restrict__ weight,
                                                                   bf16* __restrict__ out, int s, int b, int hidden,
                                                                   int64_t vocab_start, int64_t vocab_rows, float scale) {
  const int col = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  if (col >= hidden) return;
  const int64_t tokens = (int64_t)s * b;
  bf16x8 x[TOKENS];
  bool mine[TOKENS];
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    int64_t t = (int64_t)blockIdx.x * TOKENS + i;
    t = t < tokens ? t : tokens - 1;
    const int64_t si = t / b, bi = t - si * b;
    const int64_t row = ids[bi * s + si] - vocab_start;
    mine[i] = row >= 0 && row < vocab_rows;
    x[i] = ldg8(weight + (mine[i] ? row : 0) * hidden + col);
  }
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    const int64_t t = (int64_t)blockIdx.x * TOKENS + i;
    if (t >= tokens) break;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = (bf16)((float)x[i][e] * scale);
    stg8(out + t * hidden + col, mine[i] ? x[i] : zero8());
  }
}

// A token's row, or vocab_rows (behind all others) where its id belongs to another shard.  Tokens count in dout's order.
__device__ __forceinline__ unsigned row_of(const int64_t* ids, unsigned t, int s, int b, int64_t vocab_start, int64_t vocab_rows) {
  const unsigned si = t / (unsigned)b, bi = t - si * (unsigned)b;   // (tokens: below 2^26)
  const int64_t row = ids[(int64_t)bi * s + si] - vocab_start;
  return (unsigned)(row >= 0 && row < vocab_rows ? row : vocab_rows);
}

struct SortArgs {
  const int64_t* ids;
  int s, b;
  int64_t vocab_start, vocab_rows;
  const unsigned *keys, *pos;     // input of a pass behind the first
  unsigned *keys_out, *pos_out;
  unsigned* counts;               // [blocks][bins]
  unsigned* totals;               // [bins], where there are many blocks
  uint8_t* seen;                  // [vocab_rows up to a multiple of 16], cleared by the first launch (null: not wanted)
  int* joins;                     // how many runs the sums leave to be joined: cleared by the first launch
  int tokens, blocks, block, shift, bits;
};

// The workgroups behind the first `blocks` of the first launch, 16 KB each.
constexpr int kClearBytes = 16384;
__device__ __forceinline__ void clear_seen(const SortArgs& g, int block, int threads) {
  const int64_t lo = (int64_t)block * kClearBytes;
  for (int i = threadIdx.x * 16; i < kClearBytes && lo + i < g.vocab_rows; i += threads * 16)
    *reinterpret_cast<u32x4*>(g.seen + lo + i) = u32x4{0, 0, 0, 0};
}

// ---- sort of few tokens: a token's place is the number of tokens that come before it ---------------
// tokens^2 comparisons, two instructions for 64 of them, and one launch where the passes below are four.  8192 tokens take 13 us, 4 of
// them by that count: every workgroup derives all keys first, a division and a load across the ids' rows each.  A workgroup holds all keys in LDS and places 32 tokens; 32 slices of the keys are compared side by side.
constexpr int kRankMost = 8192, kRankTokens = 32, kRankThreads = 1024;
__global__ __launch_bounds__(kRankThreads) void rank_sort_kernel(SortArgs g) {
  __shared__ __attribute__((aligned(16))) unsigned keys[kRankMost];
  __shared__ unsigned below[32][kRankTokens];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= g.blocks) {
    clear_seen(g, blockIdx.x - g.blocks, kRankThreads);
    return;
  }
  if (blockIdx.x == 0 && tid == 0) *g.joins = 0;
  const int padded = (g.tokens + 127) / 128 * 128;   // 32 slices of whole 16-byte reads
#pragma unroll 8
  for (int t = tid; t < padded; t += kRankThreads)
    keys[t] = t < g.tokens ? row_of(g.ids, t, g.s, g.b, g.vocab_start, g.vocab_rows) : 0xffffffffu;
  kr_barrier();
  const int first = blockIdx.x * kRankTokens, slice = tid >> 5, mine = first + (tid & 31);
  const unsigned key = mine < g.tokens ? keys[mine] : 0;
  const int per = padded / 32, lo = slice * per, hi = lo + per;
  // of a slice in front of these tokens equal keys count as well, of one behind them they do not
  const bool mixed = hi > first && lo < first + kRankTokens;
  unsigned n = 0;
  if (__ballot(mixed) == 0) {
    const unsigned bound = key + (hi <= first ? 1u : 0u);
#pragma unroll 4
    for (int i = lo; i < hi; i += 4) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(&keys[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) n += k[e] < bound ? 1u : 0u;
    }
  } else {
    for (int i = lo; i < hi; i += 4) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(&keys[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) n += k[e] < key + (i + e < mine ? 1u : 0u) ? 1u : 0u;
    }
  }
  below[slice][tid & 31] = n;
  kr_barrier();
  if (tid < kRankTokens && mine < g.tokens) {
    unsigned at = 0;
    for (int i = 0; i < 32; ++i) at += below[i][tid];
    g.keys_out[at] = key;
    g.pos_out[at] = (unsigned)mine;
  }
}

// ---- sort of many tokens: least significant digit first, blocks of up to 2048 tokens -----------------
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
constexpr int kReps = 8;         // tokens of a thread, at most
constexpr int kFewBlocks = 64;   // up to here every block adds the others' counts up by itself

template <bool FIRST>
__device__ __forceinline__ unsigned key_at(const SortArgs& g, int64_t t) {
  return FIRST ? row_of(g.ids, (unsigned)t, g.s, g.b, g.vocab_start, g.vocab_rows) : g.keys[t];
}

template <bool FIRST>
__global__ __launch_bounds__(kThreads) void sort_count_kernel(SortArgs g) {
  __shared__ unsigned hist[kMaxBins];
  const int tid = threadIdx.x, bins = 1 << g.bits;
  if (FIRST && (int)blockIdx.x >= g.blocks) {
    clear_seen(g, blockIdx.x - g.blocks, kThreads);
    return;
  }
  if (FIRST && blockIdx.x == 0 && tid == 0) *g.joins = 0;
  for (int i = tid; i < bins; i += kThreads) hist[i] = 0;
  kr_barrier();
  for (int i = tid; i < g.block; i += kThreads) {
    const int64_t t = (int64_t)blockIdx.x * g.block + i;
    if (t < g.tokens) atomicAdd(&hist[(key_at<FIRST>(g, t) >> g.shift) & (bins - 1)], 1u);
  }
  kr_barrier();
  for (int i = tid; i < bins; i += kThreads) g.counts[(int64_t)blockIdx.x * bins + i] = hist[i];
}

// Many blocks.  One workgroup per digit value: its counts over the blocks become running sums, its total goes to totals.
__global__ __launch_bounds__(kThreads) void sort_scan_kernel(unsigned* counts, unsigned* totals, int blocks) {
  __shared__ unsigned part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned* c = counts + blockIdx.x;
  unsigned before = 0;
  for (int i0 = 0; i0 < blocks; i0 += kThreads) {
    const int i = i0 + tid;
    const unsigned v = i < blocks ? c[(int64_t)i * gridDim.x] : 0;
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
    if (i < blocks) c[(int64_t)i * gridDim.x] = base + inc - v;
    before += part[0] + part[1] + part[2] + part[3];
    kr_barrier();
  }
  if (tid == 0) totals[blockIdx.x] = before;
}

template <bool FIRST, bool SCANNED>
__global__ __launch_bounds__(kThreads) void sort_scatter_kernel(SortArgs g) {
  __shared__ unsigned start[4][kMaxBins];   // where the next token of a wave with this digit goes
  __shared__ unsigned part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = 1 << g.bits;
  const int per_wave = g.block / 4;   // at most 64 kReps
  const int64_t first = (int64_t)blockIdx.x * g.block + wave * per_wave + lane;
  unsigned key[kReps], pos[kReps];
#pragma unroll
  for (int r = 0; r < kReps; ++r) {
    const int64_t t = first + 64 * r;
    const bool in = 64 * r < per_wave && t < g.tokens;
    key[r] = in ? key_at<FIRST>(g, t) : 0;
    pos[r] = in ? (FIRST ? (unsigned)t : g.pos[t]) : 0;
  }
  for (int w = 0; w < 4; ++w)
    for (int i = tid; i < bins; i += kThreads) start[w][i] = 0;
  kr_barrier();
#pragma unroll
  for (int r = 0; r < kReps; ++r)
    if (64 * r < per_wave && first + 64 * r < g.tokens) atomicAdd(&start[wave][(key[r] >> g.shift) & (bins - 1)], 1u);
  // thread t takes the digits 2 t and 2 t + 1: all blocks' tokens with them, and those of the blocks before this
  unsigned total[2] = {0, 0}, before[2] = {0, 0};
  if (2 * tid < bins) {
    if constexpr (SCANNED) {
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        total[d] = g.totals[2 * tid + d];
        before[d] = g.counts[(int64_t)blockIdx.x * bins + 2 * tid + d];
      }
    } else {
#pragma unroll 8
      for (int k = 0; k < g.blocks; ++k) {
        const u32x2 c = *reinterpret_cast<const u32x2*>(g.counts + (int64_t)k * bins + 2 * tid);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          total[d] += c[d];
          before[d] += k < (int)blockIdx.x ? c[d] : 0u;
        }
      }
    }
  }
  unsigned inc = total[0] + total[1];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned up = __shfl_up(inc, o, 64);
    if (lane >= o) inc += up;
  }
  if (lane == 63) part[wave] = inc;
  kr_barrier();
  unsigned base = inc - total[0] - total[1];
  for (int w = 0; w < wave; ++w) base += part[w];
  if (2 * tid < bins) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int i = 2 * tid + d;
      unsigned at = base + (d ? total[0] : 0) + before[d];
      for (int w = 0; w < 4; ++w) {
        const unsigned n = start[w][i];
        start[w][i] = at;
        at += n;
      }
    }
  }
  kr_barrier();
#pragma unroll
  for (int r = 0; r < kReps; ++r) {   // (a wave's tokens in order, 64 at a time)
    if (64 * r >= per_wave) break;
    const bool in = first + 64 * r < g.tokens;
    const unsigned digit = (key[r] >> g.shift) & (bins - 1);
    unsigned long long same = __ballot(in);
    for (int bit = 0; bit < g.bits; ++bit) {
      const unsigned long long set = __ballot(digit >> bit & 1);
      same &= digit >> bit & 1 ? set : ~set;
    }
    if (in) {
      const unsigned at = start[wave][digit] + __popcll(same & ((1ull << lane) - 1));
      g.keys_out[at] = key[r];
      g.pos_out[at] = pos[r];
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
  int* joins;         // how many, then the chunks that a run begins in and goes on behind (in any order)
  int tokens, hidden, chunk, chunks;
  unsigned vocab_rows;
  float scale;
};

template <typename T>
struct Eight {
  T v[8];
};
template <typename T>
__device__ __forceinline__ Eight<T>* row_piece(const SumArgs& g, unsigned row, int col) {
  return reinterpret_cast<Eight<T>*>(reinterpret_cast<T*>(g.out) + (int64_t)row * g.hidden + col);
}
template <typename T, bool ADD>
__device__ __forceinline__ void put_row(const SumArgs& g, unsigned row, int col, const float (&sum)[8], const Eight<T>& old) {
  Eight<T> o;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = sum[e] * g.scale;
    o.v[e] = (T)(ADD ? (float)old.v[e] + v : v);
  }
  if constexpr (ADD) {
    *row_piece<T>(g, row, col) = o;
  } else {   // (a whole table leaves the caches anyway: us, plain and hinted stores, 32768 tokens x 2048 of 128256 rows 164, 154)
    u32x4* const to = reinterpret_cast<u32x4*>(row_piece<T>(g, row, col));
#pragma unroll
    for (unsigned i = 0; i < sizeof(o) / 16; ++i) __builtin_nontemporal_store(reinterpret_cast<const u32x4*>(&o)[i], to + i);
  }
}

// One wave per chunk of sorted tokens (8 or a multiple) and 512 columns, up to four of a chunk in a workgroup.  Eight tokens at a
// time: their rows of dout, and (ADD) what the gradient holds of the rows that end among them, are all asked for before the first
// is used.
constexpr int kAtOnce = 8;
template <typename T, bool ADD>
__global__ __launch_bounds__(kThreads) void sorted_sum_kernel(SumArgs g) {
  const int c = blockIdx.x;
  const int col = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  const bool live = col < g.hidden;
  const int at = live ? col : 0;                   // (lanes behind the row read its start and store nothing)
  const int lo = c * g.chunk;
  if (g.keys[lo] >= g.vocab_rows) return;          // (tokens of other shards come last)
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  bool shared = lo > 0 && g.keys[lo - 1] == g.keys[lo];   // the run has begun in an earlier chunk
  for (int i0 = lo; i0 < lo + g.chunk && i0 < g.tokens; i0 += kAtOnce) {
    unsigned row[kAtOnce + 1];
    bf16x8 v[kAtOnce];
    Eight<T> old[ADD ? kAtOnce : 1];
#pragma unroll
    for (int i = 0; i <= kAtOnce; ++i) row[i] = i0 + i < g.tokens ? g.keys[i0 + i] : g.vocab_rows;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      v[i] = ldg8(g.dout + (int64_t)(row[i] < g.vocab_rows ? g.pos[i0 + i] : 0) * g.hidden + at);
    if constexpr (ADD) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
        if (row[i] < g.vocab_rows && row[i + 1] != row[i]) old[i] = *row_piece<T>(g, row[i], at);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (row[i] >= g.vocab_rows) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += (float)v[i][e];
      const bool ends = row[i + 1] != row[i];
      if (ends || i0 + i + 1 == lo + g.chunk) {
        if (blockIdx.y == 0 && threadIdx.x == 0) {
          if constexpr (!ADD) g.seen[row[i]] = 1;
          if (!shared && !ends && i0 + i + 1 < g.tokens) g.joins[1 + atomicAdd(g.joins, 1)] = c;
        }
        if (live) {
          if (shared || !ends) {
            Eight<float> p;
#pragma unroll
            for (int e = 0; e < 8; ++e) p.v[e] = sum[e];
            *reinterpret_cast<Eight<float>*>(g.partial + ((int64_t)c * 2 + (shared ? 0 : 1)) * g.hidden + col) = p;
          } else {
            put_row<T, ADD>(g, row[i], col, sum, old[ADD ? i : 0]);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = 0.f;
        shared = false;
      }
    }
  }
}

// Behind the sums.  The first `join_groups` workgroups join the runs that go on behind the chunk they begin in (a run and 512 columns
// at a time; the waves take equal parts of the run's chunks, and the parts meet in order); the others write zeros to the rows without
// a token (none where the gradient is added to), one store per thread: `zero_rows` rows of 8 KB together, or one longer row.  (The
// whole gradient, us, 16 rows each time and 8 KB: 8192 tokens x 2048 of 128256 rows in fp32 226, 190; 32768 in bf16 148, 130; 16056 x
// 4096 of 32064 92, 88.  The zeros alone go out at 7 TB/s, as a plain fill's do.)
constexpr int kJoinWaves = 8, kJoinGroups = 512;
template <typename T, bool ADD>
__global__ __launch_bounds__(64 * kJoinWaves) void sorted_finish_kernel(SumArgs g, int join_groups, unsigned zero_rows) {
  __shared__ __attribute__((aligned(16))) float parts[kJoinWaves][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x >= join_groups) {
    if constexpr (!ADD) {
      const unsigned nv = g.hidden * sizeof(T) / 16;
      const int64_t r0 = (int64_t)(blockIdx.x - join_groups) * zero_rows;
      u32x4* const out = reinterpret_cast<u32x4*>(reinterpret_cast<T*>(g.out) + r0 * g.hidden);
      for (unsigned i = threadIdx.x; i < zero_rows * nv; i += 64 * kJoinWaves) {
        const int64_t row = r0 + i / nv;
        if (row < g.vocab_rows && !g.seen[row]) __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, out + i);
      }
    }
    return;
  }
  const int slices = (g.hidden + 511) / 512;
  const int64_t all = (int64_t)*g.joins * slices;
  for (int64_t j = blockIdx.x; j < all; j += join_groups) {
    const int which = (int)(j / slices), col = (int)(j - (int64_t)which * slices) * 512 + lane * 8;
    const int c = g.joins[1 + which], last = c * g.chunk + g.chunk - 1;
    const unsigned row = g.keys[last];
    // the first token behind the run, by halving: of the keys behind `last` those of the run come first
    int begin = last + 1, end = g.tokens;
    while (begin < end) {
      const int mid = begin + (end - begin) / 2;
      if (g.keys[mid] == row) begin = mid + 1;
      else end = mid;
    }
    const int n = (end - 1) / g.chunk - c;           // chunks behind this one that hold a part of the run
    const int per = (n + kJoinWaves - 1) / kJoinWaves;
    const int from = c + 1 + wave * per, to = from + per < c + 1 + n ? from + per : c + 1 + n;
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.f;
    const bool live = col < g.hidden;
    if (live) {
#pragma unroll 4
      for (int k = from; k < to; ++k) {
        const Eight<float> p = *reinterpret_cast<const Eight<float>*>(g.partial + (int64_t)k * 2 * g.hidden + col);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += p.v[e];
      }
    }
    kr_barrier();                                    // (the run before has been added up)
    *reinterpret_cast<Eight<float>*>(&parts[wave][lane * 8]) = *reinterpret_cast<Eight<float>*>(sum);
    kr_barrier();
    if (wave == 0 && live) {
      const Eight<float> p = *reinterpret_cast<const Eight<float>*>(g.partial + ((int64_t)c * 2 + 1) * g.hidden + col);
      Eight<T> old;
      if constexpr (ADD) old = *row_piece<T>(g, row, col);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = p.v[e];
      for (int w = 0; w < kJoinWaves; ++w)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += parts[w][lane * 8 + e];
      put_row<T, ADD>(g, row, col, sum, old);
    }
  }
}

struct Layout {
  int tokens, blocks, block, chunk, chunks, bits, passes;
  size_t counts, keys_a, pos_a, keys_b, pos_b, seen, joins, partial, bytes;
};
Layout layout(int64_t tokens, int hidden, int64_t vocab_rows) {
  Layout l{};
  l.tokens = (int)tokens;
  l.block = 512;
  while (l.block < 2048 && (tokens + l.block - 1) / l.block > kFewBlocks) l.block *= 2;
  l.blocks = (int)((tokens + l.block - 1) / l.block);
  int need = 1;
  while ((vocab_rows >> need) != 0) ++need;   // bits of vocab_rows itself: the mark of other shards' tokens
  l.passes = (need + kMaxBits - 1) / kMaxBits;
  l.bits = (need + l.passes - 1) / l.passes;
  l.chunk = tokens <= 2048 ? 8 : tokens <= 8192 ? 16 : 32;
  while ((tokens + l.chunk - 1) / l.chunk > 8192) l.chunk *= 2;
  l.chunks = (int)((tokens + l.chunk - 1) / l.chunk);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t here = at;
    at += (n + 255) / 256 * 256;
    return here;
  };
  const bool rank = tokens <= kRankMost;
  l.counts = take(rank ? 0 : 4 * ((size_t)kMaxBins * l.blocks + kMaxBins));
  l.keys_a = take(4 * tokens);
  l.pos_a = take(4 * tokens);
  l.keys_b = take(rank ? 0 : 4 * tokens);
  l.pos_b = take(rank ? 0 : 4 * tokens);
  l.seen = take(vocab_rows + 16);
  l.joins = take(4 * (1 + (size_t)l.chunks));
  l.partial = take((size_t)l.chunks * 2 * hidden * 4);
  l.bytes = at;
  return l;
}

template <typename T, bool ADD>
void launch_sums(const SumArgs& g, hipStream_t st) {
  const int slices = (g.hidden + 511) / 512;
  hipLaunchKernelGGL((sorted_sum_kernel<T, ADD>), dim3(g.chunks, (slices + 3) / 4), dim3(64 * std::min(slices, 4)), 0, st, g);
  const int groups = (int)std::min<int64_t>((int64_t)g.chunks * slices, kJoinGroups);
  unsigned zero_rows = std::max(1u, 64 * kJoinWaves * 16 / (unsigned)(g.hidden * sizeof(T)));
  while (g.vocab_rows / zero_rows >= (1u << 22)) zero_rows *= 2;   // (a launch has fewer than 2^32 threads)
  const int64_t zeros = ADD ? 0 : ((int64_t)g.vocab_rows + zero_rows - 1) / zero_rows;
  hipLaunchKernelGGL((sorted_finish_kernel<T, ADD>), dim3((unsigned)(groups + zeros)), dim3(64 * kJoinWaves), 0, st, g, groups, zero_rows);
}

}  // namespace

extern "C" int kr_embedding_fwd_scaled(const int64_t* ids, const void* weight, void* out, int s, int b, int hidden,
                                       int64_t vocab_start, int64_t vocab_rows, float scale, void* stream) {
  if (!ids || !weight || !out || s <= 0 || b <= 0 || hidden <= 0 || vocab_rows <= 0) return KR_EINVAL;
  if (hidden % 8) return KR_EUNSUPPORTED;
  if (!kr_aligned16(weight) || !kr_aligned16(out)) return KR_EINVAL;
  const int64_t tokens = (int64_t)s * b;
  const int nvec = hidden / 8, threads = nvec >= 256 ? 256 : nvec > 64 ? 128 : 64;
  const unsigned slices = (unsigned)((nvec + threads - 1) / threads);
  if (slices > 65535 || tokens >= (1 << 26)) return KR_EUNSUPPORTED;
  // four tokens per workgroup where that still leaves every unit several
  const int per = tokens * slices >= 4096 ? 4 : 1;
  hipLaunchKernelGGL((per == 4 ? embedding_scaled_kernel<4> : embedding_scaled_kernel<1>), dim3((unsigned)((tokens + per - 1) / per), slices),
                     dim3(threads), 0, (hipStream_t)stream, ids, (const bf16*)weight, (bf16*)out, s, b, hidden, vocab_start, vocab_rows, scale);
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
  a.joins = (int*)(ws + l.joins);
  a.tokens = l.tokens;
  a.blocks = l.blocks;
  a.bits = l.bits;
  a.block = l.block;
  unsigned *ka = (unsigned*)(ws + l.keys_a), *pa = (unsigned*)(ws + l.pos_a);
  unsigned *kb = (unsigned*)(ws + l.keys_b), *pb = (unsigned*)(ws + l.pos_b);
  const int clear = accumulate ? 0 : (int)((vocab_rows + kClearBytes - 1) / kClearBytes);
  if (l.tokens <= kRankMost) {
    a.keys_out = ka;
    a.pos_out = pa;
    a.blocks = (l.tokens + kRankTokens - 1) / kRankTokens;
    hipLaunchKernelGGL(rank_sort_kernel, dim3(a.blocks + clear), dim3(kRankThreads), 0, st, a);
    std::swap(ka, kb);
    std::swap(pa, pb);
  } else {
    const bool few = l.blocks <= kFewBlocks;
    for (int p = 0; p < l.passes; ++p) {
      a.shift = p * l.bits;
      a.keys = kb;
      a.pos = pb;
      a.keys_out = ka;
      a.pos_out = pa;
      hipLaunchKernelGGL((p ? sort_count_kernel<false> : sort_count_kernel<true>), dim3(l.blocks + (p ? 0 : clear)), dim3(kThreads), 0, st, a);
      if (!few) hipLaunchKernelGGL(sort_scan_kernel, dim3(1 << l.bits), dim3(kThreads), 0, st, a.counts, a.totals, l.blocks);
      hipLaunchKernelGGL((p ? few ? sort_scatter_kernel<false, false> : sort_scatter_kernel<false, true>
                            : few ? sort_scatter_kernel<true, false> : sort_scatter_kernel<true, true>),
                         dim3(l.blocks), dim3(kThreads), 0, st, a);
      std::swap(ka, kb);
      std::swap(pa, pb);
    }
  }
  const SumArgs g{kb, pb, (const bf16*)dout, dweight, (float*)(ws + l.partial), a.seen, a.joins, l.tokens, hidden, l.chunk, l.chunks,
                  (unsigned)vocab_rows, scale};
  if (out_fp32) {
    if (accumulate) launch_sums<float, true>(g, st);
    else launch_sums<float, false>(g, st);
  } else {
    if (accumulate) launch_sums<bf16, true>(g, st);
    else launch_sums<bf16, false>(g, st);
  }
  return kr_launch_status();
}
