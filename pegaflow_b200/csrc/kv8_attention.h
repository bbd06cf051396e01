// What the kernels of pf_kv8_attention share: parameters, the split of the work, partial results.
#pragma once

#include <cuda_fp16.h>

#include <atomic>

#include "kv8.h"

namespace pf {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNone = -1e30f;   // reference of a row that has seen nothing

struct AttnParams {
  Kv8View cache;
  Kv8Batch batch;
  const uint16_t *q;
  uint16_t *out;
  float *lse;
  float *weights;
  int64_t q_row, q_head, out_row, out_head, w_seq, w_head;
  int w_capacity;
  int q_heads, group, max_query;
  int row_tiles_most;   // of a sequence
  uint32_t units_most;  // units (see Work) that n_rows rows can be, however they fall on the sequences
  int causal, clear_tail, vec_q, vec_out;
  float scale;
  // Partial results: slot 2 c + k of CTA c (k = 0: the segment that its range starts in, 1: the one that it ends in).
  // part_ml holds (base, sum): the row's sum and its part_o are of terms 2^(score - base), scores in base 2.
  float *part_o;    // [slots][rows][dim]
  float2 *part_ml;  // [slots][rows]
  // Scores in base 2, kept for the weights, or null: [sequence][KV head][score_tokens][rows of the tile].
  float *scores;
  int score_tokens;
  int n_ctas, device;
};

// The work of all sequences, heads and row tiles laid end to end in units of some tokens, in equal ranges for n CTAs (the first
// ones one unit longer).  A segment is one (sequence, head, row tile).
struct Split {
  uint32_t each, longer;   // units of a range; how many ranges have one more
  int n_ctas;              // at most the units: every CTA that takes part has work
  __device__ Split(uint32_t total, int n) : n_ctas((int)min((uint32_t)n, total)) {
    each = n_ctas ? total / n_ctas : 0;
    longer = total - each * n_ctas;
  }
  __device__ uint32_t begin(int c) const { return each * c + min((uint32_t)c, longer); }
  __device__ int owner(uint32_t u) const {
    const uint32_t in_longer = longer * (each + 1);
    return (int)(u < in_longer ? u / (each + 1) : longer + (u - in_longer) / each);
  }
};

// One sequence of a call: its rows (row = query * group + head of the group) in tiles of kRows, and its tokens.  kWhole:
// one tile of all rows, that reaches over all tokens.
template <int kRows, int kUnit, bool kWhole = false>
struct Seq {
  int row0, rows, len, row_tiles;
  bool rises;
  __device__ Seq(const AttnParams &p, int s) {
    int hi;
    rises = p.batch.rows(s, row0, hi);
    rows = min(hi - row0, p.max_query);
    len = p.batch.length(s, p.cache.block_log2);
    row_tiles = kWhole ? min(rows, 1) : (rows * p.group + kRows - 1) / kRows;     // kRows is a power of two
  }
  __device__ int all_rows(const AttnParams &p) const { return rows * p.group; }
  __device__ int visible(const AttnParams &p, int row) const {   // tokens that query row `row` sees
    return p.causal && rows > 1 ? min(max(len - rows + row / p.group + 1, 0), len) : len;     // of one query: all
  }
  // Units of one row tile: those that its last row sees, one at least.
  __device__ uint32_t units(const AttnParams &p, int rt) const {
    return max(1, ((kWhole ? len : visible(p, min((rt + 1) * kRows, all_rows(p)) - 1)) + kUnit - 1) / kUnit);
  }
};

// The units of all (sequence, row tile) entries in order, kCost of them in front of each head's for what a segment costs at its
// beginning and end, as sums before every chunk of entries (one, unless there are more
// than kMost).  Every CTA of every kernel computes them for itself: lens stay on the device, and no launch and no
// workspace is spent on it.  Starts that fall and rise again claim rows more than once: where one falls the units are counted
// once more, in 64 bits, and if they are more than the host has checked 32 bits for, there is no work at all.
template <int kRows, int kUnit, bool kWhole = false>
struct Work {
  using SeqT = Seq<kRows, kUnit, kWhole>;
  static constexpr int kMost = 1024;
  // 48 requests of 700 to 16001 tokens, 8 heads of 128: a CTA took 22000 cycles, 2240 for each unit and 8150 for each segment, with
  // 1 to 9 segments to a CTA.
  static constexpr uint32_t kCost = 4;
  uint32_t *prefix;         // [chunks + 1] in shared memory
  int entries, chunk, chunks;
  bool falls, none;         // a row start falls; and there is no work for that
  static __host__ __device__ int chunk_of(int entries) { return max((entries + kMost - 1) / kMost, 1); }
  static __host__ size_t bytes(int n_seqs, int row_tiles_most) {
    const int entries = n_seqs * row_tiles_most, chunk = chunk_of(entries);
    return ((size_t)(entries + chunk - 1) / chunk + 1) * 4;
  }
  static __device__ int seq_of(const AttnParams &p, int e) { return p.row_tiles_most == 1 ? e : e / p.row_tiles_most; }
  __device__ uint32_t units_of(const AttnParams &p, int e, bool &falls) const {       // of one head
    const int s = seq_of(p, e), rt = e - s * p.row_tiles_most;
    const SeqT seq(p, s);
    falls |= !seq.rises;
    return rt < seq.row_tiles ? seq.units(p, rt) + kCost : 0u;
  }
  __device__ uint32_t units_of(const AttnParams &p, int e) const {
    bool ignored;
    return units_of(p, e, ignored);
  }
  __device__ Work(const AttnParams &p, uint32_t *prefix) : prefix(prefix), falls(false) {
    __shared__ uint32_t warp_sum[32];
    __shared__ int sh_falls;
    __shared__ unsigned long long sh_units;
    if (threadIdx.x == 0) sh_falls = 0;
    entries = p.batch.n_seqs * p.row_tiles_most;
    chunk = chunk_of(entries);
    chunks = (entries + chunk - 1) / chunk;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = (blockDim.x + 31) >> 5;
    uint32_t base = 0;
    for (int c0 = 0; c0 < chunks; c0 += blockDim.x) {
      const int c = c0 + threadIdx.x;
      uint32_t mine = 0;
      for (int e = c * chunk; c < chunks && e < min((c + 1) * chunk, entries); ++e) mine += units_of(p, e, falls) * (uint32_t)p.cache.heads;
      uint32_t x = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (lane == 31) warp_sum[warp] = x;
      __syncthreads();
      uint32_t before = base, all = 0;
      for (int w = 0; w < n_warps; ++w) {
        if (w < warp) before += warp_sum[w];
        all += warp_sum[w];
      }
      if (c < chunks) prefix[c] = before + x - mine;
      base += all;
      __syncthreads();
    }
    if (threadIdx.x == 0) prefix[chunks] = base;
    if (falls) sh_falls = 1;         // a vote of the barrier instead costs half a microsecond
    __syncthreads();
    none = falls = sh_falls;
    if (falls) {
      if (threadIdx.x == 0) sh_units = 0;
      __syncthreads();
      unsigned long long mine = 0;
#pragma unroll 1
      for (int e = threadIdx.x; e < entries; e += blockDim.x) mine += (unsigned long long)units_of(p, e) * (uint32_t)p.cache.heads;
      atomicAdd(&sh_units, mine);
      __syncthreads();
      none = sh_units > p.units_most;
    }
  }
  __device__ uint32_t total() const { return none ? 0u : prefix[chunks]; }
};

// The segment in which unit u < total lies, at or behind `from`.
struct Segment {
  int s, rt, head;
  uint32_t from, begin, units;      // where it begins with its cost; its first unit of tokens, how many of these it has
  template <int kRows, int kUnit, bool kWhole>
  __device__ Segment(const AttnParams &p, const Work<kRows, kUnit, kWhole> &work, uint32_t u) {
    int lo = 0, hi = work.chunks;      // last chunk that begins at or before u
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (work.prefix[mid] <= u) lo = mid;
      else hi = mid;
    }
    int e = lo * work.chunk;
    begin = work.prefix[lo];
    units = work.units_of(p, e);
    while (u - begin >= units * (uint32_t)p.cache.heads) {
      begin += units * (uint32_t)p.cache.heads;
      units = work.units_of(p, ++e);
    }
    s = work.seq_of(p, e);
    rt = e - s * p.row_tiles_most;
    head = (int)((u - begin) / units);
    from = begin + head * units;
    begin = from + Work<kRows, kUnit, kWhole>::kCost;
    units -= Work<kRows, kUnit, kWhole>::kCost;
  }
  // Of the range u .. u_end: the first unit of tokens, from the segment's first, and how many there are; u moves behind them.
  __device__ uint32_t take(uint32_t &u, uint32_t u_end, uint32_t &unit0) const {
    const uint32_t first = max(u, begin), last = min(begin + units, u_end);
    unit0 = first - begin;
    u = last;
    return last > first ? last - first : 0u;
  }
};

__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
  return d;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  if (!kBf16) return f16x2(lo, hi);
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// What cannot be checked before the launch, looked at by one CTA of it.
__device__ __forceinline__ void check_batch(const AttnParams &p) {
  if (p.batch.starts) p.batch.check_starts(p.max_query);
  for (int s = threadIdx.x; s < p.batch.n_seqs; s += blockDim.x)
    if (p.batch.lens[s] < 0 || p.batch.lens[s] > p.batch.length(s, p.cache.block_log2)) p.batch.report(PF_KV8_BAD_LENGTH);
}

__device__ __forceinline__ float lse_of(float base, float sum) { return sum == 0.f ? -INFINITY : (base + log2f(sum)) * kLn2; }

// Lets a kernel have all of the shared memory; asked of the driver once for each device.
template <class Kernel>
void allow_smem(Kernel kernel, std::atomic<uint64_t> &asked, int device) {
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (asked.load(std::memory_order_relaxed) & bit)) return;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 1024) != cudaSuccess)
    throw Error::storage("cudaFuncSetAttribute failed");
  if (device < 64) asked.fetch_or(bit, std::memory_order_relaxed);
}

// Few query rows (kv8_attention_few.cu): tiles of 4, 8, 16 or (not at 256 dimensions) 32
// rows, 0 when there are more.  And the accumulated weights.
int kv8_few_rows(int dim, int64_t rows);
int kv8_few_ctas(int dim, int rows);      // CTAs of an SM
void kv8_few_launch(const AttnParams &p, int rows, bool bf16, cudaStream_t stream);
void kv8_weights_launch(const AttnParams &p, bool bf16, int n_sms, cudaStream_t stream);
// Query rows by the hundred (kv8_attention_wide.cu).
struct WidePlan {
  int rows, tokens;
  size_t smem;
};
WidePlan kv8_wide_plan(int dim);
void kv8_wide_launch(const AttnParams &p, bool bf16, cudaStream_t stream);

}  // namespace pf
