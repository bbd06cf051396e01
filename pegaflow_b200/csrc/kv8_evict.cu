// Eviction from the KV cache held in 8 bits by accumulated attention weight (pf_kv8_evict): choose, then copy.
#include <cuda_fp16.h>

#include <algorithm>

#include "kv8.h"

namespace pf {
namespace {

constexpr int kSelectThreads = 1024;

struct EvictParams {
  Kv8View cache;
  Kv8Batch batch;
  const float *weights;
  int64_t w_seq, w_head;
  int w_capacity;
  const int32_t *dst_tables;
  int64_t dst_stride;
  int keep, recent, n_dst;
  int32_t *new_lens;
  float *new_weights;
  int64_t new_capacity;
  int32_t *kept;

  __device__ int length(int s) const { return min(batch.length(s, cache.block_log2), w_capacity); }
};

// Weights as integers of the same order; a NaN is the least, -0 equals +0.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Adds one to hist[bin] for every lane whose bin is not kNoBin.  Weights crowd (tokens that were never looked at all
// weigh 0): lanes of one bin add together.
constexpr uint32_t kNoBin = 0xffffffffu;
__device__ __forceinline__ void count(uint32_t *hist, uint32_t bin) {
  const uint32_t same = __match_any_sync(0xffffffffu, bin);
  if (bin != kNoBin && (same & ((1u << (threadIdx.x & 31)) - 1)) == 0) atomicAdd(hist + bin, (uint32_t)__popc(same));
}

// One CTA chooses for one (sequence, head).  The weight of the last token kept is found digit by digit (histograms of 11,
// 11 and 10 bits over the keys that agree so far); then one pass writes what lies above it and, of the equal ones, as
// many as are missing, in the tokens' order: a token's place is the number of larger ones before it plus the number
// of equal ones before it that were still taken.  Keys stay in registers up to kKeys * 1024 tokens.  Bound by the chain of
// its block-wide steps: 24 us for 128 rows of 10240 weights, 7.5 us for 8 of 1500.
constexpr int kKeys = 12;
__global__ void __launch_bounds__(kSelectThreads) kv8_select_kernel(EvictParams p) {
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t sh_prefix, sh_left;
  __shared__ uint32_t warp_total[32];
  __shared__ uint2 warp_sum[2][32];
  const int s = blockIdx.x / p.cache.heads, head = blockIdx.x % p.cache.heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  after_previous();
  const int n = p.length(s);
  if (head == 0 && tid == 0) {
    if (p.batch.lens[s] != n) p.batch.report(PF_KV8_BAD_LENGTH);
    p.new_lens[s] = min(n, p.keep);
  }
  const float *w = p.weights + s * p.w_seq + head * p.w_head;
  const int recent = min(p.recent, n), m = min(n, p.keep), candidates = n - recent, need = m - recent;
  const int rounds = (candidates + kSelectThreads - 1) / kSelectThreads;
  const bool held = rounds <= kKeys;
  float mine[kKeys];
  if (held) {
#pragma unroll
    for (int i = 0; i < kKeys; ++i) mine[i] = i * kSelectThreads + tid < candidates ? w[i * kSelectThreads + tid] : 0.f;
  }
  uint32_t bar = 0, ties = candidates;     // keep all
  if (need == 0) {
    bar = 0xffffffffu, ties = 0;
  } else if (need < candidates) {
    uint32_t prefix = 0, left = need;      // keys that agree with prefix so far, and how many of them are kept
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
      const uint32_t mask = digit == 0 ? 0u : 0xffffffffu << (shift + bits);
      hist[tid] = hist[tid + 1024] = 0;
      __syncthreads();
      auto bin_of = [&](int j, float x) {
        const uint32_t key = order_key(x);
        return j < candidates && (key & mask) == prefix ? key >> shift & ((1u << bits) - 1) : kNoBin;
      };
      if (held) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
          if (i < rounds) count(hist, bin_of(i * kSelectThreads + tid, mine[i]));
      } else {
        for (int i = 0; i < rounds; ++i) {
          const int j = i * kSelectThreads + tid;
          count(hist, bin_of(j, j < candidates ? w[j] : 0.f));
        }
      }
      __syncthreads();
      // the bin in which the left-th largest lies: thread t holds the t-th pair of bins from the top
      const uint32_t upper = hist[2047 - 2 * tid], lower = hist[2046 - 2 * tid];
      uint32_t x = upper + lower;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (lane == 31) warp_total[warp] = x;
      __syncthreads();
      uint32_t y = lane < warp ? warp_total[lane] : 0u;
      y = __reduce_add_sync(0xffffffffu, y);
      const uint32_t before = y + x - upper - lower;
      if (before < left && left <= before + upper + lower) {
        const bool first = left <= before + upper;
        sh_prefix = prefix | (uint32_t)(first ? 2047 - 2 * tid : 2046 - 2 * tid) << shift;
        sh_left = left - before - (first ? 0u : upper);
      }
      __syncthreads();
      prefix = sh_prefix, left = sh_left;
    }
    bar = prefix, ties = left;
  }
  int32_t *kept = p.kept + ((int64_t)s * p.cache.heads + head) * p.keep;
  float *out = p.new_weights + ((int64_t)s * p.cache.heads + head) * p.new_capacity;
  uint32_t above = 0, equal = 0;           // taken in by the rounds before
  auto place = [&](int i, float x) {
    const int j = i * kSelectThreads + tid;
    const uint32_t key = order_key(x);
    const bool gt = j < candidates && key > bar, eq = j < candidates && key == bar;
    const uint32_t gts = __ballot_sync(0xffffffffu, gt), eqs = __ballot_sync(0xffffffffu, eq), below = (1u << lane) - 1;
    uint2 *sums = warp_sum[i & 1];
    if (lane == 0) sums[warp] = make_uint2(__popc(gts), __popc(eqs));
    __syncthreads();
    const uint2 of = sums[lane];
    const uint32_t g = above + __reduce_add_sync(0xffffffffu, lane < warp ? of.x : 0u) + __popc(gts & below);
    const uint32_t e = equal + __reduce_add_sync(0xffffffffu, lane < warp ? of.y : 0u) + __popc(eqs & below);
    above += __reduce_add_sync(0xffffffffu, of.x);
    equal += __reduce_add_sync(0xffffffffu, of.y);
    if (gt || (eq && e < ties)) {
      const uint32_t at = g + min(e, ties);
      kept[at] = j;
      out[at] = x;
    }
  };
  if (held) {
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
      if (i < rounds) place(i, mine[i]);
  } else {
    for (int i = 0; i < rounds; ++i) place(i, i * kSelectThreads + tid < candidates ? w[i * kSelectThreads + tid] : 0.f);
  }
  for (int i = tid; i < recent; i += kSelectThreads) {
    kept[need + i] = candidates + i;
    out[need + i] = w[candidates + i];
  }
  for (int64_t i = m + tid; i < p.new_capacity; i += kSelectThreads) out[i] = 0.f;
  for (int i = m + tid; i < p.keep; i += kSelectThreads) kept[i] = -1;
}

__device__ __forceinline__ __half2 half2_of(uint32_t x) { return *reinterpret_cast<__half2 *>(&x); }

// kWarps warps make one new block of one head, K and V: a warp 2048 bytes of each, in registers.  Lane r finds where the
// warp's r-th row lies (three dependent loads, once for K and V); rows are then read 16 bytes a lane.  Where
// every row comes from a block of the scale that the new block gets, which is the common case, bytes are copied as they
// are; otherwise they are multiplied as f16, which is exact down to 2^-24 while e4m3 ends at 2^-9.
// Bound by memory, through the latency of those loads: 64 registers a thread, so that 32 warps share an SM.  16 sequences of
// 10240 tokens shortened to 4096, 8 heads of 128 (the choice included): 80 us; at 80 registers 83 us; at 128 registers, with
// the largest value looked for in converted numbers, 98 us; a warp for K and one for V 108 us.
template <int kWarps>
__global__ void __launch_bounds__(32 * (kWarps < 8 ? 8 : kWarps), kWarps < 16 ? 4 : 2) kv8_gather_kernel(EvictParams p) {
  constexpr int kCta = kWarps < 8 ? 8 : kWarps, kTiles = kCta / kWarps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % kWarps;
  const int64_t tile = (int64_t)blockIdx.x * kTiles + warp / kWarps;
  const int b = (int)(tile % p.n_dst), sh = (int)(tile / p.n_dst), s = sh / p.cache.heads, head = sh % p.cache.heads;
  const int bl = p.cache.block_log2, dim = p.cache.dim, dim_log2 = 31 - __clz(dim);
  const int row_first = part * (2048 >> dim_log2), rows_held = min(2048 >> dim_log2, 1 << bl);
  after_previous();
  const bool mine = s < p.batch.n_seqs;
  const int m = mine ? min(p.length(s), p.keep) : 0, rows = min(m - (b << bl), 1 << bl);
  // where row `lane` of this warp's share lies, and where the block goes
  const bool has = lane < rows_held && row_first + lane < rows;
  const int j = has ? p.kept[(int64_t)sh * p.keep + (b << bl) + row_first + lane] : 0;
  const uint32_t id = rows > 0 ? (uint32_t)p.dst_tables[s * p.dst_stride + b] : 0xffffffffu;
  uint32_t src = 0;
  int at = 0, e_k = kKv8MinExp, e_v = kKv8MinExp;
  bool there = false;
  if (has) {
    there = p.batch.block(p.cache, s, j >> bl, src);
    if (there) {
      at = j & ((1 << bl) - 1);
      e_k = kv8_scale_exponent(__ldg(p.cache.scale(0, src, head)));
      e_v = kv8_scale_exponent(__ldg(p.cache.scale(1, src, head)));
    } else {
      p.batch.report(PF_KV8_BAD_BLOCK);
    }
  }
  const bool write = id < p.cache.num_blocks;
  if (rows > 0 && !write && lane == 0) p.batch.report(PF_KV8_BAD_BLOCK);
  uint4 x[2][4];
  int e_row[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int el = (i * 32 + lane) * 16, row = el >> dim_log2, col = el & (dim - 1);
    const uint32_t from = __shfl_sync(0xffffffffu, src, row & 31);
    const int r = __shfl_sync(0xffffffffu, at, row & 31);
    const bool live = __shfl_sync(0xffffffffu, (int)there, row & 31) && row < rows_held;
    e_row[0][i] = __shfl_sync(0xffffffffu, e_k, row & 31);
    e_row[1][i] = __shfl_sync(0xffffffffu, e_v, row & 31);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
      x[kv][i] = live ? __ldg(reinterpret_cast<const uint4 *>(p.cache.tile(kv, from, head) + r * dim + col)) : make_uint4(0, 0, 0, 0);
  }
  __shared__ uint32_t sh_top[2][kCta];
  uint32_t top[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // magnitudes of e4m3 are ordered like their bits
      const uint32_t w[4] = {x[kv][i].x, x[kv][i].y, x[kv][i].z, x[kv][i].w};
      uint32_t even = 0, odd = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        even = __vmaxu2(even, w[k] & 0x007f007fu);
        odd = __vmaxu2(odd, w[k] >> 8 & 0x007f007fu);
      }
      even = __vmaxu2(even, odd);
      uint32_t most = max(even & 0xffff, even >> 16);
      if (most == 0x7f) {       // a NaN among them does not count
        most = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int b8 = 0; b8 < 32; b8 += 8) {
            const uint32_t m = w[k] >> b8 & 0x7f;
            if (m != 0x7f) most = max(most, m);
          }
      }
      t = max(t, __float_as_uint(__low2float(half2_of(f16x2_from_e4m3<0>(most))) * exp2i(e_row[kv][i])));
    }
    top[kv] = __reduce_max_sync(0xffffffffu, t);
    if (kWarps > 1 && lane == 0) sh_top[kv][warp] = top[kv];
  }
  if (kWarps > 1) {
    __syncthreads();
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
      for (int k = 0; k < kWarps; ++k) top[kv] = max(top[kv], sh_top[kv][warp / kWarps * kWarps + k]);
  }
  if (!write) return;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const int e = kv8_exponent(top[kv]);
    uint8_t *dst = p.cache.tile(kv, id, head) + part * 2048;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int el = (i * 32 + lane) * 16, row = el >> dim_log2;
      const int d = e_row[kv][i] - e;
      uint4 y = x[kv][i];
      if (d != 0) {
        // what is left of a factor above 2^15 goes on as a second one: only zeros and the smallest values need it
        const int d1 = min(max(d, -24), 15), d2 = min(max(d - d1, 0), 15);
        const __half2 f1 = __float2half2_rn(exp2i(d1)), f2 = __float2half2_rn(exp2i(d2));
        uint32_t *w = &y.x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t a = f16x2_from_e4m3<0>(w[k]), c = f16x2_from_e4m3<1>(w[k]);
          __half2 ha = __hmul2(*reinterpret_cast<__half2 *>(&a), f1), hc = __hmul2(*reinterpret_cast<__half2 *>(&c), f1);
          if (d2) ha = __hmul2(ha, f2), hc = __hmul2(hc, f2);
          w[k] = e4m3x4_from_f16(*reinterpret_cast<uint32_t *>(&ha), *reinterpret_cast<uint32_t *>(&hc));
        }
      }
      if (row < rows_held && row_first + row < rows) *reinterpret_cast<uint4 *>(dst + el) = y;
    }
    if (lane == 0 && part == 0) *p.cache.scale(kv, id, head) = exp2i(e);
  }
}

}  // namespace
}  // namespace pf

using namespace pf;

extern "C" int pf_kv8_evict(int device_id, const pf_kv8_cache *cache, const pf_kv8_batch *batch,
                            const pf_kv8_evict_args *args, void *stream) {
  return guarded([&] {
    const Kv8View c = kv8_check_cache(cache);
    const Kv8Batch b = kv8_check_batch(batch, 0);
    if (!args) throw Error::invalid("null eviction arguments");
    const pf_kv8_evict_args &a = *args;
    if (b.n_seqs == 0) return;
    if (a.keep == 0 || a.keep > 0x7fffffffu - 128) throw Error::invalid(strf("keep=%zu out of range", a.keep));
    if (a.recent > a.keep) throw Error::invalid(strf("recent=%zu exceeds keep=%zu", a.recent, a.keep));
    if (a.new_capacity < a.keep)
      throw Error::invalid(strf("new_capacity=%zu is below keep=%zu", a.new_capacity, a.keep));
    if (!a.weights || !a.dst_tables || !a.new_lens || !a.new_weights || !a.kept) throw Error::invalid("null eviction array");
    if (a.new_weights == a.weights) throw Error::invalid("new_weights must not be weights");
    if (a.dst_tables == b.tables) throw Error::invalid("the destination's blocks must not be the source's");
    EvictParams p{};
    p.cache = c;
    p.batch = b;
    p.weights = a.weights;
    p.w_seq = (int64_t)a.weights_seq_stride, p.w_head = (int64_t)a.weights_head_stride;
    p.w_capacity = (int)std::min<size_t>(a.weights_capacity, 0x7fffffff);
    p.dst_tables = a.dst_tables;
    p.dst_stride = (int64_t)a.dst_table_stride;
    p.keep = (int)a.keep, p.recent = (int)a.recent;
    p.n_dst = (int)((a.keep + (1 << c.block_log2) - 1) >> c.block_log2);
    p.new_lens = a.new_lens, p.new_weights = a.new_weights, p.new_capacity = (int64_t)a.new_capacity, p.kept = a.kept;
    if (b.n_seqs > 1 && a.dst_table_stride < (size_t)p.n_dst) throw Error::invalid("rows of dst_tables overlap: every sequence needs blocks of its own");
    const uint64_t tiles = (uint64_t)b.n_seqs * c.heads * p.n_dst;
    if (tiles > 0x7fffffffu) throw Error::invalid("too many blocks for one call: split the batch");
    kv8_sm_count(device_id);
    DeviceGuard on_device(device_id);
    cudaStream_t s = (cudaStream_t)stream;
    launch_after(kv8_select_kernel, b.n_seqs * c.heads, kSelectThreads, 0, s, p);
    auto gather = [&](auto kernel, int warps) {
      const int cta = std::max(8, warps), at_once = cta / warps;
      launch_after(kernel, (unsigned)((tiles + at_once - 1) / at_once), 32 * cta, 0, s, p);
    };
    switch (std::max(1, (int)(c.tile_bytes() / 2048))) {
      case 1: gather(kv8_gather_kernel<1>, 1); break;
      case 2: gather(kv8_gather_kernel<2>, 2); break;
      case 4: gather(kv8_gather_kernel<4>, 4); break;
      case 8: gather(kv8_gather_kernel<8>, 8); break;
      default: gather(kv8_gather_kernel<16>, 16); break;
    }
  });
}
