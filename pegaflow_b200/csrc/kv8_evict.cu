// Eviction from the KV cache held in 8 bits by accumulated attention weight (pf_kv8_evict): choose, then copy.
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

// One CTA chooses for one (sequence, head).  The weight of the last token kept is found digit by digit (four
// histograms of 256 bins over the keys that agree so far); then one pass writes what lies above it and, of the equal
// ones, as many as are missing, in the tokens' order: a token's place is the number of larger ones before it plus
// the number of equal ones before it that were still taken.
__global__ void __launch_bounds__(kSelectThreads) kv8_select_kernel(EvictParams p) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t sh_prefix, sh_left;
  __shared__ uint2 warp_sum[32];
  const int s = blockIdx.x / p.cache.heads, head = blockIdx.x % p.cache.heads, tid = threadIdx.x;
  const int n = p.length(s);
  if (head == 0 && tid == 0) {
    if (p.batch.lens[s] != n) p.batch.report(PF_KV8_BAD_LENGTH);
    p.new_lens[s] = min(n, p.keep);
  }
  const float *w = p.weights + s * p.w_seq + head * p.w_head;
  const int recent = min(p.recent, n), m = min(n, p.keep), candidates = n - recent, need = m - recent;
  uint32_t bar = 0, ties = candidates;     // keep all
  if (need == 0) {
    bar = 0xffffffffu, ties = 0;
  } else if (need < candidates) {
    uint32_t prefix = 0, left = need;      // keys that agree with prefix so far, and how many of them are kept
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int j = tid; j < candidates; j += kSelectThreads) {
        const uint32_t key = order_key(w[j]);
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid < 32) {      // digit in which the left-th largest lies: lane l sums bins 8 l .. 8 l + 7 from the top
        uint32_t mine = 0;
        for (int k = 0; k < 8; ++k) mine += hist[255 - (8 * tid + k)];
        uint32_t before = mine;
        for (int d = 1; d < 32; d <<= 1) {
          const uint32_t y = __shfl_up_sync(0xffffffffu, before, d);
          if (tid >= d) before += y;
        }
        before -= mine;
        if (before < left && before + mine >= left) {
          for (int k = 0; k < 8; ++k) {
            const uint32_t h = hist[255 - (8 * tid + k)];
            if (before + h >= left) {
              sh_prefix = prefix | (uint32_t)(255 - (8 * tid + k)) << shift;
              sh_left = left - before;
              break;
            }
            before += h;
          }
        }
      }
      __syncthreads();
      prefix = sh_prefix, left = sh_left;
    }
    bar = prefix, ties = left;
  }
  int32_t *kept = p.kept + ((int64_t)s * p.cache.heads + head) * p.keep;
  float *out = p.new_weights + ((int64_t)s * p.cache.heads + head) * p.new_capacity;
  uint32_t above = 0, equal = 0;           // taken in by the tiles before
  const int lane = tid & 31, warp = tid >> 5;
  for (int j0 = 0; j0 < candidates; j0 += kSelectThreads) {
    const int j = j0 + tid;
    const float x = j < candidates ? w[j] : 0.f;
    const uint32_t key = order_key(x);
    const bool gt = j < candidates && key > bar, eq = j < candidates && key == bar;
    const uint32_t gts = __ballot_sync(0xffffffffu, gt), eqs = __ballot_sync(0xffffffffu, eq), below = (1u << lane) - 1;
    if (lane == 0) warp_sum[warp] = make_uint2(__popc(gts), __popc(eqs));
    __syncthreads();
    uint32_t g = above + __popc(gts & below), e = equal + __popc(eqs & below);
    for (int k = 0; k < kSelectThreads / 32; ++k) {
      const uint2 y = warp_sum[k];
      if (k < warp) g += y.x, e += y.y;
      above += y.x, equal += y.y;
    }
    if (gt || (eq && e < ties)) {
      const uint32_t at = g + min(e, ties);
      kept[at] = j;
      out[at] = x;
    }
    __syncthreads();
  }
  for (int i = tid; i < recent; i += kSelectThreads) {
    kept[need + i] = candidates + i;
    out[need + i] = w[candidates + i];
  }
  for (int64_t i = m + tid; i < p.new_capacity; i += kSelectThreads) out[i] = 0.f;
  for (int i = m + tid; i < p.keep; i += kSelectThreads) kept[i] = -1;
}

// One CTA makes one new (block, head, K or V): block_size * head_dim / 32 threads, each with four vectors of eight
// values in registers: gathered, their largest magnitude found, scaled anew, stored.
__global__ void __launch_bounds__(1024) kv8_gather_kernel(EvictParams p) {
  const int kv = blockIdx.x & 1, b = (blockIdx.x >> 1) % p.n_dst, sh = (blockIdx.x >> 1) / p.n_dst;
  const int s = sh / p.cache.heads, head = sh % p.cache.heads;
  const int bl = p.cache.block_log2, dim = p.cache.dim, T = blockDim.x;
  const int m = min(p.length(s), p.keep), rows = min(m - (b << bl), 1 << bl);
  if (rows <= 0) return;
  const uint32_t id = (uint32_t)p.dst_tables[s * p.dst_stride + b];
  if (id >= p.cache.num_blocks) {
    if (threadIdx.x == 0) p.batch.report(PF_KV8_BAD_BLOCK);
    return;
  }
  const int32_t *kept = p.kept + (int64_t)sh * p.keep + (b << bl);
  float2 x[4][4];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = (i * T + (int)threadIdx.x) * 8, row = e / dim, col = e % dim;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[i][k] = make_float2(0.f, 0.f);
    if (row < rows) {
      const int j = kept[row];
      uint32_t src;
      if (p.batch.block(p.cache, s, j >> bl, src)) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p.cache.tile(kv, src, head) + (j & ((1 << bl) - 1)) * dim + col);
        const float f = *p.cache.scale(kv, src, head);
        x[i][0] = f32x2_from_f16x2(f16x2_from_e4m3<0>(v.x)), x[i][1] = f32x2_from_f16x2(f16x2_from_e4m3<1>(v.x));
        x[i][2] = f32x2_from_f16x2(f16x2_from_e4m3<0>(v.y)), x[i][3] = f32x2_from_f16x2(f16x2_from_e4m3<1>(v.y));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[i][k].x *= f, x[i][k].y *= f;
          top = max(top, max(kv8_magnitude(x[i][k].x), kv8_magnitude(x[i][k].y)));
        }
      } else {
        p.batch.report(PF_KV8_BAD_BLOCK);
      }
    }
  }
  __shared__ uint32_t tops[32];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < T / 32; ++w) top = max(top, tops[w]);
  const int e = kv8_exponent(top);
  const float inv = exp2i(-e);
  uint8_t *tile = p.cache.tile(kv, id, head);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int el = (i * T + (int)threadIdx.x) * 8;
    if (el / dim < rows)
      *reinterpret_cast<uint2 *>(tile + el) =
          make_uint2(e4m3x4(x[i][0].x * inv, x[i][0].y * inv, x[i][1].x * inv, x[i][1].y * inv),
                     e4m3x4(x[i][2].x * inv, x[i][2].y * inv, x[i][3].x * inv, x[i][3].y * inv));
  }
  if (threadIdx.x == 0) *p.cache.scale(kv, id, head) = exp2i(e);
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
    const uint64_t tiles = (uint64_t)b.n_seqs * c.heads * p.n_dst * 2;
    if (tiles > 0x7fffffffu) throw Error::invalid("too many blocks for one call: split the batch");
    kv8_sm_count(device_id);
    DeviceGuard on_device(device_id);
    cudaStream_t s = (cudaStream_t)stream;
    kv8_select_kernel<<<b.n_seqs * c.heads, kSelectThreads, 0, s>>>(p);
    PF_KV8_LAUNCHED();
    kv8_gather_kernel<<<(unsigned)tiles, (int)(c.tile_bytes() / 32), 0, s>>>(p);
    PF_KV8_LAUNCHED();
  });
}
