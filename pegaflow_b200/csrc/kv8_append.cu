// Writing tokens into the KV cache held in 8 bits (pf_kv8_append), and the argument checks that all calls on such a
// cache share.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "kv8.h"

namespace pf {

Kv8View kv8_check_cache(const pf_kv8_cache *c) {
  if (!c) throw Error::invalid("null cache");
  const size_t record = pf_kv8_record_bytes(c->block_size, c->kv_heads, c->head_dim);
  if (!record)
    throw Error::invalid(strf("8-bit cache: unsupported geometry block_size=%u kv_heads=%u head_dim=%u", c->block_size,
                              c->kv_heads, c->head_dim));
  if (!c->data_ptr) throw Error::invalid("8-bit cache: data_ptr must not be null");
  if (c->data_ptr % 16 || c->block_stride_bytes % 16 || c->kv_stride_bytes % 16)
    throw Error::invalid("8-bit cache: address and strides must be multiples of 16 bytes");
  if (c->num_blocks == 0 || c->num_blocks > 0x7fffffffu)
    throw Error::invalid(strf("8-bit cache: num_blocks=%zu out of range", c->num_blocks));
  if (c->num_blocks > 1 && c->block_stride_bytes < record)
    throw Error::invalid(strf("8-bit cache: block stride of %zu bytes is below the record's %zu", c->block_stride_bytes, record));
  if (c->num_blocks > 1 && c->block_stride_bytes > 0xffffffffu)
    throw Error::invalid(strf("8-bit cache: block stride of %zu bytes exceeds 4 GiB", c->block_stride_bytes));
  if (c->kv_stride_bytes < record)
    throw Error::invalid(strf("8-bit cache: K/V stride of %zu bytes is below the record's %zu", c->kv_stride_bytes, record));
  Kv8View v{};
  v.base = reinterpret_cast<char *>(c->data_ptr);
  v.block_stride = std::max(c->block_stride_bytes, record);    // of one block it may be anything
  v.kv_stride = c->kv_stride_bytes;
  v.num_blocks = (uint32_t)c->num_blocks;
  v.block_log2 = __builtin_ctz(c->block_size);
  v.heads = (int)c->kv_heads;
  v.dim = (int)c->head_dim;
  return v;
}

Kv8Batch kv8_check_batch(const pf_kv8_batch *b, size_t n_rows) {
  if (!b) throw Error::invalid("null batch");
  if (b->n_seqs > PF_KV8_MAX_SEQS)
    throw Error::invalid(strf("%u sequences exceed the limit of %d", b->n_seqs, PF_KV8_MAX_SEQS));
  if (n_rows > 0x7fffffffu) throw Error::invalid(strf("%zu rows exceed 2^31 - 1", n_rows));
  if (!b->n_seqs && !b->starts && n_rows)
    throw Error::invalid(strf("%zu rows cannot be divided evenly among 0 sequences: row starts are needed", n_rows));
  if (b->n_seqs) {
    if (!b->block_tables || !b->lens) throw Error::invalid("null block_tables or lens");
    if (b->max_blocks == 0 || b->max_blocks > 0x800000u)
      throw Error::invalid(strf("max_blocks=%u out of range", b->max_blocks));
    if (!b->starts && n_rows % b->n_seqs)
      throw Error::invalid(strf("%zu rows cannot be divided evenly among %u sequences: row starts are needed", n_rows, b->n_seqs));
  }
  Kv8Batch v{};
  v.tables = b->block_tables;
  v.table_stride = (int64_t)b->table_stride;
  v.max_blocks = (int)b->max_blocks;
  v.n_seqs = (int)b->n_seqs;
  v.lens = b->lens;
  v.starts = b->starts;
  v.rows_each = b->n_seqs ? (int)(n_rows / b->n_seqs) : 0;
  v.n_rows = (int)n_rows;
  v.status = b->status;
  return v;
}

int kv8_sm_count(int device_id) {
  static std::atomic<int> known[64];
  if (device_id >= 0 && device_id < 64) {
    const int n = known[device_id].load(std::memory_order_relaxed);
    if (n) return n;
  }
  int count = 0, sms = 0;
  cudaError_t e = cudaGetDeviceCount(&count);
  if (e != cudaSuccess) throw Error::cuda_init(cudaGetErrorString(e));
  if (device_id < 0 || device_id >= count)
    throw Error::cuda_init(strf("device %d does not exist (%d devices)", device_id, count));
  e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device_id);
  if (e != cudaSuccess) throw Error::cuda_init(cudaGetErrorString(e));
  if (device_id < 64) known[device_id].store(sms, std::memory_order_relaxed);
  return sms;
}

namespace {

struct AppendSource {
  const uint16_t *ptr[2];
  int64_t row_stride[2], head_stride[2];
};

template <bool kBf16>
__device__ __forceinline__ float2 widen(uint32_t two) {
  if (kBf16) return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
  return f32x2_from_f16x2(two);
}
// Largest finite magnitude of eight elements, as bits of their type: magnitudes order like integers.
template <bool kBf16>
__device__ __forceinline__ uint32_t finite_top(const uint4 &v) {
  constexpr uint32_t kInf = kBf16 ? 0x7f80u : 0x7c00u;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = w[j] & 0x7fff, hi = w[j] >> 16 & 0x7fff;
    top = max(top, max(lo < kInf ? lo : 0u, hi < kInf ? hi : 0u));
  }
  return top;
}

// One warp writes 2048 elements of a tile ((touched block, head, K or V), block_size * head_dim elements; kWarps warps
// hold one tile), eight vectors of eight a lane, in registers: read once, largest magnitude, scale, store.
// It is bound by HBM: 2 bytes read and 1 written for each element.  What it took to come near it: packed 16-bit maxima
// (infinities and NaN are looked at only where one was met), and eight warps to a CTA, because finding the block
// of an item is a chain of four dependent loads that many warps have to share.  8 prompts of 10240 tokens, 8 heads of 128,
// bf16: 87 us, 503 MB at 5.8 TB/s (89% of a copy's rate); one token each of 32 requests 4 us.
//
// Work items: sequence s with n > 0 new rows touches at most n / bs + 2 blocks.  Items f(s) = starts[s] / bs + 2 s
// onwards are its own; f(s + 1) - f(s) >= touched blocks, whatever lens holds, so the grid is sized without reading
// lens and a CTA finds its sequence by bisection.  Surplus items return.
__host__ __device__ constexpr int append_warps(int warps) { return warps < 8 ? 8 : warps; }   // of a CTA

template <bool kBf16, bool kVec, int kWarps>
__global__ void __launch_bounds__(32 * append_warps(kWarps), kWarps > 8 ? 2 : 4) kv8_append_kernel(Kv8View cache, Kv8Batch batch, AppendSource src) {
  constexpr int kTiles = append_warps(kWarps) / kWarps;     // tiles of a CTA
  const int bl = cache.block_log2, bs = 1 << bl, dim_log2 = 31 - __clz(cache.dim);
  const int item = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int which = blockIdx.y * kTiles + warp / kWarps, head = which >> 1, kv = which & 1, part = warp % kWarps;
  after_previous();
  if (batch.starts && item == 0 && blockIdx.y == 0) batch.check_starts(batch.n_rows);
  int lo = 0, hi = batch.n_seqs;   // last s with f(s) <= item
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const int start = batch.starts ? min(max(batch.starts[mid], 0), batch.n_rows) : mid * batch.rows_each;
    if ((start >> bl) + 2 * mid <= item) lo = mid;
    else hi = mid;
  }
  const int seq = lo;
  int row0, row1;
  batch.rows(seq, row0, row1);
  const int n = row1 - row0;
  if (n == 0) return;
  const int index = item - ((row0 >> bl) + 2 * seq);
  const int len_raw = batch.lens[seq];
  const int64_t cap = (int64_t)batch.max_blocks << bl;
  if (len_raw < 0 || len_raw + (int64_t)n > cap) {
    if (threadIdx.x == 0 && index == 0 && blockIdx.y == 0) batch.report(PF_KV8_BAD_LENGTH);
    if (len_raw < 0) return;
  }
  const int64_t len = len_raw;
  const int64_t b = (len >> bl) + index;
  const int64_t tok0 = b << bl;                           // first token of this block
  if (index < 0 || tok0 >= len + n || tok0 >= cap) return;
  uint32_t id;
  if (!batch.block(cache, seq, (int)b, id)) {
    if (threadIdx.x == 0) batch.report(PF_KV8_BAD_BLOCK);
    return;
  }
  const bool mine = head < cache.heads;                                  // the last CTA of an item may have warps to spare
  const int old_rows = (int)max((int64_t)0, len - tok0);                 // rows of the block that were there before
  const int end_row = mine ? (int)min((int64_t)bs, len + n - tok0) : 0;
  const int64_t row_stride = kv ? src.row_stride[1] : src.row_stride[0];
  // a warp's vector i lies 256 elements behind its vector i - 1: some whole rows
  const int row_step = 256 >> dim_log2, first = (part * 8 * 32 + lane) * 8, row_0 = first >> dim_log2;
  const uint16_t *x = (kv ? src.ptr[1] : src.ptr[0]) + head * (kv ? src.head_stride[1] : src.head_stride[0]) +
                      (row0 + (tok0 - len) + row_0) * row_stride + (first & (cache.dim - 1));
  const int64_t step = row_step * row_stride;

  uint4 v[8];
  uint32_t tops = 0;                                                     // of both halves of a pair
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row_0 + i * row_step;
    v[i] = make_uint4(0, 0, 0, 0);
    if (row >= old_rows && row < end_row) {
      const uint16_t *p = x + i * step;
      if (kVec) v[i] = __ldg(reinterpret_cast<const uint4 *>(p));
      else v[i] = make_uint4(p[0] | p[1] << 16, p[2] | p[3] << 16, p[4] | p[5] << 16, p[6] | p[7] << 16);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = __vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu), c = __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu);
    tops = __vmaxu2(tops, __vmaxu2(a, c));
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, max(tops & 0xffff, tops >> 16));
  if (top >= (kBf16 ? 0x7f80u : 0x7c00u)) {                              // an infinity or a NaN
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, finite_top<kBf16>(v[i]));
    top = __reduce_max_sync(0xffffffffu, top);
  }
  uint8_t *tile = cache.tile(kv, id, mine ? head : 0);
  float *scale_ptr = cache.scale(kv, id, mine ? head : 0);
  const int e_old = old_rows ? kv8_scale_exponent(*scale_ptr) : kKv8MinExp;
  if (kWarps > 1) {                          // every warp has read the old scale before one writes the new
    __shared__ uint32_t sh_top[append_warps(kWarps)];
    if (lane == 0) sh_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max(top, sh_top[warp / kWarps * kWarps + w]);
  }
  __syncwarp();
  if (!mine) return;
  const int e = max(e_old, kv8_exponent(__float_as_uint(widen<kBf16>(top).x)));
  const float inv = exp2i(-e), old_factor = exp2i(e_old - e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row_0 + i * row_step;
    uint2 *out = reinterpret_cast<uint2 *>(tile + first + 256 * i);
    if (row >= old_rows && row < end_row) {
      const float2 a = widen<kBf16>(v[i].x), c = widen<kBf16>(v[i].y), d = widen<kBf16>(v[i].z), f = widen<kBf16>(v[i].w);
      *out = make_uint2(e4m3x4(a.x * inv, a.y * inv, c.x * inv, c.y * inv), e4m3x4(d.x * inv, d.y * inv, f.x * inv, f.y * inv));
    } else if (row < old_rows && e > e_old) {
      const uint2 was = *out;
      const float2 a = f32x2_from_f16x2(f16x2_from_e4m3<0>(was.x)), c = f32x2_from_f16x2(f16x2_from_e4m3<1>(was.x));
      const float2 d = f32x2_from_f16x2(f16x2_from_e4m3<0>(was.y)), f = f32x2_from_f16x2(f16x2_from_e4m3<1>(was.y));
      const float r = old_factor;
      *out = make_uint2(e4m3x4(a.x * r, a.y * r, c.x * r, c.y * r), e4m3x4(d.x * r, d.y * r, f.x * r, f.y * r));
    }
  }
  if (lane == 0 && part == 0) *scale_ptr = exp2i(e);
}

template <bool kBf16, bool kVec>
void launch_append(const Kv8View &c, const Kv8Batch &b, const AppendSource &src, unsigned items, cudaStream_t s) {
  const int warps = std::max(1, (int)(c.tile_bytes() / 2048));      // of a tile: 1, 2, 4, 8 or 16
  auto go = [&](auto kernel, int tile_warps) {
    const int tiles = append_warps(tile_warps) / tile_warps;
    launch_after(kernel, dim3(items, (2 * c.heads + tiles - 1) / tiles), 32 * append_warps(tile_warps), 0, s, c, b, src);
  };
  switch (warps) {
    case 1: return go(kv8_append_kernel<kBf16, kVec, 1>, 1);
    case 2: return go(kv8_append_kernel<kBf16, kVec, 2>, 2);
    case 4: return go(kv8_append_kernel<kBf16, kVec, 4>, 4);
    case 8: return go(kv8_append_kernel<kBf16, kVec, 8>, 8);
    default: return go(kv8_append_kernel<kBf16, kVec, 16>, 16);
  }
}

}  // namespace
}  // namespace pf

using namespace pf;

extern "C" {

size_t pf_kv8_record_bytes(uint32_t block_size, uint32_t kv_heads, uint32_t head_dim) {
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128) return 0;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
  if (kv_heads == 0 || kv_heads > 1024) return 0;
  return (size_t)kv_heads * block_size * head_dim + (4 * (size_t)kv_heads + 15) / 16 * 16;
}

int pf_kv8_append(int device_id, const pf_kv8_cache *cache, const pf_kv8_batch *batch, const void *k, const void *v,
                  int dtype, size_t n_rows, size_t k_row_stride, size_t k_head_stride, size_t v_row_stride,
                  size_t v_head_stride, void *stream) {
  return guarded([&] {
    const Kv8View c = kv8_check_cache(cache);
    const Kv8Batch b = kv8_check_batch(batch, n_rows);
    if (dtype != PF_KV8_BF16 && dtype != PF_KV8_F16) throw Error::invalid(strf("unknown dtype %d", dtype));
    if (n_rows == 0 || b.n_seqs == 0) return;
    if (!k || !v) throw Error::invalid("null k or v");
    if ((uintptr_t)k % 2 || (uintptr_t)v % 2) throw Error::invalid("k and v must be aligned to their elements");
    AppendSource src{{(const uint16_t *)k, (const uint16_t *)v},
                     {(int64_t)k_row_stride, (int64_t)v_row_stride},
                     {(int64_t)k_head_stride, (int64_t)v_head_stride}};
    const bool vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 &&
                     (k_row_stride | k_head_stride | v_row_stride | v_head_stride) % 8 == 0;
    const size_t items = (n_rows >> c.block_log2) + 2 * (size_t)b.n_seqs;
    kv8_sm_count(device_id);
    DeviceGuard on_device(device_id);
    cudaStream_t s = (cudaStream_t)stream;
    const bool bf16 = dtype == PF_KV8_BF16;
    if (bf16) vec ? launch_append<true, true>(c, b, src, (unsigned)items, s) : launch_append<true, false>(c, b, src, (unsigned)items, s);
    else vec ? launch_append<false, true>(c, b, src, (unsigned)items, s) : launch_append<false, false>(c, b, src, (unsigned)items, s);
  });
}

}  // extern "C"
