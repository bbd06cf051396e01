// Writing tokens into the KV cache held in 8 bits (pf_kv8_append), and the argument checks that all calls on such a
// cache share.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
  if (c->kv_stride_bytes < record)
    throw Error::invalid(strf("8-bit cache: K/V stride of %zu bytes is below the record's %zu", c->kv_stride_bytes, record));
  Kv8View v{};
  v.base = reinterpret_cast<char *>(c->data_ptr);
  v.block_stride = c->block_stride_bytes;
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

// One CTA writes one (touched block, head, K or V): block_size * head_dim / 32 threads, each with four vectors of
// eight elements in registers, so that the rows are read once: largest magnitude, then scale, then store.
//
// Work items: sequence s with n > 0 new rows touches at most n / bs + 2 blocks.  Items f(s) = starts[s] / bs + 2 s
// onwards are its own; f(s + 1) - f(s) >= touched blocks, whatever lens holds, so the grid is sized without reading
// lens and a CTA finds its sequence by bisection.  Surplus items return.
template <bool kBf16, bool kVec>
__global__ void __launch_bounds__(1024) kv8_append_kernel(Kv8View cache, Kv8Batch batch, AppendSource src) {
  const int bl = cache.block_log2, bs = 1 << bl;
  const int item = blockIdx.x, head = blockIdx.y, kv = blockIdx.z;
  if (batch.starts && item == 0 && head == 0 && kv == 0) batch.check_starts(batch.n_rows);
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
  const bool reporter = threadIdx.x == 0 && index == 0 && head == 0 && kv == 0;
  if (len_raw < 0 || len_raw + (int64_t)n > cap) {
    if (reporter) batch.report(PF_KV8_BAD_LENGTH);
    if (len_raw < 0) return;
  }
  const int64_t len = len_raw;
  const int64_t first_block = len >> bl;
  const int64_t b = first_block + index;
  const int64_t tok0 = b << bl;                           // first token of this block
  if (index < 0 || tok0 >= len + n || tok0 >= cap) return;
  uint32_t id;
  if (!batch.block(cache, seq, (int)b, id)) {
    if (threadIdx.x == 0) batch.report(PF_KV8_BAD_BLOCK);
    return;
  }
  const int old_rows = (int)max((int64_t)0, len - tok0);                 // rows of the block that were there before
  const int end_row = (int)min((int64_t)bs, len + n - tok0);
  const uint16_t *x = src.ptr[kv] + head * src.head_stride[kv] + (row0 + (tok0 - len)) * src.row_stride[kv];
  uint8_t *tile = cache.tile(kv, id, head);
  float *scale_ptr = cache.scale(kv, id, head);
  const int T = blockDim.x, dim = cache.dim;

  uint4 v[4];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = (i * T + (int)threadIdx.x) * 8, row = e / dim, col = e % dim;
    v[i] = make_uint4(0, 0, 0, 0);
    if (row >= old_rows && row < end_row) {
      const uint16_t *p = x + row * src.row_stride[kv] + col;
      if (kVec) {
        v[i] = *reinterpret_cast<const uint4 *>(p);
      } else {
        v[i] = make_uint4(p[0] | p[1] << 16, p[2] | p[3] << 16, p[4] | p[5] << 16, p[6] | p[7] << 16);
      }
    }
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = widen<kBf16>(w[j]);
      top = max(top, max(kv8_magnitude(f.x), kv8_magnitude(f.y)));
    }
  }
  __shared__ uint32_t tops[32];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  const int e_old = old_rows ? kv8_scale_exponent(*scale_ptr) : kKv8MinExp;   // read before the barrier, written behind it
  __syncthreads();
  for (int w = 0; w < T / 32; ++w) top = max(top, tops[w]);
  const int e = max(e_old, kv8_exponent(top));
  const float inv = exp2i(-e), old_factor = exp2i(e_old - e);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int el = (i * T + (int)threadIdx.x) * 8, row = el / dim;
    uint2 *out = reinterpret_cast<uint2 *>(tile + el);
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
  if (threadIdx.x == 0) *scale_ptr = exp2i(e);
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
    const dim3 grid((unsigned)items, c.heads, 2);
    const int threads = (int)(c.tile_bytes() / 32);
    DeviceGuard on_device(device_id);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == PF_KV8_BF16) {
      if (vec) kv8_append_kernel<true, true><<<grid, threads, 0, s>>>(c, b, src);
      else kv8_append_kernel<true, false><<<grid, threads, 0, s>>>(c, b, src);
    } else {
      if (vec) kv8_append_kernel<false, true><<<grid, threads, 0, s>>>(c, b, src);
      else kv8_append_kernel<false, false><<<grid, threads, 0, s>>>(c, b, src);
    }
    PF_KV8_LAUNCHED();
  });
}

}  // extern "C"
