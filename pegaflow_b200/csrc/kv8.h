// The KV cache held in 8 bits: record layout and the device helpers its kernels share.
//
// A record is one block of K or of V of one layer:
//   kv_heads x block_size x head_dim e4m3 values (head-major, so that a head's rows of a block are one
//   contiguous tile), then kv_heads fp32 scales, padded to 16 bytes.
// The cache is [2 (K, V)][num_blocks] records at any strides, which is what the engine registers as a layer of two
// segments: save, load and peer copy move a block together with its scales.
//
// Scales are powers of two, 2^e with e the least integer that brings the tile's largest magnitude within e4m3's 448.
// e4m3 is a floating-point format: a finer scale would not save a mantissa bit, and a power of two makes every
// change of scale exact but for values that fall below 2^-6 of the new one (e4m3's subnormals).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "common.h"
#include "transfer.h"

namespace pf {

// 2^e, 1 / 2^e and their products with e4m3 values stay normal, but for one thing: with e = 120, which only magnitudes above
// 1.75 * 2^127 (2.97e38) ask for, values of 256 and more stand for numbers beyond fp32, which reads them as infinities.
constexpr int kKv8MinExp = -110, kKv8MaxExp = 120;

struct Kv8View {
  char *base;
  uint64_t block_stride, kv_stride;
  uint32_t num_blocks;
  int block_log2, heads, dim;

  __host__ __device__ int block_size() const { return 1 << block_log2; }
  __host__ __device__ uint64_t tile_bytes() const { return (uint64_t)dim << block_log2; }
  __device__ char *record(int kv, uint32_t block) const { return base + kv * kv_stride + block * block_stride; }
  __device__ uint8_t *tile(int kv, uint32_t block, int head) const {
    return reinterpret_cast<uint8_t *>(record(kv, block) + head * tile_bytes());
  }
  __device__ float *scale(int kv, uint32_t block, int head) const {
    return reinterpret_cast<float *>(record(kv, block) + heads * tile_bytes()) + head;
  }
};

// The sequences of one call: block tables, lengths, and where each one's rows start (null: n_rows / n_seqs each).
struct Kv8Batch {
  const int32_t *tables;
  int64_t table_stride;
  int max_blocks, n_seqs;
  const int32_t *lens, *starts;
  int rows_each;       // rows of every sequence when starts is null
  int n_rows;          // rows that the tensors of the call hold
  uint32_t *status;    // PF_KV8_* bits, or null

  // Rows [lo, hi) of a sequence, within the tensors whatever `starts` holds; false where its starts fall.
  __device__ bool rows(int s, int &lo, int &hi) const {
    if (starts) {
      const int a = starts[s], b = starts[s + 1];
      lo = min(max(a, 0), n_rows);
      hi = min(max(b, lo), n_rows);
      return a <= b;
    }
    lo = s * rows_each;
    hi = lo + rows_each;
    return true;
  }
  __device__ void report(uint32_t bits) const {
    if (status) atomicOr(status, bits);
  }
  // One CTA of a launch looks all row starts over.
  __device__ void check_starts(int most) const {
    for (int s = threadIdx.x; s < n_seqs; s += blockDim.x)
      if (starts[s] < 0 || starts[s + 1] < starts[s] || starts[s + 1] > n_rows || starts[s + 1] - starts[s] > most)
        report(PF_KV8_BAD_ROWS);
  }
  // Tokens of a sequence, within its table whatever `lens` holds.
  __device__ int length(int s, int block_log2) const {
    const int n = lens[s];
    return max(0, (int)min((int64_t)n, (int64_t)max_blocks << block_log2));
  }
  // A block id that lies in the cache, or false.
  __device__ bool block(const Kv8View &c, int s, int index, uint32_t &id) const {
    id = (uint32_t)tables[s * table_stride + index];
    return id < c.num_blocks;
  }
};

__device__ __forceinline__ float exp2i(int e) {   // 2^e; 0 below the normal numbers
  return e < -126 ? 0.f : __int_as_float((min(e, 127) + 127) << 23);
}
// Least e with amax <= 448 * 2^e, from the bits of amax >= 0 (finite): 448 = 1.75 * 2^8.
__device__ __forceinline__ int kv8_exponent(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return min(max(e, kKv8MinExp), kKv8MaxExp);
}
// Exponent of a stored scale.
__device__ __forceinline__ int kv8_scale_exponent(float scale) {
  const int e = (int)((__float_as_uint(scale) >> 23) & 255) - 127;
  return min(max(e, kKv8MinExp), kKv8MaxExp);
}

// Round to nearest even, saturating: an infinity becomes +-448 steps, a NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) { return e4m3x2(a, b) | (e4m3x2(c, d) << 16); }
__device__ __forceinline__ uint32_t e4m3x4_from_f16(uint32_t a, uint32_t b) {
  uint16_t x, y;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(x) : "r"(a));
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(y) : "r"(b));
  return x | (uint32_t)y << 16;
}
// Exact: every e4m3 value is an f16 value.  `half` selects the low or the high two bytes of `w`.
template <int half>
__device__ __forceinline__ uint32_t f16x2_from_e4m3(uint32_t w) {
  uint32_t d;
  asm("{.reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, %2;}"
      : "=r"(d)
      : "r"(w), "h"((uint16_t)(half ? w >> 16 : w & 0xffff)));
  return d;
}
__device__ __forceinline__ float2 f32x2_from_f16x2(uint32_t h) {
  float2 r;
  asm("{.reg .f16 lo, hi; mov.b32 {lo, hi}, %2; cvt.f32.f16 %0, lo; cvt.f32.f16 %1, hi;}" : "=f"(r.x), "=f"(r.y) : "r"(h));
  return r;
}

// Kernels follow each other closely: each is launched with launch_after, may start while the one before it on the stream
// drains, and every thread of it calls after_previous() before it touches what earlier work wrote.  The wait comes
// before the permission to start the next kernel, so that a kernel that has started knows that everything before its
// predecessor is complete: a call's later kernels may read the caller's lens and starts ahead of their own wait.
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
}
template <class... Params, class... Args>
void launch_after(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
  if (e != cudaSuccess) throw Error::storage(strf("kernel launch failed: %s", cudaGetErrorString(e)));
}

// Host side of every call: checks of the arguments that all of them take.
Kv8View kv8_check_cache(const pf_kv8_cache *cache);
Kv8Batch kv8_check_batch(const pf_kv8_batch *batch, size_t n_rows);
int kv8_sm_count(int device_id);   // throws CudaInit for a device that is not there

}  // namespace pf
