// Attention over the KV cache held in 8 bits (pf_kv8_attention).
//
//   s[i, j] = scale * 2^eK(j) * q[i] . K8[j]        out[i] = sum_j p[i, j] * 2^eV(j) * V8[j],  p = exp(s - lse)
//
// Few query rows per KV head (single tokens, drafted tokens): the cache is read once and each byte is used for as many
// products as there are rows, so HBM bounds it.  The tensor cores are still what makes it fit: 8 rows x 2 products x
// 7 TB/s are more multiply-adds than the ordinary pipes have beside the conversions.
//
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, as m16n8k16 f16 matrix instructions: 16 tokens (or
// 16 head dimensions) are the rows, 8 query rows the columns.  K and V come straight from global memory into the
// registers that the instruction wants, with no shared memory between: the order of the contracted index is free
// as long as both operands share it, so a lane takes 16 consecutive bytes of a row and calls them what the
// instruction's layout asks for.  Numbers:
//   K8, V8   every e4m3 value is an f16 value: converted without rounding, products and sums in fp32
//   q        scaled by a power of two for each row so that its largest element lies in [2^14, 2^15), then f16:
//            exact for f16 q, and for bf16 q but for elements 2^-28 of the row's largest and below
//   p        rounded to f16, 2^-11 / 2 relative, from fp32 scores; p is held as 2^(9 + s - ref) with a reference that
//            follows the running maximum by steps of at least 2^6, so that f16's range is used from 2^-24 to 2^15
//   scales   powers of two, applied to fp32 sums of one 16-token tile (a tile lies within one block)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kv8_attention.h"

namespace pf {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kTile = 16;                   // tokens of one warp's step
constexpr int kUnit = kTile * kWarps;       // tokens of one CTA's step, the granularity of the split
constexpr float kShift = 9.f, kSlack = 6.f;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// Query rows as the B operand of S^T = K Q^T, for rows row_first + n, n < 8 * kNt.  Lane (g, t) holds row g's elements
// 64 x + 16 t .. + 15 for each x, in the order in which K's lanes hold theirs.  factor = scale * log2(e) over the
// row's power of two, for columns 2 t and 2 t + 1 of each tile: score in log2 units = product * factor * scale of K.
template <int kDim, int kNt, bool kBf16>
struct Queries {
  uint32_t b[kNt][kDim / 16][2];
  float factor[kNt][2];

  template <class SeqT>
  __device__ void load(const AttnParams &p, const SeqT &seq, int head, int row_first) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < kNt; ++j) {
      const int row = row_first + 8 * j + g;
      float x[kDim / 4];
      const bool live = row < seq.rows * p.group;
      const int i = live ? row / p.group : 0, qh = head * p.group + (live ? row % p.group : 0);
      const uint16_t *src = p.q + (int64_t)(seq.row0 + i) * p.q_row + qh * p.q_head + 16 * t;
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < kDim / 4; k += 8) {
        const uint16_t *at = src + 64 * (k / 16) + k % 16;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (live) {
          if (p.vec_q) w = *reinterpret_cast<const uint4 *>(at);
          else w = make_uint4(at[0] | at[1] << 16, at[2] | at[3] << 16, at[4] | at[5] << 16, at[6] | at[7] << 16);
        }
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          x[k + 2 * m] = widen1<kBf16>((uint16_t)u[m]);
          x[k + 2 * m + 1] = widen1<kBf16>((uint16_t)(u[m] >> 16));
          top = fmaxf(top, fmaxf(fabsf(x[k + 2 * m]), fabsf(x[k + 2 * m + 1])));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e brings the row's largest element into [2^14, 2^15); a row of zeros or with an infinity stays as it is
      int e = (int)(__float_as_uint(top) >> 23) - 127 - 14;
      if (top == 0.f || top > 3.4e38f) e = 0;
      e = max(e, -126);
      const float down = exp2i(-e);
#pragma unroll
      for (int m = 0; m < kDim / 16; ++m) {
        b[j][m][0] = f16x2(x[4 * m] * down, x[4 * m + 1] * down);
        b[j][m][1] = f16x2(x[4 * m + 2] * down, x[4 * m + 3] * down);
      }
      const float mine = p.scale * kLog2e * exp2i(e);
      factor[j][0] = __shfl_sync(0xffffffffu, mine, (2 * t) * 4);
      factor[j][1] = __shfl_sync(0xffffffffu, mine, (2 * t + 1) * 4);
    }
  }
};

// One 16-token tile of K: lane (g, t) holds rows g and g + 8, bytes 64 x + 16 t .. + 15.
template <int kDim>
struct KTile {
  uint4 w[kDim / 64][2];
  __device__ void load(const uint8_t *tile, int row0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint8_t *at = tile + (row0 + g) * kDim + 16 * t;
#pragma unroll
    for (int x = 0; x < kDim / 64; ++x) {
      w[x][0] = __ldg(reinterpret_cast<const uint4 *>(at + 64 * x));
      w[x][1] = __ldg(reinterpret_cast<const uint4 *>(at + 64 * x + 8 * kDim));
    }
  }
  // c += K Q^T: c[0], c[1] = token g, columns 2 t, 2 t + 1; c[2], c[3] = token g + 8
  template <int kNt, bool kBf16>
  __device__ void products(const Queries<kDim, kNt, kBf16> &q, float (&c)[kNt][4]) const {
#pragma unroll
    for (int x = 0; x < kDim / 64; ++x) {
      const uint32_t lo[4] = {w[x][0].x, w[x][0].y, w[x][0].z, w[x][0].w};
      const uint32_t hi[4] = {w[x][1].x, w[x][1].y, w[x][1].z, w[x][1].w};
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const uint32_t a0 = f16x2_from_e4m3<0>(lo[m]), a1 = f16x2_from_e4m3<0>(hi[m]);
        const uint32_t a2 = f16x2_from_e4m3<1>(lo[m]), a3 = f16x2_from_e4m3<1>(hi[m]);
#pragma unroll
        for (int j = 0; j < kNt; ++j) mma_f16(c[j], a0, a1, a2, a3, q.b[j][4 * x + m][0], q.b[j][4 * x + m][1]);
      }
    }
  }
};

// One 16-token tile of V: lane (g, t) holds tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9, bytes (kDim / 8) g .. + kDim / 8 - 1.
template <int kDim>
struct VTile {
  static constexpr int kWords = kDim / 32;   // 4-byte words of one token
  uint32_t w[4][kWords];
  __device__ void load(const uint8_t *tile, int row0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint8_t *at = tile + (row0 + 2 * t) * kDim + g * (kDim / 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t *row = at + ((i & 1) + 8 * (i >> 1)) * kDim;
      if constexpr (kWords == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(row));
        w[i][0] = v.x, w[i][1] = v.y;
      } else {
#pragma unroll
        for (int x = 0; x < kWords / 4; ++x) {
          const uint4 v = __ldg(reinterpret_cast<const uint4 *>(row) + x);
          w[i][4 * x] = v.x, w[i][4 * x + 1] = v.y, w[i][4 * x + 2] = v.z, w[i][4 * x + 3] = v.w;
        }
      }
    }
  }
  __device__ bool has_nan() const {   // a byte 0x7f or 0xff
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < kWords; ++x) any |= (w[i][x] & 0x7f7f7f7fu) + 0x01010101u;
    return any & 0x80808080u;
  }
};

// Rows of the score tile that lie behind the visible tokens hold what the block held before: a NaN there would
// survive a product with p = 0.  Called for a sequence's last tile only.
template <int kDim>
__device__ __forceinline__ void clear_behind(VTile<kDim> &v, int first_hidden) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (2 * t + (i & 1) + 8 * (i >> 1) >= first_hidden)
#pragma unroll
      for (int x = 0; x < VTile<kDim>::kWords; ++x) v.w[i][x] = 0;
}

// A NaN in V reaches the rows that see its token and no other: 0 * NaN would.  In tiles that some row sees in part it is
// taken out, and the first such token is remembered for each dimension.
__device__ __noinline__ void note_nan(uint32_t word, int *nan_from, int token) {
  for (int b = 0; b < 4; ++b)
    if ((word >> (8 * b) & 0x7f) == 0x7f) atomicMin(nan_from + b, token);
}
template <int kDim>
__device__ __forceinline__ void take_nan_out(VTile<kDim> &v, int *nan_from, int tok) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int x = 0; x < VTile<kDim>::kWords; ++x) {
      const uint32_t w = v.w[i][x], mask = (((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 255u;
      if (mask) note_nan(w, nan_from + g * (kDim / 8) + 4 * x, tok + 2 * t + (i & 1) + 8 * (i >> 1));
      v.w[i][x] = w & ~mask;
    }
}

// A block of the sequence's table, looked up ahead of its use.
struct Page {
  uint32_t id;
  bool there;
  __device__ void find(const AttnParams &p, int s, int tok) { there = p.batch.block(p.cache, s, tok >> p.cache.block_log2, id); }
};

// CTAs that an SM holds: what the registers allow (128 of them at 128 dimensions and 8 rows).
constexpr int ctas_of(int dim, int nt) { return dim == 256 ? 2 : dim == 128 ? (nt == 1 ? 4 : 2) : (nt == 1 ? 5 : 4); }

template <int kDim, int kNt, bool kBf16>
__global__ void __launch_bounds__(kThreads, ctas_of(kDim, kNt)) kv8_attention_rows(AttnParams p) {
  constexpr int kRows = 8 * kNt, kMt = kDim / 16;
  using SeqT = Seq<kRows, kUnit>;
  extern __shared__ __align__(16) char smem[];
  float *sh_o = reinterpret_cast<float *>(smem);                       // [kWarps][kRows][kDim]
  float2 *sh_ml = reinterpret_cast<float2 *>(sh_o + kWarps * kRows * kDim);   // [kWarps][kRows]
  uint32_t *prefix = reinterpret_cast<uint32_t *>(sh_ml + kWarps * kRows);    // [n_seqs + 1]
  __shared__ int sh_nan_from[kDim], sh_any_nan;
  after_previous();
  for (int i = threadIdx.x; i < kDim; i += kThreads) sh_nan_from[i] = INT_MAX;
  if (threadIdx.x == 0) sh_any_nan = 0;
  scan_units(p, prefix, [&](int s) { return SeqT(p, s).all_units(p); });
  const int n_seqs = p.batch.n_seqs, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const Split split(prefix[n_seqs], p.n_ctas);
  if (blockIdx.x == 0) check_batch(p);
  if ((int)blockIdx.x >= split.n_ctas) return;
  uint32_t u = split.begin(blockIdx.x);
  const uint32_t u_end = split.begin(blockIdx.x + 1);
  bool first_segment = true;
  while (u < u_end) {
    const int s = find_seq(prefix, n_seqs, u);
    const SeqT seq(p, s);
    const Segment seg(p, seq, s, prefix[s], u);
    const int head = seg.head, row_first = seg.rt * kRows;
    const uint32_t unit0 = u - seg.begin, units = min(seg.units - unit0, u_end - u);
    const int live_rows = min(seq.all_rows(p) - row_first, kRows);
    const int most = seq.visible(p, row_first + live_rows - 1);         // tokens that any row of the tile sees
    const int least = seq.visible(p, row_first);                        // tokens that all rows see
    const int tok_end = (int)min((int64_t)(unit0 + units) * kUnit, (int64_t)most);
    int tok = (int)(unit0 * kUnit) + warp * kTile;

    // The pages of two steps ahead, the values of one: K of the next step is asked for when this step's products have
    // read K's registers, V when its own have.
    const int within = p.cache.block_size() - 1;
    Page page{}, next{};
    KTile<kDim> kt;
    VTile<kDim> vt;
    float k_scale = 0.f, v_scale = 0.f;
    if (tok < tok_end) page.find(p, s, tok);
    if (tok + kUnit < tok_end) next.find(p, s, tok + kUnit);
    if (tok < tok_end && page.there) {
      kt.load(p.cache.tile(0, page.id, head), tok & within);
      k_scale = __ldg(p.cache.scale(0, page.id, head));
      vt.load(p.cache.tile(1, page.id, head), tok & within);
      v_scale = __ldg(p.cache.scale(1, page.id, head));
    }
    Queries<kDim, kNt, kBf16> q;
    q.load(p, seq, head, row_first);
    int see[kNt][2];
#pragma unroll
    for (int j = 0; j < kNt; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) see[j][k] = seq.visible(p, min(row_first + 8 * j + 2 * t + k, seq.all_rows(p) - 1));
    float o[kNt][kMt][4], ref[kNt][2], sum[kNt][2];
#pragma unroll
    for (int j = 0; j < kNt; ++j) {
#pragma unroll
      for (int m = 0; m < kMt; ++m) o[j][m][0] = o[j][m][1] = o[j][m][2] = o[j][m][3] = 0.f;
      ref[j][0] = ref[j][1] = kNone;
      sum[j][0] = sum[j][1] = 0.f;
    }
    for (; tok < tok_end; tok += kUnit) {
      const bool there = page.there, more = tok + kUnit < tok_end && next.there;
      if (!there) p.batch.report(PF_KV8_BAD_BLOCK);
      float c[kNt][4];
#pragma unroll
      for (int j = 0; j < kNt; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
      if (there) kt.products(q, c);
#pragma unroll
      for (int j = 0; j < kNt; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float f = q.factor[j][k] * k_scale;
          c[j][k] *= f;
          c[j][k + 2] *= f;
        }
      const Page ahead = next;
      if (more) {
        kt.load(p.cache.tile(0, ahead.id, head), (tok + kUnit) & within);
        k_scale = __ldg(p.cache.scale(0, ahead.id, head));
      }
      if (tok + 2 * kUnit < tok_end) next.find(p, s, tok + 2 * kUnit);
      page = ahead;
      if (there) {
        if (tok + kTile > least) {
#pragma unroll
          for (int j = 0; j < kNt; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if (tok + g >= see[j][k]) c[j][k] = -INFINITY;
              if (tok + g + 8 >= see[j][k]) c[j][k + 2] = -INFINITY;
            }
          if (tok + kTile > seq.len) clear_behind(vt, seq.len - tok);
          if (vt.has_nan()) {
            sh_any_nan = 1;
            take_nan_out(vt, sh_nan_from, tok);
          }
        }
        bool over = false;
#pragma unroll
        for (int j = 0; j < kNt; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k) over |= fmaxf(c[j][k], c[j][k + 2]) > ref[j][k] + kSlack;
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int j = 0; j < kNt; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float top = fmaxf(c[j][k], c[j][k + 2]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              const float now = fmaxf(ref[j][k], top), r = exp2_fast(ref[j][k] - now);
              ref[j][k] = now;
              sum[j][k] *= r;
#pragma unroll
              for (int m = 0; m < kMt; ++m) {
                o[j][m][k] *= r;
                o[j][m][k + 2] *= r;
              }
            }
        }
        uint32_t pb[kNt][2];
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
#pragma unroll
          for (int k = 0; k < 4; ++k) c[j][k] = exp2_fast(c[j][k] - (ref[j][k & 1] - kShift));
          sum[j][0] += c[j][0] + c[j][2];
          sum[j][1] += c[j][1] + c[j][3];
          pb[j][0] = transpose8x8(f16x2(c[j][0], c[j][1]));
          pb[j][1] = transpose8x8(f16x2(c[j][2], c[j][3]));
        }
#pragma unroll
        for (int w = 0; w < VTile<kDim>::kWords; ++w) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362 : 0x5140;
            const uint32_t ab = __byte_perm(vt.w[0][w], vt.w[1][w], sel), ce = __byte_perm(vt.w[2][w], vt.w[3][w], sel);
            const uint32_t a0 = f16x2_from_e4m3<0>(ab), a1 = f16x2_from_e4m3<1>(ab);
            const uint32_t a2 = f16x2_from_e4m3<0>(ce), a3 = f16x2_from_e4m3<1>(ce);
#pragma unroll
            for (int j = 0; j < kNt; ++j) {
              float d[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16(d, a0, a1, a2, a3, pb[j][0], pb[j][1]);
#pragma unroll
              for (int k = 0; k < 4; ++k) o[j][2 * w + half][k] += v_scale * d[k];
            }
          }
        }
      }
      if (more) {
        vt.load(p.cache.tile(1, ahead.id, head), (tok + kUnit) & within);
        v_scale = __ldg(p.cache.scale(1, ahead.id, head));
      }
    }
    // join the four warps
#pragma unroll
    for (int j = 0; j < kNt; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum[j][k] += __shfl_xor_sync(0xffffffffu, sum[j][k], d);
        if (g == 0) sh_ml[warp * kRows + 8 * j + 2 * t + k] = make_float2(ref[j][k], sum[j][k]);
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kNt; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int n = 8 * j + 2 * t + k;
        float top = kNone;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh_ml[w * kRows + n].x);
        const float r = exp2_fast(ref[j][k] - top);
        float *dst = sh_o + (warp * kRows + n) * kDim + g * (kDim / 8);
#pragma unroll
        for (int m = 0; m < kMt; m += 2)
          *reinterpret_cast<float4 *>(dst + 2 * m) =
              make_float4(o[j][m][k] * r, o[j][m][k + 2] * r, o[j][m + 1][k] * r, o[j][m + 1][k + 2] * r);
      }
    __syncthreads();
    const bool whole = units == seg.units;
    const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
    for (int e = threadIdx.x; e < live_rows * (kDim / 4); e += kThreads) {
      const int n = e / (kDim / 4), d = e % (kDim / 4) * 4;
      float top = kNone, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh_ml[w * kRows + n].x);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = sh_ml[w * kRows + n];
        l += ml.y * exp2_fast(ml.x - top);
        const float4 x = *reinterpret_cast<const float4 *>(sh_o + (w * kRows + n) * kDim + d);
        a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
      }
      if (sh_any_nan) {
        const int see_row = seq.visible(p, row_first + n);
        float *y = &a.x;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (sh_nan_from[d + k] < see_row) y[k] = __int_as_float(0x7fffffff);
      }
      if (whole) {
        const int row = row_first + n, i = row / p.group, qh = head * p.group + row % p.group;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t *dst = p.out + (int64_t)(seq.row0 + i) * p.out_row + qh * p.out_head + d;
        const uint32_t x = narrow2<kBf16>(a.x * inv, a.y * inv), y = narrow2<kBf16>(a.z * inv, a.w * inv);
        if (p.vec_out) *reinterpret_cast<uint2 *>(dst) = make_uint2(x, y);
        else dst[0] = (uint16_t)x, dst[1] = x >> 16, dst[2] = (uint16_t)y, dst[3] = y >> 16;
        if (d == 0 && p.lse) p.lse[(int64_t)(seq.row0 + i) * p.q_heads + qh] = lse_of(top - kShift, l);
      } else {
        *reinterpret_cast<float4 *>(p.part_o + ((int64_t)slot * kRows + n) * kDim + d) = a;
        if (d == 0) p.part_ml[slot * kRows + n] = make_float2(top - kShift, l);
      }
    }
    const bool any_nan = sh_any_nan;
    __syncthreads();
    u += units;
    first_segment = false;
    if (any_nan) {
      for (int i = threadIdx.x; i < kDim; i += kThreads) sh_nan_from[i] = INT_MAX;
      if (threadIdx.x == 0) sh_any_nan = 0;
      __syncthreads();
    }
  }
}

// Joins the parts of segments that several CTAs shared, in the order of the tokens.  CTA (b, y) looks at the boundary
// between the ranges of CTAs b and b + 1: if it is the first one within a segment, it joins rows of it, a team of threads
// for each.  kDim / 4 threads hold a row of a part as float4; a team of more reads several parts at once.
constexpr int kJoinThreads = 256;
template <int kDim, int kRows, int kUnits, bool kBf16>
__global__ void __launch_bounds__(kJoinThreads) kv8_attention_join(AttnParams p, int team) {
  constexpr int kSpan = kDim / 4, kDeep = 4;
  using SeqT = Seq<kRows, kUnits>;
  extern __shared__ __align__(16) char smem[];
  uint32_t *prefix = reinterpret_cast<uint32_t *>(smem);
  __shared__ float4 sh_a[kJoinThreads];
  __shared__ float sh_l[kJoinThreads], sh_top[kJoinThreads / 32];
  const int n_seqs = p.batch.n_seqs;
  scan_units(p, prefix, [&](int s) { return SeqT(p, s).all_units(p); });
  after_previous();
  if (p.clear_tail) {
    int lo, hi = 0;
    if (n_seqs) p.batch.rows(n_seqs - 1, lo, hi);
    const int64_t id = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kJoinThreads + threadIdx.x;
    for (int64_t e = (int64_t)hi * p.q_heads * kDim + id; e < (int64_t)p.batch.n_rows * p.q_heads * kDim;
         e += (int64_t)gridDim.x * gridDim.y * kJoinThreads) {
      const int64_t row = e / (p.q_heads * kDim);
      const int qh = (int)(e / kDim % p.q_heads), d = (int)(e % kDim);
      p.out[row * p.out_row + qh * p.out_head + d] = 0;
      if (d == 0 && p.lse) p.lse[row * p.q_heads + qh] = -INFINITY;
    }
  }
  const Split split(prefix[n_seqs], p.n_ctas);
  const int c0 = blockIdx.x;
  if (c0 + 1 >= split.n_ctas) return;
  const uint32_t u = split.begin(c0 + 1);
  const int s = find_seq(prefix, n_seqs, u);
  const SeqT seq(p, s);
  const Segment seg(p, seq, s, prefix[s], u);
  if (seg.begin == u || split.owner(seg.begin) != c0) return;
  const int parts = split.owner(seg.begin + seg.units - 1) - c0 + 1, slot0 = 2 * c0 + (split.begin(c0) < seg.begin ? 1 : 0);
  const int teams = kJoinThreads / team, lane = threadIdx.x % team, part0 = lane / kSpan, at_once = team / kSpan, d = lane % kSpan * 4;
  const int live_rows = min(seq.all_rows(p) - seg.rt * kRows, kRows);
  auto slot_of = [&](int k) { return k == 0 ? slot0 : 2 * (c0 + k); };
  for (int n0 = blockIdx.y * teams; n0 < live_rows; n0 += gridDim.y * teams) {
    const int n = min(n0 + (int)threadIdx.x / team, live_rows - 1);      // surplus teams repeat the last row
    float top = kNone;
    if (at_once == 1) {
      for (int k = 0; k < parts; ++k) top = fmaxf(top, p.part_ml[slot_of(k) * kRows + n].x);
    } else {                // a team of several warps: the only one, or one of few
      for (int k = lane; k < parts; k += team) top = fmaxf(top, p.part_ml[slot_of(k) * kRows + n].x);
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k, min(team, 32)));
      if (team > 32) {
        if ((threadIdx.x & 31) == 0) sh_top[threadIdx.x >> 5] = top;
        __syncthreads();
        const int warp0 = (int)threadIdx.x / team * (team / 32);
        for (int k = 0; k < team / 32; ++k) top = fmaxf(top, sh_top[warp0 + k]);
      }
    }
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int k0 = part0; k0 < parts; k0 += kDeep * at_once) {
      float2 ml[kDeep];
      float4 x[kDeep];
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        const int k = k0 + i * at_once;
        ml[i] = make_float2(kNone, 0.f);
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k < parts) {
          ml[i] = p.part_ml[slot_of(k) * kRows + n];
          x[i] = *reinterpret_cast<const float4 *>(p.part_o + ((int64_t)slot_of(k) * kRows + n) * kDim + d);
        }
      }
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        const float r = exp2_fast(ml[i].x - top);
        l += ml[i].y * r;
        a.x += x[i].x * r, a.y += x[i].y * r, a.z += x[i].z * r, a.w += x[i].w * r;
      }
    }
    if (at_once > 1) {
      sh_a[threadIdx.x] = a;
      sh_l[threadIdx.x] = l;
      __syncthreads();
      if (part0 == 0)
        for (int k = 1; k < at_once; ++k) {
          const float4 x = sh_a[threadIdx.x + k * kSpan];
          a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
          l += sh_l[threadIdx.x + k * kSpan];
        }
    }
    if (part0 == 0 && n0 + (int)threadIdx.x / team < live_rows) {
      const int row = seg.rt * kRows + n, i = row / p.group, qh = seg.head * p.group + row % p.group;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint16_t *dst = p.out + (int64_t)(seq.row0 + i) * p.out_row + qh * p.out_head + d;
      const uint32_t x = narrow2<kBf16>(a.x * inv, a.y * inv), y = narrow2<kBf16>(a.z * inv, a.w * inv);
      if (p.vec_out) *reinterpret_cast<uint2 *>(dst) = make_uint2(x, y);
      else dst[0] = (uint16_t)x, dst[1] = x >> 16, dst[2] = (uint16_t)y, dst[3] = y >> 16;
      if (d == 0 && p.lse) p.lse[(int64_t)(seq.row0 + i) * p.q_heads + qh] = lse_of(top, l);
    }
    if (at_once > 1) __syncthreads();
  }
}

// weights[s, head, j] += sum over rows and group heads of exp(score - lse), once lse is known: the scores are taken
// again, a warp for 16 tokens, or for 64 at a time where there are more than eight rows.  Each element has one writer.
template <int kDim, bool kBf16>
__global__ void __launch_bounds__(kThreads) kv8_attention_weights(AttnParams p) {
  constexpr int kRows = 8, kDeep = 4;
  using SeqT = Seq<kRows, kUnit>;
  extern __shared__ __align__(16) char smem[];
  uint32_t *prefix = reinterpret_cast<uint32_t *>(smem);
  auto units_of = [&](const SeqT &seq) {   // of one head; none for a sequence without rows
    const int tokens = min(seq.len, p.w_capacity);
    return seq.rows ? (uint32_t)((tokens + kUnit - 1) / kUnit) : 0u;
  };
  scan_units(p, prefix, [&](int s) { return units_of(SeqT(p, s)) * (uint32_t)p.cache.heads; });
  after_previous();
  const int n_seqs = p.batch.n_seqs, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (blockIdx.x == 0)
    for (int s = threadIdx.x; s < n_seqs; s += kThreads)
      if (p.batch.lens[s] > p.w_capacity) p.batch.report(PF_KV8_BAD_LENGTH);
  const Split split(prefix[n_seqs], gridDim.x);
  if ((int)blockIdx.x >= split.n_ctas) return;
  const int within = p.cache.block_size() - 1;
  uint32_t u = split.begin(blockIdx.x);
  const uint32_t u_end = split.begin(blockIdx.x + 1);
  while (u < u_end) {
    const int s = find_seq(prefix, n_seqs, u);
    const SeqT seq(p, s);
    const uint32_t of_head = units_of(seq), unit0 = (u - prefix[s]) % of_head, units = min(of_head - unit0, u_end - u);
    const int head = (u - prefix[s]) / of_head, end = min(seq.len, p.w_capacity), rows = seq.all_rows(p);
    float *dst = p.weights + s * p.w_seq + head * p.w_head;
    // adds row tile row_first's share of the 16 tokens from tok on
    auto add = [&](const Queries<kDim, 1, kBf16> &q, const float (&base)[2], const int (&see)[2], int tok, float (&w)[2]) {
      Page page;
      page.find(p, s, tok);
      if (!page.there) return;
      KTile<kDim> kt;
      kt.load(p.cache.tile(0, page.id, head), tok & within);
      const float k_scale = __ldg(p.cache.scale(0, page.id, head));
      float c[1][4] = {{0.f, 0.f, 0.f, 0.f}};
      kt.products(q, c);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float f = q.factor[0][k] * k_scale;
        if (tok + g < see[k]) w[0] += exp2_fast(c[0][k] * f - base[k]);
        if (tok + g + 8 < see[k]) w[1] += exp2_fast(c[0][k + 2] * f - base[k]);
      }
    };
    auto rows_of = [&](Queries<kDim, 1, kBf16> &q, float (&base)[2], int (&see)[2], int row_first) {
      q.load(p, seq, head, row_first);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = row_first + 2 * t + k;
        base[k] = 0.f, see[k] = 0;
        if (row < rows) {
          see[k] = seq.visible(p, row);
          base[k] = p.lse[(int64_t)(seq.row0 + row / p.group) * p.q_heads + head * p.group + row % p.group] * kLog2e;
        }
      }
    };
    auto store = [&](int tok, float (&w)[2]) {
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        w[0] += __shfl_xor_sync(0xffffffffu, w[0], d);
        w[1] += __shfl_xor_sync(0xffffffffu, w[1], d);
      }
      if (t == 0) {
        if (tok + g < end) dst[tok + g] += w[0];
        if (tok + g + 8 < end) dst[tok + g + 8] += w[1];
      }
    };
    Queries<kDim, 1, kBf16> q;
    float base[2];
    int see[2];
    if (rows <= kRows) {
      rows_of(q, base, see, 0);
      for (uint32_t i = unit0; i < unit0 + units; ++i) {
        const int tok = (int)(i * kUnit) + warp * kTile;
        float w[2] = {0.f, 0.f};
        if (tok >= end) break;
        add(q, base, see, tok, w);
        store(tok, w);
      }
    } else {
      for (uint32_t i = unit0 + warp; i < unit0 + units; i += kWarps) {
        const int tok = (int)(i * kUnit);
        float w[kDeep][2] = {};
        for (int row_first = 0; row_first < rows; row_first += kRows) {
          if (seq.visible(p, min(row_first + kRows, rows) - 1) <= tok) continue;
          rows_of(q, base, see, row_first);
#pragma unroll
          for (int m = 0; m < kDeep; ++m)
            if (tok + m * kTile < end) add(q, base, see, tok + m * kTile, w[m]);
        }
#pragma unroll
        for (int m = 0; m < kDeep; ++m)
          if (tok + m * kTile < end) store(tok + m * kTile, w[m]);
      }
    }
    u += units;
  }
}

// ---------------------------------------------------------------------------------------------- host
struct Plan {
  int nt;               // row tiles of eight, 0: by the hundred
  int n_ctas, rows;     // rows of a part
  size_t part_o, part_ml, lse, bytes;   // offsets in the workspace
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

Plan make_plan(int device_id, const Kv8View &c, const pf_kv8_attention_args &a) {
  const size_t group = a.q_heads / c.heads;
  Plan plan{};
  const size_t rows = std::min(a.max_query, a.n_rows) * group;
  plan.nt = rows <= 8 ? 1 : rows <= 16 && c.dim != 256 ? 2 : 0;
  plan.n_ctas = kv8_sm_count(device_id) * (plan.nt ? ctas_of(c.dim, plan.nt) : 1);
  plan.rows = plan.nt ? 8 * plan.nt : kv8_wide_plan(c.dim).rows;
  const size_t slots = 2 * (size_t)plan.n_ctas * plan.rows;
  plan.part_o = 0;
  plan.part_ml = up256(slots * c.dim * 4);
  plan.lse = plan.part_ml + up256(slots * 8);
  plan.bytes = plan.lse + (a.weights && !a.lse ? up256(a.n_rows * a.q_heads * 4) : 0);
  return plan;
}

void check_args(const pf_kv8_attention_args *a, const Kv8View &c, const Kv8Batch &b) {
  if (!a) throw Error::invalid("null attention arguments");
  if (a->dtype != PF_KV8_BF16 && a->dtype != PF_KV8_F16) throw Error::invalid(strf("unknown dtype %d", a->dtype));
  if (a->q_heads == 0 || a->q_heads % c.heads || a->q_heads > 65536)
    throw Error::invalid(strf("%u query heads are not a multiple of %d KV heads", a->q_heads, c.heads));
  if (a->n_rows && b.n_seqs && a->max_query == 0) throw Error::invalid("max_query must not be 0");
  const uint64_t rows_of_group = (uint64_t)std::min<size_t>(a->max_query, a->n_rows) * (a->q_heads / c.heads);
  if (rows_of_group > 0x3fffffffu) throw Error::invalid("too many query rows");
  if (!b.starts && b.n_seqs && a->max_query < (size_t)b.rows_each)
    throw Error::invalid(strf("max_query=%zu is below the %d rows of each sequence", a->max_query, b.rows_each));
  // units are counted in 32 bits: (segments) x (units of a segment), summed over the sequences
  const uint64_t units = ((uint64_t)b.max_blocks << c.block_log2) / kUnit + 1;
  const uint64_t tiles = ((uint64_t)a->n_rows * (a->q_heads / c.heads) + 7) / 8 + b.n_seqs;
  if (units * tiles > 0xffffffffull / c.heads) throw Error::invalid("too many query rows for tables of this width: split the call");
}

template <int kDim, int kRows, int kUnits, bool kBf16>
void launch_join(const AttnParams &p, cudaStream_t stream) {
  // About n_ctas / segments parts meet in a segment: few are read one after the other by the fewest threads that hold a row,
  // many (a long sequence alone) by a whole CTA.  One rule for all: a quarter of them at a time.
  constexpr int kSpan = kDim / 4;
  const int segments = std::max(1, p.batch.n_seqs * p.cache.heads);
  int team = kSpan;
  while (team < kJoinThreads && team / kSpan * 4 * segments < p.n_ctas) team *= 2;
  const int passes = std::max(1, kRows * team / kJoinThreads);
  const dim3 grid((unsigned)p.n_ctas, (unsigned)std::min(passes, 16));
  launch_after(kv8_attention_join<kDim, kRows, kUnits, kBf16>, grid, kJoinThreads, ((size_t)p.batch.n_seqs + 1) * 4, stream, p, team);
}

template <int kDim, int kNt, bool kBf16>
void launch_rows(const AttnParams &p, cudaStream_t stream) {
  const size_t smem = kWarps * 8 * kNt * (kDim * 4 + 8) + ((size_t)p.batch.n_seqs + 1) * 4;
  auto kernel = kv8_attention_rows<kDim, kNt, kBf16>;
  if (smem > 47 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    throw Error::storage("cudaFuncSetAttribute failed");
  if (p.batch.n_seqs) launch_after(kernel, p.n_ctas, kThreads, smem, stream, p);
  launch_join<kDim, 8 * kNt, kUnit, kBf16>(p, stream);
}

template <int kDim, bool kBf16>
void launch_all(const AttnParams &p, int nt, int n_sms, cudaStream_t stream) {
  if (nt == 0) {
    if (p.batch.n_seqs) kv8_wide_launch(p, kBf16, stream);
    constexpr int kRows = kDim == 256 ? 128 : 256, kTokens = kDim == 256 ? 64 : 128;
    launch_join<kDim, kRows, kTokens, kBf16>(p, stream);
  } else if (nt == 1) {
    launch_rows<kDim, 1, kBf16>(p, stream);
  } else if constexpr (kDim != 256) {
    launch_rows<kDim, 2, kBf16>(p, stream);
  }
  if (p.weights && p.batch.n_seqs) {
    launch_after(kv8_attention_weights<kDim, kBf16>, n_sms * 4, kThreads, ((size_t)p.batch.n_seqs + 1) * 4, stream, p);
  }
}

template <bool kBf16>
void launch(const AttnParams &p, int nt, int n_sms, cudaStream_t stream) {
  if (p.cache.dim == 64) launch_all<64, kBf16>(p, nt, n_sms, stream);
  else if (p.cache.dim == 128) launch_all<128, kBf16>(p, nt, n_sms, stream);
  else launch_all<256, kBf16>(p, nt, n_sms, stream);
}

}  // namespace
}  // namespace pf

using namespace pf;

extern "C" {

int pf_kv8_attention_workspace(int device_id, const pf_kv8_cache *cache, const pf_kv8_batch *batch,
                               const pf_kv8_attention_args *args, size_t *bytes) {
  return guarded([&] {
    if (!bytes) throw Error::invalid("bytes is null");
    if (!args) throw Error::invalid("null attention arguments");
    const Kv8View c = kv8_check_cache(cache);
    const Kv8Batch b = kv8_check_batch(batch, args->n_rows);
    check_args(args, c, b);
    *bytes = make_plan(device_id, c, *args).bytes;
  });
}

int pf_kv8_attention(int device_id, const pf_kv8_cache *cache, const pf_kv8_batch *batch,
                     const pf_kv8_attention_args *args, void *workspace, size_t workspace_bytes, void *stream) {
  return guarded([&] {
    if (!args) throw Error::invalid("null attention arguments");
    const Kv8View c = kv8_check_cache(cache);
    const Kv8Batch b = kv8_check_batch(batch, args->n_rows);
    const pf_kv8_attention_args &a = *args;
    check_args(args, c, b);
    if (a.n_rows == 0 || (b.n_seqs == 0 && !a.clear_tail)) return;
    if (!a.q || !a.out) throw Error::invalid("null q or out");
    if ((uintptr_t)a.q % 2 || (uintptr_t)a.out % 2) throw Error::invalid("q and out must be aligned to their elements");
    const Plan plan = make_plan(device_id, c, a);
    if (!workspace || workspace_bytes < plan.bytes)
      throw Error::invalid(strf("workspace of %zu bytes, the call needs %zu", workspace ? workspace_bytes : 0, plan.bytes));
    if ((uintptr_t)workspace % 256) throw Error::invalid("the workspace must be 256-byte aligned");
    AttnParams p{};
    p.cache = c;
    p.batch = b;
    p.q = (const uint16_t *)a.q;
    p.out = (uint16_t *)a.out;
    char *ws = (char *)workspace;
    p.part_o = (float *)(ws + plan.part_o);
    p.part_ml = (float2 *)(ws + plan.part_ml);
    p.lse = a.lse ? a.lse : a.weights ? (float *)(ws + plan.lse) : nullptr;
    p.weights = a.weights;
    p.q_row = (int64_t)a.q_row_stride, p.q_head = (int64_t)a.q_head_stride;
    p.out_row = (int64_t)a.out_row_stride, p.out_head = (int64_t)a.out_head_stride;
    p.w_seq = (int64_t)a.weights_seq_stride, p.w_head = (int64_t)a.weights_head_stride;
    p.w_capacity = (int)std::min<size_t>(a.weights_capacity, 0x7fffffff);
    p.q_heads = (int)a.q_heads;
    p.group = (int)a.q_heads / c.heads;
    p.max_query = (int)std::min<size_t>(a.max_query, a.n_rows);
    p.causal = a.causal != 0;
    p.clear_tail = a.clear_tail != 0;
    p.vec_q = (uintptr_t)a.q % 16 == 0 && (a.q_row_stride | a.q_head_stride) % 8 == 0;
    p.vec_out = (uintptr_t)a.out % 8 == 0 && (a.out_row_stride | a.out_head_stride) % 4 == 0;
    p.scale = a.scale;
    p.n_ctas = plan.n_ctas;
    DeviceGuard on_device(device_id);
    if (a.dtype == PF_KV8_BF16) launch<true>(p, plan.nt, kv8_sm_count(device_id), (cudaStream_t)stream);
    else launch<false>(p, plan.nt, kv8_sm_count(device_id), (cudaStream_t)stream);
  });
}

}  // extern "C"
