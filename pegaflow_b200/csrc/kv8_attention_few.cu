// Attention over the KV cache held in 8 bits (pf_kv8_attention) for few query rows per KV head (single tokens, drafted
// tokens), and the accumulated weights.
//
//   s[i, j] = scale * 2^eK(j) * q[i] . K8[j]        out[i] = sum_j p[i, j] * 2^eV(j) * V8[j],  p = exp(s - lse)
//
// The cache is read once and each byte is used for as many products as there are rows, so HBM bounds it, if the arithmetic
// keeps out of the way.  It does when no thread touches K and V at all: 128 tokens at a time go from global into shared memory
// by asynchronous copies, and the tcgen05 tensor cores take the products on the e4m3 bytes as they are, transposed:
//   S^T [128 tokens, columns] = K Q^T           O^T [head dimensions, columns] += V^T P^T
// A thread holds a token's scores (a lane of tensor memory), and at the end a dimension's outputs.  What is not e4m3, q and
// p, is written as four e4m3 pieces in columns of their own, x = x0 + x1 / 16 + x2 / 256 + x3 / 4096, each piece the
// rounding of 16 times what the one before it left: a column tile of 16 holds four rows, which is the narrowest that the
// instruction takes.
//   q    scaled by a power of two for each row so that its largest element lies in [2^7, 2^8): its pieces hold a bf16 or an
//        f16 exactly down to 2^-18 of the row's largest, and smaller elements to 2^-30 of it
//   p    2^(6 + s - ref) rounded to f16 (2^-12 of p), ref following the row's running maximum in steps of 2^2; the pieces hold
//        that exactly down to 2^-11, that is 2^-17 of the largest, and smaller ones to 2^-28 of it
//   V's scale goes on p: 2^(e - e_ref), e_ref the largest so far, and the sums are in units of it; the row sum leaves it out
//   sums fp32, the tensor cores' and the row sum's; it takes p before it is rounded
// Other forms were measured at 48 requests of 700 to 16001 tokens, 8 heads of 128 (75 us at the copy rate): K and V converted
// to f16 in registers for m16n8k16 104 us, the same from rings in shared memory 108 us, m16n8k32 on e4m3 (which sm_100
// does not have: it is converted and issued as f16) 109 us: bound by the issue of conversions with few warps to hide them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kv8_attention.h"
#include "kv8_tensor.h"

namespace pf {
namespace {

constexpr int kThreads = 128, kTokens = 128, kGroups = kTokens / 16;   // tokens of a step, and of those that share a scale
constexpr float kShift = 6.f, kSlack = 2.f;

__host__ __device__ constexpr int few_ctas(int dim, int rows) {        // of an SM: by shared and by tensor memory
  return dim == 256 || rows == 64 ? 1 : rows == 32 ? 2 : dim == 128 ? 2 : 4;
}

// Offsets in shared memory behind the first 1024-byte boundary.  kWithV: attention; otherwise the weights, which read K only.
template <int kDim, int kRows, bool kWithV>
struct Few {
  static constexpr int kN = 4 * kRows;                                 // columns
  static constexpr int kKv = kWithV ? 2 : 1, kTile = kTokens * kDim, kStage = kKv * kTile;
  static constexpr int kP = 0, kQ = kP + (kWithV ? kTokens * kN : 0), kFirst = kQ + (kN * kDim < 1024 ? 1024 : kN * kDim);
  static constexpr int kRoom = 227 * 1024 / few_ctas(kDim, kRows) - 2 * 1024 - (kWithV ? 8 : 16) * 1024 - kFirst;   // Shared and Work
  static constexpr int kFit = kRoom / kStage, kStages = kFit > 4 ? 4 : kFit;
  static constexpr int kEnd = kFirst + kStages * kStage;
  static constexpr int kColumns = kN * (1 + (kWithV ? (kDim == 256 ? 2 : 1) : 0));
  static constexpr int kAlloc = kColumns <= 32 ? 32 : kColumns <= 64 ? 64 : kColumns <= 128 ? 128 : kColumns <= 256 ? 256 : 512;
  static_assert(kStages >= 2, "two tiles in flight");
  static_assert(kAlloc * few_ctas(kDim, kRows) <= 512, "tensor memory");
};

constexpr int kPass = 16;      // steps whose weights are summed over the row tiles before they are added
template <int kDim, int kRows, int kStages, bool kWithV>
struct FewShared {
  uint64_t s_full, pv_done;
  uint32_t tmem;
  int stalled, any_nan;
  float k_scale[kStages][kGroups], v_scale[kStages][kGroups];          // V's is -1 where there is no block
  float factor[kRows], ref[kRows], down[kRows], base[kRows], top[4][kRows], sum[4][kRows], v_top[4];
  int see[kRows];
  int nan_from[kDim];
  float weight[kWithV ? 1 : kPass][kThreads];
};

// Where 16-byte chunk c of row r lies: rows of 128 bytes (64 at 64 dimensions; two panels at 256) swizzled over eight rows.
template <int kDim>
__device__ __forceinline__ int place(int r, int c, int panel_rows) {
  if (kDim == 64) return r * 64 + 16 * (c ^ (r >> 1 & 3));
  return (c >> 3) * (panel_rows * 128) + r * 128 + 16 * ((c & 7) ^ (r & 7));
}

template <int kDim>
constexpr __host__ __device__ uint32_t swizzle_of() { return kDim == 64 ? kSwizzle64 : kSwizzle128; }

template <int kDim, int kRows, bool kWithV, bool kBf16>
__global__ void __launch_bounds__(kThreads, few_ctas(kDim, kRows)) kv8_attention_few(AttnParams p) {
  using L = Few<kDim, kRows, kWithV>;
  constexpr int kN = L::kN, kStages = L::kStages, kChunks = kRows / 4, kRowBytes = kDim == 64 ? 64 : 128;
  using SeqT = Seq<kRows, kTokens, !kWithV>;
  using SharedT = FewShared<kDim, kRows, kStages, kWithV>;
  extern __shared__ char raw[];
  char *smem = raw + (1024 - (shared_of(raw) & 1023));
  SharedT &sh = *reinterpret_cast<SharedT *>(smem + L::kEnd);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    bar_init(&sh.s_full, 1);
    bar_init(&sh.pv_done, 1);
    sh.stalled = 0;
    sh.any_nan = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_of(&sh.tmem)), "n"(L::kAlloc) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  for (int i = tid; i < kDim; i += kThreads) sh.nan_from[i] = INT_MAX;
  if (kWithV) after_previous();
  const Work<kRows, kTokens, !kWithV> work(p, reinterpret_cast<uint32_t *>(&sh + 1));
  if (!kWithV) after_previous();      // the kernel before it in the call has waited for what lens and starts come from
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem, lanes = tmem + ((uint32_t)warp * 32 << 16);
  const uint32_t at_p = shared_of(smem + L::kP), at_q = shared_of(smem + L::kQ), at_stage = shared_of(smem + L::kFirst);
  const Split split(work.total(), kWithV ? p.n_ctas : (int)gridDim.x);
  if (blockIdx.x == 0) {
    if (kWithV) check_batch(p);
    else
      for (int s = tid; s < p.batch.n_seqs; s += kThreads)
        if (p.batch.lens[s] > p.w_capacity) p.batch.report(PF_KV8_BAD_LENGTH);
  }
  uint32_t u = 0, u_end = 0;
  if ((int)blockIdx.x < split.n_ctas) u = split.begin(blockIdx.x), u_end = split.begin(blockIdx.x + 1);
  bool first_segment = true, ok = true;
  uint32_t n_scores = 0, n_outputs = 0;     // products waited for so far: phases of the two barriers
  const int within = p.cache.block_size() - 1;
  // a thread's copies: chunk `sub` of rows row_of, row_of + kAtOnce, ...
  constexpr int kLanes = kDim / 16, kAtOnce = kThreads / kLanes, kCopies = kTokens / kAtOnce;
  const int sub = tid % kLanes, row_of = tid / kLanes;

  while (u < u_end && ok) {
    const Segment seg(p, work, u);
    const int s = seg.s, head = seg.head;
    const SeqT seq(p, s);
    const uint32_t unit0 = u - seg.begin;
    const int all_rows = seq.all_rows(p);
    // Attention: one row tile.  Weights: all of them, one after the other, each over all units.
    const int tiles = kWithV ? 1 : (all_rows + kRows - 1) / kRows;
    const int units = (int)min(min(seg.units - unit0, u_end - u), tiles > 1 ? (uint32_t)kPass : 0xffffffffu);
    const int32_t *table = p.batch.tables + s * p.batch.table_stride;
    const char *tile_of[2] = {p.cache.base + head * p.cache.tile_bytes(), p.cache.base + p.cache.kv_stride + head * p.cache.tile_bytes()};
    const char *scale_of = p.cache.base + p.cache.heads * p.cache.tile_bytes() + 4 * head;
    if (tiles > 1)
      for (int j = 0; j < units; ++j) sh.weight[j][tid] = 0.f;         // a thread's own
    for (int tile = 0; tile < tiles && ok; ++tile) {
      const int row_first = (kWithV ? seg.rt : tile) * kRows, live_rows = min(all_rows - row_first, kRows);
      const int most = seq.visible(p, row_first + live_rows - 1);        // tokens that any row of the tile sees
      const int least = seq.visible(p, row_first);                       // tokens that all rows see
      const int tok0 = (int)(unit0 * kTokens), tok_end = min(seq.len, kWithV ? most : min(most, p.w_capacity));
      const int steps = max(0, min(units, (tok_end - tok0 + kTokens - 1) / kTokens));

      // pages of a step, looked up one step before they are asked for
      uint32_t page[kCopies];
      auto look_up = [&](int j) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int tok = tok0 + j * kTokens + i * kAtOnce + row_of;
          page[i] = tok < tok_end ? (uint32_t)table[tok >> p.cache.block_log2] : 0xffffffffu;
        }
      };
      auto ask = [&](int j) {             // always one group of copies
        if (j < steps) {
          const int stage = j % kStages, tok1 = tok0 + j * kTokens;
          const uint32_t dst = at_stage + stage * L::kStage;
#pragma unroll
          for (int i = 0; i < kCopies; ++i) {
            const int row = i * kAtOnce + row_of;
            // rows behind the last token, and of blocks that are not in the cache, become zeros
            const bool there = page[i] < p.cache.num_blocks && tok1 + row < seq.len;
            const uint64_t from = there ? (uint64_t)page[i] * (uint32_t)p.cache.block_stride + (uint32_t)(((tok1 + row) & within) * kDim + 16 * sub) : 0;
            const int bytes = there ? 16 : 0;
#pragma unroll
            for (int kv = 0; kv < L::kKv; ++kv)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + kv * L::kTile + place<kDim>(row, sub, kTokens)),
                           "l"(tile_of[kv] + from), "r"(bytes)
                           : "memory");
          }
          if (tid < kGroups) {
            const int tok = tok1 + 16 * tid;
            const uint32_t id = tok < tok_end ? (uint32_t)table[tok >> p.cache.block_log2] : 0xffffffffu;
            if (id < p.cache.num_blocks) {
              const char *at = scale_of + (uint64_t)id * (uint32_t)p.cache.block_stride;
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(shared_of(&sh.k_scale[stage][tid])), "l"(at) : "memory");
              if (kWithV)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(shared_of(&sh.v_scale[stage][tid])), "l"(at + p.cache.kv_stride) : "memory");
              else
                sh.v_scale[stage][tid] = 1.f;
            } else {
              if (tok < tok_end) p.batch.report(PF_KV8_BAD_BLOCK);
              sh.k_scale[stage][tid] = 0.f;
              sh.v_scale[stage][tid] = -1.f;
            }
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) {
        look_up(i);
        ask(i);
      }
      look_up(kStages - 1);

      // the rows' pieces, factors and lengths
      for (int e = tid; e < kRows * kLanes; e += kThreads) {
        const int r = e / kLanes, c = e % kLanes, row = row_first + r;
        const bool live = r < live_rows;
        const int i = live ? row / p.group : 0, qh = head * p.group + (live ? row % p.group : 0);
        const uint16_t *src = p.q + (int64_t)(seq.row0 + i) * p.q_row + qh * p.q_head + 16 * c;
        float x[16], top = 0.f;
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (live) {
            if (p.vec_q) w = *reinterpret_cast<const uint4 *>(src + k);
            else {
              const uint16_t *at = src + k;
              w = make_uint4(at[0] | at[1] << 16, at[2] | at[3] << 16, at[4] | at[5] << 16, at[6] | at[7] << 16);
            }
          }
          const uint32_t y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const float2 f = kBf16 ? make_float2(__uint_as_float(y[m] << 16), __uint_as_float(y[m] & 0xffff0000u)) : f32x2_from_f16x2(y[m]);
            x[k + 2 * m] = f.x, x[k + 2 * m + 1] = f.y;
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) top = fmaxf(top, __shfl_xor_sync(__activemask(), top, d));
        int ex = (int)(__float_as_uint(top) >> 23) - 127 - 7;
        if (top == 0.f || top > 3.4e38f) ex = 0;
        ex = max(ex, -126);
        const float down = exp2i(-ex);
        // an infinity would become 448
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = fabsf(x[k]) > 3.4e38f ? __int_as_float(0x7fffffff) : x[k] * down;
#pragma unroll
        for (int piece = 0; piece < 4; ++piece) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 16; k += 4) {
            const uint32_t lo = e4m3x2(x[k], x[k + 1]), hi = e4m3x2(x[k + 2], x[k + 3]);
            w[k / 4] = lo | hi << 16;
            const float2 a = f32x2_from_f16x2(f16x2_from_e4m3<0>(lo)), b = f32x2_from_f16x2(f16x2_from_e4m3<0>(hi));
            x[k] = (x[k] - a.x) * 16.f, x[k + 1] = (x[k + 1] - a.y) * 16.f;
            x[k + 2] = (x[k + 2] - b.x) * 16.f, x[k + 3] = (x[k + 3] - b.y) * 16.f;
          }
          const int n = 16 * (r / 4) + 4 * piece + r % 4;
          *reinterpret_cast<uint4 *>(smem + L::kQ + place<kDim>(n, c, kN)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (c == 0) {
          sh.factor[r] = p.scale * kLog2e * exp2i(ex);
          sh.see[r] = live ? seq.visible(p, row) : 0;
          sh.ref[r] = kNone;
          // rows that are not there, or see nothing, weigh nothing
          if (!kWithV) sh.base[r] = sh.see[r] > 0 ? p.lse[(int64_t)(seq.row0 + i) * p.q_heads + qh] * kLog2e : INFINITY;
        }
      }
      float sum[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) sum[r] = 0.f;
      float v_ref = 0.f;                     // 2^e_ref

      for (int j = 0; j < steps; ++j) {
        const int stage = j % kStages, tok1 = tok0 + j * kTokens, tok = tok1 + tid;
        const uint32_t at_k = at_stage + stage * L::kStage, at_v = at_k + L::kTile;
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        const bool partly = tok1 + kTokens > least;      // some row does not see all of it
        if (kWithV && partly) {
          // A NaN in V reaches the rows that see its token and no other: 0 * NaN would.  It is taken out, and the first such
          // token remembered for each dimension.  (A thread's own copies: no other has to be waited for.)
#pragma unroll 1
          for (int i = 0; i < kCopies; ++i) {
            const int row = i * kAtOnce + row_of;
            uint32_t *w = reinterpret_cast<uint32_t *>(smem + L::kFirst + stage * L::kStage + L::kTile + place<kDim>(row, sub, kTokens));
            uint32_t any = 0;
            for (int k = 0; k < 4; ++k) any |= (w[k] & 0x7f7f7f7fu) + 0x01010101u;
            if (!(any & 0x80808080u)) continue;
            sh.any_nan = 1;
            for (int k = 0; k < 16; ++k)
              if ((w[k / 4] >> (8 * (k % 4)) & 0x7f) == 0x7f) {
                atomicMin(&sh.nan_from[16 * sub + k], tok1 + row);
                w[k / 4] &= ~(0xffu << (8 * (k % 4)));
              }
          }
        }
        fence_to_async();
        fence_before();
        __syncthreads();
        if (tid == 0) {
          fence_after();
          constexpr uint32_t kShape = shape_of(kN, false, false);
#pragma unroll
          for (int k = 0; k < kDim / 32; ++k) {
            const uint32_t in = kDim == 64 ? k * 32 : k % 4 * 32;
            mma_e4m3_ss(tmem, operand(at_k + k / 4 * (kTokens * 128) + in, 16, 8 * kRowBytes, swizzle_of<kDim>()),
                        operand(at_q + k / 4 * (kN * 128) + in, 16, 8 * kRowBytes, swizzle_of<kDim>()), kShape, k != 0);
          }
          commit(&sh.s_full);
        }
        // the tile before is done with: its place is for the tile kStages - 1 ahead, and P for this one
        if (kWithV && j > 0) {
          ok = __syncthreads_and(bar_wait(&sh.pv_done, n_outputs++ & 1, &sh.stalled));
          if (!ok) break;
        }
        const float k_scale = sh.k_scale[stage][tid / 16], v_scale = sh.v_scale[stage][tid / 16];
        ok = __syncthreads_and(bar_wait(&sh.s_full, n_scores++ & 1, &sh.stalled));
        if (!ok) break;
        fence_after();
        ask(j + kStages - 1);
        look_up(j + kStages);
        const bool gone = v_scale < 0.f;
        auto scores = [&](int c, float (&x)[4]) {       // of rows 4 c .. 4 c + 3, for this thread's token
          uint32_t y[16];
          load16(y, lanes + 16 * c);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float lo = fmaf(__uint_as_float(y[12 + r]), 1.f / 16, __uint_as_float(y[8 + r]));
            x[r] = fmaf(fmaf(lo, 1.f / 16, __uint_as_float(y[4 + r])), 1.f / 16, __uint_as_float(y[r])) * (sh.factor[4 * c + r] * k_scale);
            if (partly || gone)
              if (gone || tok >= sh.see[4 * c + r]) x[r] = -INFINITY;
          }
        };
        if constexpr (!kWithV) {
          float w = 0.f;
#pragma unroll 2
          for (int c = 0; c < kChunks; ++c) {
            float x[4];
            scores(c, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) w += exp2_fast(x[r] - sh.base[4 * c + r]);
          }
          if (tiles > 1) sh.weight[j][tid] += w;
          else if (tok < tok_end && !gone) p.weights[s * p.w_seq + head * p.w_head + tok] += w;
        } else {
          float first[4];
          bool over = v_scale > v_ref;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            float x[4];
            scores(c, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              over |= x[r] > sh.ref[4 * c + r] + kSlack;
              if (c == 0) first[r] = x[r];
            }
          }
          if (__syncthreads_or(over)) {
            // new references: the largest scores of the tile, the largest of V's scales
            float v_top = v_scale;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, d));
            if (lane == 0) sh.v_top[warp] = v_top;
#pragma unroll 1
            for (int c = 0; c < kChunks; ++c) {
              float x[4];
              scores(c, x);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) x[r] = fmaxf(x[r], __shfl_xor_sync(0xffffffffu, x[r], d));
                if (lane == 0) sh.top[warp][4 * c + r] = x[r];
              }
            }
            __syncthreads();
            v_top = fmaxf(fmaxf(fmaxf(sh.v_top[0], sh.v_top[1]), fmaxf(sh.v_top[2], sh.v_top[3])), fmaxf(v_ref, 0x1p-110f));
            const float v_down = v_ref / v_top;          // powers of two; 0 at the start
            v_ref = v_top;
            if (tid < kRows) {
              const float was = sh.ref[tid];
              const float top = fmaxf(fmaxf(sh.top[0][tid], sh.top[1][tid]), fmaxf(sh.top[2][tid], sh.top[3][tid]));
              const float now = top > was + kSlack ? top : was;
              sh.ref[tid] = now;
              sh.down[tid] = exp2_fast(was - now);
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kRows; ++r) sum[r] *= sh.down[r];
            if (j > 0) {
#pragma unroll 1
              for (int half = 0; half < (kDim == 256 ? 2 : 1); ++half)
#pragma unroll 1
                for (int c = 0; c < kChunks; ++c) {
                  uint32_t y[16];
                  load16(y, lanes + kN * (1 + half) + 16 * c);
#pragma unroll
                  for (int k = 0; k < 16; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * (sh.down[4 * c + k % 4] * v_down));
                  store16(lanes + kN * (1 + half) + 16 * c, y);
                }
              wait_stores();
            }
          }
          // quotient of two powers of two, by their exponents; 0 where it is too small for any piece
          const float on_p = v_scale > v_ref * 0x1p-60f ? __int_as_float(0x3f800000 + __float_as_int(v_scale) - __float_as_int(v_ref)) : 0.f;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            float x[4];
            if (c == 0) x[0] = first[0], x[1] = first[1], x[2] = first[2], x[3] = first[3];
            else scores(c, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              x[r] = exp2_fast(x[r] - (sh.ref[4 * c + r] - kShift));
              sum[4 * c + r] += x[r];
            }
            uint32_t h[2] = {f16x2(x[0] * on_p, x[1] * on_p), f16x2(x[2] * on_p, x[3] * on_p)}, w[4];
#pragma unroll
            for (int piece = 0; piece < 4; ++piece) {
              w[piece] = e4m3x4_from_f16(h[0], h[1]);
              if (piece == 3) break;
              const uint32_t back[2] = {f16x2_from_e4m3<0>(w[piece]), f16x2_from_e4m3<1>(w[piece])};
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const __half2 left = __hmul2(__hsub2(*reinterpret_cast<const __half2 *>(&h[k]), *reinterpret_cast<const __half2 *>(&back[k])),
                                             __float2half2_rn(16.f));
                h[k] = *reinterpret_cast<const uint32_t *>(&left);
              }
            }
            *reinterpret_cast<uint4 *>(smem + L::kP + c * (kTokens * 16) + tid * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          fence_to_async();
          fence_before();
          __syncthreads();
          if (tid == 0) {
            fence_after();
            constexpr uint32_t kShape = shape_of(kN, true, true);
#pragma unroll
            for (int half = 0; half < (kDim == 256 ? 2 : 1); ++half)
#pragma unroll
              for (int k = 0; k < kTokens / 32; ++k)
                // at 64 dimensions the second half of the rows repeats the first: nobody reads it
                mma_e4m3_ss(tmem + kN * (1 + half), operand(at_v + half * (kTokens * 128) + k * 32 * kRowBytes, 0, 8 * kRowBytes, swizzle_of<kDim>()),
                            operand(at_p + k * 512, 128, kTokens * 16, kNoSwizzle), kShape, j > 0 || k != 0);
            commit(&sh.pv_done);
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if constexpr (kWithV) {
        if (ok && steps > 0) ok = __syncthreads_and(bar_wait(&sh.pv_done, n_outputs++ & 1, &sh.stalled));
        if (!ok) break;
        fence_after();
        // row sums over the threads
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], d);
          if (lane == 0) sh.sum[warp][r] = sum[r];
        }
        __syncthreads();
        const bool whole = units == (int)seg.units, any_nan = sh.any_nan;
        const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
#pragma unroll 1
        for (int half = 0; half < (kDim == 256 ? 2 : 1); ++half) {
          const int d = half * 128 + tid;
#pragma unroll 1
          for (int c = 0; c < (live_rows + 3) / 4; ++c) {
            uint32_t y[16];
            load16(y, lanes + kN * (1 + half) + 16 * c);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = 4 * c + k;
              if (r >= live_rows || d >= kDim) continue;
              const float l = sh.sum[0][r] + sh.sum[1][r] + sh.sum[2][r] + sh.sum[3][r];
              const float lo = fmaf(__uint_as_float(y[12 + k]), 1.f / 16, __uint_as_float(y[8 + k]));
              float a = fmaf(fmaf(lo, 1.f / 16, __uint_as_float(y[4 + k])), 1.f / 16, __uint_as_float(y[k])) * v_ref;
              if (steps == 0 || l == 0.f) a = 0.f;
              if (any_nan && sh.nan_from[d] < sh.see[r]) a = __int_as_float(0x7fffffff);
              const int row = row_first + r, i = row / p.group, qh = head * p.group + row % p.group;
              const float base = sh.ref[r] - kShift;
              if (whole) {
                a = l == 0.f ? a : a / l;
                uint16_t *dst = p.out + (int64_t)(seq.row0 + i) * p.out_row + qh * p.out_head + d;
                *dst = kBf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(a)) : __half_as_ushort(__float2half_rn(a));
                if (d == 0 && p.lse) p.lse[(int64_t)(seq.row0 + i) * p.q_heads + qh] = lse_of(base, l);
              } else {
                p.part_o[((int64_t)slot * kRows + r) * kDim + d] = a;
                if (d == 0) p.part_ml[slot * kRows + r] = make_float2(base, l);
              }
            }
          }
        }
        fence_before();
        __syncthreads();
        if (any_nan) {
          for (int i = tid; i < kDim; i += kThreads) sh.nan_from[i] = INT_MAX;
          if (tid == 0) sh.any_nan = 0;
        }
      }
      __syncthreads();         // the rows' pieces, factors and scales have been read
    }
    if (!kWithV && tiles > 1)
      for (int j = 0; j < units; ++j) {
        const int tok = (int)(unit0 + j) * kTokens + tid;
        if (tok < min(seq.len, p.w_capacity)) p.weights[s * p.w_seq + head * p.w_head + tok] += sh.weight[j][tid];
      }
    u += units;
    first_segment = false;
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (sh.stalled && tid == 0) p.batch.report(PF_KV8_STALLED);
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(L::kAlloc));
}

template <int kDim, int kRows, bool kWithV, bool kBf16>
void launch(const AttnParams &p, int n_ctas, cudaStream_t stream) {
  using L = Few<kDim, kRows, kWithV>;
  auto kernel = kv8_attention_few<kDim, kRows, kWithV, kBf16>;
  const size_t smem = 1024 + (size_t)L::kEnd + sizeof(FewShared<kDim, kRows, L::kStages, kWithV>) +
                      Work<kRows, kTokens, !kWithV>::bytes(p.batch.n_seqs, p.row_tiles_most);
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    throw Error::storage("cudaFuncSetAttribute failed");
  launch_after(kernel, n_ctas, kThreads, smem, stream, p);
}

template <int kDim, bool kBf16>
void launch(const AttnParams &p, int rows, cudaStream_t stream) {
  switch (rows) {
    case 4: return launch<kDim, 4, true, kBf16>(p, p.n_ctas, stream);
    case 8: return launch<kDim, 8, true, kBf16>(p, p.n_ctas, stream);
    case 16: return launch<kDim, 16, true, kBf16>(p, p.n_ctas, stream);
    default: return launch<kDim, 32, true, kBf16>(p, p.n_ctas, stream);
  }
}

}  // namespace

int kv8_few_rows(int64_t rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 0; }
int kv8_few_ctas(int dim, int rows) { return few_ctas(dim, rows); }

void kv8_few_launch(const AttnParams &p, int rows, bool bf16, cudaStream_t stream) {
  switch (p.cache.dim) {
    case 64: return bf16 ? launch<64, true>(p, rows, stream) : launch<64, false>(p, rows, stream);
    case 128: return bf16 ? launch<128, true>(p, rows, stream) : launch<128, false>(p, rows, stream);
    default: return bf16 ? launch<256, true>(p, rows, stream) : launch<256, false>(p, rows, stream);
  }
}

// weights[s, head, j] += sum over rows and group heads of exp(score - lse), once lse is known: the scores are taken again, from
// K alone.  Row tiles of 4 or, where there are more rows, of 16.  Each element has one writer, which adds in one order.
void kv8_weights_launch(const AttnParams &attention, bool bf16, int n_sms, cudaStream_t stream) {
  AttnParams p = attention;
  p.row_tiles_most = 1;
  const bool four = p.max_query * p.group <= 4;
  auto go = [&](auto dim, auto rows, auto type) {
    launch<decltype(dim)::value, decltype(rows)::value, false, decltype(type)::value>(
        p, n_sms * few_ctas(decltype(dim)::value, decltype(rows)::value), stream);
  };
  auto with_type = [&](auto dim, auto rows) { bf16 ? go(dim, rows, std::true_type{}) : go(dim, rows, std::false_type{}); };
  auto with_rows = [&](auto dim) {
    if (four) with_type(dim, std::integral_constant<int, 4>{});
    else with_type(dim, std::integral_constant<int, 16>{});
  };
  if (p.cache.dim == 64) with_rows(std::integral_constant<int, 64>{});
  else if (p.cache.dim == 128) with_rows(std::integral_constant<int, 128>{});
  else with_rows(std::integral_constant<int, 256>{});
}

}  // namespace pf
