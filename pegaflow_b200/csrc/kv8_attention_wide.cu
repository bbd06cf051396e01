// Attention over the 8-bit cache for many query rows (pf_kv8_attention): 256 rows of one KV head at a time on the
// tcgen05 tensor cores, sums in tensor memory.
//
// A CTA takes a row tile (two groups of 128 rows; one at 256 dimensions) along a range of tokens, kTokens per step:
//   converters  (4 warps)  read K8 and V8, turn them into f16 (exact) and lay them out in shared memory
//   issuer      (1 thread) S_g = Q_g K^T into tensor memory;  O_g += P_g V, with P_g read from tensor memory
//   softmax g   (4 warps)  a thread holds a row: scores out of tensor memory, running maximum, exponentials, P_g back into
//                          the columns that held S_g, as f16; corrects O_g when the maximum has risen by 2^6
// The two groups take turns: while one is in its exponentials, the other's products run.  Per step both cost about the same
// at 128 dimensions: 4 * 256 * 128 * 128 flops at 8192 a cycle and 256 * 128 exponentials at 16 a cycle are 2048
// cycles each.
//
// K and V have one layout in shared memory, rows of 128 bytes (64 dimensions) with 16-byte chunks swizzled over
// eight rows: as the operand of the scores its contracted index runs along the row, as the operand of the output it runs
// down the rows, which is the other of the two majors that a descriptor can name.
//
// Scales: K's goes on the scores, a block of 16 columns at a time.  V's, 2^e, goes on P: P holds
// 2^(score - ref + shift + e - e_ref), and O is in units of 2^e_ref; e_ref follows the largest e so far.  The row sums
// leave e out again.  All of these are powers of two.
#include <cuda_bf16.h>

#include "kv8_attention.h"
#include "kv8_tensor.h"

namespace pf {
namespace {

constexpr int kGroupRows = 128;
constexpr float kShift = 6.f, kSlack = 6.f;   // P <= 2^(6 + 6 + kRoom) = 2^15
constexpr int kRoom = 3;                      // by how much e may exceed e_ref
constexpr int kRing = 4;                      // steps of scales kept

constexpr int tokens_of(int dim) { return dim == 256 ? 64 : 128; }
constexpr int groups_of(int dim) { return dim == 256 ? 1 : 2; }
constexpr int threads_of(int dim) { return 128 * groups_of(dim) + 128 + 128; }   // whole warpgroups; the last one has the issuer

// Offsets in shared memory, behind the first 1024-byte boundary.
template <int kDim>
struct Layout {
  static constexpr int kTokens = tokens_of(kDim), kGroups = groups_of(kDim);
  static constexpr int q_bytes = kGroupRows * kDim * 2, kv_bytes = kTokens * kDim * 2, blocks = kTokens / 16;
  static constexpr int q = 0, k = q + kGroups * q_bytes, v = k + 2 * kv_bytes, end = v + 2 * kv_bytes;
};

struct Shared {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], scales_full[kRing];
  uint32_t tmem;
  int stalled, any_nan;
  float k_scale[kRing][8];
  int v_exp[kRing][8];       // exponent of V's scale; kHidden: the block is not in the cache
  int nan_from[256];         // first token whose V is NaN in a dimension
};
constexpr int kHidden = 1 << 20;

template <int kDim, bool kBf16>
__global__ void __launch_bounds__(threads_of(kDim), 1) kv8_attention_wide(AttnParams p) {
  using L = Layout<kDim>;
  constexpr int kTokens = L::kTokens, kGroups = L::kGroups, kRows = kGroupRows * kGroups, kBlocks = L::blocks;
  using SeqT = Seq<kRows, kTokens>;
  // columns of tensor memory: S and P of each group, then O of each group
  constexpr uint32_t kO = kDim == 256 ? 256 : 2 * kTokens;
  extern __shared__ char raw[];
  char *smem = raw + (1024 - (shared_of(raw) & 1023));
  Shared &sh = *reinterpret_cast<Shared *>(smem + L::end);
  uint32_t *prefix = reinterpret_cast<uint32_t *>(&sh + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kConvert = 4 * kGroups, kIssue = kConvert + 4;     // first warp of the converters, warp of the issuer

  if (tid == 0) {
    bar_init(&sh.q_full, kRows);
    for (int i = 0; i < 2; ++i) {
      bar_init(&sh.k_full[i], 128);
      bar_init(&sh.k_empty[i], 1);
      bar_init(&sh.v_full[i], 128);
      bar_init(&sh.v_empty[i], 1);
      bar_init(&sh.s_full[i], 1);
      bar_init(&sh.p_full[i], kGroupRows);
      bar_init(&sh.o_full[i], 1);
    }
    for (int i = 0; i < kRing; ++i) bar_init(&sh.scales_full[i], kBlocks);
    sh.stalled = 0;
    sh.any_nan = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = tid; i < kDim; i += blockDim.x) sh.nan_from[i] = INT_MAX;
  if (warp == kIssue) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_of(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  after_previous();
  const Work<kRows, kTokens> work(p, prefix);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  const Split split(work.total(), p.n_ctas);
  if (blockIdx.x == 0) check_batch(p);
  uint32_t u = 0, u_end = 0;
  if ((int)blockIdx.x < split.n_ctas) u = split.begin(blockIdx.x), u_end = split.begin(blockIdx.x + 1);
  bool first_segment = true;
  uint32_t step = 0;          // steps done in earlier segments: all roles count alike
  uint32_t n_segment = 0;
  bool ok = true;
  // Every role walks the CTA's segments by itself; behind each all threads meet.
  auto walk = [&](auto &&role) {
    while (u < u_end && ok) {
      const Segment seg(p, work, u);
      const uint32_t unit0 = u - seg.begin, units = min(seg.units - unit0, u_end - u);
      const SeqT seq(p, seg.s);
      const int row_first = seg.rt * kRows;
      role(seg, seq, unit0, units, row_first, min(seq.all_rows(p) - row_first, kRows));
      step += units;
      ++n_segment;
      u += units;
      first_segment = false;
      __syncwarp();
      // every thread is through with this segment's marks before the next one sets them
      if (u < u_end) {
        if (__syncthreads_or(sh.stalled)) break;
        if (sh.any_nan) {
          __syncthreads();
          for (int k = tid; k < kDim; k += blockDim.x) sh.nan_from[k] = INT_MAX;
          if (tid == 0) sh.any_nan = 0;
        }
        __syncthreads();
      }
    }
  };
  // Two groups: 512 threads start with 128 registers each, and 256 x 184 + 128 x 104 + 128 x 40 are as many.
  if (warp < kConvert) {
    if (kGroups == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    walk([&](const Segment &seg, const SeqT &seq, uint32_t unit0, uint32_t units, int row_first, int live_rows) {
      const int head = seg.head;
      // ------------------------------------------------------------------ softmax: a thread holds a row
      const int g = warp >> 2, r = (warp & 3) * 32 + lane;
      const int row = row_first + g * kGroupRows + r;
      const bool live = row < row_first + live_rows;
      const int i = live ? row / p.group : 0, qh = head * p.group + (live ? row % p.group : 0);
      const int see = live ? seq.visible(p, row) : 0;
      const int group_least = g * kGroupRows < live_rows ? seq.visible(p, row_first + g * kGroupRows) : 0;
      const bool dead = g * kGroupRows + (warp & 3) * 32 >= live_rows;   // no row of this warp counts
      // the row into shared memory, a power of two (and the scale's sign) taken off it
      float factor;
      {
        const uint16_t *src = p.q + (int64_t)(seq.row0 + i) * p.q_row + qh * p.q_head;
        char *dst = smem + L::q + g * L::q_bytes + r * 128;
        auto read8 = [&](int d) {
          if (!live) return make_uint4(0, 0, 0, 0);
          const uint16_t *at = src + d;
          if (p.vec_q) return *reinterpret_cast<const uint4 *>(at);
          return make_uint4(at[0] | at[1] << 16, at[2] | at[3] << 16, at[4] | at[5] << 16, at[6] | at[7] << 16);
        };
        auto wide2 = [](uint32_t two) {
          if (kBf16) return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
          return f32x2_from_f16x2(two);
        };
        float top = 0.f;
        for (int d = 0; d < kDim; d += 8) {
          const uint4 w = read8(d);
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const float2 f = wide2(x[m]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        int e = (int)(__float_as_uint(top) >> 23) - 127 - 14;
        if (top == 0.f || top > 3.4e38f) e = 0;
        e = max(e, -126);
        const float down = exp2i(-e) * (p.scale < 0.f ? -1.f : 1.f);
        factor = fabsf(p.scale) * kLog2e * exp2i(e);
        for (int d = 0; d < kDim; d += 8) {
          const uint4 w = read8(d);
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
          uint32_t h[4];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const float2 f = wide2(x[m]);
            h[m] = f16x2(f.x * down, f.y * down);
          }
          *reinterpret_cast<uint4 *>(dst + d / 64 * (kGroupRows * 128) + ((d / 8 % 8) ^ (r & 7)) * 16) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_to_async();
        bar_arrive(&sh.q_full);
      }
      const uint32_t lanes = tmem + ((uint32_t)(warp & 3) * 32 << 16);
      const uint32_t s_col = lanes + g * kTokens, o_col = lanes + kO + g * kDim;
      float ref = kNone, sum = 0.f;
      int e_ref = 0;
      for (uint32_t j = 0; j < units; ++j) {
        const uint32_t at = step + j, ring = at % kRing;
        const int tok = (int)((unit0 + j) * kTokens);
        if (!(ok = bar_wait_warp(&sh.scales_full[ring], at / kRing & 1, &sh.stalled))) break;
        if (!(ok = bar_wait_warp(&sh.s_full[g], at & 1, &sh.stalled))) break;
        fence_after();
        if (!dead) {
          uint32_t x[kTokens];
          load_all(x, s_col);
          const float *ks = sh.k_scale[ring];
          const int *ve = sh.v_exp[ring];
          // Rows that do not see the tile whole, blocks that are not there: -infinity, before anything else.  The factors below
          // are positive, so that it stays that.
          int e_top = kKv8MinExp, gone = 0;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            if (ve[b] == kHidden) gone |= 1 << b;
            else e_top = max(e_top, ve[b]);
          }
          if (tok + kTokens > group_least || gone) {
            const int n = see - tok;
#pragma unroll
            for (int k = 0; k < kTokens; ++k)
              if (k >= n || (gone >> (k / 16) & 1)) x[k] = 0xff800000u;
          }
          auto factor_of = [&](int b) { return fmaxf(factor * ks[b], 1e-37f); };
          float top = kNone;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            float m = __uint_as_float(x[16 * b]);
#pragma unroll
            for (int k = 1; k < 15; k += 2) m = fmaxf(fmaxf(m, __uint_as_float(x[16 * b + k])), __uint_as_float(x[16 * b + k + 1]));
            top = fmaxf(top, fmaxf(m, __uint_as_float(x[16 * b + 15])) * factor_of(b));
          }
          // both references, and O with them
          const bool start = j == 0;
          if (start) e_ref = e_top;
          float down = 1.f;
          bool change = false;
          if (top > ref + kSlack) {
            if (!start) down = exp2_fast(ref - top), change = true;
            sum *= exp2_fast(ref - top);
            ref = top;
          }
          if (e_top > e_ref + kRoom) {
            down *= exp2i(e_ref - e_top);
            change = true;
            e_ref = e_top;
          }
          if (__any_sync(0xffffffffu, change)) {
#pragma unroll 1
            for (int c = 0; c < kDim / 16; ++c) {
              uint32_t y[16];
              load16(y, o_col + 16 * c);
#pragma unroll
              for (int k = 0; k < 16; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * down);
              store16(o_col + 16 * c, y);
            }
          }
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            // 2^-60 of the largest scale leaves nothing of P in f16; the row sum still has it
            const int de = gone >> b & 1 ? 0 : max(ve[b] - e_ref, -60);
            const float fb = factor_of(b), minus = kShift + (float)de - ref;
            const uint64_t fb2 = pair(fb, fb), minus2 = pair(minus, minus);
            uint64_t part = pair(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              float lo, hi;
              unpair(fma2(pair(__uint_as_float(x[16 * b + k]), __uint_as_float(x[16 * b + k + 1])), fb2, minus2), lo, hi);
              lo = exp2_fast(lo), hi = exp2_fast(hi);
              part = add2(part, pair(lo, hi));
              x[8 * b + k / 2] = f16x2(lo, hi);
            }
            float lo, hi;
            unpair(part, lo, hi);
            sum = fmaf(lo + hi, exp2i(-de), sum);
          }
#pragma unroll
          for (int c = 0; c < kTokens / 32; ++c) {
            uint32_t h[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) h[k] = x[16 * c + k];
            store16(s_col + 16 * c, h);
          }
          wait_stores();
        }
        fence_before();
        bar_arrive(&sh.p_full[g]);
      }
      if (ok) ok = bar_wait_warp(&sh.o_full[g], n_segment & 1, &sh.stalled);
      const uint32_t last = step + units - 1;       // what the converters noted of NaN is seen behind their last arrival
      if (ok) ok = bar_wait_warp(&sh.v_full[last & 1], last >> 1 & 1, &sh.stalled);
      if (ok) {
        fence_after();
        const bool whole = units == seg.units;
        const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1), n = g * kGroupRows + r;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const bool nan = sh.any_nan;
        uint16_t *dst = p.out + (int64_t)(seq.row0 + i) * p.out_row + qh * p.out_head;
        float *part = p.part_o + ((int64_t)slot * kRows + n) * kDim;
        if (!dead) {
          for (int c = 0; c < kDim / 32; ++c) {
            uint32_t x[32];
            load32(x, o_col + 32 * c);
            // O is in units of 2^e_ref; the two factors are applied one after the other, their product may leave the range
            const float unit = exp2i(e_ref);
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              float y = sum == 0.f ? 0.f : __uint_as_float(x[k]) * unit;
              if (whole) y *= inv;
              if (nan && sh.nan_from[32 * c + k] < see) y = __int_as_float(0x7fffffff);
              x[k] = __float_as_uint(y);
            }
            if (!live) continue;
            if (whole) {
              if (p.vec_out) {
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                  const float *y = reinterpret_cast<const float *>(x) + k;
                  uint2 w;
                  if (kBf16) {
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w.x) : "f"(y[1]), "f"(y[0]));
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w.y) : "f"(y[3]), "f"(y[2]));
                  } else {
                    w = make_uint2(f16x2(y[0], y[1]), f16x2(y[2], y[3]));
                  }
                  *reinterpret_cast<uint2 *>(dst + 32 * c + k) = w;
                }
              } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  const float y = __uint_as_float(x[k]);
                  dst[32 * c + k] = kBf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(y)) : __half_as_ushort(__float2half_rn(y));
                }
              }
            } else {
#pragma unroll
              for (int k = 0; k < 32; k += 4) *reinterpret_cast<uint4 *>(part + 32 * c + k) = make_uint4(x[k], x[k + 1], x[k + 2], x[k + 3]);
            }
          }
        }
        if (live) {
          if (!whole) p.part_ml[slot * kRows + n] = make_float2(ref - kShift, sum);
          else if (p.lse) p.lse[(int64_t)(seq.row0 + i) * p.q_heads + qh] = lse_of(ref - kShift, sum);
        }
        fence_before();
      }
    });
  } else if (warp < kIssue) {
    if (kGroups == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    walk([&](const Segment &seg, const SeqT &seq, uint32_t unit0, uint32_t units, int, int) {
      const int s = seg.s, head = seg.head;
      // ------------------------------------------------------------------ converters
      constexpr int kLanes = kDim / 16, kVecs = kTokens * kLanes / 128;      // lanes of a row, 16-byte vectors of a thread
      const int ct = tid - kConvert * 32, sub = ct % kLanes, row_of = ct / kLanes;
      const int within = p.cache.block_size() - 1, tok_stop = seq.len;
      const int32_t *table = p.batch.tables + s * p.batch.table_stride;
      const char *tile_of[2] = {p.cache.base + head * p.cache.tile_bytes() + 16 * sub, p.cache.base + p.cache.kv_stride + head * p.cache.tile_bytes() + 16 * sub};
      auto look_up = [&](uint32_t j, uint32_t (&id)[kVecs]) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const int tok = (int)((unit0 + j) * kTokens) + v * (128 / kLanes) + row_of;
          id[v] = j < units && tok < tok_stop ? (uint32_t)table[tok >> p.cache.block_log2] : 0xffffffffu;
        }
      };
      auto fetch = [&](int kv, uint32_t j, const uint32_t (&id)[kVecs], uint4 (&x)[kVecs]) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const int tok = (int)((unit0 + j) * kTokens) + v * (128 / kLanes) + row_of;
          x[v] = make_uint4(0, 0, 0, 0);
          if (id[v] < p.cache.num_blocks)
            x[v] = __ldg(reinterpret_cast<const uint4 *>(tile_of[kv] + (uint64_t)id[v] * (uint32_t)p.cache.block_stride + (tok & within) * kDim));
        }
      };
      auto lay = [&](char *base, const uint4 (&x)[kVecs]) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const int t = v * (128 / kLanes) + row_of;
          char *dst = base + sub / 4 * (kTokens * 128) + t * 128;
          const uint4 a = make_uint4(f16x2_from_e4m3<0>(x[v].x), f16x2_from_e4m3<1>(x[v].x), f16x2_from_e4m3<0>(x[v].y), f16x2_from_e4m3<1>(x[v].y));
          const uint4 b = make_uint4(f16x2_from_e4m3<0>(x[v].z), f16x2_from_e4m3<1>(x[v].z), f16x2_from_e4m3<0>(x[v].w), f16x2_from_e4m3<1>(x[v].w));
          // lanes of odd panels store their second half first: eight lanes then fill eight different chunks
          const int c = 2 * (sub % 4), odd = sub / 4 & 1;
          *reinterpret_cast<uint4 *>(dst + ((c + odd) ^ (t & 7)) * 16) = odd ? b : a;
          *reinterpret_cast<uint4 *>(dst + ((c + 1 - odd) ^ (t & 7)) * 16) = odd ? a : b;
        }
        fence_to_async();
      };
      // pages a tile ahead of K, which is a tile ahead of V
      uint4 kx[kVecs], vx[kVecs];
      uint32_t id[kVecs], next[kVecs];
      look_up(0, id);
      look_up(1, next);
      fetch(0, 0, id, kx);
      for (uint32_t j = 0; j < units; ++j) {
        const uint32_t at = step + j, stage = at & 1;
        fetch(1, j, id, vx);
        if (!(ok = bar_wait(&sh.k_empty[stage], (at >> 1 & 1) ^ 1, &sh.stalled))) break;
        if (ct < kBlocks) {
          const int tok = (int)((unit0 + j) * kTokens) + 16 * ct;
          uint32_t id;
          float ks = 0.f;
          int ve = kHidden;
          if (tok < tok_stop) {
            if (p.batch.block(p.cache, s, tok >> p.cache.block_log2, id)) {
              ks = __ldg(p.cache.scale(0, id, head));
              ve = kv8_scale_exponent(__ldg(p.cache.scale(1, id, head)));
            } else {
              p.batch.report(PF_KV8_BAD_BLOCK);
            }
          }
          sh.k_scale[at % kRing][ct] = ks;
          sh.v_exp[at % kRing][ct] = ve;
          bar_arrive(&sh.scales_full[at % kRing]);
        }
        lay(smem + L::k + stage * L::kv_bytes, kx);
        bar_arrive(&sh.k_full[stage]);
#pragma unroll
        for (int v = 0; v < kVecs; ++v) id[v] = next[v];
        if (j + 1 < units) fetch(0, j + 1, id, kx);
        look_up(j + 2, next);
        // A NaN in V reaches the rows that see its token and no other: it is taken out here and remembered.
        bool any = false;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const uint32_t w[4] = {vx[v].x, vx[v].y, vx[v].z, vx[v].w};
#pragma unroll
          for (int m = 0; m < 4; ++m) any |= __vcmpeq4(w[m] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
        }
        if (any) {
          sh.any_nan = 1;
#pragma unroll
          for (int v = 0; v < kVecs; ++v) {
            uint32_t *w = reinterpret_cast<uint32_t *>(&vx[v]);
            const int tok = (int)((unit0 + j) * kTokens) + v * (128 / kLanes) + row_of;
            for (int b = 0; b < 16; ++b)
              if ((w[b / 4] >> (8 * (b % 4)) & 0x7f) == 0x7f) {
                atomicMin(&sh.nan_from[16 * sub + b], tok);
                w[b / 4] &= ~(0xffu << (8 * (b % 4)));
              }
          }
        }
        if (!(ok = bar_wait(&sh.v_empty[stage], (at >> 1 & 1) ^ 1, &sh.stalled))) break;
        lay(smem + L::v + stage * L::kv_bytes, vx);
        bar_arrive(&sh.v_full[stage]);
      }
    });
  } else {
    if (kGroups == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    walk([&](const Segment &, const SeqT &, uint32_t, uint32_t units, int, int live_rows) {
      if (warp != kIssue || lane != 0) return;
      // ------------------------------------------------------------------ issuer
      constexpr uint32_t kScores = shape_f16(kTokens, false), kOutput = shape_f16(kDim, true);
      auto scores = [&](int g, uint32_t stage) {
        const uint32_t a = shared_of(smem + L::q + g * L::q_bytes), b = shared_of(smem + L::k + stage * L::kv_bytes);
#pragma unroll
        for (int k = 0; k < kDim / 16; ++k)
          mma_f16_ss(tmem + g * kTokens, operand(a + k / 4 * (kGroupRows * 128) + k % 4 * 32, 16, 1024, kSwizzle128),
                 operand(b + k / 4 * (kTokens * 128) + k % 4 * 32, 16, 1024, kSwizzle128), kScores, k != 0);
      };
      auto output = [&](int g, uint32_t stage, bool add) {
        const uint32_t b = shared_of(smem + L::v + stage * L::kv_bytes);
#pragma unroll
        for (int k = 0; k < kTokens / 16; ++k)
          mma_f16_ts(tmem + kO + g * kDim, tmem + g * kTokens + 8 * k, operand(b + k * 2048, kTokens * 128, 1024, kSwizzle128), kOutput, add || k != 0);
      };
      const int n_groups = live_rows > kGroupRows ? 2 : 1;
      ok = bar_wait(&sh.q_full, n_segment & 1, &sh.stalled);
      for (uint32_t j = 0; j <= units && ok; ++j) {
        const uint32_t at = step + j, before = at - 1;
        if (j < units && !(ok = bar_wait(&sh.k_full[at & 1], at >> 1 & 1, &sh.stalled))) break;
        for (int g = 0; g < kGroups; ++g) {
          if (j > 0) {
            if (!(ok = bar_wait(&sh.p_full[g], before & 1, &sh.stalled))) break;
            if (!(ok = bar_wait(&sh.v_full[before & 1], before >> 1 & 1, &sh.stalled))) break;
            fence_after();
            if (g < n_groups) output(g, before & 1, j > 1);
            if (g == kGroups - 1) commit(&sh.v_empty[before & 1]);
            if (j == units) commit(&sh.o_full[g]);
          }
          if (j < units) {
            fence_after();
            if (g < n_groups) scores(g, at & 1);
            commit(&sh.s_full[g]);
            if (g == kGroups - 1) commit(&sh.k_empty[at & 1]);
          }
        }
      }
    });
  }
  // Everything that was issued has completed (the last commit was waited for), or a wait ran out.
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (sh.stalled && tid == 0) p.batch.report(PF_KV8_STALLED);
  if (warp == kIssue) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int kDim, bool kBf16>
void launch(const AttnParams &p, cudaStream_t stream) {
  auto kernel = kv8_attention_wide<kDim, kBf16>;
  const size_t smem = kv8_wide_plan(kDim).smem + Work<kGroupRows * groups_of(kDim), tokens_of(kDim)>::bytes(p.batch.n_seqs, p.row_tiles_most);
  static std::atomic<uint64_t> asked;
  allow_smem(kernel, asked, p.device);
  launch_after(kernel, p.n_ctas, threads_of(kDim), smem, stream, p);
}

}  // namespace

static_assert(1024 + Layout<128>::end + sizeof(Shared) + 4 * (1024 + 1) + 128 <= 227 * 1024, "shared memory");
static_assert(Layout<256>::end <= Layout<128>::end && Layout<64>::end <= Layout<128>::end, "shared memory");

WidePlan kv8_wide_plan(int dim) {
  const int end = dim == 64 ? Layout<64>::end : dim == 128 ? Layout<128>::end : Layout<256>::end;
  return WidePlan{kGroupRows * groups_of(dim), threads_of(dim), 1024 + (size_t)end + sizeof(Shared)};
}

void kv8_wide_launch(const AttnParams &p, bool bf16, cudaStream_t stream) {
  switch (p.cache.dim) {
    case 64: return bf16 ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
    case 128: return bf16 ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
    default: return bf16 ? launch<256, true>(p, stream) : launch<256, false>(p, stream);
  }
}

}  // namespace pf
