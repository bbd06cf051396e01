// Attention over the 8-bit cache for many query rows (pf_kv8_attention): 256 rows of one KV head at a time on the
// tcgen05 tensor cores, sums in tensor memory.
//
// A CTA takes a row tile (two groups of 128 rows; one at 256 dimensions) along a range of tokens, kTokens per step:
//   converters  (8 warps)  read K8 and V8 a step ahead, turn them into f16 and lay them out in shared memory, two steps deep
//   issuer      (1 thread) S_g = Q_g K^T into tensor memory;  O_g += P_g V, with P_g read from tensor memory
//   softmax g   (4 warps)  a thread holds a row: scores out of tensor memory, exponentials, P_g back into the columns that held
//                          S_g, as f16.  P is taken against the reference that stands; only a row sum above 2^15 makes it look
//                          for the maximum, move the reference there, correct O_g and compute P again.
//   a thread looks up the sequence, tile and range that come next
// The two groups take turns: while one is in its exponentials, the other's products run.  Per step at 128 dimensions the
// products cost 4 * 256 * 128 * 128 flops at 8192 a cycle, the exponentials 256 * 128 at 16 a cycle and shared memory
// (operands of the products and the converters' stores) 256 KB at 128 a cycle: 2048 cycles each.
//
// What it measured (bf16, 128 dimensions, blocks of 16): 2048 new rows of 32 query and 8 KV heads behind 10240 tokens take 527 to
// 548 us on several GPUs, about 5500 cycles a step; without the exponentials 400 us, without the products 394 us, without the conversion 388 us, so
// that the three still wait for one another.  Four converter warps with half a step of loads in flight: 750 us.  One read of
// the scores for the maximum and one for P: 623 us.  Sequence and tile in registers instead of shared memory: 600 us, by
// spilled registers that the little L1 beside 227 KB of shared memory does not hold.
//
// K and V have one layout in shared memory, rows of 128 bytes (64 dimensions) with 16-byte chunks swizzled over
// eight rows: as the operand of the scores its contracted index runs along the row, as the operand of the output it runs
// down the rows, which is the other of the two majors that a descriptor can name.
//
// Roundings to f16: P, by 2^-11 of itself at most (the row sums take it before that), because the tensor cores take no fp32; Q is
// exact but for elements below 2^-28 of their row's largest.
//
// Scales, 2^e a block: the converters multiply K and V by 2^(e - e_ref) on the way, so that one unit holds for a step.  An e4m3
// number is a multiple of 2^-9 and below 2^9: in f16 it stays exact for e - e_ref from -15 to 7, and what is lost further
// down is below 2^-40 of the largest number of the tile.  K's e_ref is the largest e of the step less 7, and goes on the scores
// in fp32.  V's stays until a step has an e larger by more than 7; O, which is in units of 2^e_ref, then follows.
#include <cuda_bf16.h>

#include "kv8_attention.h"
#include "kv8_tensor.h"

namespace pf {
namespace {

constexpr int kGroupRows = 128;
constexpr float kShift = 6.f, kMost = 32768.f;   // P at the reference is 2^6; no row of a step adds up to more than 2^15
constexpr int kRoom = 7;                      // by how much e may exceed e_ref
constexpr int kRing = 4;                      // steps of scales kept

constexpr int tokens_of(int dim) { return dim == 256 ? 64 : 128; }
constexpr int groups_of(int dim) { return dim == 256 ? 1 : 2; }
constexpr int kConverters = 256;
constexpr int threads_of(int dim) { return 128 * groups_of(dim) + kConverters + 128; }   // whole warpgroups; the last one has the issuer

// Offsets in shared memory, behind the first 1024-byte boundary.
template <int kDim>
struct Layout {
  static constexpr int kTokens = tokens_of(kDim), kGroups = groups_of(kDim);
  static constexpr int q_bytes = kGroupRows * kDim * 2, kv_bytes = kTokens * kDim * 2, blocks = kTokens / 16;
  static constexpr int q = 0, k = q + kGroups * q_bytes, v = k + 2 * kv_bytes, end = v + 2 * kv_bytes;
};

// What a CTA does next: steps unit0 .. unit0 + units of one row tile.
struct Part {
  int s, head, row0, rows, len;          // sequence and KV head; its rows begin at row0 of the query, and their number
  int row_first, live_rows;              // rows (query * group + head of the group) of the tile
  uint32_t unit0, units;                 // units 0: nothing is left
  int whole, slot;                       // all of the tile's tokens, or a partial result in this slot
};
struct Shared {
  uint64_t q_full, full[2][2], empty[2][2], s_full[2], p_full[2], o_full[2], scales_full[kRing], drained;
  uint32_t tmem;
  int stalled, late, any_nan;
  Part part[2];
  float k_unit[kRing];       // 2^e_ref of K
  int v_ref[kRing];          // e_ref of V
  uint32_t gone[kRing];      // a bit for each 16 tokens that are not in the cache
  int nan_from[256];         // first token whose V is NaN in a dimension
};
// 16 bytes that no other load of this SM wants
__device__ __forceinline__ uint4 load_once(const void *at) {
  uint4 x;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(at));
  return x;
}
constexpr int kGone = -10000;   // exponent of what is not in the cache

// 2^e as a pair of f16, 0 below the subnormal ones.
__device__ __forceinline__ uint32_t f16_power(int e) {
  const uint32_t h = e >= -14 ? (uint32_t)(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0u;
  return h | h << 16;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// acc, or NaN once one of the finite numbers' places has held one.
__device__ __forceinline__ void note_nan(uint32_t &acc, uint32_t x) {
  asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(x), "r"(0u));
}

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
  constexpr int kConvert = 4 * kGroups, kIssue = kConvert + kConverters / 32;     // first warp of the converters, warp of the issuer

  if (tid == 0) {
    bar_init(&sh.q_full, kRows);
    for (int i = 0; i < 2; ++i) {
      for (int kv = 0; kv < 2; ++kv) {
        bar_init(&sh.full[kv][i], kConverters);
        bar_init(&sh.empty[kv][i], 1);
      }
      bar_init(&sh.s_full[i], 1);
      bar_init(&sh.p_full[i], kGroupRows);
      bar_init(&sh.o_full[i], 1);
    }
    for (int i = 0; i < kRing; ++i) bar_init(&sh.scales_full[i], 1);
    bar_init(&sh.drained, 1);
    sh.stalled = sh.late = 0;
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
  if (blockIdx.x == 0) check_batch(p);
  uint32_t step = 0, n_part = 0;      // steps and parts done: all roles count alike
  bool ok = true;
  // Every role goes through the CTA's parts by itself; before and behind each all threads meet.  What a part is stays in
  // shared memory: the registers are for the inner loops.
  auto walk = [&](auto &&role) {
    for (;;) {
      __syncthreads();
      const uint32_t units = sh.part[n_part & 1].units;
      if (units == 0) break;
      role(sh.part[n_part & 1], units);
      step += units;
      ++n_part;
      __syncwarp();
      // every thread is through with this part's marks before the next one sets them
      if (__syncthreads_or(sh.stalled)) break;
      if (sh.any_nan) {
        __syncthreads();
        for (int k = tid; k < kDim; k += blockDim.x) sh.nan_from[k] = INT_MAX;
        if (tid == 0) sh.any_nan = 0;
      }
    }
  };
  // Two groups: 640 threads start with 96 registers each, and 256 x 144 + 256 x 72 + 128 x 48 are as many.
  if (warp < kConvert) {
    if (kGroups == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    walk([&](const volatile Part &part, uint32_t units) {
      const uint32_t unit0 = part.unit0;
      const int live_rows = part.live_rows;
      // ------------------------------------------------------------------ softmax: a thread holds a row
      const int g = warp >> 2, r = (warp & 3) * 32 + lane;
      // tokens that a row of the tile sees
      auto visible = [&](int row) {
        const int len = part.len, rows = part.rows;
        return p.causal && rows > 1 ? min(max(len - rows + (part.row_first + row) / p.group + 1, 0), len) : len;
      };
      const bool live = g * kGroupRows + r < live_rows;
      const int see = live ? visible(g * kGroupRows + r) : 0;
      const int group_least = g * kGroupRows < live_rows ? visible(g * kGroupRows) : 0;
      const bool dead = g * kGroupRows + (warp & 3) * 32 >= live_rows;   // no row of this warp counts
      // Q into shared memory, a power of two (and the scale's sign) taken off each row: kDim / 8 lanes read a row
      // where the thread's row is in an array of rows and heads
      auto at_row = [&](int64_t row_stride, int64_t head_stride) {
        const int row = part.row_first + g * kGroupRows + r, i = live ? row / p.group : 0;
        return (part.row0 + i) * row_stride + (part.head * p.group + (live ? row - i * p.group : 0)) * head_stride;
      };
      const int live_here = min(live_rows - g * kGroupRows - (warp & 3) * 32, 32);
      float factor;
      {
        constexpr int kPer = kDim / 8, kAtOnce = 32 / kPer;
        const int64_t q_at = at_row(p.q_row, p.q_head);
        char *dst = smem + L::q + g * L::q_bytes + lane % kPer / 8 * (kGroupRows * 128);
        auto wide2 = [](uint32_t two) {
          if (kBf16) return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
          return f32x2_from_f16x2(two);
        };
        int e_row = 0;
#pragma unroll 1
        for (int t0 = 0; t0 < 32; t0 += 4 * kAtOnce) {
          uint4 w[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int t = t0 + n * kAtOnce + lane / kPer;
            const uint16_t *at = p.q + __shfl_sync(0xffffffffu, q_at, t) + lane % kPer * 8;
            w[n] = make_uint4(0, 0, 0, 0);
            if (t < live_here) {
              if (p.vec_q) w[n] = *reinterpret_cast<const uint4 *>(at);
              else w[n] = make_uint4(at[0] | at[1] << 16, at[2] | at[3] << 16, at[4] | at[5] << 16, at[6] | at[7] << 16);
            }
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const uint32_t x[4] = {w[n].x, w[n].y, w[n].z, w[n].w};
            float top = 0.f;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const float2 f = wide2(x[m]);
              top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
#pragma unroll
            for (int m = kPer / 2; m; m /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
            int e = (int)(__float_as_uint(top) >> 23) - 127 - 14;
            if (top == 0.f || top > 3.4e38f) e = 0;
            e = max(e, -126);
            const float down = exp2i(-e) * (p.scale < 0.f ? -1.f : 1.f);
            uint32_t y[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const float2 f = wide2(x[m]);
              y[m] = f16x2(f.x * down, f.y * down);
            }
            const int first = t0 + n * kAtOnce, row_in = (warp & 3) * 32 + first + lane / kPer;
            *reinterpret_cast<uint4 *>(dst + row_in * 128 + (lane % 8 ^ (row_in & 7)) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
            const int mine = __shfl_sync(0xffffffffu, e, (lane & (kAtOnce - 1)) * kPer);
            if (lane / kAtOnce == first / kAtOnce) e_row = mine;
          }
        }
        factor = fabsf(p.scale) * kLog2e * exp2i(e_row);
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
        const float unit = fmaxf(factor * sh.k_unit[ring], 1e-37f);   // positive, so that minus infinity stays it
        const int v_ref = sh.v_ref[ring];
        const uint32_t gone = sh.gone[ring];
        const bool partly = tok + kTokens > group_least || gone;      // not all of the tile for every row
        const bool start = j == 0;
        if (start) e_ref = v_ref;
        float down = exp2i(e_ref - v_ref);                            // for O, before this step is added
        e_ref = v_ref;
        if (!(ok = bar_wait_warp(&sh.s_full[g], at & 1, &sh.stalled))) break;
        fence_after();
        if (!dead) {
          if (partly) {             // what the row does not see becomes minus infinity, in tensor memory
#pragma unroll 1
            for (int c = 0; c < kTokens / 16; ++c) {
              const int n = gone >> c & 1 ? 0 : see - tok - 16 * c;
              uint32_t x[16];
              load16(x, s_col + 16 * c);
#pragma unroll
              for (int k = 0; k < 16; ++k) x[k] = k < n ? x[k] : 0xff800000u;
              store16(s_col + 16 * c, x);
            }
            wait_stores();
          }
          const uint64_t unit2 = pair(unit, unit);
          uint32_t h[kTokens / 2];
          float total;
          // P against the reference that stands.  A sum that is not too large has no entry that is: only behind one that is
          // the row's maximum is looked for, and P computed once more.
          for (bool again = false;; again = true) {
            const uint64_t minus2 = pair(kShift - ref, kShift - ref);
            uint64_t part[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
            for (int c0 = 0; c0 < kTokens; c0 += 32) {
              uint32_t x[32];
              load32(x, s_col + c0);
#pragma unroll
              for (int k = 0; k < 32; k += 2) {
                float lo, hi;
                unpair(fma2(pair(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), unit2, minus2), lo, hi);
                lo = exp2_fast(lo), hi = exp2_fast(hi);
                part[k / 2 & 1] = add2(part[k / 2 & 1], pair(lo, hi));
                h[(c0 + k) / 2] = f16x2(lo, hi);
              }
            }
            float lo, hi;
            unpair(add2(part[0], part[1]), lo, hi);
            total = lo + hi;
            if (again || !__any_sync(0xffffffffu, !(total <= kMost))) break;
            float top = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < kTokens / 16; ++c) {
              uint32_t x[16];
              load16(x, s_col + 16 * c);
#pragma unroll
              for (int k = 0; k < 16; ++k) top = fmaxf(top, __uint_as_float(x[k]));
            }
            top *= unit;
            if (!(total <= kMost) && top > ref) {
              const float by = exp2_fast(ref - top);
              down *= by;
              sum *= by;
              ref = top;
            }
          }
          sum += total;
          if (!start && __any_sync(0xffffffffu, down != 1.f)) {
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
          for (int c = 0; c < kTokens / 32; ++c) store16(s_col + 16 * c, *reinterpret_cast<uint32_t(*)[16]>(&h[16 * c]));
          wait_stores();
        }
        fence_before();
        bar_arrive(&sh.p_full[g]);
      }
      if (ok) ok = bar_wait_warp(&sh.o_full[g], n_part & 1, &sh.stalled);
      const uint32_t last = step + units - 1;       // what the converters noted of NaN is seen behind their last arrival
      if (ok) ok = bar_wait_warp(&sh.full[1][last & 1], last >> 1 & 1, &sh.stalled);
      if (ok) {
        fence_after();
        const bool whole = part.whole;
        const int slot = part.slot, n = g * kGroupRows + r;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const bool nan = sh.any_nan;
        const int64_t out_at = at_row(p.out_row, p.out_head);
        // 32 rows x 32 dimensions at a time by way of the shared memory that held these rows of Q: whole lines go out
        char *stage = smem + L::q + g * L::q_bytes + (warp & 3) * 32 * 128;
        if (!dead) {
          const float unit = exp2i(e_ref);
#pragma unroll 1
          for (int c = 0; c < kDim / 32; ++c) {
            uint32_t x[32];
            load32(x, o_col + 32 * c);
            // O is in units of 2^e_ref; the two factors are applied one after the other, their product may leave the range
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              float y = sum == 0.f ? 0.f : __uint_as_float(x[k]) * unit;
              if (whole) y *= inv;
              if (nan && sh.nan_from[32 * c + k] < see) y = __int_as_float(0x7fffffff);
              x[k] = __float_as_uint(y);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 8; ++k)
              *reinterpret_cast<uint4 *>(stage + lane * 128 + (k ^ (lane & 7)) * 16) = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int t = 4 * k + lane / 8, d = 32 * c + lane % 8 * 4;
              const float4 y = *reinterpret_cast<const float4 *>(stage + t * 128 + (lane % 8 ^ (t & 7)) * 16);
              uint16_t *dst = p.out + __shfl_sync(0xffffffffu, out_at, t) + d;
              if (t >= live_here) continue;
              if (!whole) {
                *reinterpret_cast<float4 *>(p.part_o + ((int64_t)slot * kRows + n - lane + t) * kDim + d) = y;
              } else {
                const uint2 w = make_uint2(narrow2<kBf16>(y.x, y.y), narrow2<kBf16>(y.z, y.w));
                if (p.vec_out) {
                  *reinterpret_cast<uint2 *>(dst) = w;
                } else {
                  dst[0] = (uint16_t)w.x, dst[1] = (uint16_t)(w.x >> 16), dst[2] = (uint16_t)w.y, dst[3] = (uint16_t)(w.y >> 16);
                }
              }
            }
          }
          __syncwarp();
        }
        if (live) {
          if (!whole) p.part_ml[slot * kRows + n] = make_float2(ref - kShift, sum);
          else if (p.lse) p.lse[at_row(p.q_heads, 1)] = lse_of(ref - kShift, sum);
        }
        fence_before();
      }
    });
  } else if (warp < kIssue) {
    if (kGroups == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    walk([&](const volatile Part &part, uint32_t units) {
      const int s = part.s, head = part.head;
      const uint32_t unit0 = part.unit0;
      // ------------------------------------------------------------------ converters
      constexpr int kLanes = kDim / 16, kVecs = kTokens * kLanes / kConverters, kStride = kConverters / kLanes;
      // a thread has 16 dimensions of kVecs tokens, kStride apart; a lane looks after the block and the scale of 16 tokens
      const int ct = tid - kConvert * 32, sub = ct % kLanes, row_of = ct / kLanes;
      const int mine = lane & 7, mine_kv = lane >> 3 & 1;
      const int within = p.cache.block_size() - 1, tok_stop = part.len;
      const int32_t *table = p.batch.tables + s * p.batch.table_stride;
      const char *tile_of = p.cache.base + head * p.cache.tile_bytes() + 16 * sub;
      auto look_up = [&](uint32_t j) {
        const int tok = (int)((unit0 + j) * kTokens) + 16 * mine;
        return j < units && mine < kBlocks && tok < tok_stop ? (uint32_t)__ldg(table + (tok >> p.cache.block_log2)) : 0xffffffffu;
      };
      auto scale_of = [&](uint32_t id) { return id < p.cache.num_blocks ? __ldg(p.cache.scale(mine_kv, id, head)) : 0.f; };
      auto block_of = [&](int v) { return (v * kStride + row_of) / 16; };
      // What is not there is read from block 0 instead and multiplied by 0, what lies behind the last token is read as it is: no
      // row sees either, so that all they must not be is NaN.
      auto fetch = [&](int kv, uint32_t j, uint32_t ids, uint4 (&x)[kVecs]) {
        const char *tile = tile_of + (kv ? p.cache.kv_stride : 0);
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const int tok = (int)((unit0 + j) * kTokens) + v * kStride + row_of;
          const uint32_t id = __shfl_sync(0xffffffffu, ids < p.cache.num_blocks ? ids : 0u, block_of(v));
          x[v] = load_once(tile + (uint64_t)id * (uint32_t)p.cache.block_stride + (tok & within) * kDim);
        }
      };
      auto place = [&](int t, int c) { return (sub / 4 * kTokens + t) * 128 + ((2 * (sub % 4) + c) ^ (t & 7)) * 16; };
      // true when a NaN was among them
      auto lay = [&](char *base, int kv, uint32_t power, const uint4 (&x)[kVecs]) {
        uint32_t nan = 0;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const int t = v * kStride + row_of;
          const uint32_t m = __shfl_sync(0xffffffffu, power, 8 * kv + block_of(v));
          // lanes of odd panels store their second half first: eight lanes then fill eight different chunks
          const int odd = sub / 4 & 1;
          const uint32_t w[4] = {odd ? x[v].z : x[v].x, odd ? x[v].w : x[v].y, odd ? x[v].x : x[v].z, odd ? x[v].y : x[v].w};
          uint32_t h[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            h[2 * k] = mul_f16x2(f16x2_from_e4m3<0>(w[k]), m);
            h[2 * k + 1] = mul_f16x2(f16x2_from_e4m3<1>(w[k]), m);
            note_nan(nan, h[2 * k]);
            note_nan(nan, h[2 * k + 1]);
          }
          *reinterpret_cast<uint4 *>(base + place(t, odd)) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4 *>(base + place(t, 1 - odd)) = make_uint4(h[4], h[5], h[6], h[7]);
        }
        return nan != 0;
      };
      // K and V a tile ahead, pages two, scales one
      uint4 xk[kVecs], xv[kVecs];
      uint32_t ids = look_up(0), next = look_up(1);
      float scale = scale_of(ids);
      int v_ref = kGone;
      fetch(0, 0, ids, xk);
      fetch(1, 0, ids, xv);
      for (uint32_t j = 0; j < units && ok; ++j) {
        const uint32_t at = step + j, stage = at & 1;
        const bool there = ids < p.cache.num_blocks;
        const int e = there ? kv8_scale_exponent(scale) : kGone;
        const int k_ref = max(__reduce_max_sync(0xffffffffu, mine_kv ? kGone : e), kKv8MinExp) - kRoom;
        const int v_top = max(__reduce_max_sync(0xffffffffu, mine_kv ? e : kGone), kKv8MinExp);
        if (j == 0 || v_top > v_ref + kRoom) v_ref = v_top;
        const uint32_t power = f16_power(e - (mine_kv ? v_ref : k_ref));
        scale = scale_of(next);
        const uint32_t later = look_up(j + 2);
        if (!(ok = bar_wait_warp(&sh.empty[0][stage], (at >> 1 & 1) ^ 1, &sh.stalled))) break;
        if (warp == kConvert) {
          if (!there && mine < kBlocks && (int)((unit0 + j) * kTokens) + 16 * mine < tok_stop) p.batch.report(PF_KV8_BAD_BLOCK);
          const uint32_t gone = __ballot_sync(0xffffffffu, !there && mine < kBlocks) & 0xff;
          if (lane == 0) {
            sh.k_unit[at % kRing] = exp2i(k_ref);
            sh.v_ref[at % kRing] = v_ref;
            sh.gone[at % kRing] = gone;
            bar_arrive(&sh.scales_full[at % kRing]);
          }
        }
        lay(smem + L::k + stage * L::kv_bytes, 0, power, xk);
        fence_to_async();
        bar_arrive(&sh.full[0][stage]);
        fetch(0, j + 1, next, xk);
        if (!(ok = bar_wait_warp(&sh.empty[1][stage], (at >> 1 & 1) ^ 1, &sh.stalled))) break;
        char *base = smem + L::v + stage * L::kv_bytes;
        if (__any_sync(0xffffffffu, lay(base, 1, power, xv))) {
          // A NaN in V reaches the rows that see its token and no other: it is taken out here and remembered.
          sh.any_nan = 1;
#pragma unroll 1
          for (int t = row_of; t < kTokens; t += kStride) {
            const int tok = (int)((unit0 + j) * kTokens) + t;
            const uint32_t id = __shfl_sync(0xffffffffu, ids, t / 16);
            const bool seen = id < p.cache.num_blocks && tok < tok_stop;
            const char *src = tile_of + p.cache.kv_stride + (uint64_t)(id < p.cache.num_blocks ? id : 0u) * (uint32_t)p.cache.block_stride + (tok & within) * kDim;
#pragma unroll 1
            for (int b = 0; b < 16; ++b)
              if ((src[b] & 0x7f) == 0x7f) {
                if (seen) atomicMin(&sh.nan_from[16 * sub + b], tok);
                *reinterpret_cast<uint16_t *>(base + place(t, b / 8) + b % 8 * 2) = 0;
              }
          }
        }
        fence_to_async();
        bar_arrive(&sh.full[1][stage]);
        fetch(1, j + 1, next, xv);
        ids = next;
        next = later;
      }
    });
  } else {
    if (kGroups == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    // a thread of another warp looks up what comes next
    const bool looks = warp == kIssue + 1 && lane == 0;
    uint32_t u = 0, u_end = 0;
    bool first = true;
    auto look = [&](Part &part) {
      part.units = 0;
      if (u >= u_end) return;
      const Segment seg(p, work, u);
      uint32_t unit0;
      const uint32_t units = seg.take(u, u_end, unit0);
      const SeqT seq(p, seg.s);
      part.s = seg.s, part.head = seg.head, part.row0 = seq.row0, part.rows = seq.rows, part.len = seq.len;
      part.row_first = seg.rt * kRows, part.live_rows = min(seq.all_rows(p) - seg.rt * kRows, kRows);
      part.unit0 = unit0, part.units = units;
      part.whole = units == seg.units, part.slot = 2 * blockIdx.x + (first ? 0 : 1);
      first = false;
    };
    if (looks) {
      const Split split(work.total(), p.n_ctas);
      if ((int)blockIdx.x < split.n_ctas) u = split.begin(blockIdx.x), u_end = split.begin(blockIdx.x + 1);
      look(sh.part[0]);
    }
    walk([&](const volatile Part &part, uint32_t units) {
      if (looks) look(sh.part[~n_part & 1]);
      if (warp != kIssue || lane != 0) return;
      const int live_rows = part.live_rows;
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
      ok = bar_wait(&sh.q_full, n_part & 1, &sh.stalled);
      for (uint32_t j = 0; j <= units && ok; ++j) {
        const uint32_t at = step + j, before = at - 1;
        if (j < units && !(ok = bar_wait(&sh.full[0][at & 1], at >> 1 & 1, &sh.stalled))) break;
        for (int g = 0; g < kGroups; ++g) {
          if (j > 0) {
            if (!(ok = bar_wait(&sh.p_full[g], before & 1, &sh.stalled))) break;
            if (!(ok = bar_wait(&sh.full[1][before & 1], before >> 1 & 1, &sh.stalled))) break;
            fence_after();
            if (g < n_groups) output(g, before & 1, j > 1);
            if (g == kGroups - 1) commit(&sh.empty[1][before & 1]);
            if (j == units) commit(&sh.o_full[g]);
          }
          if (j < units) {
            fence_after();
            if (g < n_groups) scores(g, at & 1);
            commit(&sh.s_full[g]);
            if (g == kGroups - 1) commit(&sh.empty[0][at & 1]);
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
  if (sh.stalled) {          // a wait ran out: products that are still under way end before the block does
    if (tid == 0) p.batch.report(PF_KV8_STALLED);
    if (warp == kIssue && lane == 0) {
      commit(&sh.drained);
      bar_wait(&sh.drained, 0, &sh.late);
    }
    __syncthreads();
    fence_after();
  }
  if (warp == kIssue) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int kDim, bool kBf16>
void launch(const AttnParams &p, cudaStream_t stream) {
  auto kernel = kv8_attention_wide<kDim, kBf16>;
  const size_t smem = kv8_wide_plan(kDim).smem + Work<kGroupRows * groups_of(kDim), tokens_of(kDim)>::bytes(p.batch.n_seqs, p.row_tiles_most);
  static std::atomic<uint64_t> asked;
  allow_smem(kernel, asked, p.device);
  if (groups_of(kDim) == 2) {
    // what the threads take over from one another (setmaxnreg) has to be there at the start
    static const bool enough = [&] {
      cudaFuncAttributes a;
      return cudaFuncGetAttributes(&a, kernel) == cudaSuccess && (a.numRegs + 7) / 8 * 8 * threads_of(kDim) >= 256 * 144 + 256 * 72 + 128 * 48;
    }();
    if (!enough) throw Error::storage("the kernel was built with too few registers");
  }
  launch_after(kernel, p.n_ctas, threads_of(kDim), smem, stream, p);
}

}  // namespace

static_assert(1024 + Layout<128>::end + sizeof(Shared) + 4 * (1024 + 1) + 128 <= 227 * 1024, "shared memory");
static_assert(Layout<256>::end <= Layout<128>::end && Layout<64>::end <= Layout<128>::end, "shared memory");

WidePlan kv8_wide_plan(int dim) {
  const int end = dim == 64 ? Layout<64>::end : dim == 128 ? Layout<128>::end : Layout<256>::end;
  return WidePlan{kGroupRows * groups_of(dim), tokens_of(dim), 1024 + (size_t)end + sizeof(Shared)};
}

void kv8_wide_launch(const AttnParams &p, bool bf16, cudaStream_t stream) {
  switch (p.cache.dim) {
    case 64: return bf16 ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
    case 128: return bf16 ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
    default: return bf16 ? launch<256, true>(p, stream) : launch<256, false>(p, stream);
  }
}

}  // namespace pf
