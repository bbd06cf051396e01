// Attention over the KV cache held in 8 bits (pf_kv8_attention) for few query rows per KV head (single tokens, drafted
// tokens), and the accumulated weights.
//
//   s[i, j] = scale * 2^eK(j) * q[i] . K8[j]        out[i] = sum_j p[i, j] * 2^eV(j) * V8[j],  p = exp(s - lse)
//
// The cache is read once and each byte is used for as many products as there are rows, so HBM bounds it, if the arithmetic
// keeps out of the way.  It does when no thread touches K and V at all: 128 tokens at a time go from global into shared memory
// by TMA, and the tcgen05 tensor cores take the products on the e4m3 bytes as they are, transposed:
//   S^T [128 tokens, columns] = K Q^T           O^T [head dimensions, columns] += V^T P^T
// One warp feeds tiles, across the segments' ends, a thread of another issues the products, and two teams of four warps take
// tiles in turn, turn scores into P and write outputs.  Each team has references and sums of its own, joined at a segment's
// end: a tile is a chain of some hundred dependent instructions for a team (2700 cycles with one team, whatever the
// dimension, and half of HBM's rate for 64 dimensions or 8 rows), so that several have to run at a time.
// A thread of a team holds a token's scores (a lane of tensor memory), and at the end a dimension's outputs.  What is not e4m3, q and
// p, is written as four e4m3 pieces in columns of their own, x = x0 + x1 / 16 + x2 / 256 + x3 / 4096, each piece the
// rounding of 16 times what the one before it left: a column tile of 16 holds four rows, which is the narrowest that the
// instruction takes.
//   q    scaled by a power of two for each row so that its largest element lies in [2^7, 2^8): its pieces hold a bf16 or an
//        f16 exactly down to 2^-18 of the row's largest, and smaller elements to 2^-30 of it
//   p    2^(6 + s - ref) rounded to f16 (2^-11 of p at most), ref following the row's running maximum in steps of 2^2; the pieces hold
//        that exactly down to 2^-11, that is 2^-17 of the largest, and smaller ones to 2^-28 of it
//   V's scale goes on p: 2^(e - e_ref), e_ref the largest so far, and the sums are in units of it; the row sum leaves it out
//   sums fp32, the tensor cores' and the row sum's; it takes p before it is rounded
// What it measured: 48 requests of 700 to 16001 tokens, 8 heads of 128, groups of 4: 99 us with the join (75 us at the copy rate; 119 us
// with a split that does not count what a segment costs), 8 of 10240 tokens 37 us (26 us).  Long segments stream at 6.2 TB/s;
// a segment's beginning and end cost 8000 cycles of one CTA, the call 14 to 20 us.  The pass for the weights of
// more rows than scores are kept for reads K once more, 26 us for the 8 of 10240 tokens.
// Other forms were measured at the 48 requests: K and V converted
// to f16 in registers for m16n8k16 104 us, the same from rings in shared memory 108 us, m16n8k32 on e4m3 (which sm_100
// does not have: it is converted and issued as f16) 109 us: bound by the issue of conversions with few warps to hide them.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kv8_attention.h"
#include "kv8_tensor.h"

namespace pf {
namespace {

constexpr int kTeam = 128, kWorkers = 2 * kTeam, kThreads = kWorkers + 64;   // two teams, then the feeding and the issuing warp
constexpr int kTokens = 128, kGroups = kTokens / 16;                   // of a step; a group lies within a block
constexpr float kShift = 6.f, kSlack = 2.f;

__host__ __device__ constexpr int few_ctas(int dim, int rows) { return dim == 256 || rows >= 32 ? 1 : 2; }   // of an SM

// Offsets in shared memory behind the first 1024-byte boundary.  kWithV: attention; otherwise the weights, which read K only.
template <int kDim, int kRows, bool kWithV>
struct Few {
  static constexpr int kN = 4 * kRows;                                 // columns
  static constexpr int kKv = kWithV ? 2 : 1, kTile = kTokens * kDim;    // K and V take slots of a ring in turn: K's is free sooner
  static constexpr int kPBytes = kWithV ? kTokens * kN : 0;            // of a team
  static constexpr int kP = 0, kQ = 2 * kPBytes, kFirst = kQ + (kN * kDim < 1024 ? 1024 : kN * kDim);
  static constexpr int kRoom = 227 * 1024 / few_ctas(kDim, kRows) - 2 * 1024 - (kWithV ? 8 : 16) * 1024 - kFirst;   // Shared and Work
  static constexpr int kFit = kRoom / kTile, kSlots = kFit > 12 ? 12 : kFit;
  static constexpr int kEnd = kFirst + kSlots * kTile;
  static constexpr int kO = 2 * kN;                                    // first column of the teams' O behind their S
  static constexpr int kOEach = kN * (kDim == 256 ? 2 : 1), kColumns = kO + (kWithV ? 2 * kOEach : 0);
  static constexpr int kAlloc = kColumns <= 32 ? 32 : kColumns <= 64 ? 64 : kColumns <= 128 ? 128 : kColumns <= 256 ? 256 : 512;
  static_assert(kSlots >= 2 * kKv, "two tiles in flight");
  static_assert(kColumns <= 512 && kAlloc * few_ctas(kDim, kRows) <= 512, "tensor memory");
};

constexpr int kPass = 16;      // steps whose weights are summed over the row tiles before they are added
// Tiles whose scales are kept: a tile is asked for at the earliest when the one six (of the weights: twelve) before it has left
// its slot, for which the scores of that one's second successor had to be issued, which waits for the tile itself.
constexpr int kRing = 16;
template <int kDim, int kRows, int kSlots, bool kWithV>
struct FewShared {
  float scale[kRing][2][kGroups];             // of K, of V; -1: the group's block is not in the cache
  uint64_t full[kSlots], empty[kSlots], q_ready, s_full[2], p_ready[2], pv_done[2], drained;
  uint32_t tmem, fed;        // fed: slots that copies were started into, where a wait ran out
  int stalled, late, any_nan;
  float factor[kRows], base[kRows], row_top[8];
  float ref[2][kRows], down[2][kRows], top[2][4][kRows], sum[2][4][kRows], v_top[2][4], v_ref[2];
  int see[kRows];
  int nan_from[kDim];
  float weight[kWithV ? 1 : kPass][kTeam];
};

// Where 16-byte chunk c of row r lies: rows of 128 bytes (64 at 64 dimensions; two panels at 256) swizzled over eight rows.
template <int kDim>
__device__ __forceinline__ int place(int r, int c, int panel_rows) {
  if (kDim == 64) return r * 64 + 16 * (c ^ (r >> 1 & 3));
  return (c >> 3) * (panel_rows * 128) + r * 128 + 16 * ((c & 7) ^ (r & 7));
}

template <int kDim>
constexpr __host__ __device__ uint32_t swizzle_of() { return kDim == 64 ? kSwizzle64 : kSwizzle128; }

__device__ __forceinline__ float warp_max(float x) {      // leaves NaN out
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// Sums of v[r] over the warp, for all kRows rows: each step halves the rows that a lane holds, or, once it holds one, the lanes.
// Lane 0, 32 / kRows, ... hold a row each, which is returned; the others' is meaningless.
template <int kRows>
__device__ __forceinline__ float warp_sums(float (&v)[kRows], int &row) {
  const int lane = threadIdx.x & 31;
  row = 0;
#pragma unroll
  for (int m = 16, n = kRows; m > 0; m >>= 1) {
    if (n > 1) {
      n /= 2;
#pragma unroll
      for (int r = 0; r < kRows / 2; ++r)
        if (r < n) {
          const float send = lane & m ? v[r] : v[r + n], keep = lane & m ? v[r + n] : v[r];
          v[r] = keep + __shfl_xor_sync(0xffffffffu, send, m);
        }
      row += lane & m ? n : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
    }
  }
  return v[0];
}

// Barriers of a team (ids 1 and 2) and of both (3); whole warps come to them.
__device__ __forceinline__ void team_sync(int team) {
  __syncwarp();
  asm volatile("barrier.cta.sync.aligned %0, 128;" ::"r"(1 + team) : "memory");
}
template <int kCount>
__device__ __forceinline__ bool any_of(int id, bool x) {
  uint32_t y;
  __syncwarp();
  asm volatile("{.reg .pred p, q; setp.ne.u32 p, %1, 0; barrier.cta.red.or.pred.aligned q, %2, %3, p; selp.u32 %0, 1, 0, q;}"
               : "=r"(y)
               : "r"((uint32_t)x), "r"(id), "n"(kCount)
               : "memory");
  return y;
}
__device__ __forceinline__ bool team_any(int team, bool x) { return any_of<kTeam>(1 + team, x); }
__device__ __forceinline__ bool workers_all(bool x) { return !any_of<kWorkers>(3, !x); }

template <int kDim, int kRows, bool kWithV, bool kBf16>
__global__ void __launch_bounds__(kThreads, few_ctas(kDim, kRows)) kv8_attention_few(AttnParams p, const __grid_constant__ CUtensorMap map) {
  using L = Few<kDim, kRows, kWithV>;
  constexpr int kN = L::kN, kSlots = L::kSlots, kChunks = kRows / 4, kRowBytes = kDim == 64 ? 64 : 128, kHalves = kDim == 256 ? 2 : 1;
  using SeqT = Seq<kRows, kTokens, !kWithV>;
  using SharedT = FewShared<kDim, kRows, kSlots, kWithV>;
  extern __shared__ char raw[];
  char *smem = raw + (1024 - (shared_of(raw) & 1023));
  SharedT &sh = *reinterpret_cast<SharedT *>(smem + L::kEnd);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      bar_init(&sh.full[i], 1);
      bar_init(&sh.empty[i], 1);
    }
    bar_init(&sh.q_ready, kWorkers);
    bar_init(&sh.drained, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(&sh.s_full[i], 1);
      bar_init(&sh.p_ready[i], kTeam);
      bar_init(&sh.pv_done[i], 1);
    }
    sh.stalled = sh.late = 0;
    sh.any_nan = 0;
    sh.fed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
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
  const uint32_t tmem = sh.tmem;
  const uint32_t at_p = shared_of(smem + L::kP), at_q = shared_of(smem + L::kQ), at_slot = shared_of(smem + L::kFirst);
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
  // tiles so far, those of each team, and row tiles: what all roles count phases by
  uint32_t n_tiles = 0, n_of[2] = {0, 0}, n_rows = 0;

  while (u < u_end && ok) {
    const Segment seg(p, work, u);
    const int s = seg.s, head = seg.head;
    const SeqT seq(p, s);
    uint32_t unit0, next = u;
    int units = (int)seg.take(next, u_end, unit0);
    if (units == 0) break;                 // the range ends within a segment's cost
    const int all_rows = seq.all_rows(p);
    // Attention: one row tile.  Weights: all of them, one after the other, each over all units.
    const int tiles = kWithV ? 1 : (all_rows + kRows - 1) / kRows;
    if (tiles > 1 && units > kPass) units = kPass, next = seg.begin + unit0 + kPass;
    if (!kWithV && tiles > 1 && warp < 8)
      for (int j = warp >> 2; j < units; j += 2) sh.weight[j][tid % kTeam] = 0.f;         // a thread's own
    for (int tile = 0; tile < tiles && ok; ++tile) {
      const int row_first = (kWithV ? seg.rt : tile) * kRows, live_rows = min(all_rows - row_first, kRows);
      const int most = seq.visible(p, row_first + live_rows - 1);        // tokens that any row of the tile sees
      const int least = seq.visible(p, row_first);                       // tokens that all rows see
      const int tok0 = (int)(unit0 * kTokens), tok_end = min(seq.len, kWithV ? most : min(most, p.w_capacity));
      const int steps = max(0, min(units, (tok_end - tok0 + kTokens - 1) / kTokens));
      if (warp == 8) {
        // ---------------------------------------------------------------- feeding: lane = (values or scale, K or V, group)
        const int32_t *table = p.batch.tables + s * p.batch.table_stride;
        const int group = lane & 7, kv = lane >> 3 & 1, box = p.cache.block_size() / 16;      // groups of a block, and of a copy
        const char *scale_of = p.cache.base + kv * p.cache.kv_stride + p.cache.heads * p.cache.tile_bytes() + 4 * head;
        auto look_up = [&](int j) {
          const int tok = tok0 + j * kTokens + 16 * group;
          return tok < tok_end ? (uint32_t)table[tok >> p.cache.block_log2] : 0xffffffffu;
        };
        // pages two tiles ahead, scales one: both are loads that wait for memory
        auto scale_at = [&](uint32_t id) {
          return lane >= 16 && kv < L::kKv && id < p.cache.num_blocks ? __ldg(reinterpret_cast<const float *>(scale_of + (uint64_t)id * (uint32_t)p.cache.block_stride)) : -1.f;
        };
        uint32_t id = look_up(0), next = look_up(1);
        float scale = scale_at(id);
        for (int j = 0; j < steps; ++j) {
          const uint32_t at = n_tiles + j;
          const int tok = tok0 + j * kTokens + 16 * group;
          const bool there = id < p.cache.num_blocks;
          if (!there && tok < tok_end && lane < 8) p.batch.report(PF_KV8_BAD_BLOCK);
          // a block that is not there lies behind the last one: the copy fills it with zeros
          const int row = tok & (p.cache.block_size() - 1), block = there ? (int)id : (int)p.cache.num_blocks;
          id = next;
          next = look_up(j + 2);
          const float now = scale;
          scale = scale_at(id);
#pragma unroll
          for (int of = 0; of < L::kKv; ++of) {
            const uint32_t i = L::kKv * at + of, slot = i % kSlots;
            if (!(ok = bar_wait_warp(&sh.empty[slot], (i / kSlots & 1) ^ 1, &sh.stalled))) {
              sh.fed = i;
              break;
            }
            if (of == 0 && lane >= 16) sh.scale[at % kRing][kv][group] = now;
            __syncwarp();
            if (lane == 0)
              asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_of(&sh.full[slot])), "r"(L::kTile) : "memory");
            __syncwarp();
            if (lane < 16 && kv == of && (group & (box - 1)) == 0) {
#pragma unroll
              for (int half = 0; half < kHalves; ++half)
                asm volatile(
                    "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
                        at_slot + slot * L::kTile + half * (kTokens * 128) + group * 16 * kRowBytes),
                    "l"(&map), "r"(half * 128), "r"(row), "r"(head), "r"(block), "r"(kv), "r"(shared_of(&sh.full[slot]))
                    : "memory");
            }
          }
          if (!ok) break;
        }
      } else if (warp == 9) {
        // ---------------------------------------------------------------- issuing
        if (lane == 0 && steps > 0) {
          constexpr uint32_t kScores = shape_of(kN, false, false), kOutputs = shape_of(kN, true, true);
          ok = bar_wait(&sh.q_ready, n_rows & 1, &sh.stalled);
          for (int j = 0; j <= steps && ok; ++j) {
            const uint32_t at = n_tiles + j;
            if (j < steps) {
              const uint32_t i = L::kKv * at, slot = i % kSlots, at_k = at_slot + slot * L::kTile;
              if (!(ok = bar_wait(&sh.full[slot], i / kSlots & 1, &sh.stalled))) break;
              fence_after();
#pragma unroll
              for (int k = 0; k < kDim / 32; ++k) {
                const uint32_t in = kDim == 64 ? k * 32 : k % 4 * 32;
                mma_e4m3_ss(tmem + (j & 1) * kN, operand(at_k + k / 4 * (kTokens * 128) + in, 16, 8 * kRowBytes, swizzle_of<kDim>()),
                            operand(at_q + k / 4 * (kN * 128) + in, 16, 8 * kRowBytes, swizzle_of<kDim>()), kScores, k != 0);
              }
              commit(&sh.s_full[j & 1]);
              if (kWithV) commit(&sh.empty[slot]);
            }
            if (j > 0) {          // the tile before: its scores have been read, and its P written
              const int team = (j - 1) & 1;
              const uint32_t i = L::kKv * (at - 1) + L::kKv - 1, slot = i % kSlots, at_v = at_slot + slot * L::kTile;
              if (!(ok = bar_wait(&sh.p_ready[team], (n_of[team] + ((j - 1) >> 1)) & 1, &sh.stalled))) break;
              if (!kWithV) {      // K has been read
                bar_arrive(&sh.empty[slot]);
                continue;
              }
              // The workers have waited for V too, but V of two tiles need not land in order, and a team that runs ahead could take
              // the barrier's phase for its own: in this thread every phase is waited for.
              if (!(ok = bar_wait(&sh.full[slot], i / kSlots & 1, &sh.stalled))) break;
              fence_after();
#pragma unroll
              for (int half = 0; half < kHalves; ++half)
#pragma unroll
                for (int k = 0; k < kTokens / 32; ++k)
                  // at 64 dimensions the second half of the rows repeats the first: nobody reads it
                  mma_e4m3_ss(tmem + L::kO + team * L::kOEach + half * kN, operand(at_v + half * (kTokens * 128) + k * 32 * kRowBytes, 0, 8 * kRowBytes, swizzle_of<kDim>()),
                              operand(at_p + team * L::kPBytes + k * 512, 128, kTokens * 16, kNoSwizzle), kOutputs, j > 2 || k != 0);
              commit(&sh.pv_done[team]);
              commit(&sh.empty[slot]);
            }
          }
        }
      } else {
        // ---------------------------------------------------------------- workers
        const int team = warp >> 2, own = tid % kTeam;       // the token of a tile, and the dimension, that are this thread's
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) * 32 << 16), at_o = lanes + L::kO + team * L::kOEach;
        // the rows' pieces, factors and lengths
        constexpr int kLanes = kDim / 16, kFours = kDim / 4;       // 16-byte chunks of a row of bytes; threads of a row of q
        for (int e = tid; e < kRows * kFours; e += kWorkers) {     // whole warps: a row is 16 lanes, or a warp or two
          const int r = e / kFours, c = e % kFours, row = row_first + r;
          const bool live = r < live_rows;
          const int i = live ? row / p.group : 0, qh = head * p.group + (live ? row - i * p.group : 0);
          const uint16_t *src = p.q + (int64_t)(seq.row0 + i) * p.q_row + qh * p.q_head + 4 * c;
          uint2 y = make_uint2(0, 0);
          if (live) {
            if (p.vec_q) y = *reinterpret_cast<const uint2 *>(src);
            else y = make_uint2(src[0] | src[1] << 16, src[2] | src[3] << 16);
          }
          float x[4];
          const float2 lo2 = kBf16 ? make_float2(__uint_as_float(y.x << 16), __uint_as_float(y.x & 0xffff0000u)) : f32x2_from_f16x2(y.x);
          const float2 hi2 = kBf16 ? make_float2(__uint_as_float(y.y << 16), __uint_as_float(y.y & 0xffff0000u)) : f32x2_from_f16x2(y.y);
          x[0] = lo2.x, x[1] = lo2.y, x[2] = hi2.x, x[3] = hi2.y;
          float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
          if (kDim == 64) {
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          } else {
            top = warp_max(top);
          }
          if (kDim == 256) {                 // the row's other warp is this warp's neighbour
            if (lane == 0) sh.row_top[warp] = top;
            if (!workers_all(true)) break;
            top = fmaxf(top, sh.row_top[warp ^ 1]);
            if (!workers_all(true)) break;   // and has read it
          }
          int ex = (int)(__float_as_uint(top) >> 23) - 127 - 7;
          if (top == 0.f || top > 3.4e38f) ex = 0;
          ex = max(ex, -126);
          const float down = exp2i(-ex);
          // an infinity would become 448
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = fabsf(x[k]) > 3.4e38f ? __int_as_float(0x7fffffff) : x[k] * down;
#pragma unroll
          for (int piece = 0; piece < 4; ++piece) {
            const uint32_t lo = e4m3x2(x[0], x[1]), hi = e4m3x2(x[2], x[3]);
            const int n = 16 * (r / 4) + 4 * piece + r % 4;
            *reinterpret_cast<uint32_t *>(smem + L::kQ + place<kDim>(n, c / 4, kN) + 4 * (c % 4)) = lo | hi << 16;
            const float2 a = f32x2_from_f16x2(f16x2_from_e4m3<0>(lo)), b = f32x2_from_f16x2(f16x2_from_e4m3<0>(hi));
            x[0] = (x[0] - a.x) * 16.f, x[1] = (x[1] - a.y) * 16.f, x[2] = (x[2] - b.x) * 16.f, x[3] = (x[3] - b.y) * 16.f;
          }
          if (c == 0) {
            sh.factor[r] = p.scale * kLog2e * exp2i(ex);
            sh.see[r] = live ? seq.visible(p, row) : 0;
            sh.ref[0][r] = sh.ref[1][r] = kNone;
            // Rows that are not there, or see nothing (no token, or missing pages only: lse is -inf), weigh nothing.
            if (!kWithV) {
              const float lse = sh.see[r] > 0 ? p.lse[(int64_t)(seq.row0 + i) * p.q_heads + qh] : -INFINITY;
              sh.base[r] = lse == -INFINITY ? INFINITY : lse * kLog2e;
            }
          }
        }
        fence_to_async();
        if (steps > 0) bar_arrive(&sh.q_ready);
        ok = workers_all(true);
        float sum[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) sum[r] = 0.f;
        float v_ref = 0.f;                     // 2^e_ref

        uint32_t turn = n_of[team];                  // tiles that the team had before this one
        for (int j = team; j < steps; j += 2, ++turn) {
          // V's slot (of the weights: K's) is not filled again before this tile is done with, and its barrier says that the
          // scales are there too.  The scores come first: once they are issued, so is the product of the tile two before, and
          // what was in this slot before has been waited for, so that the barrier is in this tile's phase or behind it.
          const uint32_t at = n_tiles + j, i_slot = L::kKv * at + L::kKv - 1, slot = i_slot % kSlots;
          const int tok1 = tok0 + j * kTokens, tok = tok1 + own;
          ok = bar_wait_warp(&sh.s_full[team], turn & 1, &sh.stalled);
          ok = ok && bar_wait_warp(&sh.full[slot], i_slot / kSlots & 1, &sh.stalled);
          if (kWithV && j > 1) ok = ok && bar_wait_warp(&sh.pv_done[team], (turn - 1) & 1, &sh.stalled);    // P's place is free, O at rest
          fence_after();
          const bool partly = tok1 + kTokens > least;      // some row does not see all of it
          const int of_group = own >> 4;
          const float k_scale = sh.scale[at % kRing][0][of_group], v_scale = kWithV ? sh.scale[at % kRing][1][of_group] : 0.f;
          const bool gone = k_scale < 0.f;
          if (kWithV && partly) {
            // Rows behind the last token hold what the block held before.  A NaN reaches the rows that see its token and no
            // other: 0 * NaN would.  It is taken out, and the first such token remembered for each dimension.
#pragma unroll 1
            for (int e = own; e < kTokens * kLanes; e += kTeam) {
              const int row = e / kLanes, c = e % kLanes;
              uint4 *chunk = reinterpret_cast<uint4 *>(smem + L::kFirst + slot * L::kTile + place<kDim>(row, c, kTokens));
              if (tok1 + row >= seq.len) {
                *chunk = make_uint4(0, 0, 0, 0);
                continue;
              }
              uint32_t *w = reinterpret_cast<uint32_t *>(chunk), any = 0;
              for (int k = 0; k < 4; ++k) any |= (w[k] & 0x7f7f7f7fu) + 0x01010101u;
              if (!(any & 0x80808080u)) continue;
              sh.any_nan = 1;
              for (int k = 0; k < 16; ++k)
                if ((w[k / 4] >> (8 * (k % 4)) & 0x7f) == 0x7f) {
                  atomicMin(&sh.nan_from[16 * c + k], tok1 + row);
                  w[k / 4] &= ~(0xffu << (8 * (k % 4)));
                }
            }
          }
          __syncwarp();
          const uint32_t at_s = lanes + team * kN;
          auto scores = [&](int c, float (&x)[4]) {       // of rows 4 c .. 4 c + 3, for this thread's token
            uint32_t y[16];
            load16(y, at_s + 16 * c);
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
            fence_before();
            if (!ok) break;
            bar_arrive(&sh.p_ready[team]);
            if (tiles > 1) sh.weight[j][own] += w;
            else if (tok < tok_end && !gone) p.weights[s * p.w_seq + head * p.w_head + tok] += w;
          } else {
            float first[4];
            bool over = v_scale > v_ref || !ok;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              float x[4];
              scores(c, x);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                over |= x[r] > sh.ref[team][4 * c + r] + kSlack;
                if (c == 0) first[r] = x[r];
              }
            }
            if (team_any(team, over)) {
              if (!(ok = !team_any(team, !ok))) break;       // a wait of some warp ran out
              // new references: the largest scores of the tile, the largest of V's scales
              float v_top = warp_max(v_scale);
              if (lane == 0) sh.v_top[team][warp & 3] = v_top;
#pragma unroll 1
              for (int c = 0; c < kChunks; ++c) {
                float x[4];
                scores(c, x);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  x[r] = warp_max(x[r]);
                  if (lane == 0) sh.top[team][warp & 3][4 * c + r] = x[r];
                }
              }
              team_sync(team);
              const float *tops = sh.v_top[team];
              v_top = fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), fmaxf(v_ref, 0x1p-110f));
              const float v_down = v_ref / v_top;          // powers of two; 0 at the start
              v_ref = v_top;
              if (own < kRows) {
                const float was = sh.ref[team][own];
                const float top = fmaxf(fmaxf(sh.top[team][0][own], sh.top[team][1][own]), fmaxf(sh.top[team][2][own], sh.top[team][3][own]));
                const float now = top > was + kSlack ? top : was;
                sh.ref[team][own] = now;
                sh.down[team][own] = exp2_fast(was - now);
              }
              team_sync(team);
#pragma unroll
              for (int r = 0; r < kRows; ++r) sum[r] *= sh.down[team][r];
              if (j > 1) {
#pragma unroll 1
                for (int c = 0; c < kHalves * kChunks; ++c) {
                  uint32_t y[16];
                  load16(y, at_o + 16 * c);
#pragma unroll
                  for (int k = 0; k < 16; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * (sh.down[team][4 * (c % kChunks) + k % 4] * v_down));
                  store16(at_o + 16 * c, y);
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
              if (p.scores && tok < min(tok_end, p.score_tokens))
                *reinterpret_cast<float4 *>(p.scores + (((int64_t)s * p.cache.heads + head) * p.score_tokens + tok) * kRows + 4 * c) =
                    make_float4(x[0], x[1], x[2], x[3]);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                x[r] = exp2_fast(x[r] - (sh.ref[team][4 * c + r] - kShift));
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
              *reinterpret_cast<uint4 *>(smem + L::kP + team * L::kPBytes + c * (kTokens * 16) + own * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_to_async();
            fence_before();
            bar_arrive(&sh.p_ready[team]);
          }
        }
        if constexpr (kWithV) {
          if (steps > team) ok = ok && bar_wait_warp(&sh.pv_done[team], (turn - 1) & 1, &sh.stalled);
          fence_after();
          // row sums over the threads
          int row_of;
          const float row_sum = warp_sums<kRows>(sum, row_of);
          if (lane % (32 / kRows) == 0) sh.sum[team][warp & 3][row_of] = row_sum;
          if (own == 0) sh.v_ref[team] = v_ref;
          fence_before();
          if ((ok = workers_all(ok))) {
            fence_after();
            // the teams' parts together: team t writes row chunks t, t + 2, ...
            const bool whole = units == (int)seg.units, any_nan = sh.any_nan;
            const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
#pragma unroll 1
            for (int i = team; i < kHalves * ((live_rows + 3) / 4); i += 2) {
              const int half = kHalves == 2 ? i & 1 : 0, c = kHalves == 2 ? i >> 1 : i, d = half * 128 + own;
              uint32_t y[2][16];
              load16(y[0], lanes + L::kO + half * kN + 16 * c);
              load16(y[1], lanes + L::kO + L::kOEach + half * kN + 16 * c);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int r = 4 * c + k;
                if (r >= live_rows || d >= kDim) continue;
                const float base = fmaxf(sh.ref[0][r], sh.ref[1][r]);
                float a = 0.f, l = 0.f;
#pragma unroll
                for (int of = 0; of < 2; ++of) {
                  if (steps <= of) continue;               // that team had no tile: its O is not written
                  const float down = exp2_fast(sh.ref[of][r] - base);
                  const float lo = fmaf(__uint_as_float(y[of][12 + k]), 1.f / 16, __uint_as_float(y[of][8 + k]));
                  a += fmaf(fmaf(lo, 1.f / 16, __uint_as_float(y[of][4 + k])), 1.f / 16, __uint_as_float(y[of][k])) * sh.v_ref[of] * down;
                  l += (sh.sum[of][0][r] + sh.sum[of][1][r] + sh.sum[of][2][r] + sh.sum[of][3][r]) * down;
                }
                if (l == 0.f) a = 0.f;
                if (any_nan && sh.nan_from[d] < sh.see[r]) a = __int_as_float(0x7fffffff);
                const int row = row_first + r, i = row / p.group, qh = head * p.group + row % p.group;
                if (whole) {
                  a = l == 0.f ? a : a / l;
                  uint16_t *dst = p.out + (int64_t)(seq.row0 + i) * p.out_row + qh * p.out_head + d;
                  *dst = kBf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(a)) : __half_as_ushort(__float2half_rn(a));
                  if (d == 0 && p.lse) p.lse[(int64_t)(seq.row0 + i) * p.q_heads + qh] = lse_of(base - kShift, l);
                } else {
                  p.part_o[((int64_t)slot * kRows + r) * kDim + d] = a;
                  if (d == 0) p.part_ml[slot * kRows + r] = make_float2(base - kShift, l);
                }
              }
            }
            fence_before();
            if (any_nan) {
              workers_all(true);
              for (int i = tid; i < kDim; i += kWorkers) sh.nan_from[i] = INT_MAX;
              if (tid == 0) sh.any_nan = 0;
            }
          }
        }
        // what the rows of this tile left in shared memory has been read
        if ((ok = workers_all(ok)) && !kWithV && tiles > 1 && tile + 1 == tiles)
          for (int j = team; j < units; j += 2) {
            const int tok = (int)(unit0 + j) * kTokens + own;
            if (tok < min(seq.len, p.w_capacity)) p.weights[s * p.w_seq + head * p.w_head + tok] += sh.weight[j][own];
          }
      }
      n_tiles += steps;
      n_of[0] += (steps + 1) >> 1;
      n_of[1] += steps >> 1;
      n_rows += steps > 0;
    }
    u = next;
    first_segment = false;
  }
  // The tensor cores' last arrivals, at the slots that are not filled again, come before the block leaves.
  if (warp == 8 && ok)
    for (uint32_t i = L::kKv * n_tiles > (uint32_t)kSlots ? L::kKv * n_tiles - kSlots : 0; i < L::kKv * n_tiles && ok; ++i)
      if (!(ok = bar_wait_warp(&sh.empty[i % kSlots], i / kSlots & 1, &sh.stalled))) sh.fed = L::kKv * n_tiles;
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (sh.stalled) {          // a wait ran out: what is still under way, copies and products, ends before the block does
    if (tid == 0) p.batch.report(PF_KV8_STALLED);
    if (warp == 8 && lane == 0) {
      const uint32_t fed = sh.fed;
      for (uint32_t i = fed > (uint32_t)kSlots ? fed - kSlots : 0; i < fed; ++i)
        if (!bar_wait(&sh.full[i % kSlots], i / kSlots & 1, &sh.late)) break;
    }
    if (warp == 9 && lane == 0) {
      commit(&sh.drained);
      bar_wait(&sh.drained, 0, &sh.late);
    }
    __syncthreads();
    fence_after();
  }
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(L::kAlloc));
}

// The cache as [K or V][block][head][row][byte], copied by the rows of a block of (half) a head: the copies' rate is one in 45 to
// 60 cycles of an SM.  48 requests of 25600 tokens, 8 heads of 64, blocks of 64: 237 us, by copies of 16 rows 261 us.
CUtensorMap map_of(const Kv8View &c) {
  using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
    return reinterpret_cast<Encode>(f);
  }();
  if (!encode) throw Error::cuda_init("cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[5] = {(cuuint64_t)c.dim, (cuuint64_t)c.block_size(), (cuuint64_t)c.heads, c.num_blocks, 2};
  const cuuint64_t strides[4] = {(cuuint64_t)c.dim, c.tile_bytes(), c.block_stride, c.kv_stride};
  const cuuint32_t box[5] = {(cuuint32_t)std::min(c.dim, 128), (cuuint32_t)c.block_size(), 1, 1, 1}, ones[5] = {1, 1, 1, 1, 1};
  CUtensorMap map;
  if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, c.base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             c.dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    throw Error::invalid("8-bit cache: no tensor map describes it");
  return map;
}

template <int kDim, int kRows, bool kWithV, bool kBf16>
void launch(const AttnParams &p, int n_ctas, cudaStream_t stream) {
  using L = Few<kDim, kRows, kWithV>;
  auto kernel = kv8_attention_few<kDim, kRows, kWithV, kBf16>;
  const size_t smem = 1024 + (size_t)L::kEnd + sizeof(FewShared<kDim, kRows, L::kSlots, kWithV>) +
                      Work<kRows, kTokens, !kWithV>::bytes(p.batch.n_seqs, p.row_tiles_most);
  static std::atomic<uint64_t> asked;
  allow_smem(kernel, asked, p.device);
  launch_after(kernel, n_ctas, kThreads, smem, stream, p, map_of(p.cache));
}

template <int kDim, bool kBf16>
void launch(const AttnParams &p, int rows, cudaStream_t stream) {
  switch (rows) {
    case 4: return launch<kDim, 4, true, kBf16>(p, p.n_ctas, stream);
    case 8: return launch<kDim, 8, true, kBf16>(p, p.n_ctas, stream);
    case 16: return launch<kDim, 16, true, kBf16>(p, p.n_ctas, stream);
    default:
      if constexpr (kDim != 256) launch<kDim, 32, true, kBf16>(p, p.n_ctas, stream);
  }
}

}  // namespace

// Up to 32 rows go in tiles of up to 32 (at 256 dimensions 16).  16 requests of 4000 tokens, 4 KV heads of 128: 32 rows take
// 61 us here and 68 us in the form for many rows, 64 rows (two tiles, K and V read for each) 90 us and 68 us.
int kv8_few_rows(int dim, int64_t rows) {
  if (rows <= 16) return rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  return rows <= 32 ? (dim == 256 ? 16 : 32) : 0;
}
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
