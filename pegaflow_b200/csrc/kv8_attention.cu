// Attention over the KV cache held in 8 bits (pf_kv8_attention): the joining of partial results, and the host's side.  The
// attention itself is in kv8_attention_few.cu (up to 32 query rows of a KV head) and kv8_attention_wide.cu (more).
#include <algorithm>

#include "kv8_attention.h"

namespace pf {
namespace {

// Joins the parts of segments that several CTAs shared, in the order of the tokens.  CTA (b, y) looks at the boundary
// between the ranges of CTAs b and b + 1: if it is the first one within a segment, it joins rows of it, a team of threads
// for each.  kDim / 4 threads hold a row of a part as float4; a team of more reads several parts at once.  Bound by latency:
// some 5 us behind the last CTA of the attention.
constexpr int kJoinThreads = 256;
template <int kDim, int kRows, int kUnits, bool kBf16>
__device__ __forceinline__ void join(const AttnParams &p, const Work<kRows, kUnits> &work, int team) {
  constexpr int kSpan = kDim / 4, kDeep = 4;
  using SeqT = Seq<kRows, kUnits>;
  __shared__ float4 sh_a[kJoinThreads];
  __shared__ float sh_l[kJoinThreads], sh_top[kJoinThreads / 32];
  const Split split(work.total(), p.n_ctas);
  const int c0 = blockIdx.x;
  if (c0 + 1 >= split.n_ctas) return;
  const uint32_t u = split.begin(c0 + 1);
  const Segment seg(p, work, u);
  const SeqT seq(p, seg.s);
  if (u <= seg.begin || split.owner(seg.begin) != c0) return;
  const int parts = split.owner(seg.begin + seg.units - 1) - c0 + 1, slot0 = 2 * c0 + (split.begin(c0) < seg.from ? 1 : 0);
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

// Rows of no sequence, [0, first) and [last, n_rows), are cleared; where none was computed all rows, for the weights' sake too.  Where
// a row start falls, any sequence may have the first and the last ones.
template <int kDim>
__device__ __forceinline__ void clear_rows(const AttnParams &p, bool none, bool falls) {
  __shared__ int sh_first, sh_last;
  int first = 0, last = 0, ignored;
  if (falls && !none) {
    if (threadIdx.x == 0) sh_first = p.batch.n_rows, sh_last = 0;
    __syncthreads();
#pragma unroll 1
    for (int s = threadIdx.x; s < p.batch.n_seqs; s += kJoinThreads) {
      p.batch.rows(s, first, last);
      if (first < last) atomicMin(&sh_first, first), atomicMax(&sh_last, last);
    }
    __syncthreads();
    first = min(sh_first, sh_last), last = sh_last;
  } else if (!none) {
    p.batch.rows(0, first, ignored);
    p.batch.rows(p.batch.n_seqs - 1, ignored, last);
  }
#pragma unroll 1
  for (uint32_t i = blockIdx.y * gridDim.x + blockIdx.x; i < (uint32_t)(first + p.batch.n_rows - last); i += gridDim.x * gridDim.y) {
    const int64_t row = i < (uint32_t)first ? i : i - first + last;
    if (p.clear_tail == PF_KV8_CLEAR_ALL) {
#pragma unroll 1
      for (int c = threadIdx.x; c < p.q_heads * kDim; c += kJoinThreads) p.out[row * p.out_row + c / kDim * p.out_head + c % kDim] = 0;
    }
    if (p.lse) {
#pragma unroll 1
      for (int c = threadIdx.x; c < p.q_heads; c += kJoinThreads) p.lse[row * p.q_heads + c] = -INFINITY;
    }
  }
}

// 40 registers: at 48 verify-16-ragged takes 58.0 us, at 40 57.4, at 64 59.3 (decode-1x131000 29.8, 29.7, 30.3).
template <int kDim, int kRows, int kUnits, bool kBf16>
__global__ void __launch_bounds__(kJoinThreads, 6) kv8_attention_join(AttnParams p, int team) {
  extern __shared__ __align__(128) char smem[];
  const Work<kRows, kUnits> work(p, reinterpret_cast<uint32_t *>(smem));
  after_previous();
  join<kDim, kRows, kUnits, kBf16>(p, work, team);
  const bool none = work.total() == 0;
  if (p.clear_tail || (none && p.weights)) clear_rows<kDim>(p, none, work.falls);      // behind the join, which others may wait for
}

// Each token's probability from the scores that the attention kept, added to the weights: a thread a token, rows in order.
// Bound by memory, 4 bytes for each score and 8 for each weight.
constexpr int kAddThreads = 256;
template <int kRows>
__global__ void __launch_bounds__(kAddThreads) kv8_weights_add(AttnParams p) {
  after_previous();
  const int s = blockIdx.x / p.cache.heads, head = blockIdx.x % p.cache.heads;
  if (head == 0 && blockIdx.y == 0 && threadIdx.x == 0 && p.batch.lens[s] > p.w_capacity) p.batch.report(PF_KV8_BAD_LENGTH);
  const Seq<kRows, 128> seq(p, s);
  const int live_rows = min(seq.all_rows(p), kRows);
  if (live_rows <= 0) return;
  const int end = min(min(seq.visible(p, live_rows - 1), p.score_tokens), p.w_capacity);
  float base[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    base[r] = INFINITY;        // a row that sees nothing weighs nothing
    if (r < live_rows) {
      const float lse = p.lse[(int64_t)(seq.row0 + r / p.group) * p.q_heads + head * p.group + r % p.group];
      if (lse != -INFINITY) base[r] = lse * kLog2e;
    }
  }
  const float *scores = p.scores + (int64_t)blockIdx.x * p.score_tokens * kRows;
  float *weights = p.weights + s * p.w_seq + head * p.w_head;
  for (int tok = blockIdx.y * kAddThreads + threadIdx.x; tok < end; tok += gridDim.y * kAddThreads) {
    float w = 0.f;
#pragma unroll
    for (int c = 0; c < kRows / 4; ++c) {
      const float4 x = *reinterpret_cast<const float4 *>(scores + (int64_t)tok * kRows + 4 * c);
      const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) w += 4 * c + r < live_rows ? exp2_fast(y[r] - base[4 * c + r]) : 0.f;
    }
    weights[tok] += w;
  }
}

// ---------------------------------------------------------------------------------------------- host
struct Plan {
  bool wide;            // rows by the hundred
  int n_ctas, rows;     // rows of a tile, and of a part
  size_t part_o, part_ml, lse, scores, bytes;   // offsets in the workspace
  int score_tokens;     // 0: scores are not kept
  int row_tiles;        // of a sequence, at most
  uint32_t units;       // of all its rows, at most
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// The weights need every score once more, when the row's lse is known.  Of few rows the scores are kept, 8 bytes written and
// read for each, where K is dim bytes and four products a row: for 8 sequences of 10240 tokens, 8 heads of 128, groups of 4, the
// pass over the scores takes 12 us, the one over K 26 us (a call 55 and 67 us).  More rows, or more than this much workspace, read K again.
constexpr uint64_t kMostScores = 256 << 20;

Plan make_plan(int device_id, const Kv8View &c, const Kv8Batch &b, const pf_kv8_attention_args &a) {
  const size_t group = a.q_heads / c.heads;
  Plan plan{};
  const size_t rows = std::min(a.max_query, a.n_rows) * group;
  plan.rows = kv8_few_rows(c.dim, (int64_t)rows);
  plan.wide = plan.rows == 0;
  if (plan.wide) plan.rows = kv8_wide_plan(c.dim).rows;
  // As the kernels count them, in 32 bits: row tiles of all sequences x (units of tokens and a segment's cost) x heads.
  const uint64_t unit = plan.wide ? kv8_wide_plan(c.dim).tokens : 128;
  const uint64_t units = (((uint64_t)b.max_blocks << c.block_log2) / unit + 1 + Work<4, 128>::kCost) *
                         (((uint64_t)a.n_rows * group) / plan.rows + b.n_seqs) * c.heads;
  const uint64_t row_tiles = std::max<uint64_t>(1, (rows + plan.rows - 1) / plan.rows);
  if (units > 0xffffffffull || row_tiles * b.n_seqs > 1u << 29) throw Error::invalid("too many query rows for tables of this width: split the call");
  plan.units = (uint32_t)units;
  plan.row_tiles = (int)row_tiles;
  plan.n_ctas = kv8_sm_count(device_id) * (plan.wide ? 1 : kv8_few_ctas(c.dim, plan.rows));
  const size_t slots = 2 * (size_t)plan.n_ctas * plan.rows;
  plan.part_o = 0;
  plan.part_ml = up256(slots * c.dim * 4);
  plan.lse = plan.part_ml + up256(slots * 8);
  plan.scores = plan.lse + (a.weights && !a.lse ? up256(a.n_rows * a.q_heads * 4) : 0);
  plan.bytes = plan.scores;
  if (a.weights && !plan.wide && rows <= (size_t)plan.rows && plan.rows <= c.dim / 16) {      // one row tile
    const uint64_t tokens = std::min<uint64_t>((uint64_t)b.max_blocks << c.block_log2, std::min<size_t>(a.weights_capacity, 0x7fffffff));
    const uint64_t bytes = (uint64_t)b.n_seqs * c.heads * tokens * plan.rows * 4;
    if (bytes <= kMostScores) plan.score_tokens = (int)tokens, plan.bytes += up256(bytes);
  }
  return plan;
}

// Whether two elements of an array of outer x inner dense rows of n elements can be one; of a single row any stride will do.
bool overlaps_itself(size_t outer, size_t outer_stride, size_t inner, size_t inner_stride, size_t n) {
  if (outer * inner <= 1) return false;
  if (outer > 1 && (inner == 1 || inner_stride > outer_stride)) std::swap(outer, inner), std::swap(outer_stride, inner_stride);
  // now outer_stride is the larger one, or outer is 1
  const size_t whole = outer == 1 || inner > 1 ? (inner - 1) * inner_stride + n : n;
  return (inner > 1 && inner_stride < n) || (outer > 1 && outer_stride < whole);
}

// Whether out can share an element with q where the two are not one and the same: their ranges are apart, or the rests of their
// offsets modulo one of the strides are (heads or rows of one buffer that belong to q and to out in turn).
bool shares(const pf_kv8_attention_args &a, int dim) {
  const uint64_t q = (uint64_t)a.q, out = (uint64_t)a.out;
  auto bytes = [&](size_t row, size_t head) { return 2 * ((a.n_rows - 1) * row + (a.q_heads - 1) * head + dim); };
  if (q + bytes(a.q_row_stride, a.q_head_stride) <= out || out + bytes(a.out_row_stride, a.out_head_stride) <= q) return false;
  if ((out - q) % 2) return true;
  for (const size_t m : {a.q_row_stride, a.q_head_stride, a.out_row_stride, a.out_head_stride}) {
    if (!m) continue;
    auto rest = [&](size_t row, size_t head) {       // elements from the first one on that an offset's rest can be
      return (row % m ? (a.n_rows - 1) * row : 0) + (head % m ? (a.q_heads - 1) * head : 0) + dim;
    };
    const size_t apart = out >= q ? (out - q) / 2 % m : (m - (q - out) / 2 % m) % m;
    if (apart >= rest(a.q_row_stride, a.q_head_stride) && apart + rest(a.out_row_stride, a.out_head_stride) <= m) return false;
  }
  return true;
}

void check_args(const pf_kv8_attention_args *a, const Kv8View &c, const Kv8Batch &b) {
  if (!a) throw Error::invalid("null attention arguments");
  if (a->dtype != PF_KV8_BF16 && a->dtype != PF_KV8_F16) throw Error::invalid(strf("unknown dtype %d", a->dtype));
  if (a->q_heads == 0 || a->q_heads % c.heads || a->q_heads > 65536)
    throw Error::invalid(strf("%u query heads are not a multiple of %d KV heads", a->q_heads, c.heads));
  if (a->n_rows && b.n_seqs && a->max_query == 0) throw Error::invalid("max_query must not be 0");
  if (a->clear_tail < 0 || a->clear_tail > PF_KV8_CLEAR_LSE) throw Error::invalid(strf("unknown clear_tail %d", a->clear_tail));
  const uint64_t rows_of_group = (uint64_t)std::min<size_t>(a->max_query, a->n_rows) * (a->q_heads / c.heads);
  if (rows_of_group > 0x3fffffffu) throw Error::invalid("too many query rows");
  if (!b.starts && b.n_seqs && a->max_query < (size_t)b.rows_each)
    throw Error::invalid(strf("max_query=%zu is below the %d rows of each sequence", a->max_query, b.rows_each));
}

template <int kDim, int kRows, int kUnits, bool kBf16>
void launch_join(const AttnParams &p, cudaStream_t stream) {
  // About n_ctas / segments parts meet in a segment: few are read one after the other by the fewest threads that hold a row,
  // many (a long sequence alone) by a whole CTA.  One rule for all: a quarter of them at a time.
  constexpr int kSpan = kDim / 4;
  const int64_t segments = std::max<int64_t>(1, (int64_t)p.batch.n_seqs * p.cache.heads * p.row_tiles_most);
  int team = kSpan;
  while (team < kJoinThreads && team / kSpan * 4 * segments < p.n_ctas) team *= 2;
  const int passes = std::max(1, kRows * team / kJoinThreads);
  const dim3 grid((unsigned)p.n_ctas, (unsigned)std::min(passes, 16));
  launch_after(kv8_attention_join<kDim, kRows, kUnits, kBf16>, grid, kJoinThreads, Work<kRows, kUnits>::bytes(p.batch.n_seqs, p.row_tiles_most),
               stream, p, team);
}

template <int kDim, bool kBf16>
void launch(const AttnParams &p, const Plan &plan, cudaStream_t stream) {
  switch (plan.wide ? 0 : plan.rows) {
    case 4: return launch_join<kDim, 4, 128, kBf16>(p, stream);
    case 8: return launch_join<kDim, 8, 128, kBf16>(p, stream);
    case 16: return launch_join<kDim, 16, 128, kBf16>(p, stream);
    case 32: return launch_join<kDim, 32, 128, kBf16>(p, stream);
    default: return launch_join<kDim, kDim == 256 ? 128 : 256, kDim == 256 ? 64 : 128, kBf16>(p, stream);
  }
}

template <bool kBf16>
void launch(const AttnParams &p, const Plan &plan, int n_sms, cudaStream_t stream) {
  if (p.batch.n_seqs) plan.wide ? kv8_wide_launch(p, kBf16, stream) : kv8_few_launch(p, plan.rows, kBf16, stream);
  if (p.cache.dim == 64) launch<64, kBf16>(p, plan, stream);
  else if (p.cache.dim == 128) launch<128, kBf16>(p, plan, stream);
  else launch<256, kBf16>(p, plan, stream);
  if (!p.weights || !p.batch.n_seqs) return;
  if (!p.scores) return kv8_weights_launch(p, kBf16, n_sms, stream);
  auto add = [&](auto kernel) {
    launch_after(kernel, dim3((unsigned)(p.batch.n_seqs * p.cache.heads), (unsigned)std::min((p.score_tokens + 1023) / 1024, 16)), kAddThreads, 0,
                 stream, p);
  };
  if (plan.rows == 4) add(kv8_weights_add<4>);
  else if (plan.rows == 8) add(kv8_weights_add<8>);
  else add(kv8_weights_add<16>);
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
    *bytes = make_plan(device_id, c, b, *args).bytes;
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
    if (overlaps_itself(a.n_rows, a.out_row_stride, a.q_heads, a.out_head_stride, c.dim)) throw Error::invalid("elements of out overlap");
    if (a.weights && overlaps_itself(b.n_seqs, a.weights_seq_stride, c.heads, a.weights_head_stride, a.weights_capacity))
      throw Error::invalid("elements of weights overlap");
    // a row tile of q has been read when its part of out is written
    const bool in_place = a.q == a.out && a.q_row_stride == a.out_row_stride && a.q_head_stride == a.out_head_stride;
    if (!in_place && shares(a, c.dim)) throw Error::invalid("out overlaps q");
    const Plan plan = make_plan(device_id, c, b, a);
    if (in_place && a.weights && !plan.score_tokens) throw Error::invalid("out overlaps q, which these weights are computed from again");
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
    p.scores = plan.score_tokens ? (float *)(ws + plan.scores) : nullptr;
    p.score_tokens = plan.score_tokens;
    p.q_row = (int64_t)a.q_row_stride, p.q_head = (int64_t)a.q_head_stride;
    p.out_row = (int64_t)a.out_row_stride, p.out_head = (int64_t)a.out_head_stride;
    p.w_seq = (int64_t)a.weights_seq_stride, p.w_head = (int64_t)a.weights_head_stride;
    p.w_capacity = (int)std::min<size_t>(a.weights_capacity, 0x7fffffff);
    p.q_heads = (int)a.q_heads;
    p.group = (int)a.q_heads / c.heads;
    p.max_query = (int)std::min<size_t>(a.max_query, a.n_rows);
    p.row_tiles_most = plan.row_tiles;
    p.units_most = plan.units;
    p.causal = a.causal != 0;
    p.clear_tail = a.clear_tail;
    p.vec_q = (uintptr_t)a.q % 16 == 0 && (a.q_row_stride | a.q_head_stride) % 8 == 0;
    p.vec_out = (uintptr_t)a.out % 8 == 0 && (a.out_row_stride | a.out_head_stride) % 4 == 0;
    p.scale = a.scale;
    p.n_ctas = plan.n_ctas;
    p.device = device_id;
    DeviceGuard on_device(device_id);
    if (a.dtype == PF_KV8_BF16) launch<true>(p, plan, kv8_sm_count(device_id), (cudaStream_t)stream);
    else launch<false>(p, plan, kv8_sm_count(device_id), (cudaStream_t)stream);
  });
}

}  // extern "C"
