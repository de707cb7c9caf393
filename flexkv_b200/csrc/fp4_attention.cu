// Attention over the 4-bit paged cache (format: fp4_cache.cu).
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j   over the keys row i sees
//
// Row i of sequence b sits at position len_b - qlen_b + i and sees the keys
// up to its own position (causal) or all len_b.  Query head h reads key head
// h / (q_heads / kv_heads).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <random>

#include "fkv_common.h"
#include "fp4_format.cuh"
#include "fp4_launch.cuh"
#include "fp4_wait.cuh"

namespace fkv {
namespace {

struct AttnArgs {
  const uint8_t *layer;
  int64_t num_blocks, kv_stride, block_stride;
  int tokens_per_block, kv_heads, group;
  int upb;             // units of a block
  Divisor by_upb;      // positions are below 2^31, so a unit's number is below 2^27
  const uint8_t *q;
  int64_t q_token_stride, q_head_stride;  // bytes
  uint8_t *out;
  int64_t o_token_stride, o_head_stride;  // bytes
  float *lse;
  int64_t num_q;
  const int32_t *tables;
  int64_t table_stride;
  int max_blocks;
  const int32_t *seq_lens;
  const int32_t *cu;  // null: rows_each rows each
  int rows_each;
  int table_tokens;  // tokens that a table's width holds
  int num_seqs;
  float scale;
  int causal;
  int fill_rest;  // rows of no sequence: zeros, lse -inf
};

// A row's sum of weights 2^((s - centre) * mul + kLift) over its scores s, whole or of a part of its keys.
// What is joined has the row's mul in common; without a key the centre is -inf and the sum 0.
struct alignas(16) RowSum {
  float centre, l, mul, unused;
};
constexpr float kLift = 7.0f;  // see fp4_decode_kernel's weights

__device__ __forceinline__ float natural_lse(const RowSum &r) {
  return r.l == 0.0f ? -INFINITY : (fmaf(r.centre, r.mul, -kLift) + __log2f(r.l)) * 0.6931471805599453f;
}

// N channels from c on of (token, head) row `row` of a sequence.
template <bool BF16, int N>
__device__ __forceinline__ void store_row(const AttnArgs &a, int64_t first, int h, int row, int nrows, int c,
                                          const float (&v)[N], const RowSum &sum) {
  if (row >= nrows) return;
  const int i = row / a.group, qh = h * a.group + row - i * a.group;
  const float inv = sum.l == 0.0f ? 0.0f : 1.0f / sum.l;
  uint32_t w[N / 2];
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    if (BF16) {
      const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * k] * inv, v[2 * k + 1] * inv);
      w[k] = *reinterpret_cast<const uint32_t *>(&x);
    } else {
      const __half2 x = __floats2half2_rn(v[2 * k] * inv, v[2 * k + 1] * inv);
      w[k] = *reinterpret_cast<const uint32_t *>(&x);
    }
  }
  uint8_t *dst = a.out + (first + i) * a.o_token_stride + qh * a.o_head_stride + 2 * c;
  if constexpr (N >= 8) {
#pragma unroll
    for (int k = 0; k < N / 8; ++k)
      reinterpret_cast<uint4 *>(dst)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  } else {
    *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
  }
  if (a.lse && c == 0) a.lse[(first + i) * (a.kv_heads * a.group) + qh] = natural_lse(sum);
}

// Rows before the first sequence and behind the last, this CTA's share of them,
// by `n` of its threads (a kernel of its own before the call took 16 us for
// 12000 rows of 32 heads of 128, all of which the sequences then wrote).
__device__ __forceinline__ void fill_rest(const AttnArgs &a, int D, int thread, int n) {
  const int64_t lo = min((int64_t)max(a.cu[0], 0), a.num_q);
  const int64_t hi = max(min((int64_t)max(a.cu[a.num_seqs], 0), a.num_q), lo), rest = lo + a.num_q - hi;
  const int heads = a.kv_heads * a.group, pieces = heads * (D / 8);
  for (int64_t i = blockIdx.x; i < rest; i += gridDim.x) {
    const int64_t row = i < lo ? i : hi + i - lo;
    for (int j = thread; j < pieces; j += n) {
      const int h = j / (D / 8), c = j - h * (D / 8);
      *reinterpret_cast<uint4 *>(a.out + row * a.o_token_stride + h * a.o_head_stride + 16 * c) = make_uint4(0, 0, 0, 0);
      if (a.lse && c == 0) a.lse[row * heads + h] = -INFINITY;
    }
  }
}

// ---- few rows: decoding, and checking a handful of proposed tokens ----------
//
// All rows of one key head and sequence (new tokens x query heads of the
// group, R = 8 * NT of them at a time) go through the cache together, so the
// cache is read once; what bounds the kernel is that read.
//
// S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16 with the rows as the
// short side n: one new token of a group of up to 8 heads fills a tile where
// a tile with rows as the long side would be a sixteenth full.  (tcgen05's
// smallest tile has 64 rows, and its operands would have to be written to
// shared memory in 16 bits, four times the bytes that arrive.)  K and V go
// from their 4-bit bytes in shared memory straight into the fragments:
//  * the order of the contraction is free, so lane t of a quad takes D / 4
//    consecutive channels of a key: 16 bytes, two scales;
//  * V needs pairs of tokens in a register where the bytes hold pairs of
//    channels: the nibbles of two tokens are interleaved (four instructions
//    for sixteen values) before they are converted.
// x' = q * s is exact in half, so no precision is lost there; queries are
// brought into half by a power of two for each row (bfloat16's 8 bits fit).
// Weights are rounded to half for the second product (2^-11 of a weight; the
// sum of weights is taken before the rounding, in 32 bits).
//
// The sequences' units (16 tokens) x key heads x blocks of R rows form one
// line of work that is cut into equal pieces, one for each warp of the GPU,
// whatever the lengths are; they are read on the device, so a captured launch
// follows them.  A warp walks through its piece by itself, with its own ring
// of asynchronous copies that runs ahead over the borders of sequences and
// heads, and its own running sum, maximum and O.  What it holds whole it
// writes out; the rest is joined once at the end within the CTA, and pieces of
// one (sequence, head) in several CTAs by the CTA that comes last, both in a
// fixed order.
//
// Measured (B200, bfloat16, heads of 128): 48 sequences of 6000 to 16384 tokens,
// 8 key heads, 32 query heads: 130 us for 630 MB, 4.8 TB/s, 74 % of a copy's
// rate (call after call, each on other inputs), 144 where other work comes
// between; what bounds it there is the issue of 315 instructions a unit (64
// conversions, 64 multiplications, 16 products; the read alone takes 106 us).
// Why 12 warps, two units a stage and three stages: one unit and six stages take
// 144 us, 16 warps with one unit and four stages 138, 8 warps with four units
// 136, 16 warps with two stages of two 131.5 but 15.3 us instead of 13.2 for one
// sequence of 1000 tokens (at that time).  Small calls are bound by the chain
// launch, lengths, pages, keys, joins: that sequence 11 us, one of 131071 tokens
// 17.9 us.

// Warps of a CTA, units of a chunk and chunks of a warp's ring, for NT row tiles.
// Heads of 64 leave registers for more: 64 sequences of 4000 tokens, 8 key heads,
// take 50 us with 16 warps and 52 with 12 (NT 1), 63 us with 4 units a chunk and
// 69 with 2 (NT 2).
template <int D, int NT>
struct DecodeShape {
  static constexpr int kWarps = NT == 2 ? 8 : D == 64 ? 16 : 12;
  static constexpr int kUps = NT == 2 && D == 64 ? 4 : 2, kStages = 3;
};

// A weight is 2^((s - centre) * mul + kLift): s the sum q k, mul what turns it
// into a power of two.  The centre is the largest sum when it was set; it moves
// when one passes it by 8 powers of two: the largest weight of a row lies between
// 2^7 and 2^15, so its rounding to half (a step of 2^-24 at the least) takes
// at most 2^-32 of the sum of weights from any weight, however small.  The
// difference is taken first and is nearly exact, in joins too: a product rounded
// before it, s * mul - base, is off by powers of two where scores pass 2^24, and
// weights overflowed half there.
constexpr float kMove = 15.0f;
constexpr float kLowest = -3.4e38f;  // below every centre but that of a row without keys

struct Item {     // what a warp needs of one sequence
  int len;        // tokens that can be seen: the table's end at most
  int len_q;      // tokens as given: positions count from here
  int64_t first;  // first row in q
  int rows;       // new tokens
  int blocks;     // blocks of R (token, head) rows
  int units;      // units to pass, at least one where there are rows
};

template <int R>
__device__ __forceinline__ Item item_of(const AttnArgs &a, int b) {
  Item it;
  if (a.cu) {
    const int64_t lo = min((int64_t)max(a.cu[b], 0), a.num_q), hi = min((int64_t)max(a.cu[b + 1], 0), a.num_q);
    it.first = lo, it.rows = (int)max(hi - lo, (int64_t)0);
  } else {
    it.rows = a.rows_each;
    it.first = (int64_t)b * a.rows_each;
  }
  it.len_q = a.seq_lens[b];
  it.len = min(max(it.len_q, 0), a.table_tokens);
  it.blocks = (it.rows * a.group + R - 1) / R;
  it.units = it.rows ? max((it.len + 15) >> 4, 1) : 0;
  return it;
}

// The cut of all work into pieces, and where this CTA's starts; every warp
// finds it for itself.
struct Cut {
  int64_t each, more;  // a CTA has each + 1 units, from CTA `more` on each
  int64_t begin, end;
  int b;           // sequence of `begin`
  int64_t before;  // units before sequence b
  __device__ int cta_of(int64_t x) const {
    const int64_t y = (each + 1) * more;
    const int64_t n = x < y ? x : x - y, d = x < y ? each + 1 : each;
    return (int)((x < y ? 0 : more) + ((n | d) >> 32 ? n / d : (uint32_t)n / (uint32_t)d));
  }
};

template <int R, int kWarps>
__device__ __forceinline__ Cut find_cut(const AttnArgs &a) {
  const int lane = threadIdx.x & 31;
  auto work_of = [&](int b) {
    const Item it = item_of<R>(a, b);
    return (int64_t)it.units * (it.blocks * a.kv_heads);
  };
  auto scan = [&](int64_t x) {  // sum over the lanes up to this one
#pragma unroll 1
    for (int i = 1; i < 32; i <<= 1) {
      const int64_t o = __shfl_up_sync(~0u, x, i);
      if (lane >= i) x += o;
    }
    return x;
  };
  Cut cut;
  int64_t mine = lane < a.num_seqs ? work_of(lane) : 0, total = mine;
  for (int b = lane + 32; b < a.num_seqs; b += 32) total += work_of(b);
  total = __shfl_sync(~0u, scan(total), 31);
  const int64_t want = (total + kWarps - 1) / kWarps;  // a unit for each warp, at least
  uint32_t n = want < gridDim.x ? (uint32_t)want : gridDim.x;
  if (a.num_seqs == 1 && total) {
    // All (head, row block)s are as long: cut between them, and into no more than leave a warp kWhole units each
    // while that spares the second step of the join.  1000 tokens, 8 heads: 11.0 us, and 14.0 with every cut at a
    // unit a warp.  For one sequence only: two of them, cut at a unit a warp, take 14.5 us and four 15.7.
    constexpr int kWhole = 8;
    const Item it = item_of<R>(a, 0);
    const uint32_t items = it.blocks * a.kv_heads, few = (it.units + kWarps * kWhole - 1) / (kWarps * kWhole);
    if (items <= gridDim.x) n = items * max(few <= kWarps ? min(n / items, few) : n / items, 1u);
  }
  if (blockIdx.x >= n) {
    cut.begin = cut.end = total;
    return cut;
  }
  cut.each = total >> 32 ? total / n : (uint32_t)total / n;
  cut.more = total - cut.each * n;
  const int64_t c = blockIdx.x;
  cut.begin = c * cut.each + min(c, cut.more), cut.end = cut.begin + cut.each + (c < cut.more);
  // the sequence of `begin`, 32 at a time
  int64_t before = 0;
  for (int b0 = 0;; b0 += 32) {
    if (b0) mine = b0 + lane < a.num_seqs ? work_of(b0 + lane) : 0;
    const int64_t upto = scan(mine);
    const uint32_t past = __ballot_sync(~0u, before + upto > cut.begin);
    if (past) {  // `begin` lies before the total, so this comes
      const int l = __ffs(past) - 1;
      cut.b = b0 + l;
      cut.before = before + __shfl_sync(~0u, upto - mine, l);
      return cut;
    }
    before += __shfl_sync(~0u, upto, 31);
  }
}

// A walk over a warp's part of the line of work: segments (the part of one
// (sequence, head, row block) in it), and chunks of kUps units in them.
template <int R, int kUps>
struct Walk {
  int left;      // units of the part from u0 on
  int b, idx;    // sequence; (head, row block) in it
  int h, rb;
  Item it;
  int u0, u1;    // units of the segment
  int at;        // the next chunk

  // `off`: the part's start, from that of sequence `seq` on
  __device__ void start(const AttnArgs &a, int seq, int64_t off, int units) {
    left = units;
    b = seq;
    for (;;) {
      it = item_of<R>(a, b);
      const int64_t w = (int64_t)it.units * (it.blocks * a.kv_heads);
      if (off < w) break;
      off -= w, ++b;  // the part has units, so this ends
    }
    idx = (int)(off >> 32 ? off / it.units : (uint32_t)off / (uint32_t)it.units);
    u0 = (int)(off - (int64_t)idx * it.units);
    open();
  }
  __device__ void open() {
    h = it.blocks == 1 ? idx : idx / it.blocks, rb = idx - h * it.blocks;
    u1 = min(it.units, u0 + left);
    at = u0;
  }
  // To the next segment; false at the end of the part.
  __device__ bool next_segment(const AttnArgs &a) {
    left -= u1 - u0;
    if (left <= 0) return false;
    u0 = 0;
    if (++idx == it.blocks * a.kv_heads) {
      idx = 0;
      do it = item_of<R>(a, ++b);
      while (it.blocks == 0);  // there is work left, so this ends
    }
    open();
    return true;
  }
  __device__ void next_chunk() { at += kUps; }
  __device__ bool has_chunk() const { return at < u1; }
  __device__ int chunk_units() const { return min(kUps, u1 - at); }
};

__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_if(uint32_t dst, const uint8_t *src, bool on) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %2, 0;\n @p cp.async.cg.shared.global [%0], [%1], 16;\n}" ::"r"(dst), "l"(src),
               "r"((int)on)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int WORDS>
__device__ __forceinline__ void load_shared(uint32_t (&w)[WORDS], uint32_t at) {
  if constexpr (WORDS == 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
  else if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
  else
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at));
}
template <int BYTES>
__device__ __forceinline__ uint32_t load_scales(uint32_t at) {
  uint32_t r;
  if constexpr (BYTES == 2)
    asm volatile("{\n .reg .b16 h;\n ld.shared.b16 h, [%1];\n cvt.u32.u16 %0, h;\n}" : "=r"(r) : "r"(at));
  else
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(at));
  return r;
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two floats in a register pair, as the packed instructions take them.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The power of two that brings a row's largest value to [2^10, 2^11), within
// what a float holds; its inverse is exact too.
__device__ __forceinline__ float row_factor(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23) - 127;
  int k = 10 - e;
  k = k > 126 ? 126 : k;
  k = (amax > 0.0f && amax <= 3.4e38f) ? k : 0;
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

// What a row's queries are multiplied by: its factor, with the sign of softmax_scale, so that mul is positive and no
// score 0 * inf.  A row with an infinite query has the scores inf, -inf and NaN and so no softmax: they all become
// NaN, lest a row of -inf alone pass for one that sees nothing.
__device__ __forceinline__ float query_factor(float amax, float factor, float scale) {
  return amax > 3.4e38f ? __int_as_float(0x7FFFFFFF) : scale < 0.0f ? -factor : factor;
}
// From a row's q k to powers of two; its bounds keep 0 * mul and s * mul numbers.
__device__ __forceinline__ float row_mul(float scale, float factor) {
  return fminf(fmaxf(fabsf(scale) * 1.4426950408889634f * (1.0f / factor), 1e-37f), 3e38f);
}
// The sum past which the centre moves: not above centre + 8 / mul, lest a weight pass 2^15.
__device__ __forceinline__ float bar_of(float centre, float mul) {
  return __fadd_rd(centre, __fdividef(kMove - kLift, mul));
}
// What weights around `from` are around `to`, which is not below it.
__device__ __forceinline__ float moved(float from, float to, float mul) { return exp2_fast((from - to) * mul); }

// What a warp has of a (sequence, head, row block) that it does not hold whole.
template <int D, int NT>
struct Part {
  static constexpr int kPad = D + 4;  // floats of a row: quads store 16-byte pieces of rows 2 t and 2 t + 1
  alignas(16) float o[8 * NT][kPad];
  RowSum sum[8 * NT];
};
// The rows a part belongs to, and its place in the line of work.
struct PartMeta {
  int there, starts, ends;
  int h, row0, nrows;      // key head; first (token, head) row, and how many the sequence has
  int64_t first;           // the sequence's first row in q
  int64_t begin, last;     // first and last unit of the whole (sequence, head, row block)
};

template <int D, int NT>
struct DecodeSmem {
  static constexpr int kWarps = DecodeShape<D, NT>::kWarps, kUps = DecodeShape<D, NT>::kUps, kStages = DecodeShape<D, NT>::kStages;
  alignas(128) uint8_t ring[kWarps][kStages][kUps][2][9 * D];  // at the end: the part that starts in the warp
  Part<D, NT> part[kWarps];                                     // the part that goes on from the warp before
  PartMeta meta[kWarps][2];
  PartMeta open[2];  // parts of the CTA that others share: 0 goes on from another CTA, 1 starts here
  int is_last;
  static_assert(sizeof(Part<D, NT>) <= sizeof(ring[0]), "a part has to fit a warp's ring");
};

template <int D>
__host__ __device__ constexpr int slot_floats(int rows) { return rows * (D + 4); }  // and their RowSums

// Joins `count` consecutive warps' parts from that of warp w0 on, whose part
// is the one in its ring when `ring`: into rows of the output, or into a slot
// of the workspace.
template <int D, int NT, bool BF16>
__device__ __forceinline__ void join_parts(const AttnArgs &a, const DecodeSmem<D, NT> &sm, int w0, bool ring, int count,
                                           const PartMeta &pm, float *slot) {
  constexpr int R = 8 * NT, kWarps = DecodeShape<D, NT>::kWarps;
  auto part = [&](int k) -> const Part<D, NT> & {
    return k == 0 && ring ? *reinterpret_cast<const Part<D, NT> *>(sm.ring[w0]) : sm.part[w0 + k];
  };
  for (int i = threadIdx.x; i < R * (D / 4); i += kWarps * 32) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float to = kLowest, acc[4] = {};
#pragma unroll 4
    for (int k = 0; k < count; ++k) to = fmaxf(to, part(k).sum[r].centre);
    RowSum all{to, 0, part(0).sum[r].mul};
#pragma unroll 2
    for (int k = 0; k < count; ++k) {
      const RowSum of = part(k).sum[r];
      const float f = moved(of.centre, to, of.mul);
      const float4 v = *reinterpret_cast<const float4 *>(&part(k).o[r][c]);
      all.l += of.l * f;
      acc[0] += v.x * f, acc[1] += v.y * f, acc[2] += v.z * f, acc[3] += v.w * f;
    }
    if (slot) {
      *reinterpret_cast<float4 *>(slot + r * D + c) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (c == 0) reinterpret_cast<RowSum *>(slot + R * D)[r] = all;
    } else {
      store_row<BF16>(a, pm.first, pm.h, pm.row0 + r, pm.nrows, c, acc, all);
    }
  }
}

// Counts an arrival at a word of the workspace and says how many there were.
// What the word held before does not matter: a call (or a captured launch,
// which leaves its words at 0) knows its own counts by its number.
__device__ __forceinline__ int arrive(unsigned long long *word, unsigned long long call) {
  const unsigned long long old = *(volatile unsigned long long *)word;
  if ((old >> 16) != call) atomicCAS(word, old, call << 16);  // where it fails another arrival has done it
  return (int)((atomicAdd(word, 1ull) + 1) & 0xFFFF);
}

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(DecodeShape<D, NT>::kWarps * 32, 1)
fp4_decode_kernel(const __grid_constant__ AttnArgs a, float *__restrict__ slots, unsigned long long *__restrict__ arrived,
                  unsigned long long call) {
  constexpr int R = 8 * NT, KS = D / 16, KW = D / 32, VB = D / 16;  // k-steps; words of a lane's K row; bytes of its V row
  constexpr int kWarps = DecodeShape<D, NT>::kWarps, kUps = DecodeShape<D, NT>::kUps, kStages = DecodeShape<D, NT>::kStages;
  constexpr int kUnit = 9 * D, kSlot = kUps * 2 * kUnit, kBatch = 32 / kUps;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  auto &sm = *reinterpret_cast<DecodeSmem<D, NT> *>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  after_previous();
  if (lane < 2) sm.meta[warp][lane].there = 0;
  const Cut cut = find_cut<R, kWarps>(a);
  const int64_t begin = cut.begin;
  const int units_here = (int)(cut.end - begin);
  if (a.fill_rest) fill_rest(a, D, threadIdx.x, kWarps * 32);
  if (units_here <= 0) return;
  // the first warps have a unit more, or all there are
  const int share = units_here / kWarps, rest = units_here - share * kWarps;
  const int from = warp * share + min(warp, rest), to = from + share + (warp < rest);

  if (from < to) {
    Walk<R, kUps> in, cur;  // the copies' walk runs ahead
    in.start(a, cut.b, begin + from - cut.before, to - from);
    cur = in;
    const uint32_t ring = smem_addr(sm.ring[warp]);
    bool more = true;
    // Where the segment's next 32 units lie, one for each lane: bytes from the layer's start, -1 for a page
    // outside the pool; and the pages of the 32 after them, on their way.
    int64_t where = -1;
    int next_page = -1, turn = 0;
    auto page_of = [&](int u) {
      const int e = divide(u, a.by_upb);  // u / units of a block
      return u < in.u1 && e < a.max_blocks ? a.tables[in.b * a.table_stride + e] : -1;
    };
    auto take_batch = [&] {
      const int u = in.at + lane, e = divide(u, a.by_upb);
      where = next_page < 0 || next_page >= a.num_blocks
                  ? -1
                  : next_page * a.block_stride + ((int64_t)in.h * a.upb + u - e * a.upb) * kUnit;
      next_page = page_of(u + 32);
      turn = 0;
    };
    uint32_t valid = 0;  // bit kUps * stage + unit: the unit's page is in the pool and its copy was started
    auto issue = [&](int stage) {
      if (more) {
        const int n = in.chunk_units();
        uint32_t mask = 0;
#pragma unroll
        for (int u = 0; u < kUps; ++u) {
          const int64_t off = __shfl_sync(~0u, where, turn * kUps + u);
          if (u < n && off >= 0) {
            mask |= 1u << u;
            const uint32_t dst = ring + stage * kSlot + u * 2 * kUnit + lane * 16;
            const uint8_t *src = a.layer + off + lane * 16, *srcv = src + a.kv_stride;
#pragma unroll
            for (int i = 0; i < kUnit / 512; ++i) {
              copy16(dst + i * 512, src + i * 512);
              copy16(dst + kUnit + i * 512, srcv + i * 512);
            }
            // what is left of both sides goes together, V's by the lanes after K's
            constexpr int kFull = kUnit / 512 * 512, kRest = (kUnit - kFull) / 16;
            static_assert(2 * kRest <= 32, "the rests of both sides are one copy");
            const bool isv = lane >= kRest;
            copy16_if(dst + kFull + (isv ? kUnit - kRest * 16 : 0), (isv ? srcv - kRest * 16 : src) + kFull, lane < 2 * kRest);
          }
        }
        valid = (valid & ~(((1u << kUps) - 1) << (kUps * stage))) | (mask << (kUps * stage));
        in.next_chunk();
        if (!in.has_chunk()) {
          more = in.next_segment(a);
          if (more) {
            next_page = page_of(in.at + lane);
            take_batch();
          }
        } else if (++turn == kBatch) {
          take_batch();
        }
      }
      copies_commit();
    };
    next_page = page_of(in.at + lane);
    // queries of the segment, as they lie: n = g, channels D / 4 * t on
    uint32_t qx[NT][D / 8];
    auto load_queries = [&] {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = cur.rb * R + n * 8 + g;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) qx[n][i] = 0;
        if (r < cur.it.rows * a.group) {
          const int i0 = r / a.group;
          const uint8_t *p = a.q + (cur.it.first + i0) * a.q_token_stride +
                             (cur.h * a.group + r - i0 * a.group) * a.q_head_stride + t * (D / 2);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p) + i);
            qx[n][4 * i] = v.x, qx[n][4 * i + 1] = v.y, qx[n][4 * i + 2] = v.z, qx[n][4 * i + 3] = v.w;
          }
        }
      }
    };
    load_queries();
    take_batch();
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);
    int stage = 0;
    // a lane's places in a unit: its pieces of keys and values and of their scales
    const int tok = (g & 1) ? ((g >> 1) ^ 1) + 4 : (g >> 1);  // S^T: rows g, g + 8 are tokens tok, tok + 8
    const int tk[2] = {t, (t ^ 1) + 4};                       // tokens of rows 2 t, 2 t + 1
    const uint32_t at_k = tok * (D / 2) + t * (D / 8), at_ks = 8 * D + tok * (D / 16) + t * (D / 64);
    const uint32_t at_v[2] = {kUnit + tk[0] * (D / 2) + g * VB, kUnit + tk[1] * (D / 2) + g * VB};
    const uint32_t at_vs[2] = {kUnit + 8 * D + tk[0] * (D / 16) + g * D / 128,
                               kUnit + 8 * D + tk[1] * (D / 16) + g * D / 128};

    for (;;) {  // segments
      const int h = cur.h;
      const int row0 = cur.rb * R, nrows = cur.it.rows * a.group;  // of the sequence's (token, head) rows
      // queries in half; multiplier and end of the rows 2 t, 2 t + 1
      uint32_t qf[NT][KS][2];
      float mul[NT][2], bar[NT][2];  // bar: the sum q k past which the row's centre moves
      int end[NT][2], lowest = INT32_MAX, highest = 0;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t(&x)[D / 8] = qx[n];
        float amax = 0;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const float2 f = pair_to_float2<BF16>(x[i]);
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
        amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
        const float f = row_factor(amax), fs = query_factor(amax, f, a.scale);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 y = pair_to_float2<BF16>(x[2 * k + j]);
            qf[n][k][j] = pack_half2(y.x * fs, y.y * fs);
          }
        const float mine = row_mul(a.scale, f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mul[n][j] = __shfl_sync(~0u, mine, (2 * t + j) * 4);
          bar[n][j] = -INFINITY;
          const int rr = row0 + n * 8 + 2 * t + j;
          int e = 0;
          if (rr < nrows) {
            e = cur.it.len;
            if (a.causal) e = max(min(e, cur.it.len_q - cur.it.rows + rr / a.group + 1), 0);
            lowest = min(lowest, e);
          }
          end[n][j] = e;
          highest = max(highest, e);
        }
      }
#pragma unroll
      for (int i = 1; i < 4; i <<= 1) {
        lowest = min(lowest, __shfl_xor_sync(~0u, lowest, i));
        highest = max(highest, __shfl_xor_sync(~0u, highest, i));
      }

      float o[NT][KS][4], centre[NT][2], l[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][k][i] = 0;
        centre[n][0] = centre[n][1] = 0;
        l[n][0] = l[n][1] = 0;
      }

      for (; cur.has_chunk(); cur.next_chunk()) {
        const uint32_t ok = (valid >> (kUps * stage)) & ((1u << kUps) - 1);
        copies_wait<kStages - 2>();
        __syncwarp();  // the chunk is there, and every lane is done with the one before, whose slot is the next to fill
        const uint32_t slot = ring + stage * kSlot;
        issue(stage == 0 ? kStages - 1 : stage - 1);
        // The units of the chunk together: their chains of products overlap.  One that is not there (past the
        // segment, or its page outside the pool) is all hidden, whatever its place holds.
        float s[kUps][NT][4];
        uint32_t vw[kUps][4][VB / 4], vc[kUps][4];
#pragma unroll
        for (int u = 0; u < kUps; ++u) {
          const uint32_t at = slot + u * 2 * kUnit;
          uint32_t w[2][KW], sc[2][(D + 127) / 128 * 2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            load_shared(w[i], at + at_k + 8 * i * (D / 2));
            const uint32_t c = load_scales<D / 64>(at + at_ks + 8 * i * (D / 16));
            sc[i][0] = __byte_perm(c, 0, 0x0404) >> 1;
            if constexpr (D == 128) sc[i][1] = __byte_perm(c, 0, 0x1414) >> 1;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][n][i] = 0;
#pragma unroll
          for (int j = 0; j < KW; ++j) {
            uint32_t x[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              e2m1x8_to_half2(w[i][j], x[i]);
#pragma unroll
              for (int k = 0; k < 4; ++k) x[i][k] = hmul2(x[i][k], sc[i][D == 128 ? j / 2 : 0]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t f[4] = {x[0][2 * k], x[1][2 * k], x[0][2 * k + 1], x[1][2 * k + 1]};
#pragma unroll
              for (int n = 0; n < NT; ++n) mma(s[u][n], f, qf[n][2 * j + k][0], qf[n][2 * j + k][1]);
            }
          }
          // V^T: lane g takes channels D / 8 * g on, of the tokens of rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            load_shared(vw[u][i], at + at_v[i & 1] + 8 * (i >> 1) * (D / 2));
            vc[u][i] = load_scales<1>(at + at_vs[i & 1] + 8 * (i >> 1) * (D / 16));
          }
        }
        const int base = cur.at * 16;
        if (ok != (1u << kUps) - 1 || base + kUps * 16 > lowest) {  // hidden scores to -inf
#pragma unroll
          for (int u = 0; u < kUps; ++u) {
            const bool there = (ok >> u) & 1;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (!there || base + 16 * u + tok + 8 * (i >> 1) >= end[n][i & 1]) s[u][n][i] = -INFINITY;
            // what no row sees may be anything: its scale counts as zero
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!there || base + 16 * u + tk[i & 1] + 8 * (i >> 1) >= highest) vc[u][i] = 0;
          }
        }
        float top[NT][2];
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            top[n][i] = fmaxf(s[0][n][i], s[0][n][i + 2]);
#pragma unroll
            for (int u = 1; u < kUps; ++u) top[n][i] = fmaxf(top[n][i], fmaxf(s[u][n][i], s[u][n][i + 2]));
            grow |= top[n][i] > bar[n][i];
          }
        if (__any_sync(~0u, grow)) {  // rare after the first units
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float x = top[n][j];
#pragma unroll
              for (int i = 4; i < 32; i <<= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, i));
              if (x > bar[n][j]) {  // others stay: a row does not depend on its neighbours
                // a row without a key so far has no sums to move, and its centre may lie above
                const float f = fminf(moved(centre[n][j], x, mul[n][j]), 1.0f);
                centre[n][j] = x;
                bar[n][j] = bar_of(x, mul[n][j]);
                l[n][j] *= f;
#pragma unroll
                for (int k = 0; k < KS; ++k) o[n][k][j] *= f, o[n][k][j + 2] *= f;
              }
            }
        }
#pragma unroll
        for (int u = 0; u < kUps; ++u) {
          uint32_t p[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float2 e;
              if constexpr (NT == 1)  // in pairs: 48 long 133.8 us one by one, 132.0 so; with two tiles 100.4 and 102.6 (64 x 4000, 16 rows)
                e = unpair(fma2(add2(pair(s[u][n][2 * i], s[u][n][2 * i + 1]), pair(-centre[n][0], -centre[n][1])),
                                pair(mul[n][0], mul[n][1]), pair(kLift, kLift)));
              else
                e = make_float2(fmaf(s[u][n][2 * i] - centre[n][0], mul[n][0], kLift),
                                fmaf(s[u][n][2 * i + 1] - centre[n][1], mul[n][1], kLift));
              const float x = exp2_fast(e.x), y = exp2_fast(e.y);
              l[n][0] += x, l[n][1] += y;
              p[n][i] = transpose8(pack_half2(x, y));
            }
          const uint32_t vs[2] = {(vc[u][0] << 7) | (vc[u][1] << 23), (vc[u][2] << 7) | (vc[u][3] << 23)};
#pragma unroll
          for (int j = 0; j < VB / 4; ++j) {
            uint32_t x[2][2][4];  // token pair, channel parity, channel pair
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w0 = vw[u][2 * i][j], w1 = vw[u][2 * i + 1][j];
              e2m1x8_to_half2((w0 & 0x0F0F0F0Fu) | ((w1 << 4) & 0xF0F0F0F0u), x[i][0]);
              e2m1x8_to_half2(((w0 >> 4) & 0x0F0F0F0Fu) | (w1 & 0xF0F0F0F0u), x[i][1]);
#pragma unroll
              for (int k = 0; k < 4; ++k) x[i][0][k] = hmul2(x[i][0][k], vs[i]), x[i][1][k] = hmul2(x[i][1][k], vs[i]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t f[4] = {x[0][0][k], x[0][1][k], x[1][0][k], x[1][1][k]};
#pragma unroll
              for (int n = 0; n < NT; ++n) mma(o[n][4 * j + k], f, p[n][0], p[n][1]);
            }
          }
        }
        if (++stage == kStages) stage = 0;
      }

      const bool starts = cur.u0 == 0, ends = cur.u1 == cur.it.units;
      if (starts && !ends) {  // the part's last segment: the ring is free once its last copies are in
        copies_wait<0>();
        __syncwarp();
      }
      Part<D, NT> &part = starts ? *reinterpret_cast<Part<D, NT> *>(sm.ring[warp]) : sm.part[warp];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float sum = l[n][j];
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) sum += __shfl_xor_sync(~0u, sum, i);
          const int rr = n * 8 + 2 * t + j;
          const RowSum all{bar[n][j] == -INFINITY ? -INFINITY : centre[n][j], sum, mul[n][j]};
          if (starts && ends) {
            float v[D / 8];
#pragma unroll
            for (int k = 0; k < KS; ++k) v[2 * k] = o[n][k][j], v[2 * k + 1] = o[n][k][j + 2];
            store_row<BF16>(a, cur.it.first, h, row0 + rr, nrows, g * (D / 8), v, all);
          } else {
#pragma unroll
            for (int k = 0; k < KS; k += 2)
              *reinterpret_cast<float4 *>(&part.o[rr][g * (D / 8) + 2 * k]) =
                  make_float4(o[n][k][j], o[n][k][j + 2], o[n][k + 1][j], o[n][k + 1][j + 2]);
            if (g == 0) part.sum[rr] = all;
          }
        }
      if (!(starts && ends) && lane == 0) {
        const int64_t unit0 = begin + to - cur.left - cur.u0;
        sm.meta[warp][starts] = {1, starts, ends, h, row0, nrows, cur.it.first, unit0, unit0 + cur.it.units - 1};
      }
      if (!cur.next_segment(a)) break;
      load_queries();
    }
  }

  // Join the warps' parts of each (sequence, head, row block), in their order.
  if (threadIdx.x < 2) sm.open[threadIdx.x].there = 0;
  __syncthreads();
  const bool there = lane < 2 * kWarps && sm.meta[lane >> 1][lane & 1].there;
  uint32_t parts = __ballot_sync(~0u, there);
  const uint32_t ends = __ballot_sync(~0u, there && sm.meta[lane >> 1][lane & 1].ends);
  while (parts) {
    const int p0 = __ffs(parts) - 1;
    const uint32_t e = ends & ~((1u << p0) - 1);
    const int p1 = e ? __ffs(e) - 1 : 31 - __clz(parts);  // the part that ends it, or the last
    parts &= ~((2u << p1) - 1);
    const PartMeta pm = sm.meta[p0 >> 1][p0 & 1];
    const bool whole = pm.starts && e;
    join_parts<D, NT, BF16>(a, sm, p0 >> 1, p0 & 1, (p1 >> 1) - (p0 >> 1) + 1, pm,
                            whole ? nullptr : slots + (int64_t)(2 * blockIdx.x + pm.starts) * slot_floats<D>(R));
    if (!whole && threadIdx.x == 0) sm.open[pm.starts] = pm;
  }

  // The CTA that comes last joins what several CTAs have of one, in their order.
  __threadfence();
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const PartMeta pm = sm.open[i];
    if (!pm.there) continue;
    const int c0 = cut.cta_of(pm.begin), n = cut.cta_of(pm.last) - c0 + 1;
    auto slot_of = [&](int k) { return slots + (int64_t)(2 * (c0 + k) + (k == 0)) * slot_floats<D>(R); };
    // Whether this CTA is the last of `count` at a word; the word is left at 0 for a replay of this launch.
    auto last_of = [&](unsigned long long *word, int count) {
      if (threadIdx.x == 0) {
        const bool last = arrive(word, call) == count;
        __threadfence();
        if (last) *word = 0;
        sm.is_last = last;
      }
      __syncthreads();
      const bool last = sm.is_last;
      __syncthreads();
      return last;
    };
    // Joins the slots k0, k0 + step, ...: a warp gathers every kWarps-th, 8 rows at a time, into its part.
    auto join_slots = [&](int k0, int step, int count, float *to) {
      const int groups = min(count, kWarps);
      if (warp < groups) {
        Part<D, NT> &mine = sm.part[warp];
        for (int n8 = 0; n8 < NT; ++n8) {
          constexpr int kLanes = D / 4, kRows = 32 / kLanes;  // D 64: two rows at a time
          const int c = lane % kLanes * 4;
          float acc[8 / kRows][4];
          RowSum all[8 / kRows];
#pragma unroll
          for (int r = 0; r < 8 / kRows; ++r) all[r] = {kLowest, 0, 0}, acc[r][0] = acc[r][1] = acc[r][2] = acc[r][3] = 0;
#pragma unroll 1
          for (int k = warp; k < count; k += kWarps) {
            const float *slot = slot_of(k0 + k * step);
            float4 of[8 / kRows];  // a RowSum
            float4 v[8 / kRows];
#pragma unroll
            for (int r = 0; r < 8 / kRows; ++r) {
              const int rr = n8 * 8 + r * kRows + lane / kLanes;
              of[r] = __ldcg(reinterpret_cast<const float4 *>(slot + R * D) + rr);
              v[r] = __ldcg(reinterpret_cast<const float4 *>(slot + rr * D + c));
            }
#pragma unroll
            for (int r = 0; r < 8 / kRows; ++r) {
              const float mul = of[r].z, to = fmaxf(all[r].centre, of[r].x);
              const float f = moved(all[r].centre, to, mul), y = moved(of[r].x, to, mul);
              all[r] = {to, all[r].l * f + of[r].y * y, mul};
              acc[r][0] = acc[r][0] * f + v[r].x * y, acc[r][1] = acc[r][1] * f + v[r].y * y;
              acc[r][2] = acc[r][2] * f + v[r].z * y, acc[r][3] = acc[r][3] * f + v[r].w * y;
            }
          }
#pragma unroll
          for (int r = 0; r < 8 / kRows; ++r) {
            const int rr = n8 * 8 + r * kRows + lane / kLanes;
            *reinterpret_cast<float4 *>(&mine.o[rr][c]) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
            if (c == 0) mine.sum[rr] = all[r];
          }
        }
      }
      __syncthreads();
      join_parts<D, NT, BF16>(a, sm, 0, false, groups, pm, to);
      __threadfence();
      __syncthreads();
    };
    // More than a slot a warp: the CTAs join them in groups first, so that no CTA has to read them all.
    int step = 1, count = n;
    if (n > kWarps) {
      const int k0 = (blockIdx.x - c0) / kWarps * kWarps, size = min(kWarps, n - k0);
      // by slot: a CTA can end one of these and start another
      if (!last_of(arrived + gridDim.x + 2 * (c0 + k0) + (k0 == 0), size)) continue;
      join_slots(k0, 1, size, slot_of(k0));
      step = kWarps, count = (n + kWarps - 1) / kWarps;
    }
    if (last_of(arrived + c0, count)) join_slots(0, step, count, nullptr);
  }
}

// ---- many rows: prompts behind a cached prefix ------------------------------
//
// With hundreds of rows for each key the products bound the kernel, so they go
// to tcgen05.  A CTA takes kTiles * 128 (token, head) rows of one sequence and
// key head through the keys, kKeys at a time, as separate warps:
//  * four warps bring K and V in: 4-bit bytes from global memory into
//    registers (a chunk ahead), to half, into shared memory in the 128-byte
//    swizzled layout.  K as it lies is K-major for S = Q K^T, V is MN-major
//    for O = P V: no transpose;
//  * one thread for each tile of 128 rows issues its products: S into tensor
//    memory, and O += P V with P read from there;
//  * four warps for each tile of rows take S, a thread a row: weights
//    in half go back over S as P, their sum stays in the thread.  A row's
//    centre moves only when a score passes it by 8 powers of two, as in the
//    kernel above: then O is scaled in place.
// Two tiles of rows alternate: while one is in softmax the tensor core works
// on the other, and K and V are converted once for both.  A tile has two
// buffers for S, so that the next scores are there when a softmax ends.
// Tensor memory (512 columns): O of both tiles, two S of both; P lies over S.
// A block of 128 rows or fewer has one tile; the other's warps help to bring K
// and V in.  Where the blocks of rows are fewer than the SMs, several CTAs share a block's
// keys, and a second kernel joins what they have.
//
// Measured (B200, bfloat16, heads of 128, 4 query heads to a key head): three
// chunks of about 3900 tokens behind 1500 cached ones, 655 GFLOP: 732 us call after
// call, each on other inputs, 895 TFLOP/s, 54 % of a library product's rate alone
// and 64 % of its sustained one (706 us where the inputs stay the same).
// A chunk of 64 keys for both tiles takes about 2000 cycles of an SM: the tensor
// core is busy for 1300 of them (a product of S with 64 columns takes 48 cycles,
// its operands being 6 KiB of shared memory, one with P 64), the exponentials for
// 1024.  What is lost lies between them: each tile's chain softmax, P V, S.
// Tried and slower: chunks of 128 keys with one S (740 us), tiles that take turns
// at the exponentials (730), part of the exponentials as polynomials (from 810),
// the maximum found while the last weights are taken (780).

constexpr int kTiles = 2, kKeys = 64, kRing = 4;
constexpr int kFillWarps = 4;
constexpr int kManyThreads = (4 * kTiles + kFillWarps + kTiles) * 32;

template <int D>
struct ManySmem {
  static constexpr int kRows = 128 * 128, kCols = kKeys * 128;  // 64 halves of 128 rows, of kKeys keys, swizzled
  alignas(1024) uint8_t q[kTiles][D / 64][kRows];
  alignas(1024) uint8_t k[kRing][D / 64][kCols];
  alignas(1024) uint8_t v[kRing][D / 64][kCols];
  uint64_t q_full, full[kRing], empty[kRing];  // of a step: K two chunks ahead, and V
  uint64_t s_full[kTiles][2], p_full[kTiles][2], o_done[kTiles], all_done[kTiles];
  alignas(4) uint8_t bad[2 * kRing][kFillWarps];  // of a chunk of keys, a warp's unit: its page is outside the pool
  uint32_t tmem;
};

// A shared memory operand in the 128-byte swizzled layout.  K-major: 8 rows of
// 128 bytes every 1024 bytes.  MN-major: 8 rows along K every 1024 bytes, the
// next 64 columns a block of kKeys rows further.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, bool mn_major) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(mn_major ? (kKeys * 128) >> 4 : 1) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// 128 rows, N columns, half operands, float sums.
__host__ __device__ constexpr uint32_t mma_desc(int n, bool b_mn_major) {
  return 1u << 4 | (b_mn_major ? 1u << 16 : 0) | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
// The whole warp goes through the issuing code, so that operands stay in uniform
// registers; `one` picks the thread that issues.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add, uint32_t one) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(desc), "r"((int)add), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add, uint32_t one) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(desc), "r"((int)add), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *m, uint32_t one) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_addr(m)), "r"(one)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(one));
  return one;
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define FKV_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define FKV_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 16 or 32 columns of the warp's 32 lanes.
__device__ __forceinline__ void tmem_load16(uint32_t (&r)[16], uint32_t at) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : FKV_R8(r, 0), FKV_R8(r, 8)
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
               FKV_W8(r, 0), FKV_W8(r, 8)
               : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t (&r)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : FKV_R8(r, 0), FKV_R8(r, 8), FKV_R8(r, 16), FKV_R8(r, 24)
      : "r"(at)
      : "memory");
}
// What was loaded may be used from here on: the registers go through the wait.
#define FKV_RW8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
__device__ __forceinline__ void tmem_wait_load(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : FKV_RW8(r, 0), FKV_RW8(r, 8) : : "memory");
}
__device__ __forceinline__ void tmem_wait_load(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : FKV_RW8(r, 0), FKV_RW8(r, 8), FKV_RW8(r, 16), FKV_RW8(r, 24)
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Block `at` of R rows, of at most `blocks`: its sequence and its place there.
// The last blocks of a sequence have most keys, so they come first; with up to
// 32 sequences the last of each come before the second last of any.
template <int R>
__device__ __forceinline__ bool find_block(const AttnArgs &a, int at, int blocks, int &b, int &rb) {
  const int lane = threadIdx.x & 31;
  if (a.num_seqs <= 32) {
    const int mine = lane < a.num_seqs ? item_of<R>(a, lane).blocks : 0;
    int lo = 0, hi = __reduce_max_sync(~0u, mine);  // the depth d with sum min(mine, d) <= at < that of d + 1
    if (at >= (int)__reduce_add_sync(~0u, mine)) return false;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int)__reduce_add_sync(~0u, min(mine, mid)) <= at)
        lo = mid;
      else
        hi = mid;
    }
    const int nth = at - (int)__reduce_add_sync(~0u, min(mine, lo));
    b = (int)__fns(__ballot_sync(~0u, mine > lo), 0, nth + 1);
    rb = __shfl_sync(~0u, mine, b) - 1 - lo;
    return true;
  }
  const int want = blocks - 1 - at;
  int64_t before = 0;
  for (int b0 = 0; b0 < a.num_seqs; b0 += 32) {
    const int mine = b0 + lane < a.num_seqs ? item_of<R>(a, b0 + lane).blocks : 0;
    int upto = mine;
#pragma unroll 1
    for (int i = 1; i < 32; i <<= 1) {
      const int o = __shfl_up_sync(~0u, upto, i);
      if (lane >= i) upto += o;
    }
    const uint32_t past = __ballot_sync(~0u, before + upto > want);
    if (past) {
      const int l = __ffs(past) - 1;
      b = b0 + l;
      rb = (int)(want - before) - __shfl_sync(~0u, upto - mine, l);
      return true;
    }
    before += __shfl_sync(~0u, upto, 31);
  }
  return false;
}

// A block's share of the workspace where the keys are split: its rows' O, then
// their RowSums.
template <int D>
__host__ __device__ constexpr int split_floats() { return kTiles * 128 * (D + 4); }

template <int D, bool BF16>
__global__ void __launch_bounds__(kManyThreads, 1)
fp4_many_kernel(const __grid_constant__ AttnArgs a, int blocks, int splits, float *__restrict__ parts) {
  constexpr int R = kTiles * 128;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  auto &sm = *reinterpret_cast<ManySmem<D> *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a block's heads, and the parts of its keys, run together
  const int h = blockIdx.x % a.kv_heads, of = blockIdx.x / a.kv_heads, at = of / splits, split = of - at * splits;
  after_previous();

  int b, rb;
  if (!find_block<R>(a, at, blocks, b, rb)) {  // the grid is an upper bound
    if (a.fill_rest) fill_rest(a, D, threadIdx.x, kManyThreads);
    return;
  }
  const Item it = item_of<R>(a, b);
  const int row0 = rb * R, nrows = it.rows * a.group;
  const int tiles = nrows - row0 > 128 ? 2 : 1;
  auto end_of = [&](int row) {  // the keys that a row sees
    int e = it.len;
    if (a.causal) e = max(min(e, it.len_q - it.rows + row / a.group + 1), 0);
    return e;
  };
  const int most = end_of(min(nrows - 1, row0 + R - 1));
  const int all = (most + kKeys - 1) / kKeys;
  const int chunk0 = (int)((int64_t)all * split / splits), chunks = (int)((int64_t)all * (split + 1) / splits) - chunk0;

  if (threadIdx.x == 0) {
    mbar_init(&sm.q_full, 128 * tiles);
    for (int i = 0; i < kRing; ++i) mbar_init(&sm.full[i], kFillWarps * 32), mbar_init(&sm.empty[i], tiles);
    for (int t = 0; t < kTiles; ++t) {
      for (int i = 0; i < 2; ++i) mbar_init(&sm.s_full[t][i], 1), mbar_init(&sm.p_full[t][i], 128);
      mbar_init(&sm.o_done[t], 1), mbar_init(&sm.all_done[t], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * kTiles + kFillWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sm.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sm.tmem;
  auto o_at = [&](int t) { return tmem + t * 128; };
  auto s_at = [&](int t, int i) { return tmem + (kTiles + t) * 128 + i * kKeys; };
  Patience patience;

  if (warp < 4 * tiles) {
    // ---- a thread for each row ----
    const int t = warp >> 2, r = (warp & 3) * 32 + lane, row = row0 + t * 128 + r;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // the warp's 32 lanes of tensor memory
    const bool valid = row < nrows;
    const int i0 = valid ? row / a.group : 0;
    float mul = 0;
    {
      const uint8_t *p = a.q + (it.first + i0) * a.q_token_stride + (h * a.group + row - i0 * a.group) * a.q_head_stride;
      float amax = 0;
      uint4 x[D / 8];
#pragma unroll
      for (int i = 0; i < D / 8; ++i) x[i] = valid ? reinterpret_cast<const uint4 *>(p)[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = pair_to_float2<BF16>(w[j]);
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      const float f = row_factor(amax), fs = a.scale < 0.0f ? -f : f;
      mul = row_mul(a.scale, f);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 z = pair_to_float2<BF16>(w[j]);
          y[j] = pack_half2(z.x * fs, z.y * fs);
        }
        *reinterpret_cast<uint4 *>(&sm.q[t][i / 8][r * 128 + ((i % 8) ^ (r & 7)) * 16]) = make_uint4(y[0], y[1], y[2], y[3]);
      }
      // an infinite query as in query_factor; a select there instead takes 717 us in place of 697 for three prompts
      if (amax > 3.4e38f) *reinterpret_cast<uint4 *>(&sm.q[t][0][r * 128 + (r & 7) * 16]) = make_uint4(~0u, ~0u, ~0u, ~0u);
    }
    fence_async();
    mbar_arrive(&sm.q_full);

    const int end = valid ? end_of(row) : 0;
    const int lowest = __reduce_min_sync(~0u, valid ? end : INT32_MAX);
    float centre = 0, bar = -INFINITY, l[4] = {0, 0, 0, 0};
    for (int j = 0; j < chunks; ++j) {
      patience.wait(&sm.s_full[t][j & 1], (j >> 1) & 1);
      fence_after();
      const uint32_t S = s_at(t, j & 1) + lanes;
      uint32_t x[2][32];
      tmem_load32(x[0], S), tmem_load32(x[1], S + 32);
      const uint32_t bad = *(volatile uint32_t *)sm.bad[j & (2 * kRing - 1)];
      tmem_wait_load(x[0]), tmem_wait_load(x[1]);
      const int key0 = (chunk0 + j) * kKeys;
      if (key0 + kKeys > lowest || bad) {  // only what the row sees
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (key0 + 32 * c + i >= end || ((bad >> (8 * (2 * c + i / 16))) & 1)) x[c][i] = 0xFF800000u;
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(x[c][i]));
      const float most_here = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if (__any_sync(~0u, most_here > bar)) {  // rare after the first chunks
        float f = 1.0f;
        if (most_here > bar) {  // other rows stay: a row does not depend on its neighbours
          f = fminf(moved(centre, most_here, mul), 1.0f);  // 1: a row without a key so far
          centre = most_here;
          bar = bar_of(centre, mul);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) l[i] *= f;
        if (j > 0) {
          patience.wait(&sm.o_done[t], (j - 1) & 1);
          fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t y[16];
            tmem_load16(y, o_at(t) + lanes + 16 * c);
            tmem_wait_load(y);
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
            tmem_store16(o_at(t) + lanes + 16 * c, y);
          }
        }
      }
      const uint64_t mul2 = pair(mul, mul), from2 = pair(-centre, -centre), lift2 = pair(kLift, kLift);
      uint64_t l01 = pair(l[0], l[1]), l23 = pair(l[2], l[3]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 y =
              unpair(fma2(add2(pair(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1])), from2), mul2, lift2));
          const float u = exp2_fast(y.x), v = exp2_fast(y.y);
          if (i & 1)
            l23 = add2(l23, pair(u, v));
          else
            l01 = add2(l01, pair(u, v));
          p[i] = pack_half2(u, v);
        }
        tmem_store16(S + 16 * c, p);
      }
      const float2 la = unpair(l01), lb = unpair(l23);
      l[0] = la.x, l[1] = la.y, l[2] = lb.x, l[3] = lb.y;
      tmem_wait_store();
      fence_before();
      mbar_arrive(&sm.p_full[t][j & 1]);
    }

    // O / l
    if (chunks) {
      patience.wait(&sm.all_done[t], 0);
      fence_after();
    }
    const int tok_head = h * a.group + row - i0 * a.group;
    const float sum = (l[0] + l[1]) + (l[2] + l[3]);
    if (splits > 1) {  // for the kernel below to join
      float *part = parts + (int64_t)blockIdx.x * split_floats<D>(), *o = part + (t * 128 + r) * D;
      if (chunks) {
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t x[16];
          tmem_load16(x, o_at(t) + lanes + 16 * c);
          tmem_wait_load(x);
#pragma unroll
          for (int i = 0; i < 4; ++i) reinterpret_cast<uint4 *>(o)[4 * c + i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        }
      }
      reinterpret_cast<RowSum *>(part + kTiles * 128 * D)[t * 128 + r] = {bar == -INFINITY ? -INFINITY : centre, sum, mul};
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      uint8_t *dst = a.out + (it.first + i0) * a.o_token_stride + tok_head * a.o_head_stride;
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        uint32_t x[16];
        if (chunks) {
          tmem_load16(x, o_at(t) + lanes + 16 * c);
          tmem_wait_load(x);
        }
        if (valid) {
          uint32_t y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float u = sum == 0.0f ? 0.0f : __uint_as_float(x[2 * k]) * inv;
            const float v = sum == 0.0f ? 0.0f : __uint_as_float(x[2 * k + 1]) * inv;
            if (BF16) {
              const __nv_bfloat162 z = __floats2bfloat162_rn(u, v);
              y[k] = *reinterpret_cast<const uint32_t *>(&z);
            } else {
              y[k] = pack_half2(u, v);
            }
          }
          reinterpret_cast<uint4 *>(dst)[2 * c] = make_uint4(y[0], y[1], y[2], y[3]);
          reinterpret_cast<uint4 *>(dst)[2 * c + 1] = make_uint4(y[4], y[5], y[6], y[7]);
        }
      }
      if (a.lse && valid) a.lse[(it.first + i0) * (a.kv_heads * a.group) + tok_head] = natural_lse({centre, sum, mul});
    }
  } else if (warp < 4 * kTiles + kFillWarps) {
    // ---- K and V into shared memory ----
    // Warp w brings unit w of a chunk, 8 tokens at a time, a quarter of a row a lane: 8 lanes that store together
    // have 8 rows, so the swizzle spreads them over all banks.
    // Where there is no second tile its warps take every second step: four warps alone need 1500 cycles for one,
    // more than a tile's scores, softmax and products (64 sequences of 4000 tokens, 64 rows: 313 us, so 232).
    const int w = warp & 3, tok = lane & 7, quarter = lane >> 3;
    const int by = 3 - tiles, first = warp < 4 * kTiles ? -1 : -2;
    constexpr int kWords = D / 32;  // of a lane's piece, 8 channels each
    const int at_row = tok * (D / 2) + quarter * (D / 8), at_scale = 8 * D + tok * (D / 16) + quarter * (D / 64);
    uint32_t at_chunk[kWords];  // a lane's pieces of a row in shared memory
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int c = quarter * kWords + k;
      at_chunk[k] = (c >> 3) * ManySmem<D>::kCols + w * 16 * 128 + tok * 128 + ((c & 7) ^ tok) * 16;
    }
    auto page_of = [&](int j) {
      const int u = (chunk0 + j) * (kKeys / 16) + w, e = divide(u, a.by_upb);
      return u * 16 < most && e < a.max_blocks ? a.tables[b * a.table_stride + e] : -1;
    };
    uint32_t x[2][2][kWords], sc[2][2];  // pieces of K and of V of a chunk, on their way
    const uint8_t *unit;                 // none: nothing is loaded and no scale taken
    int page;
    uint32_t bad = 0;
    auto find = [&](int j) {  // the unit of chunk j, and the page of the chunk after it
      const int u = (chunk0 + j) * (kKeys / 16) + w, e = divide(u, a.by_upb);
      const bool good = page >= 0 && page < a.num_blocks;
      unit = good ? a.layer + page * a.block_stride + ((int64_t)h * a.upb + u - e * a.upb) * (9 * D) : nullptr;
      bad = !good && u * 16 < most;
      page = page_of(j + by);
    };
    auto fetch = [&](int j, int side) {
      const uint8_t *p = unit + side * a.kv_stride;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sc[side][i] = 0;  // what no row sees may be anything: its scale counts as zero
#pragma unroll
        for (int k = 0; k < kWords; ++k) x[side][i][k] = 0;
        if (unit) {
          if constexpr (D == 128) {
            const uint4 y = __ldg(reinterpret_cast<const uint4 *>(p + at_row + i * 8 * (D / 2)));
            x[side][i][0] = y.x, x[side][i][1] = y.y, x[side][i][2] = y.z, x[side][i][3] = y.w;
          } else {
            const uint2 y = __ldg(reinterpret_cast<const uint2 *>(p + at_row + i * 8 * (D / 2)));
            x[side][i][0] = y.x, x[side][i][1] = y.y;
          }
          const uint8_t *q = p + at_scale + i * 8 * (D / 16);
          if ((chunk0 + j) * kKeys + w * 16 + i * 8 + tok < most)
            sc[side][i] = D == 128 ? __ldg(reinterpret_cast<const uint16_t *>(q)) : __ldg(q);
        }
      }
    };
    auto put = [&](uint32_t dst, int side) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t s[2] = {__byte_perm(sc[side][i], 0, 0x0404) >> 1, __byte_perm(sc[side][i], 0, 0x1414) >> 1};
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          uint32_t y[4];
          e2m1x8_to_half2(x[side][i][k], y);
#pragma unroll
          for (int m = 0; m < 4; ++m) y[m] = hmul2(y[m], s[D == 128 ? k >> 1 : 0]);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + at_chunk[k] + i * 8 * 128), "r"(y[0]), "r"(y[1]),
                       "r"(y[2]), "r"(y[3])
                       : "memory");
        }
      }
    };
    const uint32_t k_at = smem_addr(sm.k[0]), v_at = smem_addr(sm.v[0]);
    constexpr uint32_t kStage = D / 64 * ManySmem<D>::kCols;
    // Steps i from -2 on: K of chunk i + 2, then V of chunk i.  Their pieces are loaded a step of the warp's ahead.
    const uint8_t *units[3];  // of the chunks i, i + 1, i + 2
    page = page_of(first + 2);
    if (first + 2 < chunks) find(first + 2), fetch(first + 2, 0);
#pragma unroll 1
    for (int i = chunks ? first : 0; i < chunks; i += by) {
      const int slot = (i + 2) & (kRing - 1);
      if (i + 2 >= kRing) patience.wait(&sm.empty[slot], ((i + 2) / kRing + 1) & 1);
      units[0] = units[1], units[1] = units[2], units[2] = unit;
      if (i + 2 < chunks) {
        put(k_at + slot * kStage, 0);
        if (lane == 0) sm.bad[(i + 2) & (2 * kRing - 1)][w] = (uint8_t)bad;  // read before the chunk 2 kRing on gets here
        if (i + 2 + by < chunks) find(i + 2 + by), fetch(i + 2 + by, 0);
      }
      if (i >= 0) put(v_at + (i & (kRing - 1)) * kStage, 1);
      fence_async();
      mbar_arrive(&sm.full[slot]);
      if (i + by >= 0 && i + by < chunks) {
        const uint8_t *keep = unit;
        unit = by == 1 ? units[1] : units[2];
        fetch(i + by, 1);
        unit = keep;
      }
    }
    if (a.fill_rest && warp >= 4 * kTiles) fill_rest(a, D, threadIdx.x - 128 * kTiles, kFillWarps * 32);
  } else {
    // ---- the products: a warp for each tile ----
    // In loops and not straight code: these warps share their instruction caches with three busier ones each.  The
    // shuffles keep what addresses and trip counts come from in uniform registers, where the instructions want them.
    constexpr uint32_t kQK = mma_desc(kKeys, false), kPV = mma_desc(D, true);
    // of descriptors, in 16 bytes: a tile of Q and its blocks, a stage of K or V and its blocks
    constexpr uint32_t kRows16 = ManySmem<D>::kRows / 16, kCols16 = ManySmem<D>::kCols / 16, kBlocks = D / 64;
    const int t = __shfl_sync(~0u, warp, 0) - (4 * kTiles + kFillWarps);
    const int n = __shfl_sync(~0u, t < tiles ? chunks : 0, 0);  // none: no step at all
    const uint32_t one = elect_one(), o = __shfl_sync(~0u, tmem, 0) + t * 128, s = o + kTiles * 128;
    const uint64_t q_desc = smem_desc(smem_addr(sm.q), false) + t * kBlocks * kRows16,
                   k_desc = smem_desc(smem_addr(sm.k), false), v_desc = smem_desc(smem_addr(sm.v), true);
    auto score = [&](int j) {  // S of chunk j
      uint64_t q = q_desc, k = k_desc + (j & (kRing - 1)) * kBlocks * kCols16;
      const uint32_t d = s + (j & 1) * kKeys;
#pragma unroll 1
      for (int c = 0; c < kBlocks; ++c, q += kRows16, k += kCols16) {
        mma_ss(d, q, k, kQK, c > 0, one);
#pragma unroll
        for (int i = 1; i < 4; ++i) mma_ss(d, q + i * 2, k + i * 2, kQK, true, one);
      }
      mma_commit(&sm.s_full[t][j & 1], one);
    };
    auto filled = [&](int i) { patience.wait(&sm.full[(i + 2) & (kRing - 1)], ((i + 2) / kRing) & 1); };
    if (n) patience.wait(&sm.q_full, 0), filled(-2);
#pragma unroll 1
    for (int i = n ? -2 : 0; i < n; ++i) {
      if (i >= 0) {
        patience.wait(&sm.p_full[t][i & 1], (i >> 1) & 1);
        fence_after();
        const uint32_t p = s + (i & 1) * kKeys;
        const uint64_t v = v_desc + (i & (kRing - 1)) * kBlocks * kCols16;
        mma_ts(o, p, v, kPV, i > 0, one);
#pragma unroll
        for (int k = 1; k < kKeys / 16; ++k) mma_ts(o, p + k * 8, v + k * 128, kPV, true, one);
        mma_commit(&sm.o_done[t], one);
      }
      if (i + 2 < n) {  // two chunks ahead: its S goes where this chunk's P lies
        if (i >= 0) patience.wait(&sm.o_done[t], i & 1);
        fence_after();
        score(i + 2);
      }
      mma_commit(&sm.empty[(i + 2) & (kRing - 1)], one);
      if (i + 1 < n) filled(i + 1);
    }
    if (n) mma_commit(&sm.all_done[t], one);
  }

  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 4 * kTiles + kFillWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Joins the parts of the keys that the kernel above has split: a warp for each
// row, in the parts' order.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) fp4_merge_kernel(const __grid_constant__ AttnArgs a, int blocks, int splits,
                                                        const float *__restrict__ parts) {
  constexpr int R = kTiles * 128, kVec = D / 32;  // floats of a lane
  const int h = blockIdx.x % a.kv_heads, at = blockIdx.x / a.kv_heads, lane = threadIdx.x & 31;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5);
  after_previous();
  int b, rb;
  if (!find_block<R>(a, at, blocks, b, rb)) return;
  const Item it = item_of<R>(a, b);
  const int row = rb * R + r, nrows = it.rows * a.group;
  if (row >= nrows) return;
  RowSum all{kLowest, 0, 0};
  float acc[kVec] = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float *part = parts + ((int64_t)(at * splits + s) * a.kv_heads + h) * split_floats<D>();
    const RowSum of = reinterpret_cast<const RowSum *>(part + R * D)[r];
    float v[kVec] = {};
    if (of.l != 0.0f) {  // a part without keys has no sums
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = part[r * D + lane * kVec + i];
    }
    const float to = fmaxf(all.centre, of.centre), f = moved(all.centre, to, of.mul), y = moved(of.centre, to, of.mul);
    all = {to, all.l * f + of.l * y, of.mul};
#pragma unroll
    for (int i = 0; i < kVec; ++i) acc[i] = acc[i] * f + v[i] * y;
  }
  const int i0 = row / a.group, qh = h * a.group + row - i0 * a.group;
  const float inv = all.l == 0.0f ? 0.0f : 1.0f / all.l;
  uint8_t *dst = a.out + (it.first + i0) * a.o_token_stride + qh * a.o_head_stride + lane * kVec * 2;
#pragma unroll
  for (int i = 0; i < kVec; i += 2) {
    if (BF16)
      reinterpret_cast<__nv_bfloat162 *>(dst)[i / 2] = __floats2bfloat162_rn(acc[i] * inv, acc[i + 1] * inv);
    else
      reinterpret_cast<uint32_t *>(dst)[i / 2] = pack_half2(acc[i] * inv, acc[i + 1] * inv);
  }
  if (a.lse && lane == 0) a.lse[(it.first + i0) * (a.kv_heads * a.group) + qh] = natural_lse(all);
}

// A number of 48 bits for each launch, from a start that differs between processes.
unsigned long long next_call() {
  static std::atomic<unsigned long long> last{[] {
    std::random_device r;
    return ((unsigned long long)r() << 32) ^ r();
  }()};
  for (;;) {
    const unsigned long long n = (last.fetch_add(1, std::memory_order_relaxed) + 1) & 0xFFFFFFFFFFFFull;
    if (n) return n;  // 0 is what a finished launch leaves
  }
}

template <int D, int NT>
int64_t decode_workspace(int ctas) {
  return (int64_t)ctas * 2 * slot_floats<D>(8 * NT) * 4 + (int64_t)ctas * 3 * 8;
}
int64_t decode_workspace(int D, int nt, int ctas) {
  if (D == 128) return nt == 1 ? decode_workspace<128, 1>(ctas) : decode_workspace<128, 2>(ctas);
  return nt == 1 ? decode_workspace<64, 1>(ctas) : decode_workspace<64, 2>(ctas);
}

template <int D, int NT, bool BF16>
int launch_decode(const AttnArgs &a, int ctas, void *workspace, cudaStream_t s) {
  const int smem = sizeof(DecodeSmem<D, NT>);
  auto kernel = fp4_decode_kernel<D, NT, BF16>;
  FKV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  float *slots = (float *)workspace;
  auto *arrived = (unsigned long long *)(slots + (int64_t)ctas * 2 * slot_floats<D>(8 * NT));
  FKV_CUDA(launch_next(kernel, dim3(ctas), DecodeShape<D, NT>::kWarps * 32, smem, s, a, slots, arrived, next_call()));
  note_launch();
  return FKV_OK;
}
template <int D, bool BF16>
int launch_decode(const AttnArgs &a, int nt, int ctas, void *workspace, cudaStream_t s) {
  return nt == 1 ? launch_decode<D, 1, BF16>(a, ctas, workspace, s) : launch_decode<D, 2, BF16>(a, ctas, workspace, s);
}

// Launch of the many-rows kernel: a bound of the blocks of rows (the sequences'
// lengths are on the device), and how many CTAs share a block's keys.
struct ManyPlan {
  int64_t blocks;
  int splits;
};
ManyPlan many_plan(int64_t num_q, int group, int kv_heads, int num_seqs, int max_q_len, int sms) {
  constexpr int R = kTiles * 128;
  ManyPlan p{num_q * group / R + num_seqs, 1};
  // as many CTAs as there are SMs where the blocks, by the lengths as told, are fewer; wrong ones cost time only
  const int64_t told = std::min(p.blocks, (int64_t)num_seqs * (((int64_t)max_q_len * group + R - 1) / R)) * kv_heads;
  if (told > 0)
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({sms / told, 4 * sms / (p.blocks * kv_heads), 64}));
  return p;
}
int64_t many_workspace(int D, const ManyPlan &p, int kv_heads) {
  return p.splits == 1 ? 0 : p.blocks * p.splits * kv_heads * 4 * (D == 128 ? split_floats<128>() : split_floats<64>());
}

template <int D, bool BF16>
int launch_many(const AttnArgs &a, const ManyPlan &p, void *workspace, cudaStream_t s) {
  const int smem = sizeof(ManySmem<D>) + 1024;
  auto kernel = fp4_many_kernel<D, BF16>;
  FKV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (p.blocks * a.kv_heads * p.splits > INT32_MAX)
    return fail(FKV_ERR_INVALID_ARG, "fkv_fp4_attention: 2^31 blocks of rows or more");
  FKV_CUDA(launch_next(kernel, dim3((unsigned)(p.blocks * a.kv_heads * p.splits)), kManyThreads, smem, s, a, (int)p.blocks,
                       p.splits, (float *)workspace));
  note_launch();
  if (p.splits > 1) {
    FKV_CUDA(launch_next(fp4_merge_kernel<D, BF16>, dim3((unsigned)(p.blocks * a.kv_heads), kTiles * 128 / 8), 256, 0, s, a,
                         (int)p.blocks, p.splits, (const float *)workspace));
    note_launch();
  }
  return FKV_OK;
}

// Rows of a key head up to which the few-rows kernel runs, 16 at a time.  8 key
// heads, sequences of 4000 tokens, us there and in the many-rows kernel:
//   heads of 128   32 rows: 16 sequences 60 and 60, 64 sequences 175 and 233
//                  64 rows:              99 and 62,               326 and 235
//   heads of 64    32 rows:              43 and 53,               114 and 204
//                  64 rows:              66 and 53,               211 and 205
constexpr int kFewRows = 32;
int row_tiles(int64_t rows) { return rows <= 8 ? 1 : 2; }

}  // namespace
}  // namespace fkv

using namespace fkv;

extern "C" {

int fkv_fp4_wait_timeouts(int64_t *count) {
  clear_error();
  if (!count) return fail(FKV_ERR_INVALID_ARG, "fkv_fp4_wait_timeouts: null pointer");
  unsigned long long n = 0;
  FKV_CUDA(cudaDeviceSynchronize());  // the copy alone does not wait for streams that are not blocking
  FKV_CUDA(cudaMemcpyFromSymbol(&n, g_wait_timeouts, sizeof(n)));
  *count = (int64_t)n;
  return FKV_OK;
}

int64_t fkv_fp4_attention_workspace(int64_t num_q_tokens, int num_q_heads, int num_kv_heads, int head_size, int num_seqs,
                                    int max_q_len) {
  ThreadDeviceCtx *ctx;
  if (num_kv_heads <= 0 || get_ctx(-1, &ctx) != FKV_OK) return 0;
  const int group = num_q_heads / num_kv_heads;
  if ((int64_t)max_q_len * group > kFewRows)
    return many_workspace(head_size, many_plan(num_q_tokens, group, num_kv_heads, num_seqs, max_q_len, ctx->num_sms), num_kv_heads);
  return decode_workspace(head_size, row_tiles((int64_t)max_q_len * (num_q_heads / num_kv_heads)), ctx->num_sms);
}

int fkv_fp4_attention(const void *layer, int64_t num_blocks, int tokens_per_block, int num_kv_heads, int head_size,
                      int64_t kv_stride_in_bytes, int64_t block_stride_in_bytes, const void *q, void *out, float *lse,
                      int64_t q_token_stride_in_bytes, int64_t q_head_stride_in_bytes, int64_t out_token_stride_in_bytes,
                      int64_t out_head_stride_in_bytes, int dtype, int64_t num_q_tokens, int num_q_heads,
                      const int32_t *block_tables, int64_t block_table_stride, int max_blocks, const int32_t *seq_lens,
                      const int32_t *cu_seqlens_q, int num_seqs, int max_q_len, float softmax_scale, int flags,
                      void *workspace, int64_t workspace_bytes, void *stream) {
  clear_error();
  const char *w = "fkv_fp4_attention: ";
  auto bad = [&](const char *m) { return fail(FKV_ERR_INVALID_ARG, std::string(w) + m); };
  if (tokens_per_block <= 0 || tokens_per_block % 16) return bad("tokens_per_block must be a positive multiple of 16");
  if (tokens_per_block > 65536) return bad("tokens_per_block must be at most 65536");
  if (head_size != 64 && head_size != 128)
    return fail(FKV_ERR_UNSUPPORTED, std::string(w) + "head_size must be 64 or 128");
  if (dtype != FKV_DTYPE_BF16 && dtype != FKV_DTYPE_FP16)
    return fail(FKV_ERR_UNSUPPORTED, std::string(w) + "queries must be bfloat16 or half");
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads)
    return bad("the query heads must be a multiple of the key heads");
  if (num_blocks < 0 || num_q_tokens < 0 || num_seqs < 0 || max_blocks < 0) return bad("counts must be non-negative");
  if (!std::isfinite(softmax_scale)) return bad("softmax_scale must be finite");
  if (flags & ~(FKV_FP4_CAUSAL | FKV_FP4_FILL_REST)) return bad("unknown flags");
  if (num_q_tokens == 0 || num_seqs == 0) return FKV_OK;
  if (num_q_tokens > INT32_MAX || num_q_tokens * num_q_heads >= INT32_MAX - 65536)
    return bad("2^31 (token, head) rows or more in one call");
  if (!q || !out || !seq_lens || (max_blocks > 0 && !block_tables) || (num_blocks > 0 && !layer)) return bad("null pointer");
  if (!cu_seqlens_q && num_q_tokens % num_seqs) return bad("without cu_seqlens_q every sequence has the same number of new tokens");
  if ((uintptr_t)layer % 16 || kv_stride_in_bytes % 16 || block_stride_in_bytes % 16 || (uintptr_t)q % 16 ||
      (uintptr_t)out % 16 || q_token_stride_in_bytes % 16 || q_head_stride_in_bytes % 16 || out_token_stride_in_bytes % 16 ||
      out_head_stride_in_bytes % 16)
    return fail(FKV_ERR_MISALIGNED, std::string(w) + "the layer and the rows of q and out must start on 16-byte boundaries");
  AttnArgs a{};
  a.layer = (const uint8_t *)layer, a.num_blocks = num_blocks, a.kv_stride = kv_stride_in_bytes;
  a.block_stride = block_stride_in_bytes, a.tokens_per_block = tokens_per_block, a.kv_heads = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.upb = tokens_per_block / 16, a.by_upb = divisor_of(a.upb);
  a.q = (const uint8_t *)q, a.q_token_stride = q_token_stride_in_bytes, a.q_head_stride = q_head_stride_in_bytes;
  a.out = (uint8_t *)out, a.o_token_stride = out_token_stride_in_bytes, a.o_head_stride = out_head_stride_in_bytes;
  a.lse = lse, a.num_q = num_q_tokens, a.tables = block_tables, a.table_stride = block_table_stride;
  a.max_blocks = max_blocks, a.seq_lens = seq_lens, a.cu = cu_seqlens_q, a.num_seqs = num_seqs;
  a.scale = softmax_scale, a.causal = flags & FKV_FP4_CAUSAL;
  a.fill_rest = cu_seqlens_q && (flags & FKV_FP4_FILL_REST);
  a.rows_each = (int)(num_q_tokens / num_seqs);
  a.table_tokens = (int)std::min<int64_t>((int64_t)max_blocks * tokens_per_block, INT32_MAX - 255);  // positions are ints
  ThreadDeviceCtx *ctx;
  const int rc = get_ctx(-1, &ctx);
  if (rc != FKV_OK) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const bool bf16 = dtype == FKV_DTYPE_BF16;
  if ((int64_t)max_q_len * a.group > kFewRows) {
    const ManyPlan p = many_plan(num_q_tokens, a.group, num_kv_heads, num_seqs, max_q_len, ctx->num_sms);
    const int64_t need = many_workspace(head_size, p, num_kv_heads);
    if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
      return bad("the workspace is too small or not aligned");
    if (head_size == 128) return bf16 ? launch_many<128, true>(a, p, workspace, s) : launch_many<128, false>(a, p, workspace, s);
    return bf16 ? launch_many<64, true>(a, p, workspace, s) : launch_many<64, false>(a, p, workspace, s);
  }
  const int nt = row_tiles((int64_t)max_q_len * a.group);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < decode_workspace(head_size, nt, ctx->num_sms))
    return bad("the workspace is too small or not aligned");
  if (head_size == 128)
    return bf16 ? launch_decode<128, true>(a, nt, ctx->num_sms, workspace, s) : launch_decode<128, false>(a, nt, ctx->num_sms, workspace, s);
  return bf16 ? launch_decode<64, true>(a, nt, ctx->num_sms, workspace, s) : launch_decode<64, false>(a, nt, ctx->num_sms, workspace, s);
}

}  // extern "C"
