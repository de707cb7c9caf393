// Attention over the 4-bit paged cache (format: fp4_cache.cu).
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j   over the keys row i sees
//
// Row i of sequence b sits at position len_b - qlen_b + i and sees the keys
// up to its own position (causal) or all len_b.  Query head h reads key head
// h / (q_heads / kv_heads).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "fkv_common.h"
#include "fp4_format.cuh"

namespace fkv {
namespace {

struct AttnArgs {
  const uint8_t *layer;
  int64_t num_blocks, kv_stride, block_stride;
  int tokens_per_block, kv_heads, group;
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
  const int32_t *cu;  // null: num_q / num_seqs rows each
  int num_seqs;
  float scale;
  int causal;
};

__device__ __forceinline__ float natural_lse(float m, float l) {  // m: in powers of two
  return l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
}

// Four channels from c on of (token, head) row `row` of a sequence.
template <bool BF16>
__device__ __forceinline__ void store_row(const AttnArgs &a, int64_t first, int h, int64_t row, int64_t nrows, int c, float4 v,
                                          float m, float l) {
  if (row >= nrows) return;
  const int64_t tok = first + row / a.group;
  const int qh = h * a.group + (int)(row % a.group);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint2 w;
  if (BF16) {
    __nv_bfloat162 x = __floats2bfloat162_rn(v.x * inv, v.y * inv), y = __floats2bfloat162_rn(v.z * inv, v.w * inv);
    w.x = *reinterpret_cast<uint32_t *>(&x), w.y = *reinterpret_cast<uint32_t *>(&y);
  } else {
    __half2 x = __floats2half2_rn(v.x * inv, v.y * inv), y = __floats2half2_rn(v.z * inv, v.w * inv);
    w.x = *reinterpret_cast<uint32_t *>(&x), w.y = *reinterpret_cast<uint32_t *>(&y);
  }
  *reinterpret_cast<uint2 *>(a.out + tok * a.o_token_stride + qh * a.o_head_stride + 2 * c) = w;
  if (a.lse && c == 0) a.lse[tok * (a.kv_heads * a.group) + qh] = natural_lse(m, l);
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
// line of work that is cut into equal pieces, one for each CTA, whatever the
// lengths are; they are read on the device, so a captured launch follows them.
// Within a CTA every warp has its own ring of bulk copies, takes chunks of up
// to kUps units in turn and keeps its own running maximum, sum and O; they are
// joined once for each (sequence, head), and pieces of one (sequence, head) in
// several CTAs by a second small kernel, in a fixed order.

constexpr int kWarps = 8;
constexpr int kUps = 2;     // units of a chunk
constexpr int kStages = 4;  // chunks of a warp's ring
constexpr float kNone = -1e30f;  // a row's base before any key
// A weight is 2^(score - base).  The base is set 7 below the largest score and
// moves when one passes it by 15: the largest weight of a row lies between
// 2^7 and 2^15, so its rounding to half (a step of 2^-24 at the least) takes
// at most 2^-32 of the sum of weights from any weight, however small.
constexpr float kLift = 7.0f, kMove = 15.0f;

struct Item {  // what a CTA needs of one sequence
  int64_t len;      // tokens that can be seen: the table's end at most
  int64_t len_q;    // tokens as given: positions count from here
  int64_t first;    // first row in q
  int rows;         // new tokens
  int blocks;       // blocks of R (token, head) rows
  int64_t units;    // units to pass, at least one where there are rows
};

template <int R>
__device__ __forceinline__ Item item_of(const AttnArgs &a, int b) {
  Item it;
  if (a.cu) {
    const int64_t lo = min((int64_t)max(a.cu[b], 0), a.num_q), hi = min((int64_t)max(a.cu[b + 1], 0), a.num_q);
    it.first = lo, it.rows = (int)max(hi - lo, (int64_t)0);
  } else {
    it.rows = (int)(a.num_q / a.num_seqs);
    it.first = (int64_t)b * it.rows;
  }
  it.len_q = a.seq_lens[b];
  it.len = min(max(it.len_q, (int64_t)0), (int64_t)a.max_blocks * a.tokens_per_block);
  it.blocks = (int)(((int64_t)it.rows * a.group + R - 1) / R);
  it.units = it.rows ? max((it.len + 15) / 16, (int64_t)1) : 0;
  return it;
}

// Where a CTA's piece starts, found by every CTA for itself.
struct Start {
  int64_t total;   // units of all work
  int64_t begin, end;
  int ctas;
  int b;           // sequence of `begin`
  int64_t before;  // units before sequence b
};

template <int R>
__device__ void find_start(const AttnArgs &a, int ctas, Start *out, int64_t *scratch /* kWarps */) {
  const int per = (a.num_seqs + kWarps * 32 - 1) / (kWarps * 32);
  const int b0 = min(threadIdx.x * per, a.num_seqs), b1 = min(b0 + per, a.num_seqs);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Item it = item_of<R>(a, b);
    mine += it.units * it.blocks * a.kv_heads;
  }
  int64_t upto = mine;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const int64_t o = __shfl_up_sync(~0u, upto, i);
    if ((threadIdx.x & 31) >= i) upto += o;
  }
  if ((threadIdx.x & 31) == 31) scratch[threadIdx.x >> 5] = upto;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < (threadIdx.x >> 5)) upto += scratch[w];
    total += scratch[w];
  }
  const int64_t want = (total + kWarps - 1) / kWarps;  // a unit for each warp, at least
  const int n = (int)(want < ctas ? want : ctas);
  const int64_t begin = blockIdx.x < n ? blockIdx.x * total / n : total;
  const int64_t end = blockIdx.x < n ? (blockIdx.x + 1) * total / n : total;
  if (threadIdx.x == 0) out->total = total, out->begin = begin, out->end = end, out->ctas = n;
  int64_t at = upto - mine;
  if (begin >= at && begin < upto) {
    for (int b = b0; b < b1; ++b) {
      const Item it = item_of<R>(a, b);
      const int64_t w = it.units * it.blocks * a.kv_heads;
      if (begin < at + w) {
        out->b = b, out->before = at;
        break;
      }
      at += w;
    }
  }
  __syncthreads();
}

// A walk over a CTA's piece: segments (the part of one (sequence, head, row
// block) in it), and a warp's chunks in them.
template <int R>
struct Walk {
  int64_t left;      // units of the piece from u0 on
  int b, idx;        // sequence; (head, row block) in it
  Item it;
  int64_t u0, u1;    // units of the segment
  int64_t at;        // this warp's next chunk
  int step;          // units of a chunk

  __device__ void start(const AttnArgs &a, const Start &s, int warp) {
    left = s.end - s.begin;
    if (left <= 0) return;
    b = s.b;
    it = item_of<R>(a, b);
    const int64_t off = s.begin - s.before;
    idx = (int)(off / it.units);
    u0 = off - (int64_t)idx * it.units;
    open(warp);
  }
  __device__ void open(int warp) {
    u1 = min(it.units, u0 + left);
    const int64_t share = (u1 - u0 + kWarps - 1) / kWarps;
    step = (int)min(share, (int64_t)kUps);
    at = u0 + (int64_t)warp * step;
  }
  // To the next segment; false at the end of the piece.
  __device__ bool next_segment(const AttnArgs &a, int warp) {
    left -= u1 - u0;
    if (left <= 0) return false;
    u0 = 0;
    if (++idx == it.blocks * a.kv_heads) {
      idx = 0;
      do it = item_of<R>(a, ++b);
      while (it.units * it.blocks == 0);  // there is work left, so this ends
    }
    open(warp);
    return true;
  }
  __device__ void next_chunk() { at += kWarps * step; }
  __device__ bool has_chunk() const { return at < u1; }
  __device__ int chunk_units() const { return (int)min((int64_t)step, u1 - at); }
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t *m, int count) {
  asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(smem_addr(m)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t *m, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(smem_addr(m)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t *m, int parity) {
  int ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared.b64 p, [%1], %2, %3;\n selp.b32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_addr(m)), "r"(parity), "r"(1000000)
      : "memory");
  return ok;
}
__device__ __forceinline__ void bulk_load(void *dst, const void *src, int bytes, uint64_t *m) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_addr(dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(m))
               : "memory");
}
// Waits with a limit (a try waits up to a millisecond by itself): one that
// runs out is counted, and the data is taken as it is.
__device__ unsigned long long g_wait_timeouts;
__device__ __forceinline__ bool mbar_wait(uint64_t *m, int parity, int tries) {
  for (int i = 0; i < tries; ++i)
    if (mbar_try(m, parity)) return true;
  if ((threadIdx.x & 31) == 0) atomicAdd(&g_wait_timeouts, 1ull);
  return false;
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

// The power of two that brings a row's largest value to [2^10, 2^11), within
// what a float holds; its inverse is exact too.
__device__ __forceinline__ float row_factor(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23) - 127;
  int k = 10 - e;
  k = k > 126 ? 126 : k;
  k = (amax > 0.0f && amax <= 3.4e38f) ? k : 0;
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

struct SplitMeta {  // of a CTA: the (sequence, head, row block) that starts in it and ends in another
  int last;         // the CTA it ends in; -1: none
  int b, idx;
};

template <int D, int NT>
struct DecodeSmem {
  static constexpr int kUnit = 9 * D;
  static constexpr int kPad = D + 4;  // floats of a row in the join: quads store 16-byte pieces of rows 2 t and 2 t + 1
  alignas(128) uint8_t ring[kWarps][kStages][kUps][2][kUnit];
  alignas(16) float o[kWarps][8][kPad];
  float m[kWarps][8 * NT], l[kWarps][8 * NT];
  uint64_t full[kWarps][kStages];
  Start start;
  int64_t scratch[kWarps];
};

template <int D>
__host__ __device__ constexpr int slot_floats(int rows) { return rows * (D + 2); }

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(kWarps * 32, 1)
fp4_decode_kernel(const __grid_constant__ AttnArgs a, float *__restrict__ parts, SplitMeta *__restrict__ meta) {
  constexpr int R = 8 * NT, KS = D / 16, KW = D / 32, VB = D / 16;  // k-steps; words of a lane's K row; bytes of its V row
  extern __shared__ uint8_t smem_raw[];
  auto &sm = *reinterpret_cast<DecodeSmem<D, NT> *>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // the next kernel only starts its CTAs early; it waits for this one's end before it reads
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&sm.full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  find_start<R>(a, gridDim.x, &sm.start, sm.scratch);
  const Start st = sm.start;
  if (threadIdx.x == 0) meta[blockIdx.x].last = -1;
  if (st.begin >= st.end) return;

  Walk<R> in, cur;  // the copies' walk runs ahead
  in.start(a, st, warp);
  cur = in;
  bool more = true;
  int64_t page = -1;
  const int units_per_block = a.tokens_per_block / 16;
  auto settle = [&] {  // to a segment with a chunk for this warp, and on to its pages
    while (more && !in.has_chunk()) more = in.next_segment(a, warp);
    if (more && lane < 2 * in.chunk_units()) {
      const int64_t u = in.at + (lane >> 1), e = u / units_per_block;
      page = e < a.max_blocks ? a.tables[in.b * a.table_stride + e] : -1;
    }
  };
  uint32_t valid = 0;  // bit kUps * stage + unit: the unit's page is in the pool and its copy was started
  int alive = 1000;    // tries of a wait; after one ran out, a single one
  auto issue = [&](int stage) {
    const int n = more ? in.chunk_units() : 0;
    if (n == 0) return;
    const bool good = lane < 2 * n && page >= 0 && page < a.num_blocks;
    const uint32_t ok = __ballot_sync(~0u, good);
    uint32_t mask = 0;
#pragma unroll
    for (int u = 0; u < kUps; ++u) mask |= ((ok >> (2 * u)) & 1) << u;
    valid = (valid & ~(((1u << kUps) - 1) << (kUps * stage))) | (mask << (kUps * stage));
    if (lane == 0) mbar_expect(&sm.full[warp][stage], __popc(ok) * 9 * D);
    __syncwarp();
    if (good) {
      const int64_t u = in.at + (lane >> 1);
      const int h = in.idx / in.it.blocks;
      const uint8_t *src = a.layer + (lane & 1) * a.kv_stride + page * a.block_stride +
                           ((int64_t)h * units_per_block + u % units_per_block) * (9 * D);
      bulk_load(sm.ring[warp][stage][lane >> 1][lane & 1], src, 9 * D, &sm.full[warp][stage]);
    }
    in.next_chunk();
    settle();
  };
  settle();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s);
  int stage = 0, phase = 0;

  for (;;) {  // segments
    const int h = cur.idx / cur.it.blocks, rb = cur.idx % cur.it.blocks;
    const int64_t row0 = (int64_t)rb * R;  // of the sequence's (token, head) rows
    const int64_t nrows = (int64_t)cur.it.rows * a.group;
    // queries, n = g, channels D / 4 * t on; multiplier and end of the rows 2 t, 2 t + 1
    uint32_t qf[NT][KS][2];
    float mul[NT][2];
    int64_t end[NT][2], lowest = INT64_MAX, highest = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int64_t r = row0 + n * 8 + g;
      float x[D / 4];
      float amax = 0;
      if (r < nrows) {
        const uint8_t *p = a.q + (cur.it.first + r / a.group) * a.q_token_stride +
                           (h * a.group + r % a.group) * a.q_head_stride + t * (D / 2);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = pair_to_float2<BF16>(w[j]);
            x[8 * i + 2 * j] = f.x, x[8 * i + 2 * j + 1] = f.y;
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 4; ++i) x[i] = 0;
      }
      amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
      const float f = row_factor(amax);
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) qf[n][k][j] = pack_half2(x[4 * k + 2 * j] * f, x[4 * k + 2 * j + 1] * f);
      const float mine = a.scale * 1.4426950408889634f * (1.0f / f);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mul[n][j] = __shfl_sync(~0u, mine, (2 * t + j) * 4);
        const int64_t rr = row0 + n * 8 + 2 * t + j;
        int64_t e = 0;
        if (rr < nrows) e = a.causal ? min(cur.it.len, cur.it.len_q - cur.it.rows + rr / a.group + 1) : cur.it.len;
        end[n][j] = e;
        if (rr < nrows) lowest = min(lowest, e);
        highest = max(highest, e);
      }
    }
#pragma unroll
    for (int i = 1; i < 4; i <<= 1) {
      lowest = min(lowest, __shfl_xor_sync(~0u, lowest, i));
      highest = max(highest, __shfl_xor_sync(~0u, highest, i));
    }

    float o[NT][KS][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][k][i] = 0;
      m[n][0] = m[n][1] = kNone;
      l[n][0] = l[n][1] = 0;
    }

    for (; cur.has_chunk(); cur.next_chunk()) {
      const uint32_t ok = (valid >> (kUps * stage)) & ((1u << kUps) - 1);
      if (!mbar_wait(&sm.full[warp][stage], phase, alive)) alive = 1;
      __syncwarp();  // and every lane is done with the chunk before, whose slot is the next to fill
      issue((stage + kStages - 1) % kStages);
      float s[kUps][NT][4];
      // S^T: rows g, g + 8 are tokens tok, tok + 8
      const int tok = (g & 1) ? ((g >> 1) ^ 1) + 4 : (g >> 1);
#pragma unroll
      for (int u = 0; u < kUps; ++u) {
        const uint8_t *K = sm.ring[warp][stage][u][0];
        uint32_t w[2][KW], sc[2][(D + 127) / 128 * 2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint8_t *row = K + (tok + 8 * i) * (D / 2) + t * (D / 8);
          if constexpr (D == 128) {
            const uint4 v = *reinterpret_cast<const uint4 *>(row);
            w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
            const uint32_t c = *reinterpret_cast<const uint16_t *>(K + 8 * D + (tok + 8 * i) * (D / 16) + 2 * t);
            sc[i][0] = __byte_perm(c, 0, 0x0404) >> 1;
            sc[i][1] = __byte_perm(c, 0, 0x1414) >> 1;
          } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(row);
            w[i][0] = v.x, w[i][1] = v.y;
            const uint32_t c = K[8 * D + (tok + 8 * i) * (D / 16) + t];
            sc[i][0] = __byte_perm(c, 0, 0x0404) >> 1;
          }
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
      }
      // scores in powers of two; hidden ones to -inf
      bool hide[kUps];
      bool grow = false;
#pragma unroll
      for (int u = 0; u < kUps; ++u) {
        const int64_t base = (cur.at + u) * 16;
        hide[u] = !((ok >> u) & 1) || base + 16 > lowest;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][n][i] *= mul[n][i & 1];
        if (hide[u]) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int64_t j = base + tok + 8 * (i >> 1);
              if (!((ok >> u) & 1) || j >= end[n][i & 1]) s[u][n][i] = -INFINITY;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) grow |= s[u][n][i] > m[n][i & 1] + kMove;
      }
      if (__any_sync(~0u, grow)) {  // rare after the first chunks
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float x = kNone;
#pragma unroll
            for (int u = 0; u < kUps; ++u) x = fmaxf(x, fmaxf(s[u][n][j], s[u][n][j + 2]));
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, i));
            const float to = x > m[n][j] + kMove ? x - kLift : m[n][j];  // others stay: a row does not depend on its neighbours
            const float f = exp2_fast(m[n][j] - to);
            m[n][j] = to;
            l[n][j] *= f;
#pragma unroll
            for (int k = 0; k < KS; ++k) o[n][k][j] *= f, o[n][k][j + 2] *= f;
          }
      }
#pragma unroll
      for (int u = 0; u < kUps; ++u) {
        uint32_t p[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float x = exp2_fast(s[u][n][2 * i] - m[n][0]), y = exp2_fast(s[u][n][2 * i + 1] - m[n][1]);
            l[n][0] += x, l[n][1] += y;
            p[n][i] = transpose8(pack_half2(x, y));
          }
        // V^T: lane g takes channels D / 8 * g on, of the tokens of rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9
        const uint8_t *V = sm.ring[warp][stage][u][1];
        const int tk[2] = {t, (t ^ 1) + 4};
        uint32_t w[4][VB / 4], sc[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t c[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int tt = tk[j] + 8 * i;
            if constexpr (D == 128) {
              const uint2 v = *reinterpret_cast<const uint2 *>(V + tt * (D / 2) + g * VB);
              w[2 * i + j][0] = v.x, w[2 * i + j][1] = v.y;
            } else {
              w[2 * i + j][0] = *reinterpret_cast<const uint32_t *>(V + tt * (D / 2) + g * VB);
            }
            c[j] = V[8 * D + tt * (D / 16) + g * D / 128];
            // what no row sees may be anything: its scale counts as zero
            if (hide[u] && (!((ok >> u) & 1) || (cur.at + u) * 16 + tt >= highest)) c[j] = 0;
          }
          sc[i] = (c[0] << 7) | (c[1] << 23);
        }
#pragma unroll
        for (int j = 0; j < VB / 4; ++j) {
          uint32_t x[2][2][4];  // token pair, channel parity, channel pair
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w0 = w[2 * i][j], w1 = w[2 * i + 1][j];
            e2m1x8_to_half2((w0 & 0x0F0F0F0Fu) | ((w1 << 4) & 0xF0F0F0F0u), x[i][0]);
            e2m1x8_to_half2(((w0 >> 4) & 0x0F0F0F0Fu) | (w1 & 0xF0F0F0F0u), x[i][1]);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i][0][k] = hmul2(x[i][0][k], sc[i]), x[i][1][k] = hmul2(x[i][1][k], sc[i]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t f[4] = {x[0][0][k], x[0][1][k], x[1][0][k], x[1][1][k]};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma(o[n][4 * j + k], f, p[n][0], p[n][1]);
          }
        }
      }
      if (++stage == kStages) stage = 0, phase ^= 1;
    }

    // join the warps' parts: row r of the block, channel c
    const bool starts = cur.u0 == 0, ends = cur.u1 == cur.it.units;
    float *slot = parts + (int64_t)(2 * blockIdx.x + (starts ? 1 : 0)) * slot_floats<D>(R);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 4; i < 32; i <<= 1) l[n][j] += __shfl_xor_sync(~0u, l[n][j], i);
#pragma unroll
        for (int k = 0; k < KS; k += 2)
          *reinterpret_cast<float4 *>(&sm.o[warp][2 * t + j][g * (D / 8) + 2 * k]) =
              make_float4(o[n][k][j], o[n][k][j + 2], o[n][k + 1][j], o[n][k + 1][j + 2]);
        if (g == 0) sm.m[warp][n * 8 + 2 * t + j] = m[n][j], sm.l[warp][n * 8 + 2 * t + j] = l[n][j];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 8 * (D / 4); i += kWarps * 32) {
        const int r = i / (D / 4), c = i % (D / 4) * 4, rr = n * 8 + r;
        float M = kNone, L = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.m[w][rr]);
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = exp2_fast(sm.m[w][rr] - M);
          const float4 v = *reinterpret_cast<const float4 *>(&sm.o[w][r][c]);
          L += sm.l[w][rr] * f;
          acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
        }
        if (starts && ends) {
          store_row<BF16>(a, cur.it.first, h, row0 + rr, nrows, c, acc, M, L);
        } else {
          *reinterpret_cast<float4 *>(slot + rr * D + c) = acc;
          if (c == 0) slot[R * D + 2 * rr] = M, slot[R * D + 2 * rr + 1] = L;
        }
      }
      __syncthreads();
    }
    if (starts && !ends && threadIdx.x == 0) {
      // the global index of the item's last unit gives the CTA that holds it
      const int64_t x = st.end - (cur.u1 - cur.u0) + cur.it.units - 1;
      meta[blockIdx.x].b = cur.b;
      meta[blockIdx.x].idx = cur.idx;
      meta[blockIdx.x].last = (int)(((x + 1) * st.ctas - 1) / st.total);
    }
    if (!cur.next_segment(a, warp)) break;
  }
}

// Joins the pieces of the (sequence, head, row block) that starts in CTA
// blockIdx.x of the kernel above, for row blockIdx.y of it.
template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(D) fp4_join_kernel(const __grid_constant__ AttnArgs a, const float *__restrict__ parts,
                                                     const SplitMeta *__restrict__ meta) {
  constexpr int R = 8 * NT, kMost = 1024;
  __shared__ float w[kMost];
  __shared__ float red[2][D / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x, r = blockIdx.y, last = meta[c].last;
  if (last < 0) return;
  const int n = last - c + 1;
  auto slot = [&](int i) { return parts + (int64_t)(2 * (c + i) + (i == 0 ? 1 : 0)) * slot_floats<D>(R); };
  float M = kNone;
  for (int i = threadIdx.x; i < n; i += D) M = fmaxf(M, slot(i)[R * D + 2 * r]);
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, i));
  if ((threadIdx.x & 31) == 0) red[0][threadIdx.x >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < D / 32; ++i) M = fmaxf(M, red[0][i]);
  float L = 0;
  for (int i = threadIdx.x; i < n; i += D) {
    const float f = exp2_fast(slot(i)[R * D + 2 * r] - M);
    w[i] = f;
    L += slot(i)[R * D + 2 * r + 1] * f;
  }
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) L += __shfl_xor_sync(~0u, L, i);
  if ((threadIdx.x & 31) == 0) red[1][threadIdx.x >> 5] = L;
  __syncthreads();
  L = 0;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) L += red[1][i];
  float acc = 0;
#pragma unroll 8
  for (int i = 0; i < n; ++i) acc += slot(i)[r * D + threadIdx.x] * w[i];
  const Item it = item_of<R>(a, meta[c].b);
  const int h = meta[c].idx / it.blocks, rb = meta[c].idx % it.blocks;
  const int64_t row = (int64_t)rb * R + r;
  if (row >= (int64_t)it.rows * a.group) return;
  const int64_t tok = it.first + row / a.group;
  const int qh = h * a.group + (int)(row % a.group);
  uint8_t *dst = a.out + tok * a.o_token_stride + qh * a.o_head_stride + threadIdx.x * 2;
  const float v = acc * (L == 0 ? 0.0f : 1.0f / L);
  if (BF16)
    *reinterpret_cast<__nv_bfloat16 *>(dst) = __float2bfloat16_rn(v);
  else
    *reinterpret_cast<__half *>(dst) = __float2half_rn(v);
  if (a.lse && threadIdx.x == 0) a.lse[tok * (a.kv_heads * a.group) + qh] = natural_lse(M, L);
}

template <int D, int NT>
int64_t decode_workspace(int ctas) {
  return (int64_t)ctas * 2 * slot_floats<D>(8 * NT) * 4 + (int64_t)ctas * sizeof(SplitMeta);
}
int64_t decode_workspace(int D, int nt, int ctas) {
  return D == 128 ? (nt == 1 ? decode_workspace<128, 1>(ctas) : nt == 2 ? decode_workspace<128, 2>(ctas) : decode_workspace<128, 4>(ctas))
                  : (nt == 1 ? decode_workspace<64, 1>(ctas) : nt == 2 ? decode_workspace<64, 2>(ctas) : decode_workspace<64, 4>(ctas));
}

template <int D, int NT, bool BF16>
int launch_decode(const AttnArgs &a, int ctas, void *workspace, cudaStream_t s) {
  const int smem = sizeof(DecodeSmem<D, NT>);
  auto kernel = fp4_decode_kernel<D, NT, BF16>;
  FKV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  float *parts = (float *)workspace;
  SplitMeta *meta = (SplitMeta *)(parts + (int64_t)ctas * 2 * slot_floats<D>(8 * NT));
  kernel<<<ctas, kWarps * 32, smem, s>>>(a, parts, meta);
  FKV_CUDA(cudaGetLastError());
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas, 8 * NT), cfg.blockDim = dim3(D), cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at, cfg.numAttrs = 1;
  FKV_CUDA(cudaLaunchKernelEx(&cfg, fp4_join_kernel<D, NT, BF16>, a, (const float *)parts, (const SplitMeta *)meta));
  note_launch(2);
  return FKV_OK;
}
template <int D, bool BF16>
int launch_decode(const AttnArgs &a, int nt, int ctas, void *workspace, cudaStream_t s) {
  switch (nt) {
    case 1: return launch_decode<D, 1, BF16>(a, ctas, workspace, s);
    case 2: return launch_decode<D, 2, BF16>(a, ctas, workspace, s);
    default: return launch_decode<D, 4, BF16>(a, ctas, workspace, s);
  }
}

// Tiles of 8 rows that go through the cache together.
int row_tiles(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

}  // namespace
}  // namespace fkv

using namespace fkv;

extern "C" {

int64_t fkv_fp4_attention_workspace(int64_t num_q_tokens, int num_q_heads, int num_kv_heads, int head_size, int num_seqs,
                                    int max_q_len) {
  ThreadDeviceCtx *ctx;
  if (num_kv_heads <= 0 || get_ctx(-1, &ctx) != FKV_OK) return 0;
  return decode_workspace(head_size, row_tiles((int64_t)max_q_len * (num_q_heads / num_kv_heads)), ctx->num_sms);
}

int fkv_fp4_attention(const void *layer, int64_t num_blocks, int tokens_per_block, int num_kv_heads, int head_size,
                      int64_t kv_stride_in_bytes, int64_t block_stride_in_bytes, const void *q, void *out, float *lse,
                      int64_t q_token_stride_in_bytes, int64_t q_head_stride_in_bytes, int64_t out_token_stride_in_bytes,
                      int64_t out_head_stride_in_bytes, int dtype, int64_t num_q_tokens, int num_q_heads,
                      const int32_t *block_tables, int64_t block_table_stride, int max_blocks, const int32_t *seq_lens,
                      const int32_t *cu_seqlens_q, int num_seqs, int max_q_len, float softmax_scale, int causal,
                      void *workspace, int64_t workspace_bytes, void *stream) {
  clear_error();
  const char *w = "fkv_fp4_attention: ";
  auto bad = [&](const char *m) { return fail(FKV_ERR_INVALID_ARG, std::string(w) + m); };
  if (tokens_per_block <= 0 || tokens_per_block % 16) return bad("tokens_per_block must be a positive multiple of 16");
  if (head_size != 64 && head_size != 128)
    return fail(FKV_ERR_UNSUPPORTED, std::string(w) + "head_size must be 64 or 128");
  if (dtype != FKV_DTYPE_BF16 && dtype != FKV_DTYPE_FP16)
    return fail(FKV_ERR_UNSUPPORTED, std::string(w) + "queries must be bfloat16 or half");
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads)
    return bad("the query heads must be a multiple of the key heads");
  if (num_blocks < 0 || num_q_tokens < 0 || num_seqs < 0 || max_blocks < 0) return bad("counts must be non-negative");
  if (!std::isfinite(softmax_scale)) return bad("softmax_scale must be finite");
  if (num_q_tokens == 0 || num_seqs == 0) return FKV_OK;
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
  a.q = (const uint8_t *)q, a.q_token_stride = q_token_stride_in_bytes, a.q_head_stride = q_head_stride_in_bytes;
  a.out = (uint8_t *)out, a.o_token_stride = out_token_stride_in_bytes, a.o_head_stride = out_head_stride_in_bytes;
  a.lse = lse, a.num_q = num_q_tokens, a.tables = block_tables, a.table_stride = block_table_stride;
  a.max_blocks = max_blocks, a.seq_lens = seq_lens, a.cu = cu_seqlens_q, a.num_seqs = num_seqs;
  a.scale = softmax_scale, a.causal = causal;
  ThreadDeviceCtx *ctx;
  const int rc = get_ctx(-1, &ctx);
  if (rc != FKV_OK) return rc;
  const int nt = row_tiles((int64_t)max_q_len * a.group);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < decode_workspace(head_size, nt, ctx->num_sms))
    return bad("the workspace is too small or not aligned");
  cudaStream_t s = (cudaStream_t)stream;
  const bool bf16 = dtype == FKV_DTYPE_BF16;
  if (head_size == 128)
    return bf16 ? launch_decode<128, true>(a, nt, ctx->num_sms, workspace, s) : launch_decode<128, false>(a, nt, ctx->num_sms, workspace, s);
  return bf16 ? launch_decode<64, true>(a, nt, ctx->num_sms, workspace, s) : launch_decode<64, false>(a, nt, ctx->num_sms, workspace, s);
}

}  // extern "C"
