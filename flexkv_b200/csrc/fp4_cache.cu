// The KV cache in 4 bits: quantising tokens as they are written, reading
// them back, and both for whole blocks of every layer (the 16-bit cache of an
// inference engine on one side, 4-bit blocks for the host and SSD tiers on
// the other).
//
// Format.  16 consecutive channels of one token and head are a group: 16
// e2m1 values q and one scale s of 5 exponent and 3 mantissa bits (a half
// without sign and low mantissa bits: code c is the half with bits c << 7).
//   s = nearest(amax / 6), at most 10240;  q = nearest_e2m1(x / s)
// both with ties to the even code; x' = q * s has at most 6 significant bits
// and is exact in half and bfloat16.  16 tokens of one head are a unit of
// 9 * D bytes: 16 rows of D / 2 payload bytes (even channel in the low four
// bits), then 16 rows of D / 16 scale bytes.  A unit is one contiguous,
// 16-byte aligned piece, which attention fetches in 16-byte copies; a block
// holds its units head after head, so a head's share of a block (and a
// tensor-parallel rank's) is one piece too.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "fkv_common.h"
#include "fp4_format.cuh"
#include "fp4_launch.cuh"

namespace fkv {
namespace {

constexpr int kMaxLayers = 128;  // layers of one launch: their pointers travel in the kernel's parameters
constexpr int kMaxListed = 256;  // pairs of blocks of one launch whose ids travel there too
constexpr int kThreads = 256;
constexpr int kUnroll = 4;

// Tokens by slot; blocks whose ids are in device memory; blocks of which one
// list of ids or both come from the host, in the parameters: nothing has to be
// copied to the device first, and a captured launch keeps its ids.  9 blocks of 28
// layers there and back take 8.4 us so, with ids on the device 7.4 (the larger
// parameters); 1000 blocks of one layer, four launches each way, 40 and 26.
enum Form { kTokens, kBlocks, kListed };

// LAYERS, PAIRS: what the call's pointers and ids need; they are copied with every launch.
template <int LAYERS, int PAIRS>
struct RowsArgsOf {
  int num_heads;
  int kv_dim;
  int tokens_per_block;
  int upb;                // units (16 tokens) of a block
  int groups;             // groups (16 channels) of a head
  Divisor by_upb, by_groups;
  bool far;               // more units in the 4-bit layer, or in a block, than by_upb is for
  int64_t num_rows;       // tokens of the call (blocks * tokens_per_block for the block form)
  int64_t num_slots;      // slots of the 4-bit layer
  int64_t num_blocks, num_row_blocks;  // of the 4-bit and of the 16-bit side (block form)
  int64_t fp4_kv_stride, fp4_block_stride;
  int64_t token_stride[2], head_stride[2];        // bytes, 16-bit side
  int64_t row_block_stride;                        // bytes, block form
  const int64_t *fp4_ids;                          // slots (token form) or blocks; null: listed[0]
  const int64_t *row_ids;                          // blocks of the 16-bit side (block form); null: listed[1]
  uint8_t *fp4[LAYERS];
  uint8_t *rows[2][LAYERS];
  int64_t listed[2][PAIRS];
};
template <int FORM>
using RowsArgs = RowsArgsOf<FORM == kTokens ? 1 : kMaxLayers, FORM == kListed ? kMaxListed : 1>;

// 32 bytes in one access where the address allows it, else two of 16.
template <bool WIDE>
__device__ __forceinline__ void load_group(const uint8_t *p, uint32_t (&r)[8]) {
  if (WIDE) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p));
  } else {
    const uint4 a = *reinterpret_cast<const uint4 *>(p), b = *reinterpret_cast<const uint4 *>(p + 16);
    r[0] = a.x, r[1] = a.y, r[2] = a.z, r[3] = a.w, r[4] = b.x, r[5] = b.y, r[6] = b.z, r[7] = b.w;
  }
}
template <bool WIDE>
__device__ __forceinline__ void store_group(uint8_t *p, const uint32_t (&r)[8]) {
  if (WIDE) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4 *>(p)[0] = make_uint4(r[0], r[1], r[2], r[3]);
    reinterpret_cast<uint4 *>(p)[1] = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

// One thread per group of 16 channels, kUnroll of them under way at a time.  A
// CTA takes R consecutive rows of the list (R = 16, or 1 for a call with fewer
// rows than 16) of one layer and side, for every head: neighbouring threads have
// neighbouring groups, then rows, so that 32 lanes store 256 payload bytes and
// 32 scale bytes of one unit next to each other.  NG: groups of a head where
// they and the rows divide the CTA's threads evenly: a thread then keeps its
// row and group through all heads and looks its slot up once.  0: at run time,
// a place for each group.
//
// Bound by memory: 2 + 9/16 bytes a value.  Measured (B200, heads of 128): 256
// blocks of 16 tokens, 8 heads, 32 layers packed and unpacked again in 215 us, 6.4
// TB/s, 98 % of a copy's rate (227 us, 93 %, where other work comes between); a call
// that reads 32768 tokens 30.5 us, 5.7 TB/s.
// With divisions for each group's place and true ones in the rounding, 9 blocks of
// 28 layers there and back took 9.9 us instead of 6.9, and quantising was bound by
// the issue of 315 instructions a group.
template <bool WRITE, bool BF16, int FORM, bool WIDE, int NG, int R>
__global__ void __launch_bounds__(kThreads) fp4_rows_kernel(const __grid_constant__ RowsArgs<FORM> a) {
  after_previous();
  const int ng = NG ? NG : a.groups, D = 16 * ng;
  const int layer = a.kv_dim == 1 ? blockIdx.y : blockIdx.y >> 1, side = a.kv_dim == 1 ? 0 : blockIdx.y & 1;
  const int64_t row0 = (int64_t)blockIdx.x * R;
  uint8_t *const fp4 = a.fp4[layer] + side * a.fp4_kv_stride;
  uint8_t *const rows = a.rows[side][layer];
  const int64_t token_stride = a.token_stride[side], head_stride = a.head_stride[side];
  const int64_t unit_step = (int64_t)a.upb * (9 * D);  // from a head's unit to the next head's

  // Unit of the first head and 16-bit row of row t of the CTA: null where there is none.
  auto find = [&](int t, uint8_t *&unit, uint8_t *&row, int &off) {
    const int64_t i = row0 + t;
    unit = row = nullptr;
    if (i >= a.num_rows) return;
    if (FORM != kTokens) {
      // a block's rows are multiples of 16, R = 16: row 0 says which block
      const int64_t u = row0 >> 4;
      const int64_t blk = a.far ? u / a.upb : divide((int)u, a.by_upb);
      const int in = (int)(u - blk * a.upb);
      const int64_t fb = FORM == kListed && !a.fp4_ids ? a.listed[0][blk] : a.fp4_ids[blk];
      const int64_t rb = FORM == kListed && !a.row_ids ? a.listed[1][blk] : a.row_ids[blk];
      if (fb < 0 || fb >= a.num_blocks || rb < 0 || rb >= a.num_row_blocks) return;
      off = t;
      unit = fp4 + fb * a.fp4_block_stride + (int64_t)in * (9 * D);
      row = rows + rb * a.row_block_stride + (in * 16 + t) * token_stride;
    } else {
      row = rows + i * token_stride;
      const int64_t slot = a.fp4_ids[i];
      if (slot < 0 || slot >= a.num_slots) return;
      const int64_t u = slot >> 4;
      const int64_t blk = a.far ? u / a.upb : divide((int)u, a.by_upb);
      off = (int)(slot & 15);
      unit = fp4 + blk * a.fp4_block_stride + (u - blk * a.upb) * (9 * D);
    }
  };
  auto load = [&](uint32_t(&x)[8], const uint8_t *unit, const uint8_t *row, int off, int g) {
    if (WRITE) {
      if (unit) load_group<WIDE>(row + g * 32, x);
    } else if (unit) {
      const uint2 p = *reinterpret_cast<const uint2 *>(unit + off * (D / 2) + g * 8);
      x[0] = p.x, x[1] = p.y, x[2] = unit[8 * D + off * ng + g];
    } else {
      x[0] = x[1] = x[2] = 0;  // a row without a slot reads as zeros
    }
  };
  auto finish = [&](uint32_t(&x)[8], uint8_t *unit, uint8_t *row, int off, int g) {
    if (WRITE) {
      if (!unit) return;
      uint2 p;
      const uint32_t code = quantise_group<BF16>(x, p);
      *reinterpret_cast<uint2 *>(unit + off * (D / 2) + g * 8) = p;
      unit[8 * D + off * ng + g] = (uint8_t)code;
    } else if (row) {
      uint32_t y[8];
      dequantise_group<BF16>(make_uint2(x[0], x[1]), x[2], y);
      store_group<WIDE>(row + g * 32, y);
    }
  };

  if (NG) {
    constexpr int kPlaces = NG ? R * NG : 1, kStep = kThreads / kPlaces;  // heads at a time
    const int t = threadIdx.x % kPlaces / (NG ? NG : 1), g = threadIdx.x % (NG ? NG : 1);
    uint8_t *unit, *row;
    int off = 0;
    find(t, unit, row, off);
    if (!row || (WRITE && !unit)) return;
    for (int h0 = threadIdx.x / kPlaces; h0 < a.num_heads; h0 += kStep * kUnroll) {
      uint32_t x[kUnroll][8];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int h = h0 + k * kStep;
        if (h < a.num_heads) load(x[k], unit ? unit + h * unit_step : nullptr, row + h * head_stride, off, g);
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int h = h0 + k * kStep;
        if (h < a.num_heads) finish(x[k], unit ? unit + h * unit_step : nullptr, row + h * head_stride, off, g);
      }
    }
  } else {
    const int work = a.num_heads * R * ng;
    for (int w0 = threadIdx.x; w0 < work; w0 += kThreads * kUnroll) {
      uint32_t x[kUnroll][8];
      uint8_t *unit[kUnroll], *row[kUnroll];
      int off[kUnroll], g[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int w = w0 + k * kThreads;
        unit[k] = row[k] = nullptr, off[k] = 0;
        if (w >= work) continue;
        const int q = divide(w, a.by_groups), h = q / R;  // w < 2^24
        g[k] = w - q * ng;
        find(q % R, unit[k], row[k], off[k]);
        if (row[k]) row[k] += h * head_stride;
        if (unit[k]) unit[k] += h * unit_step;
        if (row[k]) load(x[k], unit[k], row[k], off[k], g[k]);
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
        if (row[k]) finish(x[k], unit[k], row[k], off[k], g[k]);
    }
  }
}

template <bool WRITE, bool BF16, int FORM, bool WIDE, int R>
cudaError_t launch_ng(const RowsArgs<FORM> &a, dim3 grid, int ng, cudaStream_t s) {
  switch (ng) {
    case 4: return launch_next(fp4_rows_kernel<WRITE, BF16, FORM, WIDE, 4, R>, grid, kThreads, 0, s, a);
    case 8: return launch_next(fp4_rows_kernel<WRITE, BF16, FORM, WIDE, 8, R>, grid, kThreads, 0, s, a);
    case 16: return launch_next(fp4_rows_kernel<WRITE, BF16, FORM, WIDE, 16, R>, grid, kThreads, 0, s, a);
    default: return launch_next(fp4_rows_kernel<WRITE, BF16, FORM, WIDE, 0, R>, grid, kThreads, 0, s, a);
  }
}
template <bool WRITE, bool BF16, int FORM, bool WIDE>
cudaError_t launch_r(const RowsArgs<FORM> &a, int rows_at_once, dim3 grid, int ng, cudaStream_t s) {
  if (FORM != kTokens || rows_at_once == 16)
    return launch_ng<WRITE, BF16, FORM, WIDE, 16>(a, grid, ng, s);
  return launch_ng<WRITE, BF16, FORM, WIDE, FORM != kTokens ? 16 : 1>(a, grid, ng, s);
}
template <bool WRITE, int FORM>
cudaError_t launch_rows(const RowsArgs<FORM> &a, bool bf16, bool wide, int r, dim3 grid, int ng, cudaStream_t s) {
  if (bf16)
    return wide ? launch_r<WRITE, true, FORM, true>(a, r, grid, ng, s) : launch_r<WRITE, true, FORM, false>(a, r, grid, ng, s);
  return wide ? launch_r<WRITE, false, FORM, true>(a, r, grid, ng, s) : launch_r<WRITE, false, FORM, false>(a, r, grid, ng, s);
}

int check_geometry(const char *who, int kv_dim, int64_t num_blocks, int tpb, int heads, int head_size, int dtype) {
  const std::string w(who);
  if (kv_dim != 1 && kv_dim != 2) return fail(FKV_ERR_INVALID_ARG, w + ": kv_dim must be 1 or 2");
  if (tpb <= 0 || tpb % 16) return fail(FKV_ERR_INVALID_ARG, w + ": tokens_per_block must be a positive multiple of 16");
  if (head_size <= 0 || head_size % 16 || head_size > 65536)
    return fail(FKV_ERR_INVALID_ARG, w + ": head_size must be a positive multiple of 16");
  if (heads <= 0 || heads > 65536) return fail(FKV_ERR_INVALID_ARG, w + ": num_heads must be positive");
  if ((int64_t)heads * head_size > (int64_t)1 << 24) return fail(FKV_ERR_INVALID_ARG, w + ": a token of more than 2^24 values");
  if (num_blocks < 0 || num_blocks > INT64_MAX / tpb) return fail(FKV_ERR_INVALID_ARG, w + ": bad number of blocks");
  if (dtype != FKV_DTYPE_BF16 && dtype != FKV_DTYPE_FP16)
    return fail(FKV_ERR_UNSUPPORTED, w + ": the 16-bit side must be bfloat16 or half");
  return FKV_OK;
}

bool aligned(int64_t v, int64_t to) { return v % to == 0; }
bool aligned(const void *p, int64_t to) { return (uintptr_t)p % to == 0; }

template <bool WRITE, int FORM>
int run_rows(RowsArgs<FORM> &a, int num_layers, int head_size, int dtype, bool wide, cudaStream_t s) {
  const int ng = head_size / 16, r = a.num_rows < 16 ? 1 : 16;
  a.upb = a.tokens_per_block / 16, a.groups = ng;
  a.far = a.num_slots >> 32 || a.num_rows >> 32 || a.upb > 4096;
  if (!a.far) a.by_upb = divisor_of(a.upb);
  a.by_groups = divisor_of(ng);
  // grid.x counts row groups: 2^31 - 1 of them is the launch limit
  const int64_t gx = (a.num_rows + r - 1) / r;
  if (gx > INT32_MAX) return fail(FKV_ERR_INVALID_ARG, "more than 2^31 groups of rows in one call");
  FKV_CUDA((launch_rows<WRITE, FORM>(a, dtype == FKV_DTYPE_BF16, wide, r, dim3((unsigned)gx, num_layers * a.kv_dim), ng, s)));
  note_launch();
  return FKV_OK;
}

template <bool WRITE>
int tokens_call(const char *who, void *layer, int kv_dim, int64_t num_blocks, int tpb, int heads, int head_size,
                int64_t kv_stride, int64_t block_stride, const void *k, const void *v, int64_t k_token_stride,
                int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, int dtype, const int64_t *slots,
                int64_t num_tokens, void *stream) {
  clear_error();
  int rc = check_geometry(who, kv_dim, num_blocks, tpb, heads, head_size, dtype);
  if (rc != FKV_OK) return rc;
  const std::string w(who);
  if (num_tokens < 0) return fail(FKV_ERR_INVALID_ARG, w + ": num_tokens must be non-negative");
  if (num_tokens == 0) return FKV_OK;
  if (!k || !slots || (kv_dim == 2 && !v) || (num_blocks > 0 && !layer))
    return fail(FKV_ERR_INVALID_ARG, w + ": null pointer");
  if (kv_dim == 1 && v) return fail(FKV_ERR_INVALID_ARG, w + ": a latent layer (kv_dim 1) has no values");
  if (!aligned(layer, 16) || !aligned(kv_stride, 16) || !aligned(block_stride, 16))
    return fail(FKV_ERR_MISALIGNED, w + ": the layer and its strides must be multiples of 16 bytes");
  RowsArgs<kTokens> a{};
  a.num_heads = heads, a.kv_dim = kv_dim, a.tokens_per_block = tpb;
  a.num_rows = num_tokens, a.num_slots = num_blocks * tpb;
  a.fp4_kv_stride = kv_stride, a.fp4_block_stride = block_stride;
  a.token_stride[0] = k_token_stride, a.head_stride[0] = k_head_stride;
  a.token_stride[1] = v_token_stride, a.head_stride[1] = v_head_stride;
  a.fp4_ids = slots;
  a.fp4[0] = (uint8_t *)layer;
  a.rows[0][0] = (uint8_t *)k, a.rows[1][0] = (uint8_t *)v;
  bool wide = true;
  for (int i = 0; i < kv_dim; ++i) {
    if (!aligned(a.rows[i][0], 16) || !aligned(a.token_stride[i], 16) || !aligned(a.head_stride[i], 16))
      return fail(FKV_ERR_MISALIGNED, w + ": rows must start on 16-byte boundaries");
    wide = wide && aligned(a.rows[i][0], 32) && aligned(a.token_stride[i], 32) && aligned(a.head_stride[i], 32);
  }
  return run_rows<WRITE, kTokens>(a, 1, head_size, dtype, wide, (cudaStream_t)stream);
}

// host_lists: which ids are in host memory (kListed)
template <bool WRITE, int FORM>
int blocks_call(const char *who, int num_layers, void *const *fp4_layers, void *const *kv_layers, int kv_dim, int tpb,
                int heads, int head_size, int64_t fp4_num_blocks, int64_t fp4_kv_stride, int64_t fp4_block_stride,
                int64_t kv_num_blocks, int64_t kv_kv_stride, int64_t kv_block_stride, int dtype, const int64_t *fp4_ids,
                const int64_t *kv_ids, int64_t num, int host_lists, void *stream) {
  clear_error();
  int rc = check_geometry(who, kv_dim, fp4_num_blocks, tpb, heads, head_size, dtype);
  if (rc != FKV_OK) return rc;
  const std::string w(who);
  if (num < 0 || num_layers < 0 || kv_num_blocks < 0 || num > INT64_MAX / tpb)
    return fail(FKV_ERR_INVALID_ARG, w + ": counts must be non-negative");
  if (host_lists & ~(FKV_FP4_KV_IDS | FKV_FP4_FP4_IDS)) return fail(FKV_ERR_INVALID_ARG, w + ": unknown host_lists");
  if (num == 0 || num_layers == 0) return FKV_OK;
  if (!fp4_layers || !kv_layers || !fp4_ids || !kv_ids) return fail(FKV_ERR_INVALID_ARG, w + ": null pointer");
  if (!aligned(fp4_kv_stride, 16) || !aligned(fp4_block_stride, 16) || !aligned(kv_kv_stride, 16) ||
      !aligned(kv_block_stride, 16))
    return fail(FKV_ERR_MISALIGNED, w + ": strides must be multiples of 16 bytes");
  bool wide = aligned(kv_kv_stride, 32) && aligned(kv_block_stride, 32);
  for (int l = 0; l < num_layers; ++l) {
    if (!fp4_layers[l] || !kv_layers[l]) return fail(FKV_ERR_INVALID_ARG, w + ": null layer pointer");
    if (!aligned(fp4_layers[l], 16) || !aligned(kv_layers[l], 16))
      return fail(FKV_ERR_MISALIGNED, w + ": layers must start on 16-byte boundaries");
    wide = wide && aligned(kv_layers[l], 32);
  }
  RowsArgs<FORM> a{};
  a.num_heads = heads, a.kv_dim = kv_dim, a.tokens_per_block = tpb;
  a.num_slots = fp4_num_blocks * tpb, a.num_blocks = fp4_num_blocks, a.num_row_blocks = kv_num_blocks;
  a.fp4_kv_stride = fp4_kv_stride, a.fp4_block_stride = fp4_block_stride;
  a.row_block_stride = kv_block_stride;
  for (int i = 0; i < 2; ++i) a.head_stride[i] = 2 * head_size, a.token_stride[i] = (int64_t)2 * head_size * heads;
  for (int l0 = 0; l0 < num_layers; l0 += kMaxLayers) {
    const int n = num_layers - l0 < kMaxLayers ? num_layers - l0 : kMaxLayers;
    for (int l = 0; l < n; ++l) {
      a.fp4[l] = (uint8_t *)fp4_layers[l0 + l];
      a.rows[0][l] = (uint8_t *)kv_layers[l0 + l];
      a.rows[1][l] = (uint8_t *)kv_layers[l0 + l] + kv_kv_stride;
    }
    const int64_t step = FORM == kListed ? kMaxListed : num;
    for (int64_t i = 0; i < num; i += step) {
      const int64_t pairs = std::min(num - i, step);
      a.num_rows = pairs * tpb;
      a.fp4_ids = host_lists & FKV_FP4_FP4_IDS ? nullptr : fp4_ids + i;
      a.row_ids = host_lists & FKV_FP4_KV_IDS ? nullptr : kv_ids + i;
      if (FORM == kListed && !a.fp4_ids) std::copy_n(fp4_ids + i, pairs, a.listed[0]);
      if (FORM == kListed && !a.row_ids) std::copy_n(kv_ids + i, pairs, a.listed[1]);
      if ((rc = run_rows<WRITE, FORM>(a, n, head_size, dtype, wide, (cudaStream_t)stream)) != FKV_OK) return rc;
    }
  }
  return FKV_OK;
}

}  // namespace
}  // namespace fkv

extern "C" {

int fkv_fp4_write(void *layer, int kv_dim, int64_t num_blocks, int tokens_per_block, int num_heads, int head_size,
                  int64_t kv_stride_in_bytes, int64_t block_stride_in_bytes, const void *k, const void *v,
                  int64_t k_token_stride_in_bytes, int64_t k_head_stride_in_bytes, int64_t v_token_stride_in_bytes,
                  int64_t v_head_stride_in_bytes, int dtype, const int64_t *slots, int64_t num_tokens, void *stream) {
  return fkv::tokens_call<true>("fkv_fp4_write", layer, kv_dim, num_blocks, tokens_per_block, num_heads, head_size,
                                kv_stride_in_bytes, block_stride_in_bytes, k, v, k_token_stride_in_bytes,
                                k_head_stride_in_bytes, v_token_stride_in_bytes, v_head_stride_in_bytes, dtype, slots,
                                num_tokens, stream);
}

int fkv_fp4_read(const void *layer, int kv_dim, int64_t num_blocks, int tokens_per_block, int num_heads, int head_size,
                 int64_t kv_stride_in_bytes, int64_t block_stride_in_bytes, void *k, void *v,
                 int64_t k_token_stride_in_bytes, int64_t k_head_stride_in_bytes, int64_t v_token_stride_in_bytes,
                 int64_t v_head_stride_in_bytes, int dtype, const int64_t *slots, int64_t num_tokens, void *stream) {
  return fkv::tokens_call<false>("fkv_fp4_read", const_cast<void *>(layer), kv_dim, num_blocks, tokens_per_block,
                                 num_heads, head_size, kv_stride_in_bytes, block_stride_in_bytes, k, v,
                                 k_token_stride_in_bytes, k_head_stride_in_bytes, v_token_stride_in_bytes,
                                 v_head_stride_in_bytes, dtype, slots, num_tokens, stream);
}

int fkv_fp4_pack_blocks(int num_layers, void *const *kv_layer_ptrs, void *const *fp4_layer_ptrs, int kv_dim,
                        int tokens_per_block, int num_heads, int head_size, int64_t kv_num_blocks,
                        int64_t kv_kv_stride_in_bytes, int64_t kv_block_stride_in_bytes, int64_t fp4_num_blocks,
                        int64_t fp4_kv_stride_in_bytes, int64_t fp4_block_stride_in_bytes, int dtype,
                        const int64_t *kv_block_ids, const int64_t *fp4_block_ids, int64_t num_blocks, void *stream) {
  return fkv::blocks_call<true, fkv::kBlocks>("fkv_fp4_pack_blocks", num_layers, fp4_layer_ptrs, kv_layer_ptrs,
                                              kv_dim, tokens_per_block, num_heads, head_size, fp4_num_blocks,
                                              fp4_kv_stride_in_bytes, fp4_block_stride_in_bytes, kv_num_blocks,
                                              kv_kv_stride_in_bytes, kv_block_stride_in_bytes, dtype, fp4_block_ids,
                                              kv_block_ids, num_blocks, 0, stream);
}

int fkv_fp4_pack_blocks_listed(int num_layers, void *const *kv_layer_ptrs, void *const *fp4_layer_ptrs, int kv_dim,
                               int tokens_per_block, int num_heads, int head_size, int64_t kv_num_blocks,
                               int64_t kv_kv_stride_in_bytes, int64_t kv_block_stride_in_bytes,
                               int64_t fp4_num_blocks, int64_t fp4_kv_stride_in_bytes,
                               int64_t fp4_block_stride_in_bytes, int dtype, const int64_t *kv_block_ids,
                               const int64_t *fp4_block_ids, int64_t num_blocks, int host_lists, void *stream) {
  return fkv::blocks_call<true, fkv::kListed>("fkv_fp4_pack_blocks_listed", num_layers, fp4_layer_ptrs, kv_layer_ptrs,
                                              kv_dim, tokens_per_block, num_heads, head_size, fp4_num_blocks,
                                              fp4_kv_stride_in_bytes, fp4_block_stride_in_bytes, kv_num_blocks,
                                              kv_kv_stride_in_bytes, kv_block_stride_in_bytes, dtype, fp4_block_ids,
                                              kv_block_ids, num_blocks, host_lists, stream);
}

int fkv_fp4_unpack_blocks(int num_layers, void *const *fp4_layer_ptrs, void *const *kv_layer_ptrs, int kv_dim,
                          int tokens_per_block, int num_heads, int head_size, int64_t fp4_num_blocks,
                          int64_t fp4_kv_stride_in_bytes, int64_t fp4_block_stride_in_bytes, int64_t kv_num_blocks,
                          int64_t kv_kv_stride_in_bytes, int64_t kv_block_stride_in_bytes, int dtype,
                          const int64_t *fp4_block_ids, const int64_t *kv_block_ids, int64_t num_blocks,
                          void *stream) {
  return fkv::blocks_call<false, fkv::kBlocks>("fkv_fp4_unpack_blocks", num_layers, fp4_layer_ptrs, kv_layer_ptrs,
                                               kv_dim, tokens_per_block, num_heads, head_size, fp4_num_blocks,
                                               fp4_kv_stride_in_bytes, fp4_block_stride_in_bytes, kv_num_blocks,
                                               kv_kv_stride_in_bytes, kv_block_stride_in_bytes, dtype, fp4_block_ids,
                                               kv_block_ids, num_blocks, 0, stream);
}

int fkv_fp4_unpack_blocks_listed(int num_layers, void *const *fp4_layer_ptrs, void *const *kv_layer_ptrs, int kv_dim,
                                 int tokens_per_block, int num_heads, int head_size, int64_t fp4_num_blocks,
                                 int64_t fp4_kv_stride_in_bytes, int64_t fp4_block_stride_in_bytes,
                                 int64_t kv_num_blocks, int64_t kv_kv_stride_in_bytes,
                                 int64_t kv_block_stride_in_bytes, int dtype, const int64_t *fp4_block_ids,
                                 const int64_t *kv_block_ids, int64_t num_blocks, int host_lists, void *stream) {
  return fkv::blocks_call<false, fkv::kListed>("fkv_fp4_unpack_blocks_listed", num_layers, fp4_layer_ptrs,
                                               kv_layer_ptrs, kv_dim, tokens_per_block, num_heads, head_size,
                                               fp4_num_blocks, fp4_kv_stride_in_bytes, fp4_block_stride_in_bytes,
                                               kv_num_blocks, kv_kv_stride_in_bytes, kv_block_stride_in_bytes, dtype,
                                               fp4_block_ids, kv_block_ids, num_blocks, host_lists, stream);
}

}  // extern "C"
