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

// One warp per (new token, query head), a key at a time: the plainest form.
template <bool BF16>
__global__ void fp4_attention_plain_kernel(const __grid_constant__ AttnArgs a, int D) {
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int qh = blockIdx.y, h = qh / a.group;
  int b = 0;
  int64_t first = 0, rows = a.num_q / a.num_seqs;
  if (a.cu) {
    for (; b < a.num_seqs; ++b)
      if (row >= a.cu[b] && row < a.cu[b + 1]) break;
    if (b == a.num_seqs) return;
    first = a.cu[b], rows = a.cu[b + 1] - first;
  } else {
    b = (int)(row / rows);
    first = b * rows;
  }
  const int64_t len = min((int64_t)max(a.seq_lens[b], 0), (int64_t)a.max_blocks * a.tokens_per_block);
  const int64_t end = a.causal ? min(len, a.seq_lens[b] - rows + (row - first) + 1) : len;
  const uint8_t *q = a.q + row * a.q_token_stride + qh * a.q_head_stride;
  const int ng = D / 16;
  float m = -INFINITY, l = 0, o[8][2] = {};
  for (int64_t j = 0; j < end; ++j) {
    const int64_t page = a.tables[b * a.table_stride + j / a.tokens_per_block];
    if (page < 0 || page >= a.num_blocks) continue;
    const int off = j % a.tokens_per_block;
    const uint8_t *u = a.layer + page * a.block_stride + ((int64_t)h * (a.tokens_per_block / 16) + off / 16) * (9 * D);
    float s = 0;
    for (int c = lane; c < D / 2; c += 32) {
      const uint32_t k = hmul2(e2m1x2_to_half2(u[(off % 16) * (D / 2) + c]), scale_half2(u[8 * D + (off % 16) * ng + c / 8]));
      const float2 kf = __half22float2(*(const __half2 *)&k);
      const float2 qf = pair_to_float2<BF16>(((const uint32_t *)q)[c]);
      s += kf.x * qf.x + kf.y * qf.y;
    }
    for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(~0u, s, i);
    s *= a.scale;
    const float mn = fmaxf(m, s), p = __expf(s - mn), r = __expf(m - mn);
    m = mn, l = l * r + p;
    u += a.kv_stride;
    int i = 0;
    for (int c = lane; c < D / 2; c += 32, ++i) {
      const uint32_t v = hmul2(e2m1x2_to_half2(u[(off % 16) * (D / 2) + c]), scale_half2(u[8 * D + (off % 16) * ng + c / 8]));
      const float2 vf = __half22float2(*(const __half2 *)&v);
      o[i][0] = o[i][0] * r + p * vf.x, o[i][1] = o[i][1] * r + p * vf.y;
    }
  }
  uint8_t *dst = a.out + row * a.o_token_stride + qh * a.o_head_stride;
  const float inv = l > 0 ? 1 / l : 0;
  int i = 0;
  for (int c = lane; c < D / 2; c += 32, ++i) {
    if (BF16)
      ((__nv_bfloat162 *)dst)[c] = __floats2bfloat162_rn(o[i][0] * inv, o[i][1] * inv);
    else
      ((__half2 *)dst)[c] = __floats2half2_rn(o[i][0] * inv, o[i][1] * inv);
  }
  if (a.lse && lane == 0) a.lse[row * (a.kv_heads * a.group) + qh] = l > 0 ? m + logf(l) : -INFINITY;
}

}  // namespace
}  // namespace fkv

using namespace fkv;

extern "C" {

int64_t fkv_fp4_attention_workspace(int64_t num_q_tokens, int num_q_heads, int num_kv_heads, int head_size, int num_seqs,
                                    int max_q_len) {
  return 0;
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
  const dim3 grid((unsigned)num_q_tokens, num_q_heads);
  if (dtype == FKV_DTYPE_BF16)
    fp4_attention_plain_kernel<true><<<grid, 32, 0, (cudaStream_t)stream>>>(a, head_size);
  else
    fp4_attention_plain_kernel<false><<<grid, 32, 0, (cudaStream_t)stream>>>(a, head_size);
  FKV_CUDA(cudaGetLastError());
  note_launch();
  return FKV_OK;
}

}  // extern "C"
