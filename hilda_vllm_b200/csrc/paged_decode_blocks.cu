// Paged decode attention (one query token per sequence) over the block-scaled 8-bit KV cache:
//   out[b, hq] = sum_j p_j vs[g(j), h] Vq[j, h],  p = softmax_j(scale * ks[g(j), h] * q[b, hq] . Kq[j, h])
// over the tokens j < context_lens[b] of sequence b, h = hq / (Hq / Hk), g(j) the group of
// scale_block tokens that j's slot lies in.  mini_vllm/layers/attention.py:134-141 calls an 8-bit
// decode without scales.
#include "kv_blocks.cuh"

namespace hl {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxBatch = 4096;

struct BlockDecodeParams {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scales;
  const float* v_scales;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* context_lens;
  int batch, num_q_heads, num_kv_heads;
  int block_size, scale_block;
  int64_t num_blocks;
  float scale_log2;
  __nv_bfloat16* out;
  int64_t out_stride;
  int32_t* errors;
};

constexpr int kWarps = 8;

// One thread block per (query head, sequence); warp w takes tokens w, w + 8, ...; a lane holds four
// of the 128 dimensions.
__global__ void __launch_bounds__(32 * kWarps) decode_blocks_kernel(const BlockDecodeParams p) {
  const int hq = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = hq / (p.num_q_heads / p.num_kv_heads);
  const int64_t row_bytes = int64_t(p.num_kv_heads) * kBlockHeadDim;
  const int64_t n = min(int64_t(p.context_lens[b]), int64_t(p.max_blocks) * p.block_size);
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  const uint2 qv = *reinterpret_cast<const uint2*>(p.q + b * p.q_stride + hq * kBlockHeadDim + 4 * lane);
  q[0] = bf16lo(qv.x), q[1] = bf16hi(qv.x), q[2] = bf16lo(qv.y), q[3] = bf16hi(qv.y);
  for (int64_t j = warp; j < n; j += kWarps) {
    const int64_t page = p.block_tables[b * p.bt_stride + j / p.block_size];
    if (page < 0 || page >= p.num_blocks) {
      if (lane == 0) atomicOr(p.errors, 2);
      continue;
    }
    const int64_t slot = page * p.block_size + j % p.block_size;
    const int64_t at = slot * row_bytes + h * kBlockHeadDim + 4 * lane, sc = slot / p.scale_block * p.num_kv_heads + h;
    const uint32_t kb = *reinterpret_cast<const uint32_t*>(p.k_cache + at);
    const uint32_t vb = *reinterpret_cast<const uint32_t*>(p.v_cache + at);
    const float2 k0 = e4m3x2_to_float2(kb & 0xffffu), k1 = e4m3x2_to_float2(kb >> 16);
    const float2 v0 = e4m3x2_to_float2(vb & 0xffffu), v1 = e4m3x2_to_float2(vb >> 16);
    float s = q[0] * k0.x + q[1] * k0.y + q[2] * k1.x + q[3] * k1.y;
#pragma unroll
    for (int t = 16; t >= 1; t >>= 1) s += __shfl_xor_sync(0xffffffffu, s, t);
    s *= p.k_scales[sc] * p.scale_log2;
    const float m2 = fmaxf(m, s), a = m == -INFINITY ? 0.f : exp2f(m - m2), e = s == -INFINITY ? 0.f : exp2f(s - m2);
    const float ev = e * p.v_scales[sc];
    l = l * a + e;
    o[0] = o[0] * a + ev * v0.x, o[1] = o[1] * a + ev * v0.y, o[2] = o[2] * a + ev * v1.x, o[3] = o[3] * a + ev * v1.y;
    m = m2;
  }
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][kBlockHeadDim];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
  for (int t = 0; t < 4; ++t) so[warp][4 * lane + t] = o[t];
  __syncthreads();
  if (threadIdx.x >= kBlockHeadDim) return;
  float mm = -INFINITY, ll = 0.f, oo = 0.f;
  for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm[w]);
  for (int w = 0; w < kWarps; ++w) {
    const float a = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - mm);
    ll += sl[w] * a;
    oo += so[w][threadIdx.x] * a;
  }
  p.out[b * p.out_stride + hq * kBlockHeadDim + threadIdx.x] = __float2bfloat16_rn(ll > 0.f || ll != ll ? oo / ll : 0.f);
}

}  // namespace
}  // namespace hl

using namespace hl;

extern "C" int64_t hl_paged_decode_fp8_blocks_workspace_size(int batch, int num_q_heads, int num_kv_heads) {
  if (batch <= 0 || batch > kMaxBatch || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return -1;
  return 256;
}

extern "C" int hl_paged_decode_fp8_blocks(const void* q, int64_t q_row_stride, const void* k_cache,
                                          const void* v_cache, const float* k_scales, const float* v_scales,
                                          const int32_t* block_tables, int64_t bt_stride, int max_blocks_per_seq,
                                          const int32_t* context_lens, int batch, int num_q_heads, int num_kv_heads,
                                          int head_dim, int block_size, int scale_block, int64_t num_blocks,
                                          float softmax_scale, void* out, int64_t out_row_stride, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  clear_error();
  HL_CHECK_ARG(batch >= 0, "hl_paged_decode_fp8_blocks: batch < 0");
  if (batch == 0) return HL_OK;
  HL_CHECK_ARG(batch <= kMaxBatch, "hl_paged_decode_fp8_blocks: batch %d > %d", batch, kMaxBatch);
  HL_CHECK_ARG(q && k_cache && v_cache && k_scales && v_scales && block_tables && context_lens && out,
               "hl_paged_decode_fp8_blocks: null pointer");
  HL_CHECK_ARG(head_dim == kBlockHeadDim, "hl_paged_decode_fp8_blocks: head_dim %d != 128", head_dim);
  HL_CHECK_ARG(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0 &&
                   num_q_heads / num_kv_heads <= 16,
               "hl_paged_decode_fp8_blocks: Hq must be a multiple of Hk, at most 16 query heads per KV head");
  HL_CHECK_ARG(scale_block > 0 && scale_block % 64 == 0 && block_size > 0 && block_size % scale_block == 0,
               "hl_paged_decode_fp8_blocks: scale_block must be a multiple of 64 that divides block_size");
  HL_CHECK_ARG(max_blocks_per_seq > 0 && bt_stride >= max_blocks_per_seq && num_blocks > 0,
               "hl_paged_decode_fp8_blocks: bad block table or pool shape");
  HL_CHECK_ARG(int64_t(max_blocks_per_seq) * block_size <= 0x7fffffff,
               "hl_paged_decode_fp8_blocks: a block table row spans 2^31 tokens or more");
  HL_CHECK_ARG(aligned16(q) && q_row_stride % 8 == 0 && q_row_stride >= int64_t(num_q_heads) * head_dim &&
                   aligned16(out) && out_row_stride % 8 == 0 && out_row_stride >= int64_t(num_q_heads) * head_dim &&
                   aligned16(k_cache) && aligned16(v_cache),
               "hl_paged_decode_fp8_blocks: 16-byte alignment and row strides >= Hq*D, multiples of 8, required");
  const int64_t need = hl_paged_decode_fp8_blocks_workspace_size(batch, num_q_heads, num_kv_heads);
  if (!workspace || workspace_bytes < need || !aligned16(workspace)) {
    set_error("hl_paged_decode_fp8_blocks: workspace of %lld bytes needed (got %lld)", (long long)need,
              (long long)workspace_bytes);
    return HL_ERR_WORKSPACE;
  }
  BlockDecodeParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_row_stride;
  p.k_cache = static_cast<const uint8_t*>(k_cache);
  p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.block_tables = block_tables;
  p.bt_stride = bt_stride;
  p.max_blocks = max_blocks_per_seq;
  p.context_lens = context_lens;
  p.batch = batch;
  p.num_q_heads = num_q_heads;
  p.num_kv_heads = num_kv_heads;
  p.block_size = block_size;
  p.scale_block = scale_block;
  p.num_blocks = num_blocks;
  p.scale_log2 = softmax_scale * kLog2e;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_row_stride;
  p.errors = static_cast<int32_t*>(workspace);
  const dim3 grid(num_q_heads, batch);
  decode_blocks_kernel<<<grid, 32 * kWarps, 0, static_cast<cudaStream_t>(stream)>>>(p);
  HL_CHECK_LAUNCH("hl_paged_decode_fp8_blocks");
  return HL_OK;
}
