// KV store into the block-scaled 8-bit cache: the scale of a group (scale_block consecutive tokens
// of a page, one head) follows the data instead of being calibrated beforehand
// (mini_vllm/layers/attention.py:51-52,133 stores e4m3 without scales).
//
// Per group and head, with a = max |x| over this call's new rows (finite values) and s_old the
// group's scale if it holds rows from before this call (0 otherwise):
//   s = max(s_old, smallest power of two with a / s <= 448, 2^-100)
//   rows from before: e4m3(q * s_old / s);   new rows: e4m3(x / s), saturating;   scale := s.
// Sequence b's rows cu[b] .. cu[b+1]-1 are its tokens context_lens[b] - n .. context_lens[b]-1, so
// "rows from before" are the tokens of the group in front of its first new one, whatever the page
// held for an earlier owner.
#include "kv_blocks.cuh"

namespace hl {
namespace {

constexpr int kStoreWindow = 16;  // rows whose group runs one thread block starts
constexpr int kStoreThreads = 128;

struct StoreBlocksParams {
  const __nv_bfloat16* x[2];  // key, value
  int64_t x_stride[2];
  uint8_t* cache[2];
  float* scales[2];
  int64_t num_tokens;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* context_lens;
  const int32_t* cu;
  int num_seqs;
  int num_kv_heads;
  int block_size;
  int scale_block;
  int64_t num_blocks;
};

// The rows of a call that fall into one group: rows [row, row + count) go to offsets
// [held, held + count) of the group whose first slot is `slot0`.  count = 0: none.
struct GroupRun {
  int64_t row, slot0;
  int count, held;
};

// The run that starts at row i; count 0 where i is inside a run or belongs to no sequence.
__device__ GroupRun run_at(const StoreBlocksParams& p, int64_t i) {
  GroupRun r{i, 0, 0, 0};
  int64_t first = i, last = i + 1;  // rows of i's sequence
  int b = int(i);
  if (p.cu) {
    int lo = 0, hi = p.num_seqs;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.cu[mid + 1] > i) hi = mid; else lo = mid + 1;
    }
    b = lo;
    if (b >= p.num_seqs || p.cu[b] > i || p.cu[b] < 0) return r;
    first = p.cu[b];
    last = min(int64_t(p.cu[b + 1]), p.num_tokens);
  }
  const int64_t pos = int64_t(p.context_lens[b]) - ((p.cu ? int64_t(p.cu[b + 1]) : last) - i);
  const int64_t j = pos / p.block_size;
  if (pos < 0 || j >= p.max_blocks) return r;
  const int held = int(pos % p.scale_block);
  if (held != 0 && i != first) return r;
  const int64_t page = p.block_tables[b * p.bt_stride + j];
  if (page < 0 || page >= p.num_blocks) return r;
  r.held = held;
  r.slot0 = page * p.block_size + pos % p.block_size - held;
  r.count = int(min(int64_t(p.scale_block - held), last - i));
  return r;
}

// One warp, one run, one head, K or V: 16 lanes per row of 128 elements.
__device__ void store_run(const StoreBlocksParams& p, const GroupRun& r, int head, int kv, int lane) {
  const int sub = lane >> 4, e0 = (lane & 15) * 8;
  const __nv_bfloat16* x = p.x[kv] + r.row * p.x_stride[kv] + head * kBlockHeadDim + e0;
  const int64_t row_bytes = int64_t(p.num_kv_heads) * kBlockHeadDim;
  uint8_t* out = p.cache[kv] + r.slot0 * row_bytes + head * kBlockHeadDim + e0;
  float* scale_at = p.scales[kv] + r.slot0 / p.scale_block * p.num_kv_heads + head;
  float amax = 0.f;
  for (int i = sub; i < r.count; i += 2) {
    const uint4 v = *reinterpret_cast<const uint4*>(x + i * p.x_stride[kv]);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int t = 0; t < 4; ++t) amax = fmaxf(amax, fmaxf(finite_abs(bf16lo(w[t])), finite_abs(bf16hi(w[t]))));
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float s = scale_for(amax);
  if (r.held > 0) {
    const float old = *scale_at;
    const bool known = old > 0.f && old < INFINITY;
    if (known) s = fmaxf(s, ceil_pow2(old));
    const float ratio = known ? __fdiv_rn(old, s) : 1.f;
    if (ratio != 1.f) {
      for (int i = sub; i < r.held; i += 2) {
        uint2 v = *reinterpret_cast<const uint2*>(out + i * row_bytes);
        uint16_t* h = reinterpret_cast<uint16_t*>(&v);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float2 f = e4m3x2_to_float2(h[t]);
          h[t] = __nv_cvt_float2_to_fp8x2(make_float2(f.x * ratio, f.y * ratio), __NV_SATFINITE, __NV_E4M3);
        }
        *reinterpret_cast<uint2*>(out + i * row_bytes) = v;
      }
    }
  }
  for (int i = sub; i < r.count; i += 2) {
    const uint4 v = *reinterpret_cast<const uint4*>(x + i * p.x_stride[kv]);
    *reinterpret_cast<uint2*>(out + (r.held + i) * row_bytes) = quant8_e4m3(v, s);
  }
  __syncwarp();
  if (lane == 0) *scale_at = s;
}

__global__ void __launch_bounds__(kStoreThreads) store_kv_blocks_kernel(const StoreBlocksParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t begin = int64_t(blockIdx.x) * kStoreWindow;
  __shared__ GroupRun runs[kStoreWindow];
  if (threadIdx.x < kStoreWindow) {
    runs[threadIdx.x] = begin + threadIdx.x < p.num_tokens ? run_at(p, begin + threadIdx.x) : GroupRun{0, 0, 0, 0};
  }
  __syncthreads();
  for (int i = warp; i < 2 * kStoreWindow; i += kStoreThreads / 32) {
    const GroupRun r = runs[i >> 1];
    if (r.count > 0) store_run(p, r, blockIdx.y, i & 1, lane);
  }
}

}  // namespace
}  // namespace hl

using namespace hl;

extern "C" int hl_store_kv_fp8_blocks(const void* key, const void* value, int64_t key_row_stride,
                                      int64_t value_row_stride, int64_t num_tokens, void* k_cache, void* v_cache,
                                      float* k_scales, float* v_scales, const int32_t* block_tables,
                                      int64_t bt_stride, int max_blocks_per_seq, const int32_t* context_lens,
                                      const int32_t* cu_seqlens_q, int num_seqs, int num_kv_heads, int head_dim,
                                      int block_size, int scale_block, int64_t num_blocks, void* stream) {
  clear_error();
  HL_CHECK_ARG(num_tokens >= 0 && num_tokens <= 0x7fffffff && num_seqs >= 0,
               "hl_store_kv_fp8_blocks: num_tokens or num_seqs out of range");
  HL_CHECK_ARG(head_dim == kBlockHeadDim, "hl_store_kv_fp8_blocks: head_dim %d != 128", head_dim);
  HL_CHECK_ARG(num_kv_heads > 0 && num_kv_heads <= 65535, "hl_store_kv_fp8_blocks: bad num_kv_heads");
  HL_CHECK_ARG(scale_block > 0 && scale_block % 64 == 0 && block_size > 0 && block_size % scale_block == 0,
               "hl_store_kv_fp8_blocks: scale_block must be a multiple of 64 that divides block_size");
  HL_CHECK_ARG(cu_seqlens_q || num_tokens == num_seqs,
               "hl_store_kv_fp8_blocks: without cu_seqlens_q there is one token per sequence");
  if (num_tokens == 0 || num_seqs == 0) return HL_OK;
  HL_CHECK_ARG(key && value && k_cache && v_cache && k_scales && v_scales && block_tables && context_lens,
               "hl_store_kv_fp8_blocks: null pointer");
  HL_CHECK_ARG(max_blocks_per_seq > 0 && bt_stride >= max_blocks_per_seq && num_blocks > 0,
               "hl_store_kv_fp8_blocks: bad block table or pool shape");
  const int64_t row = int64_t(num_kv_heads) * head_dim;
  HL_CHECK_ARG(key_row_stride >= row && value_row_stride >= row, "hl_store_kv_fp8_blocks: row stride < Hk*D");
  HL_CHECK_ARG(aligned16(key) && aligned16(value) && key_row_stride % 8 == 0 && value_row_stride % 8 == 0 &&
                   aligned16(k_cache) && aligned16(v_cache),
               "hl_store_kv_fp8_blocks: 16-byte alignment required");
  StoreBlocksParams p;
  p.x[0] = static_cast<const __nv_bfloat16*>(key);
  p.x[1] = static_cast<const __nv_bfloat16*>(value);
  p.x_stride[0] = key_row_stride;
  p.x_stride[1] = value_row_stride;
  p.cache[0] = static_cast<uint8_t*>(k_cache);
  p.cache[1] = static_cast<uint8_t*>(v_cache);
  p.scales[0] = k_scales;
  p.scales[1] = v_scales;
  p.num_tokens = num_tokens;
  p.block_tables = block_tables;
  p.bt_stride = bt_stride;
  p.max_blocks = max_blocks_per_seq;
  p.context_lens = context_lens;
  p.cu = cu_seqlens_q;
  p.num_seqs = num_seqs;
  p.num_kv_heads = num_kv_heads;
  p.block_size = block_size;
  p.scale_block = scale_block;
  p.num_blocks = num_blocks;
  const dim3 grid(unsigned((num_tokens + kStoreWindow - 1) / kStoreWindow), num_kv_heads);
  store_kv_blocks_kernel<<<grid, kStoreThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  HL_CHECK_LAUNCH("hl_store_kv_fp8_blocks");
  return HL_OK;
}
