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
//
// The rows of a call that fall into one group are a run, and consecutive rows.  A thread block looks
// for the runs that start in its window of rows, for one head and K or V.  A run of up to 16 rows is
// one warp's, a longer one the whole block's; either way the rows are loaded once, all loads in
// flight together, and stay in registers between the maximum and the rounding.  HBM bounds long runs
// (3 B an element), the chain of reads (sequence, table, scale) a decode step.
#include "kv_blocks.cuh"

namespace hl {
namespace {

constexpr int kStoreThreads = 256;
constexpr int kStoreWarps = kStoreThreads / 32;
constexpr int kMaxWindow = 64;
constexpr int kWarpRun = 16;         // longest run of one warp
constexpr int kMaxSharedSeqs = 4096; // cu_seqlens_q of up to so many sequences is searched in shared memory

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
  int window;  // rows whose runs one thread block starts
};

// The rows of a call that fall into one group: rows [row, row + count) go to offsets
// [held, held + count) of the group whose first slot is `slot0`.  count = 0: none.
struct GroupRun {
  int64_t row, slot0;
  int count, held;
};

// The run that starts at row i; count 0 where i is inside a run or belongs to no sequence.
// cu: the prefix sums, or nullptr for one row per sequence.
__device__ GroupRun run_at(const StoreBlocksParams& p, const int32_t* cu, int64_t i) {
  GroupRun r{i, 0, 0, 0};
  int64_t first = i, end = i + 1;  // rows of i's sequence
  int b = int(i);
  if (cu) {
    int lo = 0, hi = p.num_seqs;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid + 1] > i) hi = mid; else lo = mid + 1;
    }
    b = lo;
    if (b >= p.num_seqs) return r;
    first = cu[b];
    end = cu[b + 1];
    if (first > i || first < 0) return r;
  }
  const int64_t pos = int64_t(p.context_lens[b]) - (end - i);
  if (pos < 0) return r;
  const unsigned at = unsigned(pos);  // < 2^31
  const unsigned j = at / unsigned(p.block_size), off = at - j * unsigned(p.block_size);
  const unsigned held = off % unsigned(p.scale_block);
  if (j >= unsigned(p.max_blocks) || (held != 0 && i != first)) return r;
  const int64_t page = p.block_tables[b * p.bt_stride + j];
  if (page < 0 || page >= p.num_blocks) return r;
  r.held = int(held);
  r.slot0 = page * p.block_size + off - held;
  r.count = int(min(int64_t(p.scale_block) - held, min(end, p.num_tokens) - i));
  return r;
}

// Largest finite |x| of a vector, as a bf16 bit pattern; patterns from 0x7f80 on are infinities and NaN.
__device__ __forceinline__ uint32_t abs_bits(uint4 v) {
  return __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
}
__device__ __forceinline__ uint32_t finite_bits(uint4 v) {
  auto keep = [](uint32_t w) {
    w &= 0x7fff7fffu;
    if ((w & 0xffffu) >= 0x7f80u) w &= 0xffff0000u;
    if ((w >> 16) >= 0x7f80u) w &= 0xffffu;
    return w;
  };
  return __vmaxu2(__vmaxu2(keep(v.x), keep(v.y)), __vmaxu2(keep(v.z), keep(v.w)));
}
__device__ __forceinline__ uint32_t larger_half(uint32_t w) { return max(w & 0xffffu, w >> 16); }

__device__ __forceinline__ uint2 scale_to_e4m3(uint4 v, float inverse) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t q[4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
    q[t] = __nv_cvt_float2_to_fp8x2(make_float2(bf16lo(w[t]) * inverse, bf16hi(w[t]) * inverse), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
}

// Rounds the rows from before to the new scale, `rows` of them at a time.
__device__ __forceinline__ void rescale_rows(uint8_t* out, int64_t row_bytes, int held, float ratio, int row, int rows) {
  for (int i = row; i < held; i += rows) {
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

// A run's place for one head of K or V.
struct RunPlace {
  const __nv_bfloat16* x;
  uint8_t* out;      // first row of the group
  float* scale;
  __device__ RunPlace(const StoreBlocksParams& p, const GroupRun& r, int kv, int head)
      : x(p.x[kv] + r.row * p.x_stride[kv] + head * kBlockHeadDim),
        out(p.cache[kv] + (r.slot0 * p.num_kv_heads + head) * kBlockHeadDim),
        scale(p.scales[kv] + r.slot0 / p.scale_block * p.num_kv_heads + head) {}
};

// The group's new scale from the largest new value and the old scale (ignored unless rows are held);
// ratio: what the rows from before are multiplied by.
__device__ __forceinline__ float new_scale(uint32_t amax_bits, bool held, float old, float& ratio) {
  float s = scale_for(__uint_as_float(amax_bits << 16));
  ratio = 1.f;
  if (held && old > 0.f && old < INFINITY) {
    s = fmaxf(s, ceil_pow2(old));
    ratio = __fdiv_rn(old, s);
  }
  return s;
}
// 1 / s of a power of two between 2^-100 and 2^126.
__device__ __forceinline__ float inverse_pow2(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// One warp, a run of at most kWarpRun rows: 16 lanes per row.
__device__ void store_warp_run(const StoreBlocksParams& p, const GroupRun& r, int kv, int head, int lane) {
  const RunPlace at(p, r, kv, head);
  const int row = lane >> 4, e0 = (lane & 15) * 8;
  const int64_t row_bytes = int64_t(p.num_kv_heads) * kBlockHeadDim;
  const float old = r.held ? *at.scale : 0.f;
  uint4 v[kWarpRun / 2];
#pragma unroll
  for (int k = 0; k < kWarpRun / 2; ++k)
    v[k] = 2 * k + row < r.count ? __ldg(reinterpret_cast<const uint4*>(at.x + (2 * k + row) * p.x_stride[kv] + e0))
                                 : make_uint4(0, 0, 0, 0);
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < kWarpRun / 2; ++k) m = __vmaxu2(m, abs_bits(v[k]));
  uint32_t amax = __reduce_max_sync(0xffffffffu, larger_half(m));
  if (amax >= 0x7f80u) {
    m = 0;
#pragma unroll
    for (int k = 0; k < kWarpRun / 2; ++k) m = __vmaxu2(m, finite_bits(v[k]));
    amax = __reduce_max_sync(0xffffffffu, larger_half(m));
  }
  float ratio;
  const float s = new_scale(amax, r.held > 0, old, ratio), inverse = inverse_pow2(s);
#pragma unroll
  for (int k = 0; k < kWarpRun / 2; ++k)
    if (2 * k + row < r.count)
      *reinterpret_cast<uint2*>(at.out + (r.held + 2 * k + row) * row_bytes + e0) = scale_to_e4m3(v[k], inverse);
  if (ratio != 1.f) rescale_rows(at.out + e0, row_bytes, r.held, ratio, row, 2);
  if (lane == 0) *at.scale = s;
}

// The whole block, a longer run: 16 rows a pass, up to P passes in registers; what is longer is read
// twice.
template <int P>
__device__ void store_block_run(const StoreBlocksParams& p, const GroupRun& r, int kv, int head, uint32_t* warp_max) {
  const RunPlace at(p, r, kv, head);
  const int row = threadIdx.x >> 4, e0 = (threadIdx.x & 15) * 8;
  const int64_t row_bytes = int64_t(p.num_kv_heads) * kBlockHeadDim;
  const float old = r.held ? *at.scale : 0.f;
  constexpr int kRows = kStoreThreads / 16;
  uint4 v[P];
  auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < P; ++k)
      v[k] = i0 + k * kRows + row < r.count
                 ? __ldg(reinterpret_cast<const uint4*>(at.x + (i0 + k * kRows + row) * p.x_stride[kv] + e0))
                 : make_uint4(0, 0, 0, 0);
  };
  auto block_max = [&](uint32_t m) {
    m = __reduce_max_sync(0xffffffffu, larger_half(m));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int w = 0; w < kStoreWarps; ++w) m = max(m, warp_max[w]);
    return m;
  };
  auto run_max = [&](auto bits) {
    uint32_t m = 0;
    for (int i0 = 0; i0 < r.count; i0 += P * kRows) {
      if (i0 > 0 || r.count > P * kRows) load(i0);
#pragma unroll
      for (int k = 0; k < P; ++k) m = __vmaxu2(m, bits(v[k]));
    }
    return block_max(m);
  };
  load(0);
  uint32_t amax = run_max([](uint4 x) { return abs_bits(x); });
  if (amax >= 0x7f80u) amax = run_max([](uint4 x) { return finite_bits(x); });
  float ratio;
  const float s = new_scale(amax, r.held > 0, old, ratio), inverse = inverse_pow2(s);
  for (int i0 = 0; i0 < r.count; i0 += P * kRows) {
    if (r.count > P * kRows) load(i0);
#pragma unroll
    for (int k = 0; k < P; ++k)
      if (i0 + k * kRows + row < r.count)
        *reinterpret_cast<uint2*>(at.out + (r.held + i0 + k * kRows + row) * row_bytes + e0) = scale_to_e4m3(v[k], inverse);
  }
  if (ratio != 1.f) rescale_rows(at.out + e0, row_bytes, r.held, ratio, row, kRows);
  if (threadIdx.x == 0) *at.scale = s;
}

template <int P>
__global__ void __launch_bounds__(kStoreThreads) store_kv_blocks_kernel(const __grid_constant__ StoreBlocksParams p) {
  extern __shared__ int32_t cu_shared[];
  __shared__ GroupRun runs[kMaxWindow];
  __shared__ int small[kMaxWindow], large[kMaxWindow], num_small, num_large;
  __shared__ uint32_t warp_max[kStoreWarps];
  const int kv = blockIdx.z, head = blockIdx.y;
  const int64_t begin = int64_t(blockIdx.x) * p.window;
  const int32_t* cu = p.cu;
  if (cu && p.num_seqs <= kMaxSharedSeqs) {
    for (int i = threadIdx.x; i <= p.num_seqs; i += kStoreThreads) cu_shared[i] = cu[i];
    cu = cu_shared;
  }
  if (threadIdx.x == 0) num_small = num_large = 0;
  __syncthreads();
  if (threadIdx.x < p.window && begin + threadIdx.x < p.num_tokens) {
    const GroupRun r = run_at(p, cu, begin + threadIdx.x);
    runs[threadIdx.x] = r;
    if (r.count > kWarpRun) large[atomicAdd(&num_large, 1)] = threadIdx.x;
    else if (r.count > 0) small[atomicAdd(&num_small, 1)] = threadIdx.x;
  }
  __syncthreads();
  for (int i = threadIdx.x >> 5; i < num_small; i += kStoreWarps)
    store_warp_run(p, runs[small[i]], kv, head, threadIdx.x & 31);
  for (int i = 0; i < num_large; ++i) store_block_run<P>(p, runs[large[i]], kv, head, warp_max);
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
  // Windows of 64 rows, which start about one run each in a prefill; of 8, a warp for each row of a
  // decode step, where those would leave SMs idle.
  const int64_t wide = (num_tokens + kMaxWindow - 1) / kMaxWindow;
  p.window = wide * num_kv_heads * 2 >= 2 * 148 ? kMaxWindow : kStoreWarps;
  const dim3 grid(unsigned((num_tokens + p.window - 1) / p.window), num_kv_heads, 2);
  const size_t shared = cu_seqlens_q && num_seqs <= kMaxSharedSeqs ? (num_seqs + 1) * sizeof(int32_t) : 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (scale_block <= 64)
    store_kv_blocks_kernel<4><<<grid, kStoreThreads, shared, s>>>(p);
  else if (scale_block <= 128)
    store_kv_blocks_kernel<8><<<grid, kStoreThreads, shared, s>>>(p);
  else
    store_kv_blocks_kernel<16><<<grid, kStoreThreads, shared, s>>>(p);
  HL_CHECK_LAUNCH("hl_store_kv_fp8_blocks");
  return HL_OK;
}
