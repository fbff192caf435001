// KV store into the block-scaled 8-bit cache: the scale of a group (scale_block consecutive tokens
// of a page, one head) follows the data instead of being calibrated beforehand
// (mini_vllm/layers/attention.py:51-52,133 stores e4m3 without scales).
//
// Per group and head, with a = max |x| over this call's new rows (finite values) and s_old the
// group's scale if it holds rows from before this call (0 otherwise):
//   s = max(s_old, smallest power of two with a / s <= 448, 2^-100)
//   rows from before: e4m3(q * s_old / s);   new rows: e4m3(x / s), saturating;   scale := s.
// A scale of this store's own is a power of two, and x / s one exact bf16 product.  A caller's own may be
// any; while it is the larger one, the new rows are divided in fp32.
// Sequence b's rows cu[b] .. cu[b+1]-1 are its tokens context_lens[b] - n .. context_lens[b]-1, so
// "rows from before" are the tokens of the group in front of its first new one, whatever the page
// held for an earlier owner.
//
// The rows of a call that fall into one group are a run, and consecutive rows.  A thread block looks
// for the runs that start in its window of rows and stores them for several items, an item being one
// head of K or of V.  A warp holds up to 2 L rows of an item in registers between the maximum and the
// rounding, L loads a lane in flight, and no warp waits for another but for the maximum of a longer
// run, which two or four warps share.  HBM bounds a prefill (3 B an element): L = 32, twelve warps of
// 16 KB an SM, or 16 warps of 8 KB where that evens out a short one.  A decode step is bound by its
// chain of reads (sequence, table, scale): L = 8, more and smaller warps.
#include "dependent_launch.cuh"
#include "kv_blocks.cuh"

namespace hl {
namespace {

constexpr int kStoreThreads = 128;
constexpr int kStoreWarps = kStoreThreads / 32;
constexpr int kMaxWindow = 256;
constexpr int kSharedSeqs = 512;  // the lengths of up to so many sequences are searched in shared memory

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
  int items;   // heads of K and V that it stores, of 2 Hk
};

// The rows of a call that fall into one group: rows [row, row + count) go to offsets
// [held, held + count) of the group whose first slot is `slot0`.  count = 0: none.
struct GroupRun {
  int64_t row, slot0, group;  // group: slot0 / scale_block
  int count, held;
};

// The run that starts at row i; count 0 where i is inside a run or belongs to no sequence.
// lens: the prefix sums (nullptr: one row per sequence) and context lengths of the sequences from
// `base` on; i lies in one of lo .. hi or in none.
struct Lengths {
  const int32_t *cu, *context;
  int base, lo, hi;
};
__device__ GroupRun run_at(const StoreBlocksParams& p, const Lengths& lens, int64_t i) {
  GroupRun r{i, 0, 0, 0, 0};
  int64_t first = i, end = i + 1;  // rows of i's sequence
  int b = int(i);
  if (lens.cu) {
    int lo = lens.lo, hi = lens.hi;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (lens.cu[mid + 1 - lens.base] > i) hi = mid; else lo = mid + 1;
    }
    b = lo;
    if (b >= p.num_seqs) return r;
    first = lens.cu[b - lens.base];
    end = lens.cu[b + 1 - lens.base];
    if (first > i || first < 0 || end <= i) return r;
  }
  const int64_t pos = int64_t(lens.context[b - lens.base]) - (end - i);
  if (pos < 0) return r;
  const unsigned at = unsigned(pos);  // < 2^31
  const unsigned j = at / unsigned(p.block_size), off = at - j * unsigned(p.block_size);
  const unsigned held = off % unsigned(p.scale_block);
  if (j >= unsigned(p.max_blocks) || (held != 0 && i != first)) return r;
  const int64_t page = p.block_tables[b * p.bt_stride + j];
  if (page < 0 || page >= p.num_blocks) return r;
  r.held = int(held);
  r.slot0 = page * p.block_size + off - held;
  r.group = page * (p.block_size / p.scale_block) + off / unsigned(p.scale_block);
  r.count = int(min(int64_t(p.scale_block) - held, min(end, p.num_tokens) - i));
  return r;
}

// The first sequence that ends behind row i (num_seqs: none), by the lanes of a warp together.
__device__ int warp_sequence_of(const StoreBlocksParams& p, int64_t i, int lane) {
  int lo = 0, n = p.num_seqs;  // it is one of lo .. lo + n
  while (n > 0) {
    const int step = (n + 31) / 32, at = min((lane + 1) * step, n) - 1;
    const int k = __popc(__ballot_sync(0xffffffffu, p.cu[lo + at + 1] <= i));
    if (k == 32) return lo + n;
    const int next = min(k * step, n);
    n = min((k + 1) * step, n) - 1 - next;
    lo += next;
  }
  return lo;
}

// Running maximum of |x| over pairs of bf16 values: NaN is passed over, infinities are not.
__device__ __forceinline__ void raise_abs(__nv_bfloat162& m, uint4 v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int t = 0; t < 4; ++t) m = __hmax2(m, __habs2(h[t]));
}
// The same over finite values only.
__device__ __forceinline__ void raise_finite(__nv_bfloat162& m, uint4 v) {
  auto keep = [](uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
    return w;
  };
  raise_abs(m, make_uint4(keep(v.x), keep(v.y), keep(v.z), keep(v.w)));
}
// Larger half of the warp's maxima, as bits: at least 0x7f80 if a value is infinite.
__device__ __forceinline__ uint32_t warp_max_bits(__nv_bfloat162 m) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(&m);
  return __reduce_max_sync(0xffffffffu, max(w & 0xffffu, w >> 16));
}

// e4m3(x * inverse), inverse a power of two: exact in bf16 but for results below 2^-126, which round to
// zero either way.
__device__ __forceinline__ uint2 scale_to_e4m3(uint4 v, __nv_bfloat162 inverse) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  uint32_t q[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const __nv_bfloat162 y = __hmul2(h[t], inverse);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&y);
    q[t] = __nv_cvt_float2_to_fp8x2(make_float2(bf16lo(w), bf16hi(w)), __NV_SATFINITE, __NV_E4M3);
  }
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
        scale(p.scales[kv] + r.group * p.num_kv_heads + head) {}
};

// The group's new scale from the largest new value and the old scale (ignored unless rows are held);
// ratio: what the rows from before are multiplied by.
__device__ __forceinline__ float new_scale(uint32_t amax_bits, bool held, float old, float& ratio) {
  float s = scale_for(__uint_as_float(amax_bits << 16));
  ratio = 1.f;
  if (held && old >= 0.f && old < INFINITY) {
    s = fmaxf(s, old);
    ratio = __fdiv_rn(old, s);
  }
  return s;
}
// s is a power of two with a normal inverse (s >= 2^-100).
__device__ __forceinline__ bool has_inverse(float s) { return (__float_as_uint(s) & 0x7fffffu) == 0 && s <= 0x1p126f; }
// Its inverse.
__device__ __forceinline__ __nv_bfloat162 inverse_pow2(float s) {
  return __float2bfloat162_rn(__uint_as_float((254u << 23) - __float_as_uint(s)));
}

// M warps, one run of one item: warp `sub` of them holds rows 2 L sub .. 2 L (sub + 1) - 1, two a load; of
// a run that is longer than 2 L M rows the same of every 2 L M, which are then read twice.  False, with
// nothing written, where the group keeps an old scale that has no exact inverse.
template <int M, int L>
__device__ __forceinline__ bool store_run(const StoreBlocksParams& p, const GroupRun& r, int kv, int head, int sub,
                                          int team, int lane, uint32_t* team_max) {
  constexpr int kHeldRows = 2 * L;
  const RunPlace at(p, r, kv, head);
  const int row = sub * kHeldRows + (lane >> 4), e0 = (lane & 15) * 8;
  const int64_t row_bytes = int64_t(p.num_kv_heads) * kBlockHeadDim, step = 2 * p.x_stride[kv];
  const float old = r.held ? *at.scale : 0.f;
  const bool twice = r.count > M * kHeldRows;
  uint4 v[L];
  auto load = [&](int i0) {
    const __nv_bfloat16* x = at.x + (i0 + row) * p.x_stride[kv] + e0;
    if (i0 + (sub + 1) * kHeldRows <= r.count) {
#pragma unroll
      for (int k = 0; k < L; ++k) v[k] = load16(x + k * step);
    } else {
#pragma unroll
      for (int k = 0; k < L; ++k)
        v[k] = i0 + row + 2 * k < r.count ? load16(x + k * step) : make_uint4(0, 0, 0, 0);
    }
  };
  auto run_max = [&](auto raise) {
    __nv_bfloat162 m = __float2bfloat162_rn(0.f);
    for (int i0 = 0; i0 < r.count; i0 += M * kHeldRows) {
      if (twice) load(i0);
#pragma unroll
      for (int k = 0; k < L; ++k) raise(m, v[k]);
    }
    uint32_t w = warp_max_bits(m);
    if constexpr (M > 1) {
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * M) : "memory");  // the last maxima have been read
      if (lane == 0) team_max[sub] = w;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * M) : "memory");
#pragma unroll
      for (int i = 0; i < M; ++i) w = max(w, team_max[i]);
    }
    return w;
  };
  if (!twice) load(0);
  uint32_t amax = run_max([](__nv_bfloat162& m, uint4 x) { raise_abs(m, x); });
  if (amax >= 0x7f80u) amax = run_max([](__nv_bfloat162& m, uint4 x) { raise_finite(m, x); });
  float ratio;
  const float s = new_scale(amax, r.held > 0, old, ratio);
  if (!has_inverse(s)) return false;  // s is the old one: what is written below but for the new rows stays
  const __nv_bfloat162 inverse = inverse_pow2(s);
  for (int i0 = 0; i0 < r.count; i0 += M * kHeldRows) {
    if (twice) load(i0);
    uint8_t* out = at.out + (r.held + i0 + row) * row_bytes + e0;
#pragma unroll
    for (int k = 0; k < L; ++k)
      if (i0 + row + 2 * k < r.count) *reinterpret_cast<uint2*>(out + 2 * k * row_bytes) = scale_to_e4m3(v[k], inverse);
  }
  if (ratio != 1.f) rescale_rows(at.out + e0, row_bytes, r.held, ratio, 2 * sub + (lane >> 4), 2 * M);
  if (sub == 0 && lane == 0) *at.scale = s;
  return true;
}

// The rows of a run whose group keeps an old scale without an exact inverse, by M warps.  Apart from
// store_run, whose loop would pay for the divisions with registers.
template <int M>
__device__ __forceinline__ void store_divided(const StoreBlocksParams& p, const GroupRun& r, int kv, int head, int sub, int lane) {
  if (r.held == 0) return;
  const RunPlace at(p, r, kv, head);
  const float s = *at.scale;
  if (has_inverse(s)) return;
  const int e0 = (lane & 15) * 8;
  const int64_t row_bytes = int64_t(p.num_kv_heads) * kBlockHeadDim;
  for (int i = 2 * sub + (lane >> 4); i < r.count; i += 2 * M) {
    const uint4 v = load16(at.x + i * p.x_stride[kv] + e0);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t q[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
      q[t] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(bf16lo(w[t]), s), __fdiv_rn(bf16hi(w[t]), s)), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint2*>(at.out + (r.held + i) * row_bytes + e0) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
  }
}

template <int M, int L>
__global__ void __launch_bounds__(kStoreThreads, L > 16 ? 3 : L > 8 ? 4 : 8) store_kv_blocks_kernel(const __grid_constant__ StoreBlocksParams p) {
  __shared__ int32_t lens_shared[2 * kSharedSeqs + 1];  // cu, context
  __shared__ int bounds[2];
  __shared__ GroupRun runs[kMaxWindow];
  __shared__ int found[kMaxWindow], num_found;
  __shared__ uint32_t team_max[kStoreWarps / M][M];
  const int item0 = blockIdx.y * p.items, items = min(p.items, 2 * p.num_kv_heads - item0);
  const int64_t begin = int64_t(blockIdx.x) * p.window;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  dependent_start();
  const int window = int(min(int64_t(p.window), p.num_tokens - begin));
  Lengths lens{p.cu, p.context_lens, 0, 0, p.num_seqs};
  if (p.cu) {
    int seqs = p.num_seqs;
    if (seqs > kSharedSeqs) {  // those of the window
      if (warp < 2) {
        const int b = warp_sequence_of(p, warp == 0 ? begin : begin + window - 1, lane);
        if (lane == 0) bounds[warp] = b;
      }
      __syncthreads();
      lens.lo = bounds[0];
      lens.hi = bounds[1];
      seqs = min(lens.hi + 1, p.num_seqs) - lens.lo;
    }
    if (seqs <= kSharedSeqs) {
      for (int i = threadIdx.x; i <= seqs; i += kStoreThreads) {
        lens_shared[i] = p.cu[lens.lo + i];
        if (i < seqs) lens_shared[kSharedSeqs + 1 + i] = p.context_lens[lens.lo + i];
      }
      lens.cu = lens_shared;
      lens.context = lens_shared + kSharedSeqs + 1;
      lens.base = lens.lo;
    }
  }
  if (threadIdx.x == 0) num_found = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < window; i += kStoreThreads) {
    const GroupRun r = run_at(p, lens, begin + i);
    runs[i] = r;
    if (r.count > 0) found[atomicAdd(&num_found, 1)] = i;
  }
  __syncthreads();
  bool stored = true;  // the same in all warps of a team
  for (int i = warp / M; i < num_found * items; i += kStoreWarps / M) {
    const int item = item0 + i % items;
    stored &= store_run<M, L>(p, runs[found[i / items]], item & 1, item >> 1, warp % M, warp / M, lane, team_max[warp / M]);
  }
  if (stored) return;
  if constexpr (M > 1)  // the team's scales are written
    asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / M), "n"(32 * M) : "memory");
  else
    __syncwarp();
  for (int i = warp / M; i < num_found * items; i += kStoreWarps / M) {
    const int item = item0 + i % items;
    store_divided<M>(p, runs[found[i / items]], item & 1, item >> 1, warp % M, lane);
  }
}

template <int M, int L>
cudaError_t launch_store_blocks(StoreBlocksParams& p, int64_t window, int64_t items, cudaStream_t stream) {
  p.window = int(window);
  p.items = int(items);
  const dim3 grid(unsigned((p.num_tokens + window - 1) / window), unsigned((2 * p.num_kv_heads + items - 1) / items));
  return launch_dependent(store_kv_blocks_kernel<M, L>, grid, kStoreThreads, 0, 1, stream, p);
}

// Blocks of kTeams teams of M warps: windows that start one run on average (more where a run has fewer
// items than the block teams), each team one item of it, more where that still makes kTeams rounds of all
// warps that the GPU holds at a time.  A block of one team of light warps (L = 16, M = 4) takes two items at
// least, for one does not pay for the lookup of its run (64 sequences of 250, 8 heads: 20.3 us, 22.8 with one
// item; 16 of 500: 9.5 and 10.7; but 2 heads: 8.1 and 6.6).
template <int M, int L>
cudaError_t launch_store(StoreBlocksParams& p, int64_t rows, int64_t runs, cudaStream_t stream) {
  constexpr int kTeams = kStoreWarps / M, kPerSm = L > 16 ? 3 : L > 8 ? 4 : 8, kLeast = L == 16 && M == 4 ? 2 : kTeams;
  const int64_t all = 2 * int64_t(p.num_kv_heads), rounds = runs * all / (kStoreWarps * kPerSm * 148);
  int64_t items = rounds > kLeast ? rounds / kTeams * kTeams : kLeast;
  items = items > all ? all : items;
  const int64_t window = rows * (kTeams > items ? kTeams / items : 1);
  return launch_store_blocks<M, L>(p, window < kMaxWindow ? window : kMaxWindow, items, stream);
}

// By the rows of an average run, as many registers and warps as hold it (128 sequences of 16 rows,
// T 128: 6.7 us, with the registers for whole groups 34; 4096 decode tokens: 42 us, one item at a time
// and all lengths in every block 124).  Up to three rounds of whole groups on the GPU, more and smaller
// pieces even the SMs' shares out: twice the warps a run, half the loads each (4096 tokens, 8 heads:
// 7.0 -> 5.9 us; 8195: 17.9 -> 16.5; 64 sequences of 100 to 400: 31 -> 27; but 65536: 67 -> 70 to 74).
cudaError_t launch_store_by_runs(StoreBlocksParams& p, cudaStream_t stream) {
  const int64_t group = p.scale_block, all = 2 * int64_t(p.num_kv_heads);
  int64_t runs = (p.num_tokens + group - 1) / group + p.num_seqs;
  runs = runs < p.num_tokens ? runs : p.num_tokens;
  int64_t rows = (p.num_tokens + runs - 1) / runs;
  if (10 * rows > 9 * group) rows = group;  // whole groups: a window each
  const bool few = runs * all <= 3 * 12 * 148;
  if (rows <= 16) return launch_store<1, 8>(p, rows, runs, stream);
  if (rows <= 32) return launch_store<1, 16>(p, rows, runs, stream);
  if (rows <= 64) return few ? launch_store<2, 16>(p, rows, runs, stream) : launch_store<1, 32>(p, rows, runs, stream);
  if (rows <= 128) return few ? launch_store<4, 16>(p, rows, runs, stream) : launch_store<2, 32>(p, rows, runs, stream);
  return launch_store<4, 32>(p, rows, runs, stream);
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
  HL_CHECK_ARG(num_kv_heads > 0 && num_kv_heads <= 32767, "hl_store_kv_fp8_blocks: bad num_kv_heads");
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = launch_store_by_runs(p, s);
  if (e != cudaSuccess) {
    set_error("hl_store_kv_fp8_blocks: launch failed: %s", cudaGetErrorString(e));
    return HL_ERR_CUDA;
  }
  return HL_OK;
}
