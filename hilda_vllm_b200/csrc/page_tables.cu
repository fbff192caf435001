// Block tables and slot maps of a batch from request lengths, on the GPU.
//
// Device form of the allocation and bookkeeping that BlockManager.allocate_uncached and
// prefill_metadata do on the host (mini_vllm/engine/block_manager.py:58-80,
// mini_vllm/engine/model_runner.py:614-650).  Sequence b holds c_b tokens in the first
// have_b = ceil(c_b / BS) pages of its table row and gets n_b more:
//   need_b = ceil((c_b + n_b) / BS) (have_b when n_b = 0), both cut at the row's width;
//   its need_b - have_b new pages are the next ones of free_blocks, sequence after sequence;
//   token i of its n_b has position c_b + i and slot row[pos / BS] * BS + pos % BS.
// Whole numbers only; the bytes are the token arrays (12 B a token) and the table rows.
#include "hl_common.cuh"

namespace hl {
namespace {

constexpr int kTableThreads = 1024;
constexpr int kMaxTableSeqs = 4096;

struct TableParams {
  const int32_t* cached_lens;
  const int32_t* query_lens;
  int num_seqs;
  int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* free_blocks;
  int64_t num_free;
  int block_size;
  int64_t max_tokens;
  int32_t* cu_seqlens_q;
  int32_t* cu_seqlens_k;
  int32_t* context_lens;
  int64_t* positions;
  int32_t* slot_mapping;
  int32_t* status;
};

__device__ __forceinline__ int64_t cached(const TableParams& p, int b) {
  return p.cached_lens ? max(p.cached_lens[b], 0) : 0;
}

// Pages of `tokens` tokens, cut at the width of a table row.
__device__ __forceinline__ int64_t pages_of(const TableParams& p, int64_t tokens) {
  const int64_t n = (tokens + p.block_size - 1) / p.block_size;
  return n < p.max_blocks ? n : p.max_blocks;
}

// One thread block: prefix sums over the sequences, then the table rows.
__global__ void __launch_bounds__(kTableThreads) extend_tables_kernel(const TableParams p) {
  __shared__ int64_t s_start[kMaxTableSeqs];
  __shared__ int s_err;
  if (threadIdx.x == 0) {
    s_err = 0;
    int64_t q = 0, k = 0, pages = 0;
    p.cu_seqlens_q[0] = 0;
    p.cu_seqlens_k[0] = 0;
    for (int b = 0; b < p.num_seqs; ++b) {
      const int64_t c = cached(p, b), n = max(p.query_lens[b], 0);
      const int64_t have = pages_of(p, c), need = n > 0 ? pages_of(p, c + n) : have;
      s_start[b] = pages;
      q += n;
      k += c + n;
      pages += need - have;
      p.cu_seqlens_q[b + 1] = int32_t(q);
      p.cu_seqlens_k[b + 1] = int32_t(k);
      p.context_lens[b] = int32_t(c + n);
      if (n > 0 && c + n > int64_t(p.max_blocks) * p.block_size) s_err |= HL_TABLES_TOO_NARROW;
    }
    if (pages > p.num_free) s_err |= HL_TABLES_NO_PAGES;
    if (q > p.max_tokens) s_err |= HL_TABLES_TOO_MANY_TOKENS;
    p.status[0] = int32_t(pages < p.num_free ? pages : p.num_free);
    p.status[1] = s_err;
  }
  __syncthreads();
  for (int b = threadIdx.x >> 5; b < p.num_seqs; b += kTableThreads / 32) {
    const int64_t c = cached(p, b), n = max(p.query_lens[b], 0);
    const int64_t have = pages_of(p, c), need = n > 0 ? pages_of(p, c + n) : have;
    for (int64_t j = have + (threadIdx.x & 31); j < p.max_blocks; j += 32) {
      const int64_t at = s_start[b] + j - have;
      p.block_tables[b * p.bt_stride + j] = j < need && at < p.num_free ? p.free_blocks[at] : -1;
    }
  }
}

// One thread per token: its sequence by binary search in cu_seqlens_q.
__global__ void __launch_bounds__(256) token_slots_kernel(const TableParams p) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.max_tokens) return;
  int lo = 0, hi = p.num_seqs;  // first sequence whose end lies behind i
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_seqlens_q[mid + 1] > i) hi = mid; else lo = mid + 1;
  }
  int64_t pos = 0;
  int32_t slot = -1;
  if (lo < p.num_seqs) {
    pos = cached(p, lo) + i - p.cu_seqlens_q[lo];
    const int64_t j = pos / p.block_size;
    const int64_t page = j < p.max_blocks ? p.block_tables[lo * p.bt_stride + j] : -1;
    const int64_t s = page * p.block_size + pos % p.block_size;
    if (page >= 0 && s <= 0x7fffffff) slot = int32_t(s);
  }
  p.positions[i] = pos;
  p.slot_mapping[i] = slot;
}

}  // namespace
}  // namespace hl

using namespace hl;

extern "C" int hl_extend_block_tables(const int32_t* cached_lens, const int32_t* query_lens, int num_seqs,
                                      int32_t* block_tables, int64_t bt_stride, int max_blocks,
                                      const int32_t* free_blocks, int64_t num_free, int block_size,
                                      int64_t max_tokens, int32_t* cu_seqlens_q, int32_t* cu_seqlens_k,
                                      int32_t* context_lens, int64_t* positions, int32_t* slot_mapping,
                                      int32_t* status, void* stream) {
  clear_error();
  HL_CHECK_ARG(num_seqs >= 0 && num_seqs <= kMaxTableSeqs, "hl_extend_block_tables: num_seqs not in [0, %d]",
               kMaxTableSeqs);
  HL_CHECK_ARG(block_size > 0, "hl_extend_block_tables: block_size <= 0");
  HL_CHECK_ARG(max_blocks > 0 && bt_stride >= max_blocks, "hl_extend_block_tables: bad block table width");
  HL_CHECK_ARG(num_free >= 0 && max_tokens >= 0 && max_tokens <= 0x7fffffff,
               "hl_extend_block_tables: num_free or max_tokens out of range");
  HL_CHECK_ARG(cu_seqlens_q && cu_seqlens_k && status && (max_tokens == 0 || (positions && slot_mapping)) &&
                   (num_free == 0 || free_blocks) &&
                   (num_seqs == 0 || (query_lens && block_tables && context_lens)),
               "hl_extend_block_tables: null pointer");
  const TableParams p{cached_lens, query_lens, num_seqs, block_tables, bt_stride, max_blocks, free_blocks, num_free,
                      block_size, max_tokens, cu_seqlens_q, cu_seqlens_k, context_lens, positions, slot_mapping,
                      status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  extend_tables_kernel<<<1, kTableThreads, 0, s>>>(p);
  HL_CHECK_LAUNCH("hl_extend_block_tables");
  if (max_tokens > 0) {
    token_slots_kernel<<<unsigned((max_tokens + 255) / 256), 256, 0, s>>>(p);
    HL_CHECK_LAUNCH("hl_extend_block_tables");
  }
  return HL_OK;
}
