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
//
// One launch.  Bound by latency up to some 100k tokens: lengths -> prefix sums -> free list or table ->
// slots are three dependent reads.  So every thread block scans all lengths itself (at most 4096, from
// L2) instead of waiting for one that does, and no thread reads a table entry that another writes: a
// token on a new page takes the page's id from the free list, as the thread that writes the row does.
#include "dependent_launch.cuh"

namespace hl {
namespace {

constexpr int kTableThreads = 256;
constexpr int kTokensPerThread = 4;
constexpr int kMaxTableSeqs = 4096;
constexpr int kMaxTableBlocks = 296;  // two per SM: more blocks would only repeat the scan

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
  bool wide;  // positions and slot_mapping are aligned for 16-byte stores
};

__device__ __forceinline__ unsigned cached(const TableParams& p, int b) {
  return p.cached_lens ? max(p.cached_lens[b], 0) : 0;
}

// Pages of `tokens` tokens, cut at the width of a table row.
__device__ __forceinline__ unsigned pages_of(const TableParams& p, unsigned tokens) {
  return min(tokens / p.block_size + (tokens % p.block_size != 0), unsigned(p.max_blocks));
}

// Where a sequence's entry stands in shared memory: threads that read 2, 4, 8 or 16 neighbours each meet no
// bank conflicts.
__host__ __device__ __forceinline__ int slot_of(int b) { return b + (b >> 5); }

struct Sums {
  int64_t query, context, pages;
  __device__ __forceinline__ Sums operator+(const Sums& o) const {
    return {query + o.query, context + o.context, pages + o.pages};
  }
};

__device__ __forceinline__ Sums shuffle_up(const Sums& s, int by) {
  return {__shfl_up_sync(0xffffffffu, s.query, by), __shfl_up_sync(0xffffffffu, s.context, by),
          __shfl_up_sync(0xffffffffu, s.pages, by)};
}

__device__ __forceinline__ int32_t to_int32(int64_t x) { return int32_t(min(x, int64_t(0x7fffffff))); }

// Position and slot of token i, which belongs to sequence b.
__device__ __forceinline__ void place_token(const TableParams& p, int i, int b, const int32_t* first_token,
                                            const int32_t* first_page, int64_t& pos, int32_t& slot) {
  const unsigned c = cached(p, b), at = c + unsigned(i - first_token[slot_of(b)]);
  const unsigned j = at / p.block_size, off = at - j * p.block_size;
  pos = at;
  slot = -1;
  int64_t page = -1;
  if (j < unsigned(p.max_blocks)) {
    const unsigned have = pages_of(p, c);
    if (j < have) {
      page = p.block_tables[b * p.bt_stride + j];
    } else {
      const int64_t k = int64_t(first_page[slot_of(b)]) + j - have;
      if (k < p.num_free) page = p.free_blocks[k];
    }
  }
  const int64_t s = page * p.block_size + off;
  if (page >= 0 && s <= 0x7fffffff) slot = int32_t(s);
}

__global__ void __launch_bounds__(kTableThreads) extend_tables_kernel(const TableParams p) {
  extern __shared__ int32_t table_smem[];
  int32_t* first_token = table_smem;                              // [num_seqs + 1], at slot_of
  int32_t* first_page = table_smem + slot_of(p.num_seqs) + 1;     // [num_seqs] index into free_blocks, at slot_of
  __shared__ Sums warp_sums[kTableThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  dependent_start();
  // ---- prefix sums over the sequences
  // The lengths first, in wide reads, to where their sums will stand (4096 sequences: 16.9 us, 26.7 with
  // each thread's lengths read from L2 one after another).
  for (int b = threadIdx.x; b < p.num_seqs; b += kTableThreads) {
    first_token[slot_of(b)] = max(p.query_lens[b], 0);
    first_page[slot_of(b)] = int(cached(p, b));
  }
  __syncthreads();
  const int per = (p.num_seqs + kTableThreads - 1) / kTableThreads;
  const int b0 = min(int(threadIdx.x) * per, p.num_seqs), b1 = min(b0 + per, p.num_seqs);
  auto of = [&](int b) {
    const unsigned c = first_page[slot_of(b)], n = first_token[slot_of(b)];
    return Sums{n, int64_t(c) + n, n ? pages_of(p, c + n) - pages_of(p, c) : 0};
  };
  Sums mine{0, 0, 0};
  for (int b = b0; b < b1; ++b) mine = mine + of(b);
  Sums upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sums v = shuffle_up(upto, o);
    if (lane >= o) upto = upto + v;
  }
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  Sums at{upto.query - mine.query, upto.context - mine.context, upto.pages - mine.pages}, total{0, 0, 0};
#pragma unroll
  for (int w = 0; w < kTableThreads / 32; ++w) {
    if (w < warp) at = at + warp_sums[w];
    total = total + warp_sums[w];
  }
  const bool writer = blockIdx.x == 0;
  bool narrow = false;
  for (int b = b0; b < b1; ++b) {
    const Sums s = of(b);
    first_token[slot_of(b)] = to_int32(at.query);
    first_page[slot_of(b)] = to_int32(at.pages);
    at = at + s;
    if (writer) {
      p.cu_seqlens_q[b + 1] = to_int32(at.query);
      p.cu_seqlens_k[b + 1] = to_int32(at.context);
      p.context_lens[b] = to_int32(s.context);
      narrow |= s.query > 0 && s.context > int64_t(p.max_blocks) * p.block_size;
    }
  }
  narrow = __syncthreads_or(narrow);
  if (threadIdx.x == 0) {
    first_token[slot_of(p.num_seqs)] = to_int32(total.query);
    if (writer) {
      p.cu_seqlens_q[0] = p.cu_seqlens_k[0] = 0;
      p.status[0] = to_int32(min(total.pages, p.num_free));
      p.status[1] = (total.pages > p.num_free ? HL_TABLES_NO_PAGES : 0) | (narrow ? HL_TABLES_TOO_NARROW : 0) |
                    (total.query > p.max_tokens ? HL_TABLES_TOO_MANY_TOKENS : 0);
    }
  }
  __syncthreads();

  // ---- table rows, one warp each
  for (int b = blockIdx.x * (kTableThreads / 32) + warp; b < p.num_seqs; b += gridDim.x * (kTableThreads / 32)) {
    const unsigned c = cached(p, b), n = max(p.query_lens[b], 0);
    const unsigned have = pages_of(p, c), need = n ? pages_of(p, c + n) : have;
    for (unsigned j = have + lane; j < unsigned(p.max_blocks); j += 32) {
      const int64_t k = int64_t(first_page[slot_of(b)]) + j - have;
      p.block_tables[b * p.bt_stride + j] = j < need && k < p.num_free ? p.free_blocks[k] : -1;
    }
  }

  // ---- tokens, four neighbours a thread
  const int64_t stride = int64_t(gridDim.x) * kTableThreads * kTokensPerThread;
  for (int64_t i0 = (int64_t(blockIdx.x) * kTableThreads + threadIdx.x) * kTokensPerThread; i0 < p.max_tokens; i0 += stride) {
    int lo = 0, hi = p.num_seqs;  // the sequence of token i0: the first that ends behind it
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (first_token[slot_of(mid + 1)] > i0) hi = mid; else lo = mid + 1;
    }
    int64_t pos[kTokensPerThread];
    int32_t slot[kTokensPerThread];
#pragma unroll
    for (int k = 0; k < kTokensPerThread; ++k) {
      const int64_t i = i0 + k;
      while (lo < p.num_seqs && first_token[slot_of(lo + 1)] <= i) ++lo;
      pos[k] = 0;
      slot[k] = -1;
      if (lo < p.num_seqs && i < p.max_tokens) place_token(p, int(i), lo, first_token, first_page, pos[k], slot[k]);
    }
    if (p.wide && i0 + kTokensPerThread <= p.max_tokens) {
      *reinterpret_cast<longlong2*>(p.positions + i0) = make_longlong2(pos[0], pos[1]);
      *reinterpret_cast<longlong2*>(p.positions + i0 + 2) = make_longlong2(pos[2], pos[3]);
      *reinterpret_cast<int4*>(p.slot_mapping + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int k = 0; k < kTokensPerThread; ++k) {
        if (i0 + k >= p.max_tokens) break;
        p.positions[i0 + k] = pos[k];
        p.slot_mapping[i0 + k] = slot[k];
      }
    }
  }
}

// The bytes of two arrays meet (a pointer of an array without entries may be anything).
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && a_bytes > 0 && b_bytes > 0 && x < y + uintptr_t(b_bytes) && y < x + uintptr_t(a_bytes);
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
  // Every block reads the lengths and the free list for itself, so none may be overwritten meanwhile.
  const int64_t seqs = 4 * int64_t(num_seqs);
  const struct { const void* at; int64_t bytes; } inputs[] = {{cached_lens, seqs}, {query_lens, seqs}, {free_blocks, 4 * num_free}},
      outputs[] = {{cu_seqlens_q, seqs + 4}, {cu_seqlens_k, seqs + 4}, {context_lens, seqs}, {status, 8},
                   {positions, 8 * max_tokens}, {slot_mapping, 4 * max_tokens}};
  for (const auto& in : inputs)
    for (const auto& out : outputs)
      HL_CHECK_ARG(!overlap(in.at, in.bytes, out.at, out.bytes),
                   "hl_extend_block_tables: a result overlaps the lengths or the free list");
  const TableParams p{cached_lens, query_lens, num_seqs, block_tables, bt_stride, max_blocks, free_blocks, num_free,
                      block_size, max_tokens, cu_seqlens_q, cu_seqlens_k, context_lens, positions, slot_mapping,
                      status, aligned16(positions) && aligned16(slot_mapping)};
  // One block per 1024 tokens or 8 table rows, whichever asks for more.
  const int64_t by_tokens = (max_tokens + kTableThreads * kTokensPerThread - 1) / (kTableThreads * kTokensPerThread);
  const int64_t by_rows = (num_seqs + kTableThreads / 32 - 1) / (kTableThreads / 32);
  const int64_t want = by_tokens > by_rows ? by_tokens : by_rows;
  const int blocks = want < 1 ? 1 : want > kMaxTableBlocks ? kMaxTableBlocks : int(want);
  const cudaError_t e = launch_dependent(extend_tables_kernel, dim3(blocks), kTableThreads,
                                         2 * (slot_of(num_seqs) + 1) * sizeof(int32_t), 1, static_cast<cudaStream_t>(stream), p);
  if (e != cudaSuccess) {
    set_error("hl_extend_block_tables: launch failed: %s", cudaGetErrorString(e));
    return HL_ERR_CUDA;
  }
  return HL_OK;
}
