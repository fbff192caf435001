// Paged decode attention (one query token per sequence) over the block-scaled 8-bit KV cache:
//   out[b, hq] = sum_j p_j vs[g(j), h] Vq[j, h],  p = softmax_j(scale * ks[g(j), h] * q[b, hq] . Kq[j, h])
// over the tokens j < context_lens[b] of sequence b, h = hq / G, G = Hq / Hk, g(j) the group of
// scale_block tokens that j's slot lies in.  mini_vllm/layers/attention.py:134-141 calls an 8-bit
// decode without scales.
//
// Bound: HBM, 256 B of K and V per token and head.  One warp walks 32-token tiles of one KV head
// with an online softmax; its K and V tiles arrive by TMA (128-byte swizzle) in a ring of three
// 4 KiB slots of its own, issued by an eighth warp whose lane w serves warp w, so page lookups and
// copies run ahead of the arithmetic and no consumer waits for another.  Seven and one, twice an SM:
// sixteen warps are four per scheduler with 128 registers each, with two more the tile loop spills
// (256 contexts of 65-1087 tokens, GQA 2: 60 us against 64 us with eight and one).
//
// Both products run on m16n8k16 f16 MMAs with the cache as the A operand, the G query heads being
// the 8 (16 for G > 8) columns: every cache byte is converted once (e4m3 -> f16, exact) and used by
// all G heads.  S^T = K Q^T: M = tokens; a lane's 32-bit word of a K row is its k-slice of one MMA, so
// the dimensions are summed in a permuted order that Q's fragments share.  O^T = V^T P^T: M =
// dimensions, a lane's pairs are two tokens' bytes of one dimension (byte permutes), P^T comes from
// the S^T accumulators by an 8x8 transpose.  The MMA row r of a block of 8 is token tile_row(r), an
// order in which every 16-byte shared load of K and of V is free of bank conflicts.
// q is bf16 times an exact power of two per head, f16 (its elements below 2^-27 of the largest lose
// bits).  With lv = log2 vs of the tile, the weights enter the second product as
// f16(2^(15 + s + lv - M)), M the running maximum of s + lv, and the sum as fp32 2^(s - m).  f16
// because it is what the MMA takes beside the cache's exact f16 values; 2^15 because half of its range
// would lie idle otherwise: a weight down to 2^-29 of the largest is rounded by 2^-12 of itself, a
// smaller one by at most 2^-40 of the largest (without it 2^-14 and 2^-25, and what many light tokens
// add beside one of weight 0.999 and little value was rounded away).  The exponentials are ex2.approx
// (2^-22), lv is lg2.approx.  Maxima, sums and outputs are fp32; M is kept relative to m, so that large
// scores do not cost its bits, and O is rescaled only when M grows.
//
// Work split: a thread block serves one KV head (neighbouring blocks the Hk heads of the same
// tokens).  The tiles of all sequences, with one unit of cost more per sequence for its queries and
// result, form a row that is cut into equal ranges, one per warp and seven per block.  A sequence
// inside one warp's range is written out directly; one cut between warps leaves a part per warp in
// the workspace (L2), and the warp that finishes last (a ticket, in shared memory where the block has
// all parts) merges them in order, so results do not depend on the order of arrival.  A sequence of
// more than kDirectMerge parts is merged by whole blocks, to one part per block first, and more than
// kFlatMerge of those in two levels, so that no warp reads many parts one after another.
#include "dependent_launch.cuh"
#include "kv_blocks.cuh"

#include <cuda.h>

#include <atomic>

namespace hl {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxBatch = 4096;
constexpr int kWarps = 7;                          // that compute; one more loads
constexpr int kTile = 32;                           // tokens of one tile
constexpr int kTileBytes = kTile * kBlockHeadDim;   // one ring slot
constexpr int kSlots = 3;
constexpr int kMaxCtas = 296;                       // two per SM of a B200
constexpr int kDirectMerge = 16;                    // warps' parts merged by one warp
constexpr int kFlatMerge = 40;
constexpr int kMinUnits = 2;                        // of a range: shorter ones cost more in merging
constexpr int kMergeFan = 16;                       // parts of a first-level group
constexpr int kMaxDevices = 64;
constexpr int kGaveUp = 0x7fffffff;                 // in place of a unit: a wait ran out
constexpr float kWeightExp = 15.f;                  // the largest weight of the second product is 2^15

struct BlockDecodeParams {
  CUtensorMap k_map, v_map;  // [num_blocks * block_size rows][Hk * 128 B], boxes of 32 rows x 128 B
  const __nv_bfloat16* q;
  int64_t q_stride;
  const float* k_scales;
  const float* v_scales;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* context_lens;
  int batch, group, num_kv_heads;
  int block_size, scale_block;
  int64_t num_blocks;
  float scale_log2;
  __nv_bfloat16* out;
  int64_t out_stride;
  int32_t* errors;
  int32_t* tickets;      // [kMaxCtas]: the blocks of the sequence that goes on behind a block
  int32_t* sub_tickets;  // [2 * kMaxCtas]: a group of kMergeFan blocks, by its first part
  // Parts of (range, head), then of (block, head), two each (slot 0: of a sequence that began before,
  // 1: of one that goes on behind): [2 * kMaxCtas * (kWarps + 1)][G], o also [128]; o in units of 2^m.
  float2* part_ml;       // (m, l)
  float* part_o;
};

constexpr int kWarpParts = 2 * kMaxCtas * kWarps;

// Workspace: error word | tickets | sub-tickets | (m, l) | o.
struct WsLayout {
  int64_t sub, ml, o, end;
};
__host__ __device__ inline WsLayout ws_layout(int group) {
  const int64_t rows = int64_t(kWarpParts + 2 * kMaxCtas) * group;
  WsLayout w;
  w.sub = 256 + kMaxCtas * 4;
  w.ml = (w.sub + 2 * kMaxCtas * 4 + 255) / 256 * 256;
  w.o = w.ml + (rows * 8 + 255) / 256 * 256;
  w.end = w.o + rows * kBlockHeadDim * 4;
  return w;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The same with 65504 in place of infinity.
__device__ __forceinline__ uint32_t pack_weights(float a, float b) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done;
}
// Token of MMA row r (mod 8).  K: lanes 0-7 of a shared load read rows 2i, 2i + 1, whose tokens
// differ in bit 2; V: rows 0, 2, 4, 6 (or 1, 3, 5, 7) of two chunks, tokens that differ in bits 1-2.
// The 128-byte swizzle XORs the 16-byte chunk with the token's low three bits: no conflicts.
__device__ __forceinline__ int tile_row(int r) { return r ^ ((r & 1) << 2); }

struct TileHead {
  float scale;    // of the tile's group
  int32_t valid;  // tokens it holds; 0: its page is outside the pool
};

struct Shared {
  uint8_t rows[kWarps][kSlots][kTileBytes];  // 1024-byte aligned slots
  uint64_t full[kWarps][kSlots], empty[kWarps][kSlots];
  TileHead head[kWarps][kSlots];
  int32_t warp_sum[kWarps + 1];
  int32_t last;             // broadcast of a ticket
  int32_t tickets[kWarps];  // sequences that begin in a warp's range and end in another's of the block
  int32_t prefix[];  // [batch + 1] first unit of each sequence: its cost unit, then its tiles
};

// The producer lane of one consumer warp: walks the tiles of the units [u, end) and copies K, then V
// of each into the next ring slot that is empty.
struct Loader {
  int u, end;      // next unit (a tile's), end of the range
  int b, b_end;    // its sequence, and the first unit behind it
  int n;           // tokens left in the sequence from this tile on
  int page_at, off, group_off, group;  // table index, token offset in the page, in its group; group in the page
  int page;        // block id, or -1
  float ks, vs;    // the group's scales

  __device__ __forceinline__ void read_page(const BlockDecodeParams& p) {
    page = p.block_tables[b * p.bt_stride + page_at];
    if (page < 0 || page >= p.num_blocks) {
      atomicOr(p.errors, 2);
      page = -1;
    }
  }
  __device__ __forceinline__ void read_scales(const BlockDecodeParams& p, int h) {
    ks = vs = 1.f;  // a tile without a page is masked; its scales have to be numbers
    if (page < 0) return;
    const int64_t at = (int64_t(page) * (p.block_size / p.scale_block) + group) * p.num_kv_heads + h;
    ks = p.k_scales[at];
    vs = p.v_scales[at];
  }
  __device__ __forceinline__ void enter(const BlockDecodeParams& p, const int* prefix, int h) {
    if (u == prefix[b] && ++u >= end) return;  // the cost unit
    const int tok = (u - prefix[b] - 1) * kTile;
    n = min(p.context_lens[b], p.max_blocks * p.block_size) - tok;
    b_end = prefix[b + 1];
    page_at = tok / p.block_size;
    off = tok - page_at * p.block_size;
    group = off / p.scale_block;
    group_off = off - group * p.scale_block;
    read_page(p);
    read_scales(p, h);
  }
  __device__ __forceinline__ void load(const BlockDecodeParams& p, Shared& sh, int w, int slot, int h, bool v) const {
    uint64_t* full = &sh.full[w][slot];
    sh.head[w][slot] = TileHead{v ? vs : ks, page < 0 ? 0 : min(n, kTile)};
    if (page < 0) {
      mbar_arrive(full);
      return;
    }
    mbar_arrive_expect_tx(full, kTileBytes);
    tma_2d(sh.rows[w][slot], v ? &p.v_map : &p.k_map, h * kBlockHeadDim, page * p.block_size + off, full);
  }
  __device__ __forceinline__ void next(const BlockDecodeParams& p, const int* prefix, int h) {
    if (++u >= end) return;
    if (u == b_end) {
      do ++b; while (prefix[b + 1] == u);  // sequences without tokens have no tiles
      enter(p, prefix, h);
      return;
    }
    n -= kTile;
    off += kTile;
    group_off += kTile;
    if (group_off < p.scale_block) return;
    group_off = 0, ++group;
    if (off == p.block_size) {
      off = 0, group = 0, ++page_at;
      read_page(p);
    }
    read_scales(p, h);
  }
};

struct Merged {
  float m, l;
  float4 o;
};

// (m, l, o) of one head over `count` parts, the first at index `first`, the i-th at rest + i * stride,
// summed in that order; a lane holds four dimensions.  All loads of up to 16 parts are in flight
// together; a call of its own, so that they take no registers from the tile loop.
__device__ __noinline__ Merged merge_parts(const float2* part_ml, const float* part_o,
                                           int count, int first, int rest, int stride, int lane) {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto index = [&](int i) { return i == 0 ? first : rest + i * stride; };
  for (int i0 = 0; i0 < count; i0 += 16) {
    const int i = i0 + (lane & 15);
    const float2 ml = i < count ? __ldcg(part_ml + index(i)) : make_float2(-INFINITY, 0.f);
    float4 v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k)
      v[k] = i0 + k < count ? __ldcg(reinterpret_cast<const float4*>(part_o + int64_t(index(i0 + k)) * kBlockHeadDim) + lane)
                            : make_float4(0.f, 0.f, 0.f, 0.f);
    float mx = ml.x;
#pragma unroll
    for (int k = 8; k >= 1; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
    mx = fmaxf(m, mx);
    const float ref = mx == -INFINITY ? 0.f : mx, keep = ex2(m - ref), w = ex2(ml.x - ref);
    float wl = w * ml.y;
#pragma unroll
    for (int k = 8; k >= 1; k >>= 1) wl += __shfl_xor_sync(0xffffffffu, wl, k);
    m = mx;
    l = fmaf(l, keep, wl);
    o.x *= keep, o.y *= keep, o.z *= keep, o.w *= keep;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      o.x = fmaf(v[k].x, wk, o.x);
      o.y = fmaf(v[k].y, wk, o.y);
      o.z = fmaf(v[k].z, wk, o.z);
      o.w = fmaf(v[k].w, wk, o.w);
    }
  }
  return Merged{m, l, o};
}

// One sequence's `count` <= 16 parts of all G heads, merged in order and written to `out` by one warp,
// GC heads at a time with 16 loads a lane in flight.
template <int GC>
__device__ __noinline__ void merge_and_write(const float2* part_ml, const float* part_o,
                                             int count, int first, int rest, int stride, int group,
                                             __nv_bfloat16* out, int lane) {
  constexpr int kParts = 16 / GC, kPairs = (GC + 1) / 2;
  for (int g0 = 0; g0 < group; g0 += GC) {
    // Lane: part lane % 16, heads g0 + kPairs (lane / 16) and the next.
    const int i = lane & 15, gl = kPairs * (lane >> 4);
    float w[kPairs], l[kPairs];
#pragma unroll
    for (int x = 0; x < kPairs; ++x) {
      const float2 ml = i < count && gl + x < GC && g0 + gl + x < group
                            ? __ldcg(part_ml + (i == 0 ? first : rest + i * stride) + g0 + gl + x)
                            : make_float2(-INFINITY, 0.f);
      w[x] = ml.x;
      l[x] = ml.y;
    }
    float4 o[GC];
#pragma unroll
    for (int g = 0; g < GC; ++g) o[g] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < count; i0 += kParts) {
      float4 v[kParts][GC];
#pragma unroll
      for (int k = 0; k < kParts; ++k)
#pragma unroll
        for (int g = 0; g < GC; ++g)
          v[k][g] = i0 + k < count && g0 + g < group
                        ? __ldcg(reinterpret_cast<const float4*>(
                                     part_o + int64_t((i0 + k == 0 ? first : rest + (i0 + k) * stride) + g0 + g) * kBlockHeadDim) +
                                 lane)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 == 0) {
#pragma unroll
        for (int x = 0; x < kPairs; ++x) {
          float m = w[x];
#pragma unroll
          for (int k = 8; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
          w[x] = ex2(w[x] - (m == -INFINITY ? 0.f : m));
          l[x] *= w[x];
#pragma unroll
          for (int k = 8; k >= 1; k >>= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], k);
        }
      }
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        if (i0 + k >= count) break;
#pragma unroll
        for (int g = 0; g < GC; ++g) {
          const float wk = __shfl_sync(0xffffffffu, w[g % kPairs], 16 * (g / kPairs) + i0 + k);
          o[g].x = fmaf(v[k][g].x, wk, o[g].x);
          o[g].y = fmaf(v[k][g].y, wk, o[g].y);
          o[g].z = fmaf(v[k][g].z, wk, o[g].z);
          o[g].w = fmaf(v[k][g].w, wk, o[g].w);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      const float sum = __shfl_sync(0xffffffffu, l[g % kPairs], 16 * (g / kPairs));
      if (g0 + g >= group) continue;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const __nv_bfloat162 lo = __floats2bfloat162_rn(o[g].x * inv, o[g].y * inv);
      const __nv_bfloat162 hi = __floats2bfloat162_rn(o[g].z * inv, o[g].w * inv);
      *reinterpret_cast<uint2*>(out + (g0 + g) * kBlockHeadDim + 4 * lane) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
}

__device__ __forceinline__ void write_part(const BlockDecodeParams& p, int at, int lane, const Merged& r) {
  __stcg(reinterpret_cast<float4*>(p.part_o + int64_t(at) * kBlockHeadDim) + lane, r.o);
  if (lane == 0) __stcg(&p.part_ml[at], make_float2(r.m, r.l));
}

__device__ __forceinline__ void write_row(const BlockDecodeParams& p, int b, int head, int lane, const Merged& r) {
  const float inv = r.l == 0.f ? 0.f : 1.f / r.l;
  const __nv_bfloat162 lo = __floats2bfloat162_rn(r.o.x * inv, r.o.y * inv);
  const __nv_bfloat162 hi = __floats2bfloat162_rn(r.o.z * inv, r.o.w * inv);
  *reinterpret_cast<uint2*>(p.out + b * p.out_stride + head * kBlockHeadDim + 4 * lane) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

// An accumulator of the second product from units of 2^(m + lead - 15) to units of 2^m / y (lead = -inf:
// nothing was summed).  In this order neither step leaves the range of fp32 where the result does not.
__device__ __forceinline__ float from_units(float o, float lead, float y) { return o * (exp2f(-kWeightExp) * y) * exp2f(lead); }

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }

// All consumer warps of the block: true if the block took the last of `count` tickets, after which
// the other blocks' parts can be read.  The counter is left at zero.
__device__ __forceinline__ bool block_is_last(Shared& sh, int32_t* ticket, int count) {
  __threadfence();
  consumers_sync();
  if (threadIdx.x == 0) {
    const int last = atomicAdd(ticket, 1) == count - 1;
    if (last) *ticket = 0;
    __threadfence();
    sh.last = last;
  }
  consumers_sync();
  return sh.last;
}

__device__ __forceinline__ int units_of(int context, int width) {
  const int n = min(context, width);
  return n <= 0 ? 0 : 1 + (n + kTile - 1) / kTile;
}

template <int NT>
__global__ void __launch_bounds__(32 * (kWarps + 1), NT == 1 ? 2 : 1)
    decode_blocks_kernel(const __grid_constant__ BlockDecodeParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  int* prefix = sh.prefix;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < kWarps) sh.tickets[threadIdx.x] = 0;
  if (threadIdx.x < kWarps * kSlots) {
    mbar_init(&sh.full[0][0] + threadIdx.x, 1);
    mbar_init(&sh.empty[0][0] + threadIdx.x, 1);
    fence_mbar_init();
  }
  dependent_start();
  // Units of each sequence and their prefix sums.
  {
    constexpr int kThreads = 32 * (kWarps + 1);
    const int per = (p.batch + kThreads - 1) / kThreads, width = p.max_blocks * p.block_size;
    const int b0 = threadIdx.x * per;
    int sum = 0;
    for (int b = b0; b < min(b0 + per, p.batch); ++b) sum += units_of(p.context_lens[b], width);
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sh.warp_sum[warp] = incl;
    __syncthreads();
    int before = incl - sum;
    for (int w = 0; w < warp; ++w) before += sh.warp_sum[w];
    for (int b = b0; b < min(b0 + per, p.batch); ++b) {
      prefix[b] = before;
      before += units_of(p.context_lens[b], width);
      if (b == p.batch - 1) prefix[p.batch] = before;
    }
    __syncthreads();
  }
  const int total = prefix[p.batch];
  const int h = blockIdx.x % p.num_kv_heads, block = blockIdx.x / p.num_kv_heads, base = block * kWarps;
  const int ranges = min(int(gridDim.x) / p.num_kv_heads * kWarps, (total + kMinUnits - 1) / kMinUnits);
  // Ranges of `share` units, the first `more` of them of one more.
  const unsigned share = unsigned(total) / unsigned(max(ranges, 1)), more = unsigned(total) - share * ranges;
  auto range_begin = [&](int r) { return int(r * share + min(unsigned(r), more)); };
  auto range_of = [&](unsigned u) {  // that unit u lies in
    const unsigned wide = more * (share + 1);
    return int(u < wide ? u / (share + 1) : more + (u - wide) / share);
  };
  auto sequence_of = [&](int u) {  // the last sequence that begins at or before u: it has tiles
    int lo = 0, hi = p.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= u) lo = mid; else hi = mid - 1;
    }
    return lo;
  };

  auto warp_sequence_of = [&](int u) {  // the same for one u, by the lanes of a warp together
    int lo = 0, n = p.batch;
    while (n > 1) {
      const int step = (n + 31) / 32, at = lane * step;
      const int k = __popc(__ballot_sync(0xffffffffu, at < n && prefix[min(lo + at, p.batch - 1)] <= u)) - 1;
      lo += k * step;
      n = min(step, n - k * step);
    }
    return lo;
  };

  if (warp == kWarps) {
    // ---- producer: lane w loads for warp w
    const int range = base + lane;
    Loader ld;
    ld.u = ld.end = 0;
    if (lane < kWarps && range < ranges) {
      ld.u = range_begin(range);
      ld.end = range_begin(range + 1);
      ld.b = sequence_of(ld.u);
      ld.enter(p, prefix, h);
    }
    int slot = 0, round = 0, idle = 0;
    bool v = false;
    while (__any_sync(0xffffffffu, ld.u < ld.end)) {
      if (ld.u < ld.end) {
        if (mbar_test(&sh.empty[lane][slot], (round & 1) ^ 1)) {
          ld.load(p, sh, lane, slot, h, v);
          if (v) ld.next(p, prefix, h);
          v = !v;
          if (++slot == kSlots) slot = 0, ++round;
          idle = 0;
        } else {
          if (++idle > int(kMaxWaitPolls)) {  // the consumer gave up
            atomicOr(p.errors, 1);
            ld.end = ld.u;
          }
          __nanosleep(40);
        }
      }
      __syncwarp();
    }
    // Copies in flight that nobody will wait for (none unless a wait gave up).
    if (idle) {
      for (int i = 0; i < kSlots; ++i) {
        const int at = slot - 1 - i, s = at < 0 ? at + kSlots : at, r = at < 0 ? round - 1 : round;
        if (r >= 0) mbar_wait(&sh.full[lane][s], r & 1);
      }
    }
    return;
  }

  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (prefix[b] != prefix[b + 1]) continue;
    uint4* o = reinterpret_cast<uint4*>(p.out + b * p.out_stride);
    for (int i = threadIdx.x; i < p.group * p.num_kv_heads * (kBlockHeadDim / 8); i += 32 * kWarps) o[i] = make_uint4(0, 0, 0, 0);
  }
  const int range = base + warp;
  int u = range < ranges ? range_begin(range) : 0;
  const int end = range < ranges ? range_begin(range + 1) : 0;
  int b = u < end ? warp_sequence_of(u) : 0;

  const int part_stride = 2 * p.num_kv_heads * p.group;  // from one range's (or block's) parts to the next's
  const int c = lane & 3, rr = lane >> 2;
  int slot = 0;
  uint32_t parity = 0;
  auto advance = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.empty[warp][slot]);
    if (++slot == kSlots) slot = 0, parity ^= 1;
  };
  while (u < end) {
    if (u == prefix[b] && ++u >= end) break;  // the cost unit
    // ---- one sequence: its query heads as B fragments
    uint32_t qf[NT][8][2];
    float qs[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int g = t * 8 + rr;
      uint32_t w[2][8];
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0;
        if (g < p.group) {
          const uint4* src = reinterpret_cast<const uint4*>(p.q + b * p.q_stride + (int64_t(h) * p.group + g) * kBlockHeadDim +
                                                            16 * (c + 4 * i));
          v0 = load16(src);
          v1 = load16(src + 1);
        }
        w[i][0] = v0.x, w[i][1] = v0.y, w[i][2] = v0.z, w[i][3] = v0.w;
        w[i][4] = v1.x, w[i][5] = v1.y, w[i][6] = v1.z, w[i][7] = v1.w;
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fmaxf(fabsf(bf16lo(w[i][k])), fabsf(bf16hi(w[i][k]))));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // The power of two that brings the largest |q| of the head into [2^10, 2^11).
      float up = 1.f, down = 1.f;
      if (amax > 0.f && amax < INFINITY) {
        const int e = max(min(264 - int(__float_as_uint(amax) >> 23), 253), 1);
        up = __uint_as_float(uint32_t(e) << 23);
        down = __uint_as_float(uint32_t(254 - e) << 23);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            qf[t][4 * i + k][x] = pack_half2(bf16lo(w[i][2 * k + x]) * up, bf16hi(w[i][2 * k + x]) * up);
      qs[t][0] = __shfl_sync(0xffffffffu, down, 8 * c) * p.scale_log2;
      qs[t][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4) * p.scale_log2;
    }
    // m: running maximum of s, lead: of s + lv, less m; o in units of 2^(m + lead - 15).
    float m[NT][2], lead[NT][2], l[NT][2], o[NT][8][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int x = 0; x < 2; ++x) m[t][x] = lead[t][x] = -INFINITY, l[t][x] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[t][j][x] = 0.f;
    }
    const int seq_end = prefix[b + 1], seq_begin = prefix[b];
    const bool begins = u == seq_begin + 1;
    const int stop = min(end, seq_end);
    for (; u < stop; ++u) {
      // ---- S^T = K Q^T
      if (!mbar_wait(&sh.full[warp][slot], parity)) {
        if (lane == 0) atomicOr(p.errors, 1);
        u = kGaveUp;
        break;
      }
      float s[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[mt][t][x] = 0.f;
      {
        const int row = tile_row(rr);
        const uint8_t* kbase = sh.rows[warp][slot] + row * kBlockHeadDim;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint8_t* at = kbase + (((c + 4 * i) ^ row) << 4);
          uint4 k[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) k[x] = *reinterpret_cast<const uint4*>(at + 8 * x * kBlockHeadDim);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            auto word = [&](int x) { return w == 0 ? k[x].x : w == 1 ? k[x].y : w == 2 ? k[x].z : k[x].w; };
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              const uint32_t wa = word(2 * mt), wb = word(2 * mt + 1);
              const uint32_t a0 = e4m3_to_f16x2(uint16_t(wa)), a2 = e4m3_to_f16x2(uint16_t(wa >> 16));
              const uint32_t a1 = e4m3_to_f16x2(uint16_t(wb)), a3 = e4m3_to_f16x2(uint16_t(wb >> 16));
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_f16(s[mt][t], a0, a1, a2, a3, qf[t][4 * i + w][0], qf[t][4 * i + w][1]);
            }
          }
        }
      }
      const TileHead head = sh.head[warp][slot];
      const float ks = head.scale;
      const int valid = head.valid;
      advance();

      // ---- softmax
      if (!mbar_wait(&sh.full[warp][slot], parity)) {
        if (lane == 0) atomicOr(p.errors, 1);
        u = kGaveUp;
        break;
      }
      const float lv = __log2f(sh.head[warp][slot].scale);
      const bool part = valid < kTile;  // the sequence's last tile: what lies behind is masked
      if (part) {                       // and its values are zero, for 0 times what is there may be NaN
        for (int i = valid * 32 + lane; i < kTile * 32; i += 32) reinterpret_cast<uint32_t*>(sh.rows[warp][slot])[i] = 0;
        fence_proxy_async_smem();  // before the slot's next copy
        __syncwarp();
      }
      uint32_t pf[NT][2][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float grow[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float f = ks * qs[t][x];
          float mx = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float& v = s[mt][t][2 * y + x];
              v *= f;
              if (part && mt * 16 + y * 8 + tile_row(rr) >= valid) v = -INFINITY;
              mx = fmaxf(mx, v);
            }
#pragma unroll
          for (int k = 4; k <= 16; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
          const float m2 = fmaxf(m[t][x], mx), ref = m2 == -INFINITY ? 0.f : m2, back = m[t][x] - ref;
          const float was = lead[t][x] + back, lead2 = fmaxf(was, (mx - ref) + lv);
          const float up = lv - (lead2 == -INFINITY ? 0.f : lead2) + kWeightExp;
          grow[x] = was == lead2 ? 1.f : ex2(was - lead2);
          float sum = 0.f;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float& v = s[mt][t][2 * y + x];
              v -= ref;
              sum += ex2(v);
              v = ex2(v + up);
            }
          l[t][x] = fmaf(l[t][x], ex2(back), sum);
          m[t][x] = m2;
          lead[t][x] = lead2;
        }
        if (__any_sync(0xffffffffu, grow[0] != 1.f || grow[1] != 1.f)) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[t][j][x] *= grow[x & 1];
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int y = 0; y < 2; ++y) pf[t][mt][y] = transpose8x8(pack_weights(s[mt][t][2 * y], s[mt][t][2 * y + 1]));
      }

      // ---- O^T += V^T P^T
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = mt * 16 + (k >> 1) * 8 + tile_row(2 * c + (k & 1));
          v[k] = *reinterpret_cast<const uint4*>(sh.rows[warp][slot] + row * kBlockHeadDim + ((rr ^ (row & 7)) << 4));
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          auto word = [&](int k) { return w == 0 ? v[k].x : w == 1 ? v[k].y : w == 2 ? v[k].z : v[k].w; };
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362u : 0x5140u;
            const uint32_t e = __byte_perm(word(0), word(1), sel), f = __byte_perm(word(2), word(3), sel);
            const uint32_t a0 = e4m3_to_f16x2(uint16_t(e)), a1 = e4m3_to_f16x2(uint16_t(e >> 16));
            const uint32_t a2 = e4m3_to_f16x2(uint16_t(f)), a3 = e4m3_to_f16x2(uint16_t(f >> 16));
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_f16(o[t][2 * w + half], a0, a1, a2, a3, pf[t][mt][0], pf[t][mt][1]);
          }
        }
      }
      advance();
    }

    // ---- the sequence (or its part in this range) is done: o in units of 2^m
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int k = 4; k <= 16; k <<= 1) l[t][x] += __shfl_xor_sync(0xffffffffu, l[t][x], k);
    if (begins && stop == seq_end) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int g = t * 8 + 2 * c + x;
          if (g >= p.group) continue;
          const float inv = l[t][x] == 0.f ? 0.f : 1.f / l[t][x], from = lead[t][x];
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const __nv_bfloat162 h2 = __floats2bfloat162_rn(from_units(o[t][j][x], from, inv), from_units(o[t][j][2 + x], from, inv));
            w[j] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          uint4* dst = reinterpret_cast<uint4*>(p.out + b * p.out_stride + (int64_t(h) * p.group + g) * kBlockHeadDim + 16 * rr);
          dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
          dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    } else {
      const int part = (2 * (range * p.num_kv_heads + h) + (begins ? 1 : 0)) * p.group;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int g = t * 8 + 2 * c + x;
          if (g >= p.group) continue;
          const float from = lead[t][x];
          float4* dst = reinterpret_cast<float4*>(p.part_o + int64_t(part + g) * kBlockHeadDim + 16 * rr);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            __stcg(dst + j, make_float4(from_units(o[t][2 * j][x], from, 1.f), from_units(o[t][2 * j][2 + x], from, 1.f),
                                        from_units(o[t][2 * j + 1][x], from, 1.f), from_units(o[t][2 * j + 1][2 + x], from, 1.f)));
          if (rr == 0) __stcg(&p.part_ml[part + g], make_float2(m[t][x], l[t][x]));
        }
      // The last warp of a sequence of few parts merges them.
      const int first = range_of(seq_begin + 1), last = range_of(seq_end - 1), parts = last - first + 1;
      if (parts <= kDirectMerge) {
        const bool own = first >= base && last < base + kWarps;
        if (own) __threadfence_block(); else __threadfence();
        __syncwarp();
        int done = 0;
        if (lane == 0) {
          if (own) {
            done = atomicAdd(&sh.tickets[first - base], 1) == parts - 1;
          } else {  // one arrival per warp; left at zero for the next launch
            int32_t* ticket = p.tickets + first / kWarps * p.num_kv_heads + h;
            done = atomicAdd(ticket, 1) == parts - 1;
            if (done) *ticket = 0;
          }
        }
        if (__shfl_sync(0xffffffffu, done, 0)) {
          if (own) __threadfence_block(); else __threadfence();
          const int from = 2 * (first * p.num_kv_heads + h) * p.group;
          __nv_bfloat16* out = p.out + b * p.out_stride + int64_t(h) * p.group * kBlockHeadDim;
          if (p.group <= 2)
            merge_and_write<2>(p.part_ml, p.part_o, parts, from + p.group, from, part_stride, p.group, out, lane);
          else
            merge_and_write<4>(p.part_ml, p.part_o, parts, from + p.group, from, part_stride, p.group, out, lane);
        }
      }
    }
    do ++b; while (u < end && prefix[b + 1] == u);
  }
  if (u == kGaveUp) {  // copies that are still in flight (no more than the ring holds), with a limit each
    for (int i = 0; i < kSlots; ++i) {
      mbar_wait(&sh.full[warp][slot], parity);
      if (++slot == kSlots) slot = 0, parity ^= 1;
    }
  }

  // ---- long sequences, which are cut at this block's first border (they came in), its last (they go
  // on), or both
  if (base >= ranges) return;
  for (int side = 0; side < 2; ++side) {
    const int border = range_begin(min(base + side * kWarps, ranges));
    if (border >= total) continue;
    const int b = warp_sequence_of(border);
    if (border <= prefix[b] + 1) continue;  // no tile of it lies in front
    const int first = range_of(prefix[b] + 1), last = range_of(prefix[b + 1] - 1);
    if (last - first < kDirectMerge || (side && first < base)) continue;
    consumers_sync();  // the block's parts are written
    const int k0 = first / kWarps, k1 = last / kWarps;
    // Part of block k: slot 1 where the sequence begins, 0 behind it.
    auto at_rest = [&](int k, int g) { return (kWarpParts + 2 * (k * p.num_kv_heads + h)) * p.group + g; };
    auto at = [&](int k, int g) { return at_rest(k, g) + (k == k0 ? p.group : 0); };
    const int w0 = max(first, base), w1 = min(last, base + kWarps - 1);
    for (int g = warp; g < p.group; g += kWarps) {
      const int from = 2 * (w0 * p.num_kv_heads + h) * p.group + g;
      write_part(p, at(block, g), lane,
                 merge_parts(p.part_ml, p.part_o, w1 - w0 + 1, w0 == first ? from + p.group : from, from, part_stride, lane));
    }
    int step = 1, count = k1 - k0 + 1;
    if (count > kFlatMerge) {
      const int head = k0 + (block - k0) / kMergeFan * kMergeFan, n = min(kMergeFan, k1 - head + 1);
      if (!block_is_last(sh, p.sub_tickets + 2 * (head * p.num_kv_heads + h) + (head == k0), n)) continue;
      for (int g = warp; g < p.group; g += kWarps) {
        const Merged r = merge_parts(p.part_ml, p.part_o, n, at(head, g), at_rest(head, g), part_stride, lane);
        write_part(p, at(head, g), lane, r);
      }
      step = kMergeFan;
      count = (count + kMergeFan - 1) / kMergeFan;
    }
    if (!block_is_last(sh, p.tickets + k0 * p.num_kv_heads + h, count)) continue;
    for (int g = warp; g < p.group; g += kWarps) {
      write_row(p, b, h * p.group + g, lane,
                merge_parts(p.part_ml, p.part_o, count, at(k0, g), at_rest(k0, g), step * part_stride, lane));
    }
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

bool encode_cache_map(CUtensorMap* map, const void* cache, int64_t rows, int num_kv_heads) {
  static const EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<EncodeTiledFn>(ptr)
               : nullptr;
  }();
  const cuuint64_t row_bytes = cuuint64_t(num_kv_heads) * kBlockHeadDim;
  const cuuint64_t dims[2] = {row_bytes, cuuint64_t(rows)}, strides[1] = {row_bytes};
  const cuuint32_t box[2] = {kBlockHeadDim, kTile}, steps[2] = {1, 1};
  return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(cache), dims, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT>
int launch_decode_blocks(const BlockDecodeParams& p, cudaStream_t s) {
  constexpr int kPerSm = NT == 1 ? 2 : 1;
  constexpr int kShared = int(sizeof(Shared));
  static std::atomic<int> sms[kMaxDevices];  // 0: this kernel is not set up on the device yet
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  int n = e == cudaSuccess && dev < kMaxDevices ? sms[dev].load(std::memory_order_relaxed) : 0;
  if (e == cudaSuccess && n == 0) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(decode_blocks_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kShared + 4 * (kMaxBatch + 1));
    if (e == cudaSuccess && dev < kMaxDevices) sms[dev].store(n, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) {
    set_error("hl_paged_decode_fp8_blocks: %s", cudaGetErrorString(e));
    return HL_ERR_CUDA;
  }
  int ctas = n * kPerSm < kMaxCtas ? n * kPerSm : kMaxCtas;
  if (ctas < p.num_kv_heads) ctas = p.num_kv_heads;
  e = launch_dependent(decode_blocks_kernel<NT>, dim3(ctas), 32 * (kWarps + 1), kShared + 4 * (p.batch + 1), 1, s, p);
  if (e != cudaSuccess) {
    set_error("hl_paged_decode_fp8_blocks: launch failed: %s", cudaGetErrorString(e));
    return HL_ERR_CUDA;
  }
  return HL_OK;
}

}  // namespace
}  // namespace hl

using namespace hl;

extern "C" int64_t hl_paged_decode_fp8_blocks_workspace_size(int batch, int num_q_heads, int num_kv_heads) {
  if (batch <= 0 || batch > kMaxBatch || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return -1;
  if (num_kv_heads > kMaxCtas) return -1;
  return ws_layout(num_q_heads / num_kv_heads).end;
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
  HL_CHECK_ARG(int64_t(max_blocks_per_seq) * block_size <= 0x7fffffff &&
                   int64_t(batch) * max_blocks_per_seq * (block_size / kTile + 1) <= 0x7fffffff,
               "hl_paged_decode_fp8_blocks: the block tables span 2^31 tokens a row or 2^36 in all");
  HL_CHECK_ARG(num_blocks <= 0x7fffffff / block_size, "hl_paged_decode_fp8_blocks: a pool of 2^31 tokens or more");
  HL_CHECK_ARG(num_kv_heads <= kMaxCtas, "hl_paged_decode_fp8_blocks: more than %d KV heads", kMaxCtas);
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
  if (!encode_cache_map(&p.k_map, k_cache, num_blocks * block_size, num_kv_heads) ||
      !encode_cache_map(&p.v_map, v_cache, num_blocks * block_size, num_kv_heads)) {
    set_error("hl_paged_decode_fp8_blocks: cuTensorMapEncodeTiled failed");
    return HL_ERR_CUDA;
  }
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.block_tables = block_tables;
  p.bt_stride = bt_stride;
  p.max_blocks = max_blocks_per_seq;
  p.context_lens = context_lens;
  p.batch = batch;
  p.num_kv_heads = num_kv_heads;
  p.block_size = block_size;
  p.scale_block = scale_block;
  p.num_blocks = num_blocks;
  p.scale_log2 = softmax_scale * kLog2e;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_row_stride;
  p.group = num_q_heads / num_kv_heads;
  const WsLayout w = ws_layout(p.group);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.errors = reinterpret_cast<int32_t*>(ws);
  p.tickets = reinterpret_cast<int32_t*>(ws + 256);
  p.sub_tickets = reinterpret_cast<int32_t*>(ws + w.sub);
  p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  p.part_o = reinterpret_cast<float*>(ws + w.o);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p.group <= 8 ? launch_decode_blocks<1>(p, s) : launch_decode_blocks<2>(p, s);
}
