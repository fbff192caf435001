// Paged decode attention (one query token per sequence) over the block-scaled 8-bit KV cache:
//   out[b, hq] = sum_j p_j vs[g(j), h] Vq[j, h],  p = softmax_j(scale * ks[g(j), h] * q[b, hq] . Kq[j, h])
// over the tokens j < context_lens[b] of sequence b, h = hq / G, G = Hq / Hk, g(j) the group of
// scale_block tokens that j's slot lies in.  mini_vllm/layers/attention.py:134-141 calls an 8-bit
// decode without scales.
//
// Bound: HBM, 256 B of K and V per token and head.  One warp walks 32-token tiles of one KV head
// with an online softmax; its K and V tiles arrive by TMA (128-byte swizzle) in a ring of three
// 4 KiB slots of its own, issued by a ninth warp whose lane w serves warp w, so page lookups and
// copies run ahead of the arithmetic and no consumer waits for another.
//
// Both products run on m16n8k16 f16 MMAs with the cache as the A operand, the G query heads being
// the 8 (16 for G > 8) columns: every cache byte is converted once (e4m3 -> f16, exact) and used by
// all G heads.  S^T = K Q^T: M = tokens; a lane's 32-bit word of a K row is its k-slice of one MMA, so
// the dimensions are summed in a permuted order that Q's fragments share.  O^T = V^T P^T: M =
// dimensions, a lane's pairs are two tokens' bytes of one dimension (byte permutes), P^T comes from
// the S^T accumulators by an 8x8 transpose.  The MMA row r of a block of 8 is token tile_row(r), an
// order in which every 16-byte shared load of K and of V is free of bank conflicts.
// q is bf16 times an exact power of two per head, f16.  With lv = log2 vs of the tile, the weights
// enter the second product as f16(2^(s + lv - M)), M the running maximum of s + lv, and the sum as
// fp32 2^(s - m): scales of any range cost no precision, and the f16 rounding (2^-12) is relative to
// the largest weighted value.  Maxima, sums and outputs are fp32; O is rescaled only when M grows.
//
// Work split: the tiles of all sequences in a row are cut into equal ranges, one per warp and head
// (Hk neighbouring warps read the Hk heads of the same tokens, a contiguous piece of the cache).  A
// sequence inside one range is written out directly; the parts of one cut across ranges go to the
// workspace and the warp that finishes last merges them in range order (tickets; results do not
// depend on the order of arrival).  More than kMergeFan parts are merged in two levels, so that the
// ~300 parts of one long sequence are not read by a single warp.
#include "kv_blocks.cuh"

#include <cuda.h>

#include <atomic>

namespace hl {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxBatch = 4096;
constexpr int kWarps = 8;
constexpr int kTile = 32;                           // tokens of one tile
constexpr int kTileBytes = kTile * kBlockHeadDim;   // one ring slot
constexpr int kSlots = 3;
constexpr int kMaxCtas = 296;                       // two per SM of a B200
constexpr int kMaxRanges = kMaxCtas * kWarps;       // (range, head) pairs at most
constexpr int kMergeFan = 16;
constexpr int kMaxDevices = 64;

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
  int32_t* tickets;      // [batch][Hk], all parts of a sequence
  int32_t* sub_tickets;  // [2 * ranges][Hk], one group of kMergeFan parts
  float2* part_ml;       // [2 * ranges][Hk][G]: (m, l)
  float* part_o;         // [2 * ranges][Hk][G][128]
};

// Workspace: error word | tickets | sub-tickets | (m, l) | o.
struct WsLayout {
  int64_t sub, ml, o, end;
};
__host__ __device__ inline WsLayout ws_layout(int batch, int num_q_heads, int num_kv_heads) {
  const int64_t parts = 2 * int64_t(kMaxRanges / num_kv_heads);
  WsLayout w;
  w.sub = 256 + (int64_t(batch) * num_kv_heads * 4 + 255) / 256 * 256;
  w.ml = w.sub + (parts * num_kv_heads * 4 + 255) / 256 * 256;
  w.o = w.ml + (parts * num_q_heads * 8 + 255) / 256 * 256;
  w.end = w.o + parts * num_q_heads * kBlockHeadDim * 4;
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
// Copies one float and arrives on the barrier once it has landed.
__device__ __forceinline__ void copy_float_arrive(float* dst, const float* src, uint64_t* bar) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Token of MMA row r (mod 8).  K: lanes 0-7 of a shared load read rows 2i, 2i + 1, whose tokens
// differ in bit 2; V: rows 0, 2, 4, 6 (or 1, 3, 5, 7) of two chunks, tokens that differ in bits 1-2.
// The 128-byte swizzle XORs the 16-byte chunk with the token's low three bits: no conflicts.
__device__ __forceinline__ int tile_row(int r) { return r ^ ((r & 1) << 2); }

struct Shared {
  uint8_t rows[kWarps][kSlots][kTileBytes];  // 1024-byte aligned slots
  uint64_t full[kWarps][kSlots], empty[kWarps][kSlots];
  float scale[kWarps][kSlots];
  int32_t valid[kWarps][kSlots];  // tokens the tile holds; 0: its page is outside the pool
  int32_t warp_sum[kWarps + 1];
  int32_t pad;
  int32_t prefix[];  // [batch + 1] first tile of each sequence
};

// The producer lane of one consumer warp: walks the tiles [u, end) and copies K, then V of each into
// the next ring slot that is empty.
struct Loader {
  int u, end;      // next tile, end of the range
  int b, b_end;    // its sequence, and that sequence's first tile index behind it
  int n;           // tokens left in the sequence from this tile on
  int page_at, off, group_off, group;  // table index, token offset in the page, in its group; group in the page
  int page;        // block id, or -1

  __device__ __forceinline__ void read_page(const BlockDecodeParams& p) {
    page = p.block_tables[b * p.bt_stride + page_at];
    if (page < 0 || page >= p.num_blocks) {
      atomicOr(p.errors, 2);
      page = -1;
    }
  }
  __device__ __forceinline__ void enter(const BlockDecodeParams& p, const int* prefix) {
    const int tok = (u - prefix[b]) * kTile;
    n = min(p.context_lens[b], p.max_blocks * p.block_size) - tok;
    b_end = prefix[b + 1];
    page_at = tok / p.block_size;
    off = tok - page_at * p.block_size;
    group = off / p.scale_block;
    group_off = off - group * p.scale_block;
    read_page(p);
  }
  __device__ __forceinline__ void load(const BlockDecodeParams& p, Shared& sh, int w, int slot, int h, bool v) const {
    uint64_t* full = &sh.full[w][slot];
    if (page < 0) {
      sh.valid[w][slot] = 0;
      sh.scale[w][slot] = 0.f;
      mbar_arrive(full);
      mbar_arrive(full);
      return;
    }
    sh.valid[w][slot] = min(n, kTile);
    mbar_arrive_expect_tx(full, kTileBytes);
    tma_2d(sh.rows[w][slot], v ? &p.v_map : &p.k_map, h * kBlockHeadDim, page * p.block_size + off, full);
    copy_float_arrive(&sh.scale[w][slot],
                      (v ? p.v_scales : p.k_scales) +
                          (int64_t(page) * (p.block_size / p.scale_block) + group) * p.num_kv_heads + h,
                      full);
  }
  __device__ __forceinline__ void next(const BlockDecodeParams& p, const int* prefix) {
    if (++u >= end) return;
    if (u == b_end) {
      do ++b; while (prefix[b + 1] == u);  // sequences without tokens have no tiles
      enter(p, prefix);
      return;
    }
    n -= kTile;
    off += kTile;
    group_off += kTile;
    if (group_off == p.scale_block) group_off = 0, ++group;
    if (off == p.block_size) {
      off = 0, group = 0, ++page_at;
      read_page(p);
    }
  }
};

// (m, l, o) of `count` parts first, first + step, ... of one (sequence, head), merged in that order into
// out (bf16, when final) or back into part `first`.
__device__ void merge_parts(const BlockDecodeParams& p, int h, int first_slot, int first, int step, int count, int b,
                            bool final, int lane) {
  for (int g = 0; g < p.group; ++g) {
    auto index = [&](int i) {  // part i of the list
      const int r = first + i * step;
      const int slot = r == first && first_slot ? 2 * r + 1 : 2 * r;
      return (int64_t(slot) * p.num_kv_heads + h) * p.group + g;
    };
    float mm = -INFINITY;
    for (int i = lane; i < count; i += 32) mm = fmaxf(mm, __ldcg(&p.part_ml[index(i)]).x);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    const float ref = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < count; i0 += 32) {
      float w = 0.f, wl = 0.f;
      if (i0 + lane < count) {
        const float2 ml = __ldcg(&p.part_ml[index(i0 + lane)]);
        w = ex2(ml.x - ref);
        wl = w * ml.y;
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) wl += __shfl_xor_sync(0xffffffffu, wl, o);
      ll += wl;
      const int k = min(32, count - i0);
#pragma unroll 8
      for (int i = 0; i < k; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + index(i0 + i) * kBlockHeadDim) + lane);
        acc.x = fmaf(v.x, wi, acc.x);
        acc.y = fmaf(v.y, wi, acc.y);
        acc.z = fmaf(v.z, wi, acc.z);
        acc.w = fmaf(v.w, wi, acc.w);
      }
    }
    if (final) {
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
      const __nv_bfloat162 hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(p.out + b * p.out_stride + (int64_t(h) * p.group + g) * kBlockHeadDim + 4 * lane) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
      const int64_t at = index(0);
      __syncwarp();
      __stcg(reinterpret_cast<float4*>(p.part_o + at * kBlockHeadDim) + lane, acc);
      if (lane == 0) __stcg(&p.part_ml[at], make_float2(mm, ll));
    }
  }
}

// 2^(mv - m), the factor from units of 2^mv to units of 2^m; 0 where nothing was summed.
__device__ __forceinline__ float unit(float mv, float m) { return mv == -INFINITY ? 0.f : exp2f(mv - m); }

// True for the warp that takes the last of `count` tickets; it leaves the counter at zero.
__device__ __forceinline__ bool last_ticket(int32_t* ticket, int count, int lane) {
  __threadfence();
  __syncwarp();
  int last = 0;
  if (lane == 0) {
    last = atomicAdd(ticket, 1) == count - 1;
    if (last) *ticket = 0;
  }
  last = __shfl_sync(0xffffffffu, last, 0);
  if (last) __threadfence();
  return last;
}

template <int NT>
__global__ void __launch_bounds__(32 * (kWarps + 1), NT == 1 ? 2 : 1)
    decode_blocks_kernel(const __grid_constant__ BlockDecodeParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  int* prefix = sh.prefix;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < kWarps * kSlots) {
    mbar_init(&sh.full[0][0] + threadIdx.x, 2);   // the tile's bytes and the scale
    mbar_init(&sh.empty[0][0] + threadIdx.x, 1);
    fence_mbar_init();
  }
  // Tiles of each sequence and their prefix sums.
  {
    constexpr int kThreads = 32 * (kWarps + 1);
    const int per = (p.batch + kThreads - 1) / kThreads, width = p.max_blocks * p.block_size;
    const int b0 = threadIdx.x * per;
    int sum = 0;
    for (int b = b0; b < min(b0 + per, p.batch); ++b) sum += (max(min(p.context_lens[b], width), 0) + kTile - 1) / kTile;
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
      before += (max(min(p.context_lens[b], width), 0) + kTile - 1) / kTile;
      if (b == p.batch - 1) prefix[p.batch] = before;
    }
    __syncthreads();
  }
  const int total = prefix[p.batch];
  const int ranges = min(int(gridDim.x) * kWarps / p.num_kv_heads, total);
  auto range_begin = [&](int r) { return int(int64_t(r) * total / ranges); };
  auto range_of = [&](int u) { return int((int64_t(u) * ranges + ranges - 1) / total); };  // that tile u lies in
  auto sequence_of = [&](int u) {  // the last sequence that begins at or before u: it has tiles
    int lo = 0, hi = p.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= u) lo = mid; else hi = mid - 1;
    }
    return lo;
  };

  if (warp == kWarps) {
    // ---- producer: lane w loads for warp w
    const int gid = blockIdx.x * kWarps + lane;
    const int h = gid % p.num_kv_heads, range = gid / p.num_kv_heads;
    Loader ld;
    ld.u = ld.end = 0;
    if (lane < kWarps && range < ranges) {
      ld.u = range_begin(range);
      ld.end = range_begin(range + 1);
      ld.b = sequence_of(ld.u);
      ld.enter(p, prefix);
    }
    int slot = 0, round = 0, idle = 0;
    bool v = false;
    while (__any_sync(0xffffffffu, ld.u < ld.end)) {
      if (ld.u < ld.end) {
        if (mbar_test(&sh.empty[lane][slot], (round & 1) ^ 1)) {
          ld.load(p, sh, lane, slot, h, v);
          if (v) ld.next(p, prefix);
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
  const int gid = blockIdx.x * kWarps + warp;
  const int h = gid % p.num_kv_heads, range = gid / p.num_kv_heads;
  if (range >= ranges) return;
  int u = range_begin(range);
  const int end = range_begin(range + 1);
  int b = sequence_of(u);

  const int c = lane & 3, rr = lane >> 2;
  int slot = 0;
  uint32_t parity = 0;
  auto advance = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.empty[warp][slot]);
    if (++slot == kSlots) slot = 0, parity ^= 1;
  };
  while (u < end) {
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
          v0 = __ldg(src);
          v1 = __ldg(src + 1);
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
    // m: running maximum of s, mv: of s + lv; o in units of 2^mv.
    float m[NT][2], mv[NT][2], l[NT][2], o[NT][8][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int x = 0; x < 2; ++x) m[t][x] = mv[t][x] = -INFINITY, l[t][x] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[t][j][x] = 0.f;
    }
    const int seq_end = prefix[b + 1], seq_begin = prefix[b];
    const bool begins = u == seq_begin;
    const int stop = min(end, seq_end);
    for (; u < stop; ++u) {
      // ---- S^T = K Q^T
      if (!mbar_wait(&sh.full[warp][slot], parity)) {
        if (lane == 0) atomicOr(p.errors, 1);
        return;
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
      const float ks = sh.scale[warp][slot];
      const int valid = sh.valid[warp][slot];
      advance();

      // ---- softmax
      if (!mbar_wait(&sh.full[warp][slot], parity)) {
        if (lane == 0) atomicOr(p.errors, 1);
        return;
      }
      const float lv = __log2f(sh.scale[warp][slot]);
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
              if (valid < kTile && mt * 16 + y * 8 + tile_row(rr) >= valid) v = -INFINITY;
              mx = fmaxf(mx, v);
            }
#pragma unroll
          for (int k = 4; k <= 16; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
          const float m2 = fmaxf(m[t][x], mx), mv2 = fmaxf(mv[t][x], mx + lv);
          const float ref = m2 == -INFINITY ? 0.f : m2, refv = mv2 == -INFINITY ? 0.f : mv2;
          grow[x] = ex2(mv[t][x] - refv);
          float sum = 0.f;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float& v = s[mt][t][2 * y + x];
              sum += ex2(v - ref);
              v = ex2(v + (lv - refv));
            }
          l[t][x] = fmaf(l[t][x], ex2(m[t][x] - ref), sum);
          if (mv2 == mv[t][x]) grow[x] = 1.f;
          m[t][x] = m2;
          mv[t][x] = mv2;
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
          for (int y = 0; y < 2; ++y) pf[t][mt][y] = transpose8x8(pack_half2(s[mt][t][2 * y], s[mt][t][2 * y + 1]));
      }

      // ---- O^T += V^T P^T
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = mt * 16 + (k >> 1) * 8 + tile_row(2 * c + (k & 1));
          v[k] = *reinterpret_cast<const uint4*>(sh.rows[warp][slot] + row * kBlockHeadDim + ((rr ^ (row & 7)) << 4));
          if (valid < kTile && row >= valid) v[k] = make_uint4(0, 0, 0, 0);  // 0 x what lies there may be NaN
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
          const float inv = l[t][x] == 0.f ? 0.f : unit(mv[t][x], m[t][x]) / l[t][x];
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const __nv_bfloat162 h2 = __floats2bfloat162_rn(o[t][j][x] * inv, o[t][j][2 + x] * inv);
            w[j] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          uint4* dst = reinterpret_cast<uint4*>(p.out + b * p.out_stride + (int64_t(h) * p.group + g) * kBlockHeadDim + 16 * rr);
          dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
          dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    } else {
      const int64_t part = (int64_t(2 * range + (begins ? 1 : 0)) * p.num_kv_heads + h) * p.group;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int g = t * 8 + 2 * c + x;
          if (g >= p.group) continue;
          const float f = unit(mv[t][x], m[t][x]);
          float4* dst = reinterpret_cast<float4*>(p.part_o + (part + g) * kBlockHeadDim + 16 * rr);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            __stcg(dst + j, make_float4(o[t][2 * j][x] * f, o[t][2 * j][2 + x] * f, o[t][2 * j + 1][x] * f, o[t][2 * j + 1][2 + x] * f));
          if (rr == 0) __stcg(&p.part_ml[part + g], make_float2(m[t][x], l[t][x]));
        }
      const int first = range_of(seq_begin), last = range_of(seq_end - 1), parts = last - first + 1;
      int32_t* ticket = p.tickets + int64_t(b) * p.num_kv_heads + h;
      if (parts <= kMergeFan) {
        if (last_ticket(ticket, parts, lane)) merge_parts(p, h, 1, first, 1, parts, b, true, lane);
      } else {
        const int sub = (range - first) / kMergeFan, subs = (parts + kMergeFan - 1) / kMergeFan;
        const int head = first + sub * kMergeFan, count = min(kMergeFan, last - head + 1);
        const int head_slot = 2 * head + (sub == 0 ? 1 : 0);
        if (last_ticket(p.sub_tickets + int64_t(head_slot) * p.num_kv_heads + h, count, lane)) {
          merge_parts(p, h, sub == 0, head, 1, count, b, false, lane);
          if (last_ticket(ticket, subs, lane)) merge_parts(p, h, 1, first, kMergeFan, subs, b, true, lane);
        }
      }
    }
    do ++b; while (u < end && prefix[b + 1] == u);
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
  if (ctas * kWarps < p.num_kv_heads) ctas = (p.num_kv_heads + kWarps - 1) / kWarps;
  decode_blocks_kernel<NT><<<ctas, 32 * (kWarps + 1), kShared + 4 * (p.batch + 1), s>>>(p);
  HL_CHECK_LAUNCH("hl_paged_decode_fp8_blocks");
  return HL_OK;
}

}  // namespace
}  // namespace hl

using namespace hl;

extern "C" int64_t hl_paged_decode_fp8_blocks_workspace_size(int batch, int num_q_heads, int num_kv_heads) {
  if (batch <= 0 || batch > kMaxBatch || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return -1;
  if (num_kv_heads > kMaxRanges) return -1;
  return ws_layout(batch, num_q_heads, num_kv_heads).end;
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
                   int64_t(batch) * max_blocks_per_seq * (block_size / kTile) <= 0x7fffffff,
               "hl_paged_decode_fp8_blocks: the block tables span 2^31 tokens a row or 2^36 in all");
  HL_CHECK_ARG(num_blocks <= 0x7fffffff / block_size, "hl_paged_decode_fp8_blocks: a pool of 2^31 tokens or more");
  HL_CHECK_ARG(num_kv_heads <= kMaxRanges, "hl_paged_decode_fp8_blocks: more than %d KV heads", kMaxRanges);
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
  const WsLayout w = ws_layout(batch, num_q_heads, num_kv_heads);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.errors = reinterpret_cast<int32_t*>(ws);
  p.tickets = reinterpret_cast<int32_t*>(ws + 256);
  p.sub_tickets = reinterpret_cast<int32_t*>(ws + w.sub);
  p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  p.part_o = reinterpret_cast<float*>(ws + w.o);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p.group <= 8 ? launch_decode_blocks<1>(p, s) : launch_decode_blocks<2>(p, s);
}
