// Log probabilities of given tokens, with the entropy of each row and its most probable tokens
// (the reference's sampler returns token ids only, mini_vllm/layers/sampler.py:12-25):
//   m = max_i x_i, Z = sum_i e^(x_i - m)
//   logprob = x_t - m - ln Z,   entropy = ln Z - (1/Z) sum_i e^(x_i - m) (x_i - m)
//   top: the top_n tokens by (logit descending, index ascending) and their log probabilities.
// Sums are fp32.  A masked token (-inf) has probability 0 and adds nothing to the entropy; a row
// with nothing but -inf has log probabilities -inf and entropy 0; a token id outside [0, vocab) has
// log probability -inf; a NaN or +inf makes the row's results NaN, and a NaN ranks below -inf.
//
// Bound: one read of the logits from HBM.  A row is split over a cluster of thread blocks when there
// are few rows (they meet in distributed shared memory), each thread keeps an online softmax of the
// 16-byte vectors tid, tid + T, ... of its block's piece (T threads): Z = sum 2^y and S = sum 2^y y, where
// y = x log2 e - R and R a whole number near its maximum, raised only when a logit exceeds it by far
// (2^16): one FMA a logit, and parts of different R meet with exact powers of two.  R stays 0 for logits
// below -1e8, which add 0 then, as masked ones do whatever the value that masks them; only a piece with
// nothing above -5e7, or with a logit above 1e8 (where R no longer resolves one), is summed again one by
// one, relative to one of its logits.  The instructions bound it next: 2048 rows of 151936 bf16 take
// 110 us, 0.87 of the copy rate, with one exponential in four as a polynomial 119, for that saves MUFU
// work (two thirds busy) but issues more.
// Alternatives come from the same pass.  The largest logit of each of 64 groups of threads is known;
// the top_n-th largest of those is a threshold that at least top_n logits reach, and few more do
// (some 24 for 20 of 151936 independent ones).  Only threads whose own maximum reaches it are looked
// through again, a warp for one thread's vectors, and the candidates are ranked by unique 64-bit
// (logit, index) keys.  Where ties at the threshold are too many for the candidate buffer, those with
// the lowest indices are taken in index order; where that many lie above it, rounds of block maxima.
#include "dependent_launch.cuh"

#include <cooperative_groups.h>

namespace hl {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTop = 32;
constexpr int kGroups = 64;                     // threads tid = g mod 64, for the threshold
constexpr int kMaxCandidates = 1024;
constexpr int kMaxCluster = 8;
constexpr int kUnroll = 4;                      // 16-byte loads in flight per thread
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
struct Row {
  static constexpr int kVec = 16 / int(sizeof(T));
  const T* x;        // the row
  int head;          // logits in front of the first 16-byte boundary
  int vectors;       // whole vectors behind it
  int tail;          // logits behind those
  __device__ __forceinline__ Row(const T* row, int vocab) : x(row) {
    const int off = int(reinterpret_cast<uintptr_t>(row) & 15u) / int(sizeof(T));
    head = min(off ? kVec - off : 0, vocab);
    vectors = (vocab - head) / kVec;
    tail = vocab - head - vectors * kVec;
  }
  __device__ __forceinline__ uint4 vector(int v) const { return load16(x + head + int64_t(v) * kVec); }
};

__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_logit(const float* p) { return *p; }

// Logits 2i and 2i + 1 of a vector.
__device__ __forceinline__ float2 pair(const uint4& v, int i, const __nv_bfloat16*) {
  const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
  return make_float2(bf16lo(w), bf16hi(w));
}
__device__ __forceinline__ float2 pair(const uint4& v, int i, const float*) {
  return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
}
// A vector with nothing below -1e38, NaN kept: what the sums below add up from a masked logit is 0 then,
// not 0 times infinity (with a second look at the batches where that happened instead, rows with masked
// logits took 1.6 to 4 times as long).  One instruction for two bf16 logits.
__device__ __forceinline__ uint4 unmasked(uint4 v, const __nv_bfloat16*) {
  auto cut = [](uint32_t w) {
    const __nv_bfloat162 h = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w), __float2bfloat162_rn(-1e38f));
    return *reinterpret_cast<const uint32_t*>(&h);
  };
  return make_uint4(cut(v.x), cut(v.y), cut(v.z), cut(v.w));
}
__device__ __forceinline__ uint4 unmasked(uint4 v, const float*) {
  auto cut = [](uint32_t w) {
    float r;
    asm("max.NaN.f32 %0, %1, 0fFE967699;" : "=f"(r) : "f"(__uint_as_float(w)));
    return __float_as_uint(r);
  };
  return make_uint4(cut(v.x), cut(v.y), cut(v.z), cut(v.w));
}
// Largest logit of a batch of vectors (NaN ignored; NaN if there is nothing else).
template <int N>
__device__ __forceinline__ float largest(const uint4 (&v)[N], const __nv_bfloat16*) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v[0]);
  __nv_bfloat162 m = h[0];
#pragma unroll
  for (int i = 1; i < 4 * N; ++i) m = __hmax2(m, h[i]);
  return fmaxf(__low2float(m), __high2float(m));
}
template <int N>
__device__ __forceinline__ float largest(const uint4 (&v)[N], const float*) {
  const float* f = reinterpret_cast<const float*>(&v[0]);
  float m = f[0];
#pragma unroll
  for (int i = 1; i < 4 * N; ++i) m = fmaxf(m, f[i]);
  return m;
}

// Whole numbers in the order of the logits: NaN lowest, then -inf ... +inf; -0 and +0 alike.  Never 0.
__device__ __forceinline__ uint32_t logit_key(float x) {
  if (x != x) return 1u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  if (k == 1u) return NAN;
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

constexpr uint32_t kMaskedKey = 0x007fffffu;  // of -inf; below it NaN only

// Unique over a row: larger for a larger logit, and for a lower index among equals.  Never 0.
__device__ __forceinline__ uint64_t entry_key(uint32_t key, int i) { return (uint64_t(key) << 32) | uint32_t(~i); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Keeps NaN (fmaxf would not); -inf becomes -1000, whose power of two is 0 and stays 0 when multiplied.
__device__ __forceinline__ float floor_exponent(float y) {
  float r;
  asm("max.NaN.f32 %0, %1, 0fC47A0000;" : "=f"(r) : "f"(y));
  return r;
}

// Below this size a reference m is taken as the whole number next to m log2 e, which fp32 holds to within
// 8 there (from 1.5e9 on it misses by 128 and more, and its own 2^y would overflow).
constexpr float kUsual = 1e8f;
constexpr float kHuge = 1e30f;  // log2 e times it is far from overflow

// y of a logit x for a part with reference m, one of its logits and no less than its maximum - 11:
// x log2 e - ceil(m log2 e), or (x - m) log2 e for an m that is not usual; -1000 at least.
__device__ __forceinline__ float origin(float m) { return ceilf(m * kLog2e); }
__device__ __forceinline__ bool usual(float m) { return fabsf(m) < kUsual; }
__device__ __forceinline__ float exponent(float x, float m) {
  return floor_exponent(usual(m) ? fmaf(x, kLog2e, -origin(m)) : (x - m) * kLog2e);
}
// What y of reference `to` is less than y of reference m; kAll: of any size, not usual ones only.
template <bool kAll>
__device__ __forceinline__ float shift(float m, float to) {
  if (!kAll) return floor_exponent(origin(m) - origin(to));
  const float d = usual(m) ? (usual(to) ? origin(m) - origin(to) : fmaf(to, -kLog2e, origin(m)))
                           : (usual(to) ? fmaf(m, kLog2e, -origin(to)) : (m - to) * kLog2e);
  return floor_exponent(d);
}

// Online softmax: z = sum 2^y, s = sum 2^y y.
struct Softmax {
  float m, z, s;

  __device__ __forceinline__ float ref() const { return m == -INFINITY ? 0.f : m; }
  template <bool kAll>
  __device__ __forceinline__ void raise(float to) {
    if (!(to > m)) return;
    if (m != -INFINITY) {  // else z and s are 0, or NaN
      const float d = shift<kAll>(m, to), f = ex2(d);
      s = f * fmaf(d, z, s);
      z *= f;
    }
    m = to;
  }
  // The same where the reference would fall behind by more than 16 = 11 log2 e.  kAll = false: not to
  // logits below -1e8; the sums are worthless once there was one above 1e8.  kAll = true: at once, since
  // m + 11 may be m + 16 or m where the logits' own steps are as large.
  template <bool kAll>
  __device__ __forceinline__ void raise_late(float to) {
    if (kAll ? !(to <= m) : !(to <= m + 11.f) && to > -kUsual) raise<kAll>(to);
  }
  template <bool kAll>
  __device__ __forceinline__ void add(float x) {
    raise_late<kAll>(x);
    const float y = exponent(x, ref()), e = ex2(y);
    z += e;
    s = fmaf(e, y, s);
  }
};

// The sums of a warp's lanes (`lanes` of them, a power of two), in every one of those lanes.
__device__ __forceinline__ Softmax warp_merge(Softmax a, int lanes) {
  float m = a.m;
  for (int o = lanes / 2; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  a.raise<true>(m);
  for (int o = lanes / 2; o >= 1; o >>= 1) {
    a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
  }
  a.m = m;
  return a;
}

__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <int NT>
struct LpShared {
  Softmax parts[(NT / 32)];
  Softmax sum;
  __align__(16) uint32_t group_key[kGroups];
  uint32_t threshold;
  int count, suspects;            // candidates; threads whose maximum reaches the threshold
  uint16_t suspect[NT];
  int scan[(NT / 32)];
  uint64_t best;
  __align__(16) uint64_t candidates[kMaxCandidates + 2];
  uint64_t top[kMaxTop];          // this block's, in order; 0 behind the last
  __align__(16) uint64_t all[kMaxCluster * kMaxTop + 2];
};

// This block's piece of a row.
template <typename T, int NT>
struct Piece {
  Row<T> row;
  int begin, end;      // vectors
  bool first, last;    // has the head, the tail
  // Calls f(logit, index) for every logit of thread `t`, vectors first.
  template <typename F>
  __device__ __forceinline__ void each_of(int t, F f) const {
    for (int v = begin + t; v < end; v += NT) each_in(v, f);
    each_single(t, f);
  }
  template <typename F>
  __device__ __forceinline__ void each_in(int v, F f) const {
    each_of(row.vector(v), v, f);
  }
  template <typename F>
  __device__ __forceinline__ void each_of(const uint4& q, int v, F f) const {  // q: vector v
#pragma unroll
    for (int i = 0; i < Row<T>::kVec / 2; ++i) {
      const float2 x = pair(q, i, row.x);
      f(x.x, row.head + v * Row<T>::kVec + 2 * i);
      f(x.y, row.head + v * Row<T>::kVec + 2 * i + 1);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each_single(int t, F f) const {
    if (first && t < row.head) f(load_logit(row.x + t), t);
    if (last && t < row.tail) {
      const int i = row.head + row.vectors * Row<T>::kVec + t;
      f(load_logit(row.x + i), i);
    }
  }
};

// Before block_top, with a barrier in between.
template <int NT>
__device__ __forceinline__ void clear_top(LpShared<NT>& sh) {
  const int tid = threadIdx.x;
  if (tid < kGroups) sh.group_key[tid] = 0;
  if (tid < kMaxTop) sh.top[tid] = 0;
  if (tid == 0) sh.count = sh.suspects = 0;
}

// The top_n largest entries of the piece, in order, into sh.top.  mine: the key of this thread's
// largest logit, 0 if it has none.
template <typename T, int NT>
__device__ void block_top(const Piece<T, NT>& piece, int top_n, uint32_t mine, LpShared<NT>& sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  atomicMax(&sh.group_key[tid % kGroups], mine);
  __syncthreads();
  if (tid < kGroups) {
    const uint32_t g = sh.group_key[tid];
    int rank = 0;
#pragma unroll
    for (int i = 0; i < kGroups; i += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&sh.group_key[i]);
      rank += (o.x > g || (o.x == g && i < tid)) + (o.y > g || (o.y == g && i + 1 < tid)) +
              (o.z > g || (o.z == g && i + 2 < tid)) + (o.w > g || (o.w == g && i + 3 < tid));
    }
    if (rank == top_n - 1) sh.threshold = g;
  }
  __syncthreads();
  const uint32_t threshold = sh.threshold;
  auto overflown = [&] { return *const_cast<volatile int*>(&sh.count) > kMaxCandidates; };  // then all are dropped
  auto collect = [&](float x, int i, uint32_t least) {
    const uint32_t key = logit_key(x);
    if (key < least) return;
    if (overflown()) return;
    const int at = atomicAdd(&sh.count, 1);
    if (at < kMaxCandidates) sh.candidates[at] = entry_key(key, i);
  };
  // The vectors of the threads whose maximum reaches `least`, spread over all threads.
  auto gather = [&](uint32_t least) {
    if (mine >= least) {
      sh.suspect[atomicAdd(&sh.suspects, 1)] = uint16_t(tid);
      piece.each_single(tid, [&](float x, int i) { collect(x, i, least); });
    }
    __syncthreads();
    // Warp w: suspects w, w + NT / 32, ..., two at a time; lane l: their vectors l, l + 32, ...
    const float reach = key_logit(least);
    const int n = sh.suspects, each = (piece.end - piece.begin + NT - 1) / NT;
    for (int s0 = warp; s0 < n && !overflown(); s0 += 2 * (NT / 32)) {
      const int s1 = s0 + NT / 32;
      const int t0 = piece.begin + sh.suspect[s0], t1 = s1 < n ? piece.begin + sh.suspect[s1] : piece.end;
      for (int k0 = lane; k0 < each; k0 += 64) {
        int v[4] = {t0 + k0 * NT, t0 + (k0 + 32) * NT, t1 + k0 * NT, t1 + (k0 + 32) * NT};
        uint4 q[4][1];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (v[k] < piece.end) q[k][0] = piece.row.vector(v[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (v[k] < piece.end && (least <= kMaskedKey || largest(q[k], piece.row.x) >= reach))
            piece.each_of(q[k][0], v[k], [&](float x, int i) { collect(x, i, least); });
      }
    }
  };
  gather(threshold);
  __syncthreads();
  int count = sh.count;
  if (count > kMaxCandidates) {
    __syncthreads();
    if (tid == 0) sh.count = sh.suspects = 0;
    __syncthreads();
    gather(threshold + 1);
    __syncthreads();
    count = sh.count;
    if (count <= kMaxCandidates) {
      // The ties at the threshold with the lowest indices: head, then vectors, then tail.
      int need = top_n - count;
      auto take = [&](int ties, auto each) {  // ties of this thread, in index order over the threads
        int upto = ties;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        __syncthreads();
        if (lane == 31) sh.scan[warp] = upto;
        __syncthreads();
        int before = upto - ties, total = 0;
        for (int w = 0; w < (NT / 32); ++w) {
          if (w < warp) before += sh.scan[w];
          total += sh.scan[w];
        }
        int at = before;
        each([&](int i) {
          if (at < need) sh.candidates[count + at] = entry_key(threshold, i);
          ++at;
        });
        const int took = min(total, need);
        need -= took;
        count += took;
      };
      auto tied = [&](float x) { return logit_key(x) == threshold; };
      auto single = [&](bool has, int i) {
        const bool t = has && tied(load_logit(piece.row.x + i));
        take(t, [&](auto put) { if (t) put(i); });
      };
      if (need > 0 && piece.first) single(tid < piece.row.head, tid);
      for (int v = piece.begin; need > 0 && v < piece.end; v += NT) {
        int ties = 0;
        if (v + tid < piece.end) piece.each_in(v + tid, [&](float x, int) { ties += tied(x); });
        take(ties, [&](auto put) {
          if (ties) piece.each_in(v + tid, [&](float x, int i) { if (tied(x)) put(i); });
        });
      }
      if (need > 0 && piece.last) single(tid < piece.row.tail, piece.row.head + piece.row.vectors * Row<T>::kVec + tid);
      __syncthreads();
    } else {
      // More above the threshold than the buffer holds: one block maximum per alternative.
      uint64_t below = ~0ull;
      for (int r = 0; r < top_n; ++r) {
        uint64_t best = 0;
        if (mine >= threshold)
          piece.each_of(tid, [&](float x, int i) {
            const uint64_t e = entry_key(logit_key(x), i);
            if (e < below && e > best) best = e;
          });
        __syncthreads();
        if (tid == 0) sh.best = 0;
        __syncthreads();
        if (best) atomicMax(reinterpret_cast<unsigned long long*>(&sh.best), best);
        __syncthreads();
        below = sh.best;
        if (tid == 0) sh.top[r] = below;
      }
      __syncthreads();
      return;
    }
  }
  if (tid < 2) sh.candidates[count + tid] = 0;  // pairs below
  __syncthreads();
  for (int i = tid; i < count; i += NT) {
    const uint64_t e = sh.candidates[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < count; j += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&sh.candidates[j]);
      rank += (o.x > e) + (o.y > e);
    }
    if (rank < top_n) sh.top[rank] = e;
  }
  __syncthreads();
}

// The sums of a piece whose logits are of any size, one by one; in every lane those of its warp.  A call,
// for inside the kernel it costs the loop registers (2048 rows: 112.8 us, 109.8 with the call).
template <typename T, int NT>
__device__ __noinline__ Softmax add_one_by_one(const Piece<T, NT> piece) {
  Softmax sm{-INFINITY, 0.f, 0.f};
  piece.each_of(threadIdx.x, [&](float x, int) { sm.add<true>(x); });
  return warp_merge(sm, 32);
}

// One cluster per row, each block a piece of it.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) token_logprobs_kernel(
    const T* logits, int64_t row_stride, int vocab, const int64_t* tokens, int top_n,
    float* logprobs, float* entropies, int64_t* top_tokens,
    float* top_logprobs) {
  __shared__ LpShared<NT> sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int64_t row_at = blockIdx.x / blocks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T> row(logits + row_at * row_stride, vocab);
  const Piece<T, NT> piece{row, int(int64_t(row.vectors) * rank / blocks), int(int64_t(row.vectors) * (rank + 1) / blocks),
                       rank == 0, rank == blocks - 1};
  dependent_start();
  if (top_n > 0) {
    clear_top(sh);
    __syncthreads();
  }
  float asked = -INFINITY;  // the logit of the row's token
  if (rank == 0 && tid == 0) {
    const int64_t t = tokens[row_at];
    if (t >= 0 && t < vocab) asked = load_logit(row.x + t);
  }
  Softmax sm{-INFINITY, 0.f, 0.f};
  float thread_max = NAN;  // NaN: nothing else
  bool any = false;        // the thread has a logit
  piece.each_single(tid, [&](float x, int) {
    sm.add<false>(x);
    thread_max = fmaxf(thread_max, x);
    any = true;
  });
  any |= piece.begin + tid < piece.end;
  // Batches of kUnroll vectors, the next one's loads in flight while one is summed.
  auto load = [&](uint4 (&q)[kUnroll], int v0) {
    if (v0 + (kUnroll - 1) * NT < piece.end) {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) q[k] = row.vector(v0 + k * NT);
    } else {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)  // behind the piece: NaN, which no maximum takes
        q[k] = v0 + k * NT < piece.end ? row.vector(v0 + k * NT) : make_uint4(~0u, ~0u, ~0u, ~0u);
    }
  };
  auto sum_batch = [&](uint4 (&q)[kUnroll], int v0) {
    if (v0 >= piece.end) return;
    const float top = largest(q, row.x);
    thread_max = fmaxf(thread_max, top);
    sm.raise_late<false>(top);
    if (v0 + (kUnroll - 1) * NT >= piece.end) {  // behind the piece: -9e29, which adds nothing to a usual reference
      const uint32_t low = sizeof(T) == 2 ? 0xf135f135u : 0xf135be37u;
#pragma unroll
      for (int k = 1; k < kUnroll; ++k)
        if (v0 + k * NT >= piece.end) q[k] = make_uint4(low, low, low, low);
    }
    const float ref = sm.ref(), minus = -origin(ref);
    const uint64_t off = f32x2(minus, minus), scale = f32x2(kLog2e, kLog2e);
    uint64_t z = 0, s = 0;  // (0.f, 0.f)
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const uint4 u = unmasked(q[k], row.x);
#pragma unroll
      for (int i = 0; i < Row<T>::kVec / 2; ++i) {
        const float2 x = pair(u, i, row.x);
        const uint64_t y = fma2(f32x2(x.x, x.y), scale, off);
        const float2 yy = unpack(y);
        const uint64_t e = f32x2(ex2(yy.x), ex2(yy.y));
        z = add2(z, e);
        s = fma2(e, y, s);
      }
    }
    const float2 zz = unpack(z), ss = unpack(s);
    sm.z += zz.x + zz.y;
    sm.s += ss.x + ss.y;
  };
  uint4 even[kUnroll], odd[kUnroll];
  load(even, piece.begin + tid);
  for (int v0 = piece.begin + tid; v0 < piece.end; v0 += 2 * kUnroll * NT) {
    load(odd, v0 + kUnroll * NT);
    sum_batch(even, v0);
    load(even, v0 + 2 * kUnroll * NT);
    sum_batch(odd, v0 + kUnroll * NT);
  }
  // ---- the block's sums
  sm = warp_merge(sm, 32);
  if (lane == 0) sh.parts[warp] = sm;
  if (top_n > 0) block_top(piece, top_n, any ? logit_key(thread_max) : 0u, sh);
  __syncthreads();
  const float part_m = sh.parts[lane % (NT / 32)].m;
  if (!__any_sync(0xffffffffu, part_m > -0.5f * kUsual) || __any_sync(0xffffffffu, part_m >= kUsual)) {
    // The same decision in every warp.  (2048 rows of -1e30 alone: 416 us, 109 of usual logits.)
    sm = add_one_by_one(piece);
    __syncthreads();
    if (lane == 0) sh.parts[warp] = sm;
    __syncthreads();
  }
  if (warp == 0) {
    sm = warp_merge(sh.parts[lane % (NT / 32)], (NT / 32));
    if (lane == 0) sh.sum = sm;
  }
  if (blocks > 1) {
    cluster.sync();
    if (rank != 0) {
      cluster.barrier_arrive();
      cluster.barrier_wait();  // until the first block has read this one's shared memory
      return;
    }
    const int n = blocks * top_n;
    if (warp == 0) sm = warp_merge(*cluster.map_shared_rank(&sh.sum, lane % blocks), blocks);
    if (tid < n) sh.all[tid] = cluster.map_shared_rank(sh.top, tid / top_n)[tid % top_n];
    if (tid < (n & 1)) sh.all[n] = 0;  // pairs below
    cluster.barrier_arrive();
    __syncthreads();
    if (tid == 0) sh.sum = sm;
    if (tid < kMaxTop) sh.top[tid] = 0;
    __syncthreads();
    if (tid < n && sh.all[tid] != 0) {
      const uint64_t e = sh.all[tid];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < n; j += 2) {
        const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&sh.all[j]);
        r += (o.x > e) + (o.y > e);
      }
      if (r < top_n) sh.top[r] = e;
    }
  }
  __syncthreads();
  // ---- results
  const Softmax sum = sh.sum;
  const float log_z = sum.z != sum.z ? sum.z : log2f(sum.z);
  const bool masked = sum.m == -INFINITY && sum.z == sum.z;  // every logit is -inf
  // Both results are differences of numbers of up to 16, which round to the wrong side of 0 by up to 1e-6
  // for a token that is nearly certain.  (Comparisons, which keep NaN.)
  auto logprob = [&](float x) {
    if (x == -INFINITY && sum.z == sum.z) return -INFINITY;
    const float p = x > -kHuge && usual(sum.m) ? (fmaf(x, kLog2e, -origin(sum.m)) - log_z) * kLn2
                                               : (x - sum.m) - log_z * kLn2;  // usual m: log z and its origin are below the rounding of x
    return p > 0.f ? 0.f : p;
  };
  if (tid == 0) {
    logprobs[row_at] = logprob(asked);
    const float entropy = (log_z - sum.s / sum.z) * kLn2;
    entropies[row_at] = masked || entropy < 0.f ? 0.f : entropy;
  }
  if (tid < top_n) {
    const uint64_t e = sh.top[tid];
    top_tokens[row_at * top_n + tid] = int(~uint32_t(e));
    top_logprobs[row_at * top_n + tid] = logprob(key_logit(uint32_t(e >> 32)));
  }
  if (blocks > 1) cluster.barrier_wait();  // completes the arrival above
}

template <typename T, int NT>
cudaError_t launch_logprobs_blocks(int blocks, const void* logits, int64_t row_stride, int64_t rows, int vocab,
                                   const int64_t* tokens, int top_n, float* logprobs, float* entropies,
                                   int64_t* top_tokens, float* top_logprobs, cudaStream_t stream) {
  return launch_dependent(token_logprobs_kernel<T, NT>, dim3(unsigned(rows * blocks)), NT, 0, blocks, stream,
                          static_cast<const T*>(logits), row_stride, vocab, tokens, top_n, logprobs, entropies,
                          top_tokens, top_logprobs);
}

template <typename T, typename... Args>
cudaError_t launch_logprobs(const void* logits, int64_t row_stride, int64_t rows, int vocab, Args... args) {
  // Up to a block of 512 threads for each half of an SM: those, and as many blocks a row as keep one an
  // SM and a full batch of loads a thread (64 rows of 151936: two blocks 11.3 us, one 13.5, four 12.3).
  // More rows: smaller blocks, whose barriers cost less, four an SM (512 rows: 35.6 us, with 512 threads
  // 39.3), and eight for short rows (2048 rows of 1000: 15.3 us, with 256 threads 20.2).
  if (rows <= 2 * 148) {
    int blocks = 1;
    while (blocks < kMaxCluster && 2 * rows * blocks <= 148 && vocab / (2 * blocks) >= 512 * kUnroll * Row<T>::kVec / 2)
      blocks *= 2;
    return launch_logprobs_blocks<T, 512>(blocks, logits, row_stride, rows, vocab, args...);
  }
  if (vocab >= 1024 * Row<T>::kVec) return launch_logprobs_blocks<T, 256>(1, logits, row_stride, rows, vocab, args...);
  return launch_logprobs_blocks<T, 128>(1, logits, row_stride, rows, vocab, args...);
}

}  // namespace
}  // namespace hl

using namespace hl;

extern "C" int hl_token_logprobs(const void* logits, int logits_fp32, int64_t row_stride, int64_t rows, int vocab,
                                 const int64_t* token_ids, int top_n, float* logprobs, float* entropies,
                                 int64_t* top_tokens, float* top_logprobs, void* stream) {
  clear_error();
  HL_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff && vocab > 0 && row_stride >= vocab,
               "hl_token_logprobs: bad logits shape");
  HL_CHECK_ARG(top_n >= 0 && top_n <= kMaxTop && top_n <= vocab, "hl_token_logprobs: top_n not in [0, min(%d, vocab)]",
               kMaxTop);
  if (rows == 0) return HL_OK;
  HL_CHECK_ARG(logits && token_ids && logprobs && entropies && (top_n == 0 || (top_tokens && top_logprobs)),
               "hl_token_logprobs: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      logits_fp32 ? launch_logprobs<float>(logits, row_stride, rows, vocab, token_ids, top_n, logprobs, entropies,
                                           top_tokens, top_logprobs, s)
                  : launch_logprobs<__nv_bfloat16>(logits, row_stride, rows, vocab, token_ids, top_n, logprobs,
                                                   entropies, top_tokens, top_logprobs, s);
  if (e != cudaSuccess) {
    set_error("hl_token_logprobs: launch failed: %s", cudaGetErrorString(e));
    return HL_ERR_CUDA;
  }
  HL_CHECK_LAUNCH("hl_token_logprobs");
  return HL_OK;
}
