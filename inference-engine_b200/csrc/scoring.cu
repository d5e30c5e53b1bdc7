// Log probabilities of given tokens, the entropy of each row and its best
// alternatives, in one pass over the logits.
//
// For a row x of V logits, with m = max x, s = sum e^(x - m) and
// u = sum (x - m) e^(x - m):
//     log p(t) = (x_t - m) - log s          H = log s - u / s
// and the `top` largest logits, ties to the lower index.  The sums are kept in
// base 2 and f32 per thread, each relative to the thread's own running maximum
// (e^x = 2^(x log2 e)), and merged by the usual rescaling.
//
// The pass is bound by HBM (f32: one exponential per 4 bytes; bf16: near the
// exponentials' limit, 16 a cycle and SM: so a logit costs one of those, a clamp, the
// unpacking and half of a maximum, two FMAs and an addition on packed pairs, and
// nothing for the top list; the next batch's loads are in flight meanwhile).  For the list a thread keeps,
// per batch of four 16-byte vectors, only the batch's largest value in shared
// memory.  After the pass the lanes of the row form groups with distinct elements
// (the CTAs of a split row send one another their groups' largest values), so the
// top-th largest group maximum is a lower bound of the row's top-th element; only batches that reach it are read again (from L2, a warp a
// batch) and the few elements at or above it are ranked by counting, as 64-bit
// (value, lower index first) keys.  Where very many equal the bound - a vocabulary
// mask's -inf, a constant row - those above it are collected and the equal ones
// taken in index order.  The list does not depend on the order of the atomics.
//
// In a graph 4095 bf16 rows of 128256 take 187 us with one alternative (5.6 TB/s) and 168 without
// (6.25 TB/s); 64 f32 rows with 20 take 13.6 us, one row 7.7.
//
// Few rows are split over a thread-block cluster (up to 8 CTAs a row), merged
// through distributed shared memory: one launch, no workspace.  With a bound for the
// row a CTA finds about 2 top / 8 candidates, which its first CTA ranks as they are (a
// bound and a sorted list per CTA: 64 rows 16.2 us, 16 bf16 rows 11.3 against 7.9).
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "f32x2.cuh"

namespace ie {
namespace score_detail {

namespace cg = cooperative_groups;

// Threads of a CTA.  Several CTAs share an SM, so that one's selection runs under the
// others' loads: four of 256, or eight of 128 where rows are short and the selection
// weighs more (2304 f16 rows of 8297 with 14 alternatives: 44 us with 256, 30 with
// 128; 4095 bf16 rows of 20000 with 5: 70 and 48; of 128256 with 1: 189 and 203).
constexpr int kMany = 256, kFew = 128;
constexpr int kShortRow = 65536;
constexpr int kVecs = 4;          // 16-byte vectors of one thread's batch
constexpr int kMaxTop = IE_LOGPROBS_MAX_TOP;
constexpr int kCap = 1024;        // collected candidates, and batches to look at
constexpr int kMaxBatches = 16384;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = -1000.0f;  // 2^kFar == 0: bounds (x - m) where its weight is zero

constexpr int kMaxGroups = 256;
static_assert(2 * kMaxTop <= kFew && kMany <= kMaxGroups && 4 * kMaxTop <= kMaxGroups,
              "the bound is the top-th of at least 2 top group maxima");
static_assert(kMaxCluster * (kMany / 32) <= 64, "one warp merges every warp's sums");

// (value, lower index first) as an unsigned key; NaN ranks with -inf.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (!(x == x)) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.0f);   // -0 and +0 are equal
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  return ((uint64_t)ordered(x) << 32) | (0xFFFFFFFFu - index);
}

// Sums relative to the reference m, the maximum held to [-kFinite, kFinite]: weights are
// 2^(x log2 e - scaled(m)).  The argument is one FMA, so it is off by the rounding of
// scaled(m), the same for all of a reference's weights and taken back at the end; within
// the range that is 1/16 at most.  A finite mask (-1e30, a type's lowest value) then
// has weight 0 under any reference, and where the row's maximum itself is out of
// range its sums are computed again from differences (`far_sums`).
struct Sums {
  float m, s, u;
};
constexpr float kFinite = 1048576.0f;
// __fmul_rn: rounded once everywhere, never contracted into an FMA with a
// following difference (whose sums would then disagree on the reference)
__device__ __forceinline__ float scaled(float m) { return __fmul_rn(m, kLog2e); }
__device__ __forceinline__ Sums no_sums() { return {-kFinite, 0.0f, 0.0f}; }
// a's sums taken relative to the larger reference m
__device__ __forceinline__ Sums rescaled(Sums a, float m) {
  const float d = scaled(a.m) - scaled(m);
  const float f = ex2(d);
  return {m, a.s * f, f * (a.u + fmaxf(d, kFar) * a.s)};
}
__device__ __forceinline__ Sums merge(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  a = rescaled(a, m);
  b = rescaled(b, m);
  return {m, a.s + b.s, a.u + b.u};
}
// the sums of all lanes together, in every lane: relative to the largest maximum, then added
__device__ __forceinline__ Sums warp_merge(Sums a) {
  a = rescaled(a, unordered(__reduce_max_sync(~0u, ordered(a.m))));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(~0u, a.s, o);
    a.u += __shfl_xor_sync(~0u, a.u, o);
  }
  return a;
}
// the same of the first n entries of a shared array, n <= 64, by a whole warp
__device__ __forceinline__ Sums warp_merge(const Sums* all, int n, int lane) {
  return warp_merge(merge(lane < n ? all[lane] : no_sums(),
                          lane + 32 < n ? all[lane + 32] : no_sums()));
}

template <typename T> struct Vec {
  static constexpr int kPer = 16 / sizeof(T);
};
template <typename T>
__device__ __forceinline__ void unpack(uint4 v, float* x);
template <>
__device__ __forceinline__ void unpack<float>(uint4 v, float* x) {
  x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y);
  x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(uint4 v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void unpack<__half>(uint4 v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// The largest of a vector's elements and of `m`; NaN only if all are.
template <typename T>
struct Max {
  uint32_t m;      // a pair of T; f32: one
  __device__ __forceinline__ void start(uint4 v);
  __device__ __forceinline__ void add(uint4 v);
  __device__ __forceinline__ float value() const;
};
template <>
__device__ __forceinline__ void Max<float>::start(uint4 v) {
  m = __float_as_uint(fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                            fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))));
}
template <>
__device__ __forceinline__ void Max<float>::add(uint4 v) {
  Max<float> o;
  o.start(v);
  m = __float_as_uint(fmaxf(__uint_as_float(m), __uint_as_float(o.m)));
}
template <>
__device__ __forceinline__ float Max<float>::value() const { return __uint_as_float(m); }
template <typename H2>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  const H2 r = __hmax2(*reinterpret_cast<const H2*>(&a), *reinterpret_cast<const H2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
#define IE_HALF_MAX(T, H2, LOW, HIGH)                                             \
  template <>                                                                     \
  __device__ __forceinline__ void Max<T>::start(uint4 v) {                        \
    m = max2<H2>(max2<H2>(v.x, v.y), max2<H2>(v.z, v.w));                         \
  }                                                                               \
  template <>                                                                     \
  __device__ __forceinline__ void Max<T>::add(uint4 v) {                          \
    m = max2<H2>(m, max2<H2>(max2<H2>(v.x, v.y), max2<H2>(v.z, v.w)));            \
  }                                                                               \
  template <>                                                                     \
  __device__ __forceinline__ float Max<T>::value() const {                        \
    const H2 p = *reinterpret_cast<const H2*>(&m);                                \
    return fmaxf(LOW(p), HIGH(p));                                                \
  }
IE_HALF_MAX(__nv_bfloat16, __nv_bfloat162, __low2float, __high2float)
IE_HALF_MAX(__half, __half2, __low2float, __high2float)
#undef IE_HALF_MAX

struct Params {
  const void* logits;
  int64_t ld, rows, vocab;
  const int64_t* tokens;
  int top, batches;       // batches: stored batch maxima per thread of a CTA
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
};

// One row as 16-byte vectors from the aligned address at or below its start.
// A vector that reaches over either end of the row is read element by element.
template <typename T, int kThreads>
struct Row {
  static constexpr int kPer = Vec<T>::kPer;
  const T* x;
  int64_t vocab, nvec;
  int off;
  __device__ Row(const Params& p, int64_t r) {
    x = static_cast<const T*>(p.logits) + r * p.ld;
    off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    vocab = p.vocab;
    nvec = (vocab + off + kPer - 1) / kPer;
  }
  __device__ __forceinline__ int64_t first(int64_t v) const { return v * kPer - off; }
  // Iteration `it`'s vectors of this thread, packed; -inf where there is no element.
  __device__ __forceinline__ void load_batch(int64_t it, int64_t end, uint4 (&raw)[kVecs]) const {
    const int64_t v0 = it * (kThreads * kVecs);
    const int64_t e0 = first(v0), e1 = first(v0 + kThreads * kVecs);
    if (v0 + kThreads * kVecs <= end && e0 >= 0 && e1 <= vocab) {
      const uint4* at = reinterpret_cast<const uint4*>(x + e0) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) raw[i] = __ldg(at + i * kThreads);
    } else {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int64_t v = v0 + i * kThreads + threadIdx.x, e = first(v);
        if (v < end && e >= 0 && e + kPer <= vocab) {
          raw[i] = __ldg(reinterpret_cast<const uint4*>(x + e));
        } else {
          T f[kPer];
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            f[j] = v < end && e + j >= 0 && e + j < vocab ? x[e + j] : from_f32<T>(-INFINITY);
          raw[i] = *reinterpret_cast<const uint4*>(f);
        }
      }
    }
  }
  __device__ __forceinline__ void load(int64_t v, int64_t end, float (&f)[kPer]) const {
    const int64_t e = first(v);
    if (v < end && e >= 0 && e + kPer <= vocab) {
      unpack<T>(__ldg(reinterpret_cast<const uint4*>(x + e)), f);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        f[j] = v < end && e + j >= 0 && e + j < vocab ? to_f32<T>(x[e + j]) : -INFINITY;
    }
  }
};

// The sums of a row whose maximum lies outside (-kFinite, kFinite), by a whole CTA that
// reads the row twice: for the maximum, then for weights 2^((x - m) log2 e).  m itself is
// not finite where the row has +inf or nothing above -inf, and the sums are then NaN.
template <typename T, int kThreads>
__device__ Sums far_sums(const Row<T, kThreads>& row, float* shared) {
  constexpr int kPer = Vec<T>::kPer, kWarps = kThreads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float m = -INFINITY;
  for (int64_t v = tid; v < row.nvec; v += kThreads) {
    float f[kPer];
    row.load(v, row.nvec, f);
#pragma unroll
    for (int j = 0; j < kPer; ++j) m = fmaxf(m, f[j]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  __syncthreads();
  if (lane == 0) shared[warp] = m;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, shared[w]);
  float s = 0.0f, u = 0.0f;
  for (int64_t v = tid; v < row.nvec; v += kThreads) {
    float f[kPer];
    row.load(v, row.nvec, f);
    float vs = 0.0f, vu = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int64_t e = row.first(v) + j;
      if (e < 0 || e >= row.vocab) continue;
      const float d = (f[j] - m) * kLog2e, w = ex2(d);
      vs += w;
      vu = fmaf(w, fmaxf(d, kFar), vu);
    }
    s += vs;
    u += vu;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(~0u, s, o);
    u += __shfl_xor_sync(~0u, u, o);
  }
  __syncthreads();
  if (lane == 0) {
    shared[2 * warp] = s;
    shared[2 * warp + 1] = u;
  }
  __syncthreads();
  s = u = 0.0f;
  for (int w = 0; w < kWarps; ++w) {
    s += shared[2 * w];
    u += shared[2 * w + 1];
  }
  return {m, s, u};
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const Params p) {
  constexpr int kWarps = kThreads / 32;
  constexpr int kPer = Vec<T>::kPer;
  extern __shared__ uint32_t batch_max[];      // [batches][kThreads], ordered values
  __shared__ uint64_t cand[kCap];
  __shared__ uint32_t hits[kCap];              // batches that reach the bound
  __shared__ __align__(16) uint32_t group_max[kMaxGroups];   // of the whole row
  __shared__ uint64_t lists[kMaxCluster * kMaxTop];      // leader: every CTA's candidates
  __shared__ int counts[kMaxCluster];
  __shared__ Sums all_sums[kMaxCluster * kWarps];        // leader: every warp's sums
  __shared__ uint64_t warp_key[kWarps];
  __shared__ uint32_t bound;
  __shared__ int n_hits, n_cand;

  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  cluster.barrier_arrive();      // every CTA of the row has started before its memory is written
  const int64_t r = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T, kThreads> row(p, r);
  // this CTA's vectors: whole iterations of the row, spread evenly
  const int64_t iters = (row.nvec + kThreads * kVecs - 1) / (kThreads * kVecs);
  const int64_t it0 = iters * rank / ranks, it1 = iters * (rank + 1) / ranks;
  const int64_t end = min(row.nvec, it1 * kThreads * kVecs);

  Sums mine = no_sums();
  uint32_t tmax = 0;       // ordered; 0 is below every value
  // the given token's logit arrives meanwhile
  int64_t token = -1;
  float given = 0.0f;
  if (tid == 0) {
    n_hits = n_cand = 0;
    token = p.tokens[r];
    if (token >= 0 && token < p.vocab) given = to_f32<T>(row.x[token]);
  }
  uint4 raw[kVecs], ahead[kVecs];
  if (it0 < it1) row.load_batch(it0, end, ahead);
  for (int64_t it = it0; it < it1; ++it) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) raw[i] = ahead[i];
    if (it + 1 < it1) row.load_batch(it + 1, end, ahead);
    Max<T> big;
    big.start(raw[0]);
#pragma unroll
    for (int i = 1; i < kVecs; ++i) big.add(raw[i]);
    const float bm = big.value();
    if (bm > mine.m) mine = rescaled(mine, fminf(bm, kFinite));
    const uint64_t ref = f32x2(-scaled(mine.m), -scaled(mine.m));
    const uint64_t log2e = f32x2(kLog2e, kLog2e);
    uint64_t s = 0, u = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      float f[kPer];
      unpack<T>(raw[i], f);
#pragma unroll
      for (int j = 0; j < kPer; j += 2) {
        float d0, d1;
        unpack2(fma2(f32x2(f[j], f[j + 1]), log2e, ref), d0, d1);
        const uint64_t e = f32x2(ex2(d0), ex2(d1));
        s = add2(s, e);
        u = fma2(e, f32x2(fmaxf(d0, kFar), fmaxf(d1, kFar)), u);
      }
    }
    float lo, hi;
    unpack2(s, lo, hi);
    mine.s += lo + hi;
    unpack2(u, lo, hi);
    mine.u += lo + hi;
    if (p.top > 0) {
      // a batch past the end holds no element and ranks below every value
      const int64_t v0 = it * (kThreads * kVecs) + tid;
      const uint32_t o = v0 < end && row.first(v0) < row.vocab ? ordered(bm) : 0u;
      batch_max[(it - it0) * kThreads + tid] = o;
      tmax = max(tmax, o);
    }
  }

  // ---- every warp's sums to the row's first CTA
  mine = warp_merge(mine);
  cluster.barrier_wait();
  if (lane == 0) *cluster.map_shared_rank(&all_sums[rank * kWarps + warp], 0) = mine;

  const int top = p.top;
  int n = 0;               // candidates of this CTA; all with which the row's list is made
  if (top > 0) {
    // ---- the bound: the top-th largest of the maxima of groups of lanes over the row.
    // Twice as many groups as wanted leave few elements above it beyond those wanted.
    int per_group = 1;
    while (per_group < 32 && ranks * kThreads / (2 * per_group) >= 2 * top) per_group *= 2;
    const int mine_of = kThreads / per_group, groups = ranks * mine_of;
    uint32_t g = tmax;
    for (int o = 1; o < per_group; o <<= 1) g = max(g, __shfl_xor_sync(~0u, g, o));
    for (int q = tid % per_group; q < ranks; q += per_group)   // the group's lanes share the CTAs
      *cluster.map_shared_rank(&group_max[rank * mine_of + tid / per_group], q) = g;
    if (ranks > 1) cluster.sync(); else __syncthreads();
    for (int k = tid; k < groups; k += kThreads) {
      g = group_max[k];
      int above = 0, equal = 0;
      const uint4* all = reinterpret_cast<const uint4*>(group_max);
      for (int i = 0; i < groups / 4; ++i) {
        const uint4 o = all[i];
        above += (o.x > g) + (o.y > g) + (o.z > g) + (o.w > g);
        equal += (o.x == g) + (o.y == g) + (o.z == g) + (o.w == g);
      }
      if (above < top && above + equal >= top) bound = g;   // all that say so say the same
    }
    __syncthreads();
    const uint32_t reach = max(bound, 1u);       // 0: fewer groups with elements than wanted

    // Collects the elements at or above `from`; false: more than fit.
    auto collect = [&](uint32_t from) {
      for (int64_t it = it0; it < it1; ++it)
        if (batch_max[(it - it0) * kThreads + tid] >= from) {
          const int at = atomicAdd(&n_hits, 1);
          if (at < kCap) hits[at] = (uint32_t)((it - it0) * kThreads + tid);
        }
      __syncthreads();
      const int hit = min(n_hits, kCap);
      for (int i = warp; i < hit; i += kWarps) {      // a warp a batch, a lane an element
        const int64_t it = it0 + hits[i] / kThreads;
        const int64_t v = it * (kThreads * kVecs) + hits[i] % kThreads +
                          (int64_t)(lane / kPer) * kThreads;
        const int64_t e = row.first(v) + lane % kPer;
        if (lane < kVecs * kPer && v < end && e >= 0 && e < row.vocab) {
          const uint32_t o = ordered(to_f32<T>(row.x[e]));
          if (o >= from) {
            const int at = atomicAdd(&n_cand, 1);
            if (at < kCap) cand[at] = ((uint64_t)o << 32) | (0xFFFFFFFFu - (uint32_t)e);
          }
        }
      }
      __syncthreads();
      return n_hits <= kCap && n_cand <= kCap;
    };
    bool found = collect(reach);
    if (!found) {
      // Many elements equal the bound (a mask's -inf, equal logits): those above it, and as
      // many that equal it as are wanted, in index order.
      __syncthreads();
      if (tid == 0) n_hits = n_cand = 0;
      __syncthreads();
      found = collect(reach + 1) && n_cand <= kCap - kThreads - kMaxTop;
      if (found) {
        const int above = n_cand;
        const int64_t e0 = max(row.first(it0 * kThreads * kVecs), (int64_t)0);
        const int64_t e1 = min(row.first(end), row.vocab);
        for (int64_t e = e0 + tid; e - tid < e1; e += kThreads) {
          __syncthreads();
          if (n_cand - above >= top) break;          // the same for all: nobody adds now
          __syncthreads();
          if (e < e1 && ordered(to_f32<T>(row.x[e])) == reach) {
            const int at = atomicAdd(&n_cand, 1);
            cand[at] = ((uint64_t)reach << 32) | (0xFFFFFFFFu - (uint32_t)e);
          }
        }
        __syncthreads();
      }
    }
    n = n_cand;
    if (!found) {
      // too many elements above the bound (an adversarial order): one pass per rank
      uint64_t below = ~0ull;
      for (n = 0; n < top; ++n) {
        uint64_t bk = 0;
        for (int64_t v = it0 * kThreads * kVecs + tid; v < end; v += kThreads) {
          float f[kPer];
          row.load(v, end, f);
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const int64_t e = row.first(v) + j;
            if (e < 0 || e >= row.vocab) continue;
            const uint64_t ke = key_of(f[j], (uint32_t)e);
            if (ke < below && ke > bk) bk = ke;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) bk = max(bk, (uint64_t)__shfl_xor_sync(~0u, bk, o));
        __syncthreads();
        if (lane == 0) warp_key[warp] = bk;
        __syncthreads();
        bk = warp_key[0];
        for (int w = 1; w < kWarps; ++w) bk = max(bk, warp_key[w]);
        if (bk == 0) break;
        if (tid == 0) cand[n] = bk;
        below = bk;
      }
      __syncthreads();
    }
  }

  // ---- the candidates, `top` at most of a CTA, to the row's first CTA
  if (ranks > 1) {
    if (tid == 0) *cluster.map_shared_rank(&counts[rank], 0) = min(n, top);
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t k = cand[i];
      int above = i;
      if (n > top) {
        above = 0;
        for (int j = 0; j < n; ++j) above += cand[j] > k;
      }
      if (above < top) *cluster.map_shared_rank(&lists[rank * kMaxTop + above], 0) = k;
    }
    cluster.sync();
    if (rank != 0) return;    // nothing reads a remote CTA's memory after this point
    n = 0;
    for (int q = 0; q < ranks; ++q) {
      if (q % kWarps == warp)
        for (int i = lane; i < counts[q]; i += 32) cand[n + i] = lists[q * kMaxTop + i];
      n += counts[q];
    }
  }
  __syncthreads();
  Sums c = warp_merge(all_sums, ranks * kWarps, lane);
  // the weights' reference is the rounded product m log2 e, or m itself
  float off = fmaf(c.m, kLog2e, -scaled(c.m));
  if (fabsf(c.m) >= kFinite) {        // the same in every thread
    __syncthreads();                  // all have read all_sums
    c = far_sums<T, kThreads>(row, reinterpret_cast<float*>(all_sums));
    off = 0.0f;
  }
  const float log2s = log2f(c.s);
  const float logs = (log2s - off) * kLn2;      // log sum e^(x - m)
  if (tid == 0) {
    p.logprobs[r] = token >= 0 && token < p.vocab ? (given - c.m) - logs : -INFINITY;
    p.entropy[r] = (log2s - c.u / c.s) * kLn2;
  }
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t k = cand[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += cand[j] > k;
    if (above < top) {
      p.top_logprobs[r * top + above] = (unordered((uint32_t)(k >> 32)) - c.m) - logs;
      p.top_tokens[r * top + above] = (int64_t)(0xFFFFFFFFu - (uint32_t)k);
    }
  }
}

template <typename T, int kThreads>
int launch(Params p, cudaStream_t s) {
  constexpr int64_t per_iter = (int64_t)kThreads * kVecs * Vec<T>::kPer;
  const int64_t iters = (p.vocab + Vec<T>::kPer - 1 + per_iter - 1) / per_iter;
  // A row is split while the rows alone leave SMs idle and there is work for
  // another CTA, and where its batch maxima would not fit one CTA.
  int ranks = 1;
  while (ranks < kMaxCluster &&
         ((p.rows * ranks * 2 <= 148 * 4 && iters >= 2 * ranks) ||
          (iters + ranks - 1) / ranks * kThreads > kMaxBatches))
    ranks *= 2;
  p.batches = (int)((iters + ranks - 1) / ranks + 1);
  const size_t smem = p.top > 0 ? (size_t)p.batches * kThreads * 4 : 0;
  // what the longest row needs of a full cluster may be above kMaxBatches
  constexpr int64_t longest =
      (IE_LOGPROBS_MAX_VOCAB + Vec<T>::kPer - 1 + per_iter - 1) / per_iter;
  constexpr int64_t most = std::max<int64_t>(kMaxBatches / kThreads,
                                             (longest + kMaxCluster - 1) / kMaxCluster) + 1;
  auto kernel = token_logprobs_kernel<T, kThreads>;
  static std::atomic<int> allowed[kMaxDevices];
  if (int rc = allow_smem(kernel, (int)most * kThreads * 4, allowed)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.rows * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  IE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return IE_OK;
}

template <typename T>
int launch(const Params& p, cudaStream_t s) {
  // short rows, and enough of them to fill the SMs with the smaller CTAs
  return p.vocab <= kShortRow && p.rows >= 148 * 4 ? launch<T, kFew>(p, s)
                                                   : launch<T, kMany>(p, s);
}

}  // namespace score_detail
}  // namespace ie

using namespace ie;

extern "C" int ie_token_logprobs(const void* logits, int64_t ld, int32_t dtype, int64_t rows,
                                 int64_t vocab, const int64_t* tokens, int32_t top,
                                 float* logprobs, float* entropy, float* top_logprobs,
                                 int64_t* top_tokens, void* stream) {
  using namespace score_detail;
  IE_CHECK(rows >= 0 && rows <= (1ll << 27), "token_logprobs: %lld rows outside [0, 2^27]",
           (long long)rows);
  IE_CHECK(vocab >= 1 && vocab <= IE_LOGPROBS_MAX_VOCAB,
           "token_logprobs: a vocabulary of %lld outside [1, %d]", (long long)vocab,
           IE_LOGPROBS_MAX_VOCAB);
  IE_CHECK(top >= 0 && top <= kMaxTop && top <= vocab,
           "token_logprobs: %d alternatives outside [0, min(%d, vocabulary)]", top, kMaxTop);
  IE_CHECK(ld >= 0, "token_logprobs: a row stride of %lld", (long long)ld);
  IE_CHECK(dtype == IE_DT_F32 || dtype == IE_DT_BF16 || dtype == IE_DT_F16,
           "token_logprobs: unsupported dtype %d", dtype);
  if (rows == 0) return IE_OK;
  IE_CHECK(logits && tokens && logprobs && entropy, "token_logprobs: null pointer");
  IE_CHECK(top == 0 || (top_logprobs && top_tokens), "token_logprobs: null top list");
  IE_CHECK(reinterpret_cast<uintptr_t>(logits) % (dtype == IE_DT_F32 ? 4 : 2) == 0,
           "token_logprobs: logits are not aligned to their type");
  Params p{logits, ld, rows, vocab, tokens, top, 0, logprobs, entropy, top_logprobs, top_tokens};
  cudaStream_t s = as_stream(stream);
  if (dtype == IE_DT_F32) return launch<float>(p, s);
  if (dtype == IE_DT_BF16) return launch<__nv_bfloat16>(p, s);
  return launch<__half>(p, s);
}
