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
// issue limit too, so a logit costs one max, one FMA, one ex2, one clamp and two
// accumulations and nothing for the top list).  For the list a thread keeps,
// per batch of four 16-byte vectors, only the batch's largest value in shared
// memory.  After the pass the largest of every four lanes form 128 groups with
// distinct elements, so the top-th largest group maximum T is a lower bound of
// the row's top-th element; only batches that reach T are read again (from L2),
// the few elements at or above T are collected and ranked by counting.
// Elements are ordered by (value, lower index first) as one 64-bit key, so equal
// logits - a vocabulary mask's -inf among them - cost no more than distinct
// ones and the list does not depend on the order of the atomics.
//
// Few rows are split over a thread-block cluster (up to 8 CTAs a row), merged
// through distributed shared memory: one launch, no workspace.
#include <cooperative_groups.h>

#include "common.cuh"

namespace ie {
namespace score_detail {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kVecs = 4;          // 16-byte vectors of one thread's batch
constexpr int kGroups = 128;      // four lanes each
constexpr int kMaxTop = IE_LOGPROBS_MAX_TOP;
constexpr int kCap = 2048;        // collected candidates
constexpr int kMaxBatches = 16384;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = -1000.0f;  // 2^kFar == 0: bounds (x - m) where its weight is zero

static_assert(kMaxTop < kGroups, "the threshold is the top-th group maximum");

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
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums relative to the maximum m: weights are 2^(x log2 e - scaled(m)).
struct Sums {
  float m, s, u;
};
// __fmul_rn: rounded once everywhere, never contracted into an FMA with a
// following difference (whose sums would then disagree on the reference)
__device__ __forceinline__ float scaled(float m) {
  return m == -INFINITY ? 0.0f : __fmul_rn(m, kLog2e);
}
// a's sums taken relative to the larger maximum m
__device__ __forceinline__ Sums rescaled(Sums a, float m) {
  const float d = a.m == -INFINITY ? -INFINITY : scaled(a.m) - scaled(m);
  const float f = ex2(d);
  return {m, a.s * f, f * (a.u + fmaxf(d, kFar) * a.s)};
}
__device__ __forceinline__ Sums merge(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  a = rescaled(a, m);
  b = rescaled(b, m);
  return {m, a.s + b.s, a.u + b.u};
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
template <typename T>
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

template <typename T>
__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const Params p) {
  constexpr int kPer = Vec<T>::kPer;
  extern __shared__ uint32_t batch_max[];      // [batches][kThreads], ordered values
  __shared__ uint64_t cand[kCap];
  __shared__ uint64_t group_key[kGroups];
  __shared__ uint64_t best[kMaxTop];           // this CTA's list, sorted
  __shared__ uint64_t all_best[kMaxCluster * kMaxTop];   // leader: every CTA's list
  __shared__ Sums all_sums[kMaxCluster];
  __shared__ Sums warp_sums[kWarps];
  __shared__ uint64_t warp_key[kWarps];
  __shared__ uint64_t thr;
  __shared__ int count;

  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  cluster.barrier_arrive();      // every CTA of the row has started before its memory is written
  const int64_t r = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T> row(p, r);
  // this CTA's vectors: whole iterations of the row, spread evenly
  const int64_t iters = (row.nvec + kThreads * kVecs - 1) / (kThreads * kVecs);
  const int64_t it0 = iters * rank / ranks, it1 = iters * (rank + 1) / ranks;
  const int64_t end = min(row.nvec, it1 * kThreads * kVecs);

  Sums mine{-INFINITY, 0.0f, 0.0f};
  uint32_t tmax = 0;       // ordered; 0 is below every value
  int tbatch = 0;
  if (tid == 0) count = 0;
  for (int64_t it = it0; it < it1; ++it) {
    const int64_t v0 = it * (kThreads * kVecs) + tid;
    float f[kVecs][kPer];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) row.load(v0 + i * kThreads, end, f[i]);
    float bm = f[0][0];
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int j = 0; j < kPer; ++j) bm = fmaxf(bm, f[i][j]);
    if (bm > mine.m) mine = rescaled(mine, bm);
    const float ref = scaled(mine.m);
    float s[2] = {0.0f, 0.0f}, u[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float d = fmaf(f[i][j], kLog2e, -ref);
        const float e = ex2(d);
        s[j & 1] += e;
        u[j & 1] = fmaf(e, fmaxf(d, kFar), u[j & 1]);
      }
    mine.s += s[0] + s[1];
    mine.u += u[0] + u[1];
    if (p.top > 0) {
      // a batch past the end holds no element and ranks below every value
      const uint32_t o = v0 < end && row.first(v0) < row.vocab ? ordered(bm) : 0u;
      batch_max[(it - it0) * kThreads + tid] = o;
      if (o > tmax) {
        tmax = o;
        tbatch = (int)(it - it0);
      }
    }
  }

  // ---- merged sums of the CTA
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums b{__shfl_xor_sync(~0u, mine.m, o), __shfl_xor_sync(~0u, mine.s, o),
           __shfl_xor_sync(~0u, mine.u, o)};
    mine = merge(mine, b);
  }
  if (lane == 0) warp_sums[warp] = mine;

  const int top = p.top;
  if (top > 0) {
    // ---- the threshold: the top-th largest of the group maxima
    uint64_t k = 0;
    if (tmax) {          // the first of this thread's elements that holds its maximum
      const int64_t v0 = (it0 + tbatch) * (kThreads * kVecs) + tid;
#pragma unroll
      for (int i = kVecs - 1; i >= 0; --i) {
        float f[kPer];
        row.load(v0 + i * kThreads, end, f);
#pragma unroll
        for (int j = kPer - 1; j >= 0; --j) {
          const int64_t e = row.first(v0 + i * kThreads) + j;
          if (v0 + i * kThreads < end && e >= 0 && e < row.vocab && ordered(f[j]) == tmax)
            k = ((uint64_t)tmax << 32) | (0xFFFFFFFFu - (uint32_t)e);
        }
      }
    }
    k = max(k, (uint64_t)__shfl_xor_sync(~0u, k, 1));
    k = max(k, (uint64_t)__shfl_xor_sync(~0u, k, 2));
    if ((tid & 3) == 0) group_key[tid >> 2] = k;
    __syncthreads();
    {
      // group g = tid / 4: its rank, counted over a quarter of the groups by each lane
      int above = 0;
#pragma unroll 8
      for (int i = 0; i < kGroups / 4; ++i) {
        const int g = (tid & 3) + 4 * i;
        const uint64_t o = group_key[g];
        above += o > k || (o == k && g < (tid >> 2));   // empty groups share the key 0
      }
      above += __shfl_xor_sync(~0u, above, 1);
      above += __shfl_xor_sync(~0u, above, 2);
      if ((tid & 3) == 0 && above == top - 1) thr = k;
    }
    __syncthreads();
    // ---- collect every element at or above it
    const uint64_t floor_key = max(thr, (uint64_t)1);
    const uint32_t floor_val = (uint32_t)(floor_key >> 32);
    for (int64_t it = it0; it < it1; ++it) {
      const uint32_t bm = batch_max[(it - it0) * kThreads + tid];
      if (bm == 0 || bm < floor_val) continue;
      const int64_t v0 = it * (kThreads * kVecs) + tid;
      // among equal values only lower indexes can still enter
      if (bm == floor_val && row.first(v0) > 0 &&
          (uint64_t)row.first(v0) > 0xFFFFFFFFu - (uint32_t)floor_key)
        continue;
      for (int i = 0; i < kVecs; ++i) {
        const int64_t v = v0 + i * kThreads;
        if (v >= end) break;
        float f[kPer];
        row.load(v, end, f);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int64_t e = row.first(v) + j;
          if (e < 0 || e >= row.vocab) continue;
          const uint64_t ke = key_of(f[j], (uint32_t)e);
          if (ke >= floor_key) {
            const int at = atomicAdd(&count, 1);
            if (at < kCap) cand[at] = ke;
          }
        }
      }
    }
    for (int i = tid; i < top; i += kThreads) best[i] = 0;
    __syncthreads();
    const int n = count;
    if (n <= kCap) {
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t mykey = cand[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += cand[j] > mykey;
        if (above < top) best[above] = mykey;
      }
    } else {
      // too many elements reach the bound (an adversarial order): one pass per rank
      uint64_t below = ~0ull;
      for (int t = 0; t < top; ++t) {
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
        if (tid == 0) best[t] = bk;
        below = bk;
        if (bk == 0) break;
      }
    }
  }
  __syncthreads();
  cluster.barrier_wait();

  // ---- merge the cluster's parts in rank order, on its first CTA
  if (tid == 0) {
    Sums c = warp_sums[0];
    for (int w = 1; w < kWarps; ++w) c = merge(c, warp_sums[w]);
    *cluster.map_shared_rank(&all_sums[rank], 0) = c;
  }
  if (ranks > 1) {
    for (int i = tid; i < top; i += kThreads)
      *cluster.map_shared_rank(&all_best[rank * kMaxTop + i], 0) = best[i];
    cluster.sync();
    if (rank != 0) return;    // nothing reads a remote CTA's memory after this point
  } else {
    for (int i = tid; i < top; i += kThreads) all_best[i] = best[i];
    __syncthreads();
  }
  Sums c = all_sums[0];
  for (int i = 1; i < ranks; ++i) c = merge(c, all_sums[i]);
  const float log2s = log2f(c.s);
  // log sum e^(x - m): the weights' reference is the rounded product m log2 e
  const float logs = (log2s - fmaf(c.m, kLog2e, -scaled(c.m))) * kLn2;
  if (tid == 0) {
    const int64_t t = p.tokens[r];
    p.logprobs[r] = t >= 0 && t < p.vocab ? (to_f32<T>(row.x[t]) - c.m) - logs : -INFINITY;
    p.entropy[r] = (log2s - c.u / c.s) * kLn2;
  }
  for (int i = tid; i < ranks * top; i += kThreads) {
    const uint64_t k = all_best[(i / top) * kMaxTop + i % top];
    if (k == 0) continue;
    int above = i;
    if (ranks > 1) {
      above = 0;
      for (int q = 0; q < ranks; ++q)
        for (int j = 0; j < top; ++j) above += all_best[q * kMaxTop + j] > k;
    }
    if (above < top) {
      p.top_logprobs[r * top + above] = (unordered((uint32_t)(k >> 32)) - c.m) - logs;
      p.top_tokens[r * top + above] = (int64_t)(0xFFFFFFFFu - (uint32_t)k);
    }
  }
}

template <typename T>
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
  auto kernel = token_logprobs_kernel<T>;
  // the attribute is per function and device: set whenever the default is exceeded
  if (smem > 16 * 1024)
    IE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)smem));
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
  IE_CHECK(ld >= vocab || rows <= 1, "token_logprobs: row stride %lld < vocabulary %lld",
           (long long)ld, (long long)vocab);
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
