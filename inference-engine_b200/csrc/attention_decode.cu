// Paged attention of one query token per sequence (decode), bf16 / f16 with heads
// of 64 or 128 elements.
//
// Every key and value of a kv head is read once for all the query heads that
// share it, so the kernel is bound by HBM: 4 flops per byte and query head,
// far below the tensor cores' rate.  The query heads of a kv head form the 16
// rows of an m16n8k16 product (more than 16 take several CTAs); its padded
// rows cost tensor time that is idle anyway, and tcgen05's 128-row tile would
// pad eight times more and keep the data path in shared memory and TMEM busy
// for nothing.
//
// A CTA takes one part of one sequence's visible keys for one kv head.  Its
// warps work alone: a warp loads 16 keys and values at a time into its own
// three-stage ring (cp.async, 16 bytes a lane, chunks XOR-swizzled by the row so
// that ldmatrix is conflict-free), and keeps its own running maximum, sum and
// output, joined at the end through shared memory.  No CTA barrier lies on the
// path, the eight warps of an SM (two CTAs of four, one of eight where there are no
// more CTAs than SMs, or four of two) keep 128 KB of loads in flight, and pages of
// any size cost one table lookup per key.  64 sequences, heads 32/8 x 128, window
// 4096 take 153 us in a graph, 6.5 TB/s; one sequence, window 1024, 7.1 us.
//
// The maximum is raised only when a score passes it by more than 2^8: the sums
// stay far inside f32 and the outputs are rescaled a few times a row instead of
// every step.  Weights are rounded to the element type for the product with
// V, the rounding that the tensor cores' operands impose; their sum is not.  A second
// product with what the rounding left would take the error of the output from that of two
// roundings to one (bf16: 2.3e-3 and 1.7e-3 of its norm); it cost 3 % at 64 sequences,
// window 4096 (151 and 156 us), 7 % at 64 of up to 4096 (105 and 113) and 11 % at 8 of up
// to 8192 (37 and 42), and is not made.  An f16 weight keeps its bits down to 2^-21 of the
// row's largest (kBelow).
//
// A few parts of a row form a thread-block cluster and are joined through
// distributed shared memory: one launch, no workspace.  A short prefix that the
// sequences share is read for each of them, through the first table row.  After a longer
// one the kernel runs beside the tiles that compute it, takes up their partial results at
// its end and writes the finished rows (a launch of its own for that took 10 of 49 us
// with 64 sequences and 16 parts).
#include <cooperative_groups.h>

#include "attention.cuh"

namespace ie {
namespace attn {
namespace {

constexpr int kStep = 16;     // keys of a step
constexpr int kStages = 3;
constexpr float kLazy = 8.0f;

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4],
                                                   uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                            uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int HD, int kWarps>
constexpr int smem_bytes() {
  return kWarps * kStages * kStep * HD * 2 * 2;
}

// Two elements of a finished row.
template <typename T>
__device__ __forceinline__ void store(const Params& p, int t, int head, int hd, int d, float a,
                                      float b, float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(p.out) + t * p.out_token + (int64_t)head * hd + d;
  out[0] = from_f32<T>(a * inv);
  out[1] = from_f32<T>(b * inv);
}

// kCluster: the parts of a row are the CTAs of one cluster and join on their own.
template <typename T, int HD, int kWarps, bool kCluster>
__global__ void __launch_bounds__(kWarps * 32, 8 / kWarps)
attention_decode_kernel(const Params p, const int per) {
  constexpr int kChunks = HD / 8;                 // 16-byte chunks of a row
  constexpr int kRowBytes = HD * 2;
  constexpr int kTile = kStep * kRowBytes;        // K or V of one stage
  constexpr int kRowsAtOnce = 32 / kChunks;       // rows one warp-wide copy covers
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_ml[kWarps][16][2];
  __shared__ float2 s_part[16];      // (m, l) of this CTA's part
  __shared__ float2 s_whole[16];     // merge: the row's reference and its sum
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row_groups = (p.group + 15) / 16;
  int b = blockIdx.x;
  const int part = b % p.parts;
  b /= p.parts;
  const int rg = b % row_groups;
  b /= row_groups;
  const int kvh = b % p.kv_heads;
  const int seq = b / p.kv_heads;                 // also the query token
  const Keys keys = keys_of(p, context_of(p, seq) - 1);
  const int rows = min(16, p.group - rg * 16);
  const int head0 = kvh * p.group + rg * 16;
  const int k0 = (int)min((int64_t)part * per, (int64_t)keys.n);
  const int k1 = part == p.parts - 1 ? keys.n : min(k0 + per, keys.n);
  const int64_t row0 = (int64_t)seq * p.heads + head0;

  // The join may be launched.  What it reads is written by this kernel and the one before
  // it: this one ends after both.
  pdl_trigger();
  if (!kCluster && !p.merge && k0 >= k1) {     // nothing of this row lies in this part
    if (p.slots) {
      if (threadIdx.x < rows)
        p.part_ml[(row0 + threadIdx.x) * p.slots + p.slot0 + part] = make_float2(-INFINITY, 0.0f);
    } else {
      T* out = static_cast<T*>(p.out) + seq * p.out_token + (int64_t)head0 * HD;
      for (int i = threadIdx.x; i < rows * HD; i += kWarps * 32) out[i] = from_f32<T>(0.0f);
    }
    pdl_wait();
    return;
  }

  // ---- the query rows as A fragments
  uint32_t qf[HD / 16][4];
  {
    const T* q = static_cast<const T*>(p.q) + seq * p.q_token + (int64_t)head0 * p.q_head;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = lane / 4 + (i & 1) * 8, c = kk * 16 + (lane % 4) * 2 + (i >> 1) * 8;
        qf[kk][i] = r < rows ? *reinterpret_cast<const uint32_t*>(q + r * p.q_head + c) : 0u;
      }
  }

  const uint32_t ring = smem_u32(smem) + warp * (kStages * 2 * kTile);
  const int32_t* table = p.tables + (int64_t)seq * p.table_stride;
  const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + (int64_t)kvh * p.head_stride * 2 +
                         (lane % kChunks) * 16;
  const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + (int64_t)kvh * p.head_stride * 2 +
                         (lane % kChunks) * 16;
  const int64_t slot_bytes = p.slot_stride * 2;
  const int steps = (k1 - k0 + kStep - 1) / kStep;
  const int mine = (steps - warp + kWarps - 1) / kWarps;    // steps of this warp

  // the cache row of key lane % 16 of this warp's step i (-1: not seen)
  auto slot_of = [&](int i) {
    const int key = k0 + (i * kWarps + warp) * kStep + (lane & 15);
    if (i >= mine || key >= k1) return -1;
    const int at = keys.at(key);
    return cache_slot(p, at < p.prefix ? p.tables : table, at);
  };
  auto load = [&](int i, int slot) {
    const uint32_t dst = ring + (i % kStages) * (2 * kTile);
#pragma unroll
    for (int j = 0; j < kStep / kRowsAtOnce; ++j) {
      const int r = j * kRowsAtOnce + lane / kChunks;
      const int s = __shfl_sync(~0u, slot, r);
      const uint32_t at = dst + r * kRowBytes + (((lane % kChunks) ^ (r & 7)) << 4);
      const int64_t off = s < 0 ? 0 : s * slot_bytes;
      cp_async16(at, kbase + off, s >= 0);
      cp_async16(at + kTile, vbase + off, s >= 0);
    }
  };

  float o[HD / 8][4] = {};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  uint32_t seen[kStages];          // which of a stage's keys are there
  int next = slot_of(0);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    seen[i] = __ballot_sync(~0u, next >= 0) & 0xFFFFu;
    if (i < mine) load(i, next);
    cp_commit();
    next = slot_of(i + 1);
  }
  seen[kStages - 1] = 0;
  for (int i = 0; i < mine; ++i) {
    const int ahead = i + kStages - 1;
    const uint32_t ahead_seen = __ballot_sync(~0u, next >= 0) & 0xFFFFu;
    if (ahead < mine) load(ahead, next);
    cp_commit();
    next = slot_of(ahead + 1);
    cp_wait<kStages - 1>();
    __syncwarp();
    const uint32_t kt = ring + (i % kStages) * (2 * kTile), vt = kt + kTile;
    const uint32_t bits = seen[0];

    // two chains of products for each 8 keys: a dependent product waits for the last
    float s[2][4] = {}, s2[2][4] = {};
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      const int r = (lane >> 4) * 8 + (lane & 7), c = kk * 2 + ((lane >> 3) & 1);
      uint32_t f[4];
      ldsm4(kt + r * kRowBytes + ((c ^ (r & 7)) << 4), f);
      mma<T>(kk & 1 ? s2[0] : s[0], qf[kk], f[0], f[1]);
      mma<T>(kk & 1 ? s2[1] : s[1], qf[kk], f[2], f[3]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] += s2[n][e];
    if (bits != 0xFFFFu) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(bits >> (n * 8 + (lane % 4) * 2 + (e & 1)) & 1u)) s[n][e] = -INFINITY;
    }
    float mx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(~0u, mx[h], 1));
      mx[h] = fmaf(fmaxf(mx[h], __shfl_xor_sync(~0u, mx[h], 2)), p.scale2, -kBelow<T>);
    }
    if (__any_sync(~0u, mx[0] > m[0] + kLazy || mx[1] > m[1] + kLazy)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float mn = fmaxf(m[h], mx[h]);
        const float f = mn == -INFINITY ? 1.0f : ex2(m[h] - mn);
        m[h] = mn;
        l[h] *= f;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          o[n][2 * h] *= f;
          o[n][2 * h + 1] *= f;
        }
      }
    }
    uint32_t pf[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float ref = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float w0 = ex2(fmaf(s[n][2 * h], p.scale2, -ref));
        const float w1 = ex2(fmaf(s[n][2 * h + 1], p.scale2, -ref));
        l[h] += w0 + w1;
        const T t0 = from_f32<T>(w0), t1 = from_f32<T>(w1);
        pf[n * 2 + h] = (uint32_t)*reinterpret_cast<const uint16_t*>(&t0) |
                        (uint32_t)*reinterpret_cast<const uint16_t*>(&t1) << 16;
      }
    }
#pragma unroll
    for (int n = 0; n < HD / 16; ++n) {
      const int r = ((lane >> 3) & 1) * 8 + (lane & 7), c = n * 2 + (lane >> 4);
      uint32_t f[4];
      ldsm4_trans(vt + r * kRowBytes + ((c ^ (r & 7)) << 4), f);
      mma<T>(o[2 * n], pf, f[0], f[1]);
      mma<T>(o[2 * n + 1], pf, f[2], f[3]);
    }
    __syncwarp();       // every lane has read the stage before it is loaded again
#pragma unroll
    for (int q = 0; q < kStages - 2; ++q) seen[q] = seen[q + 1];
    seen[kStages - 2] = ahead_seen;
  }
  cp_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(~0u, l[h], 1);
    l[h] += __shfl_xor_sync(~0u, l[h], 2);
  }

  // ---- join the warps
  __syncthreads();      // the rings are done with
  float* s_o = reinterpret_cast<float*>(smem) + warp * (16 * HD);
  if (lane % 4 == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s_ml[warp][lane / 4 + 8 * h][0] = m[h];
      s_ml[warp][lane / 4 + 8 * h][1] = l[h];
    }
  }
#pragma unroll
  for (int n = 0; n < HD / 8; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = lane / 4 + 8 * h;
      if (r < rows)
        *reinterpret_cast<float2*>(s_o + r * HD + n * 8 + (lane % 4) * 2) =
            make_float2(o[n][2 * h], o[n][2 * h + 1]);
    }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(smem);
  float* joined = reinterpret_cast<float*>(smem) + kWarps * 16 * HD;    // cluster: [16][HD]
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  // (m, l) of row r, and two of its elements relative to 2^m, over the warps of this CTA
  auto of_warps = [&](int r, int d, float& mt, float& lt, float2& v) {
    mt = s_ml[0][r][0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mt = fmaxf(mt, s_ml[w][r][0]);
    const float ref = mt == -INFINITY ? 0.0f : mt;
    lt = 0.0f;
    v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(s_ml[w][r][0] - ref);
      const float2 x = *reinterpret_cast<const float2*>(all + w * (16 * HD) + r * HD + d);
      lt = fmaf(s_ml[w][r][1], f, lt);
      v.x = fmaf(x.x, f, v.x);
      v.y = fmaf(x.y, f, v.y);
    }
  };
  // the same over the CTAs of the cluster, in order
  auto of_cluster = [&](int r, int d, float& mt, float& lt, float2& v) {
    mt = -INFINITY;
    for (int q = 0; q < p.parts; ++q) mt = fmaxf(mt, cluster.map_shared_rank(s_part, q)[r].x);
    const float ref = mt == -INFINITY ? 0.0f : mt;
    lt = 0.0f;
    v = make_float2(0.0f, 0.0f);
    for (int q = 0; q < p.parts; ++q) {
      const float2 ml = cluster.map_shared_rank(s_part, q)[r];
      const float2 x =
          *reinterpret_cast<const float2*>(cluster.map_shared_rank(joined, q) + r * HD + d);
      const float f = ex2(ml.x - ref);
      lt = fmaf(ml.y, f, lt);
      v.x = fmaf(x.x, f, v.x);
      v.y = fmaf(x.y, f, v.y);
    }
  };
  auto own = [&](int r, int d, float& mt, float& lt, float2& v) {
    if (kCluster) of_cluster(r, d, mt, lt, v);
    else of_warps(r, d, mt, lt, v);
  };
  if (kCluster) {
    for (int i = threadIdx.x; i < rows * (HD / 2); i += kWarps * 32) {
      const int r = i / (HD / 2), d = (i % (HD / 2)) * 2;
      float mt, lt;
      float2 v;
      of_warps(r, d, mt, lt, v);
      if (d == 0) s_part[r] = make_float2(mt, lt);
      *reinterpret_cast<float2*>(joined + r * HD + d) = v;
    }
    cluster.sync();
  }
  // ---- the parts of the launch before: their weights, [rows][merge], and the whole sum
  float* weight = joined + 16 * HD;
  if (p.merge) {
    pdl_wait();
    for (int r = warp; r < rows; r += kWarps) {
      const float2* ml = p.part_ml + (row0 + r) * p.slots;
      float mt, lt;
      float2 v;
      own(r, 0, mt, lt, v);
      float top = mt;
      for (int q = lane; q < p.merge; q += 32) top = fmaxf(top, __ldcg(&ml[q].x));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      for (int q = lane; q < p.merge; q += 32) {
        const float2 x = __ldcg(ml + q);
        const float w = x.y == 0.0f ? 0.0f : ex2(x.x - ref);
        weight[r * p.merge + q] = w;
        sum = fmaf(x.y, w, sum);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
      if (lane == 0) s_whole[r] = make_float2(ref, fmaf(lt, ex2(mt - ref), sum));
    }
    __syncthreads();
  }
  // ---- the result; each CTA of a cluster takes its share of the elements
  const int first = kCluster ? part * (kWarps * 32) : 0;
  const int stride = kCluster ? p.parts * (kWarps * 32) : kWarps * 32;
  for (int i = first + threadIdx.x; i < rows * (HD / 2); i += stride) {
    const int r = i / (HD / 2), d = (i % (HD / 2)) * 2;
    float mt, lt;
    float2 v;
    own(r, d, mt, lt, v);
    if (p.merge) {
      const float2 whole = s_whole[r];
      const float f = ex2(mt - whole.x);
      v.x *= f;
      v.y *= f;
      lt = whole.y;
      constexpr int kAtOnce = 8;
      const float* src = p.part_o + (row0 + r) * p.slots * HD + d;
      for (int q0 = 0; q0 < p.merge; q0 += kAtOnce) {
        float2 x[kAtOnce];
        float w[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          w[u] = q0 + u < p.merge ? weight[r * p.merge + q0 + u] : 0.0f;
          x[u] = make_float2(0.0f, 0.0f);
          if (w[u] != 0.0f)      // 0: nothing was written there
            x[u] = __ldcg(reinterpret_cast<const float2*>(src + (int64_t)(q0 + u) * HD));
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          v.x = fmaf(x[u].x, w[u], v.x);
          v.y = fmaf(x[u].y, w[u], v.y);
        }
      }
    }
    if (p.slots && !p.merge) {
      const int64_t at = (row0 + r) * p.slots + p.slot0 + part;
      if (d == 0) p.part_ml[at] = make_float2(mt, lt);
      *reinterpret_cast<float2*>(p.part_o + at * HD + d) = v;
    } else {
      store<T>(p, seq, head0 + r, HD, d, v.x, v.y, lt);
    }
  }
  if (kCluster) cluster.sync();      // the others have read this CTA's part
  pdl_wait();
}

template <typename T, int HD, int kWarps, bool kCluster>
int launch(const Params& p, int per, bool after_tiles, cudaStream_t s) {
  auto kernel = attention_decode_kernel<T, HD, kWarps, kCluster>;
  constexpr int kSmem = smem_bytes<HD, kWarps>();
  static std::atomic<int> allowed[kMaxDevices];
  if (int rc = allow_smem(kernel, kSmem, allowed)) return rc;
  const int64_t grid = (int64_t)p.seqs * p.kv_heads * ((p.group + 15) / 16) * p.parts;
  if (!kCluster) return launch_pdl(kernel, grid, kWarps * 32, kSmem, s, after_tiles, p, per);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_tiles ? 2 : 1;
  IE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p, per));
  return IE_OK;
}
template <typename T, int HD>
int launch(const Params& p, int per, int warps, bool after_tiles, cudaStream_t s) {
  const bool cluster = p.parts > 1 && (p.slots == 0 || p.merge > 0);
  if (cluster)
    return warps == 8 ? launch<T, HD, 8, true>(p, per, after_tiles, s)
                      : launch<T, HD, 4, true>(p, per, after_tiles, s);
  if (warps == 8) return launch<T, HD, 8, false>(p, per, after_tiles, s);
  if (warps == 4) return launch<T, HD, 4, false>(p, per, after_tiles, s);
  return launch<T, HD, 2, false>(p, per, after_tiles, s);
}

}  // namespace

int launch_decode(const Params& p, int dtype, int per, int warps, bool after_tiles,
                  cudaStream_t s) {
  if (dtype == IE_DT_BF16)
    return p.hd == 64 ? launch<__nv_bfloat16, 64>(p, per, warps, after_tiles, s)
                      : launch<__nv_bfloat16, 128>(p, per, warps, after_tiles, s);
  return p.hd == 64 ? launch<__half, 64>(p, per, warps, after_tiles, s)
                    : launch<__half, 128>(p, per, warps, after_tiles, s);
}

}  // namespace attn
}  // namespace ie
