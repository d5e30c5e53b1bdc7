// Paged attention for any element type, head size (up to 256) and alignment, and
// the joining of partial softmax results.
//
// One CTA takes one (query token, head) and one part of the keys that the
// query sees; its four warps take groups of four keys in turn, lanes across
// the head size, with the running maximum and sum of a softmax per warp:
//     m' = max(m, s_j),  l = l 2^(m - m') + sum 2^(s_j - m'),  o likewise,
// all in f32.  The tensor-core kernels serve 16-bit rows of 64 and 128
// elements; this kernel serves the rest (f32 models above all), where every
// query row reads the keys for itself, so it is bound by instruction issue
// (about 25 instructions a key and warp), not by memory.
#include "attention.cuh"

namespace ie {
namespace attn {
namespace {

constexpr int kWarps = 4;
constexpr int kKeys = 4;    // keys a warp takes at once

template <typename T, int NE>
__global__ void __launch_bounds__(kWarps * 32)
attention_simt_kernel(const Params p) {
  __shared__ float s_ml[kWarps][2];
  __shared__ float s_o[kWarps][NE * 32];
  const int t = blockIdx.x, part = blockIdx.y, h = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seq = sequence_of(p, t);
  const int pos = position_of(p, seq, t);
  const Keys keys = keys_of(p, pos);
  // this part of the keys, in whole groups
  const int groups = (keys.n + kKeys - 1) / kKeys;
  const int per = (groups + p.parts - 1) / p.parts * kKeys;
  const int k0 = min(part * per, keys.n), k1 = min(k0 + per, keys.n);
  const int kvh = p.group_div.div(h);
  const int32_t* table = p.tables + (int64_t)seq * p.table_stride;
  const T* q = static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head;
  const T* kc = static_cast<const T*>(p.k) + kvh * p.head_stride;
  const T* vc = static_cast<const T*>(p.v) + kvh * p.head_stride;

  float qv[NE], o[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int d = lane + 32 * i;
    qv[i] = d < p.hd ? to_f32<T>(q[d]) * p.scale2 : 0.0f;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int j = k0 + warp * kKeys; j < k1; j += kWarps * kKeys) {
    float s[kKeys];
    int64_t row[kKeys];
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const int key = keys.at(min(j + i, k1 - 1));
      const int slot = cache_slot(p, key < p.prefix ? p.tables : table, key);
      row[i] = j + i < k1 && slot >= 0 ? slot * p.slot_stride : -1;
      s[i] = 0.0f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int d = lane + 32 * e;
        if (row[i] >= 0 && d < p.hd) s[i] = fmaf(qv[e], to_f32<T>(kc[row[i] + d]), s[i]);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
#pragma unroll
      for (int i = 0; i < kKeys; ++i) s[i] += __shfl_xor_sync(~0u, s[i], off);
    float mn = m;
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
      if (row[i] >= 0) mn = fmaxf(mn, s[i]);
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float f = ex2(m - ref);
    m = mn;
    l *= f;
#pragma unroll
    for (int e = 0; e < NE; ++e) o[e] *= f;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      if (row[i] < 0) continue;     // not seen: its K and V may hold anything
      const float w = ex2(s[i] - ref);
      l += w;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int d = lane + 32 * e;
        if (d < p.hd) o[e] = fmaf(w, to_f32<T>(vc[row[i] + d]), o[e]);
      }
    }
  }
  if (lane == 0) {
    s_ml[warp][0] = m;
    s_ml[warp][1] = l;
  }
#pragma unroll
  for (int e = 0; e < NE; ++e) s_o[warp][lane + 32 * e] = o[e];
  __syncthreads();
  float mt = s_ml[0][0];
  for (int w = 1; w < kWarps; ++w) mt = fmaxf(mt, s_ml[w][0]);
  const float ref = mt == -INFINITY ? 0.0f : mt;
  float lt = 0.0f;
  for (int w = 0; w < kWarps; ++w) lt += s_ml[w][1] * ex2(s_ml[w][0] - ref);
  const int64_t r = (int64_t)t * p.heads + h;
  const int64_t at = r * p.slots + p.slot0 + part;
  if (p.slots && threadIdx.x == 0) p.part_ml[at] = make_float2(mt, lt);
  if (p.slots && lt == 0.0f) return;
  for (int d = threadIdx.x; d < p.hd; d += kWarps * 32) {
    float v = 0.0f;
    for (int w = 0; w < kWarps; ++w) v += s_o[w][d] * ex2(s_ml[w][0] - ref);
    if (p.slots) p.part_o[at * p.hd + d] = v;
    else
      static_cast<T*>(p.out)[t * p.out_token + (int64_t)h * p.hd + d] =
          from_f32<T>(lt == 0.0f ? 0.0f : v / lt);
  }
}

// Joins the parts of a row: o = sum o_i 2^(m_i - max m) / sum l_i 2^(m_i - max m), in
// slot order within each warp.  kSplit warps share a row's slots (few rows: what
// counts is the latency of the loads, so they are spread and issued eight at a
// time); its launch and reading overlap the tail of the kernel before it.
template <typename T, int NE, int kSplit>
__global__ void __launch_bounds__(128)
attention_join_kernel(const Params p) {
  constexpr int kRows = 4 / kSplit;             // rows of a CTA
  __shared__ float s_o[4][NE * 32];
  __shared__ float s_l[4];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kRows + warp / kSplit;
  const bool live = r < (int64_t)p.tokens * p.heads;
  const int part = warp % kSplit;
  float l = 0.0f, acc[NE] = {};
  if (live) {
    const float2* ml = p.part_ml + r * p.slots;
    float m = -INFINITY;
    for (int i = lane; i < p.slots; i += 32) m = fmaxf(m, ml[i].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const float ref = m == -INFINITY ? 0.0f : m;
    for (int i0 = 0; i0 < p.slots; i0 += 32) {
      // lane i: the weight and the sum of slot i0 + i (0: nothing was seen there)
      const float2 x = i0 + lane < p.slots ? ml[i0 + lane] : make_float2(-INFINITY, 0.0f);
      const float w = x.y == 0.0f ? 0.0f : ex2(x.x - ref);
      const int n = min(32, p.slots - i0);
      constexpr int kAtOnce = 8;
      for (int i = part; i < n; i += kSplit * kAtOnce) {
        float v[kAtOnce][NE], wi[kAtOnce], li[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const int q = i + u * kSplit;
          wi[u] = __shfl_sync(~0u, w, q & 31);
          li[u] = __shfl_sync(~0u, x.y, q & 31);
          const bool there = q < n && li[u] != 0.0f;     // otherwise nothing was written
          if (!there) li[u] = wi[u] = 0.0f;
          const float* o = p.part_o + (r * p.slots + i0 + q) * p.hd;
#pragma unroll
          for (int e = 0; e < NE; ++e)
            v[u][e] = there && lane + 32 * e < p.hd ? __ldcg(o + lane + 32 * e) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          l = fmaf(li[u], wi[u], l);
#pragma unroll
          for (int e = 0; e < NE; ++e) acc[e] = fmaf(v[u][e], wi[u], acc[e]);
        }
      }
    }
  }
  if (kSplit > 1) {
#pragma unroll
    for (int e = 0; e < NE; ++e) s_o[warp][lane + 32 * e] = acc[e];
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int q = 1; q < kSplit; ++q) {
      l += s_l[warp + q];
#pragma unroll
      for (int e = 0; e < NE; ++e) acc[e] += s_o[warp + q][lane + 32 * e];
    }
  }
  if (!live) return;
  const int64_t t = r / p.heads, h = r - t * p.heads;
  T* out = static_cast<T*>(p.out) + t * p.out_token + h * p.hd;
#pragma unroll
  for (int e = 0; e < NE; ++e)
    if (lane + 32 * e < p.hd) out[lane + 32 * e] = from_f32<T>(l == 0.0f ? 0.0f : acc[e] / l);
}

template <typename T, int NE>
int simt(const Params& p, cudaStream_t s) {
  const dim3 grid((unsigned)p.tokens, (unsigned)p.parts, (unsigned)p.heads);
  attention_simt_kernel<T, NE><<<grid, kWarps * 32, 0, s>>>(p);
  return launch_status("attention_simt_kernel");
}
template <typename T, int NE>
int join(const Params& p, cudaStream_t s) {
  const int64_t rows = (int64_t)p.tokens * p.heads;
  // an early launch pays where the join is short; the CTAs of a long one only wait on SMs
  // that others could use (2048 rows of 18 parts: 30 us with the tiles before it,
  // 26 without)
  if (rows <= kSms * 8)
    return launch_pdl(attention_join_kernel<T, NE, 4>, rows, 128, 0, s, true, p);
  return launch_pdl(attention_join_kernel<T, NE, 1>, (rows + 3) / 4, 128, 0, s, false, p);
}
template <typename T>
int by_size(const Params& p, bool joins, cudaStream_t s) {
  if (p.hd <= 32) return joins ? join<T, 1>(p, s) : simt<T, 1>(p, s);
  if (p.hd <= 64) return joins ? join<T, 2>(p, s) : simt<T, 2>(p, s);
  if (p.hd <= 128) return joins ? join<T, 4>(p, s) : simt<T, 4>(p, s);
  return joins ? join<T, 8>(p, s) : simt<T, 8>(p, s);
}
int by_type(const Params& p, int dtype, bool joins, cudaStream_t s) {
  if (dtype == IE_DT_F32) return by_size<float>(p, joins, s);
  if (dtype == IE_DT_BF16) return by_size<__nv_bfloat16>(p, joins, s);
  return by_size<__half>(p, joins, s);
}

}  // namespace

int launch_simt(const Params& p, int dtype, cudaStream_t s) { return by_type(p, dtype, false, s); }
int launch_join(const Params& p, int dtype, cudaStream_t s) { return by_type(p, dtype, true, s); }

}  // namespace attn
}  // namespace ie
