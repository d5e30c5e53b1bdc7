// Paged attention for any element type, head size (up to 256) and alignment, and
// the joining of partial softmax results.
//
// One CTA takes one query token, up to eight query heads of one kv head and one
// part of the keys that the query sees, so K and V are read once for those
// heads.  Its four warps take groups of kKeys keys in turn, lanes across the head
// size.  The kKeys x kHeads dot products of a group are summed over the lanes
// together: a butterfly that hands half of the values on at each step ends with one
// sum a lane after 31 shuffles instead of 5 for each of the 32.  A lane then holds the
// score of one (head, key), and the softmax's running maximum and sum
//     m' = max(m, s_j),  l = l 2^(m - m') + sum 2^(s_j - m'),  o likewise
// are kept per head, all in f32.
//
// The tensor-core kernels serve 16-bit rows of 64 and 128 elements; this kernel
// serves the rest, f32 models above all.  It is bound by latency: a group's K loads, its
// sums over the lanes and its V loads follow one another, with nothing in flight
// between them.  8 f32 sequences of up to 8192, heads 14/2 x 64, take 49 us in a graph
// (39 for this kernel, where the SMs issue 1.56 of 4 instructions a cycle and wait for
// loads six cycles an instruction, then the join of the parts); 1024 tokens prefilled 195.
#include "attention.cuh"

namespace ie {
namespace attn {
namespace {

constexpr int kWarps = 4;

// v[0 .. N): values of every lane; afterwards the result is the sum over all lanes of
// v[lane / (32 / N)].
template <int N>
__device__ __forceinline__ float sum_lanes(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = N / 2, off = 16; off > 0; off >>= 1, n >>= 1) {
    if (n > 0) {
      const bool upper = lane & off;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float give = upper ? v[i] : v[i + n], keep = upper ? v[i + n] : v[i];
        v[i] = keep + __shfl_xor_sync(~0u, give, off);
      }
    } else {
      v[0] += __shfl_xor_sync(~0u, v[0], off);
    }
  }
  return v[0];
}

template <typename T, int NE, int kHeads>
__global__ void __launch_bounds__(kWarps * 32)
attention_simt_kernel(const Params p) {
  constexpr int kKeys = kHeads == 1 ? 8 : 32 / kHeads;    // keys a warp takes at once
  constexpr int N = kKeys * kHeads, kCopies = 32 / N;     // lanes that hold one score
  __shared__ float s_ml[kWarps][kHeads][2];
  __shared__ float s_o[kWarps][kHeads][NE * 32];
  const int t = blockIdx.x, part = blockIdx.y;
  const int chunks = (p.group + kHeads - 1) / kHeads;
  const int kvh = blockIdx.z / chunks, g0 = (blockIdx.z - kvh * chunks) * kHeads;
  const int h0 = kvh * p.group + g0, heads = min(kHeads, p.group - g0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seq = sequence_of(p, t);
  const int pos = position_of(p, seq, t);
  const Keys keys = keys_of(p, pos);
  // this part of the keys, in whole groups
  const int groups = (keys.n + kKeys - 1) / kKeys;
  const int per = (groups + p.parts - 1) / p.parts * kKeys;
  const int k0 = (int)min((int64_t)part * per, (int64_t)keys.n);
  const int k1 = (int)min((int64_t)k0 + per, (int64_t)keys.n);
  const int32_t* table = p.tables + (int64_t)seq * p.table_stride;
  const T* kc = static_cast<const T*>(p.k) + kvh * p.head_stride;
  const T* vc = static_cast<const T*>(p.v) + kvh * p.head_stride;

  float q[kHeads][NE], o[kHeads][NE];
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int d = lane + 32 * e;
      q[h][e] = h < heads && d < p.hd
                    ? to_f32<T>(static_cast<const T*>(
                          p.q)[t * p.q_token + (h0 + h) * p.q_head + d]) * p.scale2
                    : 0.0f;
      o[h][e] = 0.0f;
    }
  // of head lane / (kKeys * kCopies); l of this lane's keys alone
  float m = -INFINITY, l = 0.0f;
  for (int j = k0 + warp * kKeys; j < k1; j += kWarps * kKeys) {
    // lane i < kKeys looks key i up
    int slot = -1;
    if (lane < kKeys && j + lane < k1) {
      const int key = keys.at(j + lane);
      slot = cache_slot(p, key < p.prefix ? p.tables : table, key);
    }
    const uint32_t there = __ballot_sync(~0u, slot >= 0);
    if (!there) continue;
    float s[N];
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const int at = __shfl_sync(~0u, slot, i);
      float k[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int d = lane + 32 * e;
        k[e] = at >= 0 && d < p.hd ? to_f32<T>(kc[at * p.slot_stride + d]) : 0.0f;
      }
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        float x = q[h][0] * k[0];
#pragma unroll
        for (int e = 1; e < NE; ++e) x = fmaf(q[h][e], k[e], x);
        s[h * kKeys + i] = x;
      }
    }
    float mine = sum_lanes<N>(s);
    const int my_key = lane / kCopies % kKeys;
    const bool seen = there >> my_key & 1;
    if (!seen) mine = -INFINITY;
    float mn = mine;
#pragma unroll
    for (int off = kCopies; off < kKeys * kCopies; off <<= 1)
      mn = fmaxf(mn, __shfl_xor_sync(~0u, mn, off));
    mn = fmaxf(mn, m);
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float f = ex2(m - ref), w = seen ? ex2(mine - ref) : 0.0f;
    if (__any_sync(~0u, mn > m)) {
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const float fh = __shfl_sync(~0u, f, h * kKeys * kCopies);
#pragma unroll
        for (int e = 0; e < NE; ++e) o[h][e] *= fh;
      }
      l *= f;
      m = mn;
    }
    l += w;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      if (!(there >> i & 1)) continue;     // not seen: its K and V may hold anything
      const int at = __shfl_sync(~0u, slot, i);
      float v[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int d = lane + 32 * e;
        v[e] = d < p.hd ? to_f32<T>(vc[at * p.slot_stride + d]) : 0.0f;
      }
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const float wh = __shfl_sync(~0u, w, (h * kKeys + i) * kCopies);
#pragma unroll
        for (int e = 0; e < NE; ++e) o[h][e] = fmaf(wh, v[e], o[h][e]);
      }
    }
  }
  // a head's sum over its lanes
#pragma unroll
  for (int off = kCopies; off < kKeys * kCopies; off <<= 1)
    l += __shfl_xor_sync(~0u, l, off);
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (lane == h * kKeys * kCopies) {
      s_ml[warp][h][0] = m;
      s_ml[warp][h][1] = l;
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) s_o[warp][h][lane + 32 * e] = o[h][e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * p.hd; i += kWarps * 32) {
    const int h = i / p.hd, d = i - h * p.hd;
    float mt = s_ml[0][h][0];
    for (int w = 1; w < kWarps; ++w) mt = fmaxf(mt, s_ml[w][h][0]);
    const float ref = mt == -INFINITY ? 0.0f : mt;
    float lt = 0.0f, v = 0.0f;
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(s_ml[w][h][0] - ref);
      lt = fmaf(s_ml[w][h][1], f, lt);
      v = fmaf(s_o[w][h][d], f, v);
    }
    if (p.slots) {
      const int64_t at = ((int64_t)t * p.heads + h0 + h) * p.slots + p.slot0 + part;
      if (d == 0) p.part_ml[at] = make_float2(mt, lt);
      if (lt != 0.0f) p.part_o[at * p.hd + d] = v;
    } else {
      static_cast<T*>(p.out)[t * p.out_token + (int64_t)(h0 + h) * p.hd + d] =
          from_f32<T>(lt == 0.0f ? 0.0f : v / lt);
    }
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

template <typename T, int NE, int kHeads>
int simt(const Params& p, cudaStream_t s) {
  const dim3 grid((unsigned)p.tokens, (unsigned)p.parts,
                  (unsigned)(p.kv_heads * ((p.group + kHeads - 1) / kHeads)));
  attention_simt_kernel<T, NE, kHeads><<<grid, kWarps * 32, 0, s>>>(p);
  return launch_status("attention_simt_kernel");
}
template <typename T, int NE>
int simt(const Params& p, cudaStream_t s) {
  if (p.group == 1) return simt<T, NE, 1>(p, s);
  return p.group <= 4 ? simt<T, NE, 4>(p, s) : simt<T, NE, 8>(p, s);
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
