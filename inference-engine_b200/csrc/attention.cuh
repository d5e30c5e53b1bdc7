// Shared pieces of the paged attention kernels: the launch parameters, which
// keys a query sees, and where a key's row lies in the cache.
#pragma once

#include "common.cuh"
#include "f32x2.cuh"

namespace ie {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

// n / d for 0 <= n < 2^31 by a multiplication and a shift, d fixed on the host
// (Granlund and Montgomery, Division by Invariant Integers using Multiplication).
struct FastDiv {
  uint32_t mul = 1, shift = 0, d = 1;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((1ull << shift) < div) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - div)) / div + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    return (int)((__umulhi(mul, (uint32_t)n) + (uint32_t)n) >> shift);
  }
};

// The tensor-core kernels take a row's weights relative to 2^(its maximum - kBelow): an f16
// weight keeps its 11 bits down to 2^-14, so 7 more binades of a long flat tail are
// rounded like the rest (the raised-late maximum adds 2^8: 2^15 at most, below 65504).
// bf16 has the exponents of f32.
template <typename T> constexpr float kBelow = 0.0f;
template <> constexpr float kBelow<__half> = 7.0f;

struct Params {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_token, q_head;        // strides in elements
  int64_t out_token;
  int64_t slot_stride, head_stride;   // of both caches
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* context;
  const int32_t* cu_q;            // null: one token per sequence
  int tokens, seqs, heads, kv_heads, group, hd;
  int table_width, pages, cache_rows;   // rows: slots of the cache
  FastDiv block, group_div;
  int window, sinks;              // window 0: every earlier key
  int prefix;                     // keys below it are looked up in the first table row
  int key_start, key_end;         // only keys in [key_start, key_end) (a part of the softmax)
  float scale2;                   // softmax scale * log2 e
  // Parts of a row's softmax: [token * heads + head][slots] partial results, of
  // which this launch writes [slot0, slot0 + parts).  part_o holds the sum
  // relative to 2^m, part_ml (m, l); l = 0 means nothing was seen and part_o
  // is not written.  slots = 0: the launch covers every key and writes `out`.
  float* part_o;
  float2* part_ml;
  int slots, slot0, parts;
  int merge;       // decode: the parts [0, merge), written by the launch before, join its own
};

// Cache row of `key`, or -1 when the table names no page of the cache there.
__device__ __forceinline__ int cache_slot(const Params& p, const int32_t* table, int key) {
  const int page_no = p.block.div(key);
  if (page_no >= p.table_width) return -1;
  const int page = __ldg(table + page_no);
  if (page < 0 || page >= p.pages) return -1;
  return page * (int)p.block.d + (key - page_no * (int)p.block.d);
}

// Sequence of query token t: the last s with cu_q[s] <= t.
__device__ __forceinline__ int sequence_of(const Params& p, int t) {
  if (!p.cu_q) return t;
  int lo = 0, hi = p.seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(p.cu_q + mid) <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Context length of sequence s, held to what its table row can address.
__device__ __forceinline__ int context_of(const Params& p, int s) {
  const int64_t most = (int64_t)p.table_width * p.block.d;
  const int c = __ldg(p.context + s);
  return c < 0 ? 0 : (c < most ? c : (int)most);
}

// Position of query token t of sequence s; -1: it sees nothing (a token in front of the
// first sequence or behind the last is no sequence's).
__device__ __forceinline__ int position_of(const Params& p, int s, int t) {
  const int ctx = context_of(p, s);
  if (!p.cu_q) return ctx - 1;
  const int end = __ldg(p.cu_q + s + 1);
  return t >= __ldg(p.cu_q + s) && t < end ? max(ctx - (end - t), -1) : -1;
}

// The keys that a query at `pos` sees within [key_start, key_end), numbered
// 0 .. n-1: the sinks in front of the window first, then [lo, lo + n - ns).
struct Keys {
  int ns, lo, n;
  __device__ __forceinline__ int at(int i) const { return i < ns ? i : lo + (i - ns); }
};
__device__ __forceinline__ Keys keys_of(const Params& p, int pos) {
  Keys k;
  int lo = p.key_start;
  if (p.window > 0 && pos - p.window + 1 > lo) lo = pos - p.window + 1;
  k.lo = lo;
  k.ns = p.key_start == 0 ? min(p.sinks, lo) : 0;
  const int hi = min(pos + 1, p.key_end);
  k.n = k.ns + max(hi - lo, 0);
  if (pos < 0) k.n = k.ns = 0;
  return k;
}

// ---- shared memory -----------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// 16 bytes, or zeros when !ok (the source is then not read)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(ok ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Programmatic dependent launch: a kernel lets the next one of the stream start when all
// of its CTAs have said so, and that one waits before it touches what it writes.
__device__ __forceinline__ void pdl_trigger() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... A, typename... B>
int launch_pdl(void (*kernel)(A...), int64_t grid, int threads, int smem, cudaStream_t s,
               bool dependent, const B&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  IE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  return IE_OK;
}

constexpr int kSms = 148;
constexpr int kMaxDecodeCluster = 8;

// ---- launchers -------------------------------------------------------------
// One token per sequence, 16-bit rows of 64 or 128 elements (attention_decode.cu);
// part i of a row covers its visible keys [i * per, (i + 1) * per), the last one
// to the end.  Several parts without slots form clusters (at most 8 parts).
// `after_tiles`: the kernel before on the stream is launch_tiles' of the same call; this
// one starts beside it and waits for it where it needs its parts (p.merge), or at
// its end.
int launch_decode(const Params& p, int dtype, int per, int warps, bool after_tiles,
                  cudaStream_t s);
// Rows in tiles on the tensor cores (attention_sm100.cu): every sequence's queries
// over its own table, or (prefix) all queries over the first table row's keys below
// key_end.  Part i writes slot slot0 + i, or, twin, slots slot0 + 2 i and 2 i + 1.
int launch_tiles(const Params& p, int dtype, bool prefix, bool twin, int row_tiles, int parts,
                 cudaStream_t s);
uint32_t attention_status(bool clear);
// Any type, head size up to 256 and alignment (attention_simt.cu).
int launch_simt(const Params& p, int dtype, cudaStream_t s);
// out = the joined parts [0, slots) of every row.
int launch_join(const Params& p, int dtype, cudaStream_t s);

}  // namespace attn
}  // namespace ie
