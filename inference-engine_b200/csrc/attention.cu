// C entry points of the paged attention operators: argument checks, the choice
// of kernels and of the parts that a long row is split into.
#include <algorithm>

#include "attention.cuh"

namespace ie {
namespace attn {
namespace {

constexpr int kSms = 148;

int validate(const ie_attention_args& a, const char* who) {
  IE_CHECK(a.dtype == IE_DT_BF16 || a.dtype == IE_DT_F16 || a.dtype == IE_DT_F32,
           "%s: unsupported dtype %d", who, a.dtype);
  IE_CHECK(a.heads > 0 && a.kv_heads > 0 && a.heads % a.kv_heads == 0 && a.heads <= 65535,
           "%s: %d query heads over %d kv heads", who, a.heads, a.kv_heads);
  IE_CHECK(a.head_dim > 0 && a.head_dim <= IE_ATTENTION_MAX_HEAD_DIM,
           "%s: a head size of %d outside [1, %d]", who, a.head_dim, IE_ATTENTION_MAX_HEAD_DIM);
  IE_CHECK(a.tokens >= 0 && a.tokens < (1ll << 31) / 256, "%s: %lld query tokens", who,
           (long long)a.tokens);
  IE_CHECK(a.seqs >= 0 && a.seqs <= a.tokens + (1 << 20), "%s: %lld sequences", who,
           (long long)a.seqs);
  IE_CHECK(a.cu_seqlens_q || a.seqs == a.tokens,
           "%s: %lld tokens of %lld sequences need cu_seqlens_q", who, (long long)a.tokens,
           (long long)a.seqs);
  IE_CHECK(a.tokens == 0 || a.seqs > 0, "%s: tokens without a sequence", who);
  IE_CHECK(a.block_size > 0, "%s: a block size of %d", who, a.block_size);
  IE_CHECK(a.table_width >= 0 && a.table_width * (int64_t)a.block_size < (1ll << 31) - (1 << 16),
           "%s: a table of %lld blocks of %d", who, (long long)a.table_width, a.block_size);
  IE_CHECK(a.cache_slots >= 0 && a.cache_slots < (1ll << 31), "%s: %lld cache slots", who,
           (long long)a.cache_slots);
  IE_CHECK(a.max_query_len >= 0 && a.max_context_len >= 0, "%s: negative lengths", who);
  IE_CHECK(a.window >= 0 && a.sinks >= 0 && a.prefix_len >= 0,
           "%s: negative window, sinks or prefix", who);
  IE_CHECK(a.scale == a.scale && a.scale - a.scale == 0.0f, "%s: the scale is not finite", who);
  if (a.tokens == 0) return IE_OK;
  IE_CHECK(a.q && a.out && (a.block_tables || a.table_width == 0) && a.context_lens, "%s: null pointer", who);
  IE_CHECK(a.cache_slots == 0 || (a.k_cache && a.v_cache), "%s: null cache", who);
  const uintptr_t size = a.dtype == IE_DT_F32 ? 4 : 2;
  IE_CHECK(reinterpret_cast<uintptr_t>(a.q) % size == 0 &&
               reinterpret_cast<uintptr_t>(a.out) % size == 0 &&
               reinterpret_cast<uintptr_t>(a.k_cache) % size == 0 &&
               reinterpret_cast<uintptr_t>(a.v_cache) % size == 0,
           "%s: a tensor is not aligned to its type", who);
  IE_CHECK(a.out_token_stride >= (int64_t)a.heads * a.head_dim || a.tokens == 1,
           "%s: out rows overlap", who);
  return IE_OK;
}

Params base_params(const ie_attention_args& a) {
  Params p{};
  p.q = a.q;
  p.k = a.k_cache;
  p.v = a.v_cache;
  p.out = a.out;
  p.q_token = a.q_token_stride;
  p.q_head = a.q_head_stride;
  p.out_token = a.out_token_stride;
  p.slot_stride = a.slot_stride;
  p.head_stride = a.head_stride;
  p.tables = a.block_tables;
  p.table_stride = a.table_stride;
  p.context = a.context_lens;
  p.cu_q = a.cu_seqlens_q;
  p.tokens = (int)a.tokens;
  p.seqs = (int)a.seqs;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.group = a.heads / a.kv_heads;
  p.hd = a.head_dim;
  p.table_width = (int)a.table_width;
  p.pages = (int)(a.cache_slots / a.block_size);
  p.block = FastDiv((uint32_t)a.block_size);
  p.group_div = FastDiv((uint32_t)p.group);
  const int64_t most = 1 << 30;
  p.window = (int)std::min(a.window, most);
  p.sinks = (int)std::min(a.sinks, most);
  p.key_end = 0x7FFFFFFF;
  p.scale2 = a.scale * kLog2e;
  return p;
}

// Keys that the longest row sees.
int64_t longest(const ie_attention_args& a) {
  int64_t n = a.table_width * a.block_size;
  if (a.max_context_len > 0) n = std::min(n, a.max_context_len);
  if (a.window > 0) n = std::min(n, a.window + a.sinks);
  return n;
}

struct Plan {
  int simt_parts;      // parts of the SIMT kernel
  int slots;           // 0: written to out directly
};

Plan make_plan(const ie_attention_args& a) {
  Plan plan{};
  // enough CTAs for every SM's warps, at least 64 keys each
  const int64_t rows = a.tokens * a.heads;
  const int64_t want = (kSms * 16 + rows - 1) / rows;
  plan.simt_parts = (int)std::max<int64_t>(1, std::min(want, longest(a) / 64));
  plan.slots = plan.simt_parts > 1 ? plan.simt_parts : 0;
  return plan;
}

size_t part_bytes(const ie_attention_args& a, int slots) {
  return (size_t)a.tokens * a.heads * slots * (a.head_dim * 4 + 8);
}

int run(const ie_attention_args& a, const char* who, cudaStream_t s) {
  const Plan plan = make_plan(a);
  const size_t need = part_bytes(a, plan.slots);
  IE_CHECK(need == 0 || (a.workspace && a.workspace_bytes >= need),
           "%s: a workspace of %zu bytes < %zu", who, a.workspace_bytes, need);
  IE_CHECK(reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0, "%s: unaligned workspace", who);
  Params p = base_params(a);
  p.prefix = (int)std::min<int64_t>(a.prefix_len, 0x7FFFFFFF);
  p.parts = plan.simt_parts;
  p.slots = plan.slots;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)a.tokens * a.heads * plan.slots *
                                                       a.head_dim);
  int rc = launch_simt(p, a.dtype, s);
  if (!rc && plan.slots) rc = launch_join(p, a.dtype, s);
  return rc;
}

}  // namespace
}  // namespace attn
}  // namespace ie

using namespace ie;
using namespace ie::attn;

extern "C" size_t ie_attention_workspace_size(const ie_attention_args* a) {
  if (!a || validate(*a, "attention") || a->tokens == 0) return 0;
  return part_bytes(*a, make_plan(*a).slots);
}

extern "C" int ie_window_attention(const ie_attention_args* a, void* stream) {
  IE_CHECK(a, "window_attention: null args");
  if (int rc = validate(*a, "window_attention")) return rc;
  IE_CHECK(a->prefix_len == 0, "window_attention: a shared prefix has its own entry point");
  if (a->tokens == 0) return IE_OK;
  return run(*a, "window_attention", as_stream(stream));
}

extern "C" int ie_shared_prefix_attention(const ie_attention_args* a, void* stream) {
  IE_CHECK(a, "shared_prefix_attention: null args");
  if (int rc = validate(*a, "shared_prefix_attention")) return rc;
  IE_CHECK(a->window == 0 && a->sinks == 0,
           "shared_prefix_attention: a window hides the prefix from its sequences");
  IE_CHECK(a->prefix_len <= a->table_width * a->block_size,
           "shared_prefix_attention: a prefix of %lld keys in tables of %lld",
           (long long)a->prefix_len, (long long)(a->table_width * a->block_size));
  if (a->tokens == 0) return IE_OK;
  return run(*a, "shared_prefix_attention", as_stream(stream));
}
