// C entry points of the paged attention operators: argument checks, the choice
// of kernels and of the parts that a long row is split into.
#include <algorithm>

#include "attention.cuh"

namespace ie {
namespace attn {
namespace {

int validate(const ie_attention_args& a, const char* who) {
  IE_CHECK(a.dtype == IE_DT_BF16 || a.dtype == IE_DT_F16 || a.dtype == IE_DT_F32,
           "%s: unsupported dtype %d", who, a.dtype);
  IE_CHECK(a.heads > 0 && a.kv_heads > 0 && a.heads % a.kv_heads == 0 && a.heads <= 65535,
           "%s: %d query heads over %d kv heads", who, a.heads, a.kv_heads);
  IE_CHECK(a.head_dim > 0 && a.head_dim <= IE_ATTENTION_MAX_HEAD_DIM,
           "%s: a head size of %d outside [1, %d]", who, a.head_dim, IE_ATTENTION_MAX_HEAD_DIM);
  // the launches number (token, head, part) and (row tile, head, part) in 31 bits; each
  // factor is held first, so that no product here wraps
  IE_CHECK(a.tokens >= 0 && a.tokens < (1ll << 24) && a.tokens * a.heads < (1ll << 31) / 128,
           "%s: %lld query tokens", who, (long long)a.tokens);
  IE_CHECK(a.seqs >= 0 && a.seqs <= a.tokens + (1 << 20) &&
               a.seqs * (int64_t)a.heads < (1ll << 31) / 256,
           "%s: %lld sequences", who, (long long)a.seqs);
  IE_CHECK(a.cu_seqlens_q || a.seqs == a.tokens,
           "%s: %lld tokens of %lld sequences need cu_seqlens_q", who, (long long)a.tokens,
           (long long)a.seqs);
  IE_CHECK(a.tokens == 0 || a.seqs > 0, "%s: tokens without a sequence", who);
  IE_CHECK(a.block_size > 0, "%s: a block size of %d", who, a.block_size);
  IE_CHECK(a.table_width >= 0 && a.table_width < (1ll << 31) &&
               a.table_width * a.block_size < (1ll << 31) - (1 << 16),
           "%s: a table of %lld blocks of %d", who, (long long)a.table_width, a.block_size);
  IE_CHECK(a.cache_slots >= 0 && a.cache_slots < (1ll << 31), "%s: %lld cache slots", who,
           (long long)a.cache_slots);
  IE_CHECK(a.max_query_len >= 0 && a.max_context_len >= 0, "%s: negative lengths", who);
  IE_CHECK(a.window >= 0 && a.sinks >= 0 && a.prefix_len >= 0,
           "%s: negative window, sinks or prefix", who);
  IE_CHECK(a.scale > 0.0f && a.scale - a.scale == 0.0f, "%s: the scale is not positive", who);
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
  p.cache_rows = (int)a.cache_slots;
  p.block = FastDiv((uint32_t)a.block_size);
  p.group_div = FastDiv((uint32_t)p.group);
  // a window of all that a table can address hides nothing
  const int64_t most = a.table_width * a.block_size;
  p.window = a.window < most ? (int)a.window : 0;
  p.sinks = (int)std::min(a.sinks, most);
  p.key_end = 0x7FFFFFFF;
  p.scale2 = a.scale * kLog2e;
  return p;
}

bool aligned16(const void* at) { return reinterpret_cast<uintptr_t>(at) % 16 == 0; }

// 16-bit rows that the tensor-core kernels read and write as 16-byte vectors.
bool tensor_cores(const ie_attention_args& a) {
  const int64_t strides = a.q_token_stride | a.q_head_stride | a.slot_stride | a.head_stride |
                          a.out_token_stride;
  return a.dtype != IE_DT_F32 && (a.head_dim == 64 || a.head_dim == 128) && strides % 8 == 0 &&
         aligned16(a.q) && aligned16(a.k_cache) && aligned16(a.v_cache) && aligned16(a.out) &&
         a.tokens * (a.heads / a.kv_heads) < (1ll << 31) - 512;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How one call runs: the kernels' parts of a row, and the slots they fill.
struct Plan {
  bool simt, decode, prefix;        // which kernels
  int simt_parts;
  int decode_parts, decode_per, decode_warps;     // one token per sequence, own keys
  bool twin, prefix_twin;           // row tiles: own keys, shared prefix
  int row_tiles, tile_parts, prefix_row_tiles, prefix_parts;
  int slots;                        // 0: a single part, written to out directly
  int merge;                        // the decode kernel takes up that many and writes out
};

// Cost, in keys, of `units` independent rows' worth of n keys in `parts` parts, with
// `wide` CTAs at once: the rounds of CTAs, where a CTA costs its keys (whole
// steps) and `fixed` more (its start and end).
int64_t rounds_cost(int64_t units, int64_t n, int64_t step, int64_t parts, int wide,
                    int64_t fixed) {
  return ceil_div(units * parts, wide) * (ceil_div(ceil_div(n, step), parts) * step + fixed);
}

// The cheapest number of parts, where joining them costs `join` + 4 a part.
int best_parts(int64_t units, int64_t n, int64_t step, int wide, int64_t fixed, int64_t join) {
  int64_t best = 1, least = rounds_cost(units, n, step, 1, wide, fixed);
  const int64_t most = std::min<int64_t>(n / step, 128);
  for (int64_t parts = 2; parts <= most; ++parts) {
    const int64_t cost = rounds_cost(units, n, step, parts, wide, fixed) + join + 4 * parts;
    if (cost < least) {
      least = cost;
      best = parts;
    }
  }
  return (int)best;
}

// Whether the CTAs of the decode kernel, one an SM with eight warps, all start at once.  A
// cluster lies in one GPC: 14 of eight CTAs fit (16 with eight warps each ran in two
// rounds: 2 sequences of 660, 10.8 us; with four, two CTAs an SM, 6.2), and 34 of four
// (36: 10.6 us and 8.3).
bool eight_warps(int64_t ctas, int64_t cluster) {
  return ctas <= (cluster == 8 ? 14 * 8 : cluster == 4 ? 34 * 4 : kSms);
}

// Parts of the decode kernel's rows and how they are joined.  Times are counted in
// keys of one CTA of four warps (13 ns on B200 for heads of 128), fitted to
// measurements over 1 to 64 sequences of 512 to 65536 keys:
//   - 160 such CTAs draw all of HBM; a batch's contexts are taken to be 0.7 of the
//     longest on average;
//   - up to 148 CTAs (see eight_warps) have eight warps and take 0.65 of the time; the
//     next 148 share SMs;
//   - within one round of CTAs the longest part ends it (0.3 for uneven lengths),
//     a second round that is short of half costs 0.6 of a CTA, and with more
//     rounds the scheduler evens the lengths out (0.2);
//   - of a batch's parts 0.7 have keys, and where only two CTAs share an SM (heads of
//     128) their second round costs 0.9 (2 sequences of 20000, 8 kv heads: 20 parts
//     29.9 us, 24 31.7, 28 41, 32 37);
//   - a start costs 96, a join within a cluster 70, a joining launch 400 and 16 a
//     part.
void choose_decode(const ie_attention_args& a, int64_t units, int64_t own, Plan& plan) {
  const double total = (a.seqs == 1 ? 1.0 : 0.7) * (double)(units * own) / 160;
  auto cost = [&](int64_t parts, int64_t cluster) {
    const int64_t ctas = units * parts;
    const double cta = (double)(ceil_div(ceil_div(own, 64), parts) * 64 + 96) *
                       (eight_warps(ctas, cluster) ? 0.65 : 1.0);
    if (ctas <= 2 * kSms) return std::max(total, cta) + 0.3 * cta;
    if (parts == 1 || a.seqs == 1 || a.head_dim < 128) return total + (ctas < 3 * kSms ? 0.6 : 0.2) * cta;
    const double busy = 0.7 * (double)ctas;
    return busy <= 2 * kSms ? std::max(total, cta) + 0.3 * cta
                            : total + (busy < 4 * kSms ? 0.9 : 0.2) * cta;
  };
  double least = cost(1, 1);
  plan.decode_parts = 1;
  plan.slots = 0;
  const int64_t most = std::min<int64_t>(ceil_div(own, 64), 128);
  for (int64_t parts = 2; parts <= most && units * parts <= 8 * kSms; ++parts) {
    const double join = 400.0 + 16.0 * parts;
    if (cost(parts, 1) + join < least) {
      least = cost(parts, 1) + join;
      plan.decode_parts = plan.slots = (int)parts;
    }
  }
  for (int parts = 2; parts <= kMaxDecodeCluster && units * parts <= 2 * kSms; parts *= 2) {
    if (cost(parts, parts) + 70 <= least) {
      least = cost(parts, parts) + 70;
      plan.decode_parts = parts;
      plan.slots = 0;
    }
  }
}

// A short prefix of few sequences: the decode kernel reads it for each of them, from L2
// after the first, and the tiles' launch and the parts' round trip are saved.  32/8 heads
// of 128, 60 keys of their own, us in one pass and in two: 4 sequences on 64: 4.5 and
// 10.3, on 1024: 8.0 and 10.8, on 4096: 13.8 and 14.8, 16 on 1024: 13.5 and 13.8; beyond the
// bound 8 on 4096: 21.2 and 15.2, 32 on 1024: 19.9 and 16.8.
bool prefix_in_decode(const ie_attention_args& a, int64_t units) {
  return !a.cu_seqlens_q && units * a.prefix_len <= 160 * 1024;
}

Plan make_plan(const ie_attention_args& a) {
  Plan plan{};
  const int64_t group = a.heads / a.kv_heads;
  int64_t keys = a.table_width * a.block_size;      // of the longest context
  if (a.max_context_len > 0) keys = std::min(keys, a.max_context_len);
  // (held to the keys before they are added)
  const int64_t reach = std::min(a.window, keys) + std::min(a.sinks, keys);
  const int64_t seen = a.window > 0 ? std::min(keys, reach) : keys;
  const int64_t per_tile = 128 / group;     // tokens of a row tile of the tensor cores
  // (a group of more than 128 heads has only the decode kernel)
  if (!tensor_cores(a) || (per_tile == 0 && (a.cu_seqlens_q || a.prefix_len > 0))) {
    // enough CTAs for every SM's warps, at least 64 keys each
    plan.simt = true;
    const int64_t rows = a.tokens * a.kv_heads * ceil_div(group, 8);
    plan.simt_parts = (int)std::max<int64_t>(
        1, std::min({ceil_div(kSms * 16, rows), seen / 64, (int64_t)1024}));
    plan.slots = plan.simt_parts > 1 ? plan.simt_parts : 0;
    return plan;
  }
  // (without cu_seqlens_q) the decode kernel's rows
  const int64_t units = a.seqs * a.kv_heads * ceil_div(group, 16);
  plan.prefix = a.prefix_len > 0 && !prefix_in_decode(a, units);
  if (plan.prefix) {
    plan.prefix_twin = a.tokens <= per_tile;
    plan.prefix_row_tiles = (int)ceil_div(a.tokens, plan.prefix_twin ? per_tile : 2 * per_tile);
    plan.prefix_parts = best_parts(plan.prefix_row_tiles * a.kv_heads, a.prefix_len, 128, kSms,
                                   256, 512);
  }
  const int64_t own = std::max<int64_t>(1, plan.prefix ? seen - a.prefix_len : seen);
  if (!a.cu_seqlens_q) {
    plan.decode = true;
    choose_decode(a, units, own, plan);
    const int64_t ctas = units * plan.decode_parts;
    // Eight warps an SM, as one CTA or two.  Rows that a window makes equally long also
    // fill one round of four (64 sequences, window 4096: 151 us against 157; uneven
    // ones lose: 32 sequences of up to 32768 448 against 356).
    const bool even = a.window > 0 && reach < keys;
    plan.decode_warps = eight_warps(ctas, plan.slots ? 1 : plan.decode_parts) ? 8
                        : even && plan.decode_parts == 1 && ctas > 2 * kSms && ctas <= 4 * kSms
                            ? 2
                            : 4;
    plan.decode_per = (int)(ceil_div(ceil_div(own, 64), plan.decode_parts) * 64);
  } else {
    // not known: twice the average (the kernel goes on to what lies beyond)
    const int64_t queries = std::min(
        a.tokens, a.max_query_len > 0 ? a.max_query_len : 2 * ceil_div(a.tokens, a.seqs));
    plan.twin = queries <= per_tile && own > 128;
    plan.row_tiles = (int)ceil_div(queries, plan.twin ? per_tile : 2 * per_tile);
    // a row tile sees the window of its first token and what lies up to its last
    const int64_t n = a.window > 0 ? std::min(own, seen + 2 * per_tile) : own;
    plan.tile_parts = best_parts(plan.row_tiles * a.seqs * a.kv_heads, n, 128, kSms, 256,
                                 plan.prefix ? 0 : 512);
    // work items are numbered in 31 bits; the kernel goes on to what lies beyond
    plan.row_tiles = (int)std::max<int64_t>(
        1, std::min<int64_t>(plan.row_tiles,
                             (1ll << 30) / (a.seqs * a.kv_heads * plan.tile_parts)));
    plan.slots = plan.tile_parts * (plan.twin ? 2 : 1);
  }
  if (plan.prefix) {
    const int prefix_slots = plan.prefix_parts * (plan.prefix_twin ? 2 : 1);
    if (plan.decode && plan.slots == 0) plan.merge = prefix_slots;
    plan.slots += prefix_slots;
  } else if (plan.slots == 1) {
    plan.slots = 0;
  }
  return plan;
}

// The workspace: the parts' sums in f32 from the first 32-byte boundary on (the tiles
// store that many), then their (m, l) pairs, 8-byte aligned whatever the head size.
size_t part_sums(const ie_attention_args& a, int slots) {
  return ((size_t)a.tokens * a.heads * slots * a.head_dim + 1) / 2 * 2;
}
size_t part_bytes(const ie_attention_args& a, int slots) {
  return slots ? 16 + part_sums(a, slots) * 4 + (size_t)a.tokens * a.heads * slots * 8 : 0;
}

int run(const ie_attention_args& a, void* workspace, size_t workspace_bytes, const char* who,
        cudaStream_t s) {
  const Plan plan = make_plan(a);
  const size_t need = part_bytes(a, plan.slots);
  IE_CHECK(need == 0 || (workspace && workspace_bytes >= need),
           "%s: a workspace of %zu bytes < %zu", who, workspace_bytes, need);
  IE_CHECK(aligned16(workspace), "%s: unaligned workspace", who);
  Params p = base_params(a);
  p.prefix = (int)std::min<int64_t>(a.prefix_len, 0x7FFFFFFF);
  p.slots = plan.slots;
  p.part_o = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + 31) / 32 * 32);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + part_sums(a, plan.slots));
  if (plan.simt) {
    p.parts = plan.simt_parts;
    if (int rc = launch_simt(p, a.dtype, s)) return rc;
  } else {
    if (plan.prefix) {
      Params shared = p;
      shared.key_end = p.prefix;
      if (int rc = launch_tiles(shared, a.dtype, true, plan.prefix_twin, plan.prefix_row_tiles,
                                plan.prefix_parts, s))
        return rc;
      p.key_start = p.prefix;
      p.slot0 = plan.prefix_parts * (plan.prefix_twin ? 2 : 1);
    }
    if (plan.decode) {
      p.parts = plan.decode_parts;
      p.merge = plan.merge;
      if (int rc = launch_decode(p, a.dtype, plan.decode_per, plan.decode_warps, plan.prefix, s))
        return rc;
      if (plan.merge) return IE_OK;
    } else if (int rc = launch_tiles(p, a.dtype, false, plan.twin, plan.row_tiles,
                                     plan.tile_parts, s)) {
      return rc;
    }
  }
  return plan.slots ? launch_join(p, a.dtype, s) : IE_OK;
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

extern "C" int ie_window_attention(const ie_attention_args* a, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  IE_CHECK(a, "window_attention: null args");
  if (int rc = validate(*a, "window_attention")) return rc;
  IE_CHECK(a->prefix_len == 0, "window_attention: a shared prefix has its own entry point");
  if (a->tokens == 0) return IE_OK;
  return run(*a, workspace, workspace_bytes, "window_attention", as_stream(stream));
}

extern "C" int ie_shared_prefix_attention(const ie_attention_args* a, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  IE_CHECK(a, "shared_prefix_attention: null args");
  if (int rc = validate(*a, "shared_prefix_attention")) return rc;
  IE_CHECK(a->window == 0 && a->sinks == 0,
           "shared_prefix_attention: a window hides the prefix from its sequences");
  IE_CHECK(a->prefix_len <= a->table_width * a->block_size,
           "shared_prefix_attention: a prefix of %lld keys in tables of %lld",
           (long long)a->prefix_len, (long long)(a->table_width * a->block_size));
  if (a->tokens == 0) return IE_OK;
  return run(*a, workspace, workspace_bytes, "shared_prefix_attention", as_stream(stream));
}
