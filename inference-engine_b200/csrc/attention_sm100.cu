// Paged attention of many query rows on the tensor cores (tcgen05), bf16 / f16
// with heads of 64 or 128 elements: prefill (whole or chunked, with the sliding
// window and its sinks) and the shared-prefix part of a batch's attention.
//
// Rows are (query token, query head of one kv head) pairs, so the heads that
// share a kv head share its tiles: a tile of 128 rows covers 128 / group
// tokens.  One CTA per SM, persistent, works on two row tiles at a time
// ("pair"), or, where there are at most 128 rows, on one row tile whose key
// tiles alternate between two independent softmax streams ("twin"; the
// streams are parts of the row's softmax and are joined with the others).  Per tile of
// 128 keys:
//     S = Q K^T     Q, K in shared memory, S in TMEM (f32)
//     P = 2^(scale2 S - m), rounded to the element type, over S in TMEM
//     O += P V      P from TMEM, V in shared memory read MN-major, O in TMEM
// While one stream's softmax runs on its four warps the tensor cores work on
// the other's products.  The roles: warps 0-3 and 4-7 softmax of the two
// streams (a row per thread: no shuffles), warps 8-11 load, warp 12 issues.
//
// The sinks and the window of a row tile are one run of "virtual" keys (the
// sinks, then the keys from the first one any row sees), so sinks take a few
// columns of the first tile instead of a tile of their own, and only tiles at
// the edges of the mask test their elements.
//
// K and V rows are gathered with cp.async, 16 bytes a lane, straight into the
// 128-byte-swizzled layout that the MMA descriptors name: pages of any size,
// one table lookup per key, zeros for rows that are not there.  An arrival on
// a stage's barrier follows the thread's own wait and a proxy fence, two
// stages behind the loads.
//
// Bound by the exponentials as much as by the tensor cores: a 128 x 128 tile
// costs 1024 cycles of MMA and 16384 exponentials, 1024 cycles of the SM's 16
// a cycle.  The maximum is raised only when a score passes it by more than
// 2^8, so the output is rarely rescaled (by its own softmax warps: the product
// it belongs to has finished by then).
//
// A key that some rows of a tile see and others do not enters the others'
// product with weight 0; a NaN or infinite V there would still poison them.  Rows
// that come out not finite are therefore computed again key by key, leaving out what
// they do not see.
//
// Every wait has a limit; a wait that runs out sets an error bit
// (ie_kernel_status) and all roles leave.
#include "attention.cuh"

namespace ie {
namespace attn {
namespace {

constexpr int kTile = 128;         // rows of a row tile, keys of a key tile
constexpr int kThreads = 512;
constexpr int kLoaders = 128;
constexpr float kLazy = 8.0f;
constexpr long long kWaitCycles = 4000000000ll;   // ~2 s
constexpr int kInvalidRing = 8;

__device__ uint32_t g_attention_status = 0;

enum Mode { kPrefill = 0, kPrefix = 1 };

struct TileParams {
  Params p;
  int mode;
  int twin;          // one row tile, two streams of key tiles
  int row_tiles;     // work tiles (256 rows, or 128 when twin) of a segment in the grid
  int segs;          // sequences (prefill) or 1 (prefix)
  int parts;         // key parts of a work tile
};

// ---- PTX ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// False once the limit has passed or another role has given up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* quit) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (mbar_try(bar, parity)) return true;
    if (*quit) return false;
    if (clock64() - t0 > kWaitCycles) {
      atomicOr(&g_attention_status, 1u);
      *quit = 1;
      return false;
    }
  }
}
// The same for a whole warp: all lanes get one answer.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* quit) {
  return __all_sync(~0u, mbar_wait(bar, parity, quit));
}
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
__device__ __forceinline__ void fence_proxy_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// 64 consecutive columns of this thread's lane; the registers are defined once
// the wait returns, so both are one statement.
__device__ __forceinline__ void tmem_ld64(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%2"
      "3,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%4"
      "4,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]),
        "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]),
        "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
        "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]),
        "=r"(r[62]), "=r"(r[63])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Shared-memory matrix descriptors, 128-byte swizzle, version 1.  K-major (Q, K):
// groups of 8 rows 1024 bytes apart (SBO; LBO unused).  MN-major (V): 64 elements
// along the head are adjacent, groups of 8 keys 1024 bytes apart (SBO), the next
// 64 elements 16384 bytes on (LBO).
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo) {
  constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)hi << 32) | ((lbo >> 4) << 16) | ((addr & 0x3FFFFu) >> 4);
}
// f32 accumulator, A and B of type T, M = 128, N = n; B MN-major or not.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  const uint32_t type = dtype_of<T>() == IE_DT_BF16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// ---- shared memory -------------------------------------------------------------
template <int HD>
struct Layout {
  static constexpr int kHalves = HD / 64;              // 64-element (128-byte) columns
  static constexpr int kTileBytes = kHalves * 16384;   // one tile of 128 rows
  static constexpr int kStages = HD == 128 ? 5 : 6;
  static constexpr int kQ = 0;                         // two row tiles
  static constexpr int kRing = 2 * kTileBytes;
  static constexpr int kControl = kRing + kStages * kTileBytes;
  static constexpr int kBytes = kControl + 2048 + 1024;   // + alignment of the base
};
struct Control {
  uint64_t full[8], empty[8], s_full[2], p_ready[2], o_done[2], q_free;
  int slots[2][kTile];                     // cache rows of a key tile
  alignas(16) uint32_t invalid[kInvalidRing][4];   // keys of a tile whose page is not there
  uint32_t tmem;
  int quit;
};
static_assert(sizeof(Control) <= 2048, "control block");

// ---- work ------------------------------------------------------------------------
// One work tile: rows [row0, row0 + 256 or 128) of a segment for one kv head, and the
// key tiles [j0, j1) of its virtual keys.  Every role derives it alike.
struct Work {
  int seg, kvh, part, row0, nrows;     // nrows: rows of the segment
  int tok0, ctx, ntok;                 // first token, context, tokens (prefill)
  int lo, ns, n;                       // virtual keys: ns sinks, then from lo
  int j0, j1;
};

__device__ __forceinline__ int rows_of_work(const TileParams& a) { return a.twin ? 128 : 256; }

// Segment of work item `item` and its first work tile; false: nothing there.
__device__ __forceinline__ bool segment(const TileParams& a, int item, Work& w, int& tile) {
  const Params& p = a.p;
  w.kvh = item % p.kv_heads;
  item /= p.kv_heads;
  w.seg = item % a.segs;
  item /= a.segs;
  w.part = item % a.parts;
  tile = a.row_tiles - 1 - item / a.parts;      // the longest contexts first
  if (a.mode == kPrefix) {
    w.tok0 = 0;
    w.ntok = p.tokens;
    w.ctx = 0;
  } else {
    w.tok0 = p.cu_q ? __ldg(p.cu_q + w.seg) : w.seg;
    w.ntok = p.cu_q ? __ldg(p.cu_q + w.seg + 1) - w.tok0 : 1;
    // a table of lengths that does not describe [0, tokens) reads and writes nothing
    if (w.tok0 < 0 || w.tok0 > p.tokens) w.ntok = 0;
    w.ntok = min(w.ntok, p.tokens - w.tok0);
    w.ctx = context_of(p, w.seg);
  }
  w.nrows = w.ntok * p.group;
  return w.nrows > tile * rows_of_work(a);
}
__device__ __forceinline__ void locate(const TileParams& a, Work& w, int tile) {
  const Params& p = a.p;
  w.row0 = tile * rows_of_work(a);
  if (a.mode == kPrefix) {
    w.lo = w.ns = 0;
    w.n = p.key_end;
  } else {
    const int t0 = p.group_div.div(w.row0);
    const int t1 = p.group_div.div(min(w.row0 + rows_of_work(a), w.nrows) - 1);
    const int first = max(w.ctx - w.ntok + t0, 0), last = w.ctx - w.ntok + t1;
    w.lo = p.key_start;
    if (p.window > 0) w.lo = max(w.lo, first - p.window + 1);
    w.ns = p.key_start == 0 ? min(p.sinks, w.lo) : 0;
    const int hi = min(last + 1, p.key_end);
    w.n = last < 0 ? 0 : w.ns + max(hi - w.lo, 0);
  }
  const int tiles = (w.n + kTile - 1) / kTile;
  w.j0 = (int)((int64_t)tiles * w.part / a.parts);
  w.j1 = (int)((int64_t)tiles * (w.part + 1) / a.parts);
}

// ---- a row computed key by key (see the top) ------------------------------------------
// Warp-wide: o, m, l of the row of query token t, head h at position pos over the
// key tiles of the work item (twin: of its stream `stream`).
template <typename T, int HD>
__device__ __noinline__ void row_again(const TileParams& a, const Work& w, int t, int h, int pos,
                                       int stream, float* m_out, float* l_out,
                                       float (&o)[HD / 32]) {
  const Params& p = a.p;
  const int lane = threadIdx.x & 31;
  const int32_t* table = p.tables + (a.mode == kPrefix ? 0 : (int64_t)w.seg * p.table_stride);
  const T* q = static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head;
  const T* kc = static_cast<const T*>(p.k) + w.kvh * p.head_stride;
  const T* vc = static_cast<const T*>(p.v) + w.kvh * p.head_stride;
  float qv[HD / 32];
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) {
    qv[e] = to_f32<T>(q[lane + 32 * e]) * p.scale2;
    o[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int j = w.j0; j < w.j1; ++j) {
    if (a.twin && ((j - w.j0) & 1) != stream) continue;
    for (int v = j * kTile; v < min((j + 1) * kTile, w.n); ++v) {
      const int key = v < w.ns ? v : w.lo + v - w.ns;
      if (key > pos || !(p.window == 0 || key > pos - p.window || key < p.sinks)) continue;
      const int slot = cache_slot(p, table, key);
      if (slot < 0) continue;
      const int64_t at = slot * p.slot_stride + lane;
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < HD / 32; ++e) s = fmaf(qv[e], to_f32<T>(kc[at + 32 * e]), s);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(~0u, s, off);
      const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
      const float f = ex2(m - ref), wgt = ex2(s - ref);
      m = mn;
      l = fmaf(l, f, wgt);
#pragma unroll
      for (int e = 0; e < HD / 32; ++e)
        o[e] = fmaf(wgt, to_f32<T>(vc[at + 32 * e]), o[e] * f);
    }
  }
  *m_out = m;
  *l_out = l;
}

// ---- roles ---------------------------------------------------------------------------
template <typename T, int HD>
__device__ void load_role(const TileParams& a, uint8_t* base, Control* c, int items) {
  using L = Layout<HD>;
  const Params& p = a.p;
  constexpr int kChunks = HD / 8;                  // 16-byte chunks of a row
  constexpr int kRows = kLoaders / kChunks;        // rows of one pass of the loaders
  const int t = threadIdx.x & (kLoaders - 1);
  const int chunk = t % kChunks, r0 = t / kChunks;
  const uint32_t ring = smem_u32(base + L::kRing);
  // byte offset of (row r0, chunk) in a tile; rows r0 + i * kRows follow at i * kRows * 128,
  // kRows being a multiple of the swizzle's 8 rows
  static_assert(kRows % 8 == 0, "swizzle period");
  const uint32_t lane_off = (chunk / 8) * 16384 + r0 * 128 + (((chunk & 7) ^ (r0 & 7)) << 4);
  const int64_t slot_bytes = p.slot_stride * 2;
  uint32_t item = 0;          // stages filled so far (K and V tiles alternate)
  uint32_t told = 0;          // stages whose arrival is done
  uint32_t qn = 0;            // work tiles loaded
  bool failed = false;        // a wait of this thread ran out

  // Barrier of the loaders that tells all of them whether any has failed, so that they
  // leave together.
  auto any_failed = [](bool mine) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)mine)
        : "memory");
    return any != 0;
  };
  auto tell = [&]() {
    fence_proxy_async();
    mbar_arrive(smem_u32(&c->full[told % L::kStages]));
    ++told;
  };
  auto flush = [&]() {
    cp_wait<0>();
    while (told != item) tell();
  };
  // waits until the stage of the next item is free
  auto acquire = [&]() {
    if (item < L::kStages) return true;
    const uint32_t bar = smem_u32(&c->empty[item % L::kStages]);
    const uint32_t parity = (item / L::kStages - 1) & 1;
    if (mbar_try(bar, parity)) return true;
    flush();                 // what waits for us must not wait for ever
    return mbar_wait(bar, parity, &c->quit);
  };
  auto commit = [&]() {
    cp_commit();
    ++item;
    if (item - told > 2) {
      cp_wait<2>();
      tell();
    }
  };

  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    Work w;
    int tile;
    if (!segment(a, it, w, tile)) continue;
    const int32_t* table = p.tables + (a.mode == kPrefix ? 0 : (int64_t)w.seg * p.table_stride);
    const uint8_t* kb = static_cast<const uint8_t*>(p.k) + (int64_t)w.kvh * p.head_stride * 2 +
                        chunk * 16;
    const uint8_t* vb = static_cast<const uint8_t*>(p.v) + (int64_t)w.kvh * p.head_stride * 2 +
                        chunk * 16;
    for (; tile * rows_of_work(a) < w.nrows; tile += a.row_tiles) {
      locate(a, w, tile);
      if (w.j0 >= w.j1) continue;
      auto slot_at = [&](int j) {
        const int v = j * kTile + t;
        if (j >= w.j1 || v >= w.n) return -2;
        return cache_slot(p, table, v < w.ns ? v : w.lo + v - w.ns);
      };
      int next = slot_at(w.j0);
      // the query rows; their arrival is that of the first K tile
      if (qn > 0) {
        const uint32_t bar = smem_u32(&c->q_free), parity = (qn - 1) & 1;
        if (!mbar_try(bar, parity)) {
          flush();
          failed = !mbar_wait(bar, parity, &c->quit);
        }
      }
      ++qn;
      const uint8_t* qb = static_cast<const uint8_t*>(p.q) + chunk * 16;
      for (int i = 0; i < rows_of_work(a) / kRows; ++i) {
        const int r = r0 + i * kRows, row = w.row0 + r;
        const bool ok = row < w.nrows;
        const int tok = ok ? p.group_div.div(row) : 0;
        const int g = ok ? row - tok * p.group : 0;
        const uint8_t* src = qb + ((w.tok0 + tok) * p.q_token +
                                   (int64_t)(w.kvh * p.group + g) * p.q_head) * 2;
        cp_async16(smem_u32(base + L::kQ) + (r / kTile) * L::kTileBytes + lane_off +
                       (i * kRows % kTile) * 128,
                   ok ? src : qb, ok);
      }
      for (int j = w.j0; j < w.j1; ++j) {
        const uint32_t n = item / 2;      // key tiles before this one
        int* slots = c->slots[n & 1];
        slots[t] = next;
        const uint32_t bad = __ballot_sync(~0u, next == -1);
        if ((t & 31) == 0) c->invalid[n % kInvalidRing][t >> 5] = bad;
        if (any_failed(failed)) return;
        next = slot_at(j + 1);
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          failed = failed || !acquire();
          if (failed) break;
          const uint32_t dst = ring + (item % L::kStages) * L::kTileBytes + lane_off;
          const uint8_t* src = kv ? vb : kb;
#pragma unroll
          for (int i = 0; i < kTile / kRows; ++i) {
            const int s = slots[r0 + i * kRows];
            cp_async16(dst + i * kRows * 128, src + (s < 0 ? 0 : s * slot_bytes), s >= 0);
          }
          commit();
        }
      }
    }
  }
  flush();
}

template <typename T, int HD>
__device__ void issue_role(const TileParams& a, uint8_t* base, Control* c, int items,
                           uint32_t tmem) {
  using L = Layout<HD>;
  const uint32_t q0 = smem_u32(base + L::kQ), ring = smem_u32(base + L::kRing);
  constexpr uint32_t kIdS = idesc<T>(kTile, false), kIdO = idesc<T>(HD, true);
  uint32_t item = 0;                  // stages consumed by finished work tiles
  uint32_t np[2] = {0, 0};            // p_ready phases waited for

  auto full = [&](uint32_t i) {
    return mbar_wait(smem_u32(&c->full[i % L::kStages]), (i / L::kStages) & 1, &c->quit);
  };
  auto p_ready = [&](int s) {
    const bool ok = mbar_wait(smem_u32(&c->p_ready[s]), np[s] & 1, &c->quit);
    ++np[s];
    return ok;
  };
  auto scores = [&](int s, int q, uint32_t i) {      // S_s = Q_q K_i^T
    const uint32_t k = ring + (i % L::kStages) * L::kTileBytes;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      const uint32_t off = (kk / 4) * 16384 + (kk % 4) * 32;
      mma_ss(tmem + s * kTile, desc(q0 + q * L::kTileBytes + off, 16), desc(k + off, 16), kIdS,
             kk > 0);
    }
    tc_commit(smem_u32(&c->s_full[s]));
  };
  auto product = [&](int s, uint32_t i, bool first) {   // O_s (+)= P_s V_i
    const uint32_t v = ring + (i % L::kStages) * L::kTileBytes;
#pragma unroll
    for (int kk = 0; kk < kTile / 16; ++kk)
      mma_ts(tmem + 2 * kTile + s * HD, tmem + s * kTile + kk * 8, desc(v + kk * 2048, 16384),
             kIdO, !first || kk > 0);
  };
  auto release = [&](uint32_t i) { tc_commit(smem_u32(&c->empty[i % L::kStages])); };

  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    Work w;
    int tile;
    if (!segment(a, it, w, tile)) continue;
    for (; tile * rows_of_work(a) < w.nrows; tile += a.row_tiles) {
      locate(a, w, tile);
      const int nt = w.j1 - w.j0;
      if (nt <= 0) continue;
      if (a.twin) {
        for (int i = 0; i < nt + 2; ++i) {
          const int s = i & 1;
          if (i >= 2) {       // the product of step i - 2, the same stream
            const uint32_t v = item + 2 * (i - 2) + 1;
            if (!p_ready(s) || !full(v)) return;
            tc_fence_after();
            product(s, v, i < 4);
            release(v);
            if (i >= nt) tc_commit(smem_u32(&c->o_done[s]));
          }
          if (i < nt) {
            const uint32_t k = item + 2 * i;
            if (!full(k)) return;
            tc_fence_after();
            scores(s, 0, k);
            release(k);
          }
          if (i == nt - 1) tc_commit(smem_u32(&c->q_free));
        }
      } else {
        const int streams = w.nrows - w.row0 > kTile ? 2 : 1;
        for (int j = 0; j <= nt; ++j) {
          const uint32_t k = item + 2 * j, v = k - 1;      // v: of key tile j - 1
          for (int s = 0; s < streams; ++s) {
            if (j > 0) {
              if (!p_ready(s) || !full(v)) return;
              tc_fence_after();
              product(s, v, j == 1);
              if (j == nt) tc_commit(smem_u32(&c->o_done[s]));
            }
            if (j < nt) {
              if (!full(k)) return;
              tc_fence_after();
              scores(s, s, k);
            }
          }
          if (j > 0) release(v);
          if (j < nt) release(k);
          if (j == nt - 1) tc_commit(smem_u32(&c->q_free));
        }
      }
      item += 2 * nt;
    }
  }
}

template <typename T, int HD>
__device__ void softmax_role(const TileParams& a, Control* c, int items, uint32_t tmem, int s) {
  const Params& p = a.p;
  const int r = threadIdx.x & (kTile - 1), lane = threadIdx.x & 31;
  const uint32_t lanes = (uint32_t)(r & ~31) << 16;       // this warp's TMEM lanes
  const uint32_t ts = tmem + lanes + s * kTile, to = tmem + lanes + 2 * kTile + s * HD;
  const float scale2 = p.scale2;
  uint32_t n_s = 0, n_o = 0;          // s_full and o_done phases waited for
  uint32_t tiles = 0;                 // key tiles of the work tiles before

  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    Work w;
    int tile;
    if (!segment(a, it, w, tile)) continue;
    for (; tile * rows_of_work(a) < w.nrows; tile += a.row_tiles) {
      locate(a, w, tile);
      const int row = w.row0 + (a.twin ? 0 : s * kTile) + r;
      const uint32_t tile0 = tiles;
      tiles += max(w.j1 - w.j0, 0);
      if (!a.twin && s == 1 && w.nrows - w.row0 <= kTile) continue;
      const bool live = row < w.nrows;
      const int tok = live ? p.group_div.div(row) : 0;
      const int t = w.tok0 + tok;
      const int head = w.kvh * p.group + (live ? row - tok * p.group : 0);
      int pos = -1;
      if (live) pos = a.mode == kPrefix ? position_of(p, sequence_of(p, t), t)
                                        : w.ctx - w.ntok + tok;
      // virtual key v is seen iff v <= vmax and (v >= vmin or v < sinks)
      const int shift = w.lo - w.ns;
      const int vmax = pos < 0 ? -1 : min(pos - shift, w.n - 1);
      const int vmin = p.window > 0 ? pos - p.window + 1 - shift : -1;

      float m = -INFINITY, l = 0.0f;
      int done = 0;
      for (int j = w.j0 + (a.twin ? s : 0); j < w.j1; j += a.twin ? 2 : 1) {
        if (!warp_wait(smem_u32(&c->s_full[s]), n_s & 1, &c->quit)) return;
        ++n_s;
        tc_fence_after();
        uint32_t raw[kTile];
        tmem_ld64(ts, raw);
        tmem_ld64(ts + 64, raw + 64);
        const int v0 = j * kTile;
        const uint4 bad = *reinterpret_cast<const uint4*>(c->invalid[(tile0 + (j - w.j0)) % kInvalidRing]);
        const bool whole = v0 + kTile - 1 <= vmax && (v0 >= vmin || v0 + kTile <= p.sinks) &&
                           (bad.x | bad.y | bad.z | bad.w) == 0;
        if (!__all_sync(~0u, whole)) {
          const uint32_t words[4] = {bad.x, bad.y, bad.z, bad.w};
#pragma unroll
          for (int i = 0; i < kTile; ++i) {
            const int v = v0 + i;
            const bool see = v <= vmax && (v >= vmin || v < p.sinks) &&
                             !(words[i / 32] >> (i % 32) & 1u);
            if (!see) raw[i] = 0xFF800000u;
          }
        }
        float mx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(raw[i]);
#pragma unroll
        for (int i = 4; i < kTile; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(raw[i]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
        if (__any_sync(~0u, top > m + kLazy)) {
          const float mn = fmaxf(m, top);
          const float f = mn == -INFINITY ? 1.0f : ex2(m - mn);
          m = mn;
          l *= f;
          if (done > 0) {      // S being there, every product before it has finished
#pragma unroll
            for (int h = 0; h < HD; h += 16) {
              uint32_t o[16];
              tmem_ld16(to + h, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st16(to + h, o);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i0 = 0; i0 < kTile; i0 += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float w0 = ex2(fmaf(__uint_as_float(raw[i0 + i]), scale2, -ref));
            const float w1 = ex2(fmaf(__uint_as_float(raw[i0 + i + 1]), scale2, -ref));
            sum[i & 2] += w0;
            sum[(i & 2) + 1] += w1;
            pk[i / 2] = pack2<T>(w0, w1);
          }
          tmem_st16(ts + i0 / 2, pk);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_u32(&c->p_ready[s]));
        ++done;
      }

      // ---- the row's result
      const int slot = p.slot0 + w.part * (a.twin ? 2 : 1) + (a.twin ? s : 0);
      const int64_t at = ((int64_t)t * p.heads + head) * p.slots + slot;
      T* out = static_cast<T*>(p.out) + (int64_t)t * p.out_token + (int64_t)head * HD;
      float inv = 0.0f, check = 0.0f;
      if (done > 0) {
        if (!warp_wait(smem_u32(&c->o_done[s]), n_o & 1, &c->quit)) return;
        ++n_o;
        tc_fence_after();
        inv = l == 0.0f ? 0.0f : (p.slots ? 1.0f : 1.0f / l);
        check = l * 0.0f;
      }
#pragma unroll
      for (int h = 0; h < HD; h += 64) {
        uint32_t o[64];
        if (done > 0) tmem_ld64(to + h, o);
        else
#pragma unroll
          for (int i = 0; i < 64; ++i) o[i] = 0u;
        if (l == 0.0f) {     // nothing seen: whatever the product held is not the row's
#pragma unroll
          for (int i = 0; i < 64; ++i) o[i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const float v = __uint_as_float(o[i]) * inv;
          check = fmaf(v, 0.0f, check);
          o[i] = __float_as_uint(v);
        }
        if (live && p.slots) {
          float4* dst = reinterpret_cast<float4*>(p.part_o + at * HD + h);
#pragma unroll
          for (int i = 0; i < 64; i += 4)
            dst[i / 4] = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]),
                                     __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
        } else if (live) {
          uint4* dst = reinterpret_cast<uint4*>(out + h);
#pragma unroll
          for (int i = 0; i < 64; i += 8) {
            uint32_t x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[e] = pack2<T>(__uint_as_float(o[i + 2 * e]), __uint_as_float(o[i + 2 * e + 1]));
            dst[i / 8] = make_uint4(x[0], x[1], x[2], x[3]);
          }
        }
      }
      if (done > 0) tc_fence_before();       // O has been read before the next P arrives
      if (live && p.slots) p.part_ml[at] = make_float2(m, l);

      uint32_t again = __ballot_sync(~0u, live && !(check == 0.0f));
      while (again) {
        const int src = __ffs(again) - 1;
        again &= again - 1;
        const int tt = __shfl_sync(~0u, t, src), hh = __shfl_sync(~0u, head, src);
        const int pp = __shfl_sync(~0u, pos, src);
        float o[HD / 32], m2, l2;
        row_again<T, HD>(a, w, tt, hh, pp, s, &m2, &l2, o);
        const int64_t at2 = ((int64_t)tt * p.heads + hh) * p.slots + slot;
        const float i2 = l2 == 0.0f ? 0.0f : 1.0f / l2;
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) {
          if (p.slots) p.part_o[at2 * HD + lane + 32 * e] = o[e];
          else
            static_cast<T*>(p.out)[(int64_t)tt * p.out_token + (int64_t)hh * HD + lane + 32 * e] =
                from_f32<T>(o[e] * i2);
        }
        if (p.slots && lane == 0) p.part_ml[at2] = make_float2(m2, l2);
      }
    }
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
attention_tile_kernel(const __grid_constant__ TileParams a) {
  using L = Layout<HD>;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* base = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  Control* c = reinterpret_cast<Control*>(base + L::kControl);
  const int warp = threadIdx.x >> 5;
  const int items = a.row_tiles * a.parts * a.segs * a.p.kv_heads;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) {
      mbar_init(smem_u32(&c->full[i]), kLoaders);
      mbar_init(smem_u32(&c->empty[i]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&c->s_full[s]), 1);
      mbar_init(smem_u32(&c->p_ready[s]), kTile);
      mbar_init(smem_u32(&c->o_done[s]), 1);
    }
    mbar_init(smem_u32(&c->q_free), 1);
    c->quit = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&c->tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = c->tmem;

  // 512 threads at 128 registers: 256 x 192 + 256 x 64 is the same total
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    softmax_role<T, HD>(a, c, items, tmem, warp >> 2);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp < 12) load_role<T, HD>(a, base, c, items);
    else if (warp == 12 && (threadIdx.x & 31) == 0) issue_role<T, HD>(a, base, c, items, tmem);
  }
  // every product issued has finished (the softmax warps waited for the last) unless a
  // wait ran out: then give what is in flight the time to end before TMEM goes
  cp_wait<0>();
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (c->quit) {
    if (warp == 12 && (threadIdx.x & 31) == 0) {
      mbar_init(smem_u32(&c->slots[0][0]), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      tc_commit(smem_u32(&c->slots[0][0]));
      const long long t0 = clock64();
      while (!mbar_try(smem_u32(&c->slots[0][0]), 0) && clock64() - t0 < kWaitCycles) {
      }
    }
    __syncthreads();
  }
  if (warp == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <typename T, int HD>
int launch(const TileParams& a, cudaStream_t s) {
  auto kernel = attention_tile_kernel<T, HD>;
  IE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   Layout<HD>::kBytes));
  const int64_t items = (int64_t)a.row_tiles * a.parts * a.segs * a.p.kv_heads;
  kernel<<<(unsigned)(items < kSms ? items : kSms), kThreads, Layout<HD>::kBytes, s>>>(a);
  return launch_status("attention_tile_kernel");
}

}  // namespace

int launch_tiles(const Params& p, int dtype, bool prefix, bool twin, int row_tiles, int parts,
                 cudaStream_t s) {
  TileParams a;
  a.p = p;
  a.mode = prefix ? kPrefix : kPrefill;
  a.twin = twin;
  a.row_tiles = row_tiles;
  a.segs = prefix ? 1 : p.seqs;
  a.parts = parts;
  if (dtype == IE_DT_BF16)
    return p.hd == 64 ? launch<__nv_bfloat16, 64>(a, s) : launch<__nv_bfloat16, 128>(a, s);
  return p.hd == 64 ? launch<__half, 64>(a, s) : launch<__half, 128>(a, s);
}

uint32_t attention_status(bool clear) {
  uint32_t v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attention_status, sizeof(v)) != cudaSuccess) return 0;
  if (clear) cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(zero));
  return v;
}

}  // namespace attn
}  // namespace ie
