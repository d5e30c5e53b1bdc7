// Paged attention of many query rows on the tensor cores (tcgen05), bf16 / f16
// with heads of 64 or 128 elements: prefill (whole or chunked, with the sliding
// window and its sinks) and the shared-prefix part of a batch's attention.
//
// Rows are (query token, query head of one kv head) pairs, so the heads that
// share a kv head share its tiles: a row tile is 128 / group whole tokens.  A work
// item is two row tiles ("pair") or, where one holds all tokens, one row tile
// whose key tiles alternate between two independent softmax streams ("twin": the
// streams are parts of the row's softmax, joined with the others).  Per stream
// and tile of 128 keys:
//     S = Q K^T     Q, K in shared memory, S in TMEM (f32)
//     P = 2^(scale2 S - m), rounded to the element type, over S in TMEM
//     O += P V      P from TMEM, V in shared memory read MN-major, O in TMEM
// While one stream's softmax runs on its four warps (a row per thread: no
// shuffles) the tensor cores work on the other's products; the first half of the
// weights is handed over while the exponentials of the second run.  Two streams
// are what TMEM holds: S and O of both take its 512 columns.
//
// The sinks and the window of a row tile are one run of "virtual" keys (the
// sinks, then the keys from the first one any row sees, both in whole boxes), so
// sinks take a few columns of the first tile instead of a tile of their own, and
// only tiles at the edges of the mask test their elements.
//
// K and V come by TMA in boxes of up to 32 rows, which never cross a page, into the
// 128-byte-swizzled layout that the MMA descriptors name; pages that no box of 8
// rows fits are gathered row by row with cp.async.  One CTA per SM; items are
// taken over with cluster launch control, so the next item's loads run under the
// end of the last one.
//
// What bounds it (2 x 8192 tokens, heads 32/8 x 128, window 2048: 350 us, 1.08 PFLOP/s):
// a pair of row tiles against a key tile is 2048 cycles of MMA, 2048 of the SM's 16
// exponentials a cycle, and 256 KB of shared-memory traffic (both products'
// operands and the loads' writes), 2048 cycles of its 128 bytes: none can hide
// much of another.  Under the profiler a pair takes 3690 cycles, starts and ends of the
// items included: the tensor pipe is active for 54 % of them, the exponentials' for 55 %.  Not
// kept: a polynomial for a part of the exponentials (slower at every share), two
// threads a row (registers spill), steps of 64 keys (the products of 64 columns are
// bound by shared memory).
//
// The maximum is raised only when a score passes it by more than 2^8, so the
// output is rarely rescaled (by its own softmax warps: the product it belongs to has
// finished by then).  Weights are rounded to the element type, which the MMA's
// operands have; scores, sums and outputs are f32.
//
// A key that some rows of a tile see and others do not enters the others'
// product with weight 0; a NaN or infinite V there would still spoil them.  For a row
// that comes out not finite although its weights are finite, a warp looks through the
// keys that the row met but does not see; where it finds such a value, it computes the
// row's output again over the keys that the row sees.
//
// Every wait has a limit, counted from the last sign that a long item's key tiles go on or
// rows are being computed again (both take time in proportion to their contexts); a wait
// that runs out sets an error bit (ie_kernel_status) and all roles leave.
#include <cuda.h>

#include <mutex>

#include "attention.cuh"

namespace ie {
namespace attn {
namespace {

constexpr int kTile = 128;         // rows of a row tile, keys of a key tile
constexpr int kLoaders = 128;      // threads that gather K and V rows
constexpr int kQLoaders = 64;      // threads that load the query rows
constexpr float kLazy = 8.0f;
// Rows of a TMA box.  Boxes of 16 rows leave the tensor cores waiting (490 us against 440 for
// 2 x 8192 tokens, window 2048); larger ones than 32 only add masked keys to the window.
constexpr int kMaxBox = 32;
constexpr long long kWaitCycles = 4000000000ll;   // ~2 s
constexpr int kBeatTiles = 4096;   // key tiles between two signs of a long item, some 10 ms
constexpr int kInvalidRing = 8;

__device__ uint32_t g_attention_status = 0;

enum Mode { kPrefill = 0, kPrefix = 1 };

// Warps: 0-7 softmax, then the loaders of K and V (with TMA one of each, as one could not
// issue the boxes of 16-row pages fast enough; four that gather), the issuing
// warp and one (gathering: two) for the query rows and the next work item.
template <bool kTma> struct Warps {
  static constexpr int kIssue = kTma ? 10 : 12, kQuery = kIssue + 1;
  static constexpr int kReaders = kTma ? 12 : 15;     // warps that follow the work items
  static constexpr int kThreads = kTma ? 384 : 512;
  // registers of the softmax warps and of the others: together the launch's
  // (384 x 168: 256 x 208 + 128 x 88; 512 x 128: 256 x 192 + 256 x 64)
  static constexpr int kSoftmaxRegs = kTma ? 208 : 192, kOtherRegs = kTma ? 88 : 64;
};

struct TileParams {
  Params p;
  int box;           // rows of a TMA box (0: K and V are gathered)
  int mode;
  int twin;          // one row tile, two streams of key tiles
  int per_tile;      // tokens of a row tile: 128 / group
  int row_tiles;     // work tiles (two row tiles, one when twin) of a segment in the grid
  bool wide_out;     // out rows are 32-byte aligned
  int segs;          // sequences (prefill) or 1 (prefix)
  int parts;         // key parts of a work tile
};

struct Maps {
  CUtensorMap map[4];   // K, V in boxes; K, V row by row
  CUtensorMap q;
};

// ---- PTX ---------------------------------------------------------------------
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
// What the roles tell one another: that one has given up, and when (clock64) key tiles of a
// long item were last issued or rows being computed again, for which the others wait
// as long as it takes.
struct Signals {
  long long beat;
  int quit;
};
// False once the limit has passed without a beat or another role has given up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile Signals* x) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (mbar_try(bar, parity)) return true;
    if (x->quit) return false;
    if (clock64() - t0 > kWaitCycles && clock64() - x->beat > kWaitCycles) {
      atomicOr(&g_attention_status, 1u);
      x->quit = 1;
      return false;
    }
  }
}
// The same for a whole warp: all lanes get one answer.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile Signals* x) {
  return __all_sync(~0u, mbar_wait(bar, parity, x));
}
__device__ __forceinline__ void beat(Signals& x) {
  *static_cast<volatile long long*>(&x.beat) = clock64();
}
// True in one lane of a converged warp.  The instructions of the asynchronous units take
// their operands from uniform registers: a whole warp runs the code around them
// (so that the compiler keeps the operands there) and one lane issues.
__device__ __forceinline__ bool elect() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)::"memory");
  return ok != 0;
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap* map, int x, int y,
                                          int z, int u, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(u), "r"(bar)
      : "memory");
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
__device__ __forceinline__ void tc_commit(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          bar),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
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
// The low word (address in 16-byte units, LBO above it) moves with the start address.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
  return ((lbo >> 4) << 16) | ((addr & 0x3FFFFu) >> 4);
}
__device__ __forceinline__ uint64_t desc(uint32_t lo) {
  constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)hi << 32) | lo;
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
  uint64_t full[8], empty[8], s_full[2], p_ready[2][2], o_done[2], q_full, q_free;
  uint64_t next_full, next_empty;          // the next work item
  alignas(16) uint32_t next[4];
  int slots[2][kTile];                     // cache rows of a key tile
  alignas(16) uint32_t invalid[kInvalidRing][4];   // keys of a tile whose page is not there
  uint32_t tmem;
  Signals signals;
};
static_assert(sizeof(Control) <= 2048, "control block");

// ---- work items --------------------------------------------------------------------
// The grid has a CTA for every work item.  A resident CTA takes over, one at a time,
// CTAs that have not been launched yet (cluster launch control), so items of uneven
// length spread over the SMs as they come free, and the loads of the next item
// run under the end of the last.
__device__ __forceinline__ void try_take(uint32_t answer, uint32_t bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 "
      "[%0], [%1];" ::"r"(answer),
      "r"(bar)
      : "memory");
}
// The item that was taken, or -1.
__device__ __forceinline__ int taken(uint32_t answer) {
  uint32_t x, ok;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %1, 1, 0, p;\n\t"
      "mov.u32 %0, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n\t}"
      : "=r"(x), "=r"(ok)
      : "r"(answer)
      : "memory");
  return ok ? (int)x : -1;
}
// A reader's way through the items: the CTA's own, then what it takes over.
struct Items {
  uint32_t phase = 0;
  int item;
  __device__ __forceinline__ explicit Items(int first) : item(first) {}
  // -1: no more (or another role gave up)
  __device__ __forceinline__ void next(Control* c) {
    if (!warp_wait(smem_u32(&c->next_full), phase, &c->signals)) {
      item = -1;
      return;
    }
    phase ^= 1;
    item = taken(smem_u32(c->next));
    fence_proxy_async();
    __syncwarp();
    if (elect()) mbar_arrive(smem_u32(&c->next_empty));
  }
};
// The asking, by one of the readers, once all have read the answer before (`n` asked
// so far).  A refusal ends the reader's loop: nobody asks again.
__device__ __forceinline__ void ask_next(Control* c, uint32_t n) {
  if (n > 0 && !warp_wait(smem_u32(&c->next_empty), (n - 1) & 1, &c->signals)) return;
  if (elect()) {
    mbar_expect(smem_u32(&c->next_full), 16);
    try_take(smem_u32(c->next), smem_u32(&c->next_full));
  }
  __syncwarp();
}

// ---- work ------------------------------------------------------------------------
// One work tile: the tokens from `first` on of a segment (two row tiles of
// per_tile tokens, one when twin) for one kv head, and the key tiles [j0, j1) of
// its virtual keys.  Every role derives it alike.
struct Work {
  int seg, kvh, part, first;
  int tok0, ntok, pos0;                // of the segment: first token, tokens, first position
  int lo, ns, n;                       // virtual keys: ns sinks, then from lo
  int j0, j1;
};

__device__ __forceinline__ int tokens_of_work(const TileParams& a) {
  return a.twin ? a.per_tile : 2 * a.per_tile;
}
// row tiles of the work tile that hold tokens
__device__ __forceinline__ int row_tiles_of(const TileParams& a, const Work& w) {
  return !a.twin && w.ntok - w.first > a.per_tile ? 2 : 1;
}

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
    w.tok0 = w.pos0 = 0;
    w.ntok = p.tokens;
  } else {
    w.tok0 = p.cu_q ? __ldg(p.cu_q + w.seg) : w.seg;
    w.ntok = p.cu_q ? __ldg(p.cu_q + w.seg + 1) - w.tok0 : 1;
    w.pos0 = context_of(p, w.seg) - w.ntok;
    // a table of lengths that does not describe [0, tokens) reads and writes nothing
    if (w.tok0 < 0 || w.tok0 > p.tokens) w.ntok = 0;
    w.ntok = min(w.ntok, p.tokens - w.tok0);
  }
  return w.ntok > tile * tokens_of_work(a);
}
__device__ __forceinline__ void locate(const TileParams& a, Work& w, int tile) {
  const Params& p = a.p;
  w.first = tile * tokens_of_work(a);
  if (a.mode == kPrefix) {
    w.lo = w.ns = 0;
    w.n = p.key_end;
  } else {
    const int first = max(w.pos0 + w.first, 0);
    const int last = w.pos0 + min(w.first + tokens_of_work(a), w.ntok) - 1;
    w.lo = p.key_start;
    if (p.window > 0) w.lo = max(w.lo, first - p.window + 1);
    w.ns = p.key_start == 0 ? min(p.sinks, w.lo) : 0;
    if (a.box > 1) {        // whole boxes: what they add is masked
      w.lo &= ~(a.box - 1);
      w.ns = min((w.ns + a.box - 1) & ~(a.box - 1), w.lo);
    }
    const int hi = min(last + 1, p.key_end);
    w.n = last < 0 ? 0 : w.ns + max(hi - w.lo, 0);
  }
  const int tiles = (w.n + kTile - 1) / kTile;
  w.j0 = (int)((int64_t)tiles * w.part / a.parts);
  w.j1 = (int)((int64_t)tiles * (w.part + 1) / a.parts);
}

// Rows of tokens that are no sequence's: those in front of the first sequence and behind
// the last.  The softmax warps of that sequence's items write them, the chunks of tokens
// spread over its items; whether the item has work of its own does not matter.
template <typename T, int HD>
__device__ __noinline__ void rows_of_no_sequence(const TileParams& a, const Work& w, int tile,
                                                 int s) {
  const Params& p = a.p;
  if (!p.cu_q || (!a.twin && s > 0)) return;
  const int step = tokens_of_work(a);
  for (int side = 0; side < 2; ++side) {
    if (w.seg != (side ? a.segs - 1 : 0)) continue;
    const int at = min(max(__ldg(p.cu_q + (side ? a.segs : 0)), 0), p.tokens);
    const int lo = side ? at : 0, hi = side ? p.tokens : at;
    for (int64_t c = lo + (int64_t)tile * step; c < hi; c += (int64_t)a.row_tiles * step)
      for (int r = threadIdx.x & (kTile - 1); r < min(step, hi - (int)c) * p.group; r += kTile) {
        const int tok = p.group_div.div(r);
        const int t = (int)c + tok, head = w.kvh * p.group + r - tok * p.group;
        if (p.slots) {
          const int slot = p.slot0 + w.part * (a.twin ? 2 : 1) + (a.twin ? s : 0);
          p.part_ml[((int64_t)t * p.heads + head) * p.slots + slot] = make_float2(-INFINITY, 0.0f);
        } else {
          uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + t * p.out_token +
                                                (int64_t)head * HD);
          for (int i = 0; i < HD / 8; ++i) out[i] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
  }
}

// ---- rows that a value behind their mask has spoilt (see the top) ------------------------
// The virtual keys v that a row sees: v <= vmax and (v >= vmin or v < sinks).
struct Seen {
  int vmax, vmin;
  __device__ __forceinline__ Seen(const Params& p, const Work& w, int pos) {
    const int shift = w.lo - w.ns;
    vmax = pos < 0 ? -1 : min(pos - shift, w.n - 1);
    vmin = max(p.window > 0 ? pos - p.window + 1 : 0, p.key_start) - shift;
  }
  __device__ __forceinline__ bool one(const Params& p, int v) const {
    return v <= vmax && (v >= vmin || v < p.sinks);
  }
  __device__ __forceinline__ bool tile(const Params& p, int v0) const {     // all of its keys
    return v0 + kTile - 1 <= vmax && (v0 >= vmin || v0 + kTile <= p.sinks);
  }
};
// Calls f(v, seen) for this lane's keys of the row's tiles, 32 at a time, where there is
// work: all of them, or (unseen) only in tiles that the row does not see whole.  Ends
// when f returns true, which it does in all lanes or none.
template <typename F>
__device__ __forceinline__ bool keys_of_row(const TileParams& a, const Work& w, Control* c,
                                            const Seen& see, int stream, bool unseen, F f) {
  const int lane = threadIdx.x & 31;
  for (int j = w.j0; j < w.j1; ++j) {
    if (a.twin && ((j - w.j0) & 1) != stream) continue;
    const int v0 = j * kTile;
    if (unseen && see.tile(a.p, v0)) continue;
    for (int i = 0; i < kTile && v0 + i < w.n; i += 32) {
      if (lane == 0) beat(c->signals);
      const int v = v0 + i + lane;
      if (f(v, see.one(a.p, v))) return true;
    }
  }
  return false;
}
__device__ __forceinline__ int slot_of_virtual(const TileParams& a, const Work& w, int v) {
  const Params& p = a.p;
  const int32_t* table = p.tables + (a.mode == kPrefix ? 0 : (int64_t)w.seg * p.table_stride);
  return v < w.n ? cache_slot(p, table, v < w.ns ? v : w.lo + v - w.ns) : -1;
}

// Warp-wide: whether a key that the row at `pos` does not see, but its products met, has
// a value that is not finite.  A lane looks through one key's row.
template <typename T, int HD>
__device__ __noinline__ bool spoilt(const TileParams& a, const Work& w, Control* c, int pos,
                                    int stream) {
  const Params& p = a.p;
  const T* vc = static_cast<const T*>(p.v) + w.kvh * p.head_stride;
  constexpr uint32_t kExp = dtype_of<T>() == IE_DT_BF16 ? 0x7F80u : 0x7C00u;
  return keys_of_row(a, w, c, Seen(p, w, pos), stream, true, [&](int v, bool seen) {
    const int slot = seen ? -1 : slot_of_virtual(a, w, v);
    bool bad = false;
    if (slot >= 0) {
      const uint4* row = reinterpret_cast<const uint4*>(vc + slot * p.slot_stride);
#pragma unroll
      for (int k = 0; k < HD / 8; ++k) {
        const uint4 x = __ldg(row + k);
        for (uint32_t y : {x.x, x.y, x.z, x.w})
          bad = bad || (y & kExp) == kExp || (y >> 16 & kExp) == kExp;
      }
    }
    return __any_sync(~0u, bad) != 0;
  });
}

// Warp-wide: o, relative to the 2^m that the row's sums have, of query token t, head h,
// over the keys that it sees.  A lane computes one key's score; lane + 32 e is an element
// of o.  Ends early when every element is NaN, which it then stays.
template <typename T, int HD>
__device__ __noinline__ void row_again(const TileParams& a, const Work& w, Control* c, int t,
                                       int h, int pos, int stream, float m,
                                       float (&o)[HD / 32]) {
  const Params& p = a.p;
  const int lane = threadIdx.x & 31;
  const uint4* q =
      reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head);
  const T* kc = static_cast<const T*>(p.k) + w.kvh * p.head_stride;
  const T* vc = static_cast<const T*>(p.v) + w.kvh * p.head_stride + lane;
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) o[e] = 0.0f;
  keys_of_row(a, w, c, Seen(p, w, pos), stream, false, [&](int v, bool seen) {
    const int slot = seen ? slot_of_virtual(a, w, v) : -1;
    if (!__any_sync(~0u, slot >= 0)) return false;
    float weight = 0.0f;
    if (slot >= 0) {
      const uint4* k = reinterpret_cast<const uint4*>(kc + slot * p.slot_stride);
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const uint4 x = __ldg(q + i), y = __ldg(k + i);
        const T* xs = reinterpret_cast<const T*>(&x);
        const T* ys = reinterpret_cast<const T*>(&y);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(to_f32<T>(xs[e]), to_f32<T>(ys[e]), s);
      }
      weight = ex2(fmaf(s, p.scale2, -m));
    }
    constexpr int kAtOnce = 8;      // keys whose values are in flight
#pragma unroll 1
    for (int i = 0; i < 32; i += kAtOnce) {
      float value[kAtOnce][HD / 32];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int at = max(__shfl_sync(~0u, slot, i + u), 0);
#pragma unroll
        for (int e = 0; e < HD / 32; ++e)
          value[u][e] = to_f32<T>(vc[at * p.slot_stride + 32 * e]);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const float x = __shfl_sync(~0u, weight, i + u);
        const bool there = __shfl_sync(~0u, slot, i + u) >= 0;
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) o[e] = there ? fmaf(x, value[u][e], o[e]) : o[e];
      }
    }
    bool over = true;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) over = over && o[e] != o[e];
    return __all_sync(~0u, over) != 0;
  });
}

// Warp-wide: those of the lanes' rows that `again` names are computed again where they are
// spoilt, and written over their first result.
template <typename T, int HD>
__device__ __noinline__ void mend_rows(const TileParams& a, const Work& w, Control* c,
                                       uint32_t again, int t, int head, int pos, int stream,
                                       int slot, float m, float l) {
  const Params& p = a.p;
  const int lane = threadIdx.x & 31;
  __syncwarp();       // the rows' own stores come before what other lanes write
  while (again) {
    const int src = __ffs(again) - 1;
    again &= again - 1;
    const int tt = __shfl_sync(~0u, t, src), hh = __shfl_sync(~0u, head, src);
    const int pp = __shfl_sync(~0u, pos, src);
    const float mm = __shfl_sync(~0u, m, src), ll = __shfl_sync(~0u, l, src);
    if (!spoilt<T, HD>(a, w, c, pp, stream)) continue;     // what it sees is not finite
    float o[HD / 32];
    row_again<T, HD>(a, w, c, tt, hh, pp, stream, mm, o);
    const int64_t at = ((int64_t)tt * p.heads + hh) * p.slots + slot;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) {
      if (p.slots) p.part_o[at * HD + lane + 32 * e] = o[e];
      else
        static_cast<T*>(p.out)[(int64_t)tt * p.out_token + (int64_t)hh * HD + lane + 32 * e] =
            from_f32<T>(o[e] / ll);
    }
  }
}

// 32 bytes of a thread's own row: a whole sector a store where the row allows it
__device__ __forceinline__ void store32(void* at, const uint32_t* x, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(at), "r"(x[0]),
                 "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
                 : "memory");
  } else {
    static_cast<uint4*>(at)[0] = make_uint4(x[0], x[1], x[2], x[3]);
    static_cast<uint4*>(at)[1] = make_uint4(x[4], x[5], x[6], x[7]);
  }
}
// bits 0 .. n-1
__device__ __forceinline__ uint32_t below(int n) {
  return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
}

// ---- roles ---------------------------------------------------------------------------
template <typename T, int HD>
__device__ void gather_role(const TileParams& a, uint8_t* base, Control* c) {
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
    return mbar_wait(bar, parity, &c->signals);
  };
  auto commit = [&]() {
    cp_commit();
    ++item;
    if (item - told > 2) {
      cp_wait<2>();
      tell();
    }
  };

  auto next_item = [&](Items& it) {
    flush();                               // the wait below is for those who use the loads
    it.next(c);
    return !any_failed(it.item < 0 || failed);       // all of the loaders go on, or none
  };
  Items it(blockIdx.x);
  do {
    Work w;
    int tile;
    if (!segment(a, it.item, w, tile)) continue;
    const int32_t* table = p.tables + (a.mode == kPrefix ? 0 : (int64_t)w.seg * p.table_stride);
    const uint8_t* kb = static_cast<const uint8_t*>(p.k) + (int64_t)w.kvh * p.head_stride * 2 +
                        chunk * 16;
    const uint8_t* vb = static_cast<const uint8_t*>(p.v) + (int64_t)w.kvh * p.head_stride * 2 +
                        chunk * 16;
    for (; tile * tokens_of_work(a) < w.ntok; tile += a.row_tiles) {
      locate(a, w, tile);
      if (w.j0 >= w.j1) continue;
      auto slot_at = [&](int j) {
        const int v = j * kTile + t;
        if (j >= w.j1 || v >= w.n) return -2;
        return cache_slot(p, table, v < w.ns ? v : w.lo + v - w.ns);
      };
      int next = slot_at(w.j0);
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
  } while (next_item(it));
  flush();
}

// One warp loads K (kv 0) or V (kv 1) with TMA: boxes of a.box rows (a power of two that
// divides the page, so a box lies in one page) by 64 elements.  Lane g looks up box
// g of the tile, one lane issues them all.  A box whose page is not there, and
// rows past the last key, are read outside the tensor: zeros.
template <typename T, int HD>
__device__ void tma_role(const TileParams& a, const CUtensorMap* maps, uint8_t* base, Control* c,
                         int kv) {
  using L = Layout<HD>;
  const Params& p = a.p;
  const int lane = threadIdx.x & 31;
  const int groups = kTile / a.box;
  const int v_lane = lane * a.box;         // this lane's box, if lane < groups
  const uint32_t ring = smem_u32(base + L::kRing);
  const int outside = p.cache_rows;
  uint32_t item = kv;        // K and V tiles alternate in the ring

  for (Items it(blockIdx.x); it.item >= 0; it.next(c)) {
    Work w;
    int tile;
    if (!segment(a, it.item, w, tile)) continue;
    const int32_t* table = p.tables + (a.mode == kPrefix ? 0 : (int64_t)w.seg * p.table_stride);
    for (; tile * tokens_of_work(a) < w.ntok; tile += a.row_tiles) {
      locate(a, w, tile);
      // cache row of this lane's box of key tile j: -1 no page, -2 no key
      auto row_at = [&](int j) {
        const int v = j * kTile + v_lane;
        if (lane >= groups || j >= w.j1 || v >= w.n) return -2;
        return cache_slot(p, table, v < w.ns ? v : w.lo + v - w.ns);
      };
      int next = row_at(w.j0);
      for (int j = w.j0; j < w.j1; ++j) {
        const int row = next;
        next = row_at(j + 1);
        const uint32_t n = item / 2;      // key tiles before this one
        const bool bad = row == -1;
        uint32_t words[4] = {0u, 0u, 0u, 0u};
        if (__any_sync(~0u, bad)) {
          const int bit = v_lane;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            words[i] = __reduce_or_sync(
                ~0u, bad && bit / 32 == i ? below(a.box) << (bit % 32) : 0u);
        }
        // boxes that end past the last key are read row by row
        const int rows = row < 0 ? 0 : min(w.n - (j * kTile + v_lane), a.box);
        const uint32_t ragged = __ballot_sync(~0u, rows > 0 && rows < a.box);
        const int at = rows > 0 ? row : outside;
        const uint32_t st = item % L::kStages, bar = smem_u32(&c->full[st]);
        if (item >= L::kStages &&
            !warp_wait(smem_u32(&c->empty[st]), (item / L::kStages - 1) & 1, &c->signals)) {
          // what has been started ends before the CTA does
          const long long t0 = clock64();
          constexpr uint32_t kBack = L::kStages & ~1;
          for (uint32_t i = item >= kBack ? item - kBack : kv; i < item; i += 2)
            while (!mbar_try(smem_u32(&c->full[i % L::kStages]), (i / L::kStages) & 1) &&
                   clock64() - t0 < kWaitCycles) {
            }
          return;
        }
        if (lane == 0) {
          if (kv == 0)
            *reinterpret_cast<uint4*>(c->invalid[n % kInvalidRing]) =
                make_uint4(words[0], words[1], words[2], words[3]);
          mbar_expect(bar, L::kTileBytes);
        }
        __syncwarp();
        const uint32_t dst = ring + st * L::kTileBytes;
#pragma unroll 8
        for (int g = 0; g < groups; ++g) {
          const int y = __shfl_sync(~0u, at, g);
          const int skip = ragged >> g & 1;
          if (elect()) {
#pragma unroll
            for (int h = 0; h < L::kHalves; ++h)
              if (!skip)
                tma_load(dst + h * 16384 + g * a.box * 128, maps + kv, h * 64, y, w.kvh, bar);
          }
        }
        if (ragged) {
          const int g = __ffs(ragged) - 1;      // the last box only
          const int y = __shfl_sync(~0u, row, g), n_rows = __shfl_sync(~0u, rows, g);
          for (int r = 0; r < a.box; ++r)
            if (elect())
              for (int h = 0; h < L::kHalves; ++h)
                tma_load(dst + h * 16384 + (g * a.box + r) * 128, maps + 2 + kv, h * 64,
                         r < n_rows ? y + r : outside, w.kvh, bar);
        }
        __syncwarp();
        item += 2;
      }
    }
  }
}

// The query rows of a work tile, once the last scores of the one before have been
// computed: by TMA (a box is per_tile tokens by the group's heads by 64 elements,
// which is the order of the rows) or by two warps that gather.
template <typename T, int HD, bool kTma>
__device__ void query_role(const TileParams& a, const CUtensorMap* map, uint8_t* base, Control* c) {
  using L = Layout<HD>;
  const Params& p = a.p;
  constexpr int kChunks = HD / 8, kRows = kQLoaders / kChunks;
  const int t = threadIdx.x & (kQLoaders - 1);
  const int chunk = t % kChunks, r0 = t / kChunks;
  const uint32_t q = smem_u32(base + L::kQ), bar = smem_u32(&c->q_full);
  const bool asks = kTma || t < 32;      // one warp asks for the next item
  uint32_t n = 0, asked = 0;
  // the next item is asked for after the loads of this one: the wait for the slowest
  // reader must not hold them up
  auto next_item = [&](Items& it) {
    if (asks) ask_next(c, asked++);
    it.next(c);
    return it.item >= 0;
  };
  Items it(blockIdx.x);
  do {
    Work w;
    int tile;
    if (!segment(a, it.item, w, tile)) continue;
    for (; tile * tokens_of_work(a) < w.ntok; tile += a.row_tiles) {
      locate(a, w, tile);
      if (w.j0 >= w.j1) continue;
      if (n > 0 && !warp_wait(smem_u32(&c->q_free), (n - 1) & 1, &c->signals)) break;
      ++n;
      const int tiles = row_tiles_of(a, w);
      if (kTma) {
        if (elect()) {
          mbar_expect(bar, tiles * L::kHalves * a.per_tile * p.group * 128);
          for (int s = 0; s < tiles; ++s)
            for (int h = 0; h < L::kHalves; ++h)
              tma_load4(q + s * L::kTileBytes + h * 16384, map, h * 64, 0, w.kvh,
                        w.tok0 + w.first + s * a.per_tile, bar);
        }
        __syncwarp();
      } else {
        const uint8_t* qb = static_cast<const uint8_t*>(p.q) + chunk * 16;
#pragma unroll 4
        for (int r = r0; r < tiles * kTile; r += kRows) {
          const int tok = p.group_div.div(r % kTile), g = r % kTile - tok * p.group;
          const int at = w.first + r / kTile * a.per_tile + tok;
          const bool ok = tok < a.per_tile && at < w.ntok;
          const uint8_t* src = qb + ((w.tok0 + at) * p.q_token +
                                     (int64_t)(w.kvh * p.group + g) * p.q_head) * 2;
          cp_async16(q + (r / kTile) * L::kTileBytes + (chunk / 8) * 16384 + (r % kTile) * 128 +
                         (((chunk & 7) ^ (r & 7)) << 4),
                     ok ? src : qb, ok);
        }
        cp_commit();
        cp_wait<0>();
        fence_proxy_async();
        mbar_arrive(bar);
      }
    }
  } while (next_item(it));
  // a load that nothing waited for (the others gave up) ends before the CTA does
  if (kTma && c->signals.quit && n > 0) {
    const long long t0 = clock64();
    while (!mbar_try(bar, (n - 1) & 1) && clock64() - t0 < kWaitCycles) {
    }
  }
  if (c->signals.quit && asks && asked > 0) {      // nor does an answer come after it
    const long long t0 = clock64();
    while (!mbar_try(smem_u32(&c->next_full), (asked - 1) & 1) && clock64() - t0 < kWaitCycles) {
    }
  }
}

template <typename T, int HD>
__device__ void issue_role(const TileParams& a, uint8_t* base, Control* c,
                           uint32_t tmem_lane) {
  using L = Layout<HD>;
  constexpr uint32_t kIdS = idesc<T>(kTile, false), kIdO = idesc<T>(HD, true);
  constexpr uint32_t kStep = L::kTileBytes >> 4;       // of a descriptor, per stage or row tile
  const uint32_t leader = elect() ? 1u : 0u;
  const uint32_t tmem = __shfl_sync(~0u, tmem_lane, 0);   // uniform
  const uint32_t q_lo = desc_lo(smem_u32(base + L::kQ), 16);
  const uint32_t k_lo = desc_lo(smem_u32(base + L::kRing), 16);
  const uint32_t v_lo = desc_lo(smem_u32(base + L::kRing), 16384);
  const uint32_t full0 = smem_u32(&c->full[0]), empty0 = smem_u32(&c->empty[0]);
  const uint32_t s_full0 = smem_u32(&c->s_full[0]), p_ready0 = smem_u32(&c->p_ready[0][0]);
  const uint32_t o_done0 = smem_u32(&c->o_done[0]);
  uint32_t np = 0, nq = 0;     // phase bits: of p_ready (bit s), of q_full

  // K and V tiles alternate in the ring: a cursor on the next one, in the order of arrival
  struct Cursor {
    uint32_t stage = 0, phase = 0;
    __device__ __forceinline__ void next() {
      if (++stage == L::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
  } cur;
  auto full = [&](const Cursor& x) { return warp_wait(full0 + 8 * x.stage, x.phase, &c->signals); };
  auto release = [&](const Cursor& x) { tc_commit(leader, empty0 + 8 * x.stage); };
  auto p_ready = [&](int s, int half) {
    return warp_wait(p_ready0 + 16 * s + 8 * half, np >> s & 1, &c->signals);
  };
  auto scores = [&](int s, int q, const Cursor& x) {      // S_s = Q_q K^T
    const uint32_t ql = q_lo + q * kStep, kl = k_lo + x.stage * kStep, d = tmem + s * kTile;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      const uint32_t off = ((kk / 4) * 16384 + (kk % 4) * 32) >> 4;
      mma_ss(leader, d, desc(ql + off), desc(kl + off), kIdS, kk > 0);
    }
    tc_commit(leader, s_full0 + 8 * s);
  };
  auto product = [&](int s, const Cursor& x, bool first) {   // O_s (+)= P_s V
    const uint32_t vl = v_lo + x.stage * kStep;
    const uint32_t d = tmem + 2 * kTile + s * HD, pa = tmem + s * kTile;
    // the first half of the weights arrives while the exponentials of the second run
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (!p_ready(s, half)) return false;
      tc_fence_after();
#pragma unroll
      for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
        mma_ts(leader, d, pa + kk * 8, desc(vl + kk * (2048 >> 4)), kIdO, !first || kk > 0);
    }
    np ^= 1u << s;
    return true;
  };

  for (Items it(blockIdx.x); it.item >= 0; it.next(c)) {
    Work w;
    int tile;
    if (!segment(a, it.item, w, tile)) continue;
    for (; tile * tokens_of_work(a) < w.ntok; tile += a.row_tiles) {
      locate(a, w, tile);
      const int nt = w.j1 - w.j0;
      if (nt <= 0) continue;
      if (!warp_wait(smem_u32(&c->q_full), nq, &c->signals)) return;
      nq ^= 1;
      if (a.twin) {
        Cursor v[2];        // V tile of each stream's last scores
        for (int i = 0; i < nt + 2; ++i) {
          const int s = i & 1;
          if (i % kBeatTiles == kBeatTiles - 1 && leader) beat(c->signals);
          if (i >= 2) {       // the product of step i - 2, the same stream
            const Cursor x = s ? v[1] : v[0];
            if (!full(x) || !product(s, x, i < 4)) return;
            release(x);
            if (i >= nt) tc_commit(leader, o_done0 + 8 * s);
          }
          if (i < nt) {
            if (!full(cur)) return;
            tc_fence_after();
            scores(s, 0, cur);
            release(cur);
            cur.next();
            if (s) v[1] = cur;
            else v[0] = cur;
            cur.next();
          }
          if (i == nt - 1) tc_commit(leader, smem_u32(&c->q_free));
        }
      } else {
        const int streams = row_tiles_of(a, w);
        Cursor v;           // V tile of key tile j - 1
        for (int j = 0; j <= nt; ++j) {
          if (j % kBeatTiles == kBeatTiles - 1 && leader) beat(c->signals);
          if (j > 0 && !full(v)) return;
          if (j < nt && !full(cur)) return;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (s >= streams) break;
            if (j > 0) {
              if (!product(s, v, j == 1)) return;
              if (j == nt) tc_commit(leader, o_done0 + 8 * s);
            } else {
              tc_fence_after();
            }
            if (j < nt) scores(s, s, cur);
          }
          if (j > 0) release(v);
          if (j < nt) {
            release(cur);
            cur.next();
            v = cur;
            cur.next();
          }
          if (j == nt - 1) tc_commit(leader, smem_u32(&c->q_free));
        }
      }
    }
  }
}

template <typename T, int HD>
__device__ void softmax_role(const TileParams& a, Control* c, uint32_t tmem, int s) {
  const Params& p = a.p;
  const int r = threadIdx.x & (kTile - 1);
  const uint32_t lanes = (uint32_t)(r & ~31) << 16;       // this warp's TMEM lanes
  const uint32_t ts = tmem + lanes + s * kTile, to = tmem + lanes + 2 * kTile + s * HD;
  const float scale2 = p.scale2;
  const uint64_t scale22 = f32x2(scale2, scale2);
  const int row_tok = p.group_div.div(r), row_head = r - row_tok * p.group;
  uint32_t n_s = 0, n_o = 0;          // s_full and o_done phases waited for
  uint32_t tiles = 0;                 // key tiles of the work tiles before

  for (Items it(blockIdx.x); it.item >= 0; it.next(c)) {
    Work w;
    int tile;
    const bool work = segment(a, it.item, w, tile);
    if (a.mode == kPrefill && ((w.seg == 0 && w.tok0 > 0) ||
                               (w.seg == a.segs - 1 && w.tok0 + w.ntok < p.tokens)))
      rows_of_no_sequence<T, HD>(a, w, tile, s);
    if (!work) continue;
    for (; tile * tokens_of_work(a) < w.ntok; tile += a.row_tiles) {
      locate(a, w, tile);
      const uint32_t tile0 = tiles;
      tiles += max(w.j1 - w.j0, 0);
      if (!a.twin && s >= row_tiles_of(a, w)) continue;
      const int tok = w.first + (a.twin ? 0 : s * a.per_tile) + row_tok;
      const bool live = row_tok < a.per_tile && tok < w.ntok;
      const int t = w.tok0 + (live ? tok : 0);
      const int head = w.kvh * p.group + row_head;
      int pos = -1;
      if (live) pos = a.mode == kPrefix ? position_of(p, sequence_of(p, t), t)
                                        : max(w.pos0 + tok, -1);
      const Seen seen(p, w, pos);
      const int vmax = seen.vmax, vmin = seen.vmin;

      float m = -INFINITY, l = 0.0f;
      int done = 0;
      for (int j = w.j0 + (a.twin ? s : 0); j < w.j1; j += a.twin ? 2 : 1) {
        if (!warp_wait(smem_u32(&c->s_full[s]), n_s & 1, &c->signals)) return;
        ++n_s;
        tc_fence_after();
        uint32_t raw[kTile];
        tmem_ld64(ts, raw);
        tmem_ld64(ts + 64, raw + 64);
        const int v0 = j * kTile;
        const uint4 bad = *reinterpret_cast<const uint4*>(
            c->invalid[(tile0 + (j - w.j0)) % kInvalidRing]);
        const bool whole = seen.tile(p, v0) && (bad.x | bad.y | bad.z | bad.w) == 0;
        if (!__all_sync(~0u, whole)) {
          const uint32_t words[4] = {bad.x, bad.y, bad.z, bad.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // the row's visible keys of these 32 as bits
            const int at = v0 + 32 * i;
            const uint32_t see = below(vmax + 1 - at) & (~below(vmin - at) | below(p.sinks - at)) &
                                 ~words[i];
            if (!__all_sync(~0u, see == ~0u)) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(see & (1u << e))) raw[32 * i + e] = 0xFF800000u;
            }
          }
        }
        float mx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(raw[i]);
#pragma unroll
        for (int i = 4; i < kTile; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(raw[i]));
        const float top =
            fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), scale2, -kBelow<T>);
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
        const uint64_t ref2 = f32x2(-ref, -ref);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int i0 = 0; i0 < kTile; i0 += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const uint64_t x = fma2(f32x2(__uint_as_float(raw[i0 + i]), __uint_as_float(raw[i0 + i + 1])),
                                    scale22, ref2);
            float w0, w1;
            unpack2(x, w0, w1);
            w0 = ex2(w0);
            w1 = ex2(w1);
            sum[i / 2 & 1] = add2(sum[i / 2 & 1], f32x2(w0, w1));
            pk[i / 2] = pack2<T>(w0, w1);
          }
          tmem_st16(ts + i0 / 2, pk);
          if (i0 % 64 == 32) {
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(smem_u32(&c->p_ready[s][i0 / 64]));
          }
        }
        {
          float s0, s1;
          unpack2(add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
        }
        ++done;
      }

      // ---- the row's result
      const int slot = p.slot0 + w.part * (a.twin ? 2 : 1) + (a.twin ? s : 0);
      const int64_t at = ((int64_t)t * p.heads + head) * p.slots + slot;
      T* out = static_cast<T*>(p.out) + (int64_t)t * p.out_token + (int64_t)head * HD;
      float inv = 0.0f, check = 0.0f;
      if (done > 0) {
        if (!warp_wait(smem_u32(&c->o_done[s]), n_o & 1, &c->signals)) return;
        ++n_o;
        tc_fence_after();
        inv = l == 0.0f ? 0.0f : (p.slots ? 1.0f : 1.0f / l);
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
#pragma unroll
          for (int i = 0; i < 64; i += 8) store32(p.part_o + at * HD + h + i, o + i, true);
        } else if (live) {
#pragma unroll
          for (int i = 0; i < 64; i += 16) {
            uint32_t x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              x[e] = pack2<T>(__uint_as_float(o[i + 2 * e]), __uint_as_float(o[i + 2 * e + 1]));
            store32(out + h + i, x, a.wide_out);
          }
        }
      }
      if (done > 0) tc_fence_before();       // O has been read before the next P arrives
      if (live && p.slots) p.part_ml[at] = make_float2(m, l);

      // a sum that is not finite is the row's own: only keys that it sees enter it
      const uint32_t again = __ballot_sync(~0u, live && l - l == 0.0f && !(check == 0.0f));
      if (again) mend_rows<T, HD>(a, w, c, again, t, head, pos, s, slot, m, l);
    }
  }
}

template <typename T, int HD, bool kTma>
__global__ void __launch_bounds__(Warps<kTma>::kThreads, 1)
attention_tile_kernel(const __grid_constant__ TileParams a, const __grid_constant__ Maps maps) {
  using L = Layout<HD>;
  using W = Warps<kTma>;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* base = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  Control* c = reinterpret_cast<Control*>(base + L::kControl);
  const int warp = threadIdx.x >> 5;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) {
      mbar_init(smem_u32(&c->full[i]), kTma ? 1 : kLoaders);
      mbar_init(smem_u32(&c->empty[i]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&c->s_full[s]), 1);
      mbar_init(smem_u32(&c->p_ready[s][0]), kTile);
      mbar_init(smem_u32(&c->p_ready[s][1]), kTile);
      mbar_init(smem_u32(&c->o_done[s]), 1);
    }
    mbar_init(smem_u32(&c->q_full), kTma ? 1 : kQLoaders);
    mbar_init(smem_u32(&c->q_free), 1);
    mbar_init(smem_u32(&c->next_full), 1);
    mbar_init(smem_u32(&c->next_empty), W::kReaders);
    c->signals.beat = 0;
    c->signals.quit = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == W::kIssue) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&c->tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // own keys (decode) or the join may be launched: they wait for this kernel where they
  // need it
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = c->tmem;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(W::kSoftmaxRegs));
    softmax_role<T, HD>(a, c, tmem, warp >> 2);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(W::kOtherRegs));
    if (warp < W::kIssue) {
      if (kTma) tma_role<T, HD>(a, maps.map, base, c, warp - 8);
      else gather_role<T, HD>(a, base, c);
    } else if (warp == W::kIssue) {
      issue_role<T, HD>(a, base, c, tmem);
    } else if (warp < W::kQuery + (kTma ? 1 : 2)) {
      query_role<T, HD, kTma>(a, &maps.q, base, c);
    }
  }
  // every product issued has finished (the softmax warps waited for the last) unless a
  // wait ran out: then give what is in flight the time to end before TMEM goes
  cp_wait<0>();
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (c->signals.quit) {
    if (warp == W::kIssue && (threadIdx.x & 31) == 0) {
      mbar_init(smem_u32(&c->slots[0][0]), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      tc_commit(1u, smem_u32(&c->slots[0][0]));
      const long long t0 = clock64();
      while (!mbar_try(smem_u32(&c->slots[0][0]), 0) && clock64() - t0 < kWaitCycles) {
      }
    }
    __syncthreads();
  }
  if (warp == W::kIssue)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
  });
  return fn;
}

// K and V as [kv_heads][slots][head], in boxes of 64 elements by `box` rows and by one.
bool encode(Maps& maps, const Params& p, int dtype, int box) {
  EncodeFn enc = encoder();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)p.hd, (cuuint64_t)p.cache_rows,
                              (cuuint64_t)p.kv_heads};
  const cuuint64_t strides[2] = {(cuuint64_t)p.slot_stride * 2,
                                 (cuuint64_t)(p.kv_heads > 1 ? p.head_stride : 8) * 2};
  const cuuint32_t unit[3] = {1, 1, 1};
  for (int i = 0; i < 4; ++i) {
    const cuuint32_t size[3] = {64, i < 2 ? (cuuint32_t)box : 1u, 1};
    if (enc(&maps.map[i],
            dtype == IE_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
            3, const_cast<void*>(i & 1 ? p.v : p.k), dims, strides, size, unit,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  // the query rows as [tokens][kv_heads][group][head]
  const cuuint64_t q_dims[4] = {(cuuint64_t)p.hd, (cuuint64_t)p.group, (cuuint64_t)p.kv_heads,
                                (cuuint64_t)p.tokens};
  const cuuint64_t head = (cuuint64_t)(p.heads > 1 ? p.q_head : 8) * 2;
  const cuuint64_t q_strides[3] = {head, head * p.group,
                                   (cuuint64_t)(p.tokens > 1 ? p.q_token : 8) * 2};
  const cuuint32_t q_size[4] = {64, (cuuint32_t)p.group, 1, (cuuint32_t)(kTile / p.group)};
  const cuuint32_t q_unit[4] = {1, 1, 1, 1};
  return enc(&maps.q,
             dtype == IE_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
             4, const_cast<void*>(p.q), q_dims, q_strides, q_size, q_unit,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, bool kTma>
int launch(const TileParams& a, const Maps& maps, cudaStream_t s) {
  auto kernel = attention_tile_kernel<T, HD, kTma>;
  static std::atomic<int> allowed[kMaxDevices];
  if (int rc = allow_smem(kernel, Layout<HD>::kBytes, allowed)) return rc;
  const int64_t items = (int64_t)a.row_tiles * a.parts * a.segs * a.p.kv_heads;
  kernel<<<(unsigned)items, Warps<kTma>::kThreads, Layout<HD>::kBytes,
           s>>>(a, maps);
  return launch_status("attention_tile_kernel");
}
template <typename T>
int launch(TileParams& a, int dtype, cudaStream_t s) {
  const Params& p = a.p;
  Maps maps;
  // TMA wants boxes of at least 8 rows (a swizzle period) within a page; smaller powers of
  // two and rows that a tensor map cannot name (a stride of 0) are gathered
  const int low = (int)(p.block.d & -p.block.d);
  a.box = low >= kMaxBox ? kMaxBox : low;
  if (a.box < 8 || p.pages == 0 || p.slot_stride <= 0 || (p.kv_heads > 1 && p.head_stride <= 0) ||
      (p.tokens > 1 && p.q_token <= 0) || (p.heads > 1 && p.q_head <= 0) ||
      !encode(maps, p, dtype, a.box))
    a.box = 0;
  if (a.box) return p.hd == 64 ? launch<T, 64, true>(a, maps, s) : launch<T, 128, true>(a, maps, s);
  return p.hd == 64 ? launch<T, 64, false>(a, maps, s) : launch<T, 128, false>(a, maps, s);
}

}  // namespace

int launch_tiles(const Params& p, int dtype, bool prefix, bool twin, int row_tiles, int parts,
                 cudaStream_t s) {
  TileParams a{};
  a.p = p;
  a.mode = prefix ? kPrefix : kPrefill;
  a.twin = twin;
  a.per_tile = kTile / p.group;
  a.row_tiles = row_tiles;
  a.segs = prefix ? 1 : p.seqs;
  a.parts = parts;
  a.wide_out = (reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)p.out_token * 2) % 32 == 0;
  return dtype == IE_DT_BF16 ? launch<__nv_bfloat16>(a, dtype, s) : launch<__half>(a, dtype, s);
}

uint32_t attention_status(bool clear) {
  uint32_t v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attention_status, sizeof(v)) != cudaSuccess) return 0;
  if (clear) cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(zero));
  return v;
}

}  // namespace attn
}  // namespace ie
