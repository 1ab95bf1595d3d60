// Attention of a chunk of new tokens over the paged cache (prefill, mixed
// batches, single tokens): for query token i of a request,
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - m_i),
//   over max(0, pos_i - window + 1) <= j <= pos_i,
//   pos_i = seq_len - q_len + i;  lse_i = m_i + ln sum_j p_ij.
//
// One pass over K and V with a running maximum.  A row tile is 128 rows =
// (tokens) x (the G query heads of one kv head), so K and V are read once for
// all heads of the group.  An item is two row tiles of one (request, kv head)
// -- two softmax warpgroups, one tile each -- against 128-key tiles.
//
//   warps 0-3, 4-7  softmax of row tile 0, 1: one thread per row
//   warp 8          TMA producer: Q, then K and V tiles into a ring, one copy
//                   a page (a copy takes some 80-100 cycles of the TMA unit
//                   whatever its size: at one per page and 64 columns K and V
//                   came at 26 bytes a cycle, the tensor core wants 32)
//   warp 9          issues the tcgen05 MMAs: S = Q K^T (both operands in
//                   shared memory, fp32 S in TMEM), O += P V (P in TMEM over
//                   S's columns, V as a column-major operand, fp32 O in TMEM)
//   warp 10         walks the run and tells the others its pieces
//
// While one row tile's softmax runs, the tensor core works for the other.
// O is rescaled only when a row's maximum grows by more than 2^8, so weights
// stay below 256, which both 16-bit types hold; sums stay in fp32 registers.
// The one rounding to 16 bits before the end is P's, half a step per weight:
// the tensor core takes P in V's type.  The row sum keeps the unrounded
// weights, so the result is about 1.4 times as far off as one rounded once.
//
// Work split: the (item, key tile) units of the whole batch form one flat
// list; every CTA takes an equal run of it.  Lengths live on the device, so
// each CTA scans the requests and finds its own run.  Items cut by a run's
// end leave unnormalised partials; the CTA that finishes the last one of a
// warp's rows joins them (a second kernel for that took 9 us of 20 at one
// token).  This serves a single token over a long context (all SMs read one
// request's cache) and a large prefill (no tail of uneven causal tiles) with
// one rule.
//
// Measured on a B200, bf16, 32 query / 8 kv heads of 128, back to back (and in
// runs too short to reach the power limit): 2048 tokens behind 64K 2013 us,
// 1110 TFLOP/s (1763 us, 1267), one token over 4K 12.4 us with the call; 64 / 8
// heads, six fresh prompts of 333-2047 tokens 208 us (190).  What bounds it:
// the chain scores -> softmax -> product (3300 cycles a key tile of two row
// tiles, of which the tensor core is busy 2048), then the board's power.
//
// Code size counts: hot and cold paths together are about what the instruction
// caches hold, so loops stay rolled and paths shared where a unit's time does
// not hang on it (158 KB -> 119 KB, old and new in turn, short runs: fresh
// prompts 9 % less time, with heads of 64 15 %, 2048 behind 64K 1 %).
//
// Slots behind a request's last token, or before all windows of an item's
// rows, may hold anything: K's scores there are replaced before the maximum,
// V's rows are zeroed in shared memory, whole pages are not read.
#include <cuda.h>

#include "common.cuh"

namespace amass {
namespace {

constexpr int kChThreads = 384;          // three warpgroups (warp 11 idles)
constexpr int kKeys = 128;               // keys of a tile
constexpr int kPg = 16;                  // tokens of a page
constexpr int kChMaxReq = 4096;
// cost of an item, for equal runs: a key tile of two row tiles (3300 cycles,
// softmax bound), of one row tile (2100, its loads), and what an item adds
// (query load, first scores, output); cycles of heads of 128, used for 64 too
constexpr int kCost2 = 3, kCost1 = 2, kCostItem = 6, kMinRun = 4;
constexpr float kRescaleLog2 = 8.f;
constexpr uint32_t kWaitCycles = 2000000000u;    // a second or so
constexpr int kPart = 96;                // keys whose weights go to O first

struct ChunkArgs {
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* sl;
  const int32_t* qsl;
  const int32_t* status;                 // null or 0: the request has a step
  void* out;
  int64_t o_st, o_sh;
  float* lse;                            // (T, H) or null
  float* acc;                            // [cta][2][D / 4][256][4]
  float2* ml;                            // [cta][2][256]
  int32_t* tickets;                      // [cta][8], 0 between calls
  int32_t* fault;
  float scale_log2;
  int n_req, n_kv, G, T, max_pages, nb, window, tm_log2;
  int bh;                                // head rows from block to block
};

// ------------------------------------------------------------ tcgen05 / TMA
AMASS_DEV uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(lbo >> 4) << 16) |
         ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// fp32 accumulator, 16-bit operands, A K-major
constexpr uint32_t mma_idesc(bool f16, bool b_mn, int n) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) |
         (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
AMASS_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                      bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
      :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
AMASS_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                      bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
AMASS_DEV void mma_commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 "
      "[%0];" :: "r"(bar) : "memory");
}
AMASS_DEV void tc_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
AMASS_DEV void tc_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
AMASS_DEV void tc_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
AMASS_DEV void tc_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
AMASS_DEV void tc_ld32(uint32_t* r, uint32_t t) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, "
      "[%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]),
        "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(t));
}
AMASS_DEV void tc_st32(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      :: "r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
         "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
         "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
         "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
         "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
         "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
         "r"(r[31])
      : "memory");
}
AMASS_DEV void tc_ld16(uint32_t* r, uint32_t t) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]),
        "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15])
      : "r"(t));
}
AMASS_DEV void tc_st16(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :: "r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
         "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
         "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 16 rows (TMEM lanes) of 128 columns: lane l holds columns 8 j + 2 (l % 4) and
// the next one of row l / 4 in r[4 j], r[4 j + 1], of row l / 4 + 8 in the
// other two
AMASS_DEV void tc_ld_16x256(uint32_t* r, uint32_t t) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, "
      "[%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]),
        "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
        "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]),
        "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]),
        "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]),
        "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(t));
}
// 16 rows of 64 columns: lane l's are 4 j + l % 4 of rows l / 4 and l / 4 + 8
AMASS_DEV void tc_st_16x128(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      :: "r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
         "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
         "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
         "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
         "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
         "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
         "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
         "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
AMASS_DEV float fmax_nan(float a, float b) {   // NaN when either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// two fp32 lanes at once
AMASS_DEV uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
AMASS_DEV void f2_get(uint64_t x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
AMASS_DEV uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
AMASS_DEV uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
AMASS_DEV void tma_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x,
                      int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      :: "r"(dst), "l"(m), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
AMASS_DEV void tma_5d(uint32_t dst, const CUtensorMap* m, uint32_t bar,
                      int w) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes [%0], [%1, {%2, %2, %2, %2, %3}], [%4];"
      :: "r"(dst), "l"(m), "r"(0), "r"(w), "r"(bar) : "memory");
}

// ------------------------------------------------------------- work list ---
// e / d for 0 <= e < 2^31 and a quotient below 2^20: the reciprocal's quotient
// is off by one at most (an integer division costs some 150 cycles more)
AMASS_DEV int quotient(int e, int d) {
  unsigned q = (unsigned)__fdividef((float)e, (float)d);
  q -= q * (unsigned)d > (unsigned)e;
  q += (q + 1) * (unsigned)d <= (unsigned)e;
  return (int)q;
}

// One request: its rows start at q0, ql of them; row i has position off + i.
struct ChReq {
  int q0, ql, sl, off, nt;
};
AMASS_DEV ChReq ch_req(const ChunkArgs& a, int r) {
  ChReq q;
  const int s0 = a.qsl[r], s1 = a.qsl[r + 1];
  q.q0 = max(s0, 0);
  q.ql = max(min(s1, a.T) - q.q0, 0);
  // a length beyond the block table's row is cut: no page behind it exists;
  // new tokens behind the last row are not there: the others keep their
  // positions
  const int64_t most = min((int64_t)a.sl[r], (int64_t)a.max_pages * kPg);
  q.sl = (int)max(most - (max(s1, a.T) - a.T), (int64_t)0);
  // a refused request's length is without its new tokens: no key is theirs
  if (a.status && a.status[r] != 0) q.sl = 0;
  q.off = q.sl - q.ql;
  q.nt = (q.ql + (2 << a.tm_log2) - 1) >> (a.tm_log2 + 1);
  return q;
}
// key tiles [lo, lo + n) that item i of the request visits (n >= 1: rows that
// see nothing still get their zeros written)
AMASS_DEV int ch_tiles(const ChunkArgs& a, const ChReq& q, int i, int* lo) {
  const int tl = a.tm_log2 + 1;
  const int end = q.off + min((i + 1) << tl, q.ql);
  *lo = a.window ? max(q.off + (i << tl) - a.window + 1, 0) >> 7 : 0;
  return end > 0 ? ((end + kKeys - 1) >> 7) - *lo : (*lo = 0, 1);
}
// sum over j < x of j >> s
AMASS_DEV int64_t shift_sum(int x, int s) {
  const int q = x >> s;
  return (((int64_t)q * (q - 1) / 2) << s) + (int64_t)q * (x - (q << s));
}
// sum over i in [i0, i1) of max(b + i * 2^tl, 0) >> 7; with c = b >> tl a
// summand is (c + i) >> (7 - tl) up to tl = 7, and above that (c + i) <<
// (tl - 7) plus the bits of b in between
AMASS_DEV int64_t floor_sum(int b, int i0, int i1, int tl) {
  if (b < 0) {                           // first i with a value above 0
    const int z = ((-b) >> tl) + 1;
    i0 = max(i0, z) - z;
    i1 -= z;
    b += z << tl;
  }
  if (i0 >= i1) return 0;
  const int c = b >> tl, s = max(7 - tl, 0), k = max(tl - 7, 0);
  return ((shift_sum(i1 + c, s) - shift_sum(i0 + c, s)) << k) +
         (int64_t)(i1 - i0) * ((b >> 7) & ((1 << k) - 1));
}
// cost of one key tile of item i
AMASS_DEV int ch_weight(const ChunkArgs& a, const ChReq& q, int i) {
  return q.ql - (i << (a.tm_log2 + 1)) > (1 << a.tm_log2) ? kCost2 : kCost1;
}
// cost of items 0 .. m - 1 of the request (closed form of ch_tiles' sum)
AMASS_DEV int64_t ch_cost(const ChunkArgs& a, const ChReq& q, int m) {
  const int tl = a.tm_log2 + 1;
  if (m <= 0) return 0;
  int64_t s = (int64_t)m * kCostItem;
  int full = m;
  if (m == q.nt) {                       // the last item may be short
    int lo;
    s += (int64_t)ch_tiles(a, q, m - 1, &lo) * ch_weight(a, q, m - 1);
    full = m - 1;
  }
  // items whose last position is negative visit one (empty) tile
  const int none = q.off < 0 ? min(full, (-q.off) >> tl) : 0;
  int64_t u = none + floor_sum(q.off + (1 << tl) + kKeys - 1, none, full, tl);
  if (a.window) u -= floor_sum(q.off - a.window + 1, none, full, tl);
  return s + u * kCost2;
}

// A piece of an item: key tiles [t0, t0 + n) for ntok tokens from tok0 on;
// first / last: with the item's first / last key tile; n = 0 ends the run.
struct alignas(16) ChSeg {
  int r, h, tok0, ntok;                  // request, kv head; row in q
  int pos0, sl, t0, n;                   // position of tok0, tokens, tiles
  int first, last, cta0, parts;          // a cut item's CTAs
};
struct ChPlan {
  long long u;                           // the run's start in the head's items
  ChReq q;
  int r, h, i, from, to, share;          // run [from, to) from item i's start
};

// Walks the segments of a CTA's run (one warp does, a few ahead of the others).
// Key tile k of an item belongs to the CTA whose run holds its place, item
// start + k * weight.  A first segment that starts inside its item goes last:
// then every CTA starts at its item's first key tile, and since the runs are
// equally long the late pieces of one head's items meet at the same key tiles
// again.  CTAs of a head so stream its K and V together and find them in L2
// (2048 rows behind 64K tokens: 2290 -> 1920 us).
struct ChWalk {
  ChReq q;
  int r, h, i, from, to, at;             // at: the item's start in the run
  bool late;                             // the first segment is still to come
  AMASS_DEV void start(const ChunkArgs& a, const ChPlan& p) {
    q = p.q; r = p.r; h = p.h; i = p.i; from = p.from; to = p.to;
    late = false;
    at = -from;
    if (from > 0 && to > 0) {
      int lo;
      const int w = ch_weight(a, q, i), n = ch_tiles(a, q, i, &lo);
      if (to > n * w + kCostItem) {      // the run goes on behind this item
        late = from <= (n - 1) * w;      // no tile of it: its overhead only
        step(a, n * w + kCostItem);
      }
    }
  }
  AMASS_DEV void step(const ChunkArgs& a, int cost) {
    from = 0;
    to -= cost;
    at += cost;
    if (++i < q.nt) return;
    i = 0;
    if (++h < a.n_kv) return;
    h = 0;
    if (to <= 0) return;
    do {
      if (++r >= a.n_req) { to = 0; return; }
      q = ch_req(a, r);
    } while (q.nt == 0);
  }
  AMASS_DEV bool next(const ChunkArgs& a, const ChPlan& p, ChSeg& s) {
    bool only = false;
    if (to <= 0) {
      if (!late) return false;
      late = false;
      only = true;
      q = p.q; r = p.r; h = p.h; i = p.i; from = p.from; to = p.to;
      at = -from;
    }
    const int tl = a.tm_log2 + 1, w = ch_weight(a, q, i);
    int lo;
    const int nu = ch_tiles(a, q, i, &lo);
    const auto tiles = [&](int c) {      // ceil(c / w)
      return w == kCost2 ? (c + kCost2 - 1) / kCost2
                         : (c + kCost1 - 1) / kCost1;
    };
    const int k0 = tiles(from), k1 = to >= nu * w ? nu : tiles(to);
    if (k0 >= k1) return false;          // the run is in an item's overhead
    s.r = r; s.h = h; s.sl = q.sl;
    s.tok0 = q.q0 + (i << tl);
    s.pos0 = q.off + (i << tl);
    s.ntok = min(1 << tl, q.ql - (i << tl));
    s.t0 = lo + k0;
    s.n = k1 - k0;
    s.first = k0 == 0;
    s.last = k1 == nu;
    s.cta0 = s.parts = 0;
    if (!(s.first && s.last)) {          // floor divisions by the run length
      const int b = at < 0 ? quotient(p.share - 1 - at, p.share) : 0;
      const int e = at + (nu - 1) * w;
      s.cta0 = (int)blockIdx.x - b;
      s.parts = (e < 0 ? -quotient(p.share - 1 - e, p.share)
                       : quotient(e, p.share)) + b + 1;
    }
    if (only) to = 0;
    else step(a, nu * w + kCostItem);
    return true;
  }
};

// this CTA's run of the flat list of items
AMASS_DEV void ch_plan(const ChunkArgs& a, ChPlan* out) {
  __shared__ long long wsum[kChThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int per = (a.n_req + kChThreads - 1) / kChThreads;
  const int r0 = min(a.n_req, tid * per), r1 = min(a.n_req, r0 + per);
  long long mine = 0, cost = 0;
  ChReq q;
  for (int r = r0; r < r1; ++r) {
    q = ch_req(a, r);
    cost = ch_cost(a, q, q.nt);
    mine += cost * a.n_kv;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) wsum[w] = incl;
  if (tid == 0) out->to = 0;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int i = 0; i < kChThreads / 32; ++i) {
    if (i < w) before += wsum[i];
    total += wsum[i];
  }
  const long long over = total + gridDim.x - 1;
  long long share = over >> 32 ? over / gridDim.x
                               : (long long)((uint32_t)over / gridDim.x);
  if (share < kMinRun) share = kMinRun;
  const long long begin = share * blockIdx.x;
  const long long end = min(total, begin + share);
  if (begin >= before && begin < before + mine) {
    long long u = begin - before;
    for (int r = r0; r < r1; ++r) {
      if (per > 1) {                     // one request: still in registers
        q = ch_req(a, r);
        cost = ch_cost(a, q, q.nt);
      }
      const long long all = cost * a.n_kv;
      if (u >= all) {
        u -= all;
        continue;
      }
      const int h = all >> 31 || a.n_kv >> 20 ? (int)(u / cost)
                                              : quotient((int)u, (int)cost);
      u -= h * cost;
      out->q = q;
      out->r = r;
      out->h = h;
      out->u = u;                        // for ch_plan_item
      out->to = (int)(end - begin);
      out->share = (int)share;
      break;
    }
  }
  __syncthreads();
}

// Ends the plan: the last item of the head that starts at or before the run's
// start, by a whole warp, 32 places at a time (halving by one thread took 2500
// cycles of a run's start).
AMASS_DEV void ch_plan_item(const ChunkArgs& a, ChPlan* p) {
  const int lane = threadIdx.x & 31;
  const ChReq q = p->q;
  const long long u = p->u;
  long long base = 0;
  int lo = 0, hi = p->to > 0 ? q.nt : 0;
#pragma unroll 1
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, m = lo + (lane + 1) * step;
    const long long c = m < hi ? ch_cost(a, q, m) : 0;
    const int n = __popc(__ballot_sync(~0u, m < hi && c <= u));
    const long long b = __shfl_sync(~0u, c, max(n - 1, 0));
    if (n) base = b;
    lo += n * step;
    hi = min(hi, lo + step);
  }
  __syncwarp();
  if (lane == 0) {
    p->i = lo;
    p->from = (int)(u - base);
    if (p->to > 0) p->to += p->from;
  }
  __syncwarp();
}

constexpr int kSegs = 4;
constexpr int kFewRows = 8;              // of a warp: joined by all warps
constexpr int kStage = 4096;             // a warp's 32 rows x 64 columns

template <int D>
struct ChShape {
  static constexpr int kPanels = D / 64;
  static constexpr int kTile = kKeys * D * 2;        // bytes of a K or V tile
  static constexpr int kPanel = kKeys * 128;         // Q: 128 rows x 64
  // K and V: 8 rows x 64 columns are one kilobyte, the panels of 8 rows side
  // by side, so that one copy brings a whole page
  static constexpr int kRows8 = kPanels * 1024;
  static constexpr int kPage = 2 * kRows8;
  static constexpr int kStages = 131072 / kTile;     // 128 KB of ring
  static constexpr int kOut = 2 * kTile + kStages * kTile;   // staged rows
  static constexpr int kSmem = kOut + 8 * kStage + 1024;
  static constexpr uint32_t kCols = 512;             // 2 S/P + 2 O
  static constexpr uint32_t kO = 256;
};

// Lane r's row of 64 16-bit values goes through 4 KB of shared memory, 16
// bytes at a time (chunk c of 8), so that eight lanes write a row's 128 bytes
// together: a store of 32 rows is 32 cycles of the load/store unit, one of 4
// full lines 4.
AMASS_DEV void stage_put(uint32_t stage, int c, uint4 v) {
  const uint32_t r = threadIdx.x & 31;
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
               :: "r"(stage + r * 128 + ((c ^ (r & 7)) << 4)), "r"(v.x),
                  "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// row: where the lane's 128 bytes go, null for nowhere
AMASS_DEV void stage_out(uint32_t stage, char* row) {
  const int lane = threadIdx.x & 31;
  const uint32_t c = lane & 7;
  unsigned long long p[8];
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    p[i] = __shfl_sync(~0u, reinterpret_cast<unsigned long long>(row),
                       i * 4 + (lane >> 3));
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t r = i * 4 + (lane >> 3);
    v[i] = lds128(stage + r * 128 + ((c ^ (r & 7)) << 4));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (p[i]) *reinterpret_cast<uint4*>(p[i] + c * 16) = v[i];
  __syncwarp();
}

// draws a ticket: this warp's earlier stores are visible to whoever draws a
// later one, the stores before earlier ones to this warp
AMASS_DEV int draw(int32_t* ticket) {
  int v;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;"
               : "=r"(v) : "l"(ticket) : "memory");
  return v;
}

// The rows of one warp of a cut item whose last partial was written here.
struct ChJob {
  int cta0, parts, h;                    // the item's CTAs, its kv head
  int n, row0, tok0;                     // rows, first of the item's 256, token
};                                       // of its row tile's row 0

// Joining: out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over the item's
// CTAs in order (the same result whichever CTA finishes last).
struct ChSum {
  float M = -INFINITY, l = 0.f;
  // adds NP partials, every `by`-th from c0 on, of NC groups of 4 columns
  template <int D, int NC, int NP>
  AMASS_DEV void add(const ChJob& b, const float2* ml, const float4* x,
                     int c0, int by, float4* o) {
    float4 v[NP][NC];
    float2 z[NP];
    // the first CTA's partial is its second slot, the others' their first
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      const int c = c0 + e * by, s = 2 * c + (c == 0);
      z[e] = make_float2(-INFINITY, 0.f);
      if (c < b.parts) z[e] = __ldcg(ml + s * 256);
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        v[e][k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < b.parts)
          v[e][k] = __ldcg(x + ((int64_t)s * (D / 4) + k) * 256);
      }
    }
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      const float mn = fmax_nan(M, z[e].x), ref = mn == -INFINITY ? 0.f : mn;
      const float f = ex2_approx(M - ref), w = ex2_approx(z[e].x - ref);
      M = mn;
      l = l * f + w * z[e].y;
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        o[k].x = o[k].x * f + w * v[e][k].x;
        o[k].y = o[k].y * f + w * v[e][k].y;
        o[k].z = o[k].z * f + w * v[e][k].z;
        o[k].w = o[k].w * f + w * v[e][k].w;
      }
    }
  }
  AMASS_DEV bool some() const { return l > 0.f || l != l; }
  AMASS_DEV float inv() const { return some() ? 1.f / l : 0.f; }
  AMASS_DEV float lse() const {
    return some() ? (M + log2f(l)) * 0.6931471805599453f : -INFINITY;
  }
};
template <bool kF16>
AMASS_DEV uint2 pack4(float4 o, float f) {
  return kF16 ? make_uint2(pack_h2(o.x * f, o.y * f), pack_h2(o.z * f, o.w * f))
              : make_uint2(pack_bf2(o.x * f, o.y * f),
                           pack_bf2(o.z * f, o.w * f));
}
// where row `row` of the job's item goes
AMASS_DEV char* ch_out(const ChunkArgs& a, const ChJob& b, int row,
                       int64_t* lse) {
  const int tok = (row & 127) / a.G;
  const int64_t token = b.tok0 + tok;
  const int head = b.h * a.G + (row & 127) - tok * a.G;
  *lse = token * (a.n_kv * a.G) + head;
  return (char*)a.out + 2 * (token * a.o_st + head * a.o_sh);
}
// Few rows (2^sh >= n, sh <= 3), many partials: lanes over rows, then 4 groups
// of 4 columns from cg on, then 8 >> sh groups of partials, 12 in flight each.
template <int D, bool kF16>
AMASS_DEV void ch_join_few(const ChunkArgs& a, const ChJob& b, int sh, int cg) {
  const int lane = threadIdx.x & 31, r = lane & ((1 << sh) - 1);
  const int pg = lane >> (sh + 2), pgs = 8 >> sh;
  cg += (lane >> sh) & 3;
  const int row = b.row0 + min(r, b.n - 1);
  const float2* ml = a.ml + (int64_t)b.cta0 * 512 + row;
  const float4* x = reinterpret_cast<const float4*>(a.acc) +
                    ((int64_t)b.cta0 * 2 * (D / 4) + cg) * 256 + row;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  ChSum s;
#pragma unroll 1
  for (int c = pg; c < b.parts; c += 12 * pgs)
    s.template add<D, 1, 12>(b, ml, x, c, pgs, &o);
  for (int k = 4 << sh; k < 32; k <<= 1) {
    const float m1 = __shfl_xor_sync(~0u, s.M, k);
    const float l1 = __shfl_xor_sync(~0u, s.l, k);
    const float mn = fmax_nan(s.M, m1), ref = mn == -INFINITY ? 0.f : mn;
    const float f0 = ex2_approx(s.M - ref), f1 = ex2_approx(m1 - ref);
    s.M = mn;
    s.l = s.l * f0 + l1 * f1;
    o.x = o.x * f0 + __shfl_xor_sync(~0u, o.x, k) * f1;
    o.y = o.y * f0 + __shfl_xor_sync(~0u, o.y, k) * f1;
    o.z = o.z * f0 + __shfl_xor_sync(~0u, o.z, k) * f1;
    o.w = o.w * f0 + __shfl_xor_sync(~0u, o.w, k) * f1;
  }
  if (r >= b.n || pg) return;
  int64_t li;
  char* out = ch_out(a, b, row, &li);
  *reinterpret_cast<uint2*>(out + 8 * cg) = pack4<kF16>(o, s.inv());
  if (a.lse && cg == 0) a.lse[li] = s.lse();
}
// A lane per row, 64 columns from 64 half on: two partials' 64 columns in
// flight.
template <int D, bool kF16>
AMASS_DEV void ch_join_many(const ChunkArgs& a, const ChJob& b, int half,
                            uint32_t stage) {
  const int lane = threadIdx.x & 31, row = b.row0 + min(lane, b.n - 1);
  const float2* ml = a.ml + (int64_t)b.cta0 * 512 + row;
  const float4* x = reinterpret_cast<const float4*>(a.acc) +
                    ((int64_t)b.cta0 * 2 * (D / 4) + half * 16) * 256 + row;
  float4 o[16];
  ChSum s;
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int c = 0; c < b.parts; c += 2)
    s.template add<D, 16, 2>(b, ml, x, c, 1, o);
  const float f = s.inv();
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    const uint2 lo = pack4<kF16>(o[e], f), hi = pack4<kF16>(o[e + 1], f);
    stage_put(stage, e / 2, make_uint4(lo.x, lo.y, hi.x, hi.y));
  }
  int64_t li;
  char* out = ch_out(a, b, row, &li);
  if (a.lse && half == 0 && lane < b.n) a.lse[li] = s.lse();
  stage_out(stage, lane < b.n ? out + half * 128 : nullptr);
}

template <int D, bool kF16>
__global__ void __launch_bounds__(kChThreads, 1)
chunk_kernel(const __grid_constant__ CUtensorMap mq,
             const __grid_constant__ CUtensorMap mk,
             const __grid_constant__ CUtensorMap mv, const ChunkArgs a) {
  using X = ChShape<D>;
  constexpr int NS = X::kStages;
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[2 * NS + 16 + 2 * kSegs];
  __shared__ ChJob jobs[16];             // a run cuts two items: 8 warps' rows
  __shared__ int few_jobs[16], n_few;    // those of few rows
  __shared__ ChPlan plan;
  __shared__ ChSeg segs[kSegs];          // the walk, a few pieces ahead
  __shared__ uint32_t tmem_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const uint32_t base = (smem_u32(dyn) + 1023u) & ~1023u;
  const uint32_t q_s = base, ring = base + 2 * X::kTile;
  const uint32_t b0 = smem_u32(bars);
  const auto full = [&](int s) { return b0 + 8u * s; };
  const auto empty = [&](int s) { return b0 + 8u * (NS + s); };
  // one of each per row tile
  const uint32_t q_full = b0 + 8u * (2 * NS), q_empty = q_full + 16;
  const uint32_t s_full = q_full + 32, p_part = q_full + 48;
  const uint32_t p_full = q_full + 64, o_full = q_full + 80;
  const uint32_t v_tmp = q_full + 96, drain = v_tmp + 8;
  const uint32_t pair = v_tmp + 16, pair_done = v_tmp + 24;
  const uint32_t seg_full = v_tmp + 32, seg_empty = seg_full + 8 * kSegs;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(q_full + 8 * t, 1);
      mbar_init(q_empty + 8 * t, 1);
      mbar_init(s_full + 8 * t, 1);
      mbar_init(p_part + 8 * t, 4);
      mbar_init(p_full + 8 * t, 4);
      mbar_init(o_full + 8 * t, 1);
    }
    n_few = 0;
    mbar_init(v_tmp, 1);
    mbar_init(drain, 1);
    for (int s = 0; s < kSegs; ++s) {
      mbar_init(seg_full + 8 * s, 1);
      mbar_init(seg_empty + 8 * s, 10);  // softmax, producer, MMA warps
    }
    mbar_init(pair, 4);
    mbar_init(pair_done, 4);
    mbar_init_fence();
  }
  if (warp == 9) {
    asm volatile(
        "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
        :: "r"(smem_u32(&tmem_s)), "r"(X::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // the predecessor's memory is read from here on
  grid_dep_wait();
  grid_dep_launch();
  tc_before();
  ch_plan(a, &plan);                     // ends with a barrier
  tc_after();
  const uint32_t tmem = tmem_s;

  // bounded wait: after about a second the warp unwinds, the others run into
  // their own limits, and the fault is recorded at the end
  // (mbar_wait in fewer instructions: there are some thirty of these)
  const auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    uint32_t t0 = 0;
    while (!mbar_try_wait(bar, parity)) {
      const uint32_t now = clock() | 1u;
      if (!t0) t0 = now;
      if (now - t0 >= kWaitCycles) return false;
    }
    return true;
  };
  // the same for whole warps, which have to unwind together
  const auto wait_warp = [&](uint32_t bar, uint32_t parity) -> bool {
    return __all_sync(~0u, wait(bar, parity));
  };

  // the run's next piece; false at its end
  ChSeg sg;
  int seg_at = 0;
  bool ok = true;
  const auto next_seg = [&]() -> bool {
    const int k = seg_at++;
    if (!(ok = wait_warp(seg_full + 8 * (k % kSegs), (k / kSegs) & 1)))
      return false;
    sg = segs[k % kSegs];
    __syncwarp();
    if (lane == 0) mbar_arrive(seg_empty + 8 * (k % kSegs));
    return sg.n > 0;
  };

  // a softmax thread holds a row of 128 scores: 384 * 168 registers at launch
  // = 128 * (2 * 192 + 120)
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ------------------------------------------------------------- softmax
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + t * 128 + lanes;
    const uint32_t to = tmem + X::kO + t * D + lanes;
    const int tok = row / a.G, g = row - tok * a.G, tm = 1 << a.tm_log2;
    const uint32_t stage = base + X::kOut + warp * kStage;
    // warpgroup 1's (m, l) of an item it shares with warpgroup 0: in its own
    // stage, which it does not use then
    float2* pair_ml = reinterpret_cast<float2*>(
        dyn + (base - smem_u32(dyn)) + X::kOut + (4 + (warp & 3)) * kStage) +
        lane;
    const float sl2 = a.scale_log2;
    const uint64_t sl2x2 = f2(sl2, sl2);
    uint32_t sph = 0, oph = 0, cph = 0;
    int mine = 0;                        // this warp's jobs
    while (ok && next_seg()) {
      const bool two = sg.ntok > tm;
      const int it = (two ? t * tm : 0) + tok;   // token within the item
      const bool valid = tok < tm && it < sg.ntok;
      const int pos = sg.pos0 + it;
      // rows of nobody compute on whatever Q's buffer holds, unmasked
      const int khi = valid ? max(pos + 1, 0) : 0x7fffffff;
      const int klo = valid && a.window ? max(pos - a.window + 1, 0) : 0;
      const int rows = __popc(__ballot_sync(~0u, valid));
      const bool live = rows > 0;
      // up to eight rows (one token's heads): four lanes share a row, a
      // quarter of the exponentials and of the code for a lane
      const bool few = rows <= 8;
      const int khi4 = __shfl_sync(~0u, khi, lane >> 2);
      const int klo4 = __shfl_sync(~0u, klo, lane >> 2);
      const bool valid4 = __shfl_sync(~0u, (int)valid, lane >> 2) != 0;
      // what all of the warp's rows see, and any of
      const int khi_lo = __reduce_min_sync(~0u, khi);
      const int klo_hi = __reduce_max_sync(~0u, klo);
      const int khi_hi = __reduce_max_sync(~0u, valid ? khi : 0);
      const int klo_lo = __reduce_min_sync(~0u, valid ? klo : 0x7fffffff);
      const int by = two ? 1 : 2;
      const auto rescale = [&](float f) {        // row lane of O by f
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t o[16];
          tc_ld16(o, to + c);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tc_st16(to + c, o);
        }
      };
      float m = -INFINITY, l = 0.f;
      for (int j = two ? 0 : t; j < sg.n; j += by) {
        if (!(ok = wait_warp(s_full + 8 * t, sph))) break;
        sph ^= 1;
        tc_after();
        if (live && few) {
          uint32_t s[64];
          tc_ld_16x256(s, ts);
          tc_wait_ld();
          const int k0 = (sg.t0 + j) * kKeys, col = (lane & 3) * 2;
          if (__any_sync(~0u, khi4 - k0 < kKeys || k0 < klo4)) {
            const int e = khi4 - k0 - col, b = klo4 - k0 - col;
#pragma unroll
            for (int c = 0; c < 128; c += 8) {
              if (c >= e || c < b) s[c / 2] = 0xff800000u;
              if (c + 1 >= e || c + 1 < b) s[c / 2 + 1] = 0xff800000u;
            }
          }
          float mx = -INFINITY;
#pragma unroll
          for (int c = 0; c < 64; c += 4)
            mx = fmax_nan(fmax_nan(mx, __uint_as_float(s[c])),
                          __uint_as_float(s[c + 1]));
          mx = fmax_nan(mx, __shfl_xor_sync(~0u, mx, 1));
          mx = fmax_nan(mx, __shfl_xor_sync(~0u, mx, 2));
          if (j < by) {
            m = mx;
          } else if (__any_sync(~0u,
                                valid4 && !((mx - m) * sl2 <= kRescaleLog2))) {
            const float mn = fmax_nan(m, mx);
            const float f = m == -INFINITY ? 0.f : ex2_approx((m - mn) * sl2);
            l *= f;
            m = mn;
            rescale(__shfl_sync(~0u, f, (lane & 7) * 4));
          }
          const float nm = m == -INFINITY ? 0.f : fmaf(0.f, m, -m * sl2);
          float sum = 0.f;
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float p0 =
                ex2_approx(fmaf(__uint_as_float(s[2 * c]), sl2, nm));
            const float p1 =
                ex2_approx(fmaf(__uint_as_float(s[2 * c + 1]), sl2, nm));
            sum += p0 + p1;
            s[c] = kF16 ? pack_h2(p0, p1) : pack_bf2(p0, p1);
            s[c + 1] = 0;
          }
          l += sum;
          tc_st_16x128(ts, s);
          tc_wait_st();
          tc_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_part + 8 * t);
        } else if (live) {
          // the running maximum takes in mx
          const auto grow = [&](float mx) {
            if (j < by) {                // this warpgroup's first tile
              m = mx;
            } else if (__any_sync(~0u, valid &&
                                           !((mx - m) * sl2 <= kRescaleLog2))) {
              const float mn = fmax_nan(m, mx);
              const float f =
                  m == -INFINITY ? 0.f : ex2_approx((m - mn) * sl2);
              l *= f;
              m = mn;
              rescale(f);
            }
            // a score of +inf or NaN makes the row NaN, as the formula does;
            // one of -inf has no weight
            return m == -INFINITY ? 0.f : fmaf(0.f, m, -m * sl2);
          };
          uint64_t sum[2] = {0ull, 0ull};
          // two weights from two scores, packed
          const auto weigh = [&](uint32_t s0, uint32_t s1, uint64_t nm2,
                                 int k) {
            float p0, p1;
            f2_get(f2_fma(f2(__uint_as_float(s0), __uint_as_float(s1)), sl2x2,
                          nm2), p0, p1);
            p0 = ex2_approx(p0);
            p1 = ex2_approx(p1);
            sum[k & 1] = f2_add(sum[k & 1], f2(p0, p1));
            return kF16 ? pack_h2(p0, p1) : pack_bf2(p0, p1);
          };
          const int k0 = (sg.t0 + j) * kKeys;
          if (k0 + kKeys > khi_lo || k0 < klo_hi) {
            // some row does not see all of the tile: -inf in place of what it
            // does not see, 32 keys at a time (a path of its own that leaves
            // hidden keys out takes 4 % less for 8 prompts of 200-600 tokens,
            // 2 % more for 333-2047, and more code)
#pragma unroll 1
            for (int c = 0; c < kKeys; c += 32) {
              const int k = k0 + c;
              if (k + 32 <= khi_lo && k >= klo_hi) continue;
              uint32_t s[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) s[i] = 0xff800000u;
              if (k < khi_hi && k + 32 > klo_lo) {
                tc_ld32(s, ts + c);
                tc_wait_ld();
                const int e = khi - k, b = klo - k;
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (i >= e || i < b) s[i] = 0xff800000u;
              }
              tc_st32(ts + c, s);
            }
            tc_wait_st();
          }
          uint32_t s[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tc_ld32(s + 32 * c, ts + 32 * c);
          tc_wait_ld();
          float x4[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) x4[c] = __uint_as_float(s[c]);
#pragma unroll
          for (int c = 4; c < 124; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x4[e] = fmax_nan(fmax_nan(x4[e], __uint_as_float(s[c + e])),
                               __uint_as_float(s[c + 4 + e]));
#pragma unroll
          for (int c = 0; c < 4; ++c)
            x4[c] = fmax_nan(x4[c], __uint_as_float(s[124 + c]));
          const float nm = grow(fmax_nan(fmax_nan(x4[0], x4[1]),
                                         fmax_nan(x4[2], x4[3])));
          const uint64_t nm2 = f2(nm, nm);
#pragma unroll
          for (int c = 0; c < 128; c += 2) {
            s[c >> 1] = weigh(s[c], s[c + 1], nm2, c >> 1);
            if (c + 2 == kPart) {              // the MMA may start
              tc_st32(ts, s);
              tc_st16(ts + 32, s + 32);
              tc_wait_st();
              tc_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(p_part + 8 * t);
            }
          }
          tc_st16(ts + kPart / 2, s + kPart / 2);
          tc_wait_st();
          float a0, a1;
          f2_get(f2_add(sum[0], sum[1]), a0, a1);
          l += a0 + a1;
        } else if (lane == 0) {
          mbar_arrive(p_part + 8 * t);
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * t);
      }
      if (!ok) break;
      if (few) {                                 // back to a lane per row
        l += __shfl_xor_sync(~0u, l, 1);
        l += __shfl_xor_sync(~0u, l, 2);
        l = __shfl_sync(~0u, l, (lane & 7) * 4);
        m = __shfl_sync(~0u, m, (lane & 7) * 4);
      }
      const bool paired = !two && sg.n > 1;      // both hold part of the rows
      if (t == 0 || two || paired) {
        if (!(ok = wait_warp(o_full + 8 * t, oph))) break;
        oph ^= 1;
        tc_after();
      }
      if (!two && t == 1) {
        if (!paired) continue;
        *pair_ml = make_float2(m, l);
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pair);
        // warpgroup 0 reads O_1 and (m, l) until then
        if (!(ok = wait_warp(pair_done, cph))) break;
        cph ^= 1;
        continue;
      }
      float f0 = 1.f, f1 = 0.f;
      if (paired) {
        if (!(ok = wait_warp(pair, cph))) break;
        cph ^= 1;
        tc_after();
        const float2 o = *pair_ml;
        const float mn = fmax_nan(m, o.x), ref = mn == -INFINITY ? 0.f : mn;
        f0 = ex2_approx((m - ref) * sl2);
        f1 = ex2_approx((o.x - ref) * sl2);
        l = l * f0 + o.y * f1;
        m = mn;
      }
      const bool whole = sg.first && sg.last;
      const int slot = sg.first ? 1 : 0;
      const int64_t part = (int64_t)blockIdx.x * 2 + slot;
      const bool some = l > 0.f || l != l;
      const float inv = !whole ? 1.f : some ? 1.f / l : 0.f;
      f0 *= inv;
      f1 *= inv;
      const int token = sg.tok0 + it;
      char* orow = (char*)a.out + 2 * ((int64_t)token * a.o_st +
                                       (int64_t)(sg.h * a.G + g) * a.o_sh);
      float4* prow = reinterpret_cast<float4*>(a.acc) + part * (D / 4) * 256 +
                     (two ? t : 0) * 128 + row;
      if (live) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tc_ld32(o, to + c);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            o[e] = __float_as_uint(__uint_as_float(o[e]) * f0);
          if (paired) {
            uint32_t o1[32];
            tc_ld32(o1, to + D + c);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = __float_as_uint(fmaf(__uint_as_float(o1[e]), f1,
                                          __uint_as_float(o[e])));
          }
          if (whole) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float lo = __uint_as_float(o[8 * k + 2 * x]);
                const float hi = __uint_as_float(o[8 * k + 2 * x + 1]);
                w[x] = kF16 ? pack_h2(lo, hi) : pack_bf2(lo, hi);
              }
              stage_put(stage, (c & 32) / 8 + k,
                        make_uint4(w[0], w[1], w[2], w[3]));
            }
            if (c & 32) stage_out(stage, valid ? orow + 2 * c - 64 : nullptr);
          } else if (valid) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              prow[(c + e) / 4 * 256] = make_float4(
                  __uint_as_float(o[e]), __uint_as_float(o[e + 1]),
                  __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
          }
          __syncwarp();
        }
        if (valid) {
          const float ms = m == -INFINITY ? m : m * sl2;
          if (!whole)
            a.ml[part * 256 + (two ? t : 0) * 128 + row] = make_float2(ms, l);
          else if (a.lse)
            a.lse[(int64_t)token * (a.n_kv * a.G) + sg.h * a.G + g] =
                some ? (ms + log2f(l)) * 0.6931471805599453f : -INFINITY;
        }
      }
      if (paired) {
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pair_done);
      }
      if (!whole && live) {
        // rows whose last partial this is are joined when the run is done
        __syncwarp();
        int joins = 0;
        if (lane == 0) {
          int32_t* ticket = a.tickets + sg.cta0 * 8 + warp;
          if (draw(ticket) == sg.parts - 1) {
            *ticket = 0;
            ChJob& b = jobs[warp * 2 + mine];
            b.cta0 = sg.cta0;
            b.parts = sg.parts;
            b.h = sg.h;
            b.n = rows;
            b.row0 = (two ? t : 0) * 128 + (warp & 3) * 32;
            b.tok0 = (two ? t * tm : 0) + sg.tok0;
            joins = 1;
            if (rows <= kFewRows)
              few_jobs[atomicAdd(&n_few, 1)] = warp * 2 + mine;
          }
        }
        mine += __shfl_sync(~0u, joins, 0);
        __syncwarp();
      }
    }
    for (int k = 0; k < mine; ++k) {
      const ChJob b = jobs[warp * 2 + k];
      if (b.n <= kFewRows) continue;
#pragma unroll 1
      for (int half = 0; half < X::kPanels; ++half)
        ch_join_many<D, kF16>(a, b, half, stage);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
    if (warp == 8) {
      // ------------------------------------------------------------ producer
      int st = 0;
      uint32_t ph = 1, qph = 3, vph = 0;
      while (ok && next_seg()) {
        const int tm = 1 << a.tm_log2;
        for (int t = 0; ok && t < (sg.ntok > tm ? 2 : 1); ++t) {
          if (!(ok = wait_warp(q_empty + 8 * t, (qph >> t) & 1))) break;
          qph ^= 1u << t;
          if (lane == 0) {
            mbar_arrive_expect_tx(q_full + 8 * t, X::kPanels * 128u * a.G * tm);
            for (int p = 0; p < X::kPanels; ++p)
              tma_3d(q_s + t * X::kTile + p * X::kPanel, &mq, q_full + 8 * t,
                     p * 64, sg.h * a.G, sg.tok0 + t * tm);
          }
        }
        if (!ok) break;
        const int npg = (sg.sl + kPg - 1) / kPg;
        // the first key that any of the item's rows sees
        const int lo = a.window ? max(sg.pos0 - a.window + 1, 0) : 0;
        // tiles whose V has pages with rows that somebody sees and rows that
        // nobody does
        const int tlo = lo & (kPg - 1) ? lo >> 7 : -1;
        const int thi = sg.sl & (kPg - 1) ? sg.sl >> 7 : -1;
        const int32_t* row = a.bt + (int64_t)sg.r * a.bt_stride;
        // lane 8 (t & 3) + p: block of page p of tile t, four tiles at once;
        // pages that are not the request's, or before all windows, read as
        // zeros (a block behind the cache)
        const auto blocks_of = [&](int group) {
          const int p = group * 32 + lane;
          int b = -1;
          if (p < npg && p >= (lo >> 4)) b = row[p];
          return b < 0 || b >= a.nb ? a.nb : b;
        };
        // in the order of use, `lead` tiles of K before the first of V: the
        // ring then covers the same time for both.  One loop for both: the
        // kernel is as large as the instruction caches
        const int lead = sg.ntok > tm ? 1 : 2, end = sg.t0 + sg.n;
        int kt = sg.t0, vt = sg.t0;      // the next tiles of K and of V
        int even = 0, odd = 0;           // blocks of groups of four tiles
        const auto fetch = [&](int group) {
          const int b = blocks_of(group);
          if (group & 1) odd = b; else even = b;
        };
        fetch(kt >> 2);
        if ((kt & 3) == 3) fetch((kt >> 2) + 1);
#pragma unroll 1
        while (vt < end) {
          const bool is_v = kt == end || kt - vt == lead;
          const int tile = is_v ? vt++ : kt++;
          if (!(ok = wait_warp(empty(st), ph))) break;
          const bool part = is_v && (tile == tlo || tile == thi);
          const uint32_t dst = ring + st * X::kTile;
          const uint32_t bar = part ? v_tmp : full(st);
          if (lane == 0) mbar_arrive_expect_tx(bar, X::kTile);
          __syncwarp();
          if ((lane >> 3) == (tile & 3))
            tma_5d(dst + (lane & 7) * X::kPage, is_v ? &mv : &mk, bar,
                   (tile & 4 ? odd : even) * a.bh + sg.h);
          if (!is_v && (tile & 3) == 2) fetch((tile >> 2) + 1);
          if (part) {
            // whatever the others hold, 0 * it must be 0 in P V
            if (!(ok = wait_warp(v_tmp, vph))) break;
            vph ^= 1;
            constexpr int kWords = 8 * X::kPanels;
            const int z0 = lo - tile * kKeys, z1 = sg.sl - tile * kKeys;
#pragma unroll 1
            for (int e = 0; e < 2; ++e) {
              const int r0 = e ? z1 : max(z0 & -kPg, 0);
              const int r1 = e ? min((z1 + kPg - 1) & -kPg, kKeys) : max(z0, 0);
#pragma unroll 1
              for (int i = lane; i < (r1 - r0) * kWords; i += 32) {
                const int c = i % kWords, r = r0 + i / kWords;
                const uint32_t d = dst + (r >> 3) * X::kRows8 +
                                   (c >> 3) * 1024 + (r & 7) * 128 +
                                   (c & 7) * 16;
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};"
                             :: "r"(d), "r"(0) : "memory");
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full(st));
          }
          if (++st == NS) { st = 0; ph ^= 1; }
        }
      }
      if (!ok) {
        // copies in flight end before the CTA does (a stage or a row tile
        // that never had one passes at once)
        for (int s = 0; s < NS; ++s)
          (void)mbar_wait(full(s), s < st ? ph ^ 1 : ph);
        for (int t = 0; t < 2; ++t)
          (void)mbar_wait(q_full + 8 * t, (qph >> t) & 1);
      }
    } else if (warp == 9) {
      // --------------------------------------------------------------- MMA
      // The tensor core takes the next MMA about when the last one starts, so
      // what this warp does between two MMAs is time lost.  It looks for the V
      // tile and the next K tile while it would wait for weights anyway, and
      // the whole warp walks while one elected lane issues (48 cycles a small
      // MMA in a branch of one lane, 37 elected).  Two issuing warps, one per
      // row tile, were slower: alternating MMAs of two accumulators do not
      // overlap (2048 rows behind 64K: 1900 -> 2490 us).
      constexpr uint32_t id_s = mma_idesc(kF16, false, kKeys);
      constexpr uint32_t id_o = mma_idesc(kF16, true, D);
      constexpr uint32_t kStep = X::kTile >> 4;
      const uint64_t qd = smem_desc(q_s, 16, 1024);
      const uint64_t kd = smem_desc(ring, 16, X::kRows8);
      const uint64_t vd = smem_desc(ring, 1024, X::kRows8);
      int st = 0;                        // the next ring entry and its phase
      uint32_t ph = 0, qph = 0, pph = 0;
      const auto score = [&](int t, uint64_t q0, uint64_t k0, int k) {
        mma_ss(tmem + t * 128,
               q0 + (((k >> 2) * X::kPanel + (k & 3) * 32) >> 4),
               k0 + (((k >> 2) * 1024 + (k & 3) * 32) >> 4), id_s, k > 0);
      };
      // S_t of ring entry e, which then is free when `done`
      const auto scores = [&](int t, uint64_t q0, int e, bool done) {
        const uint64_t k0 = kd + (uint32_t)e * kStep;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) score(t, q0, k0, k);
          mma_commit(s_full + 8 * t);
          if (done) mma_commit(empty(e));
        }
        __syncwarp();
      };
      // the next entry in the order of use: its index, + NS in odd phases
      const auto take = [&]() {
        const int e = st + (ph ? NS : 0);
        if (++st == NS) { st = 0; ph ^= 1; }
        return e;
      };
      const auto arrived = [&](int e) {
        return wait_warp(full(e >= NS ? e - NS : e), e >= NS);
      };
      const auto commit = [&](uint32_t bar) {
        if (elect_one()) mma_commit(bar);
        __syncwarp();
      };
      // O_t += P_t V of entry ve, the first keys of the tile as soon as their
      // weights are there, then S_t of entry ke (-1: none).  look: the entries
      // have not been seen yet (2: K may wait until P V is issued), done:
      // nothing else needs them
      const auto turn = [&](int t, int ve, bool acc, uint64_t q0, int ke,
                            int look, bool done) -> bool {
        const int v = ve >= NS ? ve - NS : ve, kn = ke >= NS ? ke - NS : ke;
        const uint64_t v0 = vd + (uint32_t)v * kStep;
        const uint64_t k0 = kd + (uint32_t)kn * kStep;
        const uint32_t p = tmem + t * 128, o = tmem + X::kO + t * D;
        const uint32_t par = (pph >> t) & 1;
        pph ^= 1u << t;
        if (look && !arrived(ve)) return false;
        if (look == 1 && ke >= 0 && !arrived(ke)) return false;
        if (!wait_warp(p_part + 8 * t, par)) return false;
        tc_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kPart / 16; ++k)
            mma_ts(o, p + k * 8, v0 + k * (X::kPage >> 4), id_o, acc || k > 0);
        }
        __syncwarp();
        if (!wait_warp(p_full + 8 * t, par)) return false;
        if (look == 2 && ke >= 0 && !arrived(ke)) return false;
        tc_after();
        if (elect_one()) {
#pragma unroll
          for (int k = kPart / 16; k < kKeys / 16; ++k)
            mma_ts(o, p + k * 8, v0 + k * (X::kPage >> 4), id_o, true);
          if (ke >= 0) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) score(t, q0, k0, k);
            mma_commit(s_full + 8 * t);
            if (done) mma_commit(empty(kn));
          } else {
            mma_commit(o_full + 8 * t);
          }
          if (done) mma_commit(empty(v));
        }
        __syncwarp();
        return true;
      };
      while (ok && next_seg()) {
        // two row tiles share every key tile; one row tile's key tiles go to
        // the two warpgroups in turn
        const int n = sg.n;
        const bool two = sg.ntok > (1 << a.tm_log2);
        int k = take(), v = 0;
        if (!(ok = wait_warp(q_full, qph & 1) && arrived(k))) break;
        const uint64_t q1 = two ? qd + kStep : qd;
#pragma unroll 1
        for (int t = 0; t < (two || n > 1 ? 2 : 1); ++t) {
          if (t) {
            if (!two) k = take();
            if (!(ok = two ? wait_warp(q_full + 8, (qph >> 1) & 1)
                           : arrived(k)))
              break;
          }
          tc_after();
          scores(t, t ? q1 : qd, k >= NS ? k - NS : k, !two || t);
        }
        if (!ok) break;
        qph ^= two ? 3 : 1;
        if (n <= (two ? 1 : 2)) commit(q_empty);
        if (two && n == 1) commit(q_empty + 8);
        const int ahead = two ? 1 : 2;
#pragma unroll 1
        for (int i = 0; i < (two ? 2 * n : n); ++i) {
          const int t = i & 1, j = two ? i >> 1 : i;
          if (!two || !t) {
            v = take();
            k = j + ahead < n ? take() : -1;
          }
          if (!(ok = turn(t, v, j >= ahead, t ? q1 : qd, k,
                          two ? 1 - t : 2, !two || t)))
            break;
          if (j + ahead + 1 == n) commit(q_empty + (two && t ? 8 : 0));
        }
      }
      // every MMA and its arrivals end before the CTA does
      commit(drain);
      ok = wait_warp(drain, 0) && ok;
    } else if (warp == 10) {
      // ------------------------------------------------------------- walk
      ch_plan_item(a, &plan);
      if (lane == 0) {
        ChWalk wk;
        wk.start(a, plan);
        for (int k = 0;; ++k) {
          ChSeg s = {};
          const bool more = wk.next(a, plan, s);
          ok = wait(seg_empty + 8 * (k % kSegs), ((k / kSegs) & 1) ^ 1);
          if (!ok) break;
          segs[k % kSegs] = s;
          mbar_arrive(seg_full + 8 * (k % kSegs));
          if (!more) break;
        }
      }
      __syncwarp();
    }
  }
  if (!ok) *a.fault = 1;
  tc_before();
  __syncthreads();
  if (warp == 9) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                 :: "r"(tmem), "r"(X::kCols));
  }
  // few rows of many partials: column blocks over all warps
  int at = warp;
  for (int k = 0; k < n_few; ++k) {
    const ChJob b = jobs[few_jobs[k]];
    const int sh = b.n <= 1 ? 0 : 32 - __clz(b.n - 1);
    for (int cg = 0; cg < D / 4; cg += 4) {
      if (at-- != 0) continue;
      at = kChThreads / 32 - 1;
      ch_join_few<D, kF16>(a, b, sh, cg);
    }
  }
}

// ------------------------------------------------------------------- host --
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t,
                             void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = []() -> EncodeFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p,
                                cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// map of a 16-bit tensor; strides (in elements) of dims 1 .. rank - 1
int make_map(CUtensorMap* m, bool f16, const void* p, int rank,
             const uint64_t* dim, const int64_t* stride, const uint32_t* box) {
  const EncodeFn fn = encode_fn();
  if (!fn) return AMASS_ERR_CUDA;
  cuuint64_t gd[5], gs[4];
  cuuint32_t bx[5], es[5];
  for (int i = 0; i < rank; ++i) {
    gd[i] = dim[i];
    bx[i] = box[i];
    es[i] = 1;
    // the stride of a dimension of one element is never used
    if (i) gs[i - 1] = dim[i] == 1 ? 16 : (cuuint64_t)stride[i] * 2;
  }
  const auto encode = [&]() {
    return fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
              (cuuint32_t)rank, const_cast<void*>(p), gd, gs, bx, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = encode();
  if (rc == CUDA_ERROR_INVALID_CONTEXT || rc == CUDA_ERROR_NOT_INITIALIZED) {
    // a host thread that has made no CUDA call yet: this one needs the
    // device's context, which the runtime's calls bind by themselves
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess)
      return AMASS_ERR_CUDA;
    rc = encode();
  }
  return rc == CUDA_SUCCESS ? AMASS_OK : AMASS_ERR_ARG;
}

template <int D, bool kF16>
int chunk_launch(const CUtensorMap& mq, const CUtensorMap& mk,
                 const CUtensorMap& mv, const ChunkArgs& a, int ctas,
                 cudaStream_t st) {
  using X = ChShape<D>;
  static DeviceOnce once;
  if (!allow_smem(once, chunk_kernel<D, kF16>, X::kSmem)) return AMASS_ERR_CUDA;
  return launch_pdl(chunk_kernel<D, kF16>, dim3(ctas), dim3(kChThreads),
                    X::kSmem, st, mq, mk, mv, a);
}

}  // namespace
}  // namespace amass

extern "C" int amass_paged_chunk_granted(const AmassChunk* args,
                                         const int32_t* status, void* stream) {
  using namespace amass;
  if (!args) return AMASS_ERR_ARG;
  const AmassChunk& x = *args;
  if (x.n_tokens < 0 || x.n_req < 0 || x.n_kv <= 0 || x.G <= 0 ||
      x.head_dim <= 0 || x.page <= 0 || x.max_pages <= 0 ||
      x.num_blocks <= 0 || x.n_ctas <= 0 || x.window < 0 ||
      !(x.scale > 0.f) || x.scale > 3e38f || x.bt_stride < 0 ||
      (x.dtype != AMASS_BF16 && x.dtype != AMASS_FP16))
    return AMASS_ERR_ARG;
  if (x.n_tokens == 0 || x.n_req == 0) return AMASS_OK;
  if (!x.q || !x.k || !x.v || !x.block_table || !x.seq_lens ||
      !x.query_start_loc || !x.acc_part || !x.ml_part || !x.tickets ||
      !x.fault || !x.out)
    return AMASS_ERR_ARG;
  if ((x.head_dim != 64 && x.head_dim != 128) || x.G > 8 || x.page != kPg ||
      x.n_req > kChMaxReq || x.max_pages > (1 << 26))
    return AMASS_ERR_UNSUPPORTED;
  // TMA and 16-byte stores: 16-byte aligned bases and strides
  const uintptr_t bases = (uintptr_t)x.q | (uintptr_t)x.k | (uintptr_t)x.v |
                          (uintptr_t)x.out | (uintptr_t)x.acc_part |
                          (uintptr_t)x.ml_part;
  if (bases & 15) return AMASS_ERR_ARG;
  const uint64_t d = (uint64_t)x.head_dim;
  const uint64_t qdim[3] = {d, (uint64_t)(x.n_kv * x.G),
                            (uint64_t)x.n_tokens};
  const int64_t qstr[3] = {1, x.q_sh, x.q_st};
  // K and V, page by page: 64 columns, 8 tokens, the panels, the page's two
  // halves, and (block, head) as one dimension of head strides
  const int panels = x.head_dim / 64;
  const auto rows = [&](int64_t sb, int64_t sh) {
    return x.n_kv == 1 ? 1 : x.num_blocks == 1 ? x.n_kv : sb / sh;
  };
  const auto bad = [](bool used, int64_t s) {
    return used && (s <= 0 || (s & 7));
  };
  if (bad(x.n_kv * x.G > 1, x.q_sh) || bad(x.n_tokens > 1, x.q_st) ||
      bad(x.n_kv * x.G > 1, x.o_sh) || bad(x.n_tokens > 1, x.o_st) ||
      bad(true, x.k_st) || bad(true, x.v_st) || bad(x.n_kv > 1, x.k_sh) ||
      bad(x.n_kv > 1, x.v_sh) || bad(x.num_blocks > 1, x.k_sb) ||
      bad(x.num_blocks > 1, x.v_sb))
    return AMASS_ERR_ARG;
  const int64_t bh = rows(x.k_sb, x.k_sh);
  if (x.n_kv > 1 && x.num_blocks > 1 &&
      (x.k_sb % x.k_sh || x.v_sb % x.v_sh || x.k_sb < x.n_kv * x.k_sh ||
       rows(x.v_sb, x.v_sh) != bh))
    return AMASS_ERR_UNSUPPORTED;
  if ((x.num_blocks + 1ll) * bh >= (1ll << 31)) return AMASS_ERR_UNSUPPORTED;
  const uint64_t kdim[5] = {64, 8, (uint64_t)panels, 2,
                            (uint64_t)((x.num_blocks - 1) * bh + x.n_kv)};
  const int64_t kstr[5] = {1, x.k_st, 64, 8 * x.k_st,
                           x.n_kv > 1 ? x.k_sh : x.k_sb};
  const int64_t vstr[5] = {1, x.v_st, 64, 8 * x.v_st,
                           x.n_kv > 1 ? x.v_sh : x.v_sb};

  ChunkArgs a = {};
  a.bt = x.block_table; a.bt_stride = x.bt_stride; a.sl = x.seq_lens;
  a.qsl = x.query_start_loc; a.status = status; a.out = x.out; a.o_st = x.o_st; a.o_sh = x.o_sh;
  a.lse = x.lse; a.acc = x.acc_part;
  a.ml = reinterpret_cast<float2*>(x.ml_part);
  a.tickets = x.tickets; a.fault = x.fault;
  a.scale_log2 = x.scale * kLog2e;
  a.n_req = x.n_req; a.n_kv = x.n_kv; a.G = x.G; a.T = x.n_tokens;
  a.bh = (int)bh; a.max_pages = x.max_pages; a.nb = x.num_blocks;
  // no request is longer than 2^30 tokens
  a.window = x.window < 1 << 30 ? x.window : 0;
  // tokens of a row tile: the largest power of two whose G heads fit 128 rows
  a.tm_log2 = x.G == 1 ? 7 : x.G == 2 ? 6 : x.G <= 4 ? 5 : 4;
  const bool f16 = x.dtype == AMASS_FP16;
  const uint32_t qbox[3] = {64, (uint32_t)x.G, 1u << a.tm_log2};
  const uint32_t kbox[5] = {64, 8, (uint32_t)panels, 2, 1};
  CUtensorMap mq, mk, mv;
  int rc = make_map(&mq, f16, x.q, 3, qdim, qstr, qbox);
  if (!rc) rc = make_map(&mk, f16, x.k, 5, kdim, kstr, kbox);
  if (!rc) rc = make_map(&mv, f16, x.v, 5, kdim, vstr, kbox);
  if (rc) return rc;
  const int ctas = x.n_ctas < num_sms() ? x.n_ctas : num_sms();
  const cudaStream_t st = (cudaStream_t)stream;
  if (x.head_dim == 128)
    return f16 ? chunk_launch<128, true>(mq, mk, mv, a, ctas, st)
               : chunk_launch<128, false>(mq, mk, mv, a, ctas, st);
  return f16 ? chunk_launch<64, true>(mq, mk, mv, a, ctas, st)
             : chunk_launch<64, false>(mq, mk, mv, a, ctas, st);
}

extern "C" int amass_paged_chunk(const AmassChunk* args, void* stream) {
  return amass_paged_chunk_granted(args, nullptr, stream);
}
