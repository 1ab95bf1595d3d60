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
//   warp 8          TMA producer: Q, then K and V tiles page by page (a 16-row
//                   box per page and 64-column panel) into a ring
//   warp 9          issues the tcgen05 MMAs: S = Q K^T (both operands in
//                   shared memory, fp32 S in TMEM), O += P V (P in TMEM over
//                   S's columns, V as a column-major operand, fp32 O in TMEM)
//
// While one row tile's softmax runs, the tensor core works for the other.
// O is rescaled only when a row's maximum grows by more than 2^8 (p stays
// below 256, exact in the 16-bit P's range); sums stay in fp32 registers; the
// one rounding to 16 bits before the end is P's (half a step per weight).
//
// Work split: the (item, key tile) units of the whole batch form one flat
// list; every CTA takes an equal run of it.  Lengths live on the device, so
// each CTA scans the requests and finds its own run.  Items cut by a run's
// end leave unnormalised partials that the merge kernel joins.  This serves a
// single token over a long context (all SMs read one request's cache) and a
// large prefill (no tail of uneven causal tiles) with one rule.
//
// Slots behind a request's last token may hold anything: K's scores there
// are replaced before the maximum, V's rows are zeroed in shared memory.
#include <cuda.h>

#include "common.cuh"

namespace amass {
namespace {

constexpr int kChThreads = 384;          // three warpgroups (two idle warps)
constexpr int kKeys = 128;               // keys of a tile
constexpr int kPg = 16;                  // tokens of a page
constexpr int kChMaxReq = 4096;
constexpr int kMinUnits = 2;             // key tiles a run has at least
constexpr float kRescaleLog2 = 8.f;
constexpr int kPart = 96;                // keys whose weights go to O first

struct ChunkArgs {
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* sl;
  const int32_t* qsl;
  void* out;
  int64_t o_st, o_sh;
  float* lse;                            // (T, H) or null
  float* acc;                            // [cta][2][D / 4][256][4]
  float2* ml;                            // [cta][2][256]
  int4* meta;                            // [cta]: parts, token, tokens, head
  int32_t* fault;
  float scale_log2;
  int n_req, n_kv, G, T, max_pages, nb, window, tm_log2;
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
AMASS_DEV uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
AMASS_DEV void tma_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x,
                      int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      :: "r"(dst), "l"(m), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
AMASS_DEV void tma_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x,
                      int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      :: "r"(dst), "l"(m), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// ------------------------------------------------------------- work list ---
// One request: its rows start at q0, ql of them; row i has position off + i.
struct ChReq {
  int q0, ql, sl, off, nt;
};
AMASS_DEV ChReq ch_req(const ChunkArgs& a, int r) {
  ChReq q;
  const int s0 = a.qsl[r], s1 = a.qsl[r + 1];
  q.q0 = max(s0, 0);
  q.ql = max(min(s1, a.T) - q.q0, 0);
  // a length beyond the block table's row is cut: no page behind it exists
  q.sl = max((int)min((int64_t)a.sl[r], (int64_t)a.max_pages * kPg), 0);
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
AMASS_DEV int64_t shift_sum(int64_t x, int s) {
  const int64_t q = x >> s;
  return ((q * (q - 1) / 2) << s) + q * (x - (q << s));
}
// sum over i in [i0, i1) of max(b + i * 2^tl, 0) >> 7
AMASS_DEV int64_t floor_sum(int64_t b, int64_t i0, int64_t i1, int tl) {
  if (b < 0) {                           // first i with a value above 0
    const int64_t z = ((-b) >> tl) + 1;
    i0 = (i0 > z ? i0 : z) - z;
    i1 -= z;
    b += z << tl;
  }
  if (i0 >= i1) return 0;
  if (tl >= 7) {
    const int64_t n = i1 - i0;
    return n * (b >> 7) + (((i0 + i1 - 1) * n / 2) << (tl - 7));
  }
  const int64_t c = b >> tl;
  return shift_sum(i1 + c, 7 - tl) - shift_sum(i0 + c, 7 - tl);
}
// units of items 0 .. m - 1 of the request (closed form of ch_tiles' sum)
AMASS_DEV int64_t ch_units(const ChunkArgs& a, const ChReq& q, int m) {
  const int tl = a.tm_log2 + 1;
  if (m <= 0) return 0;
  int64_t s = 0;
  int full = m;
  if (m == q.nt) {                       // the last item may be short
    int lo;
    s = ch_tiles(a, q, m - 1, &lo);
    full = m - 1;
  }
  // items whose last position is negative visit one (empty) tile
  const int none = q.off < 0 ? min(full, (-q.off) >> tl) : 0;
  s += none;
  s += floor_sum((int64_t)q.off + (1 << tl) + kKeys - 1, none, full, tl);
  if (a.window)
    s -= floor_sum((int64_t)q.off - a.window + 1, none, full, tl);
  return s;
}

struct ChSeg {
  int r, h, q0, tok0, ntok, off, sl, t0, n, left;
  bool first, last;
};
struct ChPlan {
  ChReq q;
  int r, h, i, uoff, rem, share;
  long long u1;
};

// Walks the segments of a CTA's run; every role keeps its own copy.  A first
// segment that starts inside its item goes last: then every CTA starts at its
// item's first key tile, and since the runs are equally long the late pieces
// of one head's items meet at the same key tiles again.  CTAs of a head so
// stream its K and V together and read them from L2 (2048 rows behind 64K
// tokens: DRAM would have to deliver 64 KB per CTA and unit otherwise).
struct ChWalk {
  ChReq q;
  int r, h, i, uoff, rem, late;          // late: units of the deferred segment
  AMASS_DEV void start(const ChunkArgs& a, const ChPlan& p) {
    q = p.q; r = p.r; h = p.h; i = p.i; uoff = p.uoff; rem = p.rem;
    late = 0;
    if (uoff > 0 && rem > 0) {
      int lo;
      const int n = min(rem, ch_tiles(a, q, i, &lo) - uoff);
      if (n < rem) {
        late = n;
        rem -= n;
        uoff = 0;
        step(a);
      }
    }
  }
  AMASS_DEV void step(const ChunkArgs& a) {
    if (++i < q.nt) return;
    i = 0;
    if (++h < a.n_kv) return;
    h = 0;
    if (rem <= 0) return;
    do {
      if (++r >= a.n_req) break;
      q = ch_req(a, r);
    } while (q.nt == 0);
  }
  AMASS_DEV bool next(const ChunkArgs& a, const ChPlan& p, ChSeg& s) {
    if (rem <= 0 || r >= a.n_req) {
      if (late == 0) return false;
      q = p.q; r = p.r; h = p.h; i = p.i; uoff = p.uoff; rem = late;
      late = 0;
    }
    const int tl = a.tm_log2 + 1;
    int lo;
    const int nu = ch_tiles(a, q, i, &lo);
    s.r = r; s.h = h; s.q0 = q.q0; s.off = q.off; s.sl = q.sl;
    s.tok0 = i << tl;
    s.ntok = min(1 << tl, q.ql - s.tok0);
    s.t0 = lo + uoff;
    s.n = min(rem, nu - uoff);
    s.first = uoff == 0;
    s.left = nu - uoff - s.n;
    s.last = s.left == 0;
    rem -= s.n;
    uoff = 0;
    step(a);
    return true;
  }
};

// this CTA's run of the flat unit list
AMASS_DEV void ch_plan(const ChunkArgs& a, ChPlan* out) {
  __shared__ long long wsum[kChThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int per = (a.n_req + kChThreads - 1) / kChThreads;
  const int r0 = min(a.n_req, tid * per), r1 = min(a.n_req, r0 + per);
  long long mine = 0, units = 0;
  ChReq q;
  for (int r = r0; r < r1; ++r) {
    q = ch_req(a, r);
    units = ch_units(a, q, q.nt);
    mine += units * a.n_kv;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) wsum[w] = incl;
  if (tid == 0) out->rem = 0;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int i = 0; i < kChThreads / 32; ++i) {
    if (i < w) before += wsum[i];
    total += wsum[i];
  }
  long long share = (total + gridDim.x - 1) / gridDim.x;
  if (share < kMinUnits) share = kMinUnits;
  long long u0 = share * blockIdx.x;
  const long long u1 = min(total, u0 + share);
  if (u0 >= before && u0 < before + mine) {
    u0 -= before;
    for (int r = r0; r < r1; ++r) {
      if (per > 1) {                     // one request: still in registers
        q = ch_req(a, r);
        units = ch_units(a, q, q.nt);
      }
      const long long all = units * a.n_kv;
      if (u0 >= all) {
        u0 -= all;
        continue;
      }
      const int h = all >> 32 ? (int)(u0 / units)
                              : (int)((uint32_t)u0 / (uint32_t)units);
      u0 -= h * units;
      int lo = 0, hi = q.nt;             // last item that starts at or before
      while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (ch_units(a, q, m) <= u0) lo = m; else hi = m;
      }
      out->q = q;
      out->r = r;
      out->h = h;
      out->i = lo;
      out->uoff = (int)(u0 - ch_units(a, q, lo));
      out->rem = (int)(u1 - share * blockIdx.x);
      out->share = (int)share;
      out->u1 = u1;
      break;
    }
  }
  __syncthreads();
}

template <int D>
struct ChShape {
  static constexpr int kPanels = D / 64;
  static constexpr int kTile = kKeys * D * 2;        // bytes of a K or V tile
  static constexpr int kPanel = kKeys * 128;         // bytes of a panel
  static constexpr int kStages = 163840 / kTile;     // 160 KB of ring
  static constexpr int kSmem = 2 * kTile + kStages * kTile + 1024;
  static constexpr uint32_t kCols = 512;             // 2 S/P + 2 O
  static constexpr uint32_t kO = 256;
};

template <int D, bool kF16>
__global__ void __launch_bounds__(kChThreads, 1)
chunk_kernel(const __grid_constant__ CUtensorMap mq,
             const __grid_constant__ CUtensorMap mk,
             const __grid_constant__ CUtensorMap mv, const ChunkArgs a) {
  using X = ChShape<D>;
  constexpr int NS = X::kStages;
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[2 * NS + 14];
  __shared__ float2 ml_s[128];           // warpgroup 1's (m, l), one-tile items
  __shared__ ChPlan plan;
  __shared__ uint32_t tmem_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const uint32_t base = (smem_u32(dyn) + 1023u) & ~1023u;
  const uint32_t q_s = base, ring = base + 2 * X::kTile;
  const uint32_t b0 = smem_u32(bars);
  const auto full = [&](int s) { return b0 + 8u * s; };
  const auto empty = [&](int s) { return b0 + 8u * (NS + s); };
  const uint32_t q_full = b0 + 8u * (2 * NS), q_empty = q_full + 8;
  const uint32_t s_full = q_full + 16, p_full = q_full + 32;   // two each
  const uint32_t o_full = q_full + 48, p_part = q_full + 64;   // two each
  const uint32_t v_tmp = q_full + 80, drain = v_tmp + 8;
  const uint32_t pair = v_tmp + 16, pair_done = v_tmp + 24;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + 8 * t, 1);
      mbar_init(p_part + 8 * t, 4);
      mbar_init(p_full + 8 * t, 4);
      mbar_init(o_full + 8 * t, 1);
    }
    mbar_init(v_tmp, 1);
    mbar_init(drain, 1);
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
  if (tid == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);

  // bounded wait: after about a second the CTA records the fault and unwinds
  const auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    if (mbar_wait(bar, parity)) return true;
    *a.fault = 1;
    return false;
  };
  // the same for whole warps, which have to unwind together
  const auto wait_warp = [&](uint32_t bar, uint32_t parity) -> bool {
    return __all_sync(~0u, wait(bar, parity));
  };

  ChWalk wk;
  wk.start(a, plan);
  ChSeg sg;

  // a softmax thread holds a row of 128 scores: 384 * 168 registers at launch
  // = 128 * (2 * 208 + 88)
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------------- softmax
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + t * 128 + lanes;
    const uint32_t to = tmem + X::kO + t * D + lanes;
    const int tok = row / a.G, g = row - tok * a.G, tm = 1 << a.tm_log2;
    const float sl2 = a.scale_log2;
    const uint64_t sl2x2 = f2(sl2, sl2);
    uint32_t sph = 0, oph = 0, cph = 0;
    bool ok = true;
    while (ok && wk.next(a, plan, sg)) {
      const bool two = sg.ntok > tm;
      const int it = (two ? t * tm : 0) + tok;   // token within the item
      const bool valid = tok < tm && it < sg.ntok;
      const int pos = sg.off + sg.tok0 + it;
      const int khi = valid ? max(pos + 1, 0) : 0;
      const int klo = a.window ? max(pos - a.window + 1, 0) : 0;
      const bool live = __any_sync(~0u, valid);
      float m = -INFINITY, l = 0.f;
      for (int j = two ? 0 : t; j < sg.n; j += two ? 1 : 2) {
        if (!(ok = wait_warp(s_full + 8 * t, sph))) break;
        sph ^= 1;
        tc_after();
        if (live) {
          uint32_t s[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tc_ld32(s + 32 * c, ts + 32 * c);
          tc_wait_ld();
          const int k0 = (sg.t0 + j) * kKeys;
          if (__any_sync(~0u, k0 + kKeys > khi || k0 < klo)) {
            const int e = khi - k0, b = klo - k0;
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if (c >= e || c < b) s[c] = 0xff800000u;
          }
          float x4[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) x4[c] = __uint_as_float(s[c]);
#pragma unroll
          for (int c = 4; c < 124; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x4[e] = fmaxf(fmaxf(x4[e], __uint_as_float(s[c + e])),
                            __uint_as_float(s[c + 4 + e]));
#pragma unroll
          for (int c = 0; c < 4; ++c)
            x4[c] = fmaxf(x4[c], __uint_as_float(s[124 + c]));
          const float mx = fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3]));
          if (j < 2 - (two ? 1 : 0)) {           // this warpgroup's first tile
            m = mx;
          } else if (__any_sync(~0u, (mx - m) * sl2 > kRescaleLog2)) {
            const float mn = fmaxf(m, mx);
            const float f = m == -INFINITY ? 0.f : ex2_approx((m - mn) * sl2);
            l *= f;
            m = mn;
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
          }
          const float nm = m == -INFINITY ? 0.f : -m * sl2;
          const uint64_t nm2 = f2(nm, nm);
          uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 128; c += 2) {
            float p0, p1;
            f2_get(f2_fma(f2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])),
                          sl2x2, nm2), p0, p1);
            p0 = ex2_approx(p0);
            p1 = ex2_approx(p1);
            sum[(c >> 1) & 1] = f2_add(sum[(c >> 1) & 1], f2(p0, p1));
            s[c >> 1] = kF16 ? pack_h2(p0, p1) : pack_bf2(p0, p1);
            if (c + 2 == kPart) {                // the MMA may start
              tc_st32(ts, s);
              tc_st16(ts + 32, s + 32);
              tc_wait_st();
              tc_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(p_part + 8 * t);
            }
          }
          tc_st16(ts + kPart / 2, s + kPart / 2);
          float a0, a1;
          f2_get(f2_add(sum[0], sum[1]), a0, a1);
          l += a0 + a1;
          tc_wait_st();
        } else if (lane == 0) {
          mbar_arrive(p_part + 8 * t);
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * t);
      }
      if (!ok) break;
      const bool paired = !two && sg.n > 1;      // both hold part of the rows
      if (t == 0 || two || paired) {
        if (!(ok = wait_warp(o_full + 8 * t, oph))) break;
        oph ^= 1;
        tc_after();
      }
      if (!two && t == 1) {
        if (!paired) continue;
        ml_s[row] = make_float2(m, l);
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pair);
        // warpgroup 0 reads O_1 and ml_s until then
        if (!(ok = wait_warp(pair_done, cph))) break;
        cph ^= 1;
        continue;
      }
      float f0 = 1.f, f1 = 0.f;
      if (paired) {
        if (!(ok = wait_warp(pair, cph))) break;
        cph ^= 1;
        tc_after();
        const float2 o = ml_s[row];
        const float mn = fmaxf(m, o.x), ref = mn == -INFINITY ? 0.f : mn;
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
      const int token = sg.q0 + sg.tok0 + it;
      char* orow = (char*)a.out + 2 * ((int64_t)token * a.o_st +
                                       (int64_t)(sg.h * a.G + g) * a.o_sh);
      float4* prow = reinterpret_cast<float4*>(a.acc) + part * (D / 4) * 256 +
                     (two ? t : 0) * 128 + row;
      if (live) {
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t o[16];
          tc_ld16(o, to + c);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[e] = __float_as_uint(__uint_as_float(o[e]) * f0);
          if (paired) {
            uint32_t o1[16];
            tc_ld16(o1, to + D + c);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = __float_as_uint(fmaf(__uint_as_float(o1[e]), f1,
                                          __uint_as_float(o[e])));
          }
          if (valid && whole) {
            uint32_t w[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const float lo = __uint_as_float(o[2 * x]);
              const float hi = __uint_as_float(o[2 * x + 1]);
              w[x] = kF16 ? pack_h2(lo, hi) : pack_bf2(lo, hi);
            }
            uint4* d = reinterpret_cast<uint4*>(orow + 2 * c);
            d[0] = make_uint4(w[0], w[1], w[2], w[3]);
            d[1] = make_uint4(w[4], w[5], w[6], w[7]);
          } else if (valid) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
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
      if (!whole && sg.first && tid == 0) {
        // the CTAs behind this one that hold the rest of the item
        const long long end = plan.u1 + sg.left;
        a.meta[blockIdx.x] =
            make_int4((int)((end - 1) / plan.share) - (int)blockIdx.x,
                      sg.q0 + sg.tok0, sg.ntok, sg.h);
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8) {
      // ------------------------------------------------------------ producer
      int st = 0, issued = 0;
      uint32_t ph = 1, qph = 1;
      bool ok = true;
      while (ok && wk.next(a, plan, sg)) {
        const int tm = 1 << a.tm_log2;
        if (!(ok = wait_warp(q_empty, qph))) break;
        qph ^= 1;
        if (lane == 0) {
          const int halves = sg.ntok > tm ? 2 : 1;
          mbar_arrive_expect_tx(q_full,
                                halves * X::kPanels * 128u * a.G * tm);
          for (int t = 0; t < halves; ++t)
            for (int p = 0; p < X::kPanels; ++p)
              tma_3d(q_s + t * X::kTile + p * X::kPanel, &mq, q_full, p * 64,
                     sg.h * a.G, sg.q0 + sg.tok0 + t * tm);
        }
        const int npg = (sg.sl + kPg - 1) / kPg;
        const int32_t* row = a.bt + (int64_t)sg.r * a.bt_stride;
        // block of the tile's page (lane & 7); pages that are not the
        // request's read as zeros (a block behind the cache)
        const auto block_of = [&](int tile) {
          const int p = tile * (kKeys / kPg) + (lane & 7);
          int b = -1;
          if (p < npg) b = row[p];
          return b < 0 || b >= a.nb ? a.nb : b;
        };
        int blk = block_of(sg.t0);
        for (int j = 0; ok && j < sg.n; ++j) {
          const int tile = sg.t0 + j;
          const int nxt = j + 1 < sg.n ? block_of(tile + 1) : 0;
          const bool part = (sg.sl & (kPg - 1)) && tile == (sg.sl - 1) >> 7;
          for (int kv = 0; kv < 2; ++kv) {
            if (!(ok = wait_warp(empty(st), ph))) break;
            const uint32_t dst = ring + st * X::kTile;
            const uint32_t bar = kv && part ? v_tmp : full(st);
            if (lane == 0) mbar_arrive_expect_tx(bar, X::kTile);
            __syncwarp();
            if (lane < 8 * X::kPanels)
              tma_4d(dst + (lane >> 3) * X::kPanel + (lane & 7) * (kPg * 128),
                     kv ? &mv : &mk, bar, (lane >> 3) * 64, sg.h, 0, blk);
            if (kv && part) {
              // rows behind the last token: whatever they hold, 0 * it must
              // be 0 in P V
              if (!(ok = wait_warp(v_tmp, (issued >> 16) & 1))) break;
              const int r0 = sg.sl & (kPg - 1);
              const int at = (((sg.sl - 1) & (kKeys - 1)) & ~(kPg - 1)) + r0;
              const int words = (kPg - r0) * 8 * X::kPanels;
              for (int i = lane; i < words; i += 32) {
                const int p = i / ((kPg - r0) * 8), x = i - p * (kPg - r0) * 8;
                const uint32_t d = dst + p * X::kPanel + at * 128 + x * 16;
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};"
                             :: "r"(d), "r"(0) : "memory");
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0) mbar_arrive(full(st));
              issued ^= 1 << 16;
            }
            if (++st == NS) { st = 0; ph ^= 1; }
          }
          blk = nxt;
        }
      }
      if (!ok) {
        // copies in flight end before the CTA does
        for (int s = 0; s < NS; ++s)
          (void)mbar_wait(full(s), s < st ? (ph ^ 1) & 1 : ph & 1);
      }
    } else if (warp == 9) {
      // ----------------------------------------------------------------- MMA
      if (lane == 0) {
        constexpr uint32_t id_s = mma_idesc(kF16, false, kKeys);
        constexpr uint32_t id_o = mma_idesc(kF16, true, D);
        uint32_t seq = 0, qph = 0, pph = 0;
        bool ok = true;
        // K of tile j is the ring's entry seq + 2 j, V the one behind it
        const auto stage = [&](uint32_t n) { return (int)(n % NS); };
        const auto arrived = [&](uint32_t n) {
          return wait(full(stage(n)), (n / NS) & 1);
        };
        const auto scores = [&](int t, int qt, uint32_t n) {
          const uint32_t qa = q_s + qt * X::kTile;
          const uint32_t ka = ring + stage(n) * X::kTile;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t o = (k >> 2) * X::kPanel + (k & 3) * 32;
            mma_ss(tmem + t * 128, smem_desc(qa + o, 16, 1024),
                   smem_desc(ka + o, 16, 1024), id_s, k > 0);
          }
          mma_commit(s_full + 8 * t);
        };
        // O_t += P_t V, the first keys of the tile as soon as their weights
        // are there
        const auto product = [&](int t, uint32_t n, bool acc) -> bool {
          const uint32_t va = ring + stage(n) * X::kTile, p = (pph >> t) & 1;
          pph ^= 1u << t;
          if (!wait(p_part + 8 * t, p)) return false;
          tc_after();
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) {
            if (k == kPart / 16) {
              if (!wait(p_full + 8 * t, p)) return false;
              tc_after();
            }
            mma_ts(tmem + X::kO + t * D, tmem + t * 128 + k * 8,
                   smem_desc(va + k * 2048, X::kPanel, 1024), id_o,
                   acc || k > 0);
          }
          return true;
        };
        while (ok && wk.next(a, plan, sg)) {
          const bool two = sg.ntok > (1 << a.tm_log2);
          const int n = sg.n;
          if (!(ok = wait(q_full, qph))) break;
          qph ^= 1;
          if (!(ok = arrived(seq))) break;
          tc_after();
          scores(0, 0, seq);
          if (two) scores(1, 1, seq);
          mma_commit(empty(stage(seq)));
          if (two) {
            if (n == 1) mma_commit(q_empty);
            for (int j = 0; ok && j < n; ++j) {
              const uint32_t v = seq + 2 * j + 1, k = v + 1;
              const bool more = j + 1 < n;
              ok = arrived(v) && (!more || arrived(k));
              for (int t = 0; ok && t < 2; ++t) {
                if (!(ok = product(t, v, j > 0))) break;
                if (more) scores(t, t, k);
                else mma_commit(o_full + 8 * t);
              }
              if (!ok) break;
              mma_commit(empty(stage(v)));
              if (more) mma_commit(empty(stage(k)));
              if (j + 2 == n) mma_commit(q_empty);
            }
          } else {
            // one row tile: the two warpgroups take its key tiles in turn
            if (n > 1) {
              if (!(ok = arrived(seq + 2))) break;
              tc_after();
              scores(1, 0, seq + 2);
              mma_commit(empty(stage(seq + 2)));
            }
            if (n <= 2) mma_commit(q_empty);
            for (int j = 0; j < n; ++j) {
              const uint32_t v = seq + 2 * j + 1, k = v + 3;
              const int t = j & 1;
              const bool more = j + 2 < n;
              ok = arrived(v) && (!more || arrived(k)) &&
                   product(t, v, j > 1);
              if (!ok) break;
              mma_commit(empty(stage(v)));
              if (more) {
                scores(t, 0, k);
                mma_commit(empty(stage(k)));
              } else {
                mma_commit(o_full + 8 * t);
              }
              if (j + 3 == n) mma_commit(q_empty);
            }
          }
          seq += 2 * n;
        }
        // every MMA and its arrivals end before the CTA does
        mma_commit(drain);
        (void)mbar_wait(drain, 0);
      }
      __syncwarp();
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 9) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                 :: "r"(tmem), "r"(X::kCols));
  }
}

// Joins the partials of the item that starts in CTA blockIdx.x's run and ends
// in a later one: out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c.  One
// thread per row and 16 columns.
template <int D, bool kF16>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const ChunkArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int4 mt = a.meta[blockIdx.x];
  if (mt.x <= 0) return;
  const int row256 = threadIdx.x, t = row256 >> 7, row = row256 & 127;
  const int tok = row / a.G, g = row - tok * a.G, tm = 1 << a.tm_log2;
  const int it = t * tm + tok;
  if (tok >= tm || it >= mt.z) return;
  const int64_t p0 = (int64_t)blockIdx.x * 2 + 1;      // then slot 0 of the
  const int64_t p1 = (int64_t)blockIdx.x * 2 + 2;      // following CTAs
  float M = -INFINITY;
  for (int c = 0; c <= mt.x; ++c)
    M = fmaxf(M, a.ml[(c ? p1 + 2 * (c - 1) : p0) * 256 + row256].x);
  const float ref = M == -INFINITY ? 0.f : M;
  const int cg = blockIdx.y * 4;
  float o[16], l = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e] = 0.f;
#pragma unroll 2
  for (int c = 0; c <= mt.x; ++c) {
    const int64_t p = c ? p1 + 2 * (c - 1) : p0;
    const float2 ml = a.ml[p * 256 + row256];
    const float w = ex2_approx(ml.x - ref);
    l += w * ml.y;
    const float4* x = reinterpret_cast<const float4*>(a.acc) +
                      (p * (D / 4) + cg) * 256 + row256;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 v = x[e * 256];
      o[4 * e] += w * v.x;
      o[4 * e + 1] += w * v.y;
      o[4 * e + 2] += w * v.z;
      o[4 * e + 3] += w * v.w;
    }
  }
  const bool some = l > 0.f || l != l;
  const float inv = some ? 1.f / l : 0.f;
  const int head = mt.w * a.G + g;
  const int64_t token = mt.y + it;
  uint4* dst = reinterpret_cast<uint4*>(
      (char*)a.out + 2 * (token * a.o_st + head * a.o_sh + cg * 4));
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    uint32_t w[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float lo = o[8 * e + 2 * x] * inv, hi = o[8 * e + 2 * x + 1] * inv;
      w[x] = kF16 ? pack_h2(lo, hi) : pack_bf2(lo, hi);
    }
    dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (a.lse && blockIdx.y == 0)
    a.lse[token * (a.n_kv * a.G) + head] =
        some ? (M + log2f(l)) * 0.6931471805599453f : -INFINITY;
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
  cuuint64_t gd[4], gs[3];
  cuuint32_t bx[4], es[4];
  for (int i = 0; i < rank; ++i) {
    gd[i] = dim[i];
    bx[i] = box[i];
    es[i] = 1;
    // the stride of a dimension of one element is never used
    if (i) gs[i - 1] = dim[i] == 1 ? 16 : (cuuint64_t)stride[i] * 2;
  }
  return fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            (cuuint32_t)rank, const_cast<void*>(p), gd, gs, bx, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? AMASS_OK : AMASS_ERR_ARG;
}

template <int D, bool kF16>
int chunk_launch(const CUtensorMap& mq, const CUtensorMap& mk,
                 const CUtensorMap& mv, const ChunkArgs& a, int ctas,
                 cudaStream_t st) {
  using X = ChShape<D>;
  static unsigned long long mask = 0;
  if (first_on_device(mask) &&
      cudaFuncSetAttribute(chunk_kernel<D, kF16>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                           X::kSmem) != cudaSuccess)
    return AMASS_ERR_CUDA;
  const int rc = launch_pdl(chunk_kernel<D, kF16>, dim3(ctas),
                            dim3(kChThreads), X::kSmem, st, mq, mk, mv, a);
  if (rc) return rc;
  return launch_pdl(chunk_merge_kernel<D, kF16>, dim3(ctas, D / 16),
                    dim3(256), 0, st, a);
}

}  // namespace
}  // namespace amass

extern "C" int amass_paged_chunk(const AmassChunk* args, void* stream) {
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
      !x.query_start_loc || !x.acc_part || !x.ml_part || !x.meta ||
      !x.fault || !x.out)
    return AMASS_ERR_ARG;
  if ((x.head_dim != 64 && x.head_dim != 128) || x.G > 8 || x.page != kPg ||
      x.n_req > kChMaxReq || x.max_pages > (1 << 26))
    return AMASS_ERR_UNSUPPORTED;
  // TMA and 16-byte stores: 16-byte aligned bases and strides
  const uintptr_t bases = (uintptr_t)x.q | (uintptr_t)x.k | (uintptr_t)x.v |
                          (uintptr_t)x.out | (uintptr_t)x.acc_part |
                          (uintptr_t)x.ml_part | (uintptr_t)x.meta;
  if ((bases & 15) || ((x.o_st | x.o_sh) & 7)) return AMASS_ERR_ARG;
  const uint64_t d = (uint64_t)x.head_dim;
  const uint64_t qdim[3] = {d, (uint64_t)(x.n_kv * x.G),
                            (uint64_t)x.n_tokens};
  const uint64_t kdim[4] = {d, (uint64_t)x.n_kv, (uint64_t)kPg,
                            (uint64_t)x.num_blocks};
  const int64_t qstr[3] = {1, x.q_sh, x.q_st};
  const int64_t kstr[4] = {1, x.k_sh, x.k_st, x.k_sb};
  const int64_t vstr[4] = {1, x.v_sh, x.v_st, x.v_sb};
  const auto bad = [](uint64_t n, int64_t s) {
    return n > 1 && (s <= 0 || (s & 7));
  };
  for (int i = 1; i < 4; ++i)
    if ((i < 3 && bad(qdim[i], qstr[i])) || bad(kdim[i], kstr[i]) ||
        bad(kdim[i], vstr[i]))
      return AMASS_ERR_ARG;

  ChunkArgs a = {};
  a.bt = x.block_table; a.bt_stride = x.bt_stride; a.sl = x.seq_lens;
  a.qsl = x.query_start_loc; a.out = x.out; a.o_st = x.o_st; a.o_sh = x.o_sh;
  a.lse = x.lse; a.acc = x.acc_part;
  a.ml = reinterpret_cast<float2*>(x.ml_part);
  a.meta = reinterpret_cast<int4*>(x.meta); a.fault = x.fault;
  a.scale_log2 = x.scale * kLog2e;
  a.n_req = x.n_req; a.n_kv = x.n_kv; a.G = x.G; a.T = x.n_tokens;
  a.max_pages = x.max_pages; a.nb = x.num_blocks; a.window = x.window;
  // tokens of a row tile: the largest power of two whose G heads fit 128 rows
  a.tm_log2 = x.G == 1 ? 7 : x.G == 2 ? 6 : x.G <= 4 ? 5 : 4;
  const bool f16 = x.dtype == AMASS_FP16;
  const uint32_t qbox[3] = {64, (uint32_t)x.G, 1u << a.tm_log2};
  const uint32_t kbox[4] = {64, 1, (uint32_t)kPg, 1};
  CUtensorMap mq, mk, mv;
  int rc = make_map(&mq, f16, x.q, 3, qdim, qstr, qbox);
  if (!rc) rc = make_map(&mk, f16, x.k, 4, kdim, kstr, kbox);
  if (!rc) rc = make_map(&mv, f16, x.v, 4, kdim, vstr, kbox);
  if (rc) return rc;
  const int ctas = x.n_ctas < num_sms() ? x.n_ctas : num_sms();
  const cudaStream_t st = (cudaStream_t)stream;
  if (x.head_dim == 128)
    return f16 ? chunk_launch<128, true>(mq, mk, mv, a, ctas, st)
               : chunk_launch<128, false>(mq, mk, mv, a, ctas, st);
  return f16 ? chunk_launch<64, true>(mq, mk, mv, a, ctas, st)
             : chunk_launch<64, false>(mq, mk, mv, a, ctas, st);
}
