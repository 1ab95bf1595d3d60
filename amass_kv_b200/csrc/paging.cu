// Page bookkeeping of a serving step on the GPU: block allocation, block
// table, query start offsets, token positions and slot mapping from the new
// token count of each request, and the way back (truncate / release).
//
//   begin   have_r = ceil(old_r / P), need_r = ceil((old_r + new_r) / P) -
//           have_r,
//           upto_r = need_0 + .. + need_r; request r is granted its pages iff
//           need_r = 0 or upto_r <= free blocks (in order: the first that
//           does not fit also refuses every later one that needs pages), its
//           row holds old_r + new_r tokens and the step 2^30;
//           its j-th new page takes
//           free_stack[top - 1 - (upto_r - need_r + j)];
//           token t of request r (start_r <= t < start_r + new_r) has position
//           old_r + t - start_r and slot table[r][pos / P] * P + pos % P.
//   trim    the pages behind the kept tokens return to the stack, last
//           request and last page first, so a trim of everything a begin
//           granted restores the stack to the same order.
//
// Bound: launch latency (a few KB to a few hundred KB move).  So each is one
// launch: every CTA scans all requests for itself (two sums, in shared
// memory), maps its share of the tokens, and takes the block of a new page
// straight from the free stack -- it never waits for another CTA's table
// write.  The token that opens a page writes that page's table entry.  What
// other CTAs still read (lengths, the stack's top) is committed by the CTA
// that draws the last ticket.
#include "common.cuh"

namespace amass {
namespace {

constexpr int kPgThreads = 512;
constexpr int kPgMaxReq = 4096;          // 32 KB of request sums
constexpr int kPgMaxTok = 1 << 30;       // tokens of a step

AMASS_DEV int pages_of(int tokens, int page) {   // tokens + page < 2^32
  return (int)(((unsigned)tokens + (unsigned)page - 1u) / (unsigned)page);
}

// exclusive prefix of (a, b) over the CTA's threads; *ta, *tb the totals
AMASS_DEV void scan2(int64_t& a, int64_t& b, int64_t* ta, int64_t* tb) {
  __shared__ int64_t wa[kPgThreads / 32], wb[kPgThreads / 32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int64_t ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t xa = __shfl_up_sync(~0u, ia, o);
    const int64_t xb = __shfl_up_sync(~0u, ib, o);
    if (lane >= o) { ia += xa; ib += xb; }
  }
  if (lane == 31) { wa[w] = ia; wb[w] = ib; }
  __syncthreads();
  int64_t oa = 0, ob = 0, sa = 0, sb = 0;
#pragma unroll
  for (int i = 0; i < kPgThreads / 32; ++i) {
    if (i < w) { oa += wa[i]; ob += wb[i]; }
    sa += wa[i];
    sb += wb[i];
  }
  __syncthreads();
  a = oa + ia - a;
  b = ob + ib - b;
  *ta = sa;
  *tb = sb;
}

// last i in [0, n) with start[i] <= t (start ascending, start[0] <= t)
AMASS_DEV int find_start(const int* start, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (start[m] <= t) lo = m; else hi = m;
  }
  return lo;
}

// true in every thread of the CTA that finishes last; its ticket is reset
AMASS_DEV bool last_cta(int32_t* ticket) {
  __shared__ int last;
  if (gridDim.x == 1) {
    __syncthreads();
    return true;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicAdd(ticket, 1) == (int)gridDim.x - 1;
    if (last) *ticket = 0;
    __threadfence();
  }
  __syncthreads();
  return last != 0;
}

__global__ void __launch_bounds__(kPgThreads)
pages_begin_kernel(const __grid_constant__ AmassPagePool p,
                   const int32_t* __restrict__ new_tokens, int n_req,
                   int n_tokens) {
  grid_dep_wait();
  grid_dep_launch();
  extern __shared__ int sm[];
  int* start = sm;                       // n_req + 1: first token
  int* pre = sm + n_req + 1;             // n_req: first new block, -1 refused
  __shared__ int used, reach;            // blocks granted, last token of one
  const int tid = threadIdx.x, most = p.max_pages * p.page;
  if (tid == 0) used = reach = 0;        // set before scan2's barriers
  const int top = min(max(*p.free_top, 0), p.num_blocks);
  const int per = (n_req + kPgThreads - 1) / kPgThreads;
  const int r0 = min(n_req, tid * per), r1 = min(n_req, r0 + per);
  int64_t sn = 0, sd = 0, all, need_all;  // 4096 rows can ask for 2^43 tokens
  for (int r = r0; r < r1; ++r) {
    const int nw = max(new_tokens[r], 0), old = max(p.seq_lens[r], 0);
    const int64_t want = (int64_t)old + nw;
    sn += nw;
    if (want <= most) sd += pages_of((int)want, p.page) - pages_of(old, p.page);
  }
  scan2(sn, sd, &all, &need_all);
  const int total = (int)min(all, (int64_t)kPgMaxTok);
  int flags = 0;
  for (int r = r0; r < r1; ++r) {
    const int nw = max(new_tokens[r], 0), old = max(p.seq_lens[r], 0);
    const int64_t want = (int64_t)old + nw;
    start[r] = (int)min(sn, (int64_t)kPgMaxTok);
    sn += nw;
    int st = 0, need = 0;
    if (want <= most)
      need = pages_of((int)want, p.page) - pages_of(old, p.page);
    if (want > most || (nw > 0 && sn > kPgMaxTok))
      st = 2;
    else if (need > 0 && sd + need > top)
      st = 1;
    pre[r] = st ? -1 : (int)min(sd, (int64_t)top);
    sd += need;
    flags |= st;
    if (st == 0 && need > 0) {           // granted: a prefix
      atomicMax(&used, (int)sd);
      atomicMax(&reach, (int)sn);
    }
    if (blockIdx.x == 0) {
      p.status[r] = st;
      p.query_start_loc[r] = start[r];
    }
  }
  if (tid == 0) {
    start[n_req] = total;
    if (blockIdx.x == 0) p.query_start_loc[n_req] = total;
  }
  __syncthreads();

  const int end = max(reach, n_tokens);
  for (int64_t t = (int64_t)blockIdx.x * kPgThreads + tid; t < end;
       t += (int64_t)gridDim.x * kPgThreads) {
    int64_t pos = 0, slot = -1;
    if (t < total) {
      const int r = find_start(start, n_req, (int)t);
      const int old = max(p.seq_lens[r], 0);   // committed after the ticket
      pos = (int64_t)old + (t - start[r]);
      const int pg = (int)((unsigned)pos / (unsigned)p.page);
      const int off = (int)pos - pg * p.page;
      if (pre[r] >= 0 && pos < most) {
        const int have = pages_of(old, p.page);
        int32_t* e = p.block_table + (int64_t)r * p.bt_stride + pg;
        int b = -1;
        if (pg < have) {
          b = *e;
        } else {
          const int k = top - 1 - (pre[r] + pg - have);
          if (k >= 0) {
            b = p.free_stack[k];
            if (off == 0) *e = b;
          }
        }
        if (b >= 0) slot = (int64_t)b * p.page + off;
      }
    }
    if (t < n_tokens) {
      p.positions[t] = pos;
      p.slot_mapping[t] = slot;
    }
  }
  const int short_f = __syncthreads_or(flags & 1);
  const int long_f = __syncthreads_or(flags & 2);
  if (!last_cta(p.ticket)) return;
  for (int r = r0; r < r1; ++r) {
    if (pre[r] < 0) continue;
    p.seq_lens[r] = max(p.seq_lens[r], 0) + (start[r + 1] - start[r]);
  }
  if (tid == 0) {
    *p.free_top = top - used;
    const int f = (short_f ? 1 : 0) | (long_f ? 2 : 0) |
                  (all > n_tokens ? 4 : 0);
    if (f) *p.overflow |= f;
  }
}

__global__ void __launch_bounds__(kPgThreads)
pages_trim_kernel(const __grid_constant__ AmassPagePool p,
                  const int32_t* __restrict__ drop, int n_req, int whole) {
  grid_dep_wait();
  grid_dep_launch();
  extern __shared__ int sm[];
  int* start = sm;                       // n_req + 1: first freed page, in
                                         // order of descending request
  int* left = sm + n_req + 1;            // n_req: tokens kept, by request
  const int tid = threadIdx.x;
  const int top = min(max(*p.free_top, 0), p.num_blocks);
  const int per = (n_req + kPgThreads - 1) / kPgThreads;
  const int i0 = min(n_req, tid * per), i1 = min(n_req, i0 + per);
  const auto kept = [&](int r, int* have) {
    const int old = min(max(p.seq_lens[r], 0), p.max_pages * p.page);
    const int d = whole ? (drop[r] != 0 ? old : 0)
                        : min(max(drop[r], 0), old);
    *have = pages_of(old, p.page);
    return old - d;
  };
  int64_t s = 0, zero = 0, all, z;
  for (int i = i0; i < i1; ++i) {
    int have;
    const int k = kept(n_req - 1 - i, &have);
    s += have - pages_of(k, p.page);
  }
  scan2(s, zero, &all, &z);
  const int total = (int)all;            // held pages: no more than blocks
  for (int i = i0; i < i1; ++i) {
    const int r = n_req - 1 - i;
    int have;
    left[r] = kept(r, &have);
    start[i] = (int)s;
    s += have - pages_of(left[r], p.page);
  }
  if (tid == 0) start[n_req] = total;
  __syncthreads();
  for (int k = blockIdx.x * kPgThreads + tid; k < total;
       k += gridDim.x * kPgThreads) {
    const int i = find_start(start, n_req, k), r = n_req - 1 - i;
    // the request's freed pages are keep .. keep + n - 1, last one first
    const int n = start[i + 1] - start[i];
    const int pg = pages_of(left[r], p.page) + n - 1 - (k - start[i]);
    int32_t* e = p.block_table + (int64_t)r * p.bt_stride + pg;
    if (top + k < p.num_blocks) p.free_stack[top + k] = *e;
    *e = -1;
  }
  if (!last_cta(p.ticket)) return;
  for (int i = i0; i < i1; ++i) p.seq_lens[n_req - 1 - i] = left[n_req - 1 - i];
  if (tid == 0) *p.free_top = min(top + total, p.num_blocks);
}

__global__ void __launch_bounds__(kPgThreads)
slot_map_kernel(const int32_t* __restrict__ block_table, int64_t bt_stride,
                const int32_t* __restrict__ seq_lens,
                const int32_t* __restrict__ query_start_loc, int n_req,
                int64_t* __restrict__ positions,
                int64_t* __restrict__ slot_mapping, int n_tokens,
                int max_pages, int page) {
  grid_dep_wait();
  grid_dep_launch();
  extern __shared__ int sm[];
  for (int i = threadIdx.x; i <= n_req; i += kPgThreads)
    sm[i] = query_start_loc[i];
  __syncthreads();
  for (int64_t t = (int64_t)blockIdx.x * kPgThreads + threadIdx.x;
       t < n_tokens; t += (int64_t)gridDim.x * kPgThreads) {
    int64_t pos = 0, slot = -1;
    if (t >= sm[0] && t < sm[n_req]) {
      const int r = find_start(sm, n_req, (int)t);
      pos = (int64_t)seq_lens[r] - (sm[r + 1] - t);
      const int pg = (int)((unsigned)pos / (unsigned)page);
      if (pos >= 0 && pos < (int64_t)max_pages * page) {
        const int b = block_table[(int64_t)r * bt_stride + pg];
        if (b >= 0) slot = (int64_t)b * page + ((int)pos - pg * page);
      }
    }
    positions[t] = pos;
    slot_mapping[t] = slot;
  }
}

int grid_for(int64_t items, int per_cta) {
  const int64_t n = (items + per_cta - 1) / per_cta;
  return (int)(n < 1 ? 1 : n > num_sms() ? num_sms() : n);
}

}  // namespace
}  // namespace amass

static bool pool_ok(const AmassPagePool* p) {
  return p && p->block_table && p->seq_lens && p->free_stack && p->free_top &&
         p->query_start_loc && p->positions && p->slot_mapping && p->status &&
         p->overflow && p->ticket && p->bt_stride >= 0 && p->num_blocks > 0 &&
         p->max_reqs > 0 && p->max_pages > 0 && p->max_tokens > 0 &&
         p->page > 0 && (int64_t)p->max_pages * p->page < (1ll << 31);
}

extern "C" int amass_pages_begin(const AmassPagePool* pool,
                                 const int32_t* new_tokens, int n_req,
                                 int n_tokens, void* stream) {
  using namespace amass;
  if (!pool_ok(pool) || n_req < 0 || n_req > pool->max_reqs || n_tokens < 0 ||
      n_tokens > pool->max_tokens || (n_req > 0 && !new_tokens))
    return AMASS_ERR_ARG;
  if (n_req > kPgMaxReq) return AMASS_ERR_UNSUPPORTED;
  return launch_pdl(pages_begin_kernel, dim3(grid_for(n_tokens, kPgThreads)),
                    dim3(kPgThreads), (2 * n_req + 1) * sizeof(int),
                    (cudaStream_t)stream, *pool, new_tokens, n_req, n_tokens);
}

extern "C" int amass_pages_trim(const AmassPagePool* pool, const int32_t* drop,
                                int n_req, int whole, void* stream) {
  using namespace amass;
  if (!pool_ok(pool) || n_req < 0 || n_req > pool->max_reqs ||
      (n_req > 0 && !drop))
    return AMASS_ERR_ARG;
  if (n_req > kPgMaxReq) return AMASS_ERR_UNSUPPORTED;
  if (n_req == 0) return AMASS_OK;
  // the number of pages that return is known on the device only: a whole
  // release may free every row, a truncation mostly a page or two per request
  const int64_t most = whole ? (int64_t)n_req * pool->max_pages : 4ll * n_req;
  return launch_pdl(pages_trim_kernel, dim3(grid_for(most, 4 * kPgThreads)),
                    dim3(kPgThreads), (2 * n_req + 1) * sizeof(int),
                    (cudaStream_t)stream, *pool, drop, n_req, whole);
}

extern "C" int amass_slot_map(const int32_t* block_table, int64_t bt_stride,
                              const int32_t* seq_lens,
                              const int32_t* query_start_loc, int n_req,
                              int64_t* positions, int64_t* slot_mapping,
                              int n_tokens, int max_pages, int page,
                              void* stream) {
  using namespace amass;
  if (n_req < 0 || n_tokens < 0 || max_pages <= 0 || page <= 0 ||
      bt_stride < 0 || !query_start_loc ||
      (n_tokens > 0 && (!positions || !slot_mapping)) ||
      (n_req > 0 && (!block_table || !seq_lens)))
    return AMASS_ERR_ARG;
  if (n_req > kPgMaxReq) return AMASS_ERR_UNSUPPORTED;
  if (n_tokens == 0) return AMASS_OK;
  return launch_pdl(slot_map_kernel, dim3(grid_for(n_tokens, kPgThreads)),
                    dim3(kPgThreads), (n_req + 1) * sizeof(int),
                    (cudaStream_t)stream, block_table, bt_stride, seq_lens,
                    query_start_loc, n_req, positions, slot_mapping, n_tokens,
                    max_pages, page);
}
