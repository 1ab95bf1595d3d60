// Rotary positions of the new tokens' q and k, with k and v written straight
// into the paged cache.
//
//   y0 = m (x0 cos a - x1 sin a),  y1 = m (x1 cos a + x0 sin a),
//   a = position * f_i,  pair i = (x_i, x_{i + r/2}) or (x_{2i}, x_{2i+1}).
//
// Angle: fp32 cannot hold position * f (at position 1e5 the product has two
// or three digits left of the turn), and a table of every position costs
// memory and a second read.  f / (2 pi) is held as the nearest 64-bit binary
// fraction of a turn; the 64-bit product with the position wraps to the
// fraction that matters, off by at most |position| * 2^-65 turns.  Its upper
// 32 bits go to sincospi in fp32, which rounds them to 24: cos and sin are
// within 2^-22 (absolute) at positions up to 2^37, twice that at 2^40.
//
// Bound: HBM.  q, k and v are read once and written once, (2H + 4 n_kv) d
// 16-bit values a token; the angles are formed once a token for all heads.
// An item is 16 elements of one head: two 16-byte loads (the two halves of 8
// pairs, or 8 neighbouring pairs), eight rotations, two 16-byte stores.  v
// and the part behind rotary_dim go through the same items with the
// rotation left out.
#include "common.cuh"

namespace amass {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotMaxDim = 256;
constexpr int kRotMaxTok = 8;            // tokens of one CTA
constexpr int kBatch = 2;
constexpr int kRotCtas = 4;              // CTAs an SM holds (64 registers)

struct RotArgs {
  const char *q, *k, *v;
  char *qo, *kd, *vd;
  int64_t q_st, q_sh, qo_st, qo_sh, k_st, k_sh, v_st, v_sh;
  int64_t kd_sb, kd_st, kd_sh, vd_sb, vd_st, vd_sh;
  const int64_t* slots;
  const void* pos;
  const uint64_t* freq;
  int64_t n_slots;
  float mscale;
  int page, pos64, rot, T, H, n_kv, d, tok;
};

template <bool kF16>
AMASS_DEV float2 unpack2(uint32_t w) {
  if (kF16) return __half22float2(*reinterpret_cast<__half2*>(&w));
  return make_float2(bf16_lo(w), bf16_hi(w));
}
template <bool kF16>
AMASS_DEV uint32_t pack2(float a, float b) {
  return kF16 ? pack_h2(a, b) : pack_bf2(a, b);
}
template <bool kF16>
AMASS_DEV float load1(const char* p) {
  const uint16_t x = *reinterpret_cast<const uint16_t*>(p);
  return unpack2<kF16>(x).x;
}
template <bool kF16>
AMASS_DEV void store1(char* p, float x) {
  *reinterpret_cast<uint16_t*>(p) = (uint16_t)pack2<kF16>(x, 0.f);
}

// row `row` (q heads, k heads, v heads) of token t
AMASS_DEV const char* rot_src(const RotArgs& a, int t, int row) {
  if (row < a.H) return a.q + 2 * (t * a.q_st + row * a.q_sh);
  row -= a.H;
  if (row < a.n_kv) return a.k + 2 * (t * a.k_st + row * a.k_sh);
  return a.v + 2 * (t * a.v_st + (row - a.n_kv) * a.v_sh);
}
// where it goes; null when there is nothing to write.  at: the slot's offset
// in the K and in the V cache, -1 without a slot
AMASS_DEV char* rot_dst(const RotArgs& a, int t, int row, longlong2 at) {
  if (row < a.H) return a.qo + 2 * (t * a.qo_st + row * a.qo_sh);
  if (at.x < 0) return nullptr;
  row -= a.H;
  if (row < a.n_kv) return a.kd + 2 * (at.x + row * a.kd_sh);
  return a.vd + 2 * (at.y + (row - a.n_kv) * a.vd_sh);
}

// Item i of n a token's `rows` times `per`, then steps of kRotThreads items:
// divisions once a thread, carries after that.
struct RotWalk {
  int j, row, c, sj, sr, sc;
  AMASS_DEV RotWalk(int rows, int per) {
    const int tok = rows * per, i = threadIdx.x;
    j = i / tok; row = (i - j * tok) / per; c = i - j * tok - row * per;
    sj = kRotThreads / tok; sr = (kRotThreads - sj * tok) / per;
    sc = kRotThreads - sj * tok - sr * per;
  }
  AMASS_DEV void step(int rows, int per) {
    c += sc;
    row += sr;
    j += sj;
    if (c >= per) { c -= per; ++row; }
    if (row >= rows) { row -= rows; ++j; }
  }
};

// kWidth: elements a lane moves at a time -- 8 (16 bytes), 2, or 1
template <bool kF16, bool kHalf, int kWidth>
__global__ void __launch_bounds__(kRotThreads, kRotCtas)
rotary_write_kernel(const __grid_constant__ RotArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  __shared__ __align__(16) float cs[kRotMaxTok][kRotMaxDim / 2];
  __shared__ __align__(16) float sn[kRotMaxTok][kRotMaxDim / 2];
  __shared__ longlong2 slot_s[kRotMaxTok];
  const int t0 = blockIdx.x * a.tok;
  const int nt = min(a.tok, a.T - t0), half = a.rot >> 1;
  const int rows = a.H + a.n_kv + (a.v ? a.n_kv : 0);
  const auto angles = [&]() {            // ends with a barrier
    for (int i = threadIdx.x; i < nt * half; i += kRotThreads) {
      const int j = i / half, p = i - j * half;
      const int64_t pos = a.pos64
          ? static_cast<const int64_t*>(a.pos)[t0 + j]
          : (int64_t)static_cast<const int32_t*>(a.pos)[t0 + j];
      const uint64_t turn = (uint64_t)pos * a.freq[p];
      // [-1/2, 1/2) turns: 2^-31 makes half turns of the upper 32 bits
      const float x = (float)(int32_t)(turn >> 32) * 4.656612873077393e-10f;
      float s, c;
      sincospif(x, &s, &c);
      cs[j][p] = c * a.mscale;
      sn[j][p] = s * a.mscale;
    }
    if ((int)threadIdx.x < nt) {
      const int64_t s = a.slots ? a.slots[t0 + threadIdx.x]
                                : (int64_t)(t0 + threadIdx.x);
      longlong2 at = make_longlong2(-1, -1);
      if (s >= 0 && s < a.n_slots) {
        const int64_t b = s / a.page, o = s - b * a.page;
        at = make_longlong2(b * a.kd_sb + o * a.kd_st,
                            b * a.vd_sb + o * a.vd_st);
      }
      slot_s[threadIdx.x] = at;
    }
    __syncthreads();
  };
  if constexpr (kWidth == 8) {
    const int per = a.d >> 4, rper = a.rot >> 4;     // items: row, rotated
    const int n = nt * rows * per;
    RotWalk wk(rows, per);
    // kBatch items of a thread in flight; the first ones' loads run while the
    // angles are formed
    for (int i0 = 0; i0 < n; i0 += kBatch * kRotThreads) {
      uint4 x[kBatch], y[kBatch];
      int at[kBatch], row[kBatch], tk[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int j = wk.j, c = wk.c;
        row[b] = wk.row;
        tk[b] = j < nt ? j : -1;
        wk.step(rows, per);
        if (j >= nt) continue;
        // the item's chunk, rotated ones with their sign bit clear
        at[b] = row[b] < a.H + a.n_kv && c < rper ? c : ~c;
        const char* src = rot_src(a, t0 + j, row[b]);
        const bool pair = kHalf && at[b] >= 0;
        const int o0 = pair ? c * 16 : c * 32, o1 = pair ? o0 + a.rot : o0 + 16;
        x[b] = *reinterpret_cast<const uint4*>(src + o0);
        y[b] = *reinterpret_cast<const uint4*>(src + o1);
      }
      if (i0 == 0) angles();
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (tk[b] < 0) continue;
        char* dst = rot_dst(a, t0 + tk[b], row[b], slot_s[tk[b]]);
        if (!dst) continue;
        const int c = at[b] >= 0 ? at[b] : ~at[b];
        if (at[b] >= 0) {
          const float4* cp = reinterpret_cast<const float4*>(&cs[tk[b]][c * 8]);
          const float4* sp = reinterpret_cast<const float4*>(&sn[tk[b]][c * 8]);
          const float4 c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
          const float cv[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
          const float sv[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
          uint32_t xw[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
          uint32_t yw[4] = {y[b].x, y[b].y, y[b].z, y[b].w};
          if (kHalf) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 u = unpack2<kF16>(xw[e]), z = unpack2<kF16>(yw[e]);
              const float ca = cv[2 * e], cb = cv[2 * e + 1];
              const float sa = sv[2 * e], sb = sv[2 * e + 1];
              xw[e] = pack2<kF16>(u.x * ca - z.x * sa, u.y * cb - z.y * sb);
              yw[e] = pack2<kF16>(z.x * ca + u.x * sa, z.y * cb + u.y * sb);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 u = unpack2<kF16>(xw[e]), z = unpack2<kF16>(yw[e]);
              xw[e] = pack2<kF16>(u.x * cv[e] - u.y * sv[e],
                                  u.y * cv[e] + u.x * sv[e]);
              yw[e] = pack2<kF16>(z.x * cv[e + 4] - z.y * sv[e + 4],
                                  z.y * cv[e + 4] + z.x * sv[e + 4]);
            }
          }
          x[b] = make_uint4(xw[0], xw[1], xw[2], xw[3]);
          y[b] = make_uint4(yw[0], yw[1], yw[2], yw[3]);
        }
        const bool pair = kHalf && at[b] >= 0;
        const int o0 = pair ? c * 16 : c * 32, o1 = pair ? o0 + a.rot : o0 + 16;
        *reinterpret_cast<uint4*>(dst + o0) = x[b];
        *reinterpret_cast<uint4*>(dst + o1) = y[b];
      }
    }
  } else if constexpr (kWidth == 2) {
    // two elements by two: a pair of neighbours, or two pairs whose halves
    // are a word each
    angles();
    const int per = kHalf ? a.d >> 2 : a.d >> 1;
    const int turned = kHalf ? half >> 1 : half;     // items of a row
    for (RotWalk wk(rows, per); wk.j < nt; wk.step(rows, per)) {
      const int j = wk.j, row = wk.row, p = wk.c;
      const char* src = rot_src(a, t0 + j, row);
      char* dst = rot_dst(a, t0 + j, row, slot_s[j]);
      if (!dst) continue;
      const bool turn = row < a.H + a.n_kv && p < turned;
      const auto ld = [&](int o) {
        return *reinterpret_cast<const uint32_t*>(src + o);
      };
      const auto st = [&](int o, uint32_t v) {
        *reinterpret_cast<uint32_t*>(dst + o) = v;
      };
      if (kHalf) {
        const int o0 = turn ? 4 * p : 8 * p, o1 = turn ? o0 + a.rot : o0 + 4;
        uint32_t x = ld(o0), y = ld(o1);
        if (turn) {
          const float2 u = unpack2<kF16>(x), z = unpack2<kF16>(y);
          const float ca = cs[j][2 * p], cb = cs[j][2 * p + 1];
          const float sa = sn[j][2 * p], sb = sn[j][2 * p + 1];
          x = pack2<kF16>(u.x * ca - z.x * sa, u.y * cb - z.y * sb);
          y = pack2<kF16>(z.x * ca + u.x * sa, z.y * cb + u.y * sb);
        }
        st(o0, x);
        st(o1, y);
      } else {
        uint32_t x = ld(4 * p);
        if (turn) {
          const float2 u = unpack2<kF16>(x);
          const float c = cs[j][p], s = sn[j][p];
          x = pack2<kF16>(u.x * c - u.y * s, u.y * c + u.x * s);
        }
        st(4 * p, x);
      }
    }
  } else {
    // pair by pair: any even rotary_dim, strides and alignment
    angles();
    const int per = a.d >> 1;
    for (RotWalk wk(rows, per); wk.j < nt; wk.step(rows, per)) {
      const int j = wk.j, row = wk.row, p = wk.c;
      const char* src = rot_src(a, t0 + j, row);
      char* dst = rot_dst(a, t0 + j, row, slot_s[j]);
      if (!dst) continue;
      const bool turn = row < a.H + a.n_kv && p < half;
      const int e0 = kHalf && turn ? p : 2 * p;
      const int e1 = kHalf && turn ? p + half : 2 * p + 1;
      if (turn) {
        const float x = load1<kF16>(src + 2 * e0);
        const float y = load1<kF16>(src + 2 * e1);
        const float c = cs[j][p], s = sn[j][p];
        store1<kF16>(dst + 2 * e0, x * c - y * s);
        store1<kF16>(dst + 2 * e1, y * c + x * s);
      } else {
        const uint16_t x = *reinterpret_cast<const uint16_t*>(src + 2 * e0);
        const uint16_t y = *reinterpret_cast<const uint16_t*>(src + 2 * e1);
        *reinterpret_cast<uint16_t*>(dst + 2 * e0) = x;
        *reinterpret_cast<uint16_t*>(dst + 2 * e1) = y;
      }
    }
  }
}

template <bool kF16, bool kHalf>
int rot_launch(const RotArgs& a, int width, cudaStream_t st) {
  const dim3 grid((unsigned)((a.T + a.tok - 1) / a.tok)), block(kRotThreads);
  if (width == 8)
    return launch_pdl(rotary_write_kernel<kF16, kHalf, 8>, grid, block, 0, st,
                      a);
  if (width == 2)
    return launch_pdl(rotary_write_kernel<kF16, kHalf, 2>, grid, block, 0, st,
                      a);
  return launch_pdl(rotary_write_kernel<kF16, kHalf, 1>, grid, block, 0, st,
                    a);
}

}  // namespace
}  // namespace amass

extern "C" int amass_rotary_write(const AmassRotary* args, void* stream) {
  using namespace amass;
  if (!args) return AMASS_ERR_ARG;
  const AmassRotary& x = *args;
  if (x.n_tokens < 0 || x.H < 0 || x.n_kv < 0 || x.head_dim <= 0 ||
      x.rotary_dim <= 0 || x.rotary_dim > x.head_dim || x.num_blocks < 0 ||
      x.page <= 0 || (x.n_tokens > 0 && (!x.positions || !x.freq)) ||
      (!x.q) != (!x.q_out) || (!x.k) != (!x.k_dst) || (!x.v) != (!x.v_dst) ||
      (x.v && !x.k) ||
      (x.layout != AMASS_ROTARY_HALF &&
       x.layout != AMASS_ROTARY_INTERLEAVED) ||
      (x.dtype != AMASS_BF16 && x.dtype != AMASS_FP16))
    return AMASS_ERR_ARG;
  if (x.head_dim > kRotMaxDim || (x.head_dim & 1) || (x.rotary_dim & 1))
    return AMASS_ERR_UNSUPPORTED;
  RotArgs a = {};
  a.q = (const char*)x.q; a.k = (const char*)x.k; a.v = (const char*)x.v;
  a.qo = (char*)x.q_out; a.kd = (char*)x.k_dst; a.vd = (char*)x.v_dst;
  a.q_st = x.q_st; a.q_sh = x.q_sh; a.qo_st = x.qo_st; a.qo_sh = x.qo_sh;
  a.k_st = x.k_st; a.k_sh = x.k_sh; a.v_st = x.v_st; a.v_sh = x.v_sh;
  a.kd_sb = x.kd_sb; a.kd_st = x.kd_st; a.kd_sh = x.kd_sh;
  a.vd_sb = x.vd_sb; a.vd_st = x.vd_st; a.vd_sh = x.vd_sh;
  a.slots = x.slot_mapping; a.pos = x.positions; a.freq = x.freq;
  a.page = x.slot_mapping ? x.page : 1;
  a.n_slots = x.slot_mapping ? (int64_t)x.num_blocks * x.page : x.n_tokens;
  a.mscale = x.mscale; a.pos64 = x.pos64; a.rot = x.rotary_dim;
  a.T = x.n_tokens; a.H = x.q ? x.H : 0; a.n_kv = x.k ? x.n_kv : 0;
  a.d = x.head_dim;
  const int head_dim = x.head_dim, rotary_dim = x.rotary_dim;
  const int n_tokens = x.n_tokens;
  if (n_tokens == 0 || a.H + a.n_kv == 0) return AMASS_OK;
  // 16-byte items need whole items in the rotated part and in the rest, and
  // 16-byte aligned rows; words need the same of two elements; what is left
  // goes one by one (8192 tokens of 8 / 2 heads of 64: rotary_dim 64 and 32
  // 8.3 us, rotary_dim 20 by words 11.0 in halves and 16.4 interleaved, one by
  // one 22.9)
  const int64_t strides = a.q_st | a.q_sh | a.qo_st | a.qo_sh | a.k_st |
                          a.k_sh | a.v_st | a.v_sh | a.kd_sb | a.kd_st |
                          a.kd_sh | a.vd_sb | a.vd_st | a.vd_sh;
  const uintptr_t base = (uintptr_t)a.q | (uintptr_t)a.qo | (uintptr_t)a.k |
                         (uintptr_t)a.kd | (uintptr_t)a.v | (uintptr_t)a.vd;
  const bool half = x.layout == AMASS_ROTARY_HALF;
  const int width =
      !(head_dim & 15) && !(rotary_dim & 15) && !(strides & 7) && !(base & 15)
          ? 8
      : !(strides & 1) && !(base & 3) &&
              (!half || (!(head_dim & 3) && !(rotary_dim & 3)))
          ? 2 : 1;
  // as many tokens a CTA as make whole waves of the CTAs that fit the GPU
  // (a last wave of a few CTAs costs as much as a full one), at least one
  const int64_t fit = (int64_t)kRotCtas * num_sms();
  const int64_t waves = (n_tokens + fit * kRotMaxTok - 1) /
                        (fit * kRotMaxTok);
  a.tok = (int)((n_tokens + fit * waves - 1) / (fit * waves));
  const cudaStream_t st = (cudaStream_t)stream;
  if (x.dtype == AMASS_FP16)
    return half ? rot_launch<true, true>(a, width, st)
                : rot_launch<true, false>(a, width, st);
  return half ? rot_launch<false, true>(a, width, st)
              : rot_launch<false, false>(a, width, st);
}
