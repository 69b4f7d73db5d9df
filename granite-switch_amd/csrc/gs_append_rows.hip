// Rows into and out of a quantised paged cache, and the norms of queries and keys for
// each head in the pass that rotates and stores them.
//
// A row (a head's key or value of one token) is kept as e4m3 values y and one power of
// two 2^e, x = y 2^e, with e the least integer that keeps the row's largest finite
// magnitude within 448 2^e (e >= -126): the product with 2^-e is exact, so a value is
// rounded once, by at most 2^-4 of itself down to 2^-6 2^e, and any factor between two
// powers of two would leave it the same relative error.  e + 127 is the scale's byte.
//
// gs_append_kv_normed: x rsqrt(mean(x^2) + eps) w over a head's columns, rotation, and for
// keys and values the row's exponent and its e4m3 values, in fp32 throughout.  A head's
// columns are held by 2^n adjacent lanes (8 for 128 bf16 columns, 16 each), which add
// squares and find the maximum by lane permutes; nothing is read twice.
//
// gs_read_kv: rows by their slots, y 2^e; both are one read and one write, the memory rate
// bounds them.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "gs_append.h"

namespace gs {
namespace {

struct RowsArgs {
  AppendArgs a;
  const void* qw;                                    // norm weights [D] or NULL
  const void* kw;
  bool w_bf16;
  float eps, inv_d;
  uint8_t* ks;                                       // scales; a head's of a page side by side
  uint8_t* vs;
  int64_t ks_ps, ks_hs, vs_ps, vs_hs;
  int lanes, lanes_log;                              // of a head
};

// Sums, and maxima, over the 2^n adjacent lanes of a head.
template <int CTRL>
__device__ __forceinline__ float dpp_other(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, false));
}
template <class F>
__device__ __forceinline__ float over_lanes(float x, int lanes, const F& f) {
  if (lanes > 1) x = f(x, dpp_other<0xB1>(x));       // lanes 1, 2 apart
  if (lanes > 2) x = f(x, dpp_other<0x4E>(x));
  if (lanes > 4) x = f(x, dpp_other<0x141>(x));      // mirrored in 8, in 16: the other four, the other eight
  if (lanes > 8) x = f(x, dpp_other<0x140>(x));
  if (lanes > 16) x = f(x, __shfl_xor(x, 16, 64));
  if (lanes > 32) x = f(x, __shfl_xor(x, 32, 64));
  return x;
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.402823466e+38f; }

// The partners x0 and x1 of a unit, turned: VE columns each of half-split pairs, or
// VE / 2 side-by-side pairs each.
template <int VE, bool PAIRS>
__device__ __forceinline__ void rotate(float* x0, float* x1, const float* cs, const float* sn) {
  const auto turn = [](float& a, float& b, float c, float s) {
    const float p = a, q = b;
    a = p * c - q * s;
    b = q * c + p * s;
  };
  if constexpr (!PAIRS || VE == 1) {
#pragma unroll
    for (int i = 0; i < VE; ++i) turn(x0[i], x1[i], cs[i], sn[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) {
      turn(x0[2 * i], x0[2 * i + 1], cs[i], sn[i]);
      turn(x1[2 * i], x1[2 * i + 1], cs[VE / 2 + i], sn[VE / 2 + i]);
    }
  }
}

// VE values as e4m3 in the low bytes; what is not finite becomes NaN.
template <int VE>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float* x, float inv) {
  float y[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) y[i] = is_finite(x[i]) ? x[i] * inv : __uint_as_float(0x7fc00000u);
  if constexpr (VE == 1) {
    *p = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[0], 0, false));
  } else {
    uint32_t w[VE / 4];
#pragma unroll
    for (int i = 0; i < VE / 4; ++i) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
      w[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], lo, true));
    }
    if constexpr (VE == 8) *reinterpret_cast<uint64_t*>(p) = w[0] | (static_cast<uint64_t>(w[1]) << 32);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// Thread mapping as append_kv_kernel's (gs_append.hip) with a head's units on a power of
// two of lanes, NU to a lane: the vector forms have one, the scalar one a wave for a head.
template <bool BF16, int VE, bool PAIRS, bool QUANT>
__global__ __launch_bounds__(256) void append_rows_kernel(RowsArgs r) {
  constexpr int NU = VE == 1 ? 4 : 1;
  constexpr int kBatch = VE == 1 ? 1 : 4;            // heads whose loads are in flight together
  const AppendArgs& a = r.a;
  const int tid = threadIdx.x;
  const int per_token = a.groups << r.lanes_log;
  const int tok = tid / per_token;
  if (tok >= a.tokens) return;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * a.tokens + tok;
  if (t >= a.T) return;
  const int in_tok = tid - tok * per_token;
  const int grp = in_tok >> r.lanes_log, u0 = in_tok & (r.lanes - 1);
  addr::AppendCols c[NU];
  float cs[NU][VE], sn[NU][VE], wq[NU][2][VE], wk[NU][2][VE];
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const int u = u0 + n * r.lanes;
    c[n] = u < a.units ? addr::append_cols(u, VE, a.D, a.R, PAIRS) : addr::AppendCols{-1, -1, false};
    if (c[n].rot) {
      const float* row = a.cos_sin + addr::append_pos(a.positions[t], a.max_pos) * a.R;
      const int j0 = addr::append_pair(u, VE);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        cs[n][i] = row[j0 + i];
        sn[n][i] = row[a.R / 2 + j0 + i];
      }
    }
    const auto weights = [&](const void* w, float (*to)[VE]) {
      if (w == nullptr) return;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = x == 0 ? c[n].c0 : c[n].c1;
#pragma unroll
        for (int i = 0; i < VE; ++i)
          to[x][i] = col < 0 ? 0.f : r.w_bf16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(w)[col + i]) : static_cast<const float*>(w)[col + i];
      }
    };
    weights(r.qw, wq[n]);
    weights(r.kw, wk[n]);
  }
  const int64_t slot = a.slots[t];
  const bool stored = addr::append_stored(slot, a.num_slots);
  const uint32_t page = stored ? static_cast<uint32_t>(static_cast<uint64_t>(slot) / a.page_size) : 0u;
  const uint32_t prow = stored ? static_cast<uint32_t>(slot - static_cast<int64_t>(page) * a.page_size) : 0u;
  const int heads = a.H + 2 * a.HK;
  for (int h0 = grp; h0 < heads; h0 += kBatch * a.groups) {
    float x0[kBatch][NU][VE], x1[kBatch][NU][VE];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * a.groups;
      if (h >= heads) continue;
      const bool isq = h < a.H, isk = !isq && h < a.H + a.HK;
      const void* src = isq ? a.q : isk ? a.k : a.v;
      const int64_t base = isq ? t * a.q_ts + h * a.q_hs
                         : isk ? t * a.k_ts + (h - a.H) * a.k_hs : t * a.v_ts + (h - a.H - a.HK) * a.v_hs;
#pragma unroll
      for (int n = 0; n < NU; ++n) {
#pragma unroll
        for (int i = 0; i < VE; ++i) x0[b][n][i] = x1[b][n][i] = 0.f;
        if (c[n].c0 >= 0) append_load<BF16, VE>(src, base + c[n].c0, x0[b][n]);
        if (c[n].c1 >= 0) append_load<BF16, VE>(src, base + c[n].c1, x1[b][n]);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * a.groups;
      if (h >= heads) continue;
      const bool isq = h < a.H, isk = !isq && h < a.H + a.HK;
      if (!isq && !stored) continue;
      if ((isq && r.qw != nullptr) || (isk && r.kw != nullptr)) {
        float ss = 0.f;
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
          for (int i = 0; i < VE; ++i) ss += x0[b][n][i] * x0[b][n][i] + x1[b][n][i] * x1[b][n][i];
        ss = over_lanes(ss, r.lanes, [](float x, float y) { return x + y; });
        const float f = rsqrtf(ss * r.inv_d + r.eps);
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            x0[b][n][i] *= f * (isq ? wq : wk)[n][0][i];
            x1[b][n][i] *= f * (isq ? wq : wk)[n][1][i];
          }
      }
#pragma unroll
      for (int n = 0; n < NU; ++n)
        if (c[n].rot && (isq || isk)) rotate<VE, PAIRS>(x0[b][n], x1[b][n], cs[n], sn[n]);
      float inv = 1.f;
      if (QUANT && !isq) {
        float m = 0.f;
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            m = is_finite(x0[b][n][i]) ? fmaxf(m, fabsf(x0[b][n][i])) : m;
            m = is_finite(x1[b][n][i]) ? fmaxf(m, fabsf(x1[b][n][i])) : m;
          }
        m = over_lanes(m, r.lanes, [](float x, float y) { return fmaxf(x, y); });
        const int code = addr::e8m0_of(__float_as_uint(m));
        inv = __uint_as_float(static_cast<uint32_t>(254 - code) << 23);
        if (u0 == 0) {
          if (isk) r.ks[page * r.ks_ps + (h - a.H) * r.ks_hs + prow] = static_cast<uint8_t>(code);
          else r.vs[page * r.vs_ps + (h - a.H - a.HK) * r.vs_hs + prow] = static_cast<uint8_t>(code);
        }
      }
      void* dst = isq ? a.q_out : isk ? a.kc : a.vc;
      const int64_t base = isq ? t * a.qo_ts + h * a.qo_hs
                         : isk ? page * a.kc_ps + (h - a.H) * a.kc_hs + prow * a.kc_rs
                               : page * a.vc_ps + (h - a.H - a.HK) * a.vc_hs + prow * a.vc_rs;
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        if (c[n].c0 < 0) continue;
        if (QUANT && !isq) {
          store_e4m3<VE>(static_cast<uint8_t*>(dst) + base + c[n].c0, x0[b][n], inv);
          if (c[n].c1 >= 0) store_e4m3<VE>(static_cast<uint8_t*>(dst) + base + c[n].c1, x1[b][n], inv);
        } else {
          append_store<BF16, VE>(dst, base + c[n].c0, x0[b][n]);
          if (c[n].c1 >= 0) append_store<BF16, VE>(dst, base + c[n].c1, x1[b][n]);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Read
// ---------------------------------------------------------------------------
struct ReadArgs {
  const void* c[2];                                  // key and value cache
  const uint8_t* s[2];                               // scales, or NULL
  void* out[2];
  int64_t ps[2], hs[2], rs[2], s_ps[2], s_hs[2], o_ts[2], o_hs[2];
  const int64_t* slots;
  int64_t num_slots;
  uint32_t page_size;
  int T, HK, D;
  int pieces, tokens;                                // of a head; of a workgroup
  uint32_t row_magic, piece_magic;                   // div_magic(HK * pieces), div_magic(pieces)
};

enum class Held { kE4m3, kBf16, kFp32 };             // a cache's elements

// VE elements of one row.  The product is exact in bf16 and fp32: e4m3 has four bits.
template <Held HELD, bool BF16, int VE>
__device__ __forceinline__ void read_piece(const ReadArgs& r, int w, int64_t at, float scale, bool live, int64_t to) {
  if constexpr (HELD != Held::kE4m3) {
    constexpr int kSize = HELD == Held::kBf16 ? 2 : 4;
    const char* p = static_cast<const char*>(r.c[w]) + at * kSize;
    char* o = static_cast<char*>(r.out[w]) + to * kSize;
    if constexpr (VE == 1 && kSize == 2) *reinterpret_cast<uint16_t*>(o) = live ? *reinterpret_cast<const uint16_t*>(p) : uint16_t(0);
    else if constexpr (VE == 1) *reinterpret_cast<uint32_t*>(o) = live ? *reinterpret_cast<const uint32_t*>(p) : 0u;
    else st16(o, sel16(live, ld16(p)));
  } else if constexpr (VE == 1) {
    const uint32_t x = static_cast<const uint8_t*>(r.c[w])[at];
    const f32x2_t f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, scale, false);
    const float y = live ? f[0] : 0.f;
    if constexpr (BF16) static_cast<uint16_t*>(r.out[w])[to] = f32_to_bf16_bits(y);
    else static_cast<float*>(r.out[w])[to] = y;
  } else {
    const u32x4 x = sel16(live, ld16(static_cast<const uint8_t*>(r.c[w]) + at));
    if constexpr (BF16) {
      u32x4 y[2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i >> 1][2 * (i & 1)] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], scale, false));
        y[i >> 1][2 * (i & 1) + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], scale, true));
      }
      uint16_t* o = static_cast<uint16_t*>(r.out[w]) + to;
      st16(o, y[0]);
      st16(o + 8, y[1]);
    } else {
      float* o = static_cast<float*>(r.out[w]) + to;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x[i], scale, false);
        const f32x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x[i], scale, true);
        *reinterpret_cast<f32x4*>(o + 4 * i) = f32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    }
  }
}

// A workgroup takes `tokens` tokens of the keys (blockIdx.y 0) or the values; a thread a
// piece of VE columns, every 256-th of the workgroup's.
template <Held HELD, bool BF16, int VE>
__global__ __launch_bounds__(256) void read_kv_kernel(ReadArgs r) {
  const int w = blockIdx.y;
  const int row = r.HK * r.pieces;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * r.tokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(r.tokens), r.T - t0)) * row;
#pragma unroll 4
  for (int x = threadIdx.x; x < n; x += 256) {
    uint32_t tok, in, h, piece;
    addr::div_by(x, row, r.row_magic, tok, in);
    addr::div_by(in, r.pieces, r.piece_magic, h, piece);
    const int64_t t = t0 + tok;
    const int64_t slot = r.slots[t];
    const bool live = addr::append_stored(slot, r.num_slots);
    const uint32_t page = live ? static_cast<uint32_t>(static_cast<uint64_t>(slot) / r.page_size) : 0u;
    const uint32_t prow = live ? static_cast<uint32_t>(slot - static_cast<int64_t>(page) * r.page_size) : 0u;
    const int col = static_cast<int>(piece) * VE;
    float scale = 1.f;
    if constexpr (HELD == Held::kE4m3) scale = live ? e8m0_scale(r.s[w][page * r.s_ps[w] + h * r.s_hs[w] + prow]) : 1.f;
    read_piece<HELD, BF16, VE>(r, w, page * r.ps[w] + h * r.hs[w] + prow * r.rs[w] + col, scale, live, t * r.o_ts[w] + h * r.o_hs[w] + col);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// Heads and tokens of a workgroup as gs_append_kv's.
void plan_rows(RowsArgs& r, int ve, int cus) {
  AppendArgs& a = r.a;
  a.units = addr::append_units(ve, a.D, a.R);
  r.lanes_log = 0;
  while ((1 << r.lanes_log) < a.units && r.lanes_log < 6) ++r.lanes_log;
  r.lanes = 1 << r.lanes_log;
  const int n = a.H + 2 * a.HK;
  const int most = 256 >> r.lanes_log;
  a.groups = std::max(1, std::min(a.T <= 2 * cus ? n : (n + 3) / 4, most));
  a.tokens = most / a.groups;
}

void plan_read(ReadArgs& r, int ve) {
  r.pieces = r.D / ve;
  const int row = r.HK * r.pieces;
  r.tokens = std::max(1, 1024 / row);
  r.row_magic = addr::div_magic(row);
  r.piece_magic = addr::div_magic(r.pieces);
}

bool multiples(int n, std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s < 0 || s % n != 0) return false;
  return true;
}
bool aligned_to(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <int VE, bool PAIRS>
void model_rows_append(PagedModel& m, const RowsArgs& r, bool quant, const int64_t* slots, const int64_t* positions) {
  constexpr int NU = VE == 1 ? 4 : 1;
  const AppendArgs& a = r.a;
  const int64_t pages = a.num_slots / a.page_size;
  const int64_t q_elems = extent3(a.T, a.q_ts, a.H, a.q_hs, 1, 0, a.D), qo_elems = extent3(a.T, a.qo_ts, a.H, a.qo_hs, 1, 0, a.D);
  const int64_t k_elems = extent3(a.T, a.k_ts, a.HK, a.k_hs, 1, 0, a.D);
  const int64_t c_elems = extent3(pages, a.kc_ps, a.HK, a.kc_hs, a.page_size, a.kc_rs, a.D);
  const int64_t s_elems = extent3(pages, r.ks_ps, a.HK, r.ks_hs, a.page_size, 1, 1);
  const int heads = a.H + 2 * a.HK;
  const int per_token = a.groups << r.lanes_log;
  if (per_token * a.tokens > 256 || a.tokens < 1) m.fail("threads of a workgroup", 0, per_token * a.tokens, 256);
  if (a.units > NU * r.lanes) m.fail("units of a head", 0, a.units, NU * r.lanes);
  std::vector<int> seen(static_cast<size_t>(heads) * a.D), scales(heads);
  for (int64_t blk = 0; blk * a.tokens < a.T && !m.bad; ++blk)
    for (int tok = 0; tok < a.tokens && blk * a.tokens + tok < a.T; ++tok) {
      const int64_t t = blk * a.tokens + tok;
      std::fill(seen.begin(), seen.end(), 0);
      std::fill(scales.begin(), scales.end(), 0);
      const bool stored = addr::append_stored(slots[t], a.num_slots);
      const int64_t page = stored ? slots[t] / a.page_size : 0, prow = stored ? slots[t] - page * a.page_size : 0;
      for (int in_tok = 0; in_tok < per_token; ++in_tok)
        for (int n = 0; n < NU; ++n) {
          const int grp = in_tok >> r.lanes_log, u0 = in_tok & (r.lanes - 1), u = u0 + n * r.lanes;
          if (u >= a.units) continue;
          const addr::AppendCols c = addr::append_cols(u, VE, a.D, a.R, PAIRS);
          if (c.rot) {
            const int64_t row = addr::append_pos(positions[t], a.max_pos) * a.R;
            m.in("cosines", row + addr::append_pair(u, VE), VE, row + a.R / 2);
            m.in("cos_sin", row + a.R / 2 + addr::append_pair(u, VE), VE, a.max_pos * a.R);
          }
          for (int h = grp; h < heads; h += a.groups) {
            if (u0 == 0 && n == 0 && h >= a.H) {
              ++scales[h];
              if (quant && stored) m.in("scales", page * r.ks_ps + (h < a.H + a.HK ? h - a.H : h - a.H - a.HK) * r.ks_hs + prow, 1, s_elems);
            }
            for (int col : {c.c0, c.c1}) {
              if (col < 0) continue;
              m.in("norm weights", col, VE, a.D);
              for (int i = 0; i < VE && col + i < a.D; ++i) ++seen[static_cast<size_t>(h) * a.D + col + i];
              if (h < a.H) {
                m.in("q", t * a.q_ts + h * a.q_hs + col, VE, q_elems);
                m.in("q_out", t * a.qo_ts + h * a.qo_hs + col, VE, qo_elems);
              } else {
                const int hk = h < a.H + a.HK ? h - a.H : h - a.H - a.HK;
                m.in("k or v", t * a.k_ts + hk * a.k_hs + col, VE, k_elems);
                if (stored) m.in("cache", page * a.kc_ps + hk * a.kc_hs + prow * a.kc_rs + col, VE, c_elems);
              }
            }
          }
        }
      for (int h = a.H; h < heads; ++h)
        if (scales[h] != 1 && !m.bad) m.fail("a scale written other than once", h, scales[h], 1);
      for (size_t i = 0; i < seen.size(); ++i)
        if (seen[i] != 1 && !m.bad) m.fail("a column taken other than once", static_cast<int64_t>(i), 1, a.D);
    }
}

void model_read(PagedModel& m, const ReadArgs& r, int ve, const int64_t* slots) {
  const int64_t pages = r.num_slots / r.page_size, row = static_cast<int64_t>(r.HK) * r.pieces;
  const int64_t c_elems = extent3(pages, r.ps[0], r.HK, r.hs[0], r.page_size, r.rs[0], r.D);
  const int64_t s_elems = extent3(pages, r.s_ps[0], r.HK, r.s_hs[0], r.page_size, 1, 1);
  const int64_t o_elems = extent3(r.T, r.o_ts[0], r.HK, r.o_hs[0], 1, 0, r.D);
  std::vector<char> seen(static_cast<size_t>(r.T) * row, 0);
  for (int64_t t0 = 0; t0 < r.T && !m.bad; t0 += r.tokens) {
    const int n = static_cast<int>(std::min<int64_t>(r.tokens, r.T - t0) * row);
    for (int x = 0; x < n; ++x) {
      uint32_t tok, in, h, piece;
      addr::div_by(x, static_cast<uint32_t>(row), r.row_magic, tok, in);
      addr::div_by(in, r.pieces, r.piece_magic, h, piece);
      const int64_t t = t0 + tok;
      m.in("slots", t, 1, r.T);
      m.in("head", h, 1, r.HK);
      if (m.bad) return;
      ++seen[t * row + h * r.pieces + piece];
      const bool live = addr::append_stored(slots[t], r.num_slots);
      const int64_t page = live ? slots[t] / r.page_size : 0, prow = live ? slots[t] - page * r.page_size : 0;
      m.in("cache", page * r.ps[0] + h * r.hs[0] + prow * r.rs[0] + piece * ve, ve, c_elems);
      m.in("scales", page * r.s_ps[0] + h * r.s_hs[0] + prow, 1, s_elems);
      m.in("out", t * r.o_ts[0] + h * r.o_hs[0] + piece * ve, ve, o_elems);
    }
  }
  for (char c : seen)
    if (c != 1 && !m.bad) m.fail("a piece taken other than once", 0, c, 1);
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

int gs_append_kv_normed(int32_t dtype, const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts,
                        int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs, int64_t num_tokens, int32_t heads,
                        int32_t kv_heads, int32_t head_dim, const void* q_norm, const void* k_norm, int32_t norm_dtype,
                        float eps, const int64_t* positions, const float* cos_sin, int64_t max_pos, int32_t rot_dim,
                        int32_t interleaved, const int64_t* slots, int32_t cache_dtype, void* k_cache, int64_t kc_ps,
                        int64_t kc_hs, int64_t kc_rs, void* v_cache, int64_t vc_ps, int64_t vc_hs, int64_t vc_rs,
                        uint8_t* k_scales, int64_t ks_ps, int64_t ks_hs, uint8_t* v_scales, int64_t vs_ps,
                        int64_t vs_hs, int64_t num_pages, int32_t page_size, void* q_out, int64_t qo_ts, int64_t qo_hs,
                        void* stream) {
  const char* who = "gs_append_kv_normed";
  GS_CHECK_ARG(dtype == GS_DTYPE_BF16 || dtype == GS_DTYPE_FP32, "%s: dtype=%d", who, dtype);
  GS_CHECK_ARG(cache_dtype == dtype || cache_dtype == GS_DTYPE_E4M3, "%s: cache_dtype=%d with dtype=%d", who, cache_dtype, dtype);
  GS_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t(1) << 31), "%s: num_tokens=%lld", who, (long long)num_tokens);
  GS_CHECK_ARG(heads >= 0 && kv_heads > 0 && heads <= 4096 && kv_heads <= 4096, "%s: heads=%d kv_heads=%d", who, heads, kv_heads);
  GS_CHECK_ARG(head_dim > 0 && head_dim <= 512, "%s: head_dim=%d (1 .. 512)", who, head_dim);
  GS_CHECK_ARG(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 2 == 0, "%s: rot_dim=%d of head_dim=%d", who, rot_dim, head_dim);
  GS_CHECK_ARG(page_size > 0 && num_pages > 0, "%s: page_size=%d num_pages=%lld", who, page_size, (long long)num_pages);
  GS_CHECK_ARG((q_norm == nullptr && k_norm == nullptr) || norm_dtype == dtype || norm_dtype == GS_DTYPE_FP32,
               "%s: norm_dtype=%d with dtype=%d", who, norm_dtype, dtype);
  GS_CHECK_ARG(eps >= 0.f, "%s: eps=%g", who, static_cast<double>(eps));
  if (num_tokens == 0) return GS_OK;
  const bool quant = cache_dtype == GS_DTYPE_E4M3;
  // the stride of a dimension of one is never used, and may be anything
  if (num_tokens == 1) q_ts = k_ts = v_ts = qo_ts = 0;
  if (heads == 1) q_hs = qo_hs = 0;
  if (kv_heads == 1) k_hs = v_hs = kc_hs = vc_hs = ks_hs = vs_hs = 0;
  if (num_pages == 1) kc_ps = vc_ps = ks_ps = vs_ps = 0;
  if (page_size == 1) kc_rs = vc_rs = 0;
  GS_CHECK_ARG(k != nullptr && v != nullptr && slots != nullptr && k_cache != nullptr && v_cache != nullptr &&
                   (heads == 0 || (q != nullptr && q_out != nullptr)) && (!quant || (k_scales != nullptr && v_scales != nullptr)),
               "%s: null tensor", who);
  GS_CHECK_ARG(rot_dim == 0 || (positions != nullptr && cos_sin != nullptr && max_pos > 0),
               "%s: rot_dim=%d without positions or cos_sin", who, rot_dim);
  const bool bf16 = dtype == GS_DTYPE_BF16;
  const int ve = bf16 ? 8 : 4;
  const auto fits = [&](const void* p, int64_t ts, int64_t hs) { return aligned16(p) && multiples(ve, {ts, hs}); };
  const int cache_align = quant ? ve : 16;           // bytes of a store
  const bool vec = head_dim % ve == 0 && rot_dim % (2 * ve) == 0 && fits(k, k_ts, k_hs) && fits(v, v_ts, v_hs) &&
                   (heads == 0 || (fits(q, q_ts, q_hs) && fits(q_out, qo_ts, qo_hs))) && aligned_to(k_cache, cache_align) &&
                   aligned_to(v_cache, cache_align) && multiples(ve, {kc_ps, kc_hs, kc_rs, vc_ps, vc_hs, vc_rs});
  RowsArgs r{};
  AppendArgs& a = r.a;
  a.q = q; a.q_ts = q_ts; a.q_hs = q_hs;
  a.k = k; a.k_ts = k_ts; a.k_hs = k_hs;
  a.v = v; a.v_ts = v_ts; a.v_hs = v_hs;
  a.q_out = q_out; a.qo_ts = qo_ts; a.qo_hs = qo_hs;
  a.kc = k_cache; a.kc_ps = kc_ps; a.kc_hs = kc_hs; a.kc_rs = kc_rs;
  a.vc = v_cache; a.vc_ps = vc_ps; a.vc_hs = vc_hs; a.vc_rs = vc_rs;
  a.slots = slots; a.positions = positions; a.cos_sin = cos_sin; a.max_pos = max_pos;
  a.num_slots = num_pages * page_size;
  a.page_size = static_cast<uint32_t>(page_size);
  a.T = static_cast<int>(num_tokens);
  a.H = heads; a.HK = kv_heads; a.D = head_dim; a.R = rot_dim;
  r.qw = heads > 0 ? q_norm : nullptr;
  r.kw = k_norm;
  r.w_bf16 = norm_dtype == GS_DTYPE_BF16;
  r.eps = eps;
  r.inv_d = 1.0f / static_cast<float>(head_dim);
  r.ks = k_scales; r.ks_ps = ks_ps; r.ks_hs = ks_hs;
  r.vs = v_scales; r.vs_ps = vs_ps; r.vs_hs = vs_hs;
  plan_rows(r, vec ? ve : 1, device_cus());
  const dim3 grid(static_cast<unsigned>((num_tokens + a.tokens - 1) / a.tokens));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, r); };
  const auto pick = [&](auto b, auto w) {
    constexpr bool B = decltype(b)::value;
    constexpr int W = decltype(w)::value;
    if (interleaved != 0) quant ? go(append_rows_kernel<B, W, true, true>) : go(append_rows_kernel<B, W, true, false>);
    else quant ? go(append_rows_kernel<B, W, false, true>) : go(append_rows_kernel<B, W, false, false>);
  };
  if (bf16) vec ? pick(std::true_type(), std::integral_constant<int, 8>()) : pick(std::true_type(), std::integral_constant<int, 1>());
  else vec ? pick(std::false_type(), std::integral_constant<int, 4>()) : pick(std::false_type(), std::integral_constant<int, 1>());
  GS_CHECK_LAUNCH(who);
  return GS_OK;
}

int gs_read_kv(int32_t dtype, int32_t cache_dtype, const void* k_cache, int64_t kc_ps, int64_t kc_hs, int64_t kc_rs,
               const void* v_cache, int64_t vc_ps, int64_t vc_hs, int64_t vc_rs, const uint8_t* k_scales, int64_t ks_ps,
               int64_t ks_hs, const uint8_t* v_scales, int64_t vs_ps, int64_t vs_hs, int64_t num_pages,
               int32_t page_size, int32_t kv_heads, int32_t head_dim, const int64_t* slots, int64_t num_tokens,
               void* k_out, int64_t ko_ts, int64_t ko_hs, void* v_out, int64_t vo_ts, int64_t vo_hs, void* stream) {
  const char* who = "gs_read_kv";
  GS_CHECK_ARG(dtype == GS_DTYPE_BF16 || dtype == GS_DTYPE_FP32, "%s: dtype=%d", who, dtype);
  GS_CHECK_ARG(cache_dtype == dtype || cache_dtype == GS_DTYPE_E4M3, "%s: cache_dtype=%d with dtype=%d", who, cache_dtype, dtype);
  GS_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t(1) << 31), "%s: num_tokens=%lld", who, (long long)num_tokens);
  GS_CHECK_ARG(kv_heads > 0 && kv_heads <= 4096 && head_dim > 0 && head_dim <= 512, "%s: kv_heads=%d head_dim=%d (1 .. 512)",
               who, kv_heads, head_dim);
  GS_CHECK_ARG(page_size > 0 && num_pages > 0, "%s: page_size=%d num_pages=%lld", who, page_size, (long long)num_pages);
  if (num_tokens == 0) return GS_OK;
  const bool quant = cache_dtype == GS_DTYPE_E4M3;
  if (num_tokens == 1) ko_ts = vo_ts = 0;
  if (kv_heads == 1) kc_hs = vc_hs = ks_hs = vs_hs = ko_hs = vo_hs = 0;
  if (num_pages == 1) kc_ps = vc_ps = ks_ps = vs_ps = 0;
  if (page_size == 1) kc_rs = vc_rs = 0;
  GS_CHECK_ARG(k_cache != nullptr && v_cache != nullptr && slots != nullptr && k_out != nullptr && v_out != nullptr &&
                   (!quant || (k_scales != nullptr && v_scales != nullptr)), "%s: null tensor", who);
  const bool bf16 = dtype == GS_DTYPE_BF16;
  const int ve = quant ? 16 : bf16 ? 8 : 4;          // 16 bytes of the cache
  const bool vec = head_dim % ve == 0 && aligned16(k_cache) && aligned16(v_cache) && aligned16(k_out) && aligned16(v_out) &&
                   multiples(ve, {kc_ps, kc_hs, kc_rs, vc_ps, vc_hs, vc_rs}) &&
                   multiples(bf16 ? 8 : 4, {ko_ts, ko_hs, vo_ts, vo_hs});
  ReadArgs r{};
  const auto side = [&](int w, const void* c, int64_t ps, int64_t hs, int64_t rs, const uint8_t* s, int64_t s_ps, int64_t s_hs,
                        void* out, int64_t o_ts, int64_t o_hs) {
    r.c[w] = c; r.ps[w] = ps; r.hs[w] = hs; r.rs[w] = rs;
    r.s[w] = s; r.s_ps[w] = s_ps; r.s_hs[w] = s_hs;
    r.out[w] = out; r.o_ts[w] = o_ts; r.o_hs[w] = o_hs;
  };
  side(0, k_cache, kc_ps, kc_hs, kc_rs, k_scales, ks_ps, ks_hs, k_out, ko_ts, ko_hs);
  side(1, v_cache, vc_ps, vc_hs, vc_rs, v_scales, vs_ps, vs_hs, v_out, vo_ts, vo_hs);
  r.slots = slots;
  r.num_slots = num_pages * page_size;
  r.page_size = static_cast<uint32_t>(page_size);
  r.T = static_cast<int>(num_tokens);
  r.HK = kv_heads; r.D = head_dim;
  plan_read(r, vec ? ve : 1);
  const dim3 grid(static_cast<unsigned>((num_tokens + r.tokens - 1) / r.tokens), 2);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, r); };
  if (quant) {
    if (vec) bf16 ? go(read_kv_kernel<Held::kE4m3, true, 16>) : go(read_kv_kernel<Held::kE4m3, false, 16>);
    else bf16 ? go(read_kv_kernel<Held::kE4m3, true, 1>) : go(read_kv_kernel<Held::kE4m3, false, 1>);
  } else if (bf16) {
    vec ? go(read_kv_kernel<Held::kBf16, true, 8>) : go(read_kv_kernel<Held::kBf16, true, 1>);
  } else {
    vec ? go(read_kv_kernel<Held::kFp32, false, 4>) : go(read_kv_kernel<Held::kFp32, false, 1>);
  }
  GS_CHECK_LAUNCH(who);
  return GS_OK;
}

int64_t gs_check_rows_addresses(int32_t dtype, int32_t quant, int32_t vec, int64_t q_ts, int64_t q_hs, int64_t k_ts,
                                int64_t k_hs, int64_t num_tokens, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                const int64_t* positions, int64_t max_pos, int32_t rot_dim, int32_t interleaved,
                                const int64_t* slots, int64_t c_ps, int64_t c_hs, int64_t c_rs, int64_t s_ps,
                                int64_t s_hs, int64_t num_pages, int32_t page_size, int32_t cus, char* msg,
                                int64_t msg_len, int64_t* checked) {
  const char* who = "gs_check_rows_addresses";
  const bool bf16 = dtype == GS_DTYPE_BF16;
  const int ve = vec ? (bf16 ? 8 : 4) : 1;
  GS_CHECK_ARG((bf16 || dtype == GS_DTYPE_FP32) && num_tokens > 0 && num_tokens < (int64_t(1) << 31) && heads >= 0 &&
                   kv_heads > 0 && head_dim > 0 && head_dim <= 512 && rot_dim >= 0 && rot_dim <= head_dim &&
                   rot_dim % 2 == 0 && head_dim % ve == 0 && rot_dim % (2 * ve) == 0 && page_size > 0 && num_pages > 0 &&
                   slots != nullptr && (rot_dim == 0 || (positions != nullptr && max_pos > 0)) && cus > 0, "%s: sizes", who);
  RowsArgs r{};
  AppendArgs& a = r.a;
  a.q_ts = a.qo_ts = q_ts; a.q_hs = a.qo_hs = q_hs;
  a.k_ts = a.v_ts = k_ts; a.k_hs = a.v_hs = k_hs;
  a.kc_ps = a.vc_ps = c_ps; a.kc_hs = a.vc_hs = c_hs; a.kc_rs = a.vc_rs = c_rs;
  r.ks_ps = r.vs_ps = s_ps; r.ks_hs = r.vs_hs = s_hs;
  a.max_pos = max_pos;
  a.num_slots = num_pages * page_size;
  a.page_size = static_cast<uint32_t>(page_size);
  a.T = static_cast<int>(num_tokens);
  a.H = heads; a.HK = kv_heads; a.D = head_dim; a.R = rot_dim;
  plan_rows(r, ve, cus);
  PagedModel m;
  const bool pr = interleaved != 0;
  if (ve == 8) pr ? model_rows_append<8, true>(m, r, quant != 0, slots, positions) : model_rows_append<8, false>(m, r, quant != 0, slots, positions);
  else if (ve == 4) pr ? model_rows_append<4, true>(m, r, quant != 0, slots, positions) : model_rows_append<4, false>(m, r, quant != 0, slots, positions);
  else pr ? model_rows_append<1, true>(m, r, quant != 0, slots, positions) : model_rows_append<1, false>(m, r, quant != 0, slots, positions);
  // the rows read back, packed
  const int re = vec ? (quant ? 16 : ve) : 1;
  if (head_dim % re == 0 && !m.bad) {
    ReadArgs x{};
    x.ps[0] = c_ps; x.hs[0] = c_hs; x.rs[0] = c_rs;
    x.s_ps[0] = s_ps; x.s_hs[0] = s_hs;
    x.o_ts[0] = static_cast<int64_t>(kv_heads) * head_dim; x.o_hs[0] = head_dim;
    x.num_slots = a.num_slots;
    x.page_size = a.page_size;
    x.T = a.T; x.HK = kv_heads; x.D = head_dim;
    plan_read(x, re);
    model_read(m, x, re, slots);
  }
  if (checked) *checked = m.checked;
  if (msg && msg_len > 0) snprintf(msg, static_cast<size_t>(msg_len), "%s", m.msg);
  return m.bad;
}

}  // extern "C"
