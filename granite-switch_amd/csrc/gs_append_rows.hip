// Rows into and out of a quantised paged cache, and the norms of queries and keys for
// each head in the pass that rotates and stores them.
//
// A row (a head's key or value of one token) is kept as e4m3 values y and one power of
// two 2^e, x = y 2^e, with e the least integer that keeps the row's largest finite
// magnitude within 448 2^e (e >= -126): the product with 2^-e is exact, so a value is
// rounded once, by at most 2^-4 of itself down to 2^-6 2^e, and any factor between two
// powers of two would leave it the same relative error.  e + 127 is the scale's byte.  A
// finite value stays finite (kMostHeld).
//
// gs_append_kv_normed: x rsqrt(mean(x^2) + eps) w over a head's columns, rotation, and for
// keys and values the row's exponent and its e4m3 values.  A head's columns are held by 2^n
// adjacent lanes (8 for 128 bf16 columns, 16 each), which add squares and find the maximum by
// lane permutes; nothing is read twice.  8192 tokens of 32 + 8 + 8 heads of 128, bf16, with
// norms, quantised: 38.3 us, 4.9 TB/s, where a bare copy reaches 6.2 and vector instructions
// take 72% of the SIMDs' cycles; 4144 tokens into a bf16 cache 19.5 us, 5.3 TB/s; 256 tokens
// 5.1 us, of which the launch and a chain of loads are most.
//
// gs_read_kv: rows by their slots, y 2^e.  One read and one write, the memory rate bounds it:
// 131071 tokens of 8 heads of 128 to bf16 139.5 us, 5.8 TB/s.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "gs_append.h"

namespace gs {
namespace {

struct RowsArgs {
  AppendArgs a;                                      // without units, groups and tokens
  const void* qw;                                    // norm weights [D] or NULL
  const void* kw;
  bool w_bf16;
  float eps;
  uint8_t* ks;                                       // scales; a head's of a page side by side
  uint8_t* vs;
  int64_t ks_ps, ks_hs, vs_ps, vs_hs;
  uint32_t page_magic;                               // div_magic(page_size) where slots fit 31 bits, or 0
  int units, lanes_log;                              // column units and lanes of a head
  int groups[3], tokens[3], blocks[3];               // queries, keys, values: heads at a time and tokens of a workgroup, workgroups
  uint32_t k_share, v_share;                         // keys' share of the workgroups, values' of the others
};
enum Kind { kQueries, kKeys, kValues };
// Workgroup b's kind, and which of that kind's it is: spread evenly, so that those that
// compute more (keys) run beside those that move more.
__device__ __host__ __forceinline__ Kind rows_kind(const RowsArgs& r, int b, int& block) {
  block = addr::spread_before(b, r.k_share, r.blocks[kKeys]);
  if (addr::spread_is(b, r.k_share, r.blocks[kKeys])) return kKeys;
  b -= block;
  block = addr::spread_before(b, r.v_share, r.blocks[kValues]);
  if (addr::spread_is(b, r.v_share, r.blocks[kValues])) return kValues;
  block = b - block;
  return kQueries;
}

// Sums, and maxima, over the 2^n adjacent lanes of a head.  Eight lanes, which are 65 .. 128
// bf16 columns or 33 .. 64 fp32 ones, have a branch of their own: 256 rows 5.1 us in a graph,
// 5.3 without; 4144 rows into a bf16 cache 20.4 and 20.8; 8192 rows no difference.
template <int CTRL>
__device__ __forceinline__ float dpp_other(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ double dpp_other(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, 0xf, 0xf, false);
  const uint32_t up = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, lo | (static_cast<uint64_t>(up) << 32));
}
template <class T, class F>
__device__ __forceinline__ T over_lanes(T x, int lanes, const F& f) {
  if (lanes == 8) {                                  // 128 bf16 columns, 64 fp32 ones
    x = f(x, dpp_other<0xB1>(x));
    x = f(x, dpp_other<0x4E>(x));
    return f(x, dpp_other<0x141>(x));
  }
  if (lanes > 1) x = f(x, dpp_other<0xB1>(x));       // lanes 1, 2 apart
  if (lanes > 2) x = f(x, dpp_other<0x4E>(x));
  if (lanes > 4) x = f(x, dpp_other<0x141>(x));      // mirrored in 8, in 16: the other four, the other eight
  if (lanes > 8) x = f(x, dpp_other<0x140>(x));
  if (lanes > 16) x = f(x, __shfl_xor(x, 16, 64));
  if (lanes > 32) x = f(x, __shfl_xor(x, 32, 64));
  return x;
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.402823466e+38f; }

// The largest magnitude that a row holds: 240 2^120 = 1.875 2^127.  The next e4m3 value times
// that power of two is 2^128, which neither type has; a larger x is kept as this one, off by
// less than 2^-4 of itself.
constexpr float kMostHeld = 0x1.ep127f;
__device__ __forceinline__ float held_finite(float x) {
  return !is_finite(x) ? __uint_as_float(0x7fc00000u) : fabsf(x) > kMostHeld ? copysignf(kMostHeld, x) : x;
}

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

// VE values as e4m3 in the low bytes.
template <int VE>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float* x, float inv) {
  float y[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) y[i] = x[i] * inv;
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

// 1 / sqrt(x) from the instruction's 24 bits, twice refined; 0 for an infinity, whose product
// with its 0 is kept out of the refinement.
__device__ __forceinline__ double rsqrt64(double x) {
  double y = __builtin_amdgcn_rsq(x);
  const double h = 0.5 * fmin(x, 1.7976931348623157e308);
#pragma unroll
  for (int i = 0; i < 2; ++i) y *= 1.5 - h * y * y;
  return y;
}
// x in fp32, to the odd neighbour where it is none: another rounding, to fewer bits, is then
// that of x itself.
__device__ __forceinline__ float round_odd(double x) {
  const float f = static_cast<float>(x);
  const double back = static_cast<double>(f);
  const uint32_t b = __float_as_uint(f);
  const bool move = back != x && (b & 1u) == 0 && is_finite(f);
  return __uint_as_float(move ? (fabs(x) > fabs(back) ? b + 1 : b - 1) : b);
}

// VE elements as they are in memory.
template <bool BF16, int VE>
struct RowVec {
  u32x4 w;
  __device__ __forceinline__ void load(const char* p) { w = ld16(p); }
  __device__ __forceinline__ void none() { w = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (BF16) return __uint_as_float((i & 1) != 0 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    else return __uint_as_float(w[i]);
  }
};
template <bool BF16>
struct RowVec<BF16, 1> {
  float w;
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (BF16) w = bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(p));
    else w = *reinterpret_cast<const float*>(p);
  }
  __device__ __forceinline__ void none() { w = 0.f; }
  __device__ __forceinline__ float at(int) const { return w; }
};

// The rows of one kind for a workgroup's tokens.  A thread takes a unit of columns as
// append_kv_kernel (gs_append.hip) does -- two vectors of VE, partners of a rotation -- of
// every groups-th head of its token; a head's units are on 2^n adjacent lanes, one to a
// lane, or up to NU (element by element: a wave to a head).  Loads of kBatch heads are in
// flight, one head's columns are unpacked.  The walk is not shared with that kernel, which needs
// no lanes in powers of two and loads partners together: with the rotation alone in common it
// got other registers, and its 8192 rows 47.3 us instead of 43.5.
//
// Keys that are normed or rotated on their way into a quantised cache take that in 64 bits:
// in 32, one in 10^6 of them ends at the other e4m3 neighbour, 2^-3 away.  A thread has one
// head of these at a time, or its 64-bit numbers leave too few registers for waves that hide
// the loads.
template <bool BF16, int VE, bool PAIRS, bool QUANT, int KIND>
__device__ __forceinline__ void append_rows(const RowsArgs& r, int block) {
  constexpr int NU = VE == 1 ? 4 : 1;
  constexpr int kES = BF16 ? 2 : 4;
  constexpr bool kE4m3 = QUANT && KIND != kQueries;
  constexpr int kBatch = VE == 1 || (kE4m3 && KIND == kKeys) ? 1 : 4;
  const AppendArgs& a = r.a;
  const int groups = r.groups[KIND], tokens = r.tokens[KIND], heads = KIND == kQueries ? a.H : a.HK;
  const int tid = threadIdx.x, lanes = 1 << r.lanes_log;
  const int g = tid >> r.lanes_log, u0 = tid & (lanes - 1);
  const int tok = g / groups, grp = g - tok * groups;
  const int64_t t = static_cast<int64_t>(block) * tokens + tok;
  if (tok >= tokens || t >= a.T) return;
  uint32_t page = 0, prow = 0;
  if (KIND != kQueries) {
    const int64_t slot = a.slots[t];
    if (!addr::append_stored(slot, a.num_slots)) return;
    if (r.page_magic != 0) {
      addr::div_by(static_cast<uint32_t>(slot), a.page_size, r.page_magic, page, prow);
    } else {
      page = static_cast<uint32_t>(static_cast<uint64_t>(slot) / a.page_size);
      prow = static_cast<uint32_t>(slot - static_cast<int64_t>(page) * a.page_size);
    }
  }
  const void* norm = KIND == kQueries ? r.qw : KIND == kKeys ? r.kw : nullptr;
  addr::AppendCols c[NU];
  float cs[NU][VE], sn[NU][VE], w[NU][2][VE];
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const int u = u0 + n * lanes;
    c[n] = u < r.units ? addr::append_cols(u, VE, a.D, a.R, PAIRS) : addr::AppendCols{-1, -1, false};
    if (KIND == kValues) continue;
    if (c[n].rot) {
      const float* row = a.cos_sin + addr::append_pos(a.positions[t], a.max_pos) * a.R;
      const int j0 = addr::append_pair(u, VE);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        cs[n][i] = row[j0 + i];
        sn[n][i] = row[a.R / 2 + j0 + i];
      }
    }
    if (norm != nullptr) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = max(x == 0 ? c[n].c0 : c[n].c1, 0);
        if (BF16 && r.w_bf16) {
          RowVec<true, VE> v;
          v.load(static_cast<const char*>(norm) + col * 2);
#pragma unroll
          for (int i = 0; i < VE; ++i) w[n][x][i] = v.at(i);
        } else {
#pragma unroll
          for (int i = 0; i < VE; i += 4) {
            RowVec<false, VE == 1 ? 1 : 4> v;
            v.load(static_cast<const char*>(norm) + (col + i) * 4);
#pragma unroll
            for (int e = 0; e < (VE == 1 ? 1 : 4); ++e) w[n][x][i + e] = v.at(e);
          }
        }
      }
    }
  }
  const char* src = static_cast<const char*>(KIND == kQueries ? a.q : KIND == kKeys ? a.k : a.v) +
                    t * (KIND == kQueries ? a.q_ts : KIND == kKeys ? a.k_ts : a.v_ts) * kES;
  const int64_t src_hs = (KIND == kQueries ? a.q_hs : KIND == kKeys ? a.k_hs : a.v_hs) * kES;
  constexpr int kDS = kE4m3 ? 1 : kES;
  char* dst = static_cast<char*>(KIND == kQueries ? a.q_out : KIND == kKeys ? a.kc : a.vc) +
              (KIND == kQueries ? t * a.qo_ts : KIND == kKeys ? page * a.kc_ps + prow * a.kc_rs : page * a.vc_ps + prow * a.vc_rs) * kDS;
  const int64_t dst_hs = (KIND == kQueries ? a.qo_hs : KIND == kKeys ? a.kc_hs : a.vc_hs) * kDS;
  const auto lane_sum = [&](auto x) { return over_lanes(x, lanes, [](auto p, auto q) { return p + q; }); };
  const int64_t src_step = groups * src_hs, dst_step = groups * dst_hs;
  src += grp * src_hs;
  dst += grp * dst_hs;
  for (int h0 = grp; h0 < heads; h0 += kBatch * groups, src += kBatch * src_step, dst += kBatch * dst_step) {
    RowVec<BF16, VE> x0[kBatch][NU], x1[kBatch][NU];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * groups;
      if (h >= heads) continue;
      const char* p = src + b * src_step;
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        if (c[n].c0 >= 0) x0[b][n].load(p + c[n].c0 * kES);
        else x0[b][n].none();
        if (c[n].c1 >= 0) x1[b][n].load(p + c[n].c1 * kES);
        else x1[b][n].none();
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * groups;
      if (h >= heads) continue;
      float f0[NU][VE], f1[NU][VE];
      if (kE4m3 && KIND == kKeys && (norm != nullptr || a.R > 0)) {
        double f = 1;
        if (norm != nullptr) {
          double ss = 0;
#pragma unroll
          for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
              const double p = x0[b][n].at(i), q = x1[b][n].at(i);
              ss = fma(p, p, fma(q, q, ss));
            }
          f = rsqrt64(lane_sum(ss) / a.D + r.eps);
        }
        // a pair of partners at a time, and what does not depend on the head not kept in 64 bits
        const auto pair = [&](float p32, float q32, float wp, float wq, float c32, float s32, bool rot, float& to_p, float& to_q) {
          asm("" : "+v"(wp), "+v"(wq), "+v"(c32), "+v"(s32));
          double p = p32, q = q32;
          if (norm != nullptr) {
            p *= f * wp;
            q *= f * wq;
          }
          if (rot) {
            const double cd = c32, sd = s32, p0 = p, q0 = q;
            p = p0 * cd - q0 * sd;
            q = q0 * cd + p0 * sd;
          }
          to_p = round_odd(p);
          to_q = round_odd(q);
        };
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          if constexpr (!PAIRS || VE == 1) {
#pragma unroll
            for (int i = 0; i < VE; ++i)
              pair(x0[b][n].at(i), x1[b][n].at(i), w[n][0][i], w[n][1][i], cs[n][i], sn[n][i], c[n].rot, f0[n][i], f1[n][i]);
          } else {
#pragma unroll
            for (int i = 0; i < VE / 2; ++i) {
              const int u = 2 * i, v = 2 * i + 1, k = VE / 2 + i;
              pair(x0[b][n].at(u), x0[b][n].at(v), w[n][0][u], w[n][0][v], cs[n][i], sn[n][i], c[n].rot, f0[n][u], f0[n][v]);
              pair(x1[b][n].at(u), x1[b][n].at(v), w[n][1][u], w[n][1][v], cs[n][k], sn[n][k], c[n].rot, f1[n][u], f1[n][v]);
            }
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            f0[n][i] = x0[b][n].at(i);
            f1[n][i] = x1[b][n].at(i);
          }
        if (KIND != kValues && norm != nullptr) {
          float ss = 0.f;
#pragma unroll
          for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int i = 0; i < VE; ++i) ss += f0[n][i] * f0[n][i] + f1[n][i] * f1[n][i];
          const float f = rsqrtf(lane_sum(ss) * (1.f / a.D) + r.eps);
#pragma unroll
          for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
              f0[n][i] *= f * w[n][0][i];
              f1[n][i] *= f * w[n][1][i];
            }
        }
        if (KIND != kValues) {
#pragma unroll
          for (int n = 0; n < NU; ++n)
            if (c[n].rot) rotate<VE, PAIRS>(f0[n], f1[n], cs[n], sn[n]);
        }
      }
      char* p = dst + b * dst_step;
      if constexpr (kE4m3) {
        const auto largest = [&] {                   // NaN is never the larger one
          float m = 0.f;
#pragma unroll
          for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int i = 0; i < VE; ++i) m = fmaxf(fmaxf(m, fabsf(f0[n][i])), fabsf(f1[n][i]));
          return over_lanes(m, lanes, [](float x, float y) { return fmaxf(x, y); });
        };
        float m = largest();
        if (!(m <= kMostHeld)) {                     // infinities become NaN, which e4m3 has
#pragma unroll
          for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
              f0[n][i] = held_finite(f0[n][i]);
              f1[n][i] = held_finite(f1[n][i]);
            }
          m = largest();
        }
        const int code = addr::e8m0_of(__float_as_uint(m));
        const float inv = __uint_as_float(static_cast<uint32_t>(254 - code) << 23);
        if (u0 == 0) {
          uint8_t* s = KIND == kKeys ? r.ks + page * r.ks_ps + h * r.ks_hs : r.vs + page * r.vs_ps + h * r.vs_hs;
          s[prow] = static_cast<uint8_t>(code);
        }
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          if (c[n].c0 >= 0) store_e4m3<VE>(reinterpret_cast<uint8_t*>(p) + c[n].c0, f0[n], inv);
          if (c[n].c1 >= 0) store_e4m3<VE>(reinterpret_cast<uint8_t*>(p) + c[n].c1, f1[n], inv);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          if (c[n].c0 >= 0) append_store<BF16, VE>(p, c[n].c0, f0[n]);
          if (c[n].c1 >= 0) append_store<BF16, VE>(p, c[n].c1, f1[n]);
        }
      }
    }
  }
}

// The kernel's only argument, to be loaded where it is used: the three kinds' fields together
// would keep the scalar registers full throughout.
__device__ __forceinline__ const RowsArgs& fresh_rows() {
  typedef const __attribute__((address_space(4))) RowsArgs* Ptr;
  Ptr p = (Ptr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const RowsArgs*)(p);
}

template <bool BF16, int VE, bool PAIRS, bool QUANT>
__global__ __launch_bounds__(256, 4) void append_rows_kernel(RowsArgs) {
  int block;
  const Kind kind = rows_kind(fresh_rows(), blockIdx.x, block);
  if (kind == kKeys) append_rows<BF16, VE, PAIRS, QUANT, kKeys>(fresh_rows(), block);
  else if (kind == kValues) append_rows<BF16, VE, PAIRS, QUANT, kValues>(fresh_rows(), block);
  else append_rows<BF16, VE, PAIRS, QUANT, kQueries>(fresh_rows(), block);
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
    else st16_nt(o, sel16(live, ld16(p)));
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
      st16_nt(o, y[0]);
      st16_nt(o + 8, y[1]);
    } else {
      float* o = static_cast<float*>(r.out[w]) + to;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x[i], scale, false);
        const f32x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x[i], scale, true);
        st16_nt(o + 4 * i, __builtin_bit_cast(u32x4, f32x4{lo[0], lo[1], hi[0], hi[1]}));
      }
    }
  }
}

// A workgroup takes `tokens` tokens of the keys (blockIdx.y 0) or the values; a thread a
// piece of VE columns, every 256-th of the workgroup's.  One piece a thread where a token has
// no more: 131071 rows of 8 heads of 128 149 us, 158 with two and 168 with four, and 140 with
// streaming stores.
template <Held HELD, bool BF16, int VE>
__global__ __launch_bounds__(256) void read_kv_kernel(ReadArgs r) {
  const int w = blockIdx.y;
  const int row = r.HK * r.pieces;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * r.tokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(r.tokens), r.T - t0)) * row;
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
constexpr int64_t kMostBlocks = int64_t(1) << 24;    // of 256 threads: a launch has less than 2^32

// Few tokens: every head of a token at once; many: each thread four heads, its cosines,
// sines and weights loaded once for them.
// False: more workgroups than a launch has.
bool plan_rows(RowsArgs& r, int ve, bool quant, int cus) {
  const AppendArgs& a = r.a;
  r.units = addr::append_units(ve, a.D, a.R);
  r.lanes_log = 0;
  while ((1 << r.lanes_log) < r.units && r.lanes_log < 6) ++r.lanes_log;
  const int most = 256 >> r.lanes_log;
  int64_t all = 0;
  for (int kind = 0; kind < 3; ++kind) {
    const int n = kind == kQueries ? a.H : a.HK;
    r.groups[kind] = std::max(1, std::min(a.T <= 2 * cus || (quant && kind == kKeys) ? n : (n + 3) / 4, most));
    r.tokens[kind] = most / r.groups[kind];
    r.blocks[kind] = n == 0 ? 0 : static_cast<int>((static_cast<int64_t>(a.T) + r.tokens[kind] - 1) / r.tokens[kind]);
    all += r.blocks[kind];
  }
  if (all >= kMostBlocks) return false;
  r.k_share = addr::spread_share(r.blocks[kKeys], r.blocks[kQueries] + r.blocks[kKeys] + r.blocks[kValues]);
  r.v_share = addr::spread_share(r.blocks[kValues], r.blocks[kQueries] + r.blocks[kValues]);
  r.page_magic = a.num_slots < (int64_t(1) << 31) ? addr::div_magic(a.page_size) : 0;
  return true;
}

void plan_read(ReadArgs& r, int ve) {
  r.pieces = r.D / ve;
  const int row = r.HK * r.pieces;
  r.tokens = std::max(1, 256 / row);
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
  if (r.units > NU << r.lanes_log) m.fail("units of a head", 0, r.units, NU << r.lanes_log);
  std::vector<int> taken[3];
  for (int kind = 0; kind < 3; ++kind) taken[kind].assign(r.blocks[kind], 0);
  for (int b = 0; b < r.blocks[0] + r.blocks[1] + r.blocks[2]; ++b) {
    int block;
    const Kind kind = rows_kind(r, b, block);
    m.in("workgroup", block, 1, r.blocks[kind]);
    if (m.bad) return;
    if (++taken[kind][block] != 1) m.fail("a workgroup's rows taken twice", block, 1, r.blocks[kind]);
  }
  for (int kind = 0; kind < 3; ++kind) {
    const int groups = r.groups[kind], tokens = r.tokens[kind], heads = kind == kQueries ? a.H : a.HK, lanes = 1 << r.lanes_log;
    if (groups * tokens * lanes > 256 || tokens < 1) m.fail("threads of a workgroup", 0, groups * tokens * lanes, 256);
    std::vector<int> seen(static_cast<size_t>(a.T) * heads * a.D, 0), scales(static_cast<size_t>(a.T) * heads, 0);
    for (int64_t block = 0; block < r.blocks[kind] && !m.bad; ++block)
      for (int tid = 0; tid < 256 && !m.bad; ++tid) {
        const int g = tid >> r.lanes_log, u0 = tid & (lanes - 1), tok = g / groups, grp = g - tok * groups;
        const int64_t t = block * tokens + tok;
        if (tok >= tokens || t >= a.T) continue;
        const bool stored = addr::append_stored(slots[t], a.num_slots);
        uint32_t page = 0, prow = 0;
        if (stored) {
          page = static_cast<uint32_t>(slots[t] / a.page_size);
          prow = static_cast<uint32_t>(slots[t] - static_cast<int64_t>(page) * a.page_size);
          uint32_t p2 = page, r2 = prow;
          if (r.page_magic != 0) addr::div_by(static_cast<uint32_t>(slots[t]), a.page_size, r.page_magic, p2, r2);
          if (p2 != page || r2 != prow) m.fail("division", slots[t], 0, a.page_size);
        }
        for (int n = 0; n < NU; ++n) {
          const int u = u0 + n * lanes;
          if (u >= r.units) continue;
          const addr::AppendCols c = addr::append_cols(u, VE, a.D, a.R, PAIRS);
          if (c.rot && kind != kValues) {
            const int64_t row = addr::append_pos(positions[t], a.max_pos) * a.R;
            m.in("cosines", row + addr::append_pair(u, VE), VE, row + a.R / 2);
            m.in("cos_sin", row + a.R / 2 + addr::append_pair(u, VE), VE, a.max_pos * a.R);
          }
          for (int h = grp; h < heads; h += groups) {
            if (u0 == 0 && n == 0 && kind != kQueries) {
              ++scales[t * heads + h];
              if (quant && stored) m.in("scales", page * r.ks_ps + h * r.ks_hs + prow, 1, s_elems);
            }
            for (int col : {c.c0, c.c1}) {
              if (col < 0) continue;
              m.in("norm weights", col, VE, a.D);
              for (int i = 0; i < VE && col + i < a.D; ++i) ++seen[(t * heads + h) * a.D + col + i];
              if (kind == kQueries) {
                m.in("q", t * a.q_ts + h * a.q_hs + col, VE, q_elems);
                m.in("q_out", t * a.qo_ts + h * a.qo_hs + col, VE, qo_elems);
              } else {
                m.in("k or v", t * a.k_ts + h * a.k_hs + col, VE, k_elems);
                if (stored) m.in("cache", page * a.kc_ps + h * a.kc_hs + prow * a.kc_rs + col, VE, c_elems);
              }
            }
          }
        }
      }
    for (int x : scales)
      if (x != 1 && kind != kQueries && !m.bad) m.fail("a scale written other than once", 0, x, 1);
    for (int x : seen)
      if (x != 1 && !m.bad) m.fail("a column taken other than once", 0, x, 1);
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
  GS_CHECK_ARG(page_size > 0 && num_pages > 0 && num_pages < (int64_t(1) << 31), "%s: page_size=%d num_pages=%lld", who, page_size,
               (long long)num_pages);
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
  const bool vec = head_dim % ve == 0 && aligned16(q_norm) && aligned16(k_norm) && rot_dim % (2 * ve) == 0 && fits(k, k_ts, k_hs) && fits(v, v_ts, v_hs) &&
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
  r.ks = k_scales; r.ks_ps = ks_ps; r.ks_hs = ks_hs;
  r.vs = v_scales; r.vs_ps = vs_ps; r.vs_hs = vs_hs;
  GS_CHECK_ARG(plan_rows(r, vec ? ve : 1, quant, device_cus()), "%s: num_tokens=%lld with %d + %d heads of %d are too many", who,
               (long long)num_tokens, heads, kv_heads, head_dim);
  const dim3 grid(static_cast<unsigned>(r.blocks[0] + r.blocks[1] + r.blocks[2]));
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
  GS_CHECK_ARG(page_size > 0 && num_pages > 0 && num_pages < (int64_t(1) << 31), "%s: page_size=%d num_pages=%lld", who, page_size,
               (long long)num_pages);
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
  const int64_t blocks = (num_tokens + r.tokens - 1) / r.tokens;
  GS_CHECK_ARG(blocks < kMostBlocks, "%s: num_tokens=%lld with %d heads of %d are too many", who, (long long)num_tokens, kv_heads, head_dim);
  const dim3 grid(static_cast<unsigned>(blocks), 2);
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
  GS_CHECK_ARG(plan_rows(r, ve, quant != 0, cus), "%s: too many rows", who);
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
