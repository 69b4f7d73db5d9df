// Paged key/value cache: rotated append, and attention over it.
//
// A cache is [pages, kv heads, page rows, head dim] with any page, head and row
// stride (a head's rows of a page side by side, or a token's heads), so token t
// of a sequence is row t % page of page table[t / page].  Pages hold a multiple
// of 8 rows: the 8 tokens from a multiple of 8 on share a page, which is the
// granule every address below is computed for.
//
// gs_append_kv (append_kv_kernel): the QKV projection's rows in, the rotated
// query rows out, the rotated keys and the values into their slots.
//
// gs_paged_attention: per query row one pass over the keys it sees with the
// running maximum and total of its softmax.  The row form here
// (paged_attention_kernel, paged_join_kernel) takes 16 rows at a time, straight
// from the pages into registers, a sequence's length split over workgroups and
// joined: one new token of a sequence.  Sequences of many rows take the chunk
// form (gs_chunk.hip).
#include <algorithm>
#include <vector>

#include "gs_paged.h"

namespace gs {
namespace {

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;      // token and head strides, elements
  void* q_out;
  int64_t qo_ts, qo_hs;
  void* kc;
  void* vc;
  int64_t kc_ps, kc_hs, kc_rs, vc_ps, vc_hs, vc_rs;   // page, head and row strides
  const int64_t* slots;
  const int64_t* positions;
  const float* cos_sin;                             // [max_pos, R]: R/2 cosines, R/2 sines
  int64_t max_pos;
  int64_t num_slots;
  uint32_t page_size;
  int T, H, HK, D, R;
  int units, groups, tokens;                        // column units of a head, head groups, tokens of a workgroup
};

template <bool BF16, int VE>
__device__ __forceinline__ void append_load(const void* p, int64_t e, float* f) {
  if constexpr (VE == 1) {
    if constexpr (BF16) f[0] = bf16_bits_to_f32(static_cast<const uint16_t*>(p)[e]);
    else f[0] = static_cast<const float*>(p)[e];
  } else if constexpr (BF16) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const f32x4 w = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = w[i];
  }
}
template <bool BF16, int VE>
__device__ __forceinline__ void append_store(void* p, int64_t e, const float* f) {
  if constexpr (VE == 1) {
    if constexpr (BF16) static_cast<uint16_t*>(p)[e] = f32_to_bf16_bits(f[0]);
    else static_cast<float*>(p)[e] = f[0];
  } else if constexpr (BF16) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = static_cast<uint32_t>(f32_to_bf16_bits(f[2 * i])) | (static_cast<uint32_t>(f32_to_bf16_bits(f[2 * i + 1])) << 16);
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + e) = w;
  } else {
    *reinterpret_cast<f32x4*>(static_cast<float*>(p) + e) = f32x4{f[0], f[1], f[2], f[3]};
  }
}

// A thread takes one unit of columns -- two vectors of VE elements, the partners
// of a rotation among them -- of every groups-th head of its token, so its
// cosines and sines are loaded once for all of them.  Half-split pairs: columns
// [VE u, +VE) and the same R/2 further; side-by-side pairs: 2 VE columns from
// 2 VE u on.  Columns from R on are copied, 2 VE at a time.
template <bool BF16, int VE, bool PAIRS>
__global__ __launch_bounds__(256) void append_kv_kernel(AppendArgs a) {
  const int tid = threadIdx.x;
  const int per_token = a.units * a.groups;
  const int tok = tid / per_token;
  if (tok >= a.tokens) return;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * a.tokens + tok;
  if (t >= a.T) return;
  const int in_tok = tid - tok * per_token;
  const int grp = in_tok / a.units, u = in_tok - grp * a.units;
  const addr::AppendCols c = addr::append_cols(u, VE, a.D, a.R, PAIRS);
  const int64_t slot = a.slots[t];
  float cs[VE], sn[VE];                              // PAIRS: VE pairs; half: VE columns' partners
  if (c.rot) {
    const int64_t pos = a.positions[t];
    const float* row = a.cos_sin + addr::append_pos(pos, a.max_pos) * a.R;
    const int j0 = addr::append_pair(u, VE);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      cs[i] = row[j0 + i];
      sn[i] = row[a.R / 2 + j0 + i];
    }
  }
  const bool stored = addr::append_stored(slot, a.num_slots);
  const uint32_t page = stored ? static_cast<uint32_t>(static_cast<uint64_t>(slot) / a.page_size) : 0u;
  const uint32_t prow = stored ? static_cast<uint32_t>(slot - static_cast<int64_t>(page) * a.page_size) : 0u;
  const int heads = a.H + 2 * a.HK;
  constexpr int kBatch = 4;                          // heads whose loads are in flight together
  for (int h0 = grp; h0 < heads; h0 += kBatch * a.groups) {
    float x0[kBatch][VE], x1[kBatch][VE];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * a.groups;
      if (h < heads) {
        const bool isq = h < a.H, isk = !isq && h < a.H + a.HK;
        const void* src = isq ? a.q : isk ? a.k : a.v;
        const int64_t base = isq ? t * a.q_ts + h * a.q_hs
                           : isk ? t * a.k_ts + (h - a.H) * a.k_hs : t * a.v_ts + (h - a.H - a.HK) * a.v_hs;
        append_load<BF16, VE>(src, base + c.c0, x0[b]);
        if (c.c1 >= 0) append_load<BF16, VE>(src, base + c.c1, x1[b]);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * a.groups;
      if (h >= heads) continue;
      const bool isq = h < a.H, isk = !isq && h < a.H + a.HK;
      if (!isq && !stored) continue;
      if (c.rot && (isq || isk)) {
        if constexpr (!PAIRS) {
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const float p = x0[b][i], s = x1[b][i];
            x0[b][i] = p * cs[i] - s * sn[i];
            x1[b][i] = s * cs[i] + p * sn[i];
          }
        } else if constexpr (VE == 1) {
          const float p = x0[b][0], s = x1[b][0];
          x0[b][0] = p * cs[0] - s * sn[0];
          x1[b][0] = s * cs[0] + p * sn[0];
        } else {
#pragma unroll
          for (int i = 0; i < VE / 2; ++i) {
            const float p = x0[b][2 * i], s = x0[b][2 * i + 1];
            x0[b][2 * i] = p * cs[i] - s * sn[i];
            x0[b][2 * i + 1] = s * cs[i] + p * sn[i];
            const float p1 = x1[b][2 * i], s1 = x1[b][2 * i + 1];
            x1[b][2 * i] = p1 * cs[VE / 2 + i] - s1 * sn[VE / 2 + i];
            x1[b][2 * i + 1] = s1 * cs[VE / 2 + i] + p1 * sn[VE / 2 + i];
          }
        }
      }
      void* dst = isq ? a.q_out : isk ? a.kc : a.vc;
      const int64_t base = isq ? t * a.qo_ts + h * a.qo_hs
                         : isk ? page * a.kc_ps + (h - a.H) * a.kc_hs + prow * a.kc_rs
                               : page * a.vc_ps + (h - a.H - a.HK) * a.vc_hs + prow * a.vc_rs;
      append_store<BF16, VE>(dst, base + c.c0, x0[b]);
      if (c.c1 >= 0) append_store<BF16, VE>(dst, base + c.c1, x1[b]);
    }
  }
}

// ---------------------------------------------------------------------------
// Slots and positions of a batch's tokens
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void cache_slots_kernel(const int32_t* table, int64_t ld_table, int max_pages,
                                                          int num_pages, int page_size, const int32_t* lens,
                                                          const int32_t* cu, int B, int T, int64_t* slots,
                                                          int64_t* positions) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  int s = t;
  bool in = t < B;
  int first = t, last = t + 1;
  if (cu != nullptr) {
    int lo = 0, hi = B - 1;                          // largest s with cu[s] <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cu[mid] <= t) lo = mid; else hi = mid - 1;
    }
    s = lo;
    in = B > 0 && cu[s] <= t && t < cu[s + 1];
    if (in) {
      first = cu[s];
      last = cu[s + 1];
    }
  }
  int64_t pos = in ? static_cast<int64_t>(lens[s]) - (last - first) + (t - first) : -1;
  int64_t slot = -1;
  if (pos >= 0 && pos < static_cast<int64_t>(max_pages) * page_size) {
    const int id = table[s * ld_table + pos / page_size];
    if (id >= 0 && id < num_pages) slot = static_cast<int64_t>(id) * page_size + pos % page_size;
  }
  slots[t] = slot;
  positions[t] = pos >= 0 ? pos : 0;
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
// What the two element types differ in.  Both use 16 x 16 products: S^T = K Q^T
// with the keys as rows, so a lane has one query row's scores of consecutive
// keys, which is the operand that O^T = V^T P^T takes them as.
template <bool BF16, int DT>
struct PagedForm;
template <int DT>
struct PagedForm<true, DT> {
  static constexpr int kBlock = 32;                 // keys of a wave's block
  static constexpr int kSteps = DT / 32;            // K pieces of 16 bytes per key row and lane
  static constexpr int kKT = 2;                     // 16-key tiles of S^T in a block
  static constexpr int kVW = DT >= 128 ? 8 : 4;     // columns of a V vector
  static constexpr int kVN = DT / (16 * kVW);       // V vectors of a lane and key
  static constexpr int kKeys = 8;                   // keys of a lane: 8 g .. 8 g + 7
  static constexpr int kES = 2;
};
template <int DT>
struct PagedForm<false, DT> {
  static constexpr int kBlock = 16;
  static constexpr int kSteps = DT / 16;
  static constexpr int kKT = 1;
  static constexpr int kVW = 4;
  static constexpr int kVN = DT / 64;
  static constexpr int kKeys = 4;                   // keys 4 g .. 4 g + 3
  static constexpr int kES = 4;
};

__device__ __forceinline__ f32x4 mfma16_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// Half h (0 low, 1 high) of two dwords, side by side.
__device__ __forceinline__ uint32_t pair16(uint32_t lo, uint32_t hi, int h) {
  return __builtin_amdgcn_perm(hi, lo, h ? 0x07060302u : 0x05040100u);
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int BYTES>
struct VVec;
template <>
struct VVec<16> {
  typedef u32x4 T;
};
template <>
struct VVec<8> {
  typedef u32x2 T;
};

// One 32-key (16-key, fp32) block's keys and values in a wave's registers.
template <bool BF16, int DT>
struct PagedBlock {
  using F = PagedForm<BF16, DT>;
  u32x4 k[F::kKT][F::kSteps];
  typename VVec<F::kVW * F::kES>::T v[F::kKeys][F::kVN];
};

constexpr int kPWaves = 4;

template <bool BF16, int DT>
__global__ __launch_bounds__(256, DT == 256 ? 1 : 2) void paged_attention_kernel(PagedArgs a) {
  using F = PagedForm<BF16, DT>;
  constexpr int kUnit = F::kBlock * kPWaves;
  constexpr int kOC = F::kVN * F::kVW;              // O^T tiles of 16 columns
  constexpr int kLd = DT + 4;
  __shared__ float s_o[kPWaves][16][kLd];
  __shared__ float s_m[kPWaves][16], s_l[kPWaves][16];
  __shared__ int64_t s_scan[kPWaves];
  __shared__ int64_t s_first;
  __shared__ int s_seq;

  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int lq = l & 15, lg = l >> 4;
  const int part = blockIdx.x, h = blockIdx.y;
  const auto seq_at = [&](int s) { return seq_of_form<false>(a, s); };

  // ---- the part's share: every part takes an equal run of the batch's units --
  const int run = (a.B + 255) / 256;
  int64_t mine = 0;
  for (int s = tid * run; s < min(a.B, (tid + 1) * run); ++s) mine += addr::paged_seq_units(seq_at(s), a.G, a.window, kUnit);
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t up = __shfl_up(incl, d, 64);
    if (l >= d) incl += up;
  }
  if (l == 63) s_scan[wave] = incl;
  __syncthreads();
  int64_t U = 0;
#pragma unroll
  for (int w = 0; w < kPWaves; ++w) {
    if (w < wave) incl += s_scan[w];
    U += s_scan[w];
  }
  const int parts = addr::paged_parts(U, a.parts);
  const int64_t u0 = part < parts ? addr::paged_part_lo(U, parts, part) : U;
  const int64_t u1 = part < parts ? addr::paged_part_lo(U, parts, part + 1) : U;
  if (mine > 0 && incl - mine <= u0 && u0 < incl) {
    s_seq = tid * run;
    s_first = incl - mine;
  }
  __syncthreads();
  int4 join = make_int4(-1, 0, 0, 0);
  if (u0 < u1) {
    int s = s_seq;
    int64_t base = s_first;                          // unit the sequence starts at
    int64_t u = u0;
    while (u < u1) {
      const addr::PagedSeq sq = seq_at(s);
      const int64_t su = addr::paged_seq_units(sq, a.G, a.window, kUnit);
      if (base + su <= u) {
        base += su;
        ++s;
        continue;
      }
      const int nu = addr::paged_tile_units(sq, a.G, a.window, kUnit);
      const int j = static_cast<int>((u - base) / nu);
      const int64_t item = base + static_cast<int64_t>(j) * nu;     // the item's first unit
      const int w0 = static_cast<int>(u - item);
      const int w1 = static_cast<int>(min(static_cast<int64_t>(nu), u1 - item));
      const addr::PagedTile tile = addr::paged_tile(sq, a.G, a.window, j);

      // ---- the lane's query row ---------------------------------------------
      const int64_t rows = static_cast<int64_t>(sq.n) * a.G;
      const int64_t r = static_cast<int64_t>(j) * 16 + lq;
      const bool live = r < rows;
      const int qi = live ? static_cast<int>(r / a.G) : tile.i0;
      const int qh = h * a.G + (live ? static_cast<int>(r - static_cast<int64_t>(qi) * a.G) : 0);
      const int hi = live ? sq.len - sq.n + qi + 1 : 0;             // sees [lo, hi)
      const int lo = a.window > 0 ? hi - a.window : 0;
      const int64_t qe = static_cast<int64_t>(sq.q0 + qi) * a.q_ts + static_cast<int64_t>(qh) * a.q_hs;
      u32x4 qf[F::kSteps];
#pragma unroll
      for (int st = 0; st < F::kSteps; ++st) {
        const int d = (16 / F::kES) * (4 * st + lg);
        const bool ok = live && d < a.D;
        const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.q) + (qe + (d < a.D ? d : 0)) * F::kES);
        qf[st] = ok ? x : u32x4{0, 0, 0, 0};
      }

      float m = -INFINITY, lsum = 0.f;
      f32x4 o[kOC];
#pragma unroll
      for (int c = 0; c < kOC; ++c) o[c] = f32x4{0, 0, 0, 0};

      // ---- its keys -----------------------------------------------------------
      const int nblk = (tile.ve - tile.first + F::kBlock - 1) / F::kBlock;
      const int b_end = min(w1 * kPWaves, nblk);
      const int32_t* trow = a.table + static_cast<int64_t>(s) * a.ld_table;
      // first keys of the 8 that the lane's K rows and its V rows are of
      const int k_oct = BF16 ? 8 * (lq >> 2) : 8 * (lq >> 3);
      const int v_oct = BF16 ? 8 * lg : 8 * (lg >> 1);
      const int k_in = BF16 ? (lq & 3) : (lq & 7);                  // K row within them (+ 4 for tile 1)
      const int v_in = BF16 ? 0 : 4 * (lg & 1);
      struct Ids {
        int k, v;
        uint32_t k_row, v_row;
      };
      const auto ids_of = [&](int b) {
        const int tb = tile.first + b * F::kBlock;
        uint32_t kp, kr, vp, vr;
        addr::div_by(static_cast<uint32_t>(addr::paged_octet(tb + k_oct, tile.ve)) >> 3, a.page_octets, a.page_magic, kp, kr);
        addr::div_by(static_cast<uint32_t>(addr::paged_octet(tb + v_oct, tile.ve)) >> 3, a.page_octets, a.page_magic, vp, vr);
        return Ids{trow[kp], trow[vp], kr * 8, vr * 8};
      };
      const auto load = [&](const Ids& id, PagedBlock<BF16, DT>& x) {
        const int64_t kb = addr::paged_page(id.k, a.num_pages) * a.k_ps + h * a.k_hs + (id.k_row + k_in) * a.k_rs;
        const int64_t vb = addr::paged_page(id.v, a.num_pages) * a.v_ps + h * a.v_hs + (id.v_row + v_in) * a.v_rs;
#pragma unroll
        for (int u2 = 0; u2 < F::kKT; ++u2)
#pragma unroll
          for (int st = 0; st < F::kSteps; ++st) {
            const int d = (16 / F::kES) * (4 * st + lg);
            x.k[u2][st] = *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.k) + (kb + 4 * u2 * a.k_rs + (d < a.D ? d : 0)) * F::kES);
          }
#pragma unroll
        for (int t = 0; t < F::kKeys; ++t)
#pragma unroll
          for (int n = 0; n < F::kVN; ++n) {
            const int d = n * 16 * F::kVW + F::kVW * lq;
            x.v[t][n] = *reinterpret_cast<const typename VVec<F::kVW * F::kES>::T*>(
                static_cast<const char*>(a.v) + (vb + t * a.v_rs + (d < a.D ? d : 0)) * F::kES);
          }
      };
      const int hi_min = sq.len - sq.n + tile.i0 + 1;               // keys below it and from lo_max on: seen by every row
      const int lo_max = a.window > 0 ? sq.len - sq.n + tile.i1 + 1 - a.window : 0;
      const auto step = [&](int b, PagedBlock<BF16, DT>& x) {
        const int tb = tile.first + b * F::kBlock;
        f32x4 sacc[F::kKT];
#pragma unroll
        for (int u2 = 0; u2 < F::kKT; ++u2) sacc[u2] = f32x4{0, 0, 0, 0};
        const bool pad = DT > a.D;
#pragma unroll
        for (int st = 0; st < F::kSteps; ++st)
#pragma unroll
          for (int u2 = 0; u2 < F::kKT; ++u2) {
            u32x4 kx = x.k[u2][st];
            if (pad && (16 / F::kES) * (4 * st + lg) >= a.D) kx = u32x4{0, 0, 0, 0};
            if constexpr (BF16) {
              sacc[u2] = mfma16_bf16(kx, qf[st], sacc[u2]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sacc[u2] = mfma16_f32(__uint_as_float(kx[e]), __uint_as_float(qf[st][e]), sacc[u2]);
            }
          }
        float sc[F::kKeys];
#pragma unroll
        for (int i = 0; i < F::kKeys; ++i) sc[i] = sacc[i >> 2][i & 3] * a.scale_log2;
        const int t0 = tb + F::kKeys * lg;                           // the lane's first key
        if (tb + F::kBlock > hi_min || tb < lo_max) {
#pragma unroll
          for (int i = 0; i < F::kKeys; ++i) {
            const int t = t0 + i;
            if (t >= hi || t < lo) sc[i] = -INFINITY;
            // a key that no row of the tile sees may hold anything: 0 * NaN is not 0
            if (t >= tile.ve || t < tile.vs) {
#pragma unroll
              for (int n = 0; n < F::kVN; ++n)
#pragma unroll
                for (int w = 0; w < F::kVW * F::kES / 4; ++w) x.v[i][n][w] = 0;
            }
          }
        }
        float mx = sc[0];
#pragma unroll
        for (int i = 1; i < F::kKeys; ++i) mx = fmaxf(mx, sc[i]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (__any(mx > m)) {
          const float mn = fmaxf(m, mx);
          const float f = m == mn ? 1.f : exp2f(m - mn);             // m = mn = -inf: nothing summed yet
          m = mn;
          lsum *= f;
#pragma unroll
          for (int c = 0; c < kOC; ++c) o[c] *= f;
        }
        const float ms = m == -INFINITY ? 0.f : m;
        float p[F::kKeys];
#pragma unroll
        for (int i = 0; i < F::kKeys; ++i) {
          p[i] = __builtin_amdgcn_exp2f(sc[i] - ms);
          lsum += p[i];
        }
        if constexpr (BF16) {
          // probabilities enter the product in bf16 (relative error 2^-8, as
          // the values and the result have); their total stays in fp32
          u32x4 pf;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            pf[i] = static_cast<uint32_t>(f32_to_bf16_bits(p[2 * i])) | (static_cast<uint32_t>(f32_to_bf16_bits(p[2 * i + 1])) << 16);
#pragma unroll
          for (int n = 0; n < F::kVN; ++n)
#pragma unroll
            for (int c = 0; c < F::kVW; ++c) {
              u32x4 vf;
#pragma unroll
              for (int i = 0; i < 4; ++i) vf[i] = pair16(x.v[2 * i][n][c >> 1], x.v[2 * i + 1][n][c >> 1], c & 1);
              o[n * F::kVW + c] = mfma16_bf16(vf, pf, o[n * F::kVW + c]);
            }
        } else {
#pragma unroll
          for (int n = 0; n < F::kVN; ++n)
#pragma unroll
            for (int c = 0; c < F::kVW; ++c)
#pragma unroll
              for (int t = 0; t < 4; ++t)
                o[n * F::kVW + c] = mfma16_f32(__uint_as_float(x.v[t][n][c]), p[t], o[n * F::kVW + c]);
        }
      };
      int b = w0 * kPWaves + wave;
      if (b < b_end) {
        PagedBlock<BF16, DT> cur, nxt;
        Ids id = ids_of(b);
        load(id, cur);
        id = ids_of(b + kPWaves);
        for (; b + kPWaves < b_end; b += kPWaves) {
          const Ids id2 = ids_of(b + 2 * kPWaves);
          load(id, nxt);
          step(b, cur);
          cur = nxt;
          id = id2;
        }
        step(b, cur);
      }

      // ---- the four waves' results, joined --------------------------------------
      lsum += __shfl_xor(lsum, 16, 64);
      lsum += __shfl_xor(lsum, 32, 64);
      if (lg == 0) {
        s_m[wave][lq] = m;
        s_l[wave][lq] = lsum;
      }
#pragma unroll
      for (int n = 0; n < F::kVN; ++n)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          // O^T row 4 lg + v of tile (n, c): column 16 kVW n + kVW (4 lg + v) + c
          const int d = n * 16 * F::kVW + F::kVW * (4 * lg + v);
#pragma unroll
          for (int c = 0; c < F::kVW; c += 4)
            *reinterpret_cast<f32x4*>(&s_o[wave][lq][d + c]) =
                f32x4{o[n * F::kVW + c][v], o[n * F::kVW + c + 1][v], o[n * F::kVW + c + 2][v], o[n * F::kVW + c + 3][v]};
        }
      __syncthreads();
      const bool whole = w0 == 0 && w1 == nu;
      const int nrow = static_cast<int>(min(static_cast<int64_t>(16), rows - static_cast<int64_t>(j) * 16));
      float* slot = nullptr;
      if (!whole)
        slot = a.ws + ((static_cast<int64_t>(part) * a.HK + h) * 2 + (w0 == 0 ? 1 : 0)) * addr::paged_partial_floats(DT);
      for (int it = tid; it < nrow * (DT / 4); it += 256) {
        const int q = it / (DT / 4), d = (it - q * (DT / 4)) * 4;
        float M = s_m[0][q];
#pragma unroll
        for (int w = 1; w < kPWaves; ++w) M = fmaxf(M, s_m[w][q]);
        const float ms = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kPWaves; ++w) {
          const float f = exp2f(s_m[w][q] - ms);
          L += f * s_l[w][q];
          acc += f * *reinterpret_cast<const f32x4*>(&s_o[w][q][d]);
        }
        if (!whole) {
          *reinterpret_cast<f32x4*>(slot + q * DT + d) = acc;
          if (d == 0) {
            slot[16 * DT + q] = M;
            slot[16 * DT + 16 + q] = L;
          }
        } else if (d < a.D) {
          const int64_t rr = static_cast<int64_t>(j) * 16 + q;
          const int qi2 = static_cast<int>(rr / a.G);
          const int64_t tok = sq.q0 + qi2;
          const int head = h * a.G + static_cast<int>(rr - static_cast<int64_t>(qi2) * a.G);
          const float inv = L == 0.f ? 0.f : 1.0f / L;
          if (L == 0.f) acc = f32x4{0, 0, 0, 0};
          const int64_t e = tok * a.o_ts + head * a.o_hs + d;
          if constexpr (BF16) {
            u32x2 w2;
            w2[0] = static_cast<uint32_t>(f32_to_bf16_bits(acc[0] * inv)) | (static_cast<uint32_t>(f32_to_bf16_bits(acc[1] * inv)) << 16);
            w2[1] = static_cast<uint32_t>(f32_to_bf16_bits(acc[2] * inv)) | (static_cast<uint32_t>(f32_to_bf16_bits(acc[3] * inv)) << 16);
            *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + e) = w2;
          } else {
            *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + e) = acc * inv;
          }
          if (a.lse != nullptr && d == 0)
            a.lse[tok * a.H + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
        }
      }
      if (!whole && w0 > 0 && w1 == nu)                // the item ends here: this part names it for the join
        join = make_int4(s, j, addr::paged_part_of(U, parts, item), nrow);
      __syncthreads();
      u = item + w1;
    }
  }
  if (tid == 0) a.join[static_cast<int64_t>(part) * a.HK + h] = join;
}

// The parts of an item that was split, joined in the order of its keys: grid
// (parts, kv heads), the workgroup of the part that the item ends in.
template <bool BF16, int DT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  const int part = blockIdx.x, h = blockIdx.y;
  const int4 jn = a.join[static_cast<int64_t>(part) * a.HK + h];
  if (jn.x < 0) return;
  const int s = jn.x, j = jn.y, first = jn.z, nrow = jn.w;
  const int q0 = a.cu != nullptr ? addr::paged_seq(a.cu[s], a.cu[s + 1], 0, a.T, 0).q0 : s;
  const auto slot_of = [&](int p) {
    return a.ws + ((static_cast<int64_t>(p) * a.HK + h) * 2 + (p == first ? 1 : 0)) * addr::paged_partial_floats(DT);
  };
  for (int it = threadIdx.x; it < nrow * (DT / 4); it += 256) {
    const int q = it / (DT / 4), d = (it - q * (DT / 4)) * 4;
    float M = -INFINITY;
    for (int p = first; p <= part; ++p) M = fmaxf(M, slot_of(p)[16 * DT + q]);
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4 acc = {0, 0, 0, 0};
    for (int p = first; p <= part; ++p) {
      const float* sl = slot_of(p);
      const float f = exp2f(sl[16 * DT + q] - ms);
      L += f * sl[16 * DT + 16 + q];
      acc += f * *reinterpret_cast<const f32x4*>(sl + q * DT + d);
    }
    if (d >= a.D) continue;
    const int64_t rr = static_cast<int64_t>(j) * 16 + q;
    const int qi = static_cast<int>(rr / a.G);
    const int64_t tok = q0 + qi;
    const int head = h * a.G + static_cast<int>(rr - static_cast<int64_t>(qi) * a.G);
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    if (L == 0.f) acc = f32x4{0, 0, 0, 0};
    const int64_t e = tok * a.o_ts + head * a.o_hs + d;
    if constexpr (BF16) {
      u32x2 w2;
      w2[0] = static_cast<uint32_t>(f32_to_bf16_bits(acc[0] * inv)) | (static_cast<uint32_t>(f32_to_bf16_bits(acc[1] * inv)) << 16);
      w2[1] = static_cast<uint32_t>(f32_to_bf16_bits(acc[2] * inv)) | (static_cast<uint32_t>(f32_to_bf16_bits(acc[3] * inv)) << 16);
      *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + e) = w2;
    } else {
      *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + e) = acc * inv;
    }
    if (a.lse != nullptr && d == 0)
      a.lse[tok * a.H + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
int paged_width(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// Parts of the batch for each key/value head: two workgroups to a compute unit.
int paged_parts_for(int HK, int cus) { return std::max(1, 2 * cus / HK); }

int64_t paged_ws_bytes(int HK, int D, int cus) {
  const int64_t n = static_cast<int64_t>(paged_parts_for(HK, cus)) * HK;
  return n * (2 * addr::paged_partial_floats(paged_width(D)) * 4 + static_cast<int64_t>(sizeof(int4)));
}

// Whether ragged calls of these sizes have a chunk form, and the rows up to
// which a sequence stays with the row form.
bool chunk_form(bool bf16, int G, int D) { return bf16 && D <= 128 && G <= kChunkRows; }
constexpr int kRowFormRows = 16;

int64_t attention_ws_bytes(bool bf16, bool ragged, int G, int HK, int D, int cus) {
  return paged_ws_bytes(HK, D, cus) + (ragged && chunk_form(bf16, G, D) ? chunk_workspace_bytes(HK, paged_width(D), cus) : 0);
}

// What follows from the sizes alone.
void plan_paged(PagedArgs& a, bool bf16, int cus, int max_pages, int page_size, float scale) {
  a.parts = paged_parts_for(a.HK, cus);
  a.max_len = std::min<int64_t>(static_cast<int64_t>(max_pages) * page_size, (int64_t(1) << 31) - (1 << 16));
  a.page_octets = static_cast<uint32_t>(page_size / 8);
  a.page_magic = addr::div_magic(a.page_octets);
  a.row_limit = a.cu != nullptr && chunk_form(bf16, a.G, a.D) ? kRowFormRows : INT32_MAX;
  a.chunk_slots = chunk_slots_for(cus);
  a.chunk_share = static_cast<double>(a.HK) / (2.0 * a.chunk_slots);
  a.tq.tq = std::max(1, addr::chunk_tq(kChunkRows, a.G));
  a.tq.magic = addr::div_magic(a.tq.tq);
  a.g_magic = addr::div_magic(a.G);
  a.scale_log2 = scale * 1.44269504088896340736f;
}

template <bool BF16, int DT>
void launch_paged(const PagedArgs& a, hipStream_t st) {
  const dim3 grid(a.parts, a.HK);
  hipLaunchKernelGGL((paged_attention_kernel<BF16, DT>), grid, dim3(256), 0, st, a);
  hipLaunchKernelGGL((paged_join_kernel<BF16, DT>), grid, dim3(256), 0, st, a);
}

// Few tokens: every head of a token at once; many: each thread four heads or more.
void plan_append(AppendArgs& a, int cus) {
  const int n = a.H + 2 * a.HK;
  const int most = 256 / a.units;                        // units <= 256
  a.groups = std::max(1, std::min(a.T <= cus ? n : (n + 3) / 4, most));
  a.tokens = 256 / (a.units * a.groups);
}

bool strides_ok(int64_t a, int64_t b, int n) { return a >= 0 && b >= 0 && a % n == 0 && b % n == 0; }

// ---------------------------------------------------------------------------
// Address model: the kernels' global accesses for given tables, replayed with
// the kernels' own arithmetic.
// ---------------------------------------------------------------------------
struct PagedModel {
  int64_t bad = 0, checked = 0;
  std::vector<char> rows;                           // output rows written
  char msg[256] = "";
  void fail(const char* what, int64_t at, int64_t n, int64_t cap) {
    if (bad++ == 0) snprintf(msg, sizeof(msg), "%s: elements [%lld, %lld) of %lld", what, (long long)at, (long long)(at + n), (long long)cap);
  }
  void in(const char* what, int64_t at, int64_t n, int64_t cap) {
    ++checked;
    if (at < 0 || at + n > cap) fail(what, at, n, cap);
  }
};
int64_t extent3(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t cols) {
  return (n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + cols;
}

// The attention kernels for one width and element type.
template <bool BF16, int DT>
void model_attention(PagedModel& m, const PagedArgs& a) {
  using F = PagedForm<BF16, DT>;
  constexpr int kUnit = F::kBlock * kPWaves;
  constexpr int kVec = 16 / F::kES;
  const int max_pages = static_cast<int>(a.max_len / (8 * a.page_octets));
  const int64_t page_rows = 8 * a.page_octets;
  const int64_t k_elems = extent3(a.num_pages, a.k_ps, a.HK, a.k_hs, page_rows, a.k_rs, a.D);
  const int64_t v_elems = extent3(a.num_pages, a.v_ps, a.HK, a.v_hs, page_rows, a.v_rs, a.D);
  const int64_t q_elems = extent3(a.T, a.q_ts, a.H, a.q_hs, 1, 0, a.D);
  const int64_t o_elems = extent3(a.T, a.o_ts, a.H, a.o_hs, 1, 0, a.D);
  const auto seq_at = [&](int s) { return seq_of_form<false>(a, s); };
  std::vector<int64_t> start(a.B + 1, 0);
  for (int s = 0; s < a.B; ++s) start[s + 1] = start[s] + addr::paged_seq_units(seq_at(s), a.G, a.window, kUnit);
  const int64_t U = start[a.B];
  const int parts = addr::paged_parts(U, a.parts);
  std::vector<char> slots(static_cast<size_t>(a.parts) * a.HK * 2, 0);
  std::vector<char>& rows = m.rows;
  const auto written = [&](const addr::PagedSeq& sq, int j, int h, int nrow) {
    for (int q = 0; q < nrow; ++q) {
      const int64_t rr = static_cast<int64_t>(j) * 16 + q;
      const int64_t tok = sq.q0 + rr / a.G;
      const int64_t head = h * a.G + rr % a.G;
      m.in("output row", tok * a.H + head, 1, static_cast<int64_t>(a.T) * a.H);
      if (m.bad) return;
      if (rows[tok * a.H + head]++) m.fail("output row written twice", tok * a.H + head, 1, static_cast<int64_t>(a.T) * a.H);
      for (int d = 0; d < a.D; d += 4) m.in("out", tok * a.o_ts + head * a.o_hs + d, 4, o_elems);
    }
  };
  struct Join {
    int part, h, s, j, first, nrow;
  };
  std::vector<Join> joins;
  for (int part = 0; part < parts && !m.bad; ++part) {
    const int64_t u0 = addr::paged_part_lo(U, parts, part), u1 = addr::paged_part_lo(U, parts, part + 1);
    if (u0 >= u1) m.fail("a part without a unit", part, 1, parts);
    int s = 0;
    int64_t u = u0;
    while (u < u1 && !m.bad) {
      while (start[s + 1] <= u) ++s;
      const addr::PagedSeq sq = seq_at(s);
      const int nu = addr::paged_tile_units(sq, a.G, a.window, kUnit);
      const int j = static_cast<int>((u - start[s]) / nu);
      const int64_t item = start[s] + static_cast<int64_t>(j) * nu;
      const int w0 = static_cast<int>(u - item), w1 = static_cast<int>(std::min<int64_t>(nu, u1 - item));
      const addr::PagedTile t = addr::paged_tile(sq, a.G, a.window, j);
      const int64_t nrows = static_cast<int64_t>(sq.n) * a.G;
      const int nblk = (t.ve - t.first + F::kBlock - 1) / F::kBlock;
      if (nblk > nu * kPWaves) m.fail("blocks past the item's units", nblk, 0, nu * kPWaves);
      const int b_end = std::min(w1 * kPWaves, nblk);
      const int nrow = static_cast<int>(std::min<int64_t>(16, nrows - static_cast<int64_t>(j) * 16));
      for (int h = 0; h < a.HK; ++h) {
        for (int l = 0; l < 64; ++l) {
          const int lq = l & 15, lg = l >> 4;
          const int64_t r = static_cast<int64_t>(j) * 16 + lq;
          const bool live = r < nrows;
          const int qi = live ? static_cast<int>(r / a.G) : t.i0;
          const int64_t qh = h * a.G + (live ? r - static_cast<int64_t>(qi) * a.G : 0);
          for (int st = 0; st < F::kSteps; ++st) {
            const int d = kVec * (4 * st + lg);
            m.in("q", (sq.q0 + qi) * a.q_ts + qh * a.q_hs + (d < a.D ? d : 0), kVec, q_elems);
          }
          const int k_oct = BF16 ? 8 * (lq >> 2) : 8 * (lq >> 3), v_oct = BF16 ? 8 * lg : 8 * (lg >> 1);
          const int k_in = BF16 ? (lq & 3) : (lq & 7), v_in = BF16 ? 0 : 4 * (lg & 1);
          for (int b = w0 * kPWaves; b < b_end + 2 * kPWaves && t.ve > 0 && b_end > w0 * kPWaves; ++b) {   // ids are read up to two rounds ahead
            const int tb = t.first + b * F::kBlock;
            uint32_t kp, kr, vp, vr;
            const int kt = addr::paged_octet(tb + k_oct, t.ve), vt = addr::paged_octet(tb + v_oct, t.ve);
            addr::div_by(static_cast<uint32_t>(kt) >> 3, a.page_octets, a.page_magic, kp, kr);
            addr::div_by(static_cast<uint32_t>(vt) >> 3, a.page_octets, a.page_magic, vp, vr);
            if (kp != static_cast<uint32_t>(kt / page_rows) || kr * 8 != static_cast<uint32_t>(kt % page_rows)) m.fail("division", kt, 0, page_rows);
            m.in("page table row", kp, 1, max_pages);
            m.in("page table row", vp, 1, max_pages);
            if (m.bad) return;
            const int64_t kb = addr::paged_page(a.table[s * a.ld_table + kp], a.num_pages) * a.k_ps + h * a.k_hs + (kr * 8 + k_in) * a.k_rs;
            const int64_t vb = addr::paged_page(a.table[s * a.ld_table + vp], a.num_pages) * a.v_ps + h * a.v_hs + (vr * 8 + v_in) * a.v_rs;
            m.in("page row", kr * 8 + k_in + 4 * (F::kKT - 1), 1, page_rows);
            m.in("page row", vr * 8 + v_in + F::kKeys - 1, 1, page_rows);
            for (int u2 = 0; u2 < F::kKT; ++u2)
              for (int st = 0; st < F::kSteps; ++st) {
                const int d = kVec * (4 * st + lg);
                m.in("k cache", kb + 4 * u2 * a.k_rs + (d < a.D ? d : 0), kVec, k_elems);
              }
            for (int tt = 0; tt < F::kKeys; ++tt)
              for (int n = 0; n < F::kVN; ++n) {
                const int d = n * 16 * F::kVW + F::kVW * lq;
                m.in("v cache", vb + tt * a.v_rs + (d < a.D ? d : 0), F::kVW, v_elems);
              }
          }
        }
        if (w0 == 0 && w1 == nu) {
          written(sq, j, h, nrow);
        } else {
          const int64_t slot = (static_cast<int64_t>(part) * a.HK + h) * 2 + (w0 == 0 ? 1 : 0);
          m.in("workspace slot", slot, 1, static_cast<int64_t>(slots.size()));
          if (m.bad) return;
          if (slots[slot]++) m.fail("workspace slot written twice", slot, 1, static_cast<int64_t>(slots.size()));
          if (w0 > 0 && w1 == nu) joins.push_back({part, h, s, j, addr::paged_part_of(U, parts, item), nrow});
        }
      }
      u = item + w1;
    }
  }
  for (const Join& jn : joins) {
    for (int p = jn.first; p <= jn.part && !m.bad; ++p) {
      const int64_t slot = (static_cast<int64_t>(p) * a.HK + jn.h) * 2 + (p == jn.first ? 1 : 0);
      m.in("joined slot", slot, 1, static_cast<int64_t>(slots.size()));
      if (m.bad) return;
      if (slots[slot] != 1) m.fail("a joined slot that no part writes, or two joins read", slot, 1, static_cast<int64_t>(slots.size()));
      slots[slot] = 2;
    }
    written(seq_at(jn.s), jn.j, jn.h, jn.nrow);
  }
  for (char c : slots)
    if (c == 1 && !m.bad) m.fail("a partial result that no join reads", 0, 1, 0);
}

// The chunk form.
template <int DT>
void model_chunk(PagedModel& m, const PagedArgs& a) {
  constexpr int kWaves = 4, kRowB = DT * 2, kTileB = 64 * kRowB, kRowsPer = 1024 / kRowB;
  // what the transfers leave in LDS, and what the operand reads take from it
  std::vector<int> k_lds(kTileB / 16, -1), v_lds(kTileB / 16, -1);
  for (int w = 0; w < kWaves; ++w)
    for (int x = 0; x < 16 / kRowsPer; ++x)
      for (int l = 0; l < 64; ++l) {
        const int row = 16 * w + x * kRowsPer + l / (64 / kRowsPer), pos = l % (64 / kRowsPer);
        const int at = ((16 * w + x * kRowsPer) * kRowB + l * 16) / 16;
        k_lds[at] = row * 64 + addr::chunk_k_pos(DT, row, pos);
        v_lds[at] = row * 64 + addr::chunk_v_pos(DT, row, pos);
      }
  for (int l = 0; l < 64; ++l) {
    const int lq = l & 31, hl = l >> 5, v_row = 4 * hl + ((l & 15) >> 2);
    for (int u = 0; u < 2; ++u)
      for (int st = 0; st < DT / 16; ++st) {
        const int at = lq * kRowB + addr::chunk_k_pos(DT, lq, 2 * st + hl) * 16 + u * 32 * kRowB;
        m.in("K operand (LDS)", at, 16, kTileB);
        if (k_lds[at / 16] != (32 * u + lq) * 64 + 2 * st + hl) m.fail("K operand of another piece", at, 16, kTileB);
      }
    for (int d = 0; d < DT / 32; ++d)
      for (int g = 0; g < 4; ++g)
        for (int x = 0; x < 2; ++x) {
          const int piece = 4 * d + 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
          const int at = v_row * kRowB + addr::chunk_v_pos(DT, v_row, piece) * 16 + (l & 1) * 8 + (g * 16 + 8 * x) * kRowB;
          m.in("V operand (LDS)", at, 8, kTileB);
          if (v_lds[at / 16] != (g * 16 + 8 * x + v_row) * 64 + piece) m.fail("V operand of another piece", at, 8, kTileB);
        }
  }
  const int max_pages = static_cast<int>(a.max_len / (8 * a.page_octets));
  const int64_t page_rows = 8 * a.page_octets;
  const int64_t k_elems = extent3(a.num_pages, a.k_ps, a.HK, a.k_hs, page_rows, a.k_rs, a.D);
  const int64_t v_elems = extent3(a.num_pages, a.v_ps, a.HK, a.v_hs, page_rows, a.v_rs, a.D);
  const int64_t q_elems = extent3(a.T, a.q_ts, a.H, a.q_hs, 1, 0, a.D), o_elems = extent3(a.T, a.o_ts, a.H, a.o_hs, 1, 0, a.D);
  const addr::ChunkTq& tq = a.tq;
  int64_t U2 = 0, n = 0, slots = 0, split = 0;
  for (int s = 0; s < a.B; ++s) U2 += addr::chunk_work2(seq_of_form<true>(a, s), tq, a.window);
  const int pt = addr::chunk_part_tiles(U2, a.chunk_share, kChunkLeast);
  for (int s = 0; s < a.B && !m.bad; ++s) {
    const addr::PagedSeq sq = seq_of_form<true>(a, s);
    const int nt = addr::chunk_tiles(sq, tq), np = addr::chunk_parts(sq, tq, a.window, pt, addr::div_magic(pt));
    n += static_cast<int64_t>(nt) * np;
    if (np > 1) {
      slots += static_cast<int64_t>(nt) * np;
      split += nt;
    }
    for (int j = 0; j < nt && !m.bad; ++j) {
      const addr::PagedTile t = addr::chunk_tile(sq, tq.tq, a.window, j);
      const int nkt = addr::chunk_key_tiles(t);
      const int nrow = (t.i1 - t.i0 + 1) * a.G;
      if (nrow < 1 || nrow > kChunkRows) m.fail("rows of a tile", 0, nrow, kChunkRows);
      for (int h = 0; h < a.HK && !m.bad; ++h) {
        for (int r = 0; r < nrow; ++r) {
          const int64_t tok = sq.q0 + t.i0 + r / a.G, head = h * a.G + r % a.G;
          m.in("output row", tok * a.H + head, 1, static_cast<int64_t>(a.T) * a.H);
          if (m.bad) return;
          if (m.rows[tok * a.H + head]++) m.fail("output row written twice", tok, 1, a.T);
          m.in("q", tok * a.q_ts + head * a.q_hs, a.D, q_elems);
          m.in("out", tok * a.o_ts + head * a.o_hs, a.D, o_elems);
        }
        for (int kt = 0; kt < nkt + 2 && nkt > 0; ++kt)       // ids are read past the last tile, too
          for (int w = 0; w < 8; ++w) {
            uint32_t pg, row;
            addr::div_by(static_cast<uint32_t>(addr::paged_octet(t.first + kt * 64 + 8 * w, t.ve)) >> 3, a.page_octets, a.page_magic, pg, row);
            m.in("page table row", pg, 1, max_pages);
            if (m.bad) return;
            if (kt >= nkt) continue;
            const int64_t page = addr::paged_page(a.table[s * a.ld_table + pg], a.num_pages);
            for (int rr = 0; rr < 8; ++rr) {
              m.in("page row", row * 8 + rr, 1, page_rows);
              m.in("k cache", page * a.k_ps + h * a.k_hs + (row * 8 + rr) * a.k_rs, a.D, k_elems);
              m.in("v cache", page * a.v_ps + h * a.v_hs + (row * 8 + rr) * a.v_rs, a.D, v_elems);
            }
          }
      }
    }
  }
  m.in("partial results", 0, slots, addr::chunk_slots_per_head(a.HK, a.chunk_slots));
  m.in("split tiles", 0, 2 * split, addr::chunk_slots_per_head(a.HK, a.chunk_slots));
  const int64_t per = (n * a.HK + 7) >> 3;
  m.in("workgroups", 0, 8 * per, chunk_grid(a));
}

void model_rows(PagedModel& m, const PagedArgs& a) {
  for (int s = 0; s < a.B && !m.bad; ++s) {
    const addr::PagedSeq sq = a.cu != nullptr ? addr::paged_seq(a.cu[s], a.cu[s + 1], 0, a.T, 0) : addr::PagedSeq{s, 1, 0};
    for (int i = 0; i < sq.n; ++i)
      for (int h = 0; h < a.H; ++h)
        if (!m.rows[static_cast<int64_t>(sq.q0 + i) * a.H + h] && !m.bad) m.fail("output row never written", sq.q0 + i, 1, a.T);
  }
}

template <int VE, bool PAIRS>
void model_append(PagedModel& m, const AppendArgs& a, const int64_t* slots, const int64_t* positions) {
  const int64_t pages = a.num_slots / a.page_size;
  const int64_t q_elems = extent3(a.T, a.q_ts, a.H, a.q_hs, 1, 0, a.D), qo_elems = extent3(a.T, a.qo_ts, a.H, a.qo_hs, 1, 0, a.D);
  const int64_t k_elems = extent3(a.T, a.k_ts, a.HK, a.k_hs, 1, 0, a.D), v_elems = extent3(a.T, a.v_ts, a.HK, a.v_hs, 1, 0, a.D);
  const int64_t kc_elems = extent3(pages, a.kc_ps, a.HK, a.kc_hs, a.page_size, a.kc_rs, a.D);
  const int64_t vc_elems = extent3(pages, a.vc_ps, a.HK, a.vc_hs, a.page_size, a.vc_rs, a.D);
  const int heads = a.H + 2 * a.HK;
  const int per_token = a.units * a.groups;
  if (per_token * a.tokens > 256 || a.tokens < 1) m.fail("threads of a workgroup", 0, per_token * a.tokens, 256);
  std::vector<int> seen(static_cast<size_t>(heads) * a.D, 0);
  for (int64_t blk = 0; blk * a.tokens < a.T && !m.bad; ++blk)
    for (int tok = 0; tok < a.tokens && blk * a.tokens + tok < a.T; ++tok) {
      const int64_t t = blk * a.tokens + tok;
      std::fill(seen.begin(), seen.end(), 0);
      for (int in_tok = 0; in_tok < per_token; ++in_tok) {
        const int grp = in_tok / a.units, u = in_tok - grp * a.units;
        const addr::AppendCols c = addr::append_cols(u, VE, a.D, a.R, PAIRS);
        if (c.rot) {
          const int64_t row = addr::append_pos(positions[t], a.max_pos) * a.R;
          m.in("cosines", row + addr::append_pair(u, VE), VE, row + a.R / 2);
          m.in("cos_sin", row + a.R / 2 + addr::append_pair(u, VE), VE, a.max_pos * a.R);
        }
        const bool stored = addr::append_stored(slots[t], a.num_slots);
        const int64_t page = stored ? slots[t] / a.page_size : 0, prow = stored ? slots[t] - page * a.page_size : 0;
        for (int h0 = grp; h0 < heads; h0 += 4 * a.groups)
          for (int b = 0; b < 4; ++b) {
            const int h = h0 + b * a.groups;
            if (h >= heads) continue;
            for (int col : {c.c0, c.c1}) {
              if (col < 0) continue;
              for (int i = 0; i < VE && col + i < a.D; ++i) ++seen[static_cast<size_t>(h) * a.D + col + i];
              if (h < a.H) {
                m.in("q", t * a.q_ts + h * a.q_hs + col, VE, q_elems);
                m.in("q_out", t * a.qo_ts + h * a.qo_hs + col, VE, qo_elems);
              } else if (h < a.H + a.HK) {
                m.in("k", t * a.k_ts + (h - a.H) * a.k_hs + col, VE, k_elems);
                if (stored) m.in("k cache", page * a.kc_ps + (h - a.H) * a.kc_hs + prow * a.kc_rs + col, VE, kc_elems);
              } else {
                m.in("v", t * a.v_ts + (h - a.H - a.HK) * a.v_hs + col, VE, v_elems);
                if (stored) m.in("v cache", page * a.vc_ps + (h - a.H - a.HK) * a.vc_hs + prow * a.vc_rs + col, VE, vc_elems);
              }
            }
          }
      }
      for (size_t i = 0; i < seen.size(); ++i)
        if (seen[i] != 1 && !m.bad) m.fail("a column taken other than once", static_cast<int64_t>(i), 1, a.D);
    }
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

int gs_append_kv(int32_t dtype, const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs,
                 const void* v, int64_t v_ts, int64_t v_hs, int64_t num_tokens, int32_t heads, int32_t kv_heads,
                 int32_t head_dim, const int64_t* positions, const float* cos_sin, int64_t max_pos, int32_t rot_dim,
                 int32_t interleaved, const int64_t* slots, void* k_cache, int64_t kc_ps, int64_t kc_hs, int64_t kc_rs,
                 void* v_cache, int64_t vc_ps, int64_t vc_hs, int64_t vc_rs, int64_t num_pages, int32_t page_size,
                 void* q_out, int64_t qo_ts, int64_t qo_hs, void* stream) {
  const char* who = "gs_append_kv";
  GS_CHECK_ARG(dtype == GS_DTYPE_BF16 || dtype == GS_DTYPE_FP32, "%s: dtype=%d", who, dtype);
  GS_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t(1) << 31), "%s: num_tokens=%lld", who, (long long)num_tokens);
  GS_CHECK_ARG(heads >= 0 && kv_heads > 0 && heads <= 4096 && kv_heads <= 4096, "%s: heads=%d kv_heads=%d", who, heads, kv_heads);
  GS_CHECK_ARG(head_dim > 0 && head_dim <= 512, "%s: head_dim=%d (1 .. 512)", who, head_dim);
  GS_CHECK_ARG(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 2 == 0, "%s: rot_dim=%d of head_dim=%d", who, rot_dim, head_dim);
  GS_CHECK_ARG(page_size > 0 && num_pages > 0, "%s: page_size=%d num_pages=%lld", who, page_size, (long long)num_pages);
  if (num_tokens == 0) return GS_OK;
  // the stride of a dimension of one is never used, and may be anything
  if (num_tokens == 1) q_ts = k_ts = v_ts = qo_ts = 0;
  if (heads == 1) q_hs = qo_hs = 0;
  if (kv_heads == 1) k_hs = v_hs = kc_hs = vc_hs = 0;
  if (num_pages == 1) kc_ps = vc_ps = 0;
  if (page_size == 1) kc_rs = vc_rs = 0;
  GS_CHECK_ARG(k != nullptr && v != nullptr && slots != nullptr && k_cache != nullptr && v_cache != nullptr &&
                   (heads == 0 || (q != nullptr && q_out != nullptr)), "%s: null tensor", who);
  GS_CHECK_ARG(rot_dim == 0 || (positions != nullptr && cos_sin != nullptr && max_pos > 0),
               "%s: rot_dim=%d without positions or cos_sin", who, rot_dim);
  const bool bf16 = dtype == GS_DTYPE_BF16;
  const int ve = bf16 ? 8 : 4;
  const bool vec = head_dim % ve == 0 && rot_dim % (2 * ve) == 0 && aligned16(k) && aligned16(v) && aligned16(k_cache) &&
                   aligned16(v_cache) && strides_ok(k_ts, k_hs, ve) && strides_ok(v_ts, v_hs, ve) &&
                   strides_ok(kc_ps, kc_hs, ve) && strides_ok(vc_ps, vc_hs, ve) && strides_ok(kc_rs, vc_rs, ve) &&
                   (heads == 0 || (aligned16(q) && aligned16(q_out) && strides_ok(q_ts, q_hs, ve) && strides_ok(qo_ts, qo_hs, ve)));
  const int VE = vec ? ve : 1;
  AppendArgs a{};
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
  a.units = addr::append_units(VE, head_dim, rot_dim);
  plan_append(a, device_cus());
  const dim3 grid(static_cast<unsigned>((num_tokens + a.tokens - 1) / a.tokens));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a); };
  const bool pr = interleaved != 0;
  if (bf16) {
    if (vec) pr ? go(append_kv_kernel<true, 8, true>) : go(append_kv_kernel<true, 8, false>);
    else pr ? go(append_kv_kernel<true, 1, true>) : go(append_kv_kernel<true, 1, false>);
  } else {
    if (vec) pr ? go(append_kv_kernel<false, 4, true>) : go(append_kv_kernel<false, 4, false>);
    else pr ? go(append_kv_kernel<false, 1, true>) : go(append_kv_kernel<false, 1, false>);
  }
  GS_CHECK_LAUNCH(who);
  return GS_OK;
}

int gs_cache_slots(const int32_t* page_table, int64_t ld_table, int32_t max_pages, int64_t num_pages, int32_t page_size,
                   const int32_t* kv_lens, const int32_t* cu_seqlens, int32_t num_seqs, int64_t num_tokens,
                   int64_t* slots, int64_t* positions, void* stream) {
  const char* who = "gs_cache_slots";
  GS_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t(1) << 31) && num_seqs >= 0, "%s: num_tokens=%lld num_seqs=%d",
               who, (long long)num_tokens, num_seqs);
  GS_CHECK_ARG(page_size > 0 && max_pages >= 0 && ld_table >= max_pages && num_pages >= 0 && num_pages < (int64_t(1) << 31),
               "%s: page_size=%d max_pages=%d ld_table=%lld num_pages=%lld", who, page_size, max_pages,
               (long long)ld_table, (long long)num_pages);
  if (num_tokens == 0) return GS_OK;
  GS_CHECK_ARG(slots != nullptr && positions != nullptr &&
                   (num_seqs == 0 || (kv_lens != nullptr && (page_table != nullptr || max_pages == 0))),
               "%s: null tensor", who);
  hipLaunchKernelGGL(cache_slots_kernel, dim3(static_cast<unsigned>((num_tokens + 255) / 256)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), page_table, ld_table, max_pages, static_cast<int>(num_pages),
                     page_size, kv_lens, cu_seqlens, num_seqs, static_cast<int>(num_tokens), slots, positions);
  GS_CHECK_LAUNCH(who);
  return GS_OK;
}

int64_t gs_paged_attention_workspace_bytes(int32_t dtype, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t ragged) {
  if ((dtype != GS_DTYPE_BF16 && dtype != GS_DTYPE_FP32) || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
      head_dim <= 0 || head_dim > 256) {
    set_error("gs_paged_attention_workspace_bytes: dtype=%d heads=%d kv_heads=%d head_dim=%d", dtype, heads, kv_heads, head_dim);
    return -GS_ERR_INVALID;
  }
  return attention_ws_bytes(dtype == GS_DTYPE_BF16, ragged != 0, heads / kv_heads, kv_heads, head_dim, device_cus());
}

int gs_paged_attention(int32_t dtype, const void* q, int64_t q_ts, int64_t q_hs, const void* k_cache, int64_t k_ps,
                       int64_t k_hs, int64_t k_rs, const void* v_cache, int64_t v_ps, int64_t v_hs, int64_t v_rs,
                       int64_t num_pages, int32_t page_size, const int32_t* page_table, int64_t ld_table,
                       int32_t max_pages, const int32_t* kv_lens, const int32_t* cu_seqlens, int32_t num_seqs,
                       int64_t num_tokens, int32_t max_q, int32_t heads, int32_t kv_heads, int32_t head_dim,
                       float scale, int32_t window, void* out, int64_t o_ts, int64_t o_hs, float* lse,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "gs_paged_attention";
  GS_CHECK_ARG(dtype == GS_DTYPE_BF16 || dtype == GS_DTYPE_FP32, "%s: dtype=%d", who, dtype);
  GS_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t(1) << 31) && num_seqs >= 0, "%s: num_tokens=%lld num_seqs=%d", who,
               (long long)num_tokens, num_seqs);
  GS_CHECK_ARG(cu_seqlens != nullptr || num_tokens == num_seqs, "%s: num_tokens=%lld of num_seqs=%d without cu_seqlens", who,
               (long long)num_tokens, num_seqs);
  GS_CHECK_ARG(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65536, "%s: heads=%d kv_heads=%d", who, heads, kv_heads);
  const bool bf16 = dtype == GS_DTYPE_BF16;
  const int ve = bf16 ? 8 : 4;
  GS_CHECK_ARG(head_dim > 0 && head_dim <= 256 && head_dim % ve == 0, "%s: head_dim=%d must be a multiple of %d up to 256", who,
               head_dim, ve);
  GS_CHECK_ARG(page_size > 0 && page_size % 8 == 0, "%s: page_size=%d must be a multiple of 8", who, page_size);
  GS_CHECK_ARG(num_pages > 0 && num_pages < (int64_t(1) << 31) && max_pages >= 0 && ld_table >= max_pages,
               "%s: num_pages=%lld max_pages=%d ld_table=%lld", who, (long long)num_pages, max_pages, (long long)ld_table);
  GS_CHECK_ARG(window >= 0 && max_q >= 0, "%s: window=%d max_q=%d", who, window, max_q);
  if (num_tokens == 0 || num_seqs == 0) return GS_OK;
  // the stride of a dimension of one is never used, and may be anything
  if (num_tokens == 1) q_ts = o_ts = 0;
  if (heads == 1) q_hs = o_hs = 0;
  if (kv_heads == 1) k_hs = v_hs = 0;
  if (num_pages == 1) k_ps = v_ps = 0;
  GS_CHECK_ARG(q != nullptr && k_cache != nullptr && v_cache != nullptr && out != nullptr && kv_lens != nullptr &&
                   (page_table != nullptr || max_pages == 0), "%s: null tensor", who);
  GS_CHECK_ARG(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out) && strides_ok(q_ts, q_hs, ve) &&
                   strides_ok(k_ps, k_hs, ve) && strides_ok(v_ps, v_hs, ve) && strides_ok(k_rs, v_rs, ve) &&
                   strides_ok(o_ts, o_hs, ve),
               "%s: q, the caches and out must be 16-byte aligned with strides that are multiples of %d elements", who, ve);
  const int cus = device_cus();
  const int64_t need = attention_ws_bytes(bf16, cu_seqlens != nullptr, heads / kv_heads, kv_heads, head_dim, cus);
  if (workspace == nullptr || workspace_bytes < need) {
    set_error("%s: workspace of %lld bytes needed (got %lld)", who, (long long)need, (long long)(workspace ? workspace_bytes : 0));
    return GS_ERR_WORKSPACE;
  }
  GS_CHECK_ARG(aligned16(workspace), "%s: workspace must be 16-byte aligned", who);
  PagedArgs a{};
  a.q = q; a.q_ts = q_ts; a.q_hs = q_hs;
  a.out = out; a.o_ts = o_ts; a.o_hs = o_hs;
  a.k = k_cache; a.k_ps = k_ps; a.k_hs = k_hs; a.k_rs = k_rs;
  a.v = v_cache; a.v_ps = v_ps; a.v_hs = v_hs; a.v_rs = v_rs;
  a.table = page_table; a.ld_table = ld_table;
  a.lens = kv_lens; a.cu = cu_seqlens; a.lse = lse;
  a.num_pages = static_cast<int>(num_pages);
  a.B = num_seqs; a.T = static_cast<int>(num_tokens);
  a.H = heads; a.HK = kv_heads; a.G = heads / kv_heads; a.D = head_dim;
  a.window = window;
  plan_paged(a, bf16, cus, max_pages, page_size, scale);
  const int DT = paged_width(head_dim);
  a.ws = static_cast<float*>(workspace);
  const int64_t partials = static_cast<int64_t>(a.parts) * kv_heads * 2 * addr::paged_partial_floats(DT);
  a.join = reinterpret_cast<int4*>(a.ws + partials);
  a.chunk_ws = reinterpret_cast<float*>(a.join + static_cast<int64_t>(a.parts) * kv_heads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.row_limit != INT32_MAX && (max_q == 0 || static_cast<int64_t>(max_q) * a.G > a.row_limit)) {
    GS_CHECK_ARG(chunk_grid(a) < (int64_t(1) << 31), "%s: too many tiles", who);
    launch_chunk(a, DT, st);
  }
  switch (DT) {
    case 64: bf16 ? launch_paged<true, 64>(a, st) : launch_paged<false, 64>(a, st); break;
    case 128: bf16 ? launch_paged<true, 128>(a, st) : launch_paged<false, 128>(a, st); break;
    default: bf16 ? launch_paged<true, 256>(a, st) : launch_paged<false, 256>(a, st); break;
  }
  GS_CHECK_LAUNCH(who);
  return GS_OK;
}

int64_t gs_check_paged_addresses(int32_t dtype, int64_t q_ts, int64_t q_hs, int64_t k_ps, int64_t k_hs, int64_t k_rs,
                                 int64_t v_ps, int64_t v_hs, int64_t v_rs, int64_t num_pages, int32_t page_size,
                                 const int32_t* page_table, int64_t ld_table, int32_t max_pages,
                                 const int32_t* kv_lens, const int32_t* cu_seqlens, int32_t num_seqs,
                                 int64_t num_tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t window,
                                 int64_t o_ts, int64_t o_hs, int32_t cus, char* msg, int64_t msg_len,
                                 int64_t* checked) {
  const char* who = "gs_check_paged_addresses";
  const bool bf16 = dtype == GS_DTYPE_BF16;
  GS_CHECK_ARG((bf16 || dtype == GS_DTYPE_FP32) && num_tokens > 0 && num_seqs > 0 && num_tokens < (int64_t(1) << 31) &&
                   heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && head_dim > 0 && head_dim <= 256 &&
                   head_dim % (bf16 ? 8 : 4) == 0 && page_size > 0 && page_size % 8 == 0 && num_pages > 0 &&
                   max_pages >= 0 && ld_table >= max_pages && kv_lens != nullptr && window >= 0 && cus > 0 &&
                   (cu_seqlens != nullptr || num_tokens == num_seqs), "%s: sizes", who);
  PagedArgs a{};
  a.q_ts = q_ts; a.q_hs = q_hs; a.o_ts = o_ts; a.o_hs = o_hs;
  a.k_ps = k_ps; a.k_hs = k_hs; a.k_rs = k_rs;
  a.v_ps = v_ps; a.v_hs = v_hs; a.v_rs = v_rs;
  a.table = page_table; a.ld_table = ld_table; a.lens = kv_lens; a.cu = cu_seqlens;
  a.num_pages = static_cast<int>(num_pages);
  a.B = num_seqs; a.T = static_cast<int>(num_tokens);
  a.H = heads; a.HK = kv_heads; a.G = heads / kv_heads; a.D = head_dim;
  a.window = window;
  plan_paged(a, bf16, cus, max_pages, page_size, 1.f);
  PagedModel m;
  m.rows.assign(static_cast<size_t>(a.T) * a.H, 0);
  if (a.row_limit != INT32_MAX) paged_width(head_dim) == 64 ? model_chunk<64>(m, a) : model_chunk<128>(m, a);
  switch (paged_width(head_dim)) {
    case 64: bf16 ? model_attention<true, 64>(m, a) : model_attention<false, 64>(m, a); break;
    case 128: bf16 ? model_attention<true, 128>(m, a) : model_attention<false, 128>(m, a); break;
    default: bf16 ? model_attention<true, 256>(m, a) : model_attention<false, 256>(m, a); break;
  }
  model_rows(m, a);
  if (checked) *checked = m.checked;
  if (msg && msg_len > 0) snprintf(msg, static_cast<size_t>(msg_len), "%s", m.msg);
  return m.bad;
}

int64_t gs_check_append_addresses(int32_t dtype, int32_t vec, int64_t q_ts, int64_t q_hs, int64_t k_ts, int64_t k_hs,
                                  int64_t num_tokens, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                  const int64_t* positions, int64_t max_pos, int32_t rot_dim, int32_t interleaved,
                                  const int64_t* slots, int64_t c_ps, int64_t c_hs, int64_t c_rs, int64_t num_pages,
                                  int32_t page_size, int32_t cus, char* msg, int64_t msg_len, int64_t* checked) {
  const char* who = "gs_check_append_addresses";
  const bool bf16 = dtype == GS_DTYPE_BF16;
  const int ve = vec ? (bf16 ? 8 : 4) : 1;
  GS_CHECK_ARG((bf16 || dtype == GS_DTYPE_FP32) && num_tokens > 0 && num_tokens < (int64_t(1) << 31) && heads >= 0 &&
                   kv_heads > 0 && head_dim > 0 && head_dim <= 512 && rot_dim >= 0 && rot_dim <= head_dim &&
                   rot_dim % 2 == 0 && head_dim % ve == 0 && rot_dim % (2 * ve) == 0 && page_size > 0 && num_pages > 0 &&
                   slots != nullptr && (rot_dim == 0 || (positions != nullptr && max_pos > 0)) && cus > 0, "%s: sizes", who);
  AppendArgs a{};
  a.q_ts = a.qo_ts = q_ts; a.q_hs = a.qo_hs = q_hs;
  a.k_ts = a.v_ts = k_ts; a.k_hs = a.v_hs = k_hs;
  a.kc_ps = a.vc_ps = c_ps; a.kc_hs = a.vc_hs = c_hs; a.kc_rs = a.vc_rs = c_rs;
  a.max_pos = max_pos;
  a.num_slots = num_pages * page_size;
  a.page_size = static_cast<uint32_t>(page_size);
  a.T = static_cast<int>(num_tokens);
  a.H = heads; a.HK = kv_heads; a.D = head_dim; a.R = rot_dim;
  a.units = addr::append_units(ve, head_dim, rot_dim);
  plan_append(a, cus);
  PagedModel m;
  const bool pr = interleaved != 0;
  if (ve == 8) pr ? model_append<8, true>(m, a, slots, positions) : model_append<8, false>(m, a, slots, positions);
  else if (ve == 4) pr ? model_append<4, true>(m, a, slots, positions) : model_append<4, false>(m, a, slots, positions);
  else pr ? model_append<1, true>(m, a, slots, positions) : model_append<1, false>(m, a, slots, positions);
  if (checked) *checked = m.checked;
  if (msg && msg_len > 0) snprintf(msg, static_cast<size_t>(msg_len), "%s", m.msg);
  return m.bad;
}

}  // extern "C"
