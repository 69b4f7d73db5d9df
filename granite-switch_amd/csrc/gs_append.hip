// Rotated append to a paged key/value cache, and the slots of a batch's tokens.
//
// A cache is [pages, kv heads, page rows, head dim] with any page, head and row
// stride (a head's rows of a page side by side, or a token's heads), so token t
// of a sequence is row t % page of page table[t / page].
//
// gs_append_kv: the QKV projection's rows in, the rotated query rows out, the
// rotated keys and the values into their slots -- one read and one write of
// every element, 2 to 3 operations on it: the memory rate bounds it.  8192 tokens of 32
// query and 8 key/value heads of 128, bf16: 43.3 us, 4.7 TB/s, where a bare copy reaches
// 6.2; 256 tokens 4.0 us, of which the launch is most.
#include <algorithm>

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
// Host
// ---------------------------------------------------------------------------
// Few tokens: every head of a token at once; many: each thread four heads or more, its
// cosines and sines loaded once for them.  bf16, 32 + 8 + 8 heads of 128: 256 tokens 4.9
// and 6.2 us, 512 5.6 and 6.6, 2048 12.6 and 11.7, 8192 45.7 and 43.5.
void plan_append(AppendArgs& a, int cus) {
  const int n = a.H + 2 * a.HK;
  const int most = 256 / a.units;                        // units <= 256
  a.groups = std::max(1, std::min(a.T <= 2 * cus ? n : (n + 3) / 4, most));
  a.tokens = 256 / (a.units * a.groups);
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
