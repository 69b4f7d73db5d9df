// What the kernels that store rows into a paged cache share (gs_append.hip, gs_append_rows.hip).
#pragma once

#include "gs_paged.h"

namespace gs {
namespace {

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

}  // namespace
}  // namespace gs
