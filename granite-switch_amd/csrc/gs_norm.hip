// Residual add between two blocks of a decoder layer, with the norms around it:
//
//   b  = x                                        the block's output
//   b  = b * rsqrt(mean(b^2) + eps) * post_weight (norm after the block, optional)
//   b  = b * act(gate)                            (optional)
//   r' = r + scale * b                            the residual stream
//   y  = r' * rsqrt(mean(r'^2) + eps) * weight    norm before the next block
//
// One pass: a row's values stay in registers between the two sums, so x, r and
// the gate are read once and r' and y written once -- 8 bytes an element in
// bf16 against 2 to 3 operations a byte: the memory rate bounds it.  4144 rows of
// 4096, bf16: 23.4 us, 5.8 TB/s.  Sums and r' are held in fp32; y is taken from the r'
// before its rounding.
#include <hip/hip_runtime.h>

#include "gs_common.h"

namespace gs {
namespace {

struct NormArgs {
  const void* x;
  int64_t ldx;
  const void* r;
  int64_t ldr;
  void* r_out;
  int64_t ldro;
  void* y;
  int64_t ldy;
  const void* weight;
  const void* post;
  const void* gate;
  int64_t gate_row, gate_col;       // element strides; 0: one value for all rows / columns
  int rows, hidden;
  float eps, scale, inv_hidden;
  int w_f32;                        // weight and post are fp32 whatever x is
  int act;
};

__device__ __forceinline__ float gate_value(float g, int act) {
  if (act == GS_GATE_SIGMOID) return 1.0f / (1.0f + expf(-g));
  if (act == GS_GATE_TANH) return tanhf(g);
  return g;
}

template <bool BF16>
struct NormVec;
template <>
struct NormVec<true> {
  static constexpr int N = 8;
};
template <>
struct NormVec<false> {
  static constexpr int N = 4;
};

// N elements from element `e` of p (16-byte aligned), bf16 or fp32.
template <int N, bool BF16>
__device__ __forceinline__ void load_vec(const void* p, int64_t e, float* f) {
  if constexpr (BF16) {
    static_assert(N == 8);
    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4 w = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + e + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) f[i + k] = w[k];
    }
  }
}

template <int N, bool BF16>
__device__ __forceinline__ void store_vec(void* p, int64_t e, const float* f) {
  if constexpr (BF16) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = static_cast<uint32_t>(f32_to_bf16_bits(f[2 * i])) | (static_cast<uint32_t>(f32_to_bf16_bits(f[2 * i + 1])) << 16);
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + e) = w;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<f32x4*>(static_cast<float*>(p) + e + i) = f32x4{f[i], f[i + 1], f[i + 2], f[i + 3]};
  }
}

template <bool BF16>
__device__ __forceinline__ float load_one(const void* p, int64_t e) {
  if constexpr (BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[e]);
  return static_cast<const float*>(p)[e];
}
template <bool BF16>
__device__ __forceinline__ void store_one(void* p, int64_t e, float f) {
  if constexpr (BF16) static_cast<uint16_t*>(p)[e] = f32_to_bf16_bits(f);
  else static_cast<float*>(p)[e] = f;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// Sum over the WAVES waves of a row; `red` is used by one call only.
template <int WAVES>
__device__ __forceinline__ float row_sum(float v, float* red, int wave) {
  v = wave_sum(v);
  if (lane_id() == 0) red[wave] = v;
  lds_barrier();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) v += red[w];
  return v;
}

// WAVES waves to a row, NV vectors of 16 bytes to a lane: the row in registers.
template <bool BF16, bool RF32, int WAVES, int NV>
__global__ __launch_bounds__(64 * WAVES) void residual_norm_kernel(NormArgs a) {
  constexpr int N = NormVec<BF16>::N;
  constexpr int kRowThreads = 64 * WAVES;
  __shared__ float red[2][WAVES];
  const int wave = threadIdx.x >> 6;
  const int row = blockIdx.x;
  const int t = threadIdx.x;
  const int nvec = a.hidden / N;
  float b[NV][N], r[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * kRowThreads + t) * N;
    if (i * kRowThreads + t < nvec) {
      if (a.x != nullptr) load_vec<N, BF16>(a.x, row * a.ldx + e, b[i]);
      load_vec<N, BF16 && !RF32>(a.r, row * a.ldr + e, r[i]);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) b[i][k] = r[i][k] = 0.f;
    }
  }
  float w[NV][N];
  if (NV <= 4) {                                   // the weight row on its way during the sums
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * kRowThreads + t < nvec) {
        if (!BF16 || a.w_f32) load_vec<N, false>(a.weight, (i * kRowThreads + t) * N, w[i]);
        else load_vec<N, BF16>(a.weight, (i * kRowThreads + t) * N, w[i]);
      }
  }
  if (a.x != nullptr) {
    if (a.post != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) ss += b[i][k] * b[i][k];
      const float inv = rsqrtf(row_sum<WAVES>(ss, red[0], wave) * a.inv_hidden + a.eps);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i * kRowThreads + t < nvec) {
          float pw[N];
          if (!BF16 || a.w_f32) load_vec<N, false>(a.post, (i * kRowThreads + t) * N, pw);
          else load_vec<N, BF16>(a.post, (i * kRowThreads + t) * N, pw);
#pragma unroll
          for (int k = 0; k < N; ++k) b[i][k] = b[i][k] * inv * pw[k];
        }
    }
    if (a.gate != nullptr) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i * kRowThreads + t < nvec) {
          const int e = (i * kRowThreads + t) * N;
          float g[N];
          if (a.gate_col == 1) {
            load_vec<N, BF16>(a.gate, row * a.gate_row + e, g);
          } else {
            g[0] = load_one<BF16>(a.gate, row * a.gate_row);
#pragma unroll
            for (int k = 1; k < N; ++k) g[k] = g[0];
          }
#pragma unroll
          for (int k = 0; k < N; ++k) b[i][k] *= gate_value(g[k], a.act);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * kRowThreads + t < nvec) {
#pragma unroll
        for (int k = 0; k < N; ++k) r[i][k] += a.scale * b[i][k];
        store_vec<N, BF16 && !RF32>(a.r_out, row * a.ldro + (i * kRowThreads + t) * N, r[i]);
      }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) ss += r[i][k] * r[i][k];
  const float inv = rsqrtf(row_sum<WAVES>(ss, red[1], wave) * a.inv_hidden + a.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * kRowThreads + t < nvec) {
      const int e = (i * kRowThreads + t) * N;
      if (NV > 4) {
        if (!BF16 || a.w_f32) load_vec<N, false>(a.weight, e, w[i]);
        else load_vec<N, BF16>(a.weight, e, w[i]);
      }
      float o[N];
#pragma unroll
      for (int k = 0; k < N; ++k) o[k] = r[i][k] * inv * w[i][k];
      store_vec<N, BF16>(a.y, row * a.ldy + e, o);
    }
}

// Any hidden size, stride and alignment: one element at a time, 256 threads to
// a row, the row read again for the second sum and for the outputs.
template <bool BF16, bool RF32>
__global__ __launch_bounds__(256) void residual_norm_any_kernel(NormArgs a) {
  __shared__ float red[2][4];
  const int wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const auto wt = [&](const void* p, int e) { return !BF16 || a.w_f32 ? load_one<false>(p, e) : load_one<BF16>(p, e); };
  float post_inv = 1.f;
  if (a.x != nullptr && a.post != nullptr) {
    float ss = 0.f;
    for (int e = threadIdx.x; e < a.hidden; e += 256) {
      const float v = load_one<BF16>(a.x, row * a.ldx + e);
      ss += v * v;
    }
    post_inv = rsqrtf(row_sum<4>(ss, red[0], wave) * a.inv_hidden + a.eps);
  }
  const auto value = [&](int e) {
    float r = load_one<BF16 && !RF32>(a.r, row * a.ldr + e);
    if (a.x != nullptr) {
      float b = load_one<BF16>(a.x, row * a.ldx + e);
      if (a.post != nullptr) b = b * post_inv * wt(a.post, e);
      if (a.gate != nullptr) b *= gate_value(load_one<BF16>(a.gate, row * a.gate_row + e * a.gate_col), a.act);
      r += a.scale * b;
    }
    return r;
  };
  float ss = 0.f;
  for (int e = threadIdx.x; e < a.hidden; e += 256) {
    const float r = value(e);
    ss += r * r;
  }
  const float inv = rsqrtf(row_sum<4>(ss, red[1], wave) * a.inv_hidden + a.eps);
  for (int e = threadIdx.x; e < a.hidden; e += 256) {   // each element is read before it is written: in place works
    const float r = value(e);
    if (a.x != nullptr) store_one<BF16 && !RF32>(a.r_out, row * a.ldro + e, r);
    store_one<BF16>(a.y, row * a.ldy + e, r * inv * wt(a.weight, e));
  }
}

template <bool BF16, bool RF32, int WAVES, int NV>
void launch_norm(const NormArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((residual_norm_kernel<BF16, RF32, WAVES, NV>), dim3(a.rows), dim3(64 * WAVES), 0, st, a);
}

// Four waves to a row of up to 512 vectors, sixteen to a longer one, and where there is
// at most a row for each compute unit.  bf16, four and sixteen waves: 64 x 4096 4.2 and
// 3.5 us, 4144 x 2048 13.5 and 19.5, 4144 x 4096 24.0 and 25.2, 2048 x 12800 47.0 and
// 44.2, 2048 x 16384 58.7 and 52.4.
template <bool BF16, bool RF32>
void launch_norm_type(bool vec, const NormArgs& a, hipStream_t st) {
  const int nvec = a.hidden / NormVec<BF16>::N;
  if (!vec || nvec > 16 * 64 * 8) {
    hipLaunchKernelGGL((residual_norm_any_kernel<BF16, RF32>), dim3(a.rows), dim3(256), 0, st, a);
  } else if (nvec <= 256) {
    launch_norm<BF16, RF32, 4, 1>(a, st);
  } else if (nvec <= 512 && a.rows > device_cus()) {
    launch_norm<BF16, RF32, 4, 2>(a, st);
  } else if (nvec <= 1024) {
    launch_norm<BF16, RF32, 16, 1>(a, st);
  } else if (nvec <= 2048) {
    launch_norm<BF16, RF32, 16, 2>(a, st);
  } else if (nvec <= 4096) {
    launch_norm<BF16, RF32, 16, 4>(a, st);
  } else {
    launch_norm<BF16, RF32, 16, 8>(a, st);
  }
}

// Rows of a matrix in memory, in bytes.
struct Operand {
  const char* name;
  const void* p;
  int64_t rows, ld, cols;
};
// Whether two operands share a byte.  Rows of equal stride may lie side by
// side (column slices of one buffer); others are compared by their spans.
bool overlap(const Operand& a, const Operand& b) {
  if (a.p == nullptr || b.p == nullptr) return false;
  const int64_t d = static_cast<const char*>(b.p) - static_cast<const char*>(a.p);
  if (d >= (a.rows - 1) * a.ld + a.cols || -d >= (b.rows - 1) * b.ld + b.cols) return false;
  if (a.ld != b.ld || a.ld <= 0) return true;
  const int64_t m = ((d % a.ld) + a.ld) % a.ld;      // b's columns start m bytes into a's rows
  return m < a.cols || m + b.cols > a.ld;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_residual_norm(int32_t dtype, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                int32_t residual_dtype, const void* gate, int64_t gate_row_stride,
                                int64_t gate_col_stride, int32_t gate_act, const void* post_weight,
                                const void* weight, int32_t weight_dtype, float eps, float scale, int64_t rows,
                                int32_t hidden, void* residual_out, int64_t ldro, void* y, int64_t ldy, void* stream) {
  const char* who = "gs_residual_norm";
  GS_CHECK_ARG(dtype == GS_DTYPE_BF16 || dtype == GS_DTYPE_FP32, "%s: dtype=%d", who, dtype);
  GS_CHECK_ARG(residual_dtype == dtype || residual_dtype == GS_DTYPE_FP32, "%s: residual_dtype=%d with dtype=%d", who,
               residual_dtype, dtype);
  GS_CHECK_ARG(weight_dtype == dtype || weight_dtype == GS_DTYPE_FP32, "%s: weight_dtype=%d with dtype=%d", who,
               weight_dtype, dtype);
  GS_CHECK_ARG(rows >= 0 && rows < (int64_t(1) << 31) && hidden > 0, "%s: rows=%lld hidden=%d", who, (long long)rows,
               hidden);
  GS_CHECK_ARG(gate_act == GS_GATE_NONE || gate_act == GS_GATE_SIGMOID || gate_act == GS_GATE_TANH, "%s: gate_act=%d",
               who, gate_act);
  GS_CHECK_ARG(eps >= 0.f, "%s: eps=%g", who, static_cast<double>(eps));
  if (rows == 0) return GS_OK;
  GS_CHECK_ARG(residual != nullptr && weight != nullptr && y != nullptr, "%s: residual, weight and y are needed", who);
  GS_CHECK_ARG(x != nullptr || (gate == nullptr && post_weight == nullptr), "%s: a gate or post_weight without x", who);
  GS_CHECK_ARG(x == nullptr || residual_out != nullptr, "%s: x without residual_out", who);
  GS_CHECK_ARG(ldr >= hidden && ldy >= hidden && (x == nullptr || (ldx >= hidden && ldro >= hidden)),
               "%s: ldx=%lld ldr=%lld ldro=%lld ldy=%lld below hidden=%d", who, (long long)ldx, (long long)ldr,
               (long long)ldro, (long long)ldy, hidden);
  GS_CHECK_ARG(gate == nullptr || ((gate_col_stride == 0 || gate_col_stride == 1) &&
                                   (gate_row_stride == 0 || gate_row_stride >= (gate_col_stride ? hidden : 1))),
               "%s: gate strides %lld, %lld", who, (long long)gate_row_stride, (long long)gate_col_stride);
  const bool bf16 = dtype == GS_DTYPE_BF16;
  const int es = bf16 ? 2 : 4, rs = residual_dtype == GS_DTYPE_BF16 ? 2 : 4, ws = weight_dtype == GS_DTYPE_BF16 ? 2 : 4;
  // an output may be x or the residual itself (in place), and shares a byte with nothing else
  const Operand ins[] = {{"x", x, rows, ldx * es, int64_t(hidden) * es},
                         {"residual", residual, rows, ldr * rs, int64_t(hidden) * rs},
                         {"gate", gate, gate_row_stride ? rows : 1, gate_row_stride * es,
                          (gate_col_stride ? hidden : 1) * int64_t(es)},
                         {"weight", weight, 1, int64_t(hidden) * ws, int64_t(hidden) * ws},
                         {"post_weight", post_weight, 1, int64_t(hidden) * ws, int64_t(hidden) * ws}};
  const Operand yo = {"y", y, rows, ldy * es, int64_t(hidden) * es};
  const Operand ro = {"residual_out", x != nullptr ? residual_out : nullptr, rows, ldro * rs, int64_t(hidden) * rs};
  for (const Operand& in : ins) {
    const bool same_y = &in == &ins[0] && x == y && ldx == ldy;
    const bool same_r = &in == &ins[1] && residual == residual_out && ldr == ldro;
    GS_CHECK_ARG(same_y || !overlap(in, yo), "%s: y overlaps %s", who, in.name);
    GS_CHECK_ARG(same_r || !overlap(in, ro), "%s: residual_out overlaps %s", who, in.name);
  }
  GS_CHECK_ARG(!overlap(yo, ro), "%s: y overlaps residual_out", who);
  const int n = bf16 ? 8 : 4;
  bool vec = hidden % n == 0 && aligned16(residual) && ldr % n == 0 && aligned16(y) && ldy % n == 0 && aligned16(weight);
  if (x != nullptr) vec = vec && aligned16(x) && ldx % n == 0 && aligned16(residual_out) && ldro % n == 0;
  if (post_weight != nullptr) vec = vec && aligned16(post_weight);
  if (gate != nullptr && gate_col_stride == 1) vec = vec && aligned16(gate) && gate_row_stride % n == 0;
  NormArgs a{};
  a.x = x;
  a.ldx = ldx;
  a.r = residual;
  a.ldr = ldr;
  a.r_out = residual_out;
  a.ldro = ldro;
  a.y = y;
  a.ldy = ldy;
  a.weight = weight;
  a.post = post_weight;
  a.gate = gate;
  a.gate_row = gate_row_stride;
  a.gate_col = gate_col_stride;
  a.rows = static_cast<int>(rows);
  a.hidden = hidden;
  a.eps = eps;
  a.scale = scale;
  a.inv_hidden = 1.0f / static_cast<float>(hidden);
  a.w_f32 = weight_dtype == GS_DTYPE_FP32;
  a.act = gate_act;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!bf16) launch_norm_type<false, true>(vec, a, st);
  else if (residual_dtype == GS_DTYPE_FP32) launch_norm_type<true, true>(vec, a, st);
  else launch_norm_type<true, false>(vec, a, st);
  GS_CHECK_LAUNCH(who);
  return GS_OK;
}
