// The row form of attention over a paged cache: 16 (query, head) rows at a time,
// keys and values from the pages straight into registers.  Shared by the decode
// kernel (gs_paged.hip) and the kernel for ragged batches (gs_chunk.hip).
//
// Every item -- a tile of 16 rows of a sequence, for one key/value head -- is a
// run of units of 128 keys (fp32: 64); the batch's units in order are dealt to
// `parts` workgroups in equal runs, so long and short sequences load them alike.
// A workgroup whose run ends inside an item leaves a partial result; the last of
// an item's workgroups to be done joins them, in the order of the keys.
#pragma once

#include "gs_paged.h"

namespace gs {
namespace {

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

template <int DT>
struct RowShared {
  float o[kPWaves][16][DT + 4];
  float m[kPWaves][16], l[kPWaves][16];
  float red[256][5];
  int64_t first;
  int seq, q0, n, len;
  int last;
};

// The batch's schedule, kept in LDS so that a part is found without the registers
// or the loads: thread t has the sequences from t * run on, run = ceil(B / 256).
struct Schedule {
  int64_t row_at[257];               // row form: units before a thread's sequences; of the batch
  int q0[256], n[256], len[256];     // a thread's first sequence: its only one up to 256
  int64_t sum[kPWaves];
};
// One of a form's sequences from the schedule.
template <bool CHUNK>
__device__ __forceinline__ addr::PagedSeq first_seq(const PagedArgs& a, const Schedule& sd) {
  const int t = threadIdx.x;
  return only_form<CHUNK>(a, addr::PagedSeq{sd.q0[t], sd.n[t], sd.len[t]});
}

// Each thread's own entries: no barrier between writing and reading them.
__device__ __forceinline__ void load_schedule(const PagedArgs& a, Schedule& sd) {
  const int tid = threadIdx.x;
  const int run = (a.B + 255) >> 8;
  addr::PagedSeq sq{0, 0, 0};
  if (tid * run < a.B) sq = any_seq(a, tid * run);
  sd.q0[tid] = sq.q0;
  sd.n[tid] = sq.n;
  sd.len[tid] = sq.len;
}

template <bool BF16, int DT>
__device__ __forceinline__ void row_scan(const PagedArgs& a, Schedule& sd) {
  constexpr int kUnit = PagedForm<BF16, DT>::kBlock * kPWaves;
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int run = (a.B + 255) >> 8;
  const int s0 = min(tid * run, a.B), s1 = min(s0 + run, a.B);
  int64_t mine = addr::paged_seq_units(first_seq<false>(a, sd), a.G, a.window, kUnit);
  for (int s = s0 + 1; s < s1; ++s) mine += addr::paged_seq_units(seq_of_form<false>(a, s), a.G, a.window, kUnit);
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t up = __shfl_up(incl, d, 64);
    if (l >= d) incl += up;
  }
  if (l == 63) sd.sum[wave] = incl;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPWaves; ++w)
    if (w < wave) incl += sd.sum[w];
  sd.row_at[tid] = incl - mine;
  if (tid == 255) sd.row_at[256] = incl;
  __syncthreads();
}

// A row of the result from its sums.
template <bool BF16>
__device__ __forceinline__ void row_store(const PagedArgs& a, int64_t tok, int head, int d, f32x4 acc, float M, float L) {
  if (d >= a.D) return;
  const f32x4 x = L == 0.f ? f32x4{0, 0, 0, 0} : acc * (1.0f / L);
  const int64_t e = tok * a.o_ts + static_cast<int64_t>(head) * a.o_hs + d;
  if constexpr (BF16) {
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + e) = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
  } else {
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + e) = x;
  }
  if (a.lse != nullptr && d == 0)
    a.lse[tok * a.H + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

// Partial results are written and read by workgroups of different XCDs, whose L2s
// do not see each other's lines: agent-scope accesses, which go through to memory
// (writing an L2 back at a release instead took 30 us of a decode call's 114).
__device__ __forceinline__ void put_partial(float* p, f32x4 x) {
  uint64_t* w = reinterpret_cast<uint64_t*>(p);
  const u32x4 b = __builtin_bit_cast(u32x4, x);
  __hip_atomic_store(w, b[0] | (static_cast<uint64_t>(b[1]) << 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(w + 1, b[2] | (static_cast<uint64_t>(b[3]) << 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put_partial(float* p, float x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4 get_partial4(const float* p) {
  const uint64_t* w = reinterpret_cast<const uint64_t*>(p);
  const uint64_t x = __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint64_t y = __hip_atomic_load(w + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return __builtin_bit_cast(f32x4, u32x4{static_cast<uint32_t>(x), static_cast<uint32_t>(x >> 32), static_cast<uint32_t>(y),
                                         static_cast<uint32_t>(y >> 32)});
}
__device__ __forceinline__ float get_partial(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Counts one of an item's workgroups that is done; true in every thread of the
// last one.  Every thread's partial results have reached memory when the counter
// moves (stores that were waited for), so the last one reads all of them.  The
// counter ends at zero.
__device__ __forceinline__ bool last_to_arrive(int* count, int of, int& shared) {
  mem_fence_compiler();
  __builtin_amdgcn_s_waitcnt(wait_vm(0));
  __syncthreads();
  if (threadIdx.x == 0) {
    const int n = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    shared = n == of - 1;
    if (n == of - 1) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  mem_fence_compiler();
  return shared != 0;
}

// Joins an item's partial results, parts first .. last of head h: the maxima of 8
// rows at a time through LDS, then each thread 4 columns of a row of every
// groups-th part.
template <bool BF16, int DT>
__device__ __forceinline__ void row_join(const PagedArgs& a, const addr::PagedSeq& sq, int j, int nrow, int h, int first,
                                         int last, RowShared<DT>& sh) {
  constexpr int kRows = 8;                           // kRows * np maxima fit into sh.o: np <= kMostParts
  const int64_t slot_floats = addr::paged_partial_floats(DT);
  const int tid = threadIdx.x;
  const int np = last - first + 1;
  float* sm = &sh.o[0][0][0];                        // [np][8]
  const auto slot_of = [&](int p) {
    return a.ws + ((static_cast<int64_t>(first + p) * a.HK + h) * 2 + (p == 0 ? 1 : 0)) * slot_floats;
  };
  for (int r0 = 0; r0 < nrow; r0 += kRows) {
    const int nr = min(kRows, nrow - r0);
    __syncthreads();
    for (int x = tid; x < np * kRows; x += 256) {
      const int q = x & (kRows - 1);
      sm[x] = q < nr ? get_partial(slot_of(x / kRows) + 16 * DT + r0 + q) : -INFINITY;
    }
    __syncthreads();
    const int items = nr * (DT / 4);                 // (row, 4 columns)
    const int groups = max(1, 256 / items);
    for (int base = 0; base < items; base += 256) {
      const int x = base + (groups > 1 ? tid % items : tid);
      const int g = groups > 1 ? tid / items : 0;
      const bool in = x < items && g < groups;
      const int q = in ? x / (DT / 4) : 0, d = in ? (x - q * (DT / 4)) * 4 : 0;
      float M = -INFINITY, L = 0.f;
      f32x4 acc = {0, 0, 0, 0};
      if (in) {
        for (int p = 0; p < np; ++p) M = fmaxf(M, sm[p * kRows + q]);
        const float ms = M == -INFINITY ? 0.f : M;
        // 16 parts' loads in flight at a time; past the last they repeat it with weight 0
        for (int p0 = g; p0 < np; p0 += 16 * groups) {
          f32x4 x[16];
          float lx[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float* sl = slot_of(min(p0 + k * groups, np - 1));
            x[k] = get_partial4(sl + (r0 + q) * DT + d);
            lx[k] = get_partial(sl + 16 * DT + 16 + r0 + q);
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int p = p0 + k * groups;
            const float f = p < np ? __builtin_amdgcn_exp2f(sm[min(p, np - 1) * kRows + q] - ms) : 0.f;
            L += f * lx[k];
            acc += f * x[k];
          }
        }
      }
      if (groups > 1) {
        sh.red[tid][0] = L;
#pragma unroll
        for (int i = 0; i < 4; ++i) sh.red[tid][1 + i] = acc[i];
        __syncthreads();
        if (in && g == 0)
          for (int k = 1; k < groups; ++k) {
            L += sh.red[k * items + tid][0];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += sh.red[k * items + tid][1 + i];
          }
      }
      if (in && g == 0) {
        const int64_t rr = static_cast<int64_t>(j) * 16 + r0 + q;
        const int qi = static_cast<int>(rr / a.G);
        row_store<BF16>(a, sq.q0 + qi, h * a.G + static_cast<int>(rr - static_cast<int64_t>(qi) * a.G), d, acc, M, L);
      }
    }
  }
}

// Part `part` of `parts` of the batch, for key/value head h.
template <bool BF16, int DT>
__device__ __forceinline__ void row_part(const PagedArgs& a, const Schedule& sd, int part, int parts, int h, RowShared<DT>& sh) {
  using F = PagedForm<BF16, DT>;
  constexpr int kUnit = F::kBlock * kPWaves;
  constexpr int kOC = F::kVN * F::kVW;               // O^T tiles of 16 columns
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int lq = l & 15, lg = l >> 4;
  const int64_t U = sd.row_at[256];
  const int64_t u0 = addr::paged_part_lo(U, parts, part), u1 = addr::paged_part_lo(U, parts, part + 1);
  __syncthreads();
  if (sd.row_at[tid] <= u0 && u0 < sd.row_at[tid + 1]) {
    // the sequence that unit u0 is of
    const int run = (a.B + 255) >> 8;
    int s = tid * run;
    int64_t at = sd.row_at[tid];
    addr::PagedSeq sq = first_seq<false>(a, sd);
    for (;;) {
      const int64_t n = addr::paged_seq_units(sq, a.G, a.window, kUnit);
      if (u0 < at + n) break;
      at += n;
      sq = seq_of_form<false>(a, ++s);
    }
    sh.seq = s;
    sh.first = at;
    sh.q0 = sq.q0;
    sh.n = sq.n;
    sh.len = sq.len;
  }
  __syncthreads();
  const auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  int s = uni(sh.seq);
  int64_t base = sh.first;                           // unit the sequence starts at
  addr::PagedSeq sq{uni(sh.q0), uni(sh.n), uni(sh.len)};
  int64_t u = u0;
  while (u < u1) {
    const int64_t su = addr::paged_seq_units(sq, a.G, a.window, kUnit);
    if (base + su <= u) {
      base += su;
      ++s;
      sq = seq_of_form<false>(a, s);
      continue;
    }
    const int nu = addr::paged_tile_units(sq, a.G, a.window, kUnit);
    int j = 0;
    if (sq.n * static_cast<int64_t>(a.G) > 16) j = static_cast<int>((u - base) / nu);
    const int64_t item = base + static_cast<int64_t>(j) * nu;       // the item's first unit
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


    // ---- the four waves' results, joined ------------------------------------------
    lsum += __shfl_xor(lsum, 16, 64);
    lsum += __shfl_xor(lsum, 32, 64);
    if (lg == 0) {
      sh.m[wave][lq] = m;
      sh.l[wave][lq] = lsum;
    }
#pragma unroll
    for (int n = 0; n < F::kVN; ++n)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        // O^T row 4 lg + v of tile (n, c): column 16 kVW n + kVW (4 lg + v) + c
        const int d = n * 16 * F::kVW + F::kVW * (4 * lg + v);
#pragma unroll
        for (int c = 0; c < F::kVW; c += 4)
          *reinterpret_cast<f32x4*>(&sh.o[wave][lq][d + c]) =
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
      float M = sh.m[0][q];
#pragma unroll
      for (int w = 1; w < kPWaves; ++w) M = fmaxf(M, sh.m[w][q]);
      const float ms = M == -INFINITY ? 0.f : M;
      float L = 0.f;
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kPWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(sh.m[w][q] - ms);
        L += f * sh.l[w][q];
        acc += f * *reinterpret_cast<const f32x4*>(&sh.o[w][q][d]);
      }
      if (!whole) {
        put_partial(slot + q * DT + d, acc);
        if (d == 0) {
          put_partial(slot + 16 * DT + q, M);
          put_partial(slot + 16 * DT + 16 + q, L);
        }
      } else {
        const int64_t rr = static_cast<int64_t>(j) * 16 + q;
        const int qo = static_cast<int>(rr / a.G);
        row_store<BF16>(a, sq.q0 + qo, h * a.G + static_cast<int>(rr - static_cast<int64_t>(qo) * a.G), d, acc, M, L);
      }
    }
    if (!whole) {
      const int first = addr::paged_part_of(U, parts, item), last = addr::paged_part_of(U, parts, item + nu - 1);
      if (last_to_arrive(a.row_count + static_cast<int64_t>(last) * a.HK + h, last - first + 1, sh.last))
        row_join<BF16, DT>(a, sq, j, nrow, h, first, last, sh);
    }
    __syncthreads();
    u = item + w1;
  }
}

}  // namespace
}  // namespace gs
