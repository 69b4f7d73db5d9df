// The row form of attention over a paged cache: 16 (query, head) rows at a time,
// keys and values from the pages straight into registers.  Shared by the decode
// kernel (gs_paged.hip) and the kernel for ragged batches (gs_chunk.hip).
//
// An item is a tile of 16 rows of a sequence for one key/value head, a run of units
// of 128 keys (fp32: 64).  A workgroup has one item, or one part of an item of more
// units than a workgroup's equal share.  A part leaves a partial result; the last of an
// item's workgroups to be done joins them, in the order of the keys.  The longest parts
// start first: 110 us against 117 for 256 sequences of 16 .. 2047 keys (4 key/value
// heads of 128, bf16).  Equal runs of the batch's units, cut wherever they end, cost two
// joins a workgroup and took 114.
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
  int last;
};

// The batch's schedule in LDS: thread t has the sequences from t * run on, run =
// ceil(B / 256).
struct Schedule {
  int q0[256], n[256], len[256];     // a thread's first sequence: its only one up to 256
  int64_t sum[kPWaves];
  uint64_t lo[kPWaves], hi[kPWaves];
  int slots[kPWaves];
  int found[8];
};
// The thread's first sequence as a form sees it.
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

// One part of the row form's work.
struct RowItem {
  int s, j, part, nparts, slot;      // slot: of the item's first partial result, or -1
  int units;                         // of the item
  addr::PagedSeq sq;
};

// The r-th part of the batch for one head, in order of sequences, tiles and parts; s <
// 0: there is none.  Every thread of a workgroup of 256 calls it, after load_schedule.
template <bool BF16, int DT>
__device__ __forceinline__ RowItem find_row(const PagedArgs& a, Schedule& sd, int r) {
  constexpr int kUnit = PagedForm<BF16, DT>::kBlock * kPWaves;
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int run = (a.B + 255) >> 8;
  const int s0 = min(tid * run, a.B), s1 = min(s0 + run, a.B);
  const addr::PagedSeq first = first_seq<false>(a, sd);
  addr::PagedSeq sq = first;
  int64_t U = 0;
  for (int s = s0; s < s1; ++s) {
    if (s > s0) sq = seq_of_form<false>(a, s);
    U += addr::paged_seq_units(sq, a.G, a.window, kUnit);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) U += __shfl_xor(U, d, 64);
  if (l == 0) sd.sum[wave] = U;
  if (tid == 0) sd.found[0] = -1;
  __syncthreads();
  U = 0;
#pragma unroll
  for (int w = 0; w < kPWaves; ++w) U += sd.sum[w];
  const int most = addr::row_part_units(U, a.HK, a.row_wgs);
  const uint32_t magic = addr::div_magic(most);
  int parts = 0, slots = 0, longest = 0;
  sq = first;
  for (int s = s0; s < s1; ++s) {
    if (s > s0) sq = seq_of_form<false>(a, s);
    const int nt = addr::paged_tiles(sq, a.G);
    const int nu = addr::paged_tile_units(sq, a.G, a.window, kUnit);
    const int np = addr::row_parts(nu, most, magic);
    parts += nt * np;
    slots += np > 1 ? nt * np : 0;
    longest = max(longest, np > 1 ? most : nu);
  }
  // Order: by length, in eight classes, the longest first; within one by sequence.
  // Eight 16-bit counts in two words; too many parts for them, one class.
  const bool classes = a.row_parts < 65536;
  uint32_t cls, rest;
  addr::div_by(static_cast<uint32_t>(8 * (most - longest)), static_cast<uint32_t>(most), magic, cls, rest);
  cls = classes ? min(cls, 7u) : 0;
  const uint64_t one = static_cast<uint64_t>(parts) << (classes ? 16 * (cls & 3) : 0);
  uint64_t lo = cls < 4 ? one : 0, hi = cls < 4 ? 0 : one;
  int sl = slots;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t u = __shfl_up(lo, d, 64), v = __shfl_up(hi, d, 64);
    const int w = __shfl_up(sl, d, 64);
    if (l >= d) {
      lo += u;
      hi += v;
      sl += w;
    }
  }
  if (l == 63) {
    sd.lo[wave] = lo;
    sd.hi[wave] = hi;
    sd.slots[wave] = sl;
  }
  __syncthreads();
  uint64_t all_lo = 0, all_hi = 0;
  sl -= slots;
#pragma unroll
  for (int w = 0; w < kPWaves; ++w) {
    const uint64_t x = sd.lo[w], y = sd.hi[w];
    all_lo += x;
    all_hi += y;
    if (w < wave) {
      lo += x;
      hi += y;
      sl += sd.slots[w];
    }
  }
  int at;
  if (classes) {
    constexpr uint64_t kOnes = 0x0001000100010001;   // times it: sums of the fields up to each
    const uint64_t to_lo = all_lo * kOnes, to_hi = all_hi * kOnes + (to_lo >> 48) * kOnes;
    const int sh16 = 16 * (cls & 3);
    const uint64_t to = cls < 4 ? to_lo : to_hi, all = cls < 4 ? all_lo : all_hi, own = cls < 4 ? lo : hi;
    at = static_cast<int>(((to >> sh16) & 65535) - ((all >> sh16) & 65535) + ((own >> sh16) & 65535)) - parts;
  } else {
    at = static_cast<int>(lo) - parts;
  }
  if (r >= at && r < at + parts) {
    sq = first;
    for (int s = s0;; ++s) {
      if (s > s0) sq = seq_of_form<false>(a, s);
      const int nt = addr::paged_tiles(sq, a.G);
      const int nu = addr::paged_tile_units(sq, a.G, a.window, kUnit);
      const int np = addr::row_parts(nu, most, magic);
      if (r < at + nt * np) {
        const int x = r - at;
        const int j = np > 1 ? x / np : x;
        sd.found[0] = s;
        sd.found[1] = j;
        sd.found[2] = x - j * np;
        sd.found[3] = np;
        sd.found[4] = np > 1 ? sl + j * np : -1;
        sd.found[5] = sq.q0;
        sd.found[6] = sq.n;
        sd.found[7] = sq.len;
        break;
      }
      at += nt * np;
      sl += np > 1 ? nt * np : 0;
    }
  }
  __syncthreads();
  const int* f = sd.found;
  const auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };   // uniform, and known to be
  RowItem it{u(f[0]), u(f[1]), u(f[2]), u(f[3]), u(f[4]), 0, {u(f[5]), u(f[6]), u(f[7])}};
  it.units = addr::paged_tile_units(it.sq, a.G, a.window, kUnit);
  return it;
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

// Joins an item's np partial results: the maxima of 8 rows at a time through LDS, then
// each thread 4 columns of a row of every groups-th part.
template <bool BF16, int DT>
__device__ __forceinline__ void row_join(const PagedArgs& a, const addr::PagedSeq& sq, int j, int nrow, int h,
                                         const float* first, int np, RowShared<DT>& sh) {
  constexpr int kRows = 8;                           // kRows * np maxima fit into sh.o: np <= addr::kMostParts
  const int tid = threadIdx.x;
  float* sm = &sh.o[0][0][0];                        // [np][8]
  const auto slot_of = [&](int p) { return first + p * addr::paged_partial_floats(DT); };
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

// One part of an item, for key/value head h.
template <bool BF16, int DT>
__device__ __forceinline__ void row_part(const PagedArgs& a, const RowItem& it, int h, RowShared<DT>& sh) {
  using F = PagedForm<BF16, DT>;
  constexpr int kOC = F::kVN * F::kVW;               // O^T tiles of 16 columns
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int lq = l & 15, lg = l >> 4;
  const int s = it.s, j = it.j;
  const addr::PagedSeq& sq = it.sq;
  const addr::PagedTile tile = addr::paged_tile(sq, a.G, a.window, j);
  int w0 = 0, w1 = it.units;
  if (it.nparts > 1) addr::chunk_part_range(it.units, it.part, it.nparts, w0, w1);

  // ---- the lane's query row ---------------------------------------------------------
  const int64_t rows = static_cast<int64_t>(sq.n) * a.G;
  const int64_t r = static_cast<int64_t>(j) * 16 + lq;
  const bool live = r < rows;
  int qi = tile.i0, qh = h * a.G;
  if (live) {
    if (rows <= 16) {                                // the one tile: small numbers
      uint32_t x, y;
      addr::div_by(lq, a.G, a.g_magic, x, y);
      qi = static_cast<int>(x);
      qh += static_cast<int>(y);
    } else {
      qi = static_cast<int>(r / a.G);
      qh += static_cast<int>(r - static_cast<int64_t>(qi) * a.G);
    }
  }
  const int hi = live ? sq.len - sq.n + qi + 1 : 0;  // sees [lo, hi)
  const int lo = a.window > 0 ? hi - a.window : 0;
  const int64_t qe = static_cast<int64_t>(sq.q0 + qi) * a.q_ts + static_cast<int64_t>(qh) * a.q_hs;
  constexpr int kVec = 16 / F::kES;
  u32x4 qf[F::kSteps];
#pragma unroll
  for (int st = 0; st < F::kSteps; ++st) {
    const int d = kVec * (4 * st + lg);
    const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.q) + (qe + (d < a.D ? d : 0)) * F::kES);
    qf[st] = live && d < a.D ? x : u32x4{0, 0, 0, 0};
  }
  float m = -INFINITY, lsum = 0.f;
  f32x4 o[kOC];
#pragma unroll
  for (int c = 0; c < kOC; ++c) o[c] = f32x4{0, 0, 0, 0};

  // ---- its keys ---------------------------------------------------------------------
  const int nblk = (tile.ve - tile.first + F::kBlock - 1) / F::kBlock;
  const int b_end = min(w1 * kPWaves, nblk);
  const int32_t* trow = a.table + static_cast<int64_t>(s) * a.ld_table;
  // first keys of the 8 that the lane's K rows and its V rows are of
  const int k_oct = BF16 ? 8 * (lq >> 2) : 8 * (lq >> 3);
  const int v_oct = BF16 ? 8 * lg : 8 * (lg >> 1);
  const int k_in = BF16 ? (lq & 3) : (lq & 7);       // K row within them (+ 4 for tile 1)
  const int v_in = BF16 ? 0 : 4 * (lg & 1);
  const char* k_head = static_cast<const char*>(a.k) + static_cast<int64_t>(h) * a.k_hs * F::kES;
  const char* v_head = static_cast<const char*>(a.v) + static_cast<int64_t>(h) * a.v_hs * F::kES;
  struct Ids {
    int k, v;
    uint32_t k_row, v_row;
  };
  const auto ids_of = [&](int b) {
    const int tb = tile.first + b * F::kBlock;
    uint32_t kp, kr, vp, vr;
    addr::div_by(static_cast<uint32_t>(addr::paged_octet(tb + k_oct, tile.ve)) >> 3, a.page_octets, a.page_magic, kp, kr);
    addr::div_by(static_cast<uint32_t>(addr::paged_octet(tb + v_oct, tile.ve)) >> 3, a.page_octets, a.page_magic, vp, vr);
    return Ids{trow[kp], trow[vp], kr * 8 + k_in, vr * 8 + v_in};
  };
  const auto load = [&](const Ids& id, PagedBlock<BF16, DT>& x) {
    const char* kp = k_head + (addr::paged_page(id.k, a.num_pages) * a.k_ps + id.k_row * a.k_rs) * F::kES;
    const char* vp = v_head + (addr::paged_page(id.v, a.num_pages) * a.v_ps + id.v_row * a.v_rs) * F::kES;
#pragma unroll
    for (int t = 0; t < F::kKT; ++t)
#pragma unroll
      for (int st = 0; st < F::kSteps; ++st) {
        const int d = kVec * (4 * st + lg);
        x.k[t][st] = *reinterpret_cast<const u32x4*>(kp + (4 * t * a.k_rs + (d < a.D ? d : 0)) * F::kES);
      }
#pragma unroll
    for (int t = 0; t < F::kKeys; ++t)
#pragma unroll
      for (int n = 0; n < F::kVN; ++n) {
        const int d = n * 16 * F::kVW + F::kVW * lq;
        x.v[t][n] = *reinterpret_cast<const typename VVec<F::kVW * F::kES>::T*>(vp + (t * a.v_rs + (d < a.D ? d : 0)) * F::kES);
      }
  };
  const int hi_min = sq.len - sq.n + tile.i0 + 1;    // keys below it and from lo_max on: seen by every row
  const int lo_max = a.window > 0 ? sq.len - sq.n + tile.i1 + 1 - a.window : 0;
  const bool pad = DT > a.D;

  const auto step = [&](int b, PagedBlock<BF16, DT>& x) {
    const int tb = tile.first + b * F::kBlock;
    f32x4 sacc[F::kKT];
#pragma unroll
    for (int t = 0; t < F::kKT; ++t) sacc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int st = 0; st < F::kSteps; ++st)
#pragma unroll
      for (int t = 0; t < F::kKT; ++t) {
        u32x4 kx = x.k[t][st];
        if (pad && kVec * (4 * st + lg) >= a.D) kx = u32x4{0, 0, 0, 0};
        if constexpr (BF16) {
          sacc[t] = mfma16_bf16(kx, qf[st], sacc[t]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) sacc[t] = mfma16_f32(__uint_as_float(kx[e]), __uint_as_float(qf[st][e]), sacc[t]);
        }
      }
    float sc[F::kKeys];
#pragma unroll
    for (int i = 0; i < F::kKeys; ++i) sc[i] = sacc[i >> 2][i & 3] * a.scale_log2;
    if (tb + F::kBlock > hi_min || tb < lo_max) {
      const int t0 = tb + F::kKeys * lg;           // the lane's first key
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
    // the reference point follows the maximum once it has grown by 2^8: the sums
    // stay far from their limits, and o is rarely scaled
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx);
      const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);   // m = mn = -inf: nothing summed yet
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
      // probabilities enter the product in bf16 (relative error 2^-8, as the
      // values and the result have); their total stays in fp32
      u32x4 pf;
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
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
  // A block's loads are issued before the one ahead of it is used (one buffer, its keys
  // and its values refilled in turn, and three workgroups a CU: 141 us against 124 for
  // 256 sequences of 16 .. 2047 keys then), and page ids one block before them.
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

  // ---- the four waves' results, joined --------------------------------------------
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
  const int nrow = static_cast<int>(min(static_cast<int64_t>(16), rows - static_cast<int64_t>(j) * 16));
  const int64_t slot0 = static_cast<int64_t>(h) * a.row_slots + it.slot;
  float* first = a.ws + slot0 * addr::paged_partial_floats(DT);
  float* slot = first + it.part * addr::paged_partial_floats(DT);
  for (int x = tid; x < nrow * (DT / 4); x += 256) {
    const int q = x / (DT / 4), d = (x - q * (DT / 4)) * 4;
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
    if (it.nparts > 1) {
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
  if (it.nparts > 1 && last_to_arrive(a.row_count + slot0, it.nparts, sh.last))
    row_join<BF16, DT>(a, sq, j, nrow, h, first, it.nparts, sh);
}

}  // namespace
}  // namespace gs
